// Attention of many tokens per sequence under a score rule, over rows that are in a 16-bit cache.
//
// Token t of a sequence with T tokens and L rows is the query at position i = L - T + t; z_j, out and lse are those of
// decode_rule.cu, over the rows j that the rule lets position i see (shady_score_rule).
#include <type_traits>

#include "rowq.cuh"
#include "rule.cuh"

namespace shady {
namespace pr {

struct Args {
    RuleArgs rule;
    const void *q;
    void *out;
    float *lse;
    const char *k_base, *v_base;
    const uint32_t *page_table;
    uint32_t page_rows, max_pages;
    unsigned long long seq_rows, cache_rows;
    const uint32_t *q_starts, *kv_starts, *kv_lens;
    uint32_t num_seqs, total_q, nkv, nh, G;
};

// One warp per (token, head), the rows one after the other, running maximum and sum in f32.
template <typename T, int HD>
__global__ void __launch_bounds__(128) prefill_rule_kernel(const __grid_constant__ Args a) {
    constexpr int E = HD / 32;
    const uint32_t lane = threadIdx.x & 31;
    const unsigned long long unit = (unsigned long long)blockIdx.x * 4 + (threadIdx.x >> 5);
    const uint32_t tok = (uint32_t)(unit / a.nh), h = (uint32_t)(unit % a.nh);
    if (tok >= min(a.total_q, __ldg(a.q_starts + a.num_seqs))) return;
    const uint32_t seq = warp_find_seq(a.q_starts, a.num_seqs, tok, lane);
    const uint32_t L = __ldg(a.kv_lens + seq), q1 = __ldg(a.q_starts + seq + 1);
    const long long pos = (long long)L - (q1 - tok);
    const uint32_t doc = a.rule.doc ? __ldg(a.rule.doc + tok) : 0u, pre = a.rule.prefix ? min(__ldg(a.rule.prefix + seq), L) : 0u;
    const long long wlo = a.rule.window ? max((long long)doc, pos + 1 - (long long)a.rule.window) : (long long)doc;
    const float slope = a.rule.slopes ? __ldg(a.rule.slopes + h) : 0.f;
    float q[E], o[E], m = -INFINITY, l = 0.f;
    const size_t qo = ((size_t)tok * a.nh + h) * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) { q[e] = to_f32<T>(reinterpret_cast<const T *>(a.q)[qo + e]); o[e] = 0.f; }
    for (uint32_t j = doc; pos >= 0 && j < L; ++j) {
        if (!((long long)j <= pos && (long long)j >= wlo) && j >= pre) continue;
        unsigned long long row;
        if (a.page_table) row = (unsigned long long)__ldg(a.page_table + (size_t)seq * a.max_pages + j / a.page_rows) * a.page_rows + j % a.page_rows;
        else row = (a.kv_starts ? __ldg(a.kv_starts + seq) : seq * a.seq_rows) + j;
        if (row >= a.cache_rows) continue;
        const size_t off = (row * a.nkv + h / a.G) * HD + lane * E;
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) s += q[e] * to_f32<T>(reinterpret_cast<const T *>(a.k_base)[off + e]);
        float z = warp_sum(s) * a.rule.scale;
        if (a.rule.cap > 0.f) z = a.rule.cap * rule_tanh_of_exp(z * a.rule.inv_cap * (2.0f * kRuleLog2e));
        z -= slope * fabsf((float)(pos - (long long)j));
        const float mn = fmaxf(m, z), c = expf(m - mn), p = expf(z - mn);
        l = l * c + p;
        m = mn;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = o[e] * c + p * to_f32<T>(reinterpret_cast<const T *>(a.v_base)[off + e]);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) reinterpret_cast<T *>(a.out)[qo + e] = from_f32<T>(l > 0.f ? o[e] / l : 0.f);
    if (lane == 0 && a.lse) a.lse[(size_t)tok * a.nh + h] = l > 0.f ? m + logf(l) : -INFINITY;
}

}  // namespace pr

int launch_prefill_rule(shady_ctx *ctx, const shady_prefill_params *p, const shady_score_rule *rule, const void *d_q,
                        const shady_kv_cache *cache, uint64_t cache_rows, const uint32_t *d_q_starts, uint32_t total_q,
                        const uint32_t *d_kv_starts, const uint32_t *d_kv_lens, void *d_out, float *d_lse) {
    const std::string w("prefill_rule");
    SHADY_REQUIRE(ctx, p && d_q && cache && d_q_starts && d_kv_lens && d_out, SHADY_ERR_BAD_ARG, w + ": null argument");
    SHADY_REQUIRE(ctx, p->num_kv_heads && p->num_q_heads && p->num_seqs && cache_rows, SHADY_ERR_BAD_ARG, w + ": zero-sized problem");
    SHADY_REQUIRE(ctx, p->num_q_heads % p->num_kv_heads == 0, SHADY_ERR_BAD_ARG, w + ": num_q_heads must be a multiple of num_kv_heads");
    const uint32_t G = p->num_q_heads / p->num_kv_heads;
    SHADY_REQUIRE(ctx, p->head_dim == 128 || p->head_dim == 256, SHADY_ERR_UNSUPPORTED, w + ": head_dim must be 128 or 256");
    SHADY_REQUIRE(ctx, G <= 128 && p->num_q_heads <= 65536, SHADY_ERR_UNSUPPORTED, w + ": at most 128 query heads per kv head");
    SHADY_REQUIRE(ctx, p->dtype == SHADY_F16 || p->dtype == SHADY_BF16, SHADY_ERR_UNSUPPORTED, w + ": dtype must be f16 or bf16");
    SHADY_REQUIRE(ctx, cache->dtype == p->dtype, SHADY_ERR_UNSUPPORTED, w + ": the cache must have the dtype of Q");
    SHADY_REQUIRE(ctx, !cache->d_k_ptrs && !cache->d_v_ptrs, SHADY_ERR_UNSUPPORTED, w + ": pointer-array caches are not supported");
    SHADY_REQUIRE(ctx, cache_rows < 0x7fffff00ull, SHADY_ERR_UNSUPPORTED, w + ": too many cache rows");
    for (const void *ptr : {d_q, (const void *)d_out, (const void *)cache->d_k_base, (const void *)cache->d_v_base})
        SHADY_REQUIRE(ctx, ((uintptr_t)ptr & 15) == 0, SHADY_ERR_BAD_ARG, w + ": tensors must be 16-byte aligned");
    KvAddr kv;
    if (const int st = fill_kv_addr(ctx, cache, p->num_kv_heads, p->head_dim, "prefill_rule", &kv)) return st;
    pr::Args a{};
    if (const int st = fill_rule(ctx, rule, p->head_dim, "prefill_rule", &a.rule)) return st;
    const uint64_t row = (uint64_t)p->num_kv_heads * p->head_dim;
    if (cache->d_page_table) {
        SHADY_REQUIRE(ctx, !d_kv_starts, SHADY_ERR_BAD_ARG, w + ": a paged cache takes no kv_starts");
        SHADY_REQUIRE(ctx, cache_rows % cache->page_rows == 0, SHADY_ERR_BAD_ARG, w + ": cache_rows of a paged cache is pages * page_rows");
    } else if (!d_kv_starts) {
        SHADY_REQUIRE(ctx, cache->seq_stride % row == 0, SHADY_ERR_BAD_ARG, w + ": seq_stride must be a whole number of cache rows");
    }
    if (!total_q) return SHADY_OK;
    a.q = d_q; a.out = d_out; a.lse = d_lse; a.k_base = kv.k_base; a.v_base = kv.v_base;
    a.page_table = kv.page_table; a.page_rows = kv.page_rows; a.max_pages = kv.max_pages;
    a.seq_rows = cache->seq_stride / row; a.cache_rows = cache_rows;
    a.q_starts = d_q_starts; a.kv_starts = d_kv_starts; a.kv_lens = d_kv_lens;
    a.num_seqs = p->num_seqs; a.total_q = total_q; a.nkv = p->num_kv_heads; a.nh = p->num_q_heads; a.G = G;
    const unsigned long long blocks = ((unsigned long long)total_q * a.nh + 3) / 4;
    SHADY_REQUIRE(ctx, blocks <= 0x7fffffffull, SHADY_ERR_UNSUPPORTED, w + ": too many tokens");
    auto go = [&](auto kern) { kern<<<(unsigned)blocks, 128, 0, ctx->stream>>>(a); };
    if (p->dtype == SHADY_F16) {
        if (p->head_dim == 128) go(pr::prefill_rule_kernel<__half, 128>);
        else go(pr::prefill_rule_kernel<__half, 256>);
    } else {
        if (p->head_dim == 128) go(pr::prefill_rule_kernel<__nv_bfloat16, 128>);
        else go(pr::prefill_rule_kernel<__nv_bfloat16, 256>);
    }
    ctx->launches++;
    SHADY_CUDA_OK(ctx, cudaGetLastError());
    return SHADY_OK;
}

}  // namespace shady
