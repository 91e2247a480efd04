"""Attention under a score rule, one new token per sequence and many, against 64-bit references (bounds in ``_rule_ref``)."""
import math

import numpy as np
import pytest
import torch

from _rule_ref import attend
from _util import TORCH_DT
from shady_thinker_b200 import ops
from shady_thinker_b200._lib import BF16, F16, F32, ShadyError
from test_gpu_rowq import Cache, dev_u32

pytestmark = pytest.mark.gpu
NONE = 0xFFFFFFFF   # a first visible row behind every row


class Rows16:
    """K and V rows of sequences of the given lengths in a 16-bit cache; every row nobody owns holds NaN.  kind: 'stride',
    'ptrs', 'packed' or 'paged'."""

    def __init__(self, lens, nkv, hd, dt, kind, page_rows=16, seed=0):
        g = torch.Generator().manual_seed(seed + sum(lens))
        t, S = TORCH_DT[dt], len(lens)
        self.kv = [[torch.randn(L, nkv, hd, generator=g).to(t) for L in lens] for _ in range(2)]
        self.kv_starts = None
        nan = float("nan")
        if kind == "paged":
            need = [(L + page_rows - 1) // page_rows for L in lens]
            pages = sum(need) + 2
            order = torch.randperm(pages, generator=g)
            table = torch.full((S, max(need + [1])), pages - 1, dtype=torch.int32)
            pools = [torch.full((pages, page_rows, nkv, hd), nan, dtype=t) for _ in range(2)]
            at = 0
            for s, n in enumerate(need):
                ids = order[at:at + n]
                at += n
                table[s, :n] = ids.to(torch.int32)
                for i in range(2):
                    for p in range(n):
                        rows = self.kv[i][s][p * page_rows:(p + 1) * page_rows]
                        pools[i][ids[p], :rows.shape[0]] = rows
            self.keep = [p.cuda() for p in pools] + [table.cuda()]
            self.view = ops.KvCacheView(dt, self.keep[0], self.keep[1], 0, None, None, self.keep[2], page_rows, table.shape[1])
            self.rows = pages * page_rows
        elif kind == "packed":
            gap = 3
            starts = [gap + sum(lens[:s]) + gap * s for s in range(S)]
            self.rows = starts[-1] + lens[-1] + gap
            flat = [torch.full((self.rows, nkv, hd), nan, dtype=t) for _ in range(2)]
            for i in range(2):
                for s, L in enumerate(lens):
                    flat[i][starts[s]:starts[s] + L] = self.kv[i][s]
            self.keep = [f.cuda() for f in flat]
            self.kv_starts = dev_u32(starts)
            self.view = ops.KvCacheView(dt, self.keep[0], self.keep[1], 0)
        else:
            cap = max(lens + [1]) + 5
            full = [torch.full((S, cap, nkv, hd), nan, dtype=t) for _ in range(2)]
            for i in range(2):
                for s, L in enumerate(lens):
                    full[i][s, :L] = self.kv[i][s]
            self.keep = [f.cuda() for f in full]
            self.rows = S * cap
            if kind == "ptrs":
                ptrs = [torch.tensor([f[s].data_ptr() for s in range(S)], dtype=torch.int64).cuda() for f in self.keep]
                self.keep += ptrs
                self.view = ops.KvCacheView(dt, k_ptrs=ptrs[0], v_ptrs=ptrs[1])
            else:
                self.view = ops.KvCacheView(dt, self.keep[0], self.keep[1], cap * nkv * hd)

    def values(self, s):
        return self.kv[0][s].double(), self.kv[1][s].double()


class RowsQ(Cache):
    def __init__(self, lens, nkv, hd, page_rows=0, seed=0, spread=1.0):
        super().__init__(lens, nkv, hd, page_rows, seed)
        g = torch.Generator().manual_seed(seed + 5)
        self.lens = lens
        for s, L in enumerate(lens):
            if L:
                self.fill(s, [torch.randn(L, nkv, hd, generator=g) * torch.exp(spread * torch.randn(L, nkv, 1, generator=g)) for _ in range(2)])

    def held(self):
        out = []
        for s, L in enumerate(self.lens):
            k, v = self.values(s, L)
            out.append((k.double(), v.double()))
        return out


def workspace(gpu, hd, nkv, nh, S):
    kw = dict(head_dim=hd, num_kv_heads=nkv, num_q_heads=nh, num_seqs=S)
    n = ops.decode_rule_workspace_size(gpu, **kw)
    ws = torch.full((n,), 0xAB, dtype=torch.uint8, device="cuda")
    ops.decode_rule_workspace_init(gpu, ws, n, **kw)
    return ws, n


def make_rule(rule, nh, lens):
    """(ops.ScoreRule, per-sequence dicts of the reference's arguments without the slope, slopes)."""
    r = dict(rule)
    slopes = [2.0 ** (-8 * (h + 1) / nh) * r["bias"] for h in range(nh)] if r.get("bias") else [0.0] * nh
    pre, docs = r.get("prefix"), r.get("docs")
    obj = ops.ScoreRule(scale=r.get("scale", 0.0), cap=r.get("cap", 0.0), window=r.get("window", 0),
                        slopes=torch.tensor(slopes).cuda() if r.get("bias") else None,
                        prefix_lens=dev_u32([pre] * len(lens)) if pre is not None else None,
                        doc_start=dev_u32(docs) if docs is not None else None)
    base = dict(scale=obj.scale, cap=obj.cap, window=obj.window)
    return obj, [dict(base, prefix=min(pre or 0, L)) for L in lens], [float(torch.tensor(s)) for s in slopes]


def check_decode(gpu, cache, values, lens, nkv, G, hd, q_dt, out_dt, wt, rule, seed=1, ws=None):
    S, nh = len(lens), nkv * G
    g = torch.Generator().manual_seed(seed)
    q = (2 * torch.randn(S, nh, hd, generator=g)).to(TORCH_DT[q_dt])
    obj, kws, slopes = make_rule(rule, nh, lens)
    out = torch.full((S, nh, hd), float("nan"), dtype=TORCH_DT[out_dt], device="cuda")
    lse = torch.full((S, nh), float("nan"), device="cuda")
    ws, n = ws or workspace(gpu, hd, nkv, nh, S)
    qd, ld = q.cuda(), dev_u32(lens)
    call = lambda: ops.attn_decode_rule(gpu, q=qd, cache=cache.view, seq_lens=ld, out=out, lse=lse, rule=obj, head_dim=hd, num_kv_heads=nkv,  # noqa: E731
                                        num_q_heads=nh, num_seqs=S, q_dtype=q_dt, out_dtype=out_dt, workspace=ws, workspace_bytes=n)
    call()
    gpu.synchronize()
    first = out.clone(), lse.clone()
    call()                                   # the workspace is ready again, and the result is the same to the bit
    gpu.synchronize()
    assert torch.equal(first[0], out) and torch.equal(first[1], lse)
    qr = q.to(wt).double()                   # Q is rounded to the cache's type
    o, z = out.cpu().double(), lse.cpu().double()
    docs = rule.get("docs")
    for s, L in enumerate(lens):
        k, v = values(s) if L else (torch.zeros(0, nkv, hd).double(),) * 2
        for h in range(nh):
            want, wl, b, bl = attend(qr[s, h], k[:, h // G], v[:, h // G], L - 1, L, slope=slopes[h], doc=docs[s] if docs else 0, wt=wt,
                                     out_dt=TORCH_DT[out_dt], **kws[s])
            assert bool(((o[s, h] - want).abs() <= b).all()), (s, h, float(((o[s, h] - want).abs() - b).max()))
            assert z[s, h] == wl if wl == -math.inf else abs(float(z[s, h]) - wl) <= bl, (s, h, float(z[s, h]), wl, bl)


RULES = [
    {},
    dict(cap=50.0),
    dict(cap=5.0, bias=1.0),
    dict(window=1),
    dict(window=33, prefix=4),
    dict(window=100, prefix=70, cap=30.0),
    dict(scale=0.3, bias=-0.01),
]


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("dt,kind", [(F16, "stride"), (BF16, "paged"), (BF16, "ptrs")])
def test_decode_16_bit(gpu_ctx, dt, kind, rule):
    lens = [1, 0, 16, 17, 515, 130]
    c = Rows16(lens, 2, 128, dt, kind, page_rows=48)
    check_decode(gpu_ctx, c, c.values, lens, 2, 4, 128, dt, dt, TORCH_DT[dt], rule)


@pytest.mark.parametrize("hd,nkv,G,kind,pr", [(64, 3, 1, "paged", 16), (256, 1, 7, "stride", 0), (64, 1, 16, "stride", 0), (128, 2, 12, "paged", 64),
                                              (256, 2, 9, "paged", 256), (128, 1, 1, "ptrs", 0)])
def test_decode_16_bit_shapes(gpu_ctx, hd, nkv, G, kind, pr):
    lens = [300, 2, 77]
    for dt, q_dt, out_dt in ((F16, F16, F32), (BF16, F32, F16)):
        c = Rows16(lens, nkv, hd, dt, kind, page_rows=pr or 16)
        check_decode(gpu_ctx, c, c.values, lens, nkv, G, hd, q_dt, out_dt, TORCH_DT[dt], dict(cap=20.0, window=64, prefix=3))


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("hd,nkv,G,pr,q_dt", [(128, 2, 4, 0, BF16), (64, 2, 5, 16, F16), (256, 1, 8, 64, F32), (128, 1, 10, 32, F16)])
def test_decode_row_scaled(gpu_ctx, hd, nkv, G, pr, q_dt, rule):
    lens = [1, 0, 31, 400, 64]
    c = RowsQ(lens, nkv, hd, pr, seed=hd + G)
    held = c.held()
    check_decode(gpu_ctx, c, lambda s: held[s], lens, nkv, G, hd, q_dt, F32, torch.float16, rule)


def test_decode_row_scaled_with_scales_far_apart(gpu_ctx):
    """Row scales over forty powers of two: the weights' reference takes them in, so nothing overflows or vanishes in f16."""
    lens = [200]
    c = RowsQ(lens, 2, 128, 0, seed=3, spread=0.0)
    c.scales[0] *= 0.1
    c.scales[1] *= torch.exp2(torch.randint(-20, 21, c.scales[1].shape, generator=torch.Generator().manual_seed(1)).float()).cuda()
    held = c.held()
    check_decode(gpu_ctx, c, lambda s: held[s], lens, 2, 4, 128, F16, F32, torch.float16, {})


@pytest.mark.parametrize("docs", [[0, 5, 99, NONE], [16, 0, 40, 100]])
def test_decode_document_starts_and_rows_that_see_nothing(gpu_ctx, docs):
    lens = [40, 6, 100, 101]
    c = Rows16(lens, 1, 128, BF16, "paged", page_rows=16)
    for rule in (dict(docs=docs), dict(docs=docs, window=20, prefix=30)):
        check_decode(gpu_ctx, c, c.values, lens, 1, 3, 128, BF16, BF16, torch.bfloat16, rule)


def test_decode_reads_no_row_that_is_not_seen(gpu_ctx):
    """Rows outside the window, and their pages, may hold anything: the pages are gone (table entries point nowhere)."""
    L, pr = 600, 16
    c = RowsQ([L], 1, 64, pr, seed=2)
    held = c.held()
    for p in range(1, (L - 50) // pr):
        c.table[0, p] = 0x7ffffff0
    c.view.page_table = c.table.cuda()
    check_decode(gpu_ctx, c, lambda s: held[s], [L], 1, 4, 64, F16, F16, torch.float16, dict(window=50, prefix=7))
    c16 = Rows16([L], 1, 64, F16, "stride")
    for t in c16.keep[:2]:
        t[0, 8:L - 50] = float("nan")
    check_decode(gpu_ctx, c16, c16.values, [L], 1, 4, 64, F16, F16, torch.float16, dict(window=50, prefix=8))


def test_decode_many_sequences_and_one_long(gpu_ctx):
    g = torch.Generator().manual_seed(0)
    lens = [int(x) for x in torch.randint(0, 90, (150,), generator=g)]
    c = RowsQ(lens, 2, 64, 16, seed=8)
    held = c.held()
    check_decode(gpu_ctx, c, lambda s: held[s], lens, 2, 2, 64, F16, F32, torch.float16, dict(cap=10.0, window=40, prefix=2))
    c = Rows16([40_000], 2, 128, BF16, "stride")
    check_decode(gpu_ctx, c, c.values, [40_000], 2, 8, 128, BF16, F32, torch.bfloat16, dict(cap=30.0))


def test_decode_captured_launch_serves_growing_lengths(gpu_ctx):
    """One captured launch, replayed with other lengths in the same device buffer."""
    from shady_thinker_b200.gpu import GpuContext
    nkv, G, hd, S = 2, 4, 128, 3
    nh = nkv * G
    stream = torch.cuda.Stream()
    gpu = GpuContext(0, stream=stream.cuda_stream)
    c = Rows16([500, 500, 500], nkv, hd, F16, "stride")
    q = torch.randn(S, nh, hd, generator=torch.Generator().manual_seed(3)).to(torch.float16)
    with torch.cuda.stream(stream):
        qd, lens = q.cuda(), dev_u32([1, 1, 1])
        out = torch.zeros(S, nh, hd, dtype=torch.float16, device="cuda")
        ws, n = workspace(gpu, hd, nkv, nh, S)
        call = lambda: ops.attn_decode_rule(gpu, q=qd, cache=c.view, seq_lens=lens, out=out, head_dim=hd, num_kv_heads=nkv, num_q_heads=nh,  # noqa: E731
                                            num_seqs=S, q_dtype=F16, out_dtype=F16, workspace=ws, workspace_bytes=n)
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for now in ([0, 500, 37], [1, 2, 300]):
            lens.copy_(dev_u32(now))
            graph.replay()
            stream.synchronize()
            for s, L in enumerate(now):
                k, v = (x[:L] for x in c.values(s))
                for h in range(nh):
                    want, _, b, _ = attend(q[s, h].double(), k[:, h // G], v[:, h // G], L - 1, L, wt=torch.float16, out_dt=torch.float16)
                    assert bool(((out[s, h].cpu().double() - want).abs() <= b).all()), (s, h)
    gpu.synchronize()
    del graph
    gpu.close()


# ---- many tokens ----------------------------------------------------------------------------------------------------

def check_prefill(gpu, rows, values, q_lens, kv_lens, nkv, G, hd, dt, rule, spare=3, seed=1, heads=None):
    S, nh, n, t = len(q_lens), nkv * G, sum(q_lens), TORCH_DT[dt]
    g = torch.Generator().manual_seed(seed)
    q = (2 * torch.randn(n + spare, nh, hd, generator=g)).to(t)
    q[n:] = float("nan")
    starts = [0] + [int(x) for x in np.cumsum(q_lens)]
    r = dict(rule)
    if r.get("docs") is not None:
        r["docs"] = list(r["docs"]) + [0] * spare
    obj, kws, slopes = make_rule(r, nh, kv_lens)
    out = torch.full((n + spare, nh, hd), 7.0, dtype=t, device="cuda")
    lse = torch.full((n + spare, nh), 7.0, device="cuda")
    ops.attn_prefill_rule(gpu, q=q.cuda(), cache=rows.view, cache_rows=rows.rows, q_starts=dev_u32(starts), kv_starts=rows.kv_starts,
                          kv_lens=dev_u32(kv_lens), out=out, lse=lse, rule=obj, head_dim=hd, num_kv_heads=nkv, num_q_heads=nh, num_seqs=S,
                          total_q=n + spare, dtype=dt)
    gpu.synchronize()
    o, z = out.cpu().double(), lse.cpu().double()
    assert bool((o[n:] == 7.0).all()) and bool((z[n:] == 7.0).all())
    for s in range(S):
        k, v = values(s)
        step = max(1, q_lens[s] // 40)
        for i in sorted(set(range(0, q_lens[s], step)) | {q_lens[s] - 1, max(0, q_lens[s] - 2)} if q_lens[s] else []):
            tok, pos = starts[s] + i, kv_lens[s] - q_lens[s] + i
            for h in heads or range(nh):
                want, wl, b, bl = attend(q[tok, h].double(), k[:, h // G], v[:, h // G], pos, kv_lens[s], slope=slopes[h],
                                         doc=r["docs"][tok] if r.get("docs") is not None else 0, wt=t, out_dt=t, **kws[s])
                # a weight may lie up to 2^8 above the reference of its row's maximum: same relative rounding
                assert bool(((o[tok, h] - want).abs() <= b).all()), (s, i, h, float(((o[tok, h] - want).abs() - b).max()))
                assert z[tok, h] == wl if wl == -math.inf else abs(float(z[tok, h]) - wl) <= bl, (s, i, h, float(z[tok, h]), wl)


PREFILL_RULES = [{}, dict(cap=50.0), dict(cap=5.0, bias=1.0), dict(window=1), dict(window=150, prefix=4), dict(prefix=10_000), dict(prefix=140, bias=0.5),
                 dict(window=70, prefix=200, cap=30.0), dict(scale=0.25, bias=-0.01)]


@pytest.mark.parametrize("rule", PREFILL_RULES)
@pytest.mark.parametrize("hd,kind", [(128, "packed"), (256, "paged")])
def test_prefill_rules(gpu_ctx, hd, kind, rule):
    q_lens, kv_lens = [300, 1, 0, 129], [300, 200, 64, 515]
    c = Rows16(kv_lens, 2, hd, BF16, kind, page_rows=16)
    check_prefill(gpu_ctx, c, c.values, q_lens, kv_lens, 2, 2, hd, BF16, rule)


@pytest.mark.parametrize("hd,nkv,G,kind,pr,dt", [(128, 1, 1, "stride", 0, F16), (128, 2, 7, "paged", 48, F16), (128, 1, 128, "packed", 0, BF16),
                                                 (256, 1, 3, "stride", 0, BF16), (256, 2, 16, "paged", 128, F16), (128, 3, 5, "paged", 256, BF16),
                                                 (256, 1, 65, "packed", 0, F16)])
def test_prefill_shapes(gpu_ctx, hd, nkv, G, kind, pr, dt):
    q_lens, kv_lens = [1, 130, 7], [1, 260, 128]
    c = Rows16(kv_lens, nkv, hd, dt, kind, page_rows=pr or 16)
    check_prefill(gpu_ctx, c, c.values, q_lens, kv_lens, nkv, G, hd, dt, dict(cap=20.0, window=100, prefix=5), heads=sorted({0, nkv * G - 1, nkv * G // 2}))


@pytest.mark.parametrize("hd", [128, 256])
def test_prefill_documents_and_tokens_that_see_nothing(gpu_ctx, hd):
    q_lens, kv_lens = [400, 300], [400, 350]
    docs = [0] * 100 + [100] * 157 + [257] * 140 + [NONE] * 3 + [0] * 20 + [60] * 200 + [NONE] * 80
    c = Rows16(kv_lens, 1, hd, BF16, "packed")
    for rule in (dict(docs=docs), dict(docs=docs, window=40), dict(docs=docs, prefix=120, cap=30.0)):
        check_prefill(gpu_ctx, c, c.values, q_lens, kv_lens, 1, 2, hd, BF16, rule)


def test_prefill_more_tokens_than_rows(gpu_ctx):
    """Tokens in front of the first row see nothing; the last ones see the rows there are."""
    c = Rows16([20, 5], 1, 128, F16, "packed")
    check_prefill(gpu_ctx, c, c.values, [30, 5], [20, 5], 1, 4, 128, F16, {})


@pytest.mark.parametrize("hd,kind", [(128, "packed"), (256, "stride")])
def test_prefill_long(gpu_ctx, hd, kind):
    q_lens, kv_lens = [1500, 40], [5000, 3500]
    c = Rows16(kv_lens, 2, hd, BF16, kind)
    check_prefill(gpu_ctx, c, c.values, q_lens, kv_lens, 2, 4, hd, BF16, dict(cap=40.0), heads=[0, 7])
    check_prefill(gpu_ctx, c, c.values, q_lens, kv_lens, 2, 4, hd, BF16, dict(window=1000, prefix=64), heads=[0, 5])


def test_prefill_equals_the_causal_prefill(gpu_ctx):
    """Without a rule, whole prompts: what shady_attn_prefill computes, within both kernels' roundings of the weights."""
    B, T, nkv, G, hd = 2, 384, 2, 4, 128
    c = Rows16([T] * B, nkv, hd, BF16, "stride")
    cap = T + 5
    q = torch.randn(B * T, nkv * G, hd, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).cuda()
    a, b = torch.empty_like(q), torch.empty_like(q)
    for t in c.keep[:2]:
        t[:, T:] = 0                                     # shady_attn_prefill wants finite rows behind the prompt
    ops.attn_prefill(gpu_ctx, q=q, cache=c.view, out=a, head_dim=hd, num_kv_heads=nkv, num_q_heads=nkv * G, num_seqs=B, seq_len=T, dtype=BF16)
    ops.attn_prefill_rule(gpu_ctx, q=q, cache=c.view, cache_rows=B * cap, q_starts=dev_u32([0, T, 2 * T]), kv_lens=dev_u32([T, T]), out=b,
                          head_dim=hd, num_kv_heads=nkv, num_q_heads=nkv * G, num_seqs=B, total_q=B * T, dtype=BF16)
    gpu_ctx.synchronize()
    # each side: a weight rounding (2^-8 of A) and an output rounding (2^-8 of |out|), |out| and A at most max|v| of the row's mean
    bound = 4 * 2.0 ** -8 * float(c.keep[1].nan_to_num(0).abs().max())
    assert float((a.float() - b.float()).abs().max()) <= bound


def test_prompt_chunk_and_decode_over_one_cache(gpu_ctx):
    """The operators as they are used together: a prompt is appended and attends to the stored rows, its next chunk
    attends to rows read back from the cache, and a decode step attends to the cache itself; every output is that of
    one reference over the values that the cache holds."""
    nkv, G, hd, dt, S = 2, 4, 128, BF16, 2
    nh, t = nkv * G, torch.bfloat16
    first, chunk = [70, 33], [40, 90]
    total = [a + b for a, b in zip(first, chunk)]
    rule = dict(cap=30.0, window=60, prefix=4)
    g = torch.Generator().manual_seed(6)
    cache = Cache([n + 1 for n in total], nkv, hd, 16)
    w = (torch.randn(2, hd, generator=g) * 0.1).to(t)
    obj, kws, _ = make_rule(rule, nh, total)
    got = []

    def append(counts, pos):
        n, starts = sum(counts), [0] + [int(x) for x in np.cumsum(counts)]
        q, k, v = (torch.randn(n, h, hd, generator=g).to(t).cuda() for h in (nh, nkv, nkv))
        qo, ko, vo = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        ops.kv_append_rowq(gpu_ctx, q_proj_full=q, k_proj=k, v_proj=v, q_out=qo, q_gate=None, k_out=ko, v_out=vo, cache=cache.view,
                           pos_start=dev_u32(pos), num_heads=nh, num_kv_heads=nkv, head_dim=hd, rope_theta=1e6, rotary_dim=hd, num_seqs=S,
                           tok_start=dev_u32(starts), total_tokens=n, tokens_per_seq=0, in_dtype=dt, q_dtype=dt, has_gate=False,
                           qk_norm_bf16=w.cuda())
        return qo, ko, vo, starts

    def prefill(qo, k, v, starts, kv_starts, kv_lens):
        out = torch.empty_like(qo)
        ops.attn_prefill_rule(gpu_ctx, q=qo, cache=ops.KvCacheView(dt, k, v, 0), cache_rows=k.shape[0], q_starts=dev_u32(starts),
                              kv_starts=dev_u32(kv_starts), kv_lens=dev_u32(kv_lens), out=out, rule=obj, head_dim=hd, num_kv_heads=nkv,
                              num_q_heads=nh, num_seqs=S, total_q=qo.shape[0], dtype=dt)
        return out

    qo, ko, vo, starts = append(first, [0, 0])
    got.append((qo, prefill(qo, ko, vo, starts, starts[:-1], first), starts, first, 16))
    qo, _, _, starts = append(chunk, first)
    kr, vr = (torch.empty(sum(total), nkv, hd, dtype=t, device="cuda") for _ in range(2))
    rows = [0] + [int(x) for x in np.cumsum(total)]
    ops.kv_read_rowq(gpu_ctx, cache=cache.view, k_out=kr, v_out=vr, out_start=dev_u32(rows), total_rows=rows[-1], num_seqs=S, num_kv_heads=nkv,
                     head_dim=hd, out_dtype=dt)
    got.append((qo, prefill(qo, kr, vr, starts, rows[:-1], total), starts, total, 16))
    qo, _, _, starts = append([1, 1], total)
    out = torch.empty_like(qo)
    ws, n = workspace(gpu_ctx, hd, nkv, nh, S)
    after = [x + 1 for x in total]
    ops.attn_decode_rule(gpu_ctx, q=qo, cache=cache.view, seq_lens=dev_u32(after), out=out, rule=obj, head_dim=hd, num_kv_heads=nkv, num_q_heads=nh,
                         num_seqs=S, q_dtype=dt, out_dtype=dt, workspace=ws, workspace_bytes=n)
    got.append((qo, out, starts, after, 8))
    gpu_ctx.synchronize()
    for q, o, st, lens, bits in got:
        for s in range(S):
            k, v = (x.to(t).double() if bits == 16 else x.double() for x in cache.values(s, lens[s]))
            T = st[s + 1] - st[s]
            for i in {0, T // 2, T - 1}:
                for h in (0, nh - 1):
                    want, _, b, _ = attend(q[st[s] + i, h].cpu().double(), k[:, h // G], v[:, h // G], lens[s] - T + i, lens[s],
                                           wt=t if bits == 16 else torch.float16, out_dt=t, **kws[s])
                    assert bool(((o[st[s] + i, h].cpu().double() - want).abs() <= b).all()), (bits, s, i, h)


def test_refusals(gpu_ctx):
    hd, nkv, nh, S = 128, 2, 8, 2
    c = Rows16([20, 20], nkv, hd, F16, "stride")
    cq = RowsQ([20, 20], nkv, hd)
    q = torch.zeros(S, nh, hd, dtype=torch.float16, device="cuda")
    ws, n = workspace(gpu_ctx, hd, nkv, nh, S)
    kw = dict(q=q, cache=c.view, seq_lens=dev_u32([3, 4]), out=q, head_dim=hd, num_kv_heads=nkv, num_q_heads=nh, num_seqs=S, q_dtype=F16, out_dtype=F16,
              workspace=ws, workspace_bytes=n)
    bad = [dict(head_dim=96), dict(num_q_heads=7), dict(num_seqs=0), dict(q_dtype=BF16), dict(out_dtype=4), dict(workspace=None),
           dict(workspace_bytes=n - 1), dict(workspace=ws.data_ptr() + 4), dict(q=q.data_ptr() + 2),
           dict(rule=ops.ScoreRule(scale=-1.0)), dict(rule=ops.ScoreRule(cap=float("inf"))), dict(rule=ops.ScoreRule(cap=-2.0)),
           dict(rule=ops.ScoreRule(scale=float("nan"))), dict(rule=ops.ScoreRule(cap=1e-45)),
           dict(cache=ops.KvCacheView(F32, c.keep[0], c.keep[1], 0)), dict(cache=ops.KvCacheView(F16)),
           dict(cache=ops.KvCacheView(F16, c.keep[0].data_ptr() + 8, c.keep[1], 0))]
    before = gpu_ctx.launch_count
    for b in bad:
        with pytest.raises(ShadyError):
            ops.attn_decode_rule(gpu_ctx, **{**kw, **b})
    p = dict(q=q, cache=c.view, cache_rows=c.rows, q_starts=dev_u32([0, 1, 2]), kv_lens=dev_u32([3, 4]), out=q, head_dim=hd, num_kv_heads=nkv,
             num_q_heads=nh, num_seqs=S, total_q=2, dtype=F16)
    for b in [dict(head_dim=64), dict(num_q_heads=9), dict(num_q_heads=129 * nkv), dict(dtype=F32), dict(dtype=BF16), dict(cache_rows=0),
              dict(cache_rows=1 << 31), dict(num_seqs=0), dict(cache=ops.KvCacheView(F16, c.keep[0], c.keep[1], 100)),
              dict(cache=ops.KvCacheView(F16, c.keep[0].data_ptr() + 8, c.keep[1], 0)), dict(q=q.data_ptr() + 2),
              dict(cache=ops.KvCacheView(F16, k_ptrs=q, v_ptrs=q)), dict(rule=ops.ScoreRule(scale=float("inf"))),
              dict(cache=ops.KvCacheView(F16, c.keep[0], c.keep[1], 0, page_table=dev_u32([0, 0]), page_rows=16, max_pages_per_seq=1), cache_rows=40)]:
        with pytest.raises(ShadyError):
            ops.attn_prefill_rule(gpu_ctx, **{**p, **b})
    assert gpu_ctx.launch_count == before
    with pytest.raises(ShadyError):
        ops.decode_rule_workspace_size(gpu_ctx, head_dim=100, num_kv_heads=nkv, num_q_heads=nh, num_seqs=S)
    assert cq.view.seq_rows == 20


# ---- calls that the documentation allows and a careless kernel gets wrong --------------------------------------------

def test_decode_workspace_serves_several_shapes(gpu_ctx):
    """One workspace, initialised for the largest batch, used by calls of other head_dims, groups and cache kinds in turn."""
    ws = workspace(gpu_ctx, 64, 3, 48, 40)                    # 40 sequences, 3 kv heads of two head groups
    for hd, nkv, G, lens in ((128, 2, 4, [700, 3]), (64, 3, 16, [90] * 40), (256, 1, 8, [3000]), (128, 2, 4, [900, 44, 0, 17])):
        c = Rows16(lens, nkv, hd, F16, "stride")
        check_decode(gpu_ctx, c, c.values, lens, nkv, G, hd, F16, F16, torch.float16, dict(cap=20.0), ws=ws)
        cq = RowsQ(lens, nkv, hd, 16, seed=hd)
        held = cq.held()
        check_decode(gpu_ctx, cq, lambda s: held[s], lens, nkv, G, hd, F16, F32, torch.float16, {}, ws=ws)


def test_decode_two_calls_at_once(gpu_ctx):
    """Two contexts on two streams, a workspace each, many launches in flight together."""
    from shady_thinker_b200.gpu import GpuContext
    nkv, G, hd, lens = 2, 4, 128, [600, 41]
    c = Rows16(lens, nkv, hd, F16, "stride")
    g = torch.Generator().manual_seed(1)
    q = [(2 * torch.randn(2, nkv * G, hd, generator=g)).half().cuda() for _ in range(2)]
    ld = dev_u32(lens)
    want = []
    for i in range(2):
        ws, n = workspace(gpu_ctx, hd, nkv, nkv * G, 2)
        o = torch.empty_like(q[i])
        ops.attn_decode_rule(gpu_ctx, q=q[i], cache=c.view, seq_lens=ld, out=o, head_dim=hd, num_kv_heads=nkv, num_q_heads=nkv * G, num_seqs=2,
                             q_dtype=F16, out_dtype=F16, workspace=ws, workspace_bytes=n)
        want.append(o)
    gpu_ctx.synchronize()
    ctx = [GpuContext(0) for _ in range(2)]
    wss = [workspace(x, hd, nkv, nkv * G, 2) for x in ctx]
    outs = [[torch.empty_like(q[0]) for _ in range(30)] for _ in range(2)]
    for x in ctx:
        x.synchronize()
    torch.cuda.synchronize()
    for k in range(30):
        for i in range(2):
            ops.attn_decode_rule(ctx[i], q=q[i], cache=c.view, seq_lens=ld, out=outs[i][k], head_dim=hd, num_kv_heads=nkv, num_q_heads=nkv * G,
                                 num_seqs=2, q_dtype=F16, out_dtype=F16, workspace=wss[i][0], workspace_bytes=wss[i][1])
    for x in ctx:
        x.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in outs[i])
    for x in ctx:
        x.close()


def test_decode_length_behind_the_cache_reads_no_other_sequence(gpu_ctx):
    """A length larger than a row-scaled sequence's cache: rows that it does not have count as zero rows, none of the next
    sequence's (here NaN) is read."""
    c = RowsQ([40, 40], 1, 64, seed=1)
    c.scales[0][40:] = float("nan")
    q = torch.randn(1, 4, 64, generator=torch.Generator().manual_seed(1)).half().cuda()
    out = torch.empty_like(q)
    ws, n = workspace(gpu_ctx, 64, 1, 4, 1)
    ops.attn_decode_rule(gpu_ctx, q=q, cache=c.view, seq_lens=dev_u32([70]), out=out, head_dim=64, num_kv_heads=1, num_q_heads=4, num_seqs=1,
                         q_dtype=F16, out_dtype=F16, workspace=ws, workspace_bytes=n)
    gpu_ctx.synchronize()
    assert bool(torch.isfinite(out).all())


@pytest.mark.parametrize("cap", [0.0, 3.0])
def test_nan_queries_give_nan_and_stay_in_their_row(gpu_ctx, cap):
    nkv, G, hd, L = 1, 4, 128, 200
    c = Rows16([L], nkv, hd, BF16, "stride")
    cq = RowsQ([L], nkv, hd, seed=2)
    rule = ops.ScoreRule(cap=cap)
    q = torch.randn(1, G, hd, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    q[0, 2, 5] = float("nan")
    ws, n = workspace(gpu_ctx, hd, nkv, G, 1)
    for cache, kw in ((c.view, {}), (cq.view, {})):
        out, lse = torch.zeros(1, G, hd, dtype=torch.bfloat16, device="cuda"), torch.zeros(1, G, device="cuda")
        ops.attn_decode_rule(gpu_ctx, q=q.cuda(), cache=cache, seq_lens=dev_u32([L]), out=out, lse=lse, rule=rule, head_dim=hd, num_kv_heads=nkv,
                             num_q_heads=G, num_seqs=1, q_dtype=BF16, out_dtype=BF16, workspace=ws, workspace_bytes=n)
        gpu_ctx.synchronize()
        assert bool(out[0, 2].isnan().all()) and bool(lse[0, 2].isnan())
        assert bool(out[0, [0, 1, 3]].isfinite().all()) and bool(lse[0, [0, 1, 3]].isfinite().all())
    qp = torch.randn(L, G, hd, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    qp[100, 1, 7] = float("nan")
    out, lse = torch.zeros(L, G, hd, dtype=torch.bfloat16, device="cuda"), torch.zeros(L, G, device="cuda")
    ops.attn_prefill_rule(gpu_ctx, q=qp.cuda(), cache=c.view, cache_rows=c.rows, q_starts=dev_u32([0, L]), kv_lens=dev_u32([L]), out=out, lse=lse,
                          rule=rule, head_dim=hd, num_kv_heads=nkv, num_q_heads=G, num_seqs=1, total_q=L, dtype=BF16)
    gpu_ctx.synchronize()
    bad = torch.zeros(L, G, dtype=torch.bool)
    bad[100, 1] = True
    assert torch.equal(out.isnan().all(-1).cpu(), bad) and torch.equal(out.isnan().any(-1).cpu(), bad) and torch.equal(lse.isnan().cpu(), bad)


@pytest.mark.parametrize("scale,cap", [(1.0, 1e6), (1e-3, 1e6), (5.0, 1.0), (1.0, 0.01), (0.088, 2.0)])
def test_caps_far_from_the_scores(gpu_ctx, scale, cap):
    """Caps that no score comes near (the polynomial's coefficients would leave f32's range), and that every score exceeds."""
    rule = dict(scale=scale, cap=cap)
    lens = [150]
    c = Rows16(lens, 1, 128, BF16, "packed")
    check_prefill(gpu_ctx, c, c.values, [150], lens, 1, 2, 128, BF16, rule)
    d = Rows16(lens, 1, 128, BF16, "stride")
    check_decode(gpu_ctx, d, d.values, lens, 1, 2, 128, BF16, BF16, torch.bfloat16, rule)


def test_prefill_captured_launch_serves_other_lengths(gpu_ctx):
    """One captured launch, replayed with other token counts and lengths in the same device buffers, padded behind."""
    from shady_thinker_b200.gpu import GpuContext
    nkv, G, hd, S, most = 1, 2, 128, 3, 260
    nh = nkv * G
    stream = torch.cuda.Stream()
    gpu = GpuContext(0, stream=stream.cuda_stream)
    c = Rows16([300, 300, 300], nkv, hd, F16, "stride")
    q = (2 * torch.randn(most, nh, hd, generator=torch.Generator().manual_seed(3))).half()
    with torch.cuda.stream(stream):
        qd, starts, lens = q.cuda(), dev_u32([0, 1, 2, 3]), dev_u32([1, 1, 1])
        out = torch.zeros(most, nh, hd, dtype=torch.float16, device="cuda")
        call = lambda: ops.attn_prefill_rule(gpu, q=qd, cache=c.view, cache_rows=c.rows, q_starts=starts, kv_lens=lens, out=out, head_dim=hd,  # noqa: E731
                                             num_kv_heads=nkv, num_q_heads=nh, num_seqs=S, total_q=most, dtype=F16)
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for counts, rows in (([100, 0, 160], [300, 7, 200]), ([1, 130, 5], [1, 130, 299])):
            at = [0] + [int(x) for x in np.cumsum(counts)]
            starts.copy_(dev_u32(at))
            lens.copy_(dev_u32(rows))
            out.fill_(7.0)
            graph.replay()
            stream.synchronize()
            assert bool((out[at[-1]:] == 7.0).all())
            for s in range(S):
                k, v = (x[:rows[s]] for x in c.values(s))
                for i in {0, counts[s] // 2, counts[s] - 1} if counts[s] else ():
                    want, _, b, _ = attend(q[at[s] + i, 1].double(), k[:, 0], v[:, 0], rows[s] - counts[s] + i, rows[s], wt=torch.float16, out_dt=torch.float16)
                    assert bool(((out[at[s] + i, 1].cpu().double() - want).abs() <= b).all()), (s, i)
    gpu.synchronize()
    del graph
    gpu.close()


def test_prefill_pages_that_the_pool_does_not_have(gpu_ctx):
    """Table entries behind the pool read as zero rows instead of faulting."""
    L, pr = 100, 16
    c = Rows16([L], 1, 128, F16, "paged", page_rows=pr)
    table = c.keep[2].clone()
    table[0, 2], table[0, 4] = 0x7ffffff0, -1                # rows 32..47 and 64..79
    c.view.page_table = table
    c.kv[0][0], c.kv[1][0] = c.kv[0][0].clone(), c.kv[1][0].clone()
    for t in (c.kv[0][0], c.kv[1][0]):
        t[32:48] = 0
        t[64:80] = 0
    check_prefill(gpu_ctx, c, c.values, [L], [L], 1, 2, 128, F16, {})


def test_prefill_many_short_sequences_and_gaps(gpu_ctx):
    """More sequences than a warp has lanes, some without tokens, contexts of very different lengths (levels with gaps)."""
    g = torch.Generator().manual_seed(3)
    kv_lens = [int(x) for x in torch.randint(1, 60, (70,), generator=g)]
    kv_lens[5], kv_lens[40] = 3000, 900
    q_lens = [min(L, int(x)) for L, x in zip(kv_lens, torch.randint(0, 9, (70,), generator=g))]
    q_lens[5], q_lens[40], q_lens[69] = 3, 700, 0
    c = Rows16(kv_lens, 1, 128, BF16, "packed")
    check_prefill(gpu_ctx, c, c.values, q_lens, kv_lens, 1, 4, 128, BF16, dict(cap=25.0), heads=[0, 3])


def test_launches_wait_for_an_uncollected_timeout(gpu_ctx):
    """A wait of an earlier launch ran out and nobody has asked: the operators refuse until shady_synchronize has said so."""
    from shady_thinker_b200._lib import ERR_TIMEOUT
    from shady_thinker_b200.gpu import GpuContext
    from shady_thinker_b200.p2p import ShardCombiner
    gpu = GpuContext(0, stream=0x1)
    gpu.set_wait_limits(peer_polls=1 << 12)
    lone = ShardCombiner(gpu, rank=0, world=2, num_heads=8, head_dim=128, loopback=True)   # rank 1 does not exist
    lone.combine(torch.zeros(8, 130, device="cuda"), torch.zeros(8, 128, device="cuda"))
    torch.cuda.synchronize()
    x = torch.ones(1, 2, 128, dtype=torch.float16, device="cuda")
    codes, scales = torch.full((1, 2, 128), 128, dtype=torch.uint8, device="cuda"), torch.ones(1, 2, device="cuda")
    rowq = ops.RowqCacheView(codes, codes, scales, scales, 1)
    shape = dict(head_dim=128, num_kv_heads=2, num_q_heads=2, num_seqs=1)
    n = ops.decode_rule_workspace_size(gpu, **shape)
    ws = torch.zeros(n, dtype=torch.uint8, device="cuda")
    one, span = dev_u32([1]), dev_u32([0, 1])
    out = torch.empty_like(x)
    calls = [lambda: ops.attn_decode_rule(gpu, q=x, cache=rowq, seq_lens=one, out=out, q_dtype=F16, out_dtype=F16, workspace=ws, workspace_bytes=n, **shape),
             lambda: ops.attn_prefill_rule(gpu, q=x, cache=ops.KvCacheView(F16, x, x, 256), cache_rows=1, q_starts=span, total_q=1, kv_lens=one, out=out,
                                           dtype=F16, **shape),
             lambda: ops.kv_read_rowq(gpu, cache=rowq, k_out=out, out_start=span, total_rows=1, num_seqs=1, num_kv_heads=2, head_dim=128, out_dtype=F16),
             lambda: ops.kv_append_rowq(gpu, q_proj_full=x, k_proj=x, v_proj=x, q_out=out, q_gate=None, cache=rowq, pos_start=one, num_heads=2,
                                        num_kv_heads=2, head_dim=128, rope_theta=1e4, rotary_dim=0, has_gate=False, in_dtype=F16, q_dtype=F16)]
    for call in calls:
        with pytest.raises(ShadyError) as e:
            call()
        assert e.value.code == ERR_TIMEOUT
    with pytest.raises(ShadyError):
        gpu.synchronize()
    for call in calls:
        call()
    gpu.synchronize()
    lone.close()
    gpu.close()


@pytest.mark.parametrize("rule", [dict(), dict(cap=50.0), dict(cap=55.0), dict(cap=60.0), dict(cap=50.0, slopes=True)])
@pytest.mark.parametrize("hd,dt", [(128, BF16), (256, BF16), (128, F16)])
def test_a_query_that_sees_one_row_returns_its_value(gpu_ctx, hd, dt, rule):
    """The one weight is exactly 1 whatever the score, so the first token of a prompt gets its own V row to the last bit; an
    approximate reference of the weights would leave a rounding of half a step."""
    S, nkv, G, t = 9, 2, 4, TORCH_DT[dt]
    g = torch.Generator().manual_seed(hd)
    q = (torch.randn(S, nkv * G, hd, generator=g) * 2).to(t).cuda()
    k, v = (torch.randn(S, nkv, hd, generator=g).to(t).cuda() for _ in range(2))
    r = ops.ScoreRule(cap=rule.get("cap", 0.0), slopes=torch.full((nkv * G,), 0.3, device="cuda") if rule.get("slopes") else None)
    out = torch.full_like(q, float("nan"))
    ops.attn_prefill_rule(gpu_ctx, q=q, cache=ops.KvCacheView(dt, k, v, nkv * hd), cache_rows=S, q_starts=dev_u32(list(range(S + 1))), total_q=S,
                          kv_lens=dev_u32([1] * S), out=out, head_dim=hd, num_kv_heads=nkv, num_q_heads=nkv * G, num_seqs=S, dtype=dt, rule=r)
    gpu_ctx.synchronize()
    assert torch.equal(out, v.repeat_interleave(G, dim=1))
