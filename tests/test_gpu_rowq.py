"""The row-scaled 8-bit KV cache: quantising append and read-back, against 64-bit references (bounds in ``_rule_ref``)."""
import numpy as np
import pytest
import torch

from _rule_ref import U32, norm_rope, quantise, u
from _util import TORCH_DT
from shady_thinker_b200 import ops
from shady_thinker_b200._lib import BF16, F16, F32, ShadyError

pytestmark = pytest.mark.gpu


def dev_u32(v):
    """u32 device array (torch holds it as int32)."""
    return torch.from_numpy(np.asarray(v, np.int64).astype(np.uint32).view(np.int32).copy()).cuda()


class Cache:
    """A row-scaled cache for sequences of the given capacities; rows nobody owns hold garbage codes and NaN scales."""

    def __init__(self, caps, nkv, hd, page_rows=0, seed=0, spare=3):
        self.nkv, self.hd, self.pr, self.caps = nkv, hd, page_rows, caps
        g = torch.Generator().manual_seed(seed)
        if page_rows:
            need = [(c + page_rows - 1) // page_rows for c in caps]
            pages = sum(need) + spare
            order = torch.randperm(pages, generator=g)
            self.table = torch.full((len(caps), max(need + [1]) + 1), 0x7fffffff, dtype=torch.int32)   # entries nobody owns point nowhere
            at = 0
            for s, n in enumerate(need):
                self.table[s, :n] = order[at:at + n].to(torch.int32)
                at += n
            rows, kw = pages * page_rows, dict(page_table=self.table.cuda(), page_rows=page_rows, max_pages_per_seq=self.table.shape[1],
                                               num_pages=pages)
        else:
            self.seq_rows = max(caps + [1])
            rows, kw = len(caps) * self.seq_rows, dict(seq_rows=self.seq_rows)
        self.codes = [torch.randint(0, 256, (rows, nkv, hd), dtype=torch.uint8, generator=g).cuda() for _ in range(2)]
        self.scales = [torch.full((rows, nkv), float("nan")).cuda() for _ in range(2)]
        self.view = ops.RowqCacheView(self.codes[0], self.codes[1], self.scales[0], self.scales[1], **kw)

    def row(self, s, r):
        if self.pr:
            return int(self.table[s, r // self.pr]) * self.pr + r % self.pr
        return s * self.seq_rows + r

    def fill(self, s, kv):
        """Rows 0.. of sequence s from f32 rows (k, v) [n, nkv, hd]."""
        idx = torch.tensor([self.row(s, r) for r in range(kv[0].shape[0])], dtype=torch.long)
        for i in range(2):
            c, sc = quantise(kv[i])
            self.codes[i][idx.cuda()] = c.cuda()
            self.scales[i][idx.cuda()] = sc.cuda()

    def values(self, s, n):
        """Rows 0 .. n-1 of sequence s in f32."""
        idx = torch.tensor([self.row(s, r) for r in range(n)], dtype=torch.long)
        return [(c.cpu()[idx].float() - 128) * sc.cpu()[idx][..., None] for c, sc in zip(self.codes, self.scales)]


def run_append(gpu, cache, q, k, v, starts, pos, *, dt, q_dt, gate, norm, theta, rd, interleaved, total=None, ragged=True, spare=0,
               pos_h=None, pos_w=None, s1=None):
    n, nh, hd = q.shape[0], q.shape[1], k.shape[2]
    nkv = k.shape[1]
    S = len(starts) - 1
    tq = TORCH_DT[q_dt]
    qo = torch.full((n + spare, nh, hd), 7.0, dtype=tq, device="cuda")
    go = torch.full((n + spare, nh, hd), 7.0, device="cuda") if gate else None
    ko, vo = (torch.full((n + spare, nkv, hd), 7.0, dtype=tq, device="cuda") for _ in range(2))
    pad = lambda t: torch.cat([t, torch.full((spare, *t.shape[1:]), float("nan"), dtype=t.dtype)]).cuda()   # noqa: E731
    ops.kv_append_rowq(gpu, q_proj_full=pad(q), k_proj=pad(k), v_proj=pad(v), q_out=qo, q_gate=go, k_out=ko, v_out=vo, cache=cache.view,
                       pos_start=dev_u32(pos), num_heads=nh, num_kv_heads=nkv, head_dim=hd, rope_theta=theta, rotary_dim=rd,
                       interleaved=interleaved, qk_norm_bf16=norm.cuda() if norm is not None else None, num_seqs=S,
                       tokens_per_seq=0 if ragged else n // S, tok_start=dev_u32(starts) if ragged else None, total_tokens=n + spare,
                       in_dtype=dt, q_dtype=q_dt, has_gate=gate, pos_h=pos_h, pos_w=pos_w, s1_limit=s1, s2_limit=s1)
    gpu.synchronize()
    return qo, go, ko, vo


@pytest.mark.parametrize("hd,nkv,G,dt,q_dt,gate,rd,inter,norm,pr,counts", [
    (128, 2, 4, BF16, BF16, False, 128, True, True, 0, [1, 1, 1]),
    (256, 2, 8, BF16, BF16, True, 64, True, True, 64, [5, 1, 0, 17]),
    (64, 3, 1, F16, F16, False, 64, False, True, 16, [33, 2]),
    (128, 1, 7, F32, F32, True, 32, False, True, 48, [1, 0, 0, 9, 3]),
    (256, 4, 2, F32, BF16, False, 0, True, False, 0, [40]),
    (128, 8, 3, F16, F32, False, 6, False, False, 32, [3, 70]),
    (64, 2, 16, BF16, F16, True, 48, True, True, 256, [1] * 40),
    (256, 1, 3, BF16, BF16, False, 256, False, True, 16, [300]),
])
def test_append_matches_the_definition(gpu_ctx, hd, nkv, G, dt, q_dt, gate, rd, inter, norm, pr, counts):
    g = torch.Generator().manual_seed(hd + nkv + len(counts))
    nh, n, S, t = nkv * G, sum(counts), len(counts), TORCH_DT[dt]
    rnd = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    q = rnd(n, nh, hd * (1 + gate)).to(t)
    k, v = (rnd(n, nkv, hd) * 3).to(t), (rnd(n, nkv, hd) * torch.exp(2 * rnd(n, nkv, 1))).to(t)
    if n > 2:
        v[1] = 0                              # an all-zero row
    w = (rnd(2, hd) * 0.1).to(torch.bfloat16) if norm else None
    pos = [int(x) for x in torch.randint(0, 3000, (S,), generator=g)]
    if S > 1:
        pos[-1] = 100_003 if hd == 64 else 0
    starts = [0] + list(np.cumsum(counts))
    caps = [p + c for p, c in zip(pos, counts)]
    if max(caps) > 50_000 and not pr:
        pos, caps = [p % 3000 for p in pos], [p % 3000 + c for p, c in zip(pos, counts)]
    cache = Cache(caps, nkv, hd, pr)
    before = [c.clone() for c in cache.codes], [s.clone() for s in cache.scales]
    qo, go, ko, vo = run_append(gpu_ctx, cache, q, k, v, starts, pos, dt=dt, q_dt=q_dt, gate=gate, norm=w, theta=1e6, rd=rd,
                                interleaved=inter, spare=4)
    seq = np.repeat(np.arange(S), counts)
    at = torch.tensor([pos[s] + i - starts[s] for i, s in enumerate(seq)])
    kw = dict(theta=1e6, rd=rd, interleaved=inter)
    # angle: sincosf (2 ulp) of the f32 angle, whose frequency may be an ulp of powf away: up to 2 u32 |angle|
    da = 2 * U32 * float(at.max()) + 8 * U32
    rq, rk = norm_rope(q[..., :hd], w[0] if norm else None, at, **kw), norm_rope(k, w[1] if norm else None, at, **kw)
    slack = lambda r: (16 * U32 + (2 * da if rd else 0)) * r.abs().amax(-1, keepdim=True)   # noqa: E731
    assert bool(((qo[:n].cpu().double() - rq).abs() <= u(TORCH_DT[q_dt]) * rq.abs() + slack(rq)).all())
    if gate:
        assert torch.equal(go[:n].cpu(), q[..., hd:].float())
    for i, r in enumerate((rk, v.double())):
        rows = torch.tensor([cache.row(s, int(p)) for s, p in zip(seq, at)], dtype=torch.long)
        codes, scales = cache.codes[i].cpu()[rows], cache.scales[i].cpu()[rows]
        want_scale = (r.abs().amax(-1) / 127).clamp(2.0 ** -60, 2.0 ** 60)
        rel = (16 * U32 + (2 * da if rd and i == 0 else 0))
        assert bool(((scales.double() - want_scale).abs() <= rel * want_scale).all())
        held = (codes.float() - 128) * scales[..., None]
        assert int(codes.min()) >= 1                                            # -127 .. 127 only
        assert bool(((held.double() - r).abs() <= 0.5 * want_scale[..., None] * (1 + 2.0 ** -12) + (slack(r) if i == 0 else 4 * U32 * r.abs())).all())
        assert torch.equal((ko, vo)[i][:n].cpu(), held.to(TORCH_DT[q_dt]))      # the stored rows, rounded once
        # nothing else was written
        mask = torch.ones(before[0][i].shape[0], dtype=torch.bool)
        mask[rows] = False
        assert torch.equal(cache.codes[i].cpu()[mask], before[0][i].cpu()[mask])
        assert torch.equal(cache.scales[i].cpu()[mask].nan_to_num(-1), before[1][i].cpu()[mask].nan_to_num(-1))
    for t_ in (qo, go, ko, vo):
        assert t_ is None or bool((t_[n:] == 7.0).all())                        # rows behind the last token


def test_append_uniform_equals_packed(gpu_ctx):
    """The uniform call and the packed call with equal counts write the same bytes."""
    g = torch.Generator().manual_seed(4)
    S, T, nkv, G, hd = 3, 5, 2, 4, 128
    n, nh = S * T, nkv * G
    q, k, v = (torch.randn(n, h, hd, generator=g).to(torch.bfloat16) for h in (nh, nkv, nkv))
    w = (torch.randn(2, hd, generator=g) * 0.1).to(torch.bfloat16)
    a, b = Cache([40] * S, nkv, hd, 16), Cache([40] * S, nkv, hd, 16)
    kw = dict(dt=BF16, q_dt=BF16, gate=False, norm=w, theta=1e4, rd=hd, interleaved=True)
    ra = run_append(gpu_ctx, a, q, k, v, [0, 5, 10, 15], [3, 0, 35], ragged=False, **kw)
    rb = run_append(gpu_ctx, b, q, k, v, [0, 5, 10, 15], [3, 0, 35], ragged=True, **kw)
    for x, y in zip(ra[:1] + ra[2:], rb[:1] + rb[2:]):
        assert torch.equal(x, y)
    for i in range(2):
        assert torch.equal(a.codes[i], b.codes[i])


def test_append_and_read_captured(gpu_ctx):
    """Append and read-back captured together and replayed with other positions, counts and rows in the same device buffers."""
    from shady_thinker_b200.gpu import GpuContext
    S, nkv, G, hd, most = 3, 2, 2, 64, 12
    stream = torch.cuda.Stream()
    gpu = GpuContext(0, stream=stream.cuda_stream)
    c = Cache([50] * S, nkv, hd, 16)
    g = torch.Generator().manual_seed(7)
    k, v = (torch.randn(most, nkv, hd, generator=g) for _ in range(2))
    with torch.cuda.stream(stream):
        kd, vd, q = k.cuda(), v.cuda(), torch.randn(most, nkv * G, hd, generator=g).cuda()
        qo, ko, vo = torch.zeros_like(q), torch.zeros_like(kd), torch.zeros_like(vd)
        kr, vr = torch.zeros_like(kd), torch.zeros_like(vd)
        pos, starts = dev_u32([0, 0, 0]), dev_u32([0, 1, 2, 3])

        def call():
            ops.kv_append_rowq(gpu, q_proj_full=q, k_proj=kd, v_proj=vd, q_out=qo, q_gate=None, k_out=ko, v_out=vo, cache=c.view, pos_start=pos,
                               num_heads=nkv * G, num_kv_heads=nkv, head_dim=hd, rope_theta=1e4, rotary_dim=0, num_seqs=S, tokens_per_seq=0,
                               tok_start=starts, total_tokens=most, has_gate=False)
            ops.kv_read_rowq(gpu, cache=c.view, k_out=kr, v_out=vr, row_start=pos, out_start=starts, total_rows=most, num_seqs=S,
                             num_kv_heads=nkv, head_dim=hd, out_dtype=F32)
        call()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            call()
        for p, counts in (([5, 49, 17], [3, 1, 8]), ([40, 0, 3], [0, 9, 1])):
            pos.copy_(dev_u32(p))
            starts.copy_(dev_u32([0] + list(np.cumsum(counts))))
            for t in (ko, vo, kr, vr):
                t.fill_(7.0)
            graph.replay()
            stream.synchronize()
            n = sum(counts)
            for x, out, back in ((k, ko, kr), (v, vo, vr)):
                code, scale = quantise(x[:n])
                held = (code.float() - 128) * scale[..., None]
                assert torch.equal(back, out) and bool((out[n:] == 7.0).all())
                assert float((out[:n].cpu() - held).abs().max()) <= float(scale.max()) * (1 + 2.0 ** -12)   # a code at most one apart
    gpu.synchronize()
    del graph
    gpu.close()


def test_mrope_sections_match_the_16_bit_append(gpu_ctx):
    """Height and width positions of their own: the rotated Q equals the existing append's."""
    g = torch.Generator().manual_seed(9)
    nh, nkv, hd = 4, 2, 128
    q, k, v = (torch.randn(2, h, hd, generator=g).to(torch.bfloat16) for h in (nh, nkv, nkv))
    c = Cache([60, 60], nkv, hd)
    ph, pw = dev_u32([7, 11]), dev_u32([23, 2])
    got = run_append(gpu_ctx, c, q, k, v, [0, 1, 2], [31, 50], dt=BF16, q_dt=F32, gate=False, norm=None, theta=1e4, rd=64, interleaved=True,
                     ragged=False, pos_h=ph, pos_w=pw, s1=20)
    qo = torch.empty(2, nh, hd, device="cuda")
    kc = torch.zeros(2, 60, nkv, hd, dtype=torch.bfloat16, device="cuda")
    ops.kv_append_rope(gpu_ctx, q_proj_full=q.cuda(), k_proj=k.cuda(), v_proj=v.cuda(), q_out=qo, q_gate=None,
                       cache=ops.KvCacheView(BF16, kc, torch.zeros_like(kc), 60 * nkv * hd), pos_start=dev_u32([31, 50]), num_heads=nh,
                       num_kv_heads=nkv, head_dim=hd, rope_theta=1e4, rotary_dim=64, num_seqs=2, in_dtype=BF16, q_dtype=F32, has_gate=False,
                       write_k_back=False, pos_h=ph, pos_w=pw, s1_limit=20, s2_limit=20)
    gpu_ctx.synchronize()
    # both evaluate the same f32 products; a fused multiply-add in one of them is at most 2 roundings of x and y apart
    assert float((got[0] - qo).abs().max()) <= 4 * U32 * float(qo.abs().max())


def test_append_extreme_rows(gpu_ctx):
    """NaN, infinities, the smallest and the largest values, and positions behind the cache."""
    nkv, hd = 1, 64
    v = torch.zeros(6, nkv, hd)
    v[0, 0, 3] = float("nan"); v[0, 0, 4] = 2.0
    v[1, 0, 0] = float("inf"); v[1, 0, 1] = 1.0
    v[2] = 1e-30
    v[3] = 3e38
    v[4, 0, 5] = -1.5
    c = Cache([5], nkv, hd)
    k = v.clone()
    _, _, ko, vo = run_append(gpu_ctx, c, torch.zeros(6, 1, hd), k, v, [0, 6], [0], dt=F32, q_dt=F32, gate=False, norm=None, theta=1e4, rd=0,
                              interleaved=True)
    want_c, want_s = quantise(v)
    held = (want_c.float() - 128) * want_s[..., None]
    assert torch.equal(vo.cpu(), held) and torch.equal(ko.cpu(), held)     # row 5 does not fit the cache; its output is there
    assert torch.equal(c.codes[1].cpu()[:5], want_c[:5]) and torch.equal(c.scales[1].cpu()[:5], want_s[:5])
    assert float(held[0, 0, 3]) == 0.0 and float(held[2].abs().max()) == 0.0 and float(held[3, 0, 0]) == 127 * 2.0 ** 60


@pytest.mark.parametrize("hd,nkv,out,pr,ranges", [
    (128, 2, F16, 16, [(0, 5), (3, 0), (7, 130), (0, 1)]),
    (256, 1, BF16, 0, [(100, 33)]),
    (64, 3, F32, 48, [(0, 0), (1, 200), (50, 1)]),
    (64, 1, BF16, 16, [(i, i % 3) for i in range(70)]),
    (128, 8, BF16, 256, [(17, 600), (0, 2)]),
])
def test_read_back_is_exact(gpu_ctx, hd, nkv, out, pr, ranges):
    g = torch.Generator().manual_seed(hd)
    c = Cache([f + n for f, n in ranges], nkv, hd, pr)
    for s, (f, n) in enumerate(ranges):
        c.fill(s, [torch.randn(f + n, nkv, hd, generator=g) * 10 for _ in range(2)])
    starts = [0] + list(np.cumsum([n for _, n in ranges]))
    total = starts[-1]
    ko, vo = (torch.full((total + 5, nkv, hd), 7.0, dtype=TORCH_DT[out], device="cuda") for _ in range(2))
    ops.kv_read_rowq(gpu_ctx, cache=c.view, k_out=ko, v_out=vo, row_start=dev_u32([f for f, _ in ranges]), out_start=dev_u32(starts),
                     total_rows=total + 5, num_seqs=len(ranges), num_kv_heads=nkv, head_dim=hd, out_dtype=out)
    gpu_ctx.synchronize()
    for i, o in enumerate((ko, vo)):
        want = torch.cat([c.values(s, f + n)[i][f:] for s, (f, n) in enumerate(ranges)]).to(TORCH_DT[out])
        assert torch.equal(o[:total].cpu(), want)
        assert bool((o[total:] == 7.0).all())


def test_read_back_of_rows_behind_the_cache_and_of_one_tensor(gpu_ctx):
    c = Cache([20], 2, 64, 16)
    c.fill(0, [torch.randn(20, 2, 64) for _ in range(2)])
    vo = torch.full((40, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.kv_read_rowq(gpu_ctx, cache=c.view, v_out=vo, out_start=dev_u32([0, 40]), total_rows=40, num_seqs=1, num_kv_heads=2, head_dim=64)
    gpu_ctx.synchronize()
    assert torch.equal(vo[:20].cpu(), c.values(0, 20)[1].to(torch.bfloat16))
    assert bool((vo[32:] == 0).all())      # rows of a page that the pool does not have


def test_refusals(gpu_ctx):
    c = Cache([16], 2, 64)
    x = torch.zeros(1, 2, 64, device="cuda")
    kw = dict(q_proj_full=x, k_proj=x, v_proj=x, q_out=x, q_gate=None, cache=c.view, pos_start=dev_u32([0]), num_heads=2, num_kv_heads=2,
              head_dim=64, rope_theta=1e4, rotary_dim=64, has_gate=False)
    bad = [dict(head_dim=96), dict(rotary_dim=63), dict(rotary_dim=66), dict(num_kv_heads=0), dict(in_dtype=3), dict(q_dtype=9), dict(has_gate=True),
           dict(k_out=x), dict(total_tokens=2), dict(tokens_per_seq=0), dict(num_seqs=0),
           dict(cache=ops.RowqCacheView(c.codes[0], c.codes[1], c.scales[0], None, 16)),
           dict(cache=ops.RowqCacheView(c.codes[0], c.codes[1], c.scales[0], c.scales[1], 0)),
           dict(cache=ops.RowqCacheView(c.codes[0].data_ptr() + 8, c.codes[1], c.scales[0], c.scales[1], 16)),
           dict(cache=ops.RowqCacheView(c.codes[0], c.codes[1], c.scales[0], c.scales[1], 0, dev_u32([0]), 24, 1)),
           dict(q_out=x.data_ptr() + 4)]
    n = gpu_ctx.launch_count
    for b in bad:
        with pytest.raises(ShadyError):
            ops.kv_append_rowq(gpu_ctx, **{**kw, **b})
    rd = dict(cache=c.view, k_out=x, v_out=x, out_start=dev_u32([0, 1]), total_rows=1, num_seqs=1, num_kv_heads=2, head_dim=64, out_dtype=F32)
    for b in [dict(head_dim=80), dict(out_dtype=3), dict(num_seqs=0), dict(k_out=None, v_out=None), dict(k_out=x.data_ptr() + 8), dict(num_kv_heads=0)]:
        with pytest.raises(ShadyError):
            ops.kv_read_rowq(gpu_ctx, **{**rd, **b})
    assert gpu_ctx.launch_count == n


def test_positions_past_2_to_the_32_touch_no_row(gpu_ctx):
    """A range that runs past the largest position ends there: it does not come round to row 0."""
    c = Cache([8], 1, 64)
    g = torch.Generator().manual_seed(5)
    before = [t.clone() for t in (*c.codes, *c.scales)]
    x = torch.randn(6, 1, 64, generator=g)
    _, _, ko, _ = run_append(gpu_ctx, c, x, x, x, [0, 6], [2 ** 32 - 3], dt=F32, q_dt=F32, gate=False, norm=None, theta=1e4, rd=0, interleaved=True)
    for a, b in zip((*c.codes, *c.scales), before):
        assert torch.equal(a.nan_to_num(9.0), b.nan_to_num(9.0))
    want_c, want_s = quantise(x)
    assert torch.equal(ko.cpu(), (want_c.float() - 128) * want_s[..., None])
    c.fill(0, [x, x])
    out = torch.full((6, 1, 64), 7.0, device="cuda")
    ops.kv_read_rowq(gpu_ctx, cache=c.view, k_out=out, row_start=dev_u32([2 ** 32 - 3]), out_start=dev_u32([0, 6]), total_rows=6, num_seqs=1,
                     num_kv_heads=1, head_dim=64, out_dtype=F32)
    gpu_ctx.synchronize()
    assert bool((out == 0).all())
