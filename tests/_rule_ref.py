"""64-bit references of the row-scaled cache and of attention under a score rule (CPU, torch), with the error bounds the
GPU tests hold the kernels to.

Bounds.  u(t) = torch.finfo(t).eps / 2 is the largest relative error of one rounding to t, u32 that of f32.
* A score z = sum of hd products in f32: |dz| <= (hd + 8) u32 * scale * sum|q k| (any order of summation, the multiplications
  by scale and the row's scale among the 8); a tanh cap computed as 1 - 2/(1 + e) adds at most 16 u32 * cap, a distance
  bias 4 u32 * |slope * distance|, and exp2/log2/rcp approximations (2 ulp each, argument up to 2^8) 2^-15 in all.
* A weight rounded to t: relative u(t); f16 weights below 2^-14 of the running maximum: absolute 2^-25.
* out = sum w v / sum w:  |dout| <= (u(t) + 2 dz) * A + n * 2^-25 * max|v| (f16 only) + u(out) |out|, A = sum p |v|.
"""
import math

import torch

U32 = 2.0 ** -24


def u(dt):
    return torch.finfo(dt).eps / 2


def quantise(x):
    """Row-scaled codes (as stored, +128) and scales of x [..., hd] in f32, as the header defines them."""
    x = x.float()
    amax = torch.where(torch.isnan(x), torch.zeros_like(x), x.abs()).amax(-1)
    scale = (amax / 127).clamp(2.0 ** -60, 2.0 ** 60)
    code = torch.round(x / scale[..., None]).nan_to_num(0.0, 127.0, -127.0).clamp(-127, 127)
    return (code + 128).to(torch.uint8), scale


def attend(q, k, v, pos, L, *, scale=0.0, cap=0.0, slope=0.0, window=0, prefix=0, doc=0, wt=torch.float32, out_dt=torch.float32):
    """One head: q [hd] at position pos over k, v [L, hd] (all f64).  Returns out, lse, bound on |dout| [hd], bound on |dlse|."""
    hd = q.shape[-1]
    scale = scale or 1.0 / math.sqrt(hd)
    j = torch.arange(L)
    seen = (j >= doc) & ((j < prefix) | ((j <= pos) & ((pos - j < window) if window else (j >= 0))))
    if pos < 0 or not bool(seen.any()):
        z = torch.zeros(hd, dtype=torch.float64)
        return z, -math.inf, z, 0.0
    k, v, j = k[seen], v[seen], j[seen]
    z = k @ q * scale
    dz = (hd + 8) * U32 * scale * float((k.abs() @ q.abs()).max()) + 2.0 ** -15
    if cap:
        z = cap * torch.tanh(z / cap)
        dz += 16 * U32 * cap
    if slope:
        z = z - slope * (pos - j).abs().double()
        dz += 4 * U32 * abs(slope) * float((pos - j).abs().max())
    lse = float(torch.logsumexp(z, 0))
    p = torch.exp(z - lse)
    out, A = p @ v, p @ v.abs()
    n = int(seen.sum())
    tiny = n * 2.0 ** -25 * float(v.abs().max()) if wt == torch.float16 else 0.0
    return out, lse, (u(wt) + 2 * dz) * A + tiny + u(out_dt) * out.abs() + 1e-30, dz + 4 * U32 * (1 + abs(lse))


def norm_rope(x, w, pos, *, theta, rd, interleaved, eps=1e-6):
    """x [n, heads, hd] f64 at positions pos [n]: RMSNorm(1 + w) and rotation, angles rounded to f32 as the library does."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + eps) * (1 + w.double())
    if rd:
        i = torch.arange(rd // 2)
        freq = torch.tensor([1.0], dtype=torch.float32) / torch.pow(torch.tensor(theta, dtype=torch.float32), 2.0 * i.float() / rd)
        ang = (pos.float()[:, None] * freq).double()
        c, s = ang.cos()[:, None], ang.sin()[:, None]
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rd // 2)
        y = x.clone()
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., b] * c + x[..., a] * s
        x = y
    return x
