"""The 4-bit cache from its definition: the quantiser in fp32 as the format is
defined, everything else in float64, on the CPU."""
import math

import torch


def floor_bf16(x):
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    return torch.where((cut != bits) & (bits < 0), cut + 65536, cut).view(torch.float32)


def ceil_bf16(x):
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    return torch.where(cut != bits, cut + 65536, cut).view(torch.float32)


def quantise(x):
    """(..., d) -> codes, scale, zero (float32 CPU)."""
    x = x.float().cpu()
    zero = floor_bf16(x.amin(-1))
    scale = ceil_bf16((x.amax(-1) - zero) / torch.full_like(zero, 15.0))
    codes = ((x - zero[..., None]) / scale[..., None]).round().clamp(0, 15)
    codes = torch.where(scale[..., None] > 0, codes, torch.zeros_like(codes))
    return codes, scale, zero


def values(x):
    c, s, z = quantise(x)
    return c.double() * s.double()[..., None] + z.double()[..., None]


def attention(q, k, v, scale=None):
    """One sequence: rows q (r, H, d) at its newest positions over quantised keys and
    values k, v (n, hk, d).  Returns the output and a bound on a kernel's error.

    The kernel's roundings: logits summed in fp32 (d products and the pair's two,
    each sum within (d + 8) 2^-24 of the sum of magnitudes) and a 2^-22 exponential;
    weights p * s in fp16 (2^-11 of each term), and where p * s is below fp16's
    normal range an absolute 2^-25 of the largest scale per token and code; fp32
    output sums (n 2^-24); q in fp16 (2^-11, fp32 queries only)."""
    r, H, d = q.shape
    n, hk, _ = k.shape
    scale = d ** -0.5 if scale is None else scale
    exact_q = q.dtype == torch.bfloat16
    q = q.double().cpu().view(r, hk, H // hk, d)
    kc, ks, kz = (t.double() for t in quantise(k))
    vc, vs, vz = (t.double() for t in quantise(v))
    kk = kc * ks[..., None] + kz[..., None]
    vv = vc * vs[..., None] + vz[..., None]
    logit = torch.einsum("rhgd,nhd->hgrn", q, kk) * scale
    mag = torch.einsum("rhgd,nhd->hgrn", q.abs(), kc * ks[..., None] + kz.abs()[..., None]) * abs(scale)
    seen = torch.arange(n) <= (n - r + torch.arange(r))[:, None]
    logit = logit.masked_fill(~seen, -math.inf)
    some = seen.any(-1)
    w = torch.exp(logit - logit.amax(-1, keepdim=True).clamp(min=-1e300))
    total = w.sum(-1, keepdim=True).clamp(min=1e-300)
    p = w / total
    y = torch.einsum("hgrn,nhd->rhgd", p, vv)
    rel = (mag.masked_fill(~seen, 0).amax(-1, keepdim=True) * ((d + 8) * 2.0 ** -24 + (0 if exact_q else 2.0 ** -11)))
    rel = 2 * rel + 2.0 ** -21 + n * 2.0 ** -24
    codes = torch.einsum("hgrn,nhd->rhgd", p, vc * vs[..., None])
    whole = torch.einsum("hgrn,nhd->rhgd", p, vc * vs[..., None] + vz.abs()[..., None])
    tiny = 15 * 2.0 ** -25 * vs.amax(0) if n else torch.zeros(hk)
    tiny = (seen.sum(-1)[None, None] / total[..., 0]) * tiny[:, None, None]  # (hk, g, r)
    bound = 2.0 ** -11 * codes + rel.permute(2, 0, 1, 3) * whole + tiny.permute(2, 0, 1)[..., None]
    y[~some] = 0
    return y.reshape(r, H, d), bound.reshape(r, H, d)
