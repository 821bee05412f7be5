"""Rotation, shared prefixes and page selection from their definitions, on the CPU:
rotation in fp32 as it is defined and in float64, everything else in float64."""
import torch

import kv4_oracle as oracle


def rotate(x, cos, sin, interleaved, at, dtype=torch.float32):
    """x (rows, heads, d) rotated by entries `at` (rows) of the tables, elementwise in dtype."""
    x = x.cpu().to(dtype)
    c, s = cos.cpu()[at][:, None].to(dtype), sin.cpu()[at][:, None].to(dtype)
    n = 2 * cos.shape[1]
    y = x.clone()
    a, b = (slice(0, n, 2), slice(1, n, 2)) if interleaved else (slice(0, n // 2), slice(n // 2, n))
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    return y


def join_bound(q, k, v, scale=None):
    """What joining two partial results may add to an attention's error: their totals'
    logarithms are fp32 numbers (a rounding of 2^-24 each of the logarithm, 2^-22 for the
    function), the weights 2^-22 exponentials and three roundings, all relative, of results no
    larger than the largest value."""
    d = q.shape[-1]
    scale = d ** -0.5 if scale is None else scale
    n = k.shape[0]
    kk, vv = oracle.values(k), oracle.values(v)
    hk = k.shape[1]
    qq = q.double().cpu().view(q.shape[0], hk, -1, d)
    logit = torch.einsum("rhgd,nhd->rhgn", qq, kk).abs().amax(-1) * scale * 1.4427 + 30 + torch.log2(torch.tensor(float(n)))
    rel = 2 * (logit * 2.0 ** -23 + 2.0 ** -21)
    return (rel[..., None] * vv.abs().amax(0)[None, :, None]).reshape(q.shape[0], -1, d)


def means(k, page):
    """Mean keys (pages, hk, d) of a sequence's quantised keys k (n, hk, d), as held: bf16."""
    vals = oracle.values(k)
    return torch.stack([p.mean(0) for p in vals.split(page)]).float().to(torch.bfloat16)


def choose(q, mean, pos, page, top, first, last):
    """Pages that one row at `pos` attends to: q (H, d), mean (pages, hk, d) bf16; a list per kv head."""
    hk = mean.shape[1]
    total = q.double().cpu().view(hk, -1, q.shape[-1]).sum(1)
    score = torch.einsum("hd,phd->hp", total, mean.double().cpu())
    mine = pos // page
    got = []
    for h in range(hk):
        forced = [i for i in range(mine + 1) if i < first or i > mine - last]
        free = [i for i in range(mine + 1) if i not in forced]
        value = lambda i: float("-inf") if torch.isnan(score[h, i]) else float(score[h, i])
        free.sort(key=lambda i: (bool(torch.isnan(score[h, i])), -value(i), i))
        got.append(sorted(forced + free[:top]))
    return got
