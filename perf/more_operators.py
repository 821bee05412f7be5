"""Operators of serving over the paged 4-bit cache, as cases to time: each in its
plain form (elementary torch operations) and, with `own` set, as the calls a user
makes of this package.

    rotary     queries, keys and values of a projection: positions rotated into
               queries and keys, keys and values stored in the cache, read back as
               the values they stand for (penta_cache.kv4_append_rotary, kv4_gather)
    prefix     causal attention of the newest rows of sequences that share a long
               prefix by groups, the prefix held once (penta_cache.kv4_prefix_attention)
    sparse     the mean key of each page kept up to date, and attention of the newest
               rows over the pages that a score of the means selects for each row and
               kv head (penta_cache.kv4_page_means, kv4_sparse_attention)

The cache: uint8 (pages, kv heads, 2, page * (d / 2 + 4)), keys at index 0 of
the third axis and values at 1.  Each of the two is page * d / 2 bytes of 4-bit
codes, then page pairs of bf16 (scale, zero); a code c stands for
scale * c + zero.  Keys: token by token, two dims per byte, the even one in the
low half.  Values: two tokens (2i, 2i + 1) side by side, 32-bit words of four
dims of the first token then the same four dims of the second.
"""
import math
import os
import sys

import torch

own = False
_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "pentanet-v1.0_b200")


def _cache():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import penta_cache
    return penta_cache


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    return [
        # one decoded token of a GPT of 12 heads of 64 dims
        dict(name="rotary, one token", op="rotary", batch=1, q_len=1, ragged=False, kv_heads=12, group=1, head_dim=64,
             page=64, length=1024, rotated=64, interleaved=False, offset=0, dtype="bf16"),
        # one decode step of 64 requests behind a shared prefix, grouped heads
        dict(name="rotary, decode step", op="rotary", batch=64, q_len=1, ragged=False, kv_heads=8, group=8, head_dim=128,
             page=64, length=4096, rotated=128, interleaved=False, offset=8192, dtype="bf16"),
        # the prompts of several requests at once, of unequal lengths; half of the dims rotated, neighbours paired
        dict(name="rotary, ragged prompts", op="rotary", batch=7, q_len=2047, ragged=True, kv_heads=8, group=4, head_dim=128,
             page=32, length=2047, rotated=64, interleaved=True, offset=0, dtype="bf16"),
        # a few samples of one short prompt, 12 heads of 64 dims
        dict(name="prefix, short", op="prefix", batch=8, groups=1, q_len=1, ragged=False, kv_heads=12, group=1, head_dim=64,
             page=64, prefix=513, length=65),
        # a decode step of 64 requests behind one system prompt, grouped heads
        dict(name="prefix, decode step", op="prefix", batch=64, groups=1, q_len=1, ragged=False, kv_heads=8, group=8,
             head_dim=128, page=64, prefix=8192, length=1000),
        # sixteen samples over one very long document
        dict(name="prefix, long document", op="prefix", batch=16, groups=1, q_len=1, ragged=False, kv_heads=8, group=4,
             head_dim=128, page=128, prefix=131071, length=257),
        # chunks of unequal lengths behind three prefixes of unequal lengths
        dict(name="prefix, ragged chunks", op="prefix", batch=24, groups=3, q_len=33, ragged=True, kv_heads=8, group=4,
             head_dim=128, page=32, prefix=8191, length=500),
        # one decoded token of a GPT of 12 heads of 64 dims, small pages
        dict(name="sparse, one short row", op="sparse", batch=1, q_len=1, ragged=False, kv_heads=12, group=1, head_dim=64,
             page=16, length=4095, top=24, first=1, last=4),
        # a decode step of 32 requests of very different ages, grouped heads
        dict(name="sparse, ragged decode", op="sparse", batch=32, q_len=1, ragged=False, kv_heads=8, group=8, head_dim=128,
             page=64, length=32768, top=32, first=1, last=2),
        # one very long document, a single new token
        dict(name="sparse, long decode", op="sparse", batch=1, q_len=1, ragged=False, kv_heads=8, group=4, head_dim=128,
             page=64, length=262143, top=64, first=1, last=4),
        # a piece of a prompt, every row with a selection of its own
        dict(name="sparse, chunk", op="sparse", batch=2, q_len=251, ragged=True, kv_heads=8, group=4, head_dim=128, page=64,
             length=16000, top=16, first=1, last=2),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rotary", "prefix", "sparse"])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 2, 3, 4, 6, 8, 16])
    head_dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "rotary":
        q_len = 1 if rng.random() < 0.4 else min(_log(rng, 2, 2047), 240000 // (kv_heads * group))
        batch = _log(rng, 1, max(1, min(128, 240000 // (q_len * kv_heads * group))))
        return dict(op=op, batch=batch, q_len=q_len, ragged=q_len > 1 and rng.random() < 0.6, kv_heads=kv_heads, group=group,
                    head_dim=head_dim, page=page, length=max(q_len, _log(rng, 64, 4096)),
                    rotated=rng.choice([head_dim, head_dim, head_dim // 2, 16, 48]), interleaved=rng.random() < 0.4,
                    offset=rng.choice([0, _log(rng, 1, 100000)]), dtype=rng.choice(["bf16", "bf16", "f32"]))
    if op == "prefix":
        prefix, length = _log(rng, 33, 65536), _log(rng, 1, 1500)
        q_len = rng.choice([1, 1, 1, 3, 17, 64])
        # no more logits than 64 sequences x 64 heads over 8192 tokens
        prefix = min(prefix, max(33, 64 * 64 * 8192 // (q_len * kv_heads * group) - length))
        batch = _log(rng, 1, max(1, min(96, 64 * 64 * 8192 // ((prefix + length) * q_len * kv_heads * group))))
        return dict(op=op, batch=batch, groups=rng.randint(1, max(1, min(4, batch))), q_len=q_len,
                    ragged=q_len > 1 and rng.random() < 0.6, kv_heads=kv_heads, group=group, head_dim=head_dim, page=page,
                    prefix=prefix, length=max(q_len, length))
    top, long, first, last = _log(rng, 1, 64), _log(rng, 64, 131072), rng.choice([0, 1, 2]), rng.choice([1, 2, 4])
    if rng.random() < 0.6:
        q_len, batch = rng.choice([1, 1, 2, 5]), _log(rng, 1, max(2, min(48, 262144 * 8 // (long * kv_heads) // 2)))
    else:
        q_len, batch, long = _log(rng, 8, 200), rng.choice([1, 2]), min(max(long, 256), 16384)
        group = min(group, max(1, 32 // kv_heads))
    # no more tokens read than 256 rows of 8 heads with 2048 tokens each
    while q_len > 1 and q_len * batch * kv_heads * (first + last + 1) * page > 256 * 8 * 2048:
        q_len = (q_len + 1) // 2
    top = max(1, min(top, 256 * 8 * 2048 // (q_len * batch * kv_heads * page) - first - last))
    return dict(op=op, batch=batch, q_len=min(q_len, long), ragged=q_len > 1 and rng.random() < 0.5, kv_heads=kv_heads,
                group=group, head_dim=head_dim, page=page, length=long, top=top, first=first, last=last)


def _rows_of(case):
    """New rows of each sequence: all alike, or from the longest down to a quarter of it."""
    b, n = case["batch"], case["q_len"]
    if not case["ragged"]:
        return [n] * b
    return [max(1, n - (3 * n * i) // (4 * b)) for i in range(b)]


def _lengths_of(case):
    """Tokens of each sequence with its new rows (behind its prefix): from the longest down to a tenth of it, none a
    round number."""
    b, n = case["batch"], case["length"]
    return [max(r, n - (9 * n * i) // (10 * b) - (37 * i) % 13) for i, r in enumerate(_rows_of(case))]


def _prefixes_of(case):
    """Tokens of each prefix, and how many sequences share it: unequal, from the longest prefix down to a third."""
    b, n, groups = case["batch"], case["prefix"], case["groups"]
    tokens = [max(1, n - (2 * n * g) // (3 * groups) - 5 * g) for g in range(groups)]
    ends = [b * (g + 1) * (g + 2) // (groups * (groups + 1)) for g in range(groups)]
    return tokens, [e - s for s, e in zip([0] + ends, ends)]


# ── inputs ───────────────────────────────────────────────────────────────────

def _gen(seed, device):
    return torch.Generator(device=device).manual_seed(7654321 + int(seed))


def _round_down(x):
    """fp32 rounded to a bf16 value towards -infinity (kept in fp32)."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    cut = torch.where((cut != bits) & (bits < 0), cut + 65536, cut)
    return cut.view(torch.float32)


def _round_up(x):
    """A non-negative fp32 rounded to a bf16 value upwards (kept in fp32)."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    return torch.where(cut != bits, cut + 65536, cut).view(torch.float32)


def _quantise(x):
    """(..., d) -> codes (..., d) uint8, scale (...), zero (...): the range of each vector in 15 steps."""
    x = x.float()
    zero = _round_down(x.amin(-1))
    span = x.amax(-1) - zero
    scale = _round_up(span / torch.full_like(span, 15))  # (a division by a Python number multiplies by its reciprocal)
    codes = ((x - zero[..., None]) / scale[..., None]).round().clamp(0, 15)
    return torch.where(scale[..., None] > 0, codes, torch.zeros_like(codes)).to(torch.uint8), scale, zero


def _pairs(scale, zero):
    """bf16 (scale, zero) as bytes: (..., page) -> (..., page * 4)."""
    p = torch.stack((scale, zero), -1).to(torch.bfloat16).contiguous()
    return p.view(torch.uint8).flatten(-2)


def _lay_out(k, v):
    """Keys and values (pages, heads, page, d) as a cache."""
    n, h, page, d = k.shape
    c, s, z = _quantise(k)
    kb = torch.cat(((c[..., 0::2] | (c[..., 1::2] << 4)).flatten(-2), _pairs(s, z)), -1)
    c, s, z = _quantise(v)
    c = c.view(n, h, page // 2, 2, d // 4, 4).transpose(3, 4)
    vb = torch.cat(((c[..., 0::2] | (c[..., 1::2] << 4)).reshape(n, h, -1), _pairs(s, z)), -1)
    return torch.stack((kb, vb), 2).contiguous()


def prepare(case, seed):
    device = torch.device("cuda", torch.cuda.current_device())
    g = _gen(seed, device)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=device)

    s = dict(case)
    b, hk, group, d, page = case["batch"], case["kv_heads"], case["group"], case["head_dim"], case["page"]
    rows, lengths = _rows_of(case), _lengths_of(case)
    prefixes, shared = _prefixes_of(case) if case["op"] == "prefix" else ([], [])
    # pages in any order: the sequences' own, then the prefixes'
    need = [-(-n // page) for n in lengths + prefixes]
    order = torch.randperm(sum(need) + 1, generator=g, device=device, dtype=torch.int32)
    tables = []
    for part in (need[:b], need[b:]):
        table = torch.zeros(len(part), max(part, default=0), dtype=torch.int32, device=device)
        for i, m in enumerate(part):
            table[i, :m] = order[:m]
            order = order[m:]
        tables.append(table)
    s["table"], s["prefix_table"] = tables
    s["lens"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    s["prefix_lens"] = torch.tensor(prefixes, dtype=torch.int32, device=device)
    s["shared"] = shared
    s["cu_prefix"] = torch.tensor([0] + shared, device=device).cumsum(0).to(torch.int32)
    s["new"] = torch.tensor(rows, device=device)
    s["cu"] = torch.tensor([0] + rows, device=device).cumsum(0).to(torch.int32) if case["ragged"] else None
    # per row: its sequence and its position there
    s["seq"] = torch.repeat_interleave(torch.arange(b, device=device), torch.tensor(rows, device=device))
    s["pos"] = torch.cat([torch.arange(n - r, n, device=device) for r, n in zip(rows, lengths)])
    total = sum(need) + 1
    loud = torch.where(torch.rand(hk, 1, d, generator=g, device=device) < 0.03, 5.0, 1.0)
    dtype = {"bf16": torch.bfloat16, "f32": torch.float32}[case.get("dtype", "bf16")]
    topic = None
    if case["op"] == "rotary":
        s["cache"] = torch.zeros(total, hk, 2, page * (d // 2 + 4), dtype=torch.uint8, device=device)
        # the tables that a model keeps: one row per position
        half = case["rotated"] // 2
        rate = 10000.0 ** (-torch.arange(half, device=device, dtype=torch.float64) / half)
        angle = torch.arange(case["offset"] + case["length"], device=device, dtype=torch.float64)[:, None] * rate
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["offsets"] = torch.full((b,), case["offset"], dtype=torch.int32, device=device) if case["offset"] else None
    else:
        # what a page is about differs from page to page
        topic = normal(total, hk, 1, d) * 0.4
        k = (normal(total, hk, page, d) + topic) * loud
        s["cache"] = _lay_out(k.to(torch.bfloat16), normal(total, hk, page, d).to(torch.bfloat16))
        del k
    if case["op"] == "sparse":
        s["means"] = torch.cat([_unpack(part, page, d)[0].double().mean(-2).float() for part in s["cache"].split(1024)]
                               ).to(torch.bfloat16)
    # one projection's output holds queries, keys and values side by side
    qkv = normal(sum(rows), (group + 2) * hk, d)
    qkv[:, group * hk:(group + 1) * hk] *= loud[:, 0]
    if case["op"] == "sparse":  # a query asks after a few pages' topics
        asked = torch.randint(0, total, (sum(rows), 4), generator=g, device=device)
        qkv[:, :group * hk] += topic[asked, :, 0].sum(1).repeat_interleave(group, dim=1)
    qkv = qkv.to(dtype)
    if case["ragged"]:
        parts = qkv.split((group * hk, hk, hk), dim=1)
    else:
        parts = qkv.view(b, case["q_len"], -1, d).split((group * hk, hk, hk), dim=2)
    s["q"], s["k"], s["v"] = parts
    return s


# ── one pass ─────────────────────────────────────────────────────────────────

def run(s):
    return {"rotary": _rotary, "prefix": _prefix, "sparse": _sparse}[s["op"]](s)


def _turn(x, cos, sin, interleaved):
    """(rows, heads, d) with its first dims rotated by the rows' angles, in fp32."""
    x = x.float()
    n = 2 * cos.shape[-1]
    cos, sin = cos[:, None], sin[:, None]
    a, b = (x[..., 0:n:2], x[..., 1:n:2]) if interleaved else (x[..., :n // 2], x[..., n // 2:n])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., n:]), -1)


def _rotary(s):
    if own:
        pc = _cache()
        q = pc.kv4_append_rotary(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["cache"], s["table"], s["lens"], cu_q=s["cu"],
                                 offsets=s["offsets"], interleaved=s["interleaved"])
        k, v = pc.kv4_gather(s["cache"], s["head_dim"], s["table"], s["lens"], s["k"].shape[:-2], cu_q=s["cu"])
        return {"q": q, "k": k, "v": v}
    hk, group, d, page, cache = s["kv_heads"], s["group"], s["head_dim"], s["page"], s["cache"]
    at = s["pos"] if s["offsets"] is None else s["pos"] + s["offsets"][s["seq"]]
    cos, sin = s["cos"][at], s["sin"][at]
    q = _turn(s["q"].reshape(-1, hk * group, d), cos, sin, s["interleaved"]).to(s["q"].dtype)
    k = _turn(s["k"].reshape(-1, hk, d), cos, sin, s["interleaved"])
    page_at = s["table"][s["seq"], s["pos"] // page].long()
    tok = s["pos"] % page
    kc, ks, kz = _quantise(k)
    vc, vs, vz = _quantise(s["v"].reshape(-1, hk, d))
    codes = cache[..., :page * d // 2]
    pairs = cache[..., page * d // 2:].view(torch.bfloat16).view(-1, hk, 2, page, 2)
    codes[:, :, 0].view(-1, hk, page, d // 2)[page_at, :, tok] = kc[..., 0::2] | (kc[..., 1::2] << 4)
    codes[:, :, 1].view(-1, hk, page // 2, d // 4, 2, 2)[page_at, :, tok // 2, :, tok % 2] = (
        vc[..., 0::2] | (vc[..., 1::2] << 4)).view(-1, hk, d // 4, 2)
    pairs[page_at, :, 0, tok] = torch.stack((ks, kz), -1).to(torch.bfloat16)
    pairs[page_at, :, 1, tok] = torch.stack((vs, vz), -1).to(torch.bfloat16)
    k, v = [(c.float() * scale[..., None] + zero[..., None]).to(torch.bfloat16).reshape(s["k"].shape)
            for c, scale, zero in ((kc, ks, kz), (vc, vs, vz))]
    return {"q": q.reshape(s["q"].shape), "k": k, "v": v}


def _unpack(pages, page, d):
    """Cache pages (..., 2, bytes) as fp32 keys and values (..., page, d)."""
    codes = pages[..., :page * d // 2]
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    pair = pages[..., page * d // 2:].contiguous().view(torch.bfloat16).unflatten(-1, (page, 2)).float()
    scale, zero = pair[..., :1], pair[..., 1:]
    k = codes[..., 0, :].unflatten(-1, (page, d))
    v = codes[..., 1, :].unflatten(-1, (page // 2, d // 4, 2, 4)).transpose(-3, -2).flatten(-2).flatten(-3, -2)
    return k * scale[..., 0, :, :] + zero[..., 0, :, :], v * scale[..., 1, :, :] + zero[..., 1, :, :]


def _side_by_side(s):
    """Rows of unequal sequences in one array (b, n, heads, d): row i of a sequence at its place from the end, and
    where that is."""
    n = s["q_len"]
    at = n - s["lens"][s["seq"]] + s["pos"]
    q = torch.zeros(s["batch"], n, s["kv_heads"] * s["group"], s["head_dim"], device=s["q"].device)
    q[s["seq"], at] = s["q"].reshape(-1, *q.shape[2:]).float()
    return q, at


def _prefix(s):
    if own:
        return _cache().kv4_prefix_attention(s["q"], s["cache"], s["table"], s["lens"], s["prefix_table"], s["prefix_lens"],
                                             cu_q=s["cu"], cu_prefix=s["cu_prefix"])
    b, hk, group, d, page, n = s["batch"], s["kv_heads"], s["group"], s["head_dim"], s["page"], s["q_len"]
    q, at = _side_by_side(s)
    q = q.view(b, n, hk, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)  # (b, heads, group * n, d)
    keys, values = (x.transpose(1, 2).flatten(2, 3) for x in _unpack(s["cache"][s["table"].long()], page, d))
    w = q @ keys.transpose(2, 3) / math.sqrt(d)
    seen = s["lens"][:, None] - n + torch.arange(n, device=w.device)  # the last own position that each row sees
    hidden = torch.arange(w.shape[-1], device=w.device) > seen[..., None]
    w = w.view(b, hk, group, n, -1).masked_fill_(hidden[:, None, None], float("-inf")).flatten(2, 3)
    ahead, before = _unpack(s["cache"][s["prefix_table"].long()], page, d)  # (groups, pages, heads, page, d)
    y = torch.empty_like(q)
    first = 0
    for i, many in enumerate(s["shared"]):
        of = slice(first, first + many)
        first += many
        if many == 0:
            continue
        pk, pv = (x[i].transpose(0, 1).flatten(1, 2) for x in (ahead, before))  # (heads, tokens, d)
        u = torch.einsum("bhrd,htd->bhrt", q[of], pk) / math.sqrt(d)
        u.masked_fill_(torch.arange(u.shape[-1], device=u.device) >= s["prefix_lens"][i], float("-inf"))
        top = torch.maximum(u.amax(-1, keepdim=True), w[of].amax(-1, keepdim=True)).clamp(min=-3e38)
        u, x = torch.exp(u - top), torch.exp(w[of] - top)
        y[of] = (torch.einsum("bhrt,htd->bhrd", u, pv) + x @ values[of]) / (u.sum(-1) + x.sum(-1))[..., None]
    y = y.view(b, hk, group, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, hk * group, d)
    return y[s["seq"], at].to(s["q"].dtype).reshape(s["q"].shape)


def _touched(s):
    """The pages that the new rows are in: their sequence and their number there (the last one repeated where a
    sequence's rows are in fewer pages than another's)."""
    last = s["lens"].long() - 1
    first = last + 1 - s["new"]
    most = (s["q_len"] - 2) // s["page"] + 2
    i = (first // s["page"])[:, None] + torch.arange(most, device=last.device)
    i = torch.minimum(i, (last // s["page"])[:, None])
    return torch.arange(s["batch"], device=last.device).repeat_interleave(most), i.flatten()


def _sparse(s):
    top, first, last = s["top"], s["first"], s["last"]
    if own:
        pc = _cache()
        pc.kv4_page_means(s["cache"], s["means"], s["table"], s["lens"], s["q"].shape[:-2], cu_q=s["cu"])
        y, pages = pc.kv4_sparse_attention(s["q"], s["cache"], s["means"], s["table"], s["lens"], top, first_pages=first,
                                           last_pages=last, cu_q=s["cu"], return_pages=True)
        return {"y": y, "pages": pages.flatten(0, -3), "means": s["means"]}
    b, hk, group, d, page = s["batch"], s["kv_heads"], s["group"], s["head_dim"], s["page"]
    # the means of the pages that the rows are in, over the tokens held so far
    seq, i = _touched(s)
    phys = s["table"][seq, i].long()
    keys = _unpack(s["cache"][phys], page, d)[0].double()
    held = (s["lens"][seq] - i * page).clamp(max=page)
    keys = keys * (torch.arange(page, device=keys.device) < held[:, None])[:, None, :, None]
    s["means"][phys] = (keys.sum(2) / held[:, None, None]).float().to(torch.bfloat16)
    # scores in 64 bits: two that are close decide which page is read
    means = s["means"][s["table"].long()].double()  # (b, pages, heads, d)
    total = s["q"].reshape(-1, hk, group, d).double().sum(2)
    n = s["q_len"]
    at = n - s["lens"][s["seq"]] + s["pos"]
    side = torch.zeros(b, n, hk, d, dtype=torch.float64, device=total.device)
    side[s["seq"], at] = total
    score = torch.einsum("bnhd,bphd->bnhp", side, means)[s["seq"], at]  # (rows, heads, pages)
    index = torch.arange(score.shape[-1], device=score.device)
    mine = (s["pos"] // page)[:, None, None]
    forced = (index < first) & (index <= mine) | (index > mine - last) & (index <= mine)
    score = score.masked_fill(forced | (index > mine), float("-inf"))
    value, order = torch.sort(score, dim=-1, descending=True, stable=True)
    picked = torch.zeros_like(forced.expand(score.shape)).scatter(-1, order[..., :top], value[..., :top] > float("-inf"))
    width = first + top + last
    beyond = max(score.shape[-1], 1) + width
    pages = torch.where(picked | forced, index, beyond)
    pages = torch.nn.functional.pad(pages, (0, width), value=beyond).sort(-1).values[..., :width]
    pages = torch.where(pages < beyond, pages, -1)
    # attention over them
    phys = s["table"][s["seq"][:, None, None], pages.clamp(min=0)].long()
    keys, values = _unpack(s["cache"][phys, torch.arange(hk, device=phys.device)[:, None]], page, d)
    keys, values = keys.flatten(2, 3), values.flatten(2, 3)  # (rows, heads, tokens, d)
    token = (pages[..., None] * page + torch.arange(page, device=pages.device)).flatten(2)
    hidden = (pages < 0).repeat_interleave(page, -1) | (token > s["pos"][:, None, None])
    q = s["q"].reshape(-1, hk, group, d).float()
    w = (q @ keys.transpose(2, 3) / math.sqrt(d)).masked_fill(hidden[:, :, None], float("-inf"))
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-3e38))
    y = (w @ values) / w.sum(-1, keepdim=True)
    return {"y": y.to(s["q"].dtype).reshape(s["q"].shape), "pages": pages.to(torch.int32), "means": s["means"]}


# ── what a pass cannot do without ────────────────────────────────────────────

def work(case):
    rows, lengths = _rows_of(case), _lengths_of(case)
    hk, group, d, page = case["kv_heads"], case["group"], case["head_dim"], case["page"]
    held = 2 * hk * (d // 2 + 4)  # bytes of one token in the cache
    n = sum(rows)
    if case["op"] == "rotary":
        wide = 2 if case["dtype"] == "bf16" else 4
        moved = n * (2 * hk * group * d * wide + 2 * hk * d * wide + held + 2 * hk * d * 2)
        tables = max(lengths) * case["rotated"] * 4 if case["q_len"] > 1 else len(set(lengths)) * case["rotated"] * 4
        return {"bytes": moved + tables, "flops": n * (hk * (group + 1) * case["rotated"] * 3 + 2 * hk * d * 4)}
    pairs = sum(r * t - r * (r - 1) // 2 for r, t in zip(rows, lengths))
    queries = 2 * 2 * n * hk * group * d
    if case["op"] == "prefix":
        tokens, shared = _prefixes_of(case)
        at = 0
        for t, many in zip(tokens, shared):
            pairs += t * sum(rows[at:at + many])
            at += many
        return {"bytes": (sum(lengths) + sum(t for t, many in zip(tokens, shared) if many)) * held + queries,
                "flops": 4 * pairs * hk * group * d}
    width = case["first"] + case["top"] + case["last"]
    read = means = seen = 0
    for r, t in zip(rows, lengths):
        pages = -(-t // page)
        means += pages
        read += min(t, r * width * page)
        seen += sum(min(p + 1, width * page) for p in range(t - r, t))
    return {"bytes": means * hk * d * 2 + read * held + queries + 4 * n * hk * width,
            "flops": 4 * seen * hk * group * d + 2 * d * hk * sum(r * -(-t // page) for r, t in zip(rows, lengths))}


# ── the same from the definitions, in 64 bits ────────────────────────────────

def _tokens(s, entries):
    """Keys and values of whole pages, (heads, tokens, d) in 64 bits, read code by code."""
    d, page = s["head_dim"], s["page"]
    kv = s["cache"][entries.long()].to(torch.int64)  # (pages, heads, 2, bytes)
    size = page * d // 2
    pair = (kv[..., size + 1::2] << 24 | kv[..., size::2] << 16).to(torch.int32).view(torch.float32).double()
    token, dim = torch.arange(page, device=kv.device)[:, None], torch.arange(d, device=kv.device)
    got = []
    for j in (0, 1):
        byte = (token * (d // 2) + dim // 2) if j == 0 else (token // 2 * d + dim // 4 * 4 + token % 2 * 2 + dim % 4 // 2)
        code = kv[:, :, j][:, :, byte] >> (dim % 2 * 4) & 15
        x = pair[:, :, j, 0::2, None] * code + pair[:, :, j, 1::2, None]
        got.append(x.transpose(0, 1).flatten(1, 2))
    return got


def exact(case, seed):
    s = prepare(case, seed)
    hk, group, d, page = case["kv_heads"], case["group"], case["head_dim"], case["page"]
    rows, lengths = _rows_of(case), _lengths_of(case)
    if case["op"] == "rotary":
        at = s["pos"] + case["offset"]
        turn = torch.complex(s["cos"].double(), s["sin"].double())[at][:, None]
        n = case["rotated"]
        out = {}
        for name in ("q", "k"):
            x = s[name].reshape(sum(rows), -1, d).double()
            lead = x[..., :n]
            if case["interleaved"]:
                z = torch.view_as_complex(lead.unflatten(-1, (n // 2, 2)).contiguous()) * turn
                lead = torch.view_as_real(z).flatten(-2)
            else:
                z = torch.complex(lead[..., :n // 2].contiguous(), lead[..., n // 2:].contiguous()) * turn
                lead = torch.cat((z.real, z.imag), -1)
            out[name] = torch.cat((lead, x[..., n:]), -1).reshape(s[name].shape)
        out["v"] = s["v"].double()
        for name in ("k", "v"):
            y = out[name]
            low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            power = torch.frexp(low).exponent  # (eight bits are kept)
            low = torch.ldexp(torch.floor(torch.ldexp(low, 8 - power)), power - 8)
            step = (high - low) / 15
            power = torch.frexp(step).exponent
            step = torch.ldexp(torch.ceil(torch.ldexp(step, 8 - power)), power - 8)
            out[name] = low + step * torch.round((y - low) / step)
        return out
    q = s["q"].reshape(-1, hk, group, d).double()
    got, at = [], 0
    if case["op"] == "prefix":
        group_of = [g for g, many in enumerate(s["shared"]) for _ in range(many)]
        ahead = [_tokens(s, s["prefix_table"][g, :-(-int(t) // page)]) for g, t in enumerate(s["prefix_lens"])]
        for i, (r, t) in enumerate(zip(rows, lengths)):
            m = int(s["prefix_lens"][group_of[i]])
            k, v = (torch.cat((x[:, :m], y[:, :t]), 1)
                    for x, y in zip(ahead[group_of[i]], _tokens(s, s["table"][i, :-(-t // page)])))
            w = torch.einsum("rhgd,hnd->hgrn", q[at:at + r], k) * d ** -0.5
            later = torch.ones(r, m + t, dtype=torch.bool, device=w.device).triu(m + t - r + 1)
            w = torch.softmax(w.masked_fill(later, -math.inf), -1)
            got.append(torch.einsum("hgrn,hnd->rhgd", w, v).reshape(r, hk * group, d))
            at += r
        return torch.cat(got).reshape(s["q"].shape)
    means, chosen = s["means"].double(), []
    width = case["first"] + case["top"] + case["last"]
    for i, (r, t) in enumerate(zip(rows, lengths)):
        entries = s["table"][i, :-(-t // page)].long()
        for j in range((t - r) // page, entries.numel()):
            k, _ = _tokens(s, entries[j:j + 1])
            means[entries[j]] = k[:, :t - j * page].mean(1)
    held = means.float().to(torch.bfloat16).double()  # what the next step reads
    for i, (r, t) in enumerate(zip(rows, lengths)):
        entries = s["table"][i, :-(-t // page)].long()
        for p in range(t - r, t):
            mine = p // page
            free = torch.arange(case["first"], max(mine - case["last"] + 1, case["first"]), device=entries.device)
            score = (held[entries[free]] * q[at].sum(1)).sum(-1)  # (pages, heads)
            best = free[torch.argsort(-score, dim=0, stable=True)[:case["top"]]]  # (picked, heads)
            taken = torch.zeros(mine + 1, hk, dtype=torch.bool, device=entries.device)
            taken[:case["first"]] = True
            taken[max(mine + 1 - case["last"], 0):] = True
            taken[best, torch.arange(hk, device=entries.device)] = True
            many = int(taken[:, 0].sum())
            mark = taken.T.nonzero()[:, 1].view(hk, many)  # ascending
            kv = s["cache"][entries[mark], torch.arange(hk, device=entries.device)[:, None]]  # (heads, pages, 2, bytes)
            k, v = _tokens({**s, "cache": kv.flatten(0, 1)[:, None]}, torch.arange(hk * many, device=entries.device))
            k, v = k.view(hk, many * page, d), v.view(hk, many * page, d)
            place = (mark[..., None] * page + torch.arange(page, device=entries.device)).flatten(1)
            w = torch.einsum("hgd,hnd->hgn", q[at], k) * d ** -0.5
            w = torch.softmax(w.masked_fill(place[:, None] > p, -math.inf), -1)
            got.append(torch.einsum("hgn,hnd->hgd", w, v).reshape(hk * group, d))
            chosen.append(torch.nn.functional.pad(mark, (0, width - many), value=-1))
            at += 1
    return {"y": torch.stack(got).reshape(s["q"].shape), "pages": torch.stack(chosen).to(torch.int32), "means": means}
