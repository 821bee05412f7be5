"""Operators of a serving step, as cases to time: each in its plain form
(elementary torch operations) and, with `own` set, as the calls a user makes of
this package.

    norm       residual add + root-mean-square norm, rounded to the input of a
               projection: bf16, or int8 per token with its scale and row sum
               (penta_kernel.rms_norm, rms_norm_i8)
    append     new keys and values quantised into a paged 4-bit cache, read
               back as the values they stand for (penta_cache.kv4_append,
               kv4_gather)
    attention  causal attention of the newest rows of each sequence over that
               cache (penta_cache.kv4_attention)
    sample     one token per row from given uniform numbers, after temperature,
               top-k, min-p and top-p (penta_kernel.sample_tokens)

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


def _kernel():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import penta_kernel
    return penta_kernel


def _cache():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    import penta_cache
    return penta_cache


# ── cases ────────────────────────────────────────────────────────────────────

def listed():
    return [
        # one decoded token of the 124M GPT (width 768), into its int8 projection
        dict(name="norm i8, one token", op="norm", rows=1, width=768, dtype="bf16", out="i8", residual=True),
        # a prefill chunk of an 8192-wide decoder, into its int8 projection
        dict(name="norm i8, prefill 8192", op="norm", rows=4096, width=8192, dtype="bf16", out="i8", residual=True),
        # an odd width with fp32 activations and no residual: the last norm before the lm_head
        dict(name="norm bf16, odd rows", op="norm", rows=1021, width=1001, dtype="f32", out="bf16", residual=False),
        # the keys and values of one decode step of 64 sequences
        dict(name="append, decode step", op="append", batch=64, q_len=1, ragged=False, kv_heads=8, group=8, head_dim=128,
             page=64, length=4096),
        # the prompts of several requests stored at once, of unequal lengths
        dict(name="append, ragged prompts", op="append", batch=7, q_len=2047, ragged=True, kv_heads=8, group=8,
             head_dim=128, page=32, length=2047),
        # one sequence of the 124M GPT at the end of its block
        dict(name="attention, one short row", op="attention", batch=1, q_len=1, ragged=False, kv_heads=12, group=1,
             head_dim=64, page=64, length=1024),
        # a decode step of 32 requests of very different ages, grouped heads
        dict(name="attention, ragged decode", op="attention", batch=32, q_len=1, ragged=False, kv_heads=8, group=8,
             head_dim=128, page=64, length=8191),
        # one very long document, a single new token
        dict(name="attention, long decode", op="attention", batch=1, q_len=1, ragged=False, kv_heads=8, group=4,
             head_dim=128, page=128, length=131072),
        # prompt chunks of unequal lengths behind what is cached already
        dict(name="attention, ragged chunks", op="attention", batch=5, q_len=512, ragged=True, kv_heads=8, group=4,
             head_dim=128, page=64, length=4096),
        # one sequence, the 124M GPT's vocabulary
        dict(name="sample, one row", op="sample", rows=1, vocab=50257, dtype="bf16", temperature=0.8, top_k=50, top_p=0.95,
             min_p=0.0, per_row=False),
        # a batch whose requests each have settings of their own
        dict(name="sample, settings per row", op="sample", rows=64, vocab=50257, dtype="f32", temperature=1.0, top_k=40,
             top_p=0.9, min_p=0.05, per_row=True),
        # a large batch over a large vocabulary, nucleus only
        dict(name="sample, large nucleus", op="sample", rows=256, vocab=131071, dtype="bf16", temperature=1.0, top_k=0,
             top_p=0.9, min_p=0.0, per_row=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "append", "attention", "attention", "sample"])
    if op == "norm":
        width = _log(rng, 64, 16384)
        width = width if rng.random() < 0.3 else max(64, width // 64 * 64)
        rows = _log(rng, 1, max(2, min(8192, (2048 * 8192) // width)))
        return dict(op=op, rows=rows, width=width, dtype=rng.choice(["bf16", "bf16", "f32"]),
                    out=rng.choice(["i8", "i8", "bf16"]), residual=rng.random() < 0.7)
    if op == "sample":
        vocab = _log(rng, 257, 131071)
        return dict(op=op, rows=_log(rng, 1, max(2, min(256, 256 * 131071 // vocab))), vocab=vocab,
                    dtype=rng.choice(["bf16", "f32"]), temperature=round(rng.uniform(0.3, 1.5), 3),
                    top_k=rng.choice([0, 1, 20, 50, 200, 1000]), top_p=rng.choice([1.0, 0.95, 0.9, 0.5]),
                    min_p=rng.choice([0.0, 0.0, 0.02, 0.1]), per_row=rng.random() < 0.5)
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    group = rng.choice([1, 2, 3, 4, 6, 8, 16])
    head_dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128, 256])
    if op == "append":
        q_len = 1 if rng.random() < 0.4 else _log(rng, 2, 2047)
        batch = _log(rng, 1, max(2, min(128, 8192 // q_len)))
        return dict(op=op, batch=batch, q_len=q_len, ragged=q_len > 1 and rng.random() < 0.6, kv_heads=kv_heads, group=group,
                    head_dim=head_dim, page=page, length=max(q_len, _log(rng, 64, 4096)))
    long = _log(rng, 64, 65536)
    if rng.random() < 0.6:
        q_len = rng.choice([1, 1, 1, 2, 4, 7])
        batch = _log(rng, 1, max(2, min(64, 262144 * 8 // (long * kv_heads) // 2)))
    else:
        long = min(long, 4096)
        q_len = _log(rng, 8, min(512, long))
        batch = _log(rng, 1, 4)
        group = min(group, max(1, 32 // kv_heads))
    return dict(op="attention", batch=batch, q_len=min(q_len, long), ragged=q_len > 1 and rng.random() < 0.5,
                kv_heads=kv_heads, group=group, head_dim=head_dim, page=page, length=long)


def _rows_of(case):
    """New rows of each sequence: all alike, or from the longest down to a quarter of it."""
    b, n = case["batch"], case["q_len"]
    if not case["ragged"]:
        return [n] * b
    return [max(1, n - (3 * n * i) // (4 * b)) for i in range(b)]


def _lengths_of(case):
    """Tokens of each sequence with its new rows: from the longest down to a tenth of it, none a round number."""
    b, n = case["batch"], case["length"]
    return [max(r, n - (9 * n * i) // (10 * b) - (37 * i) % 13) for i, r in enumerate(_rows_of(case))]


# ── inputs ───────────────────────────────────────────────────────────────────

def _gen(seed, device):
    return torch.Generator(device=device).manual_seed(1234567 + int(seed))


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


def _over(x, n):
    """x / n, correctly rounded (a division by a Python number multiplies by its reciprocal on the GPU)."""
    return x / torch.full_like(x, n)


def _quantise(x):
    """(..., d) -> codes (..., d) uint8, scale (...), zero (...): the range of each vector in 15 steps."""
    x = x.float()
    zero = _round_down(x.amin(-1))
    scale = _round_up(_over(x.amax(-1) - zero, 15))
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
    dtype = {"bf16": torch.bfloat16, "f32": torch.float32}[case.get("dtype", "bf16")]
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        # a residual stream with a few loud channels, as decoders have
        loud = torch.where(torch.rand(width, generator=g, device=device) < 0.01, 12.0, 1.0)
        s["x"] = (normal(rows, width) * loud).to(dtype)
        s["r"] = (normal(rows, width) * loud * 2).to(dtype) if case["residual"] else None
        s["w"] = 1 + 0.2 * normal(width)
        s["eps"] = 1e-6
        return s
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a bulk of unlikely tokens and a few hundred that compete
        likely = torch.rand(rows, vocab, generator=g, device=device) * vocab < 300
        s["x"] = (normal(rows, vocab) * 2 + normal(rows, vocab).abs() * 5 * likely).to(dtype)
        s["u"] = torch.rand(rows, generator=g, device=device)
        s["t"], s["k"], s["p"], s["m"] = case["temperature"], case["top_k"], case["top_p"], case["min_p"]
        if case["per_row"]:
            def spread(v):
                return v * (0.5 + 0.5 * torch.rand(rows, generator=g, device=device))
            s["t"], s["p"], s["m"] = spread(s["t"]), spread(s["p"]), spread(s["m"])
            s["k"] = torch.randint(case["top_k"] // 2, case["top_k"] + 1, (rows,), generator=g, device=device, dtype=torch.int32)
        return s
    b, hk, group, d, page = case["batch"], case["kv_heads"], case["group"], case["head_dim"], case["page"]
    rows, lengths = _rows_of(case), _lengths_of(case)
    per = -(-max(lengths) // page)
    used = sum(-(-n // page) for n in lengths)
    order = torch.randperm(used + 1, generator=g, device=device, dtype=torch.int32)
    table = torch.zeros(b, per, dtype=torch.int32, device=device)
    at = 0
    for i, n in enumerate(lengths):
        m = -(-n // page)
        table[i, :m] = order[at:at + m]
        at += m
    s["table"] = table
    s["lens"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    s["cu"] = torch.tensor([0] + rows, device=device).cumsum(0).to(torch.int32) if case["ragged"] else None
    # per row: its sequence and its position there
    s["seq"] = torch.repeat_interleave(torch.arange(b, device=device), torch.tensor(rows, device=device))
    s["pos"] = torch.cat([torch.arange(n - r, n, device=device) for r, n in zip(rows, lengths)])
    loud = torch.where(torch.rand(hk, 1, d, generator=g, device=device) < 0.03, 5.0, 1.0)
    if case["op"] == "append":
        s["cache"] = torch.zeros(used + 1, hk, 2, page * (d // 2 + 4), dtype=torch.uint8, device=device)
    else:
        s["cache"] = _lay_out((normal(used + 1, hk, page, d) * loud).to(torch.bfloat16),
                              normal(used + 1, hk, page, d).to(torch.bfloat16))
    # one projection's output holds queries, keys and values side by side
    qkv = normal(sum(rows), (group + 2) * hk, d)
    qkv[:, group * hk:(group + 1) * hk] *= loud[:, 0]
    qkv = qkv.to(torch.bfloat16)
    if case["ragged"]:
        parts = qkv.split((group * hk, hk, hk), dim=1)
    else:
        parts = qkv.view(b, case["q_len"], -1, d).split((group * hk, hk, hk), dim=2)
    s["q"], s["k"], s["v"] = parts
    return s


# ── one pass ─────────────────────────────────────────────────────────────────

def run(s):
    return {"norm": _norm, "append": _append, "attention": _attention, "sample": _sample}[s["op"]](s)


def _norm(s):
    if own:
        pk = _kernel()
        if s["out"] == "i8":
            q, scale, total, *h = pk.rms_norm_i8(s["x"], s["w"], s["eps"], residual=s["r"])
            return {"y": pk.dequantize_activations_i8(q, scale, s["width"]), "scale": scale, "total": total, "h": h}
        if s["r"] is None:
            return {"y": pk.rms_norm(s["x"], s["w"], s["eps"]), "h": []}
        y, h = pk.rms_norm(s["x"], s["w"], s["eps"], residual=s["r"])
        return {"y": y, "h": [h]}
    x = s["x"]
    h = x if s["r"] is None else (x.float() + s["r"].float()).to(x.dtype)
    rstd = (1 / (h.double().square().mean(-1, keepdim=True) + s["eps"]).sqrt()).float()
    y = h.float() * rstd * s["w"].float()
    h = [] if s["r"] is None else [h]
    if s["out"] == "bf16":
        return {"y": y.to(torch.bfloat16), "h": h}
    scale = _over(y.abs().amax(-1), 127)
    scale = torch.where(scale > 0, scale, torch.ones_like(scale))
    q = (y / scale[:, None]).round().clamp(-128, 127)
    return {"y": (q * scale[:, None]).to(torch.bfloat16), "scale": scale, "total": q.sum(-1).to(torch.int32), "h": h}


def _append(s):
    if own:
        pc = _cache()
        pc.kv4_append(s["k"], s["v"], s["cache"], s["table"], s["lens"], cu_q=s["cu"])
        rows = s["k"].shape[:-2]
        return pc.kv4_gather(s["cache"], s["head_dim"], s["table"], s["lens"], rows, cu_q=s["cu"])
    hk, d, page, cache = s["kv_heads"], s["head_dim"], s["page"], s["cache"]
    k, v = s["k"].reshape(-1, hk, d), s["v"].reshape(-1, hk, d)
    at = s["table"][s["seq"], s["pos"] // page].long()
    tok = s["pos"] % page
    kc, ks, kz = _quantise(k)
    vc, vs, vz = _quantise(v)
    codes = cache[..., :page * d // 2]
    pairs = cache[..., page * d // 2:].view(torch.bfloat16).view(-1, hk, 2, page, 2)
    codes[:, :, 0].view(-1, hk, page, d // 2)[at, :, tok] = kc[..., 0::2] | (kc[..., 1::2] << 4)
    codes[:, :, 1].view(-1, hk, page // 2, d // 4, 2, 2)[at, :, tok // 2, :, tok % 2] = (
        vc[..., 0::2] | (vc[..., 1::2] << 4)).view(-1, hk, d // 4, 2)
    pairs[at, :, 0, tok] = torch.stack((ks, kz), -1).to(torch.bfloat16)
    pairs[at, :, 1, tok] = torch.stack((vs, vz), -1).to(torch.bfloat16)
    shape = s["k"].shape
    return [(c.float() * scale[..., None] + zero[..., None]).to(torch.bfloat16).reshape(shape)
            for c, scale, zero in ((kc, ks, kz), (vc, vs, vz))]


def _unpack(pages, page, d):
    """Cache pages (..., heads, 2, bytes) as fp32 keys and values (..., heads, page, d)."""
    codes = pages[..., :page * d // 2]
    codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).float()
    pair = pages[..., page * d // 2:].contiguous().view(torch.bfloat16).unflatten(-1, (page, 2)).float()
    scale, zero = pair[..., :1], pair[..., 1:]
    k = codes[..., 0, :].unflatten(-1, (page, d))
    v = codes[..., 1, :].unflatten(-1, (page // 2, d // 4, 2, 4)).transpose(-3, -2).flatten(-2).flatten(-3, -2)
    return k * scale[..., 0, :, :] + zero[..., 0, :, :], v * scale[..., 1, :, :] + zero[..., 1, :, :]


def _attention(s):
    if own:
        return _cache().kv4_attention(s["q"], s["cache"], s["table"], s["lens"], cu_q=s["cu"])
    b, hk, group, d, page, n = s["batch"], s["kv_heads"], s["group"], s["head_dim"], s["page"], s["q_len"]
    keys, values = _unpack(s["cache"][s["table"].long()], page, d)
    keys = keys.transpose(1, 2).flatten(2, 3)  # (b, heads, tokens, d)
    values = values.transpose(1, 2).flatten(2, 3)
    # rows of unequal sequences side by side: row i of a sequence at its place from the end
    at = n - s["lens"][s["seq"]] + s["pos"]
    q = torch.zeros(b, n, hk * group, d, device=s["q"].device)
    q[s["seq"], at] = s["q"].reshape(-1, hk * group, d).float()
    q = q.view(b, n, hk, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)  # (b, heads, group * n, d)
    w = q @ keys.transpose(2, 3) / math.sqrt(d)
    seen = s["lens"][:, None] - n + torch.arange(n, device=w.device)  # the last position that each row sees
    hidden = torch.arange(w.shape[-1], device=w.device) > seen[..., None]
    w = w.view(b, hk, group, n, -1).masked_fill_(hidden[:, None, None], float("-inf"))
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-3e38))
    w = (w / w.sum(-1, keepdim=True)).flatten(2, 3)
    y = (w @ values).view(b, hk, group, n, d).permute(0, 3, 1, 2, 4).reshape(b, n, hk * group, d)
    return y[s["seq"], at].to(torch.bfloat16).reshape(s["q"].shape)


def _sample(s):
    if own:
        return _kernel().sample_tokens(s["x"], s["u"], temperature=s["t"], top_k=s["k"], top_p=s["p"], min_p=s["m"])
    x = s["x"].double()  # a number next to a border decides for a token: 64 bits
    rows, vocab = x.shape

    def column(v, dtype):
        return torch.as_tensor(v, device=x.device).to(dtype).expand(rows)[:, None]

    t, p, m = (column(v, torch.float32).double() for v in (s["t"], s["p"], s["m"]))
    k = column(s["k"], torch.int64)
    x, order = torch.sort(x, dim=-1, descending=True, stable=True)
    w = torch.exp((x - x[:, :1]) / t)
    rank = torch.arange(vocab, device=x.device)
    w = torch.where(((k <= 0) | (rank < k)) & (w >= m), w, torch.zeros_like(w))
    before = w.cumsum(-1) - w
    w = torch.where((p >= 1) | (before < p * w.sum(-1, keepdim=True)), w, torch.zeros_like(w))
    w = torch.zeros_like(w).scatter_(1, order, w)
    upto = w.cumsum(-1)
    return (upto > s["u"].double()[:, None] * upto[:, -1:]).to(torch.uint8).argmax(-1)


# ── what a pass cannot do without ────────────────────────────────────────────

def work(case):
    if case["op"] == "norm":
        n, wide = case["rows"] * case["width"], 2 if case["dtype"] == "bf16" else 4
        moved = n * wide * (3 if case["residual"] else 1) + n * (1 if case["out"] == "i8" else 2)
        return {"bytes": moved + 4 * case["width"] + (8 * case["rows"] if case["out"] == "i8" else 0), "flops": 6 * n}
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (2 if case["dtype"] == "bf16" else 4) + case["rows"] * (28 if case["per_row"] else 12), "flops": 4 * n}
    rows, lengths = _rows_of(case), _lengths_of(case)
    hk, group, d = case["kv_heads"], case["group"], case["head_dim"]
    held = 2 * hk * (d // 2 + 4)  # bytes of one token in the cache
    if case["op"] == "append":
        n = sum(rows)
        return {"bytes": n * (2 * 2 * hk * d * 2 + held), "flops": n * 2 * hk * d * 4}
    pairs = sum(r * n - r * (r - 1) // 2 for r, n in zip(rows, lengths))
    return {"bytes": sum(lengths) * held + 2 * 2 * sum(rows) * hk * group * d, "flops": 4 * pairs * hk * group * d}


# ── the same from the definitions, in 64 bits ────────────────────────────────

def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        h = s["x"].double()
        if s["r"] is not None:
            h = (h + s["r"].double()).to(s["x"].dtype).double()  # the stream itself is kept in its own type
        y = h / torch.sqrt((h * h).sum(1, keepdim=True) / case["width"] + s["eps"]) * s["w"].double()
        h = [h] if s["r"] is not None else []
        if case["out"] == "bf16":
            return {"y": y, "h": h}
        scale = torch.linalg.vector_norm(y, ord=float("inf"), dim=1) / 127
        return {"y": torch.round(y / scale[:, None]) * scale[:, None], "scale": scale, "total": None, "h": h}
    if case["op"] == "sample":
        got = []
        for i in range(case["rows"]):
            t, k, p, m = (float(v[i]) if case["per_row"] else v for v in (s["t"], s["k"], s["p"], s["m"]))
            if not case["per_row"]:  # a setting is held in 32 bits
                t, p, m = (float(torch.tensor(v, dtype=torch.float32)) for v in (t, p, m))
            x = s["x"][i].double()
            z = (x - x.max()) / t
            by = torch.argsort(-x, stable=True)
            by = by[:int(k)] if k > 0 else by
            by = by[torch.exp(z[by]) >= m]
            c = torch.softmax(z[by], 0).cumsum(0)
            if p < 1:
                by = by[:int((c < p).sum()) + 1]
            kept = by.sort().values
            c = torch.softmax(z[kept], 0).cumsum(0)
            got.append(kept[min(int((c <= float(s["u"][i]) * c[-1]).sum()), kept.numel() - 1)])
        return torch.stack(got)
    hk, group, d, page = case["kv_heads"], case["group"], case["head_dim"], case["page"]
    rows, lengths = _rows_of(case), _lengths_of(case)
    if case["op"] == "append":
        got = []
        for x in (s["k"], s["v"]):
            y = x.double()
            low, high = y.min(-1, keepdim=True).values, y.max(-1, keepdim=True).values
            step = (high - low) / 15
            step = torch.ldexp(torch.ceil(torch.ldexp(step, 8 - torch.frexp(step).exponent)), torch.frexp(step).exponent - 8)
            got.append(low + step * torch.round((y - low) / step))
        return got
    got, at = [], 0
    q = s["q"].reshape(-1, hk, group, d)
    for i, (r, n) in enumerate(zip(rows, lengths)):
        kv = s["cache"][s["table"][i, :-(-n // page)].long()].to(torch.int64)  # (pages, heads, 2, bytes)
        size = page * d // 2
        pair = (kv[..., size + 1::2] << 24 | kv[..., size::2] << 16).to(torch.int32).view(torch.float32).double()
        values = []
        for j in (0, 1):
            token, dim = torch.arange(page, device=kv.device)[:, None], torch.arange(d, device=kv.device)
            byte = (token * (d // 2) + dim // 2) if j == 0 else (token // 2 * d + dim // 4 * 4 + token % 2 * 2 + dim % 4 // 2)
            code = kv[:, :, j][:, :, byte] >> (dim % 2 * 4) & 15
            x = pair[:, :, j, 0::2, None] * code + pair[:, :, j, 1::2, None]
            values.append(x.transpose(0, 1).reshape(hk, -1, d)[:, :n])
        w = torch.einsum("rhgd,hnd->hgrn", q[at:at + r].double(), values[0]) * d ** -0.5
        ahead = torch.ones(r, n, dtype=torch.bool, device=w.device).triu(n - r + 1)
        w = torch.softmax(w.masked_fill(ahead, -math.inf), -1)
        got.append(torch.einsum("hgrn,hnd->rhgd", w, values[1]).reshape(r, hk * group, d))
        at += r
    return torch.cat(got).reshape(s["q"].shape)
