"""penta_cache -- keys and values of past tokens held in 4 bits, in pages, and
causal attention over them.  Not in the reference, whose GPT recomputes the
whole prefix for every token (train_pentagpt.py:46-136).

    cache = kv4_cache(n_pages, n_kv_heads, head_dim, page_size=64)
    kv4_append(k, v, cache, block_table, seq_lens)        store new tokens
    y = kv4_attention(q, cache, block_table, seq_lens)    attend over the cache
    k, v = kv4_gather(cache, head_dim, block_table, seq_lens, rows)

and, of the same cache, for decoders with rotated positions, for batches that share a
prefix, and for long contexts read in part:

    q = kv4_append_rotary(q, k, v, cos, sin, cache, block_table, seq_lens)
    y = kv4_prefix_attention(q, cache, block_table, seq_lens, prefix_table, prefix_lens)
    kv4_page_means(cache, means, block_table, seq_lens, rows)
    y = kv4_sparse_attention(q, cache, means, block_table, seq_lens, top_pages)

One vector of head_dim values takes head_dim / 2 bytes of codes and four bytes of
bf16 (scale, zero): 3.8x (head_dim 128) or 3.6x (64) less than bf16.  Every value
is held to within half a step, a step being a fifteenth of the vector's range, so
what four bits cost depends on how alike a vector's dims are.  Measured on normal
random data (1024 tokens), the attention output moves against unquantised keys and
values by 13 % (head_dim 64) or 14 % (128) of its norm; with two key dims 5x louder
than the rest, which take the range of every key, by 28 % or 26 %, 12x louder by 46 %
or 63 %.  A vector whose range is no finite number reads back as NaN.

A sequence's page i (block_table[b, i]) holds its positions [i * page_size,
(i + 1) * page_size).  seq_lens[b] counts the sequence's tokens WITH the rows of
the call: the rows are its newest positions.  Rows come as (B, L, heads,
head_dim), L for each sequence, or as (T, heads, head_dim) with cu_q (B + 1)
int32, never falling, sequence b having rows [cu_q[b], cu_q[b + 1]) (without cu_q:
T / B each).
Lengths, tables and cu_q are read on the GPU, so a captured CUDA graph follows
their contents.  A block-table entry outside the cache, and a position behind the
table's end, is skipped (not stored, not attended to) and shows in
penta_native.device_status().  Sequences may share a page that the call stores
nothing to.
"""
from __future__ import annotations

import functools

import torch

try:
    from . import penta_native as _nat
except ImportError:  # flat import (this directory on sys.path, as a drop-in)
    import penta_native as _nat

_FLOATS = {torch.float32: _nat.PN_F32, torch.bfloat16: _nat.PN_BF16}
HEAD_DIMS = (64, 128)


def block_bytes(page_size: int, head_dim: int) -> int:
    """Bytes of one page of one kv head's keys (or values)."""
    return page_size * (head_dim // 2 + 4)


def kv4_cache(n_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64, device="cuda") -> torch.Tensor:
    """An empty cache: uint8 (n_pages, n_kv_heads, 2, block_bytes), keys at index 0
    of the third axis, values at 1."""
    assert head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {head_dim}"
    assert page_size >= 16 and page_size % 16 == 0, f"page_size must be a multiple of 16, got {page_size}"
    return torch.zeros(n_pages, n_kv_heads, 2, block_bytes(page_size, head_dim), dtype=torch.uint8, device=device)


def _cache_args(cache, head_dim, block_table, seq_lens, cu_q, device):
    """(n_pages, kv heads, page size) after the checks that every call shares.
    device: the rows' (index)."""
    assert head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {head_dim}"
    assert cache.dtype == torch.uint8 and cache.dim() == 4 and cache.shape[2] == 2 and cache.is_contiguous(), \
        "cache must be a contiguous uint8 tensor of kv4_cache"
    n, hk, _, size = cache.shape
    page, rest = divmod(size, head_dim // 2 + 4)
    assert rest == 0 and page >= 16 and page % 16 == 0, f"cache blocks of {size} bytes do not fit head_dim {head_dim}"
    assert block_table.dtype == torch.int32 and block_table.dim() == 2, "block_table must be a (B, pages) int32 tensor"
    B, W = block_table.shape
    assert W <= 1 or block_table.stride(1) == 1, "block_table rows must be contiguous"
    assert B <= 1 or block_table.stride(0) >= W, "block_table rows must not overlap"
    assert seq_lens.dtype == torch.int32 and seq_lens.shape == (B,) and seq_lens.is_contiguous(), \
        f"seq_lens must be a contiguous ({B},) int32 tensor"
    assert cache.get_device() == block_table.get_device() == seq_lens.get_device() == device, \
        "cache, block_table and seq_lens must be on the rows' device"
    if cu_q is not None:
        assert cu_q.dtype == torch.int32 and cu_q.shape == (B + 1,) and cu_q.is_contiguous() and cu_q.get_device() == device, \
            f"cu_q must be a contiguous ({B + 1},) int32 tensor on the rows' device"
    return n, hk, page


@functools.lru_cache(maxsize=4096)
def _attention_workspace(B, T, H, hk, D, device_index):
    with torch.cuda.device(device_index):
        return int(_nat.load().pn_kv4_attention_workspace_size(B, T, H, hk, D))


def _rows(x, B, cu_q, what):
    """Strides (sequence, row, head) in elements and the number of rows of
    (B, L, heads, head_dim) or (T, heads, head_dim)."""
    if x.dim() == 4:
        assert cu_q is None and x.shape[0] == B, f"{what}: (B, L, heads, head_dim) goes without cu_q, B as in block_table"
        return x.stride(0), x.stride(1), x.stride(2), x.shape[0] * x.shape[1]
    assert x.dim() == 3, f"{what} must be (B, L, heads, head_dim) or (T, heads, head_dim)"
    T = x.shape[0]
    if cu_q is None:
        assert T == 0 if B == 0 else T % B == 0, f"{what}: {T} rows over {B} sequences need cu_q"
        return x.stride(0) * (T // B if B else 0), x.stride(0), x.stride(1), T
    return 0, x.stride(0), x.stride(1), T


def _count(rows, B, cu_q):
    """The number of rows of a leading shape (B, L) or (T,)."""
    if len(rows) == 2:
        assert cu_q is None and rows[0] == B, "rows: (B, L) goes without cu_q, B as in block_table"
        return rows[0] * rows[1]
    assert len(rows) == 1, "rows must be (B, L) or (T,)"
    assert cu_q is not None or (rows[0] == 0 if B == 0 else rows[0] % B == 0), f"{rows[0]} rows over {B} sequences need cu_q"
    return rows[0]


def _inner(x):
    """x with a contiguous last dimension."""
    return x if x.stride(-1) == 1 else x.contiguous()


def _out(q, out, cu_q):
    """`out` after its checks, or a new tensor for rows like q's."""
    if out is None:
        return (torch.empty if cu_q is None else torch.zeros)(q.shape, dtype=q.dtype, device=q.device)
    assert out.shape == q.shape and out.dtype == q.dtype and out.get_device() == q.get_device() and out.is_contiguous(), \
        "out must be a contiguous tensor of q's shape, type and device"
    return out


def kv4_append(k: torch.Tensor, v: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
               cu_q: torch.Tensor | None = None) -> None:
    """Quantise the rows' keys and values (bf16/fp32, any row and head strides)
    into the cache, at the newest positions of their sequences."""
    assert k.is_cuda, "kv4_append requires CUDA tensors"
    assert k.dtype in _FLOATS and v.dtype == k.dtype and v.shape == k.shape and v.get_device() == k.get_device(), \
        "k and v must be bfloat16 or float32 tensors of one shape, type and device"
    D = k.shape[-1]
    n, hk, page = _cache_args(cache, D, block_table, seq_lens, cu_q, k.get_device())
    assert k.shape[-2] == hk, f"k has {k.shape[-2]} heads, the cache {hk}"
    k, v = _inner(k), _inner(v)
    B, W = block_table.shape
    kb, kl, kh, T = _rows(k, B, cu_q, "k")
    vb, vl, vh, _ = _rows(v, B, cu_q, "v")
    with _nat.device_of(k):
        _nat.check(_nat.load().pn_kv4_append(k.data_ptr(), kb, kl, kh, v.data_ptr(), vb, vl, vh, _FLOATS[k.dtype],
                                             cache.data_ptr(), n, hk, page, D, block_table.data_ptr(),
                                             max(block_table.stride(0), W), W, seq_lens.data_ptr(), _nat.ptr(cu_q), B, T,
                                             _nat.stream_of(k)), "kv4_append")


def kv4_append_rotary(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                      cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                      cu_q: torch.Tensor | None = None, offsets: torch.Tensor | None = None, interleaved: bool = False,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate the rows' positions into their queries and keys, store keys and values as
    kv4_append does, and return the queries (q's shape and type).

    q, k, v: bf16/fp32 rows of one type, any row and head strides, as a projection leaves
    them side by side.  cos, sin: (positions, R / 2) float32 tables, R a multiple of 16 up
    to head_dim: of the first R dims pair (a, b) becomes (a cos - b sin, b cos + a sin) in
    fp32, pairs being (i, i + R / 2), or (2i, 2i + 1) where interleaved; the other dims pass
    as they are.  A row at position p of sequence b takes entry p + offsets[b] ((B,) int32;
    p without them), so a sequence behind a shared prefix has its length there.  A row
    whose entry the tables do not have is not stored, gives zeros, and shows in
    penta_native.device_status().  Keys are quantised without a rounding to bf16 in between.

    out: a contiguous tensor for the queries, which may be q itself but overlaps neither q
    otherwise nor k or v; rows of it behind cu_q[B] are left as they were (zeros where no out is
    given)."""
    assert q.is_cuda, "kv4_append_rotary requires CUDA tensors"
    dev, dtype, D = q.get_device(), q.dtype, q.shape[-1]
    assert dtype in _FLOATS and k.dtype == dtype and v.dtype == dtype and k.get_device() == v.get_device() == dev, \
        "q, k and v must be bfloat16 or float32 tensors of one type and device"
    n, hk, page = _cache_args(cache, D, block_table, seq_lens, cu_q, dev)
    H = q.shape[-2]
    assert H > 0 and k.shape == v.shape == (*q.shape[:-2], hk, D), \
        f"q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} must be the same rows, k and v of {hk} heads"
    assert cos.dtype == sin.dtype == torch.float32 and cos.dim() == 2 and cos.shape == sin.shape and \
        cos.stride() == sin.stride() and cos.get_device() == sin.get_device() == dev and cos.stride(1) == 1, \
        "cos and sin must be (positions, R / 2) float32 tensors alike, with contiguous rows, on the rows' device"
    P, half = cos.shape
    assert P <= 1 or cos.stride(0) >= half, "rows of cos and sin must not overlap"
    B, W = block_table.shape
    if offsets is not None:
        assert offsets.dtype == torch.int32 and offsets.shape == (B,) and offsets.is_contiguous() and \
            offsets.get_device() == dev, f"offsets must be a contiguous ({B},) int32 tensor on the rows' device"
    q, k, v = _inner(q), _inner(k), _inner(v)
    qb, ql, qh, T = _rows(q, B, cu_q, "q")
    kb, kl, kh, _ = _rows(k, B, cu_q, "k")
    vb, vl, vh, _ = _rows(v, B, cu_q, "v")
    rest = out is None and B > 0  # (the kernel writes the zeros: a fill of all rows cost a fifth of the call)
    out = torch.empty(q.shape, dtype=dtype, device=q.device) if rest else _out(q, out, cu_q)
    with _nat.device_of(q):
        _nat.check(_nat.load().pn_kv4_append_rotary(
            q.data_ptr(), qb, ql, qh, H, k.data_ptr(), kb, kl, kh, v.data_ptr(), vb, vl, vh, _FLOATS[dtype], cos.data_ptr(),
            sin.data_ptr(), P, max(cos.stride(0), half), 2 * half, int(interleaved), _nat.ptr(offsets), cache.data_ptr(), n, hk,
            page, D, block_table.data_ptr(), max(block_table.stride(0), W), W, seq_lens.data_ptr(), _nat.ptr(cu_q), B, T,
            out.data_ptr(), int(rest), _nat.stream_of(q)), "kv4_append_rotary")
    return out


def kv4_gather(cache: torch.Tensor, head_dim: int, block_table: torch.Tensor, seq_lens: torch.Tensor, rows,
               cu_q: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16
               ) -> tuple[torch.Tensor, torch.Tensor]:
    """The keys and values of the newest rows of each sequence as the cache holds
    them: rows is (B, L) or (T,), the leading shape of the result (*rows, heads,
    head_dim).  Rows behind cu_q[B], and rows before a sequence's start, are zeros."""
    assert cache.is_cuda, "kv4_gather requires CUDA tensors"
    assert dtype in _FLOATS
    rows = tuple(rows)
    n, hk, page = _cache_args(cache, head_dim, block_table, seq_lens, cu_q, cache.get_device())
    k = torch.empty((*rows, hk, head_dim), dtype=dtype, device=cache.device)
    v = torch.empty((*rows, hk, head_dim), dtype=dtype, device=cache.device)
    B, W = block_table.shape
    T = _rows(k, B, cu_q, "rows")[3]
    with _nat.device_of(cache):
        _nat.check(_nat.load().pn_kv4_gather(cache.data_ptr(), n, hk, page, head_dim, block_table.data_ptr(),
                                             max(block_table.stride(0), W), W, seq_lens.data_ptr(), _nat.ptr(cu_q), B, T,
                                             k.data_ptr(), v.data_ptr(), _FLOATS[dtype], _nat.stream_of(cache)),
                   "kv4_gather")
    return k, v


def kv4_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                  cu_q: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None
                  ) -> torch.Tensor:
    """Causal attention of the rows q (bf16/fp32, any row and head strides) over
    their sequences' cached tokens: the row at position p sees positions 0 .. p,
    its own included, so append the rows' keys and values first.  Returns q's
    shape and type.

    Query heads are a multiple of the cache's kv heads; head h reads kv head
    h // (heads / kv heads).  scale > 0 defaults to head_dim ** -0.5.  A row that sees
    nothing gives zeros.  out: a contiguous tensor to write to; rows of it
    behind cu_q[B] are left as they were (zeros where no out is given).

    The products take 11 bits of fp32 queries (all of bf16 ones) and 11 of a token's
    weight times its value scale, relative to the largest such scale that the row
    sees; sums and the softmax are fp32, and 16 tokens' products cost a sum no more than
    2^-24 of the result, however far its terms cancel.  A value vector's range
    (largest less smallest) is taken from 2^-50 to 2^110: smaller ones lose some of
    these 11 bits, larger ones may give infinities."""
    assert q.is_cuda and q.dtype in _FLOATS, "kv4_attention takes bfloat16 or float32 CUDA queries"
    D = q.shape[-1]
    dev = q.get_device()
    n, hk, page = _cache_args(cache, D, block_table, seq_lens, cu_q, dev)
    H = q.shape[-2]
    assert H > 0 and H % hk == 0, f"{H} query heads are no multiple of {hk} kv heads"
    q = _inner(q)
    B, W = block_table.shape
    sb, sl, sh, T = _rows(q, B, cu_q, "q")
    out = _out(q, out, cu_q)
    size = _attention_workspace(B, T, H, hk, D, dev)
    with _nat.device_of(q):
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        _nat.check(_nat.load().pn_kv4_attention(q.data_ptr(), sb, sl, sh, _FLOATS[q.dtype], H, cache.data_ptr(), n, hk, page,
                                                D, block_table.data_ptr(), max(block_table.stride(0), W), W,
                                                seq_lens.data_ptr(), _nat.ptr(cu_q), B, T,
                                                D ** -0.5 if scale is None else scale, out.data_ptr(), ws.data_ptr(), size,
                                                _nat.stream_of(q)), "kv4_attention")
    return out


@functools.lru_cache(maxsize=4096)
def _prefix_workspace(B, T, P, H, hk, D, device_index):
    with torch.cuda.device(device_index):
        return int(_nat.load().pn_kv4_prefix_attention_workspace_size(B, T, P, H, hk, D))


def kv4_prefix_attention(q: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                         prefix_table: torch.Tensor, prefix_lens: torch.Tensor, cu_q: torch.Tensor | None = None,
                         cu_prefix: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None
                         ) -> torch.Tensor:
    """kv4_attention of sequences behind shared prefixes, whose tokens are read once for
    all rows that see them.

    prefix_table (P, pages) int32 and prefix_lens (P,) int32 hold P prefixes as block_table
    and seq_lens hold the B sequences, in pages of the same cache.  Sequences
    [cu_prefix[g], cu_prefix[g + 1]) share prefix g (cu_prefix (P + 1) int32, never falling;
    without it B / P sequences each); sequences outside have none.  A row sees all of its
    prefix and then its sequence's own tokens up to its position, which block_table and
    seq_lens count from 0.  The rest is as in kv4_attention, its precision over either
    part included; the two parts are joined in fp32."""
    assert q.is_cuda and q.dtype in _FLOATS, "kv4_prefix_attention takes bfloat16 or float32 CUDA queries"
    D = q.shape[-1]
    dev = q.get_device()
    n, hk, page = _cache_args(cache, D, block_table, seq_lens, cu_q, dev)
    _cache_args(cache, D, prefix_table, prefix_lens, None, dev)
    H = q.shape[-2]
    assert H > 0 and H % hk == 0, f"{H} query heads are no multiple of {hk} kv heads"
    B, W = block_table.shape
    P, PW = prefix_table.shape
    if cu_prefix is not None:
        assert cu_prefix.dtype == torch.int32 and cu_prefix.shape == (P + 1,) and cu_prefix.is_contiguous() and \
            cu_prefix.get_device() == dev, f"cu_prefix must be a contiguous ({P + 1},) int32 tensor on the rows' device"
    else:
        assert P == 0 or B % P == 0, f"{B} sequences over {P} prefixes need cu_prefix"
    q = _inner(q)
    sb, sl, sh, T = _rows(q, B, cu_q, "q")
    out = _out(q, out, cu_q)
    size = _prefix_workspace(B, T, P, H, hk, D, dev)
    with _nat.device_of(q):
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        _nat.check(_nat.load().pn_kv4_prefix_attention(
            q.data_ptr(), sb, sl, sh, _FLOATS[q.dtype], H, cache.data_ptr(), n, hk, page, D, block_table.data_ptr(),
            max(block_table.stride(0), W), W, seq_lens.data_ptr(), _nat.ptr(cu_q), B, T, prefix_table.data_ptr(),
            max(prefix_table.stride(0), PW), PW, prefix_lens.data_ptr(), _nat.ptr(cu_prefix), P,
            D ** -0.5 if scale is None else scale, out.data_ptr(), ws.data_ptr(), size, _nat.stream_of(q)),
            "kv4_prefix_attention")
    return out


def kv4_means(cache: torch.Tensor, head_dim: int) -> torch.Tensor:
    """A bf16 tensor (n_pages, n_kv_heads, head_dim) for the mean keys of the cache's pages."""
    assert head_dim in HEAD_DIMS, f"head_dim must be one of {HEAD_DIMS}, got {head_dim}"
    return torch.zeros(cache.shape[0], cache.shape[1], head_dim, dtype=torch.bfloat16, device=cache.device)


def _means_args(means, cache, dev):
    assert means.dtype == torch.bfloat16 and means.dim() == 3 and means.shape[:2] == cache.shape[:2] and \
        means.is_contiguous() and means.get_device() == dev, \
        "means must be a contiguous bfloat16 (n_pages, n_kv_heads, head_dim) tensor on the cache's device (kv4_means)"


def kv4_page_means(cache: torch.Tensor, means: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, rows,
                   cu_q: torch.Tensor | None = None) -> None:
    """Bring means up to date for the pages that the newest rows of each sequence are in
    (rows as in kv4_gather: (B, L) or (T,)): the mean of the keys that a page holds, summed
    in 64 bits.  After kv4_append or kv4_append_rotary of the same rows."""
    assert cache.is_cuda, "kv4_page_means requires CUDA tensors"
    dev = cache.get_device()
    _means_args(means, cache, dev)
    D = means.shape[2]
    n, hk, page = _cache_args(cache, D, block_table, seq_lens, cu_q, dev)
    B, W = block_table.shape
    rows = tuple(rows)
    T = _count(rows, B, cu_q)
    with _nat.device_of(cache):
        _nat.check(_nat.load().pn_kv4_page_means(cache.data_ptr(), n, hk, page, D, block_table.data_ptr(),
                                                 max(block_table.stride(0), W), W, seq_lens.data_ptr(), _nat.ptr(cu_q), B, T,
                                                 means.data_ptr(), _nat.stream_of(cache)), "kv4_page_means")


@functools.lru_cache(maxsize=4096)
def _sparse_workspace(T, H, hk, D, W, width, device_index):
    with torch.cuda.device(device_index):
        return int(_nat.load().pn_kv4_sparse_attention_workspace_size(T, H, hk, D, W, width))


def kv4_sparse_attention(q: torch.Tensor, cache: torch.Tensor, means: torch.Tensor, block_table: torch.Tensor,
                         seq_lens: torch.Tensor, top_pages: int, first_pages: int = 1, last_pages: int = 2,
                         cu_q: torch.Tensor | None = None, scale: float | None = None, out: torch.Tensor | None = None,
                         return_pages: bool = False):
    """kv4_attention over some of the cached pages, chosen for each row and kv head.

    A row whose position is in page j of its sequence attends to the first first_pages
    pages, to the last last_pages (at least one: page j itself, up to its position) and to
    the top_pages of the others with the largest scores (sum of the kv head's queries) .
    mean key (means, kept by kv4_page_means), in 64 bits, ties by the lowest page, a NaN score
    and an entry that is no page last; all pages where there are no more.  With return_pages also the choice: int32 (*rows, kv heads,
    first_pages + top_pages + last_pages), the pages' numbers in the sequence, ascending,
    then -1.

    What is read is the means (head_dim * 2 bytes per page and kv head) and the chosen
    pages; a row's pages are its own, so rows of a prompt that choose alike read them
    again.  The rest is as in kv4_attention."""
    assert q.is_cuda and q.dtype in _FLOATS, "kv4_sparse_attention takes bfloat16 or float32 CUDA queries"
    D = q.shape[-1]
    dev = q.get_device()
    n, hk, page = _cache_args(cache, D, block_table, seq_lens, cu_q, dev)
    _means_args(means, cache, dev)
    assert means.shape[2] == D, f"means of {means.shape[2]} dims, heads of {D}"
    H = q.shape[-2]
    assert H > 0 and H % hk == 0, f"{H} query heads are no multiple of {hk} kv heads"
    assert top_pages >= 0 and first_pages >= 0 and last_pages >= 1, \
        f"top_pages={top_pages}, first_pages={first_pages}, last_pages={last_pages} (the last at least 1)"
    q = _inner(q)
    B, W = block_table.shape
    sb, sl, sh, T = _rows(q, B, cu_q, "q")
    out = _out(q, out, cu_q)
    width = first_pages + top_pages + last_pages
    size = _sparse_workspace(T, H, hk, D, W, width, dev)
    with _nat.device_of(q):
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        chosen = None
        if return_pages:
            shape = (*q.shape[:-2], hk, width)
            chosen = torch.empty(shape, dtype=torch.int32, device=q.device)
            if B == 0:  # (rows of no sequence)
                chosen.fill_(-1)
        _nat.check(_nat.load().pn_kv4_sparse_attention(
            q.data_ptr(), sb, sl, sh, _FLOATS[q.dtype], H, cache.data_ptr(), means.data_ptr(), n, hk, page, D,
            block_table.data_ptr(), max(block_table.stride(0), W), W, seq_lens.data_ptr(), _nat.ptr(cu_q), B, T, first_pages,
            last_pages, top_pages, D ** -0.5 if scale is None else scale, out.data_ptr(), _nat.ptr(chosen), ws.data_ptr(), size,
            _nat.stream_of(q)), "kv4_sparse_attention")
    return (out, chosen) if return_pages else out
