"""penta_cache -- keys and values of past tokens held in 4 bits, in pages, and
causal attention over them.  Not in the reference, whose GPT recomputes the
whole prefix for every token (train_pentagpt.py:46-136).

    cache = kv4_cache(n_pages, n_kv_heads, head_dim, page_size=64)
    kv4_append(k, v, cache, block_table, seq_lens)        store new tokens
    y = kv4_attention(q, cache, block_table, seq_lens)    attend over the cache
    k, v = kv4_gather(cache, head_dim, block_table, seq_lens, rows)

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


def _inner(x):
    """x with a contiguous last dimension."""
    return x if x.stride(-1) == 1 else x.contiguous()


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
    sees; sums and the softmax are fp32."""
    assert q.is_cuda and q.dtype in _FLOATS, "kv4_attention takes bfloat16 or float32 CUDA queries"
    D = q.shape[-1]
    dev = q.get_device()
    n, hk, page = _cache_args(cache, D, block_table, seq_lens, cu_q, dev)
    H = q.shape[-2]
    assert H > 0 and H % hk == 0, f"{H} query heads are no multiple of {hk} kv heads"
    q = _inner(q)
    B, W = block_table.shape
    sb, sl, sh, T = _rows(q, B, cu_q, "q")
    if out is None:
        out = (torch.empty if cu_q is None else torch.zeros)(q.shape, dtype=q.dtype, device=q.device)
    else:
        assert out.shape == q.shape and out.dtype == q.dtype and out.get_device() == dev and out.is_contiguous(), \
            "out must be a contiguous tensor of q's shape, type and device"
    size = _attention_workspace(B, T, H, hk, D, dev)
    with _nat.device_of(q):
        ws = torch.empty(size, dtype=torch.uint8, device=q.device)
        _nat.check(_nat.load().pn_kv4_attention(q.data_ptr(), sb, sl, sh, _FLOATS[q.dtype], H, cache.data_ptr(), n, hk, page,
                                                D, block_table.data_ptr(), max(block_table.stride(0), W), W,
                                                seq_lens.data_ptr(), _nat.ptr(cu_q), B, T,
                                                D ** -0.5 if scale is None else scale, out.data_ptr(), ws.data_ptr(), size,
                                                _nat.stream_of(q)), "kv4_attention")
    return out
