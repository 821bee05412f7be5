"""Calls of the 4-bit cache's further operators (penta_cache) that follow one another closely, and
the attention kernels that they reach with wide groups and many rows."""
import pytest
import torch

import kv4_more_oracle as more
import kv4_oracle as oracle
import penta_cache as pc
import penta_native as nat
from test_kv4_gpu import Batch
from test_kv4_more_gpu import Shared, cu_of, ints, sparse_check, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,rows,hk,G", [(1, 1, 1, 2), (5, 3, 2, 4), (60, 2, 2, 20)])
def test_sparse_calls_one_behind_the_other(cuda_device, B, rows, hk, G):
    """The choice of one call is written while its attention may wait already, into memory where the call before
    had its own: every call must see its own choice.  Back to back, in a graph, and one by one."""
    d, page, n = 64, 16, 40
    s = Batch([n * page - 3 * i for i in range(B)], hk, d, page, cuda_device, seed=B)
    means = pc.kv4_means(s.cache, d)
    pc.kv4_page_means(s.cache, means, s.table, s.lens, (sum(s.lengths),), cu_q=cu_of(s.lengths, cuda_device))
    g = torch.Generator().manual_seed(rows)
    qs = [torch.randn(B * rows, G * hk, d, generator=g).to(torch.bfloat16).to(cuda_device) for _ in range(8)]
    lens = [s.lens - 16 * page * (i % 2) for i in range(8)]  # other lengths too
    run = lambda i: pc.kv4_sparse_attention(qs[i], s.cache, means, s.table, lens[i], 5, return_pages=True)
    want = []
    for i in range(8):
        want.append([t.clone() for t in run(i)])
        torch.cuda.synchronize()
    assert not torch.equal(want[0][1], want[2][1])
    for _ in range(5):
        got = [run(i) for i in range(8)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(got, want) for a, b in zip(x, y))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = [run(i) for i in range(8)]
    for _ in range(5):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for x, y in zip(held, want) for a, b in zip(x, y))
    assert nat.device_status() == 0


def sparse_rows(s, q, cu, G, top, some, first=1, last=1):
    """One call over all rows; the rows `some`, (row, sequence, position), against the definition."""
    means = pc.kv4_means(s.cache, s.d)
    pc.kv4_page_means(s.cache, means, s.table, s.lens, (sum(s.lengths),), cu_q=cu_of(s.lengths, s.device))
    out = torch.full_like(q, 7.0)
    y, pages = pc.kv4_sparse_attention(q, s.cache, means, s.table, s.lens, top, first_pages=first, last_pages=last, cu_q=cu,
                                       out=out, return_pages=True)
    end = int(cu[-1])
    assert (y[end:] == 7).all() and (pages[end:] == -1).all()
    for row, i, pos in some:
        if pos < 0:
            assert not y[row].any() and (pages[row] == -1).all()
            continue
        want = more.choose(q[row].cpu(), more.means(s.k[i], s.page), pos, s.page, top, first, last)
        for h, chosen in enumerate(want):
            assert pages[row, h].tolist() == chosen + [-1] * (top + first + last - len(chosen)), (row, h)
            tok = torch.cat([torch.arange(p * s.page, min((p + 1) * s.page, pos + 1)) for p in chosen])
            part = slice(h * G, (h + 1) * G)
            ref, bound = oracle.attention(q[row][None, part].cpu(), s.k[i][tok][:, h:h + 1], s.v[i][tok][:, h:h + 1], None)
            bound = bound + 2.0 ** -8 * (ref.abs() + bound)
            err = (y[row, part].double().cpu() - ref[0]).abs()
            assert (err <= bound[0] + 1e-30).all(), (row, h, err.max())
    assert nat.device_status() == 0


# per sequence and kv head, G rows to a tile; tiles of 16 rows above four times the SMs take the kernel for 64 rows, and
# more than 64 of them per head and eight times the SMs the one for 128: 300 x 2 x 2 and x 3 tiles, 600 x 2 x 5
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("G,n_rows", [(20, 300), (40, 300), (70, 600)])
def test_sparse_wide_groups_and_many_rows(cuda_device, d, G, n_rows):
    """Tables per kv head in the kernels for many rows, rows before the sequence's start, rows of no sequence."""
    hk, page = 2, 16
    s = Batch([700, 5, 333], hk, d, page, cuda_device, seed=G + d)
    rows = [n_rows - 150, 9, 141]
    q = torch.randn(n_rows + 25, G * hk, d, generator=torch.Generator().manual_seed(G)).to(torch.bfloat16).to(cuda_device)
    at = [0, rows[0], rows[0] + 9]
    some = [(at[i] + r, i, s.lengths[i] - rows[i] + r) for i, some in
            enumerate(([0, 1, 77, rows[0] - 1], [0, 3, 4, 8], [0, 64, 140])) for r in some]
    sparse_rows(s, q, cu_of(rows, cuda_device), G, 4, some)


@pytest.mark.parametrize("d", [64, 128])
def test_prefix_own_rows_on_the_chunk_kernel(cuda_device, d):
    """40 sequences x 12 rows of 4 query heads each: their own tokens in the kernel for 64 rows, causal, ragged
    lengths, some rows before their sequence's start and some sequences without a prefix."""
    B, G, hk = 42, 4, 8
    own = [(53 * i) % 120 + 1 for i in range(B)]
    rows = [12 if i % 5 else 17 for i in range(B)]
    assert any(n < r for n, r in zip(own, rows))
    s = Shared(own, [200, 33, 0], [25, 10, 5], hk, d, 16, cuda_device, seed=d)
    q = torch.randn(sum(rows), G * hk, d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    y = s.call(q.to(cuda_device), rows)
    some = [0, 1, 7, 24, 25, 34, 35, 39, 40, 41] + [i for i in range(B) if own[i] < rows[i]][:3]
    part, x = y.split(rows), q.split(rows)
    whole = s.own, s.of, s.b.k, s.b.v
    for i in some:  # (all of them would take minutes)
        s.own, s.of = [whole[0][i]], [whole[1][i]]
        s.b.k, s.b.v = ([t[i]] + t[B:] for t in whole[2:])
        s.check([part[i]], [x[i]])
        s.own, s.of, s.b.k, s.b.v = whole
    assert nat.device_status() == 0


@pytest.mark.parametrize("d", [64, 128])
def test_page_means_of_the_largest_keys(cuda_device, d):
    """Keys whose range is nearly fp32's: fifteen times the scale, which is rounded up, is no fp32 number, the keys
    read back and their mean are."""
    page, n = 16, 37
    low, top = -2.0 ** 127, 2.0 ** 127 * (1 - 2.0 ** -8)  # (apart by less than the largest fp32 number)
    s = Batch([n], 2, d, page, cuda_device, seed=d)
    for i in range(n):
        s.k[0][i, :, i % d], s.k[0][i, :, (i + 7) % d] = low, top
    s.store([n])
    k, _ = pc.kv4_gather(s.cache, d, s.table, s.lens, (n,), dtype=torch.float32)
    assert k.isfinite().all()
    assert (oracle.quantise(s.k[0])[1] * 15).isinf().all()
    means = pc.kv4_means(s.cache, d)
    pc.kv4_page_means(s.cache, means, s.table, s.lens, (n,))
    assert torch.equal(means[s.table[0].long()].cpu(), more.means(s.k[0], page))


def test_sparse_workspace(cuda_device):
    """What a call holds for its scores has a limit, is nothing where none are made, and a list holds no more pages
    than there are, however many are asked for."""
    size = lambda T, W, width: pc._sparse_workspace(T, 32, 8, 128, W, width, cuda_device.index or 0)
    some = size(4096, 64, 64)  # no scores
    assert size(4096, 64, 1 << 20) == some and some < size(4096, 65, 64)
    assert size(4096, 8192, 64) - some < 300 << 20  # (2 GB of scores)
    assert size(1, 64, 1 << 20) < 64 << 20
    s = Batch([300, 170], 2, 64, 16, cuda_device, seed=2)
    means = pc.kv4_means(s.cache, 64)
    pc.kv4_page_means(s.cache, means, s.table, s.lens, (470,), cu_q=cu_of(s.lengths, cuda_device))
    q = torch.randn(2, 8, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda_device)
    want = pc.kv4_sparse_attention(q, s.cache, means, s.table, s.lens, 19)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    assert torch.equal(pc.kv4_sparse_attention(q, s.cache, means, s.table, s.lens, 50_000_000), want)
    assert torch.cuda.max_memory_allocated() - before < 64 << 20
    assert nat.device_status() == 0


@pytest.mark.parametrize("rows,hk,pages", [([2000, 1100], 4, 3000), ([1] * 70, 2, 300000)])
def test_sparse_rows_in_turn(cuda_device, rows, hk, pages):
    """Rows whose scores together are beyond the workspace's share of them: they are chosen for in turn."""
    G, d, page = 1, 64, 16
    assert sum(rows) * hk * pages * 8 > 256 << 20
    B, held = len(rows), 200
    s = Batch([held * page] * 2, hk, d, page, cuda_device, seed=hk)
    table = torch.zeros(B, pages, dtype=torch.int32, device=cuda_device)  # wide tables, of which little is used
    table[:, :held] = s.table[torch.arange(B) % 2]
    lens = ints([held * page - (7 * i) % 50 for i in range(B)], cuda_device)
    means = pc.kv4_means(s.cache, d)
    pc.kv4_page_means(s.cache, means, s.table, s.lens, (2 * held * page,), cu_q=cu_of(s.lengths, cuda_device))
    q = torch.randn(sum(rows), hk, d, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).to(cuda_device)
    cu = cu_of(rows, cuda_device)
    y, chosen = pc.kv4_sparse_attention(q, s.cache, means, table, lens, 4, cu_q=cu, return_pages=True)
    narrow = table[:, :held].contiguous()  # in one
    z, again = pc.kv4_sparse_attention(q, s.cache, means, narrow, lens, 4, cu_q=cu, return_pages=True)
    assert torch.equal(chosen, again) and torch.equal(y, z)
    assert nat.device_status() == 0
    mean = [more.means(k, page) for k in s.k]
    for row in range(0, sum(rows), 97):
        b = int((cu <= row).sum()) - 1
        pos = int(lens[b]) - rows[b] + row - int(cu[b])
        assert chosen[row].tolist() == [c + [-1] * (7 - len(c)) for c in more.choose(q[row].cpu(), mean[b % 2], pos, page, 4, 1, 2)]
