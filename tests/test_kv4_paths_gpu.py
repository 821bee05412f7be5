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
