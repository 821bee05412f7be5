"""The 4-bit cache (penta_cache): what is stored, what is read back, and attention
over it, against the definition (kv4_oracle)."""
import threading

import pytest
import torch

import kv4_oracle as oracle
import penta_cache as pc
import penta_kernel as pk
import penta_native as nat

pytestmark = pytest.mark.gpu


class Batch:
    """Sequences with all their keys and values, and a cache that holds them."""

    def __init__(self, lengths, hk, d, page, device, seed=0, dtype=torch.bfloat16, spare=2, width=None):
        g = torch.Generator().manual_seed(seed)
        self.lengths, self.hk, self.d, self.page, self.device = lengths, hk, d, page, device
        loud = torch.where(torch.rand(hk, d, generator=g) < 0.05, 4.0, 1.0)
        self.k = [(torch.randn(n, hk, d, generator=g) * loud + 0.3).to(dtype) for n in lengths]
        self.v = [torch.randn(n, hk, d, generator=g).to(dtype) for n in lengths]
        need = [-(-n // page) for n in lengths]
        order = torch.randperm(sum(need) + spare, generator=g, dtype=torch.int32)
        self.table = torch.full((len(lengths), width or max(max(need), 1)), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.table = self.table.to(device)
        self.lens = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.cache = pc.kv4_cache(sum(need) + spare, hk, d, page, device)
        self.cache.fill_(0xFF)  # whatever is not stored is NaN
        self.store(lengths)

    def store(self, rows, lens=None):
        """Append the newest rows[i] of sequence i (of its first lens[i])."""
        lens = lens or self.lengths
        cut = lambda x: torch.cat([t[n - r:n] for t, r, n in zip(x, rows, lens)]).to(self.device)
        cu = torch.tensor([0] + list(rows), device=self.device).cumsum(0).to(torch.int32)
        at = torch.tensor(lens, dtype=torch.int32, device=self.device)
        pc.kv4_append(cut(self.k), cut(self.v), self.cache, self.table, at, cu_q=cu)

    def attend(self, rows, G, dtype=torch.bfloat16, seed=1, scale=None, **kw):
        g = torch.Generator().manual_seed(seed)
        q = [torch.randn(r, G * self.hk, self.d, generator=g).to(dtype) for r in rows]
        cu = torch.tensor([0] + list(rows), device=self.device).cumsum(0).to(torch.int32)
        got = pc.kv4_attention(torch.cat(q).to(self.device), self.cache, self.table, self.lens, cu_q=cu, scale=scale, **kw)
        self.check(got.split(list(rows)), q, scale)
        return got

    def check(self, got, q, scale=None):
        for i, (y, x) in enumerate(zip(got, q)):
            n = self.lengths[i]
            if n == 0 or x.shape[0] == 0:
                assert not y.any()
                continue
            lead = max(x.shape[0] - n, 0)  # rows before the sequence's start
            assert not y[:lead].any()
            want, bound = oracle.attention(x[lead:], self.k[i], self.v[i], scale)
            if y.dtype == torch.bfloat16:
                bound = bound + 2.0 ** -8 * (want.abs() + bound)
            err = (y[lead:].double().cpu() - want).abs()
            assert (err <= bound + 1e-30).all(), (i, (err - bound).max(), err.max())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hk", [1, 3, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_and_gather(cuda_device, d, hk, dtype):
    lengths = [1, 0, 17, 64, 5, 131]
    for page in (16, 48, 64):
        s = Batch(lengths, hk, d, page, cuda_device, seed=page + d, dtype=dtype)
        cu = torch.tensor([0] + lengths, device=cuda_device).cumsum(0).to(torch.int32)
        for out, tol in ((torch.float32, 2.0 ** -24), (torch.bfloat16, 2.0 ** -8)):
            k, v = pc.kv4_gather(s.cache, d, s.table, s.lens, (sum(lengths),), cu_q=cu, dtype=out)
            for got, x in ((k, s.k), (v, s.v)):
                want = oracle.values(torch.cat(x))
                assert got.dtype == out
                # codes, scales and zeros are exact: one rounding of the value
                assert ((got.double().cpu() - want).abs() <= tol * want.abs()).all()
        c, scale, zero = oracle.quantise(torch.cat(s.k))
        off = (oracle.values(torch.cat(s.k)) - torch.cat(s.k).double()).abs()
        # the format: within half a step (fp32 quotients add 16 * 2^-24 of one)
        assert (off <= scale[..., None].double() * 0.500002).all()


@pytest.mark.parametrize("d", [64, 128])
def test_stored_bytes(cuda_device, d):
    """The documented layout, byte by byte."""
    page, n, hk = 32, 45, 2
    s = Batch([n], hk, d, page, cuda_device, seed=4)
    cache = s.cache.cpu()
    for j, x in enumerate((s.k[0], s.v[0])):
        c, scale, zero = oracle.quantise(x)
        for t in range(n):
            blk = cache[s.table[0, t // page].item(), :, j]
            tok = t % page
            dim = torch.arange(d)
            at = tok * (d // 2) + dim // 2 if j == 0 else tok // 2 * d + dim // 4 * 4 + tok % 2 * 2 + dim % 4 // 2
            assert torch.equal((blk[:, at] >> (dim % 2 * 4).to(torch.uint8) & 15).float(), c[t])
            pair = blk[:, page * d // 2 + 4 * tok:][:, :4].contiguous().view(torch.bfloat16).float()
            assert torch.equal(pair, torch.stack((scale[t], zero[t]), -1))


def test_step_by_step_equals_at_once(cuda_device):
    """Tokens appended one by one, in runs that end inside pages and pairs, and all
    at once leave the same bytes; nothing else is touched."""
    lengths = [70, 33, 1]
    whole = Batch(lengths, 2, 64, 16, cuda_device, seed=3)
    steps = Batch(lengths, 2, 64, 16, cuda_device, seed=3)
    steps.cache.fill_(0xFF)
    for upto, rows in (([7, 0, 0], [7, 0, 0]), ([8, 20, 0], [1, 20, 0]), ([69, 33, 1], [61, 13, 1]), ([70, 33, 1], [1, 0, 0])):
        steps.store(rows, upto)
    assert torch.equal(whole.cache, steps.cache)
    free = set(range(whole.cache.shape[0])) - set(whole.table.flatten().tolist())
    assert len(free) == 2 and all((whole.cache[p] == 0xFF).all() for p in free)


def test_strided_views_and_rows_of_a_projection(cuda_device):
    """Queries, keys and values as views of one projection's output, at any offset."""
    B, L, H, hk, d = 3, 5, 6, 2, 64
    g = torch.Generator().manual_seed(2)
    for off in (0, 1, 8):
        buf = torch.randn(B, L, off + (H + 2 * hk) * d + 8, generator=g).to(torch.bfloat16).to(cuda_device)
        q, k, v = buf[..., off:off + (H + 2 * hk) * d].split((H * d, hk * d, hk * d), dim=2)
        q, k, v = q.view(B, L, H, d), k.view(B, L, hk, d), v.view(B, L, hk, d)
        lens = torch.full((B,), L, dtype=torch.int32, device=cuda_device)
        table = torch.tensor([[2], [0], [1]], dtype=torch.int32, device=cuda_device)
        cache = pc.kv4_cache(3, hk, d, 16, cuda_device)
        pc.kv4_append(k, v, cache, table, lens)
        y = pc.kv4_attention(q, cache, table, lens)
        again = pc.kv4_cache(3, hk, d, 16, cuda_device)
        pc.kv4_append(k.contiguous(), v.contiguous().transpose(1, 2).contiguous().transpose(1, 2), again, table, lens)
        assert torch.equal(cache, again)
        assert torch.equal(y, pc.kv4_attention(q.contiguous().view(B * L, H, d), cache, table, lens).view(y.shape))
        kk, vv = pc.kv4_gather(cache, d, table, lens, (B, L), dtype=torch.float32)
        assert kk.shape == (B, L, hk, d)
        for b in range(B):
            want, bound = oracle.attention(q[b], k[b].cpu(), v[b].cpu())
            assert ((y[b].double().cpu() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("G", [1, 2, 5, 8, 12, 16, 33])
def test_decode(cuda_device, d, G):
    lengths = [1, 15, 16, 17, 64, 65, 200, 777, 3]
    s = Batch(lengths, 2, d, 64, cuda_device, seed=G)
    s.attend([1] * len(lengths), G)
    s.attend([1] * len(lengths), G, dtype=torch.float32, scale=0.5)


@pytest.mark.parametrize("rows", [2, 3, 7, 16, 33, 64, 100, 129])
def test_several_new_rows(cuda_device, rows):
    for d, G, page in ((64, 1, 16), (128, 4, 32), (64, 3, 48)):
        lengths = [rows, rows + 1, rows + 63, 3 * rows + 200]
        s = Batch(lengths, 2, d, page, cuda_device, seed=rows)
        s.attend([rows] * 4, G)


def test_rows_of_unequal_sequences(cuda_device):
    """Decodes and prompt chunks in one call, sequences without rows or without tokens."""
    lengths = [500, 1, 0, 300, 64, 129, 1000, 0, 40]
    rows = [1, 1, 0, 300, 0, 65, 128, 2, 40]
    for d, G in ((64, 1), (128, 6)):
        s = Batch(lengths, 2, d, 64, cuda_device, seed=d)
        y = s.attend(rows, G)
        assert torch.equal(y, s.attend(rows, G))  # the same bits on every run


def test_more_rows_than_tokens(cuda_device):
    """Rows before a sequence's start see nothing: zeros, and nothing is stored."""
    s = Batch([5, 0, 20], 1, 64, 16, cuda_device)
    s.attend([9, 3, 20], 2)
    before = s.cache.clone()
    k = torch.randn(3, 9, 1, 64, device=cuda_device)
    pc.kv4_append(k, k, s.cache, s.table, torch.tensor([0, -5, 0], dtype=torch.int32, device=cuda_device))
    assert torch.equal(before, s.cache)
    kk, _ = pc.kv4_gather(s.cache, 64, s.table, torch.tensor([2, -1, 0], dtype=torch.int32, device=cuda_device), (3, 4))
    assert not kk[0, :2].any() and kk[0, 2:].any() and not kk[1:].any()


@pytest.mark.parametrize("B,length,hk,G", [(1, 40000, 2, 4), (1, 5000, 1, 1), (40, 100, 4, 2), (300, 30, 1, 2), (2, 9000, 8, 8)])
def test_work_split(cuda_device, B, length, hk, G):
    """Long sequences over all blocks, many short ones, more sequences than threads."""
    lengths = [max(1, length - 7 * i) for i in range(B)]
    s = Batch(lengths, hk, 128, 128, cuda_device, seed=B)
    s.attend([1] * B, G)


def test_peaked_and_shifted_logits(cuda_device):
    """A maximum that grows along the sequence, then one dominant token, value
    vectors of very different ranges, constant vectors."""
    n = 700
    s = Batch([n, n, n, n], 2, 64, 64, cuda_device, seed=6)
    ramp = torch.linspace(-6, 6, n)[:, None, None]
    s.k[0] = (s.k[0].float() * 0.1 + ramp).to(torch.bfloat16)
    s.k[1][n // 2] = 20.0
    s.v[2] = (s.v[2].float() * torch.logspace(-4, 4, n)[torch.randperm(n, generator=torch.Generator().manual_seed(1))][:, None, None]).to(torch.bfloat16)
    s.k[3] = torch.ones_like(s.k[3])
    s.v[3] = torch.full_like(s.v[3], 0.37)
    s.store([n] * 4)
    for rows in (1, 4, 40):
        s.attend([rows] * 4, 4, seed=rows)


@pytest.mark.parametrize("d,G", [(64, 1), (128, 4), (128, 8)])
def test_value_scales_from_zero_up(cuda_device, d, G):
    """Constant values first (their scale is zero), then ever larger ones, and the reverse."""
    n = 900
    s = Batch([n, n, n], 2, d, 64, cuda_device, seed=12)
    grow = torch.logspace(-6, 3, n)[:, None, None]
    s.v[0] = (s.v[0].float() * grow).to(torch.bfloat16)
    s.v[0][:300] = 0.75
    s.v[1] = (s.v[1].float() * grow.flip(0)).to(torch.bfloat16)
    s.v[2][:] = torch.arange(n)[:, None, None] % 7
    s.store([n] * 3)
    for rows in (1, 3, 20, 150):
        s.attend([rows] * 3, G, seed=rows)


def test_tables_wider_than_the_sequences(cuda_device):
    """Entries behind a sequence's end are never looked at."""
    s = Batch([100, 3], 2, 128, 16, cuda_device, width=4096)
    s.attend([1, 1], 4)
    s.attend([50, 3], 4)
    assert nat.device_status() == 0


def test_vectors_that_are_not_finite(cuda_device):
    """They read back as NaN, and only rows that see them turn NaN."""
    s = Batch([40, 40], 1, 64, 16, cuda_device, seed=8)
    s.v[0][20, 0, 3] = float("inf")
    s.store([40, 40])
    k, v = pc.kv4_gather(s.cache, 64, s.table, s.lens, (2, 40), dtype=torch.float32)
    assert torch.isnan(v[0, 20]).all() and torch.isfinite(v[1]).all() and torch.isfinite(k).all()
    q = torch.randn(2, 30, 2, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda_device)
    y = pc.kv4_attention(q, s.cache, s.table, s.lens)
    assert torch.isfinite(y[0, :10]).all() and torch.isnan(y[0, 10:]).all() and torch.isfinite(y[1]).all()
    s.v[0][20, 0, 3] = 1.0
    s.k[0][25, 0, 0] = float("nan")
    s.store([40, 40])
    y = pc.kv4_attention(q, s.cache, s.table, s.lens)
    assert torch.isfinite(y[0, :15]).all() and torch.isnan(y[0, 15:]).all() and torch.isfinite(y[1]).all()
    y = pc.kv4_attention(q[:, -1:], s.cache, s.table, s.lens)
    assert torch.isnan(y[0]).all() and torch.isfinite(y[1]).all()


def test_block_table_entries_outside_the_cache(cuda_device):
    """Skipped and reported, never read."""
    s = Batch([64, 64], 1, 64, 16, cuda_device, seed=9)
    assert nat.device_status() == 0
    good = s.table[0, 1].item()
    for wrong in (-1, s.cache.shape[0], 2 ** 31 - 1, -2 ** 31):
        s.table[0, 1] = wrong
        q = torch.randn(2, 1, 2, 64, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
        y = pc.kv4_attention(q.to(cuda_device), s.cache, s.table, s.lens)
        assert nat.device_status(reset=True) == nat.PN_ERR_ARG
        keep = [i for i in range(64) if not 16 <= i < 32]
        want, bound = oracle.attention(q[0], s.k[0][keep], s.v[0][keep])
        assert ((y[0].double().cpu() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()
        k, _ = pc.kv4_gather(s.cache, 64, s.table, s.lens, (2, 64))
        assert not k[0, 16:32].any() and k[0, :16].any() and nat.device_status(reset=True) == nat.PN_ERR_ARG
        before = s.cache.clone()
        s.store([64, 64])
        assert torch.equal(before, s.cache) and nat.device_status(reset=True) == nat.PN_ERR_ARG
    s.table[0, 1] = good
    s.attend([1, 1], 2)
    assert nat.device_status() == 0


@pytest.mark.parametrize("rows", [3, 20, 90])
def test_lengths_past_the_table(cuda_device, rows):
    """Positions that the table has no entry for are not stored, not attended to and
    reported; what lies in the table stays as it was."""
    n, held, page, hk, G = 200, 160, 16, 2, 4
    s = Batch([n, 50], hk, 128, page, cuda_device, seed=rows)
    s.table = s.table[:, :held // page].contiguous()
    before = s.cache.clone()
    s.store([rows, 0])  # of its positions 200 - rows .. 199 those below 160 are there already
    assert torch.equal(before, s.cache)
    assert nat.device_status(reset=True) == nat.PN_ERR_ARG
    k, _ = pc.kv4_gather(s.cache, 128, s.table, s.lens, (n,), cu_q=torch.tensor([0, n, n], dtype=torch.int32, device=cuda_device))
    assert not k[held:].any() and k[held - 1].any() and nat.device_status(reset=True) == nat.PN_ERR_ARG
    q = torch.randn(rows, hk * G, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    cu = torch.tensor([0, rows, rows], dtype=torch.int32, device=cuda_device)
    y = pc.kv4_attention(q.to(cuda_device), s.cache, s.table, s.lens, cu_q=cu)
    assert nat.device_status(reset=True) == nat.PN_ERR_ARG
    for r in range(rows):  # a row at position p sees positions up to min(p, 159)
        end = min(n - rows + r + 1, held)
        want, bound = oracle.attention(q[r:r + 1], s.k[0][:end], s.v[0][:end])
        assert ((y[r].double().cpu() - want[0]).abs() <= bound[0] + 2.0 ** -8 * (want[0].abs() + bound[0])).all(), r


@pytest.mark.parametrize("rows", [4, 40, 100])
def test_row_starts_that_fall(cuda_device, rows):
    """Reported, and nothing is computed."""
    s = Batch([50, 60, 20], 1, 64, 16, cuda_device)
    q = torch.randn(3 * rows, 2, 64, device=cuda_device).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    assert nat.device_status() == 0
    cu = torch.tensor([0, 3 * rows, rows, 3 * rows], dtype=torch.int32, device=cuda_device)
    pc.kv4_attention(q, s.cache, s.table, s.lens, cu_q=cu, out=out)
    assert (out == 7).all() and nat.device_status(reset=True) == nat.PN_ERR_ARG


def test_rows_behind_the_last_sequence(cuda_device):
    s = Batch([30, 20], 2, 64, 16, cuda_device)
    cu = torch.tensor([0, 1, 3], dtype=torch.int32, device=cuda_device)
    q = torch.randn(8, 4, 64, device=cuda_device).to(torch.bfloat16)
    out = torch.full_like(q, 7.0)
    got = pc.kv4_attention(q, s.cache, s.table, s.lens, cu_q=cu, out=out)
    assert got is out and (out[3:] == 7).all()
    assert torch.equal(out[:3], pc.kv4_attention(q[:3].contiguous(), s.cache, s.table, s.lens, cu_q=cu))
    assert not pc.kv4_attention(q, s.cache, s.table, s.lens, cu_q=cu)[3:].any()
    before = s.cache.clone()
    k, v = pc.kv4_gather(s.cache, 64, s.table, s.lens, (8,), cu_q=cu)
    assert not k[3:].any()
    x = torch.randn(8, 2, 64, device=cuda_device)
    x[:3] = pc.kv4_gather(s.cache, 64, s.table, s.lens, (3,), cu_q=cu, dtype=torch.float32)[0]
    pc.kv4_append(x, x, s.cache, s.table, s.lens, cu_q=cu)
    assert torch.equal(pc.kv4_gather(s.cache, 64, s.table, s.lens, (3,), cu_q=cu)[0], k[:3])
    assert (before != s.cache).any()


def test_graph_follows_lengths_and_tables(cuda_device):
    """A captured step (append, attend) replays with new contents, and two captured
    steps of one cache keep apart."""
    B, hk, G, d, page = 4, 2, 4, 64, 16
    s = Batch([90, 50, 17, 70], hk, d, page, cuda_device, seed=5, width=8)
    q = torch.randn(B, 1, hk * G, d, device=cuda_device).to(torch.bfloat16)
    k = torch.randn(B, 1, hk, d, device=cuda_device).to(torch.bfloat16)
    lens = s.lens.clone()

    def step():
        pc.kv4_append(k, k, s.cache, s.table, lens)
        return pc.kv4_attention(q, s.cache, s.table, lens)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    one, two = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(one):
        y1 = step()
    with torch.cuda.graph(two):
        y2 = step()
    for n in ([90, 50, 17, 70], [33, 49, 1, 64], [64, 3, 17, 5]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        q.normal_()
        k.normal_()
        one.replay()
        two.replay()
        want = step()
        assert torch.equal(y1, want) and torch.equal(y2, want)


def test_offsets_past_32_bits(cuda_device):
    """A cache of more than 4 GiB, used at its far end."""
    page, hk, d = 256, 8, 128
    n_pages = (1 << 32) // (2 * hk * pc.block_bytes(page, d)) + 8
    cache = torch.empty(n_pages, hk, 2, pc.block_bytes(page, d), dtype=torch.uint8, device=cuda_device)
    n = 300
    table = torch.tensor([[n_pages - 1, 0], [n_pages - 3, n_pages - 2]], dtype=torch.int32, device=cuda_device)
    lens = torch.full((2,), n, dtype=torch.int32, device=cuda_device)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(2, n, hk, d, generator=g).to(torch.bfloat16) for _ in range(2))
    pc.kv4_append(k.to(cuda_device), v.to(cuda_device), cache, table, lens)
    for r in (1, 70):
        q = torch.randn(2, r, hk * 4, d, generator=g).to(torch.bfloat16)
        y = pc.kv4_attention(q.to(cuda_device), cache, table, lens)
        for b in range(2):
            want, bound = oracle.attention(q[b], k[b], v[b])
            assert ((y[b].double().cpu() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all()


def test_empty_calls(cuda_device):
    cache = pc.kv4_cache(0, 2, 64, 16, cuda_device)
    table = torch.zeros(2, 0, dtype=torch.int32, device=cuda_device)
    lens = torch.ones(2, dtype=torch.int32, device=cuda_device)
    q = torch.randn(2, 1, 4, 64, device=cuda_device)
    pc.kv4_append(q[..., :2, :], q[..., :2, :], cache, table, lens)
    assert not pc.kv4_attention(q, cache, table, lens).any()
    assert pc.kv4_attention(q[:, :0], cache, table, lens).shape == (2, 0, 4, 64)
    none = torch.zeros(0, 3, dtype=torch.int32, device=cuda_device)
    assert pc.kv4_attention(q[:0], cache, none, lens[:0]).shape == (0, 1, 4, 64)
    assert nat.device_status() == 0


def test_no_sequences(cuda_device):
    """Rows behind the last sequence, of which there is none: zeros."""
    cache = pc.kv4_cache(3, 2, 64, 16, cuda_device)
    table = torch.zeros(0, 3, dtype=torch.int32, device=cuda_device)
    lens = torch.zeros(0, dtype=torch.int32, device=cuda_device)
    cu = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    for dtype in (torch.bfloat16, torch.float32):
        junk = [torch.full((40, 2, 64), 7.0, dtype=dtype, device=cuda_device) for _ in range(4)]
        torch.cuda.synchronize()
        del junk  # what the allocator hands out next
        k, v = pc.kv4_gather(cache, 64, table, lens, (40,), cu_q=cu, dtype=dtype)
        assert k.shape == v.shape == (40, 2, 64) and not k.any() and not v.any()
        k, v = (torch.full((5, 2, 64), 7.0, dtype=dtype, device=cuda_device) for _ in range(2))
        st = nat.load().pn_kv4_gather(cache.data_ptr(), 3, 2, 16, 64, None, 3, 3, None, cu.data_ptr(), 0, 4, k.data_ptr(),
                                      v.data_ptr(), nat.PN_F32 if dtype == torch.float32 else nat.PN_BF16, nat.stream_of(k))
        assert st == nat.PN_OK
        assert not k[:4].any() and not v[:4].any() and (k[4] == 7).all() and (v[4] == 7).all()
        x = torch.ones(40, 2, 64, dtype=dtype, device=cuda_device)
        before = cache.clone()
        pc.kv4_append(x, x, cache, table, lens, cu_q=cu)
        assert torch.equal(before, cache) and not pc.kv4_attention(x, cache, table, lens, cu_q=cu).any()
    assert nat.device_status() == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("loud", [1.0, 5.0, 12.0])
def test_what_four_bits_cost(cuda_device, d, loud):
    """Against attention over the keys and values as they were given, before rounding to 4 bits.

    Rounding moves each value by an error of variance s^2 / 12.  A logit then moves by D of
    variance (scale |q| s_k)^2 / 12 and its weight by the factor 1 + D, so with independent
    errors the output sum_t p_t v_t moves by sum_t p_t (D_t v_t + e_t): relative to p_t and
    the values' mean square, by D^2 + s_v^2 / (12 mean v^2) in the square.  The bound allows a
    quarter more than that root (products of the two, the exponential's curvature)."""
    n, hk, G, rows = 1024, 2, 4, 8
    s = Batch([n], hk, d, 64, cuda_device, seed=3)
    g = torch.Generator().manual_seed(11)
    k, v = (torch.randn(n, hk, d, generator=g) for _ in range(2))
    k[:, :, [3, d // 2]] *= loud
    s.k, s.v = [k.to(torch.bfloat16)], [v.to(torch.bfloat16)]
    s.store([n])
    q = torch.randn(rows, hk * G, d, generator=g).to(torch.bfloat16)
    cu = torch.tensor([0, rows], dtype=torch.int32, device=cuda_device)
    y = pc.kv4_attention(q.to(cuda_device), s.cache, s.table, s.lens, cu_q=cu).double().cpu().view(rows, hk, G, d)
    qq, kk, vv = q.double().view(rows, hk, G, d), s.k[0].double(), s.v[0].double()
    logit = torch.einsum("rhgd,nhd->hgrn", qq, kk) * d ** -0.5
    logit.masked_fill_(torch.arange(n) > (n - rows + torch.arange(rows))[:, None], -float("inf"))
    p = torch.softmax(logit, -1)
    want = torch.einsum("hgrn,nhd->rhgd", p, vv)
    sk, sv = (oracle.quantise(x)[1].double() for x in (s.k[0], s.v[0]))  # (n, hk)
    moved = qq.square().sum(-1).permute(1, 2, 0)[..., None] / d * (sk * sk).t()[:, None, None] / 12  # D^2: (hk, G, rows, n)
    part = moved + ((sv * sv).t() / (12 * vv.square().mean((0, 2)))[:, None])[:, None, None]
    part = (p * p * part).sum() / (p * p).sum()
    off, cost = ((y - want).norm() / want.norm()).item(), 1.25 * part.sqrt().item()
    print(f"\n4 bits, head_dim {d}, two key dims {loud:g}x louder: {off:.3f} of the output's norm (bound {cost:.3f})")
    assert off <= cost


# Calls of many row tiles (more than four per SM) take larger ones: 64 rows up to 64 rows
# per sequence and head (here 12 x 4), 128 above (21 x 4).
def wide(device, d, rows, **kw):
    g = torch.Generator().manual_seed(rows + d)
    lengths = torch.randint(1, 260, (32,), generator=g).tolist()
    lengths[:4] = [300, 255, 64, 5]
    return Batch(lengths, 8, d, kw.pop("page", 64), device, seed=rows, **kw)


def wide_rows(rows):
    """`rows` each on average: long ones, single ones, none, more than the sequence has."""
    r = [rows] * 32
    r[:6] = [3 * rows, 1, 0, rows, rows - 1, 2]
    r[6] += 6 * rows - sum(r[:6])
    assert sum(r) == 32 * rows and min(r) >= 0
    return r


@pytest.mark.parametrize("d,page", [(64, 64), (128, 16), (128, 48), (64, 128)])
@pytest.mark.parametrize("rows", [12, 21])
def test_many_row_tiles(cuda_device, d, page, rows):
    s = wide(cuda_device, d, rows, page=page)
    s.attend(wide_rows(rows), 4)
    s.attend(wide_rows(rows), 4, dtype=torch.float32, scale=0.2)
    assert nat.device_status() == 0


@pytest.mark.parametrize("rows", [12, 21])
def test_many_row_tiles_hard_values(cuda_device, rows):
    """Growing maxima and value scales, one dominant token, constant vectors."""
    s = wide(cuda_device, 128, rows)
    n = s.lengths
    s.k[0] = (s.k[0].float() * 0.1 + torch.linspace(-6, 6, n[0])[:, None, None]).to(torch.bfloat16)
    s.k[1][n[1] // 2] = 20.0
    s.v[0] = (s.v[0].float() * torch.logspace(-6, 3, n[0])[:, None, None]).to(torch.bfloat16)
    s.v[0][:100] = 0.75
    s.v[1] = (s.v[1].float() * torch.logspace(-4, 4, n[1]).flip(0)[:, None, None]).to(torch.bfloat16)
    s.k[3] = torch.ones_like(s.k[3])
    s.v[3] = torch.full_like(s.v[3], 0.37)
    s.store(n)
    s.attend([rows] * 32, 4)
    s.attend(wide_rows(rows), 4)


@pytest.mark.parametrize("rows", [12, 21])
def test_many_row_tiles_not_finite(cuda_device, rows):
    """Only rows that see a vector that is not finite turn NaN."""
    s = wide(cuda_device, 64, rows)
    s.v[0][290, 3, 5] = float("inf")
    s.k[1][250, 2, 0] = float("nan")
    s.store(s.lengths)
    q = torch.randn(32, rows, 32, 64, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16).to(cuda_device)
    y = pc.kv4_attention(q, s.cache, s.table, s.lens).view(32, rows, 8, 4, 64)
    bad = torch.zeros(32, rows, 8, dtype=torch.bool, device=cuda_device)
    for r in range(rows):
        bad[0, r, 3] = 300 - rows + r >= 290
        bad[1, r, 2] = 255 - rows + r >= 250
    assert bad.any() and torch.equal(torch.isnan(y).all(-1).all(-1), bad)
    assert torch.equal(~torch.isfinite(y).all(-1).all(-1), bad)


@pytest.mark.parametrize("rows", [12, 21])
def test_many_row_tiles_lost_pages(cuda_device, rows):
    """Entries outside the cache and lengths past the table: skipped and reported."""
    s = wide(cuda_device, 128, rows, page=16)
    q = torch.randn(32, rows, 32, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    s.table[0, 2] = -1
    s.table[1, 0] = s.cache.shape[0]
    table = s.table[:, :256 // 16].contiguous()  # sequence 0 has 300 tokens
    assert nat.device_status() == 0
    y = pc.kv4_attention(q.to(cuda_device), s.cache, table, s.lens)
    assert nat.device_status(reset=True) == nat.PN_ERR_ARG
    near = lambda got, want, bound: ((got.double().cpu() - want).abs() <= bound + 2.0 ** -8 * (want.abs() + bound)).all().item()
    behind = set(range(256, 300))
    for i, n in enumerate(s.lengths):
        lost = behind | (set(range(32, 48)) if i == 0 else set(range(16)) if i == 1 else set())
        if lost.isdisjoint(range(n)):
            lead = max(rows - n, 0)
            assert not y[i, :lead].any() and near(y[i, lead:], *oracle.attention(q[i, lead:], s.k[i], s.v[i])), i
            continue
        for r in range(max(rows - n, 0), rows):
            keep = [t for t in range(n - rows + r + 1) if t not in lost]
            want, bound = oracle.attention(q[i, r:r + 1], s.k[i][keep], s.v[i][keep])
            assert near(y[i, r], want[0], bound[0]), (i, r)


@pytest.mark.parametrize("rows", [12, 21])
def test_many_row_tiles_captured(cuda_device, rows):
    """Strided queries of a joint projection; replays follow the lengths; twice the same bits."""
    s = wide(cuda_device, 128, rows)
    qkv = torch.randn(32, rows, 48 * 128, device=cuda_device).to(torch.bfloat16)
    q = qkv[..., :32 * 128].view(32, rows, 32, 128)
    want = pc.kv4_attention(q.contiguous(), s.cache, s.table, s.lens)
    assert torch.equal(pc.kv4_attention(q, s.cache, s.table, s.lens), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = pc.kv4_attention(q, s.cache, s.table, s.lens)
    for _ in range(2):
        graph.replay()
        assert torch.equal(y, want)
        s.lens -= 3
        s.lens.clamp_(min=0)
        want = pc.kv4_attention(q, s.cache, s.table, s.lens)


def check_rows_apart(y, q, k, v):
    """Every row against the tokens that it sees, as if there were no others: the
    oracle's bound then knows the value ranges of these alone."""
    r, n = q.shape[0], k.shape[0]
    for i in range(max(r - n, 0), r):
        end = n - r + i + 1
        want, bound = oracle.attention(q[i:i + 1], k[:end], v[:end])
        assert ((y[i].double().cpu() - want[0]).abs() <= bound[0] + 2.0 ** -8 * (want[0].abs() + bound[0])).all(), i


@pytest.mark.parametrize("d,rows,G", [(64, 6, 1), (128, 7, 1), (64, 5, 3), (128, 4, 4), (128, 30, 4), (64, 150, 1)])
def test_values_that_a_row_does_not_see(cuda_device, d, rows, G):
    """However large, they cost it nothing (few row tiles)."""
    lengths = [rows, rows + 40, 200, 333]
    s = Batch(lengths, 2, d, 16, cuda_device, seed=rows + d)
    for i, n in enumerate(lengths):
        for back, up in ((1, 2.0 ** 27), (2, 2.0 ** 24), (3, 2.0 ** 20), (4, 2.0 ** 12)):
            s.v[i][n - back] *= up
    s.store(lengths)
    q = torch.randn(4, rows, 2 * G, d, generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16)
    y = pc.kv4_attention(q.to(cuda_device), s.cache, s.table, s.lens)
    for i in range(4):
        check_rows_apart(y[i], q[i], s.k[i], s.v[i])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [12, 21])
def test_values_that_a_row_does_not_see_many_row_tiles(cuda_device, d, rows):
    s = wide(cuda_device, d, rows)
    for i, n in enumerate(s.lengths):
        for back in range(1, min(rows, n)):
            s.v[i][n - back] *= 2.0 ** (9 * (-back % 4))  # up to 2^27 between rows of one warp
    s.store(s.lengths)
    q = torch.randn(32, rows, 32, d, generator=torch.Generator().manual_seed(rows)).to(torch.bfloat16)
    y = pc.kv4_attention(q.to(cuda_device), s.cache, s.table, s.lens)
    for i in range(8):
        check_rows_apart(y[i], q[i], s.k[i], s.v[i])
    # the same rows before the last token is there
    s.lens -= 1
    again = pc.kv4_attention(q[:, :-1].contiguous().to(cuda_device), s.cache, s.table, s.lens)
    for i in range(8):
        check_rows_apart(again[i], q[i, :-1], s.k[i][:-1], s.v[i][:-1])


@pytest.mark.parametrize("rows,G", [(1, 4), (2, 4), (2, 8), (2, 40)])
def test_quiet_values_beside_loud_ones(cuda_device, rows, G):
    """A few tokens whose values lie 2^16 to 2^24 below those of others but carry the weight:
    within the bound that counts an error of 2^-25 of the largest scale per token."""
    lengths = [2 + i % 5 for i in range(96)]
    s = Batch(lengths, 3, 64, 16, cuda_device, seed=G)
    for i, n in enumerate(lengths):
        s.v[i][i % n] *= 2.0 ** (16 + i % 9)
        s.v[i] *= 2.0 ** -20
    s.store(lengths)
    s.attend([rows] * 96, G, scale=1.0, seed=G)


@pytest.mark.parametrize("rows", [1, 12, 21])
def test_between_products(cuda_device, rows):
    """Queries straight from a packed product, the output straight into the next, on two
    streams at once: both kernels start before the one before them ends and take tensor memory."""
    s = wide(cuda_device, 64, rows)
    g = torch.Generator().manual_seed(rows)
    w_q = pk.quantize_and_pack(torch.randn(32 * 64, 256, generator=g).to(cuda_device))
    w_o = pk.quantize_and_pack(torch.randn(256, 32 * 64, generator=g).to(cuda_device))
    x = torch.randn(32 * rows, 256, generator=g).to(torch.bfloat16).to(cuda_device)

    def block(wait=lambda: None):
        q = pk.penta_linear(x, w_q[0], w_q[2], w_q[1])
        wait()
        y = pc.kv4_attention(q.view(32, rows, 32, 64), s.cache, s.table, s.lens)
        wait()
        return pk.penta_linear(y.view(32 * rows, 32 * 64), w_o[0], w_o[2], w_o[1])

    want = block(torch.cuda.synchronize)
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for side in streams:
        side.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        for side in streams:
            with torch.cuda.stream(side):
                got.append(block())
    torch.cuda.synchronize()
    assert all(torch.equal(y, want) for y in got) and nat.device_status() == 0


def test_calls_of_several_threads(cuda_device):
    """Each on a stream of its own, all kernels at once: every call gives its own result."""
    s = wide(cuda_device, 128, 21)
    q = torch.randn(32, 21, 32, 128, device=cuda_device).to(torch.bfloat16)
    calls = [q[:, :n] for n in (1, 4, 12, 21)]
    want = [pc.kv4_attention(x, s.cache, s.table, s.lens) for x in calls]
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                wrong.extend(n for n, x in enumerate(calls)
                             if not torch.equal(pc.kv4_attention(x, s.cache, s.table, s.lens), want[n]))

    threads = [threading.Thread(target=work) for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and nat.device_status() == 0
