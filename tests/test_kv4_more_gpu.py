"""Rotated append, attention behind shared prefixes and attention over chosen pages
(penta_cache), against their definitions (kv4_more_oracle, kv4_oracle)."""
import pytest
import torch

import kv4_more_oracle as more
import kv4_oracle as oracle
import penta_cache as pc
import penta_native as nat
from test_kv4_gpu import Batch

pytestmark = pytest.mark.gpu


def cu_of(rows, device):
    return torch.tensor([0] + list(rows), device=device).cumsum(0).to(torch.int32)


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


# ── rotation ─────────────────────────────────────────────────────────────────

def tables(n, R, device, seed=0):
    rate = 10000.0 ** (-torch.arange(R // 2, dtype=torch.float64) * 2 / R)
    angle = (torch.arange(n, dtype=torch.float64) + 0.37 * seed)[:, None] * rate
    return angle.cos().float().to(device), angle.sin().float().to(device)


class Rows:
    """Rows of ragged sequences, a cache and a table for them."""

    def __init__(self, lengths, rows, H, hk, d, page, dtype, device, seed=0):
        g = torch.Generator().manual_seed(seed)
        T = sum(rows)
        self.lengths, self.rows, self.hk, self.d = lengths, rows, hk, d
        self.q, self.k, self.v = (torch.randn(T, h, d, generator=g).to(dtype) for h in (H, hk, hk))
        self.pos = torch.cat([torch.arange(n - r, n) for r, n in zip(rows, lengths)])
        self.seq = torch.repeat_interleave(torch.arange(len(rows)), torch.tensor(rows))
        per = max(-(-max(lengths) // page), 1)
        self.table = torch.randperm(len(rows) * per, generator=g).to(torch.int32).view(len(rows), per).to(device)
        self.lens, self.cu = ints(lengths, device), cu_of(rows, device)
        self.empty = torch.full_like(pc.kv4_cache(len(rows) * per, hk, d, page, device), 0xFF)

    def expect(self, cos, sin, interleaved, offsets=None):
        """Rotated queries, and the cache after kv4_append of the rotated keys."""
        at = self.pos if offsets is None else self.pos + offsets.cpu()[self.seq].long()
        q = more.rotate(self.q, cos, sin, interleaved, at)
        k = more.rotate(self.k, cos, sin, interleaved, at)
        cache = self.empty.clone()
        dev = cache.device
        pc.kv4_append(k.to(dev), self.v.float().to(dev), cache, self.table, self.lens, cu_q=self.cu)
        return q.to(self.q.dtype), cache


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("H,hk,d,R,page", [(1, 1, 64, 64, 16), (12, 12, 64, 16, 64), (6, 2, 64, 48, 48), (8, 8, 128, 128, 32),
                                           (9, 3, 128, 64, 16), (40, 5, 128, 112, 128)])
def test_rotary(cuda_device, dtype, interleaved, H, hk, d, R, page):
    lengths, rows = [130, 1, 40, 77], [97, 1, 0, 33]
    s = Rows(lengths, rows, H, hk, d, page, dtype, cuda_device, seed=H + R)
    cos, sin = tables(400, R, cuda_device)
    for offsets in (None, ints([200, 0, 5, 323], cuda_device)):
        want, cache = s.expect(cos, sin, interleaved, offsets)
        got = s.empty.clone()
        q = pc.kv4_append_rotary(s.q.to(cuda_device), s.k.to(cuda_device), s.v.to(cuda_device), cos, sin, got, s.table, s.lens,
                                 cu_q=s.cu, offsets=offsets, interleaved=interleaved)
        assert torch.equal(q.cpu(), want)  # fp32 as defined, one rounding: bit for bit
        assert torch.equal(got, cache)
        at = s.pos if offsets is None else s.pos + offsets.cpu()[s.seq].long()
        exact = more.rotate(s.q, cos, sin, interleaved, at, torch.float64)
        # the sum of magnitudes, |a cos| + |b sin| and |b cos| + |a sin|
        mag = torch.maximum(*(more.rotate(s.q.abs(), cos.abs(), sign * sin.abs(), interleaved, at, torch.float64)
                              for sign in (1, -1)))
        # two products and their sum, each off by half an ulp of no more than that; the output's rounding
        half = torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 0.0
        assert ((q.double().cpu() - exact).abs() <= 2.01 * 2.0 ** -24 * mag + half * 1.001 * mag).all()
    assert nat.device_status() == 0


@pytest.mark.parametrize("B,L", [(1, 1), (64, 1), (5, 7), (3, 700)])
def test_rotary_rows_of_a_projection(cuda_device, B, L):
    """Equal rows per sequence, as views of one buffer at any alignment; few rows and many."""
    H, hk, d, R = 8, 2, 128, 128
    g = torch.Generator().manual_seed(B)
    lens = [L + 3 * i for i in range(B)]
    cos, sin = tables(max(lens) + 1, R, cuda_device)
    page, per = 16, -(-max(lens) // 16)
    table = torch.arange(B * per, dtype=torch.int32, device=cuda_device).view(B, per).flip(0).contiguous()
    pos = torch.stack([torch.arange(n - L, n) for n in lens]).flatten()
    for off in (0, 1, 8):
        buf = torch.randn(B, L, off + (H + 2 * hk) * d + 8, generator=g).to(torch.bfloat16).to(cuda_device)
        q, k, v = (x.view(B, L, -1, d) for x in buf[..., off:off + (H + 2 * hk) * d].split((H * d, hk * d, hk * d), dim=2))
        cache, again = (pc.kv4_cache(B * per, hk, d, page, cuda_device) for _ in range(2))
        got = pc.kv4_append_rotary(q, k, v, cos, sin, cache, table, ints(lens, cuda_device))
        assert torch.equal(got.cpu().view(-1, H, d), more.rotate(q.reshape(-1, H, d), cos, sin, False, pos).to(torch.bfloat16))
        turned = more.rotate(k.reshape(-1, hk, d), cos, sin, False, pos).to(cuda_device).view(B, L, hk, d)
        pc.kv4_append(turned, v.float(), again, table, ints(lens, cuda_device))
        assert torch.equal(cache, again)
        same = q.contiguous().clone()  # in place
        assert pc.kv4_append_rotary(same, k, v, cos, sin, cache, table, ints(lens, cuda_device), out=same) is same
        assert torch.equal(same, got)
        wide = torch.zeros(cos.shape[0], 3 * R // 2 + off, device=cuda_device)  # tables inside wider rows
        wide[:, off:off + R // 2], wide[:, -R // 2:] = cos, sin
        assert torch.equal(got, pc.kv4_append_rotary(q, k, v, wide[:, off:off + R // 2], wide[:, -R // 2:], cache, table,
                                                     ints(lens, cuda_device)))


def test_rotary_edges(cuda_device):
    """Rows before a sequence's start, behind the last sequence, and outside the tables."""
    H, hk, d, page = 4, 2, 64, 16
    lengths, rows = [3, 20, 9], [5, 2, 1]
    s = Rows([5, 20, 9], rows, H, hk, d, page, torch.bfloat16, cuda_device)
    s.lens = ints(lengths, cuda_device)
    cos, sin = tables(19, 64, cuda_device)  # the last row of sequence 1 has no entry
    dev = lambda x: torch.cat((x, x[:2])).to(cuda_device)  # two rows more than cu_q knows
    out = torch.full((10, H, d), 7.0, dtype=torch.bfloat16, device=cuda_device)
    cache = s.empty.clone()
    assert nat.device_status() == 0
    got = pc.kv4_append_rotary(dev(s.q), dev(s.k), dev(s.v), cos, sin, cache, s.table, s.lens, cu_q=s.cu, out=out)
    assert got is out and nat.device_status() == nat.PN_ERR_ARG
    pos = torch.tensor([0, 0, 0, 1, 2, 18, 0, 8])
    want = more.rotate(s.q, cos, sin, False, pos).to(torch.bfloat16)
    zero = torch.tensor([1, 1, 0, 0, 0, 0, 1, 0], dtype=torch.bool)
    assert not got[:8].cpu()[zero].any() and torch.equal(got[:8].cpu()[~zero], want[~zero])
    assert (got[8:] == 7).all()
    kept = torch.arange(8)[~zero]
    lone = s.empty.clone()
    turned = more.rotate(s.k, cos, sin, False, pos)
    for i in kept.tolist():  # one by one
        b = int(s.seq[i])
        pc.kv4_append(turned[i:i + 1].to(cuda_device), s.v[i:i + 1].float().to(cuda_device), lone, s.table[b:b + 1],
                      ints([int(pos[i]) + 1], cuda_device))
    assert torch.equal(cache, lone)
    # without an out, rows behind the last sequence are zeros; no sequence at all; no rows
    y = pc.kv4_append_rotary(dev(s.q), dev(s.k), dev(s.v), cos, sin, cache, s.table, s.lens, cu_q=s.cu)
    assert not y[8:].any()
    none = pc.kv4_append_rotary(dev(s.q), dev(s.k), dev(s.v), cos, sin, cache, s.table[:0], s.lens[:0], cu_q=s.cu[:1])
    assert not none.any()
    assert pc.kv4_append_rotary(dev(s.q)[:0], dev(s.k)[:0], dev(s.v)[:0], cos, sin, cache, s.table, s.lens).shape == (0, H, d)
    nat.device_status()
    # negative entries, a page that is none of the cache, tables of no positions
    far = ints([-30, 0, 0], cuda_device)
    y = pc.kv4_append_rotary(s.q.to(cuda_device), s.k.to(cuda_device), s.v.to(cuda_device), *tables(64, 64, cuda_device), cache,
                             s.table, s.lens, cu_q=s.cu, offsets=far)
    assert not y[:5].any() and y[5:].any() and nat.device_status() == nat.PN_ERR_ARG
    before = cache.clone()
    bad = torch.full_like(s.table, 10 ** 6)
    y = pc.kv4_append_rotary(s.q.to(cuda_device), s.k.to(cuda_device), s.v.to(cuda_device), *tables(64, 64, cuda_device), cache,
                             bad, s.lens, cu_q=s.cu)
    assert y[2:].any() and nat.device_status() == nat.PN_ERR_ARG and torch.equal(cache, before)
    y = pc.kv4_append_rotary(s.q.to(cuda_device), s.k.to(cuda_device), s.v.to(cuda_device), cos[:0], sin[:0], cache, s.table,
                             s.lens, cu_q=s.cu)
    assert not y.any() and nat.device_status() == nat.PN_ERR_ARG


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,rows", [(64, [1]), (128, [3, 0, 400])])
def test_rotary_rows_of_no_sequence(cuda_device, dtype, d, rows):
    """Behind the last sequence: zeros in a new tensor, whatever its memory held, and for calls without sequences."""
    s = Rows([r + 3 for r in rows], rows, 3, 1, d, 16, dtype, cuda_device)
    cos, sin = tables(500, d, cuda_device)
    T = sum(rows)
    dev = lambda x: torch.cat((x, x[:1].expand(37, -1, -1))).to(cuda_device)
    junk = torch.full((T + 37, 3, d), 7.0, dtype=dtype, device=cuda_device)
    del junk
    got = pc.kv4_append_rotary(dev(s.q), dev(s.k), dev(s.v), cos, sin, s.empty.clone(), s.table, s.lens, cu_q=s.cu)
    assert got[:T].any() and not got[T:].any()
    none = pc.kv4_append_rotary(dev(s.q), dev(s.k), dev(s.v), cos, sin, s.empty.clone(), s.table[:0], s.lens[:0],
                                cu_q=ints([0], cuda_device))
    assert not none.any() and nat.device_status() == 0


def test_rotary_not_finite(cuda_device):
    """A key vector with an inf or NaN reads back as NaN, and no other does."""
    s = Rows([6], [6], 2, 2, 64, 16, torch.float32, cuda_device)
    s.k[1, 0, 3], s.k[4, 1, 60] = float("inf"), float("nan")
    cos, sin = tables(6, 32, cuda_device)
    cache = s.empty.clone()
    pc.kv4_append_rotary(s.q.to(cuda_device), s.k.to(cuda_device), s.v.to(cuda_device), cos, sin, cache, s.table, s.lens)
    k, v = pc.kv4_gather(cache, 64, s.table, s.lens, (6,), dtype=torch.float32)
    lost = torch.zeros(6, 2, dtype=torch.bool)
    lost[1, 0] = lost[4, 1] = True
    assert torch.equal(k.isnan().all(-1).cpu(), lost) and torch.equal(k.isnan().any(-1).cpu(), lost) and not v.isnan().any()


# ── shared prefixes ──────────────────────────────────────────────────────────

class Shared:
    """Sequences behind prefixes, all in one cache: prefixes are the last of a Batch."""

    def __init__(self, own, prefixes, shares, hk, d, page, device, seed=0, dtype=torch.bfloat16):
        self.b = Batch(own + prefixes, hk, d, page, device, seed=seed, dtype=dtype)
        B = len(own)
        self.own, self.prefixes, self.shares = own, prefixes, shares
        self.table, self.lens = self.b.table[:B], self.b.lens[:B].contiguous()
        self.ptable, self.plens = self.b.table[B:], self.b.lens[B:].contiguous()
        self.cu_prefix = cu_of(shares, device)
        self.of = [g for g, n in enumerate(shares) for _ in range(n)]
        self.of += [None] * (B - len(self.of))
        self.device = device

    def call(self, q, rows, **kw):
        return pc.kv4_prefix_attention(q, self.b.cache, self.table, self.lens, self.ptable, self.plens,
                                       cu_q=cu_of(rows, self.device), cu_prefix=self.cu_prefix, **kw)

    def attend(self, rows, G, dtype=torch.bfloat16, seed=1, scale=None, **kw):
        g = torch.Generator().manual_seed(seed)
        q = [torch.randn(r, G * self.b.hk, self.b.d, generator=g).to(dtype) for r in rows]
        got = self.call(torch.cat(q).to(self.device), rows, scale=scale, **kw)
        self.check(got.split(list(rows)), q, scale)
        return got

    def check(self, got, q, scale=None):
        B = len(self.own)
        for i, (y, x) in enumerate(zip(got, q)):
            p, n, r = self.of[i], self.own[i], x.shape[0]
            m = 0 if p is None else self.prefixes[p]
            lead = max(r - n, 0)  # rows before the sequence's start: they see the prefix alone
            for part, rows in ((slice(0, lead), False), (slice(lead, r), True)):
                if x[part].shape[0] == 0:
                    continue
                k, v = ([t[B + p]] if p is not None else [] for t in (self.b.k, self.b.v))
                if rows:
                    k, v = k + [self.b.k[i]], v + [self.b.v[i]]
                if sum(t.shape[0] for t in k) == 0:
                    assert not y[part].any()
                    continue
                k, v = torch.cat(k), torch.cat(v)
                if rows:
                    want, bound = oracle.attention(x[part], k, v, scale)
                else:  # every row sees all of the prefix
                    each = [oracle.attention(t[None], k, v, scale) for t in x[part]]
                    want, bound = (torch.cat(t) for t in zip(*each))
                bound = bound + more.join_bound(x[part], k, v, scale)
                if y.dtype == torch.bfloat16:
                    bound = bound + 2.0 ** -8 * (want.abs() + bound)
                err = (y[part].double().cpu() - want).abs()
                assert (err <= bound + 1e-30).all(), (i, part, (err - bound).max(), err.max())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("G,hk", [(1, 3), (4, 2), (8, 1), (16, 1)])
def test_prefix_decode(cuda_device, d, G, hk):
    """One row per sequence: 4 to 176 rows behind a prefix, every kernel of the prefix pass."""
    for shares, prefixes, page in (([4], [77], 16), ([1, 2, 0, 8], [300, 129, 50, 1], 32), ([11], [1000], 64)):
        own = [(37 * i) % 90 + 1 for i in range(sum(shares))]
        s = Shared(own, prefixes, shares, hk, d, page, cuda_device, seed=d + G)
        s.attend([1] * len(own), G)
    assert nat.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d,G,hk,page", [(64, 1, 2, 16), (64, 3, 1, 48), (128, 4, 2, 64), (128, 2, 1, 128)])
def test_prefix_ragged(cuda_device, dtype, d, G, hk, page):
    """Chunks, single rows, rows before their sequence's start, sequences without rows, without
    tokens and without a prefix; empty prefixes and prefixes of nobody."""
    own = [70, 5, 0, 200, 1, 33, 64, 3]
    rows = [70, 0, 2, 120, 1, 40, 1, 3]
    s = Shared(own, [63, 0, 257, 17], [3, 1, 2, 0], hk, d, page, cuda_device, seed=G, dtype=dtype)
    s.attend(rows, G, dtype)
    s.attend(rows, G, dtype, scale=0.5)
    assert nat.device_status() == 0


@pytest.mark.parametrize("d", [64, 128])
def test_prefix_many_rows(cuda_device, d):
    """More rows than one tile, ragged at both ends; long prefixes split over blocks."""
    s = Shared([40, 300, 7], [2049, 700], [2, 1], 2, d, 64, cuda_device, seed=2)
    s.attend([40, 210, 7], 4)
    s = Shared([9] * 33, [5000], [33], 1, d, 32, cuda_device, seed=3)
    s.attend([9] * 33, 8)


def test_prefix_and_own_on_the_long_kernel(cuda_device):
    """Chunks long enough that both passes take the kernel for many rows, one right behind the other."""
    B, L, G, hk, d = 40, 96, 2, 8, 64
    s = Shared([L] * B, [300, 77], [30, 10], hk, d, 64, cuda_device, seed=3)
    q = torch.randn(B * L, G * hk, d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    y = s.call(q.to(cuda_device), [L] * B)
    assert nat.device_status() == 0
    some = [0, 1, 17, 29, 30, 39]  # (the 64-bit attention of all of them would take minutes)
    for i in some:
        k, v = (torch.cat((t[B + s.of[i]], t[i])) for t in (s.b.k, s.b.v))
        x = q[i * L:(i + 1) * L]
        want, bound = oracle.attention(x, k, v, None)
        bound = bound + more.join_bound(x, k, v)
        bound = bound + 2.0 ** -8 * (want.abs() + bound)
        assert ((y[i * L:(i + 1) * L].double().cpu() - want).abs() <= bound + 1e-30).all(), i


def test_prefix_equal_shares(cuda_device):
    """Without cu_prefix; (B, L) rows of a projection; against the same tokens laid out as whole sequences."""
    B, L, H, hk, d, page = 6, 2, 8, 2, 128, 16
    s = Shared([20 + i for i in range(B)], [64, 128], [3, 3], hk, d, page, cuda_device)
    g = torch.Generator().manual_seed(5)
    for off in (0, 1):
        buf = torch.randn(B, L, H * d + off, generator=g).to(torch.bfloat16).to(cuda_device)
        q = buf[..., off:].view(B, L, H, d)
        y = pc.kv4_prefix_attention(q, s.b.cache, s.table, s.lens, s.ptable, s.plens)
        s.check(y, list(q.cpu()))
        z = s.call(q.reshape(-1, H, d), [L] * B)
        s.check(z.view(y.shape), list(q.cpu()))
        # the prefix's pages in front of each sequence's own
        whole = torch.full((B, 8 + s.table.shape[1]), -1, dtype=torch.int32, device=cuda_device)
        for b in range(B):
            n = s.prefixes[b // 3] // page
            whole[b, :n] = s.ptable[b // 3, :n]
            whole[b, n:n + s.table.shape[1]] = s.table[b]
        lens = s.lens + torch.tensor([s.prefixes[b // 3] for b in range(B)], dtype=torch.int32, device=cuda_device)
        x = pc.kv4_attention(q, s.b.cache, whole, lens)
        assert (x.float() - y.float()).abs().max() <= 2.0 ** -6 * x.float().abs().max()


def test_prefix_edges(cuda_device):
    """Rows behind the last sequence; shares that fall or run over; no prefixes; bad pages; NaN behind a prefix's end."""
    own, hk, d, page, G = [10, 20, 30], 2, 64, 16, 2
    s = Shared(own, [50, 33], [1, 2], hk, d, page, cuda_device)
    q = torch.randn(8, G * hk, d, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(cuda_device)
    rows = [2, 1, 3]
    out = torch.full_like(q, 5.0)
    y = pc.kv4_prefix_attention(q, s.b.cache, s.table, s.lens, s.ptable, s.plens, cu_q=cu_of(rows, cuda_device),
                                cu_prefix=s.cu_prefix, out=out)
    assert y is out and (y[6:] == 5).all()
    s.check(y[:6].split(rows), list(q[:6].cpu().split(rows)))
    assert not s.call(q, rows)[6:].any()
    s.cu_prefix = ints([1, 2, 2], cuda_device)  # sequence 1 alone has a prefix
    s.of = [None, 0, None]
    s.check(s.call(q, rows)[:6].split(rows), list(q[:6].cpu().split(rows)))
    s.cu_prefix = ints([0, 2, 99], cuda_device)  # counts past the sequences: up to the last
    s.of = [0, 0, 1]
    s.check(s.call(q, rows)[:6].split(rows), list(q[:6].cpu().split(rows)))
    assert nat.device_status() == 0
    s.cu_prefix = ints([0, 3, 1], cuda_device)
    out.fill_(5.0)
    assert (s.call(q, rows, out=out) == 5).all() and nat.device_status() == nat.PN_ERR_ARG
    s.cu_prefix = ints([0, 1, 3], cuda_device)
    out.fill_(5.0)
    assert (pc.kv4_prefix_attention(q, s.b.cache, s.table, s.lens, s.ptable, s.plens, cu_q=ints([0, 4, 2, 6], cuda_device),
                                    cu_prefix=s.cu_prefix, out=out) == 5).all() and nat.device_status() == nat.PN_ERR_ARG
    none = pc.kv4_prefix_attention(q, s.b.cache, s.table, s.lens, s.ptable[:0], s.plens[:0], cu_q=cu_of(rows, cuda_device))
    assert torch.equal(none, pc.kv4_attention(q, s.b.cache, s.table, s.lens, cu_q=cu_of(rows, cuda_device)))
    # pages that are none: their tokens are not attended to, and reported
    assert nat.device_status() == 0
    lost = s.ptable.clone()
    lost[1, 1] = 10 ** 6
    y = pc.kv4_prefix_attention(q, s.b.cache, s.table, s.lens, lost, s.plens, cu_q=cu_of(rows, cuda_device), cu_prefix=s.cu_prefix)
    assert nat.device_status() == nat.PN_ERR_ARG
    for t in (s.b.k, s.b.v):
        t[4] = torch.cat((t[4][:page], t[4][2 * page:]))
    s.prefixes[1], s.of = 33 - page, [0, 1, 1]
    s.check(y[:6].split(rows), list(q[:6].cpu().split(rows)))
    # longer than its table: reported, the rest attended to
    longer = s.plens.clone()
    longer[0] += 1000
    pc.kv4_prefix_attention(q, s.b.cache, s.table, s.lens, s.ptable, longer, cu_q=cu_of(rows, cuda_device), cu_prefix=s.cu_prefix)
    assert nat.device_status() == nat.PN_ERR_ARG
    assert pc.kv4_prefix_attention(q[:0], s.b.cache, s.table, s.lens, s.ptable, s.plens, cu_prefix=s.cu_prefix).shape[0] == 0


@pytest.mark.parametrize("G", [1, 8, 40])
def test_prefix_quiet_and_loud(cuda_device, G):
    """Prefix and own values far apart in size, and logits far apart: each part's weight counts."""
    own, prefixes, hk, d, page = [60, 30, 45], [200], 1, 64, 16
    for up, sharp in ((2.0 ** 12, 1.0), (2.0 ** -12, 1.0), (1.0, 30.0), (2.0 ** 20, 8.0)):
        s = Shared(own, prefixes, [3], hk, d, page, cuda_device, seed=int(sharp))
        s.b.v[3] = (s.b.v[3].float() * up).to(torch.bfloat16)
        for i in range(3):
            s.b.k[i] = (s.b.k[i].float() * sharp).to(torch.bfloat16)
        s.b.store(s.b.lengths)
        s.attend([1, 2, 1], G)


def test_prefix_not_finite(cuda_device):
    """A NaN vector in a prefix reaches the rows of its group and no others."""
    s = Shared([5, 6, 7], [40, 40], [1, 2], 1, 64, 16, cuda_device)
    s.b.v[3][11, 0, 5] = float("inf")
    s.b.store(s.b.lengths)
    q = torch.randn(3, 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda_device)
    y = s.call(q, [1, 1, 1])
    assert y[0].isnan().all() and not y[1:].isnan().any()


@pytest.mark.parametrize("B,G", [(4, 2), (8, 4), (36, 8)])
def test_prefix_again_and_again(cuda_device, B, G):
    """A long prefix behind few and many rows: the same bits from every call."""
    s = Shared([9] * B, [5000], [B], 1, 128, 64, cuda_device, seed=B)
    q = torch.randn(9 * B, G, 128, device=cuda_device, dtype=torch.bfloat16)
    want = s.call(q, [9] * B)
    assert all(torch.equal(s.call(q, [9] * B), want) for _ in range(10))
    assert nat.device_status() == 0


def test_prefix_captured(cuda_device):
    """A captured call follows lengths, tables and shares; two calls on two streams."""
    s = Shared([20, 31, 8, 40], [200, 90], [2, 2], 2, 128, 16, cuda_device)
    q = torch.randn(4, 8, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda_device)
    run = lambda: pc.kv4_prefix_attention(q, s.b.cache, s.table, s.lens, s.ptable, s.plens, cu_prefix=s.cu_prefix)
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = run()
    for lens, plens, cu in (([20, 31, 8, 40], [200, 90], [0, 2, 4]), ([3, 0, 8, 17], [64, 17], [0, 1, 4]), ([20, 1, 8, 4], [0, 90], [0, 3, 3])):
        s.lens.copy_(ints(lens, cuda_device)), s.plens.copy_(ints(plens, cuda_device)), s.cu_prefix.copy_(ints(cu, cuda_device))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, run())
    want = run()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


# ── chosen pages ─────────────────────────────────────────────────────────────

def sparse_check(s, q, rows, y, pages, means, top, first, last, scale=None):
    """Every row against the definition: the choice exactly, the attention within its bound."""
    at = 0
    for i, r in enumerate(rows):
        n = s.lengths[i]
        mean = more.means(s.k[i], s.page) if n else None
        for j in range(r):
            x, pos = q[at], n - r + j
            if pos < 0:
                assert not y[at].any() and (pages[at] == -1).all()
                at += 1
                continue
            want = more.choose(x, mean, pos, s.page, top, first, last)
            G = x.shape[0] // s.hk
            for h, chosen in enumerate(want):
                assert pages[at, h].tolist() == chosen + [-1] * (top + first + last - len(chosen)), (i, j, h)
                tok = torch.cat([torch.arange(p * s.page, min((p + 1) * s.page, pos + 1)) for p in chosen])
                part = slice(h * G, (h + 1) * G)
                ref, bound = oracle.attention(x[None, part], s.k[i][tok][:, h:h + 1], s.v[i][tok][:, h:h + 1], scale)
                if y.dtype == torch.bfloat16:
                    bound = bound + 2.0 ** -8 * (ref.abs() + bound)
                err = (y[at, part].double().cpu() - ref[0]).abs()
                assert (err <= bound[0] + 1e-30).all(), (i, j, h, err.max())
            at += 1


def sparse_call(s, rows, G, top, first, last, dtype=torch.bfloat16, seed=1, **kw):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(rows), G * s.hk, s.d, generator=g).to(dtype)
    cu = cu_of(rows, s.device)
    means = pc.kv4_means(s.cache, s.d)
    pc.kv4_page_means(s.cache, means, s.table, s.lens, (sum(s.lengths),), cu_q=cu_of(s.lengths, s.device))
    y, pages = pc.kv4_sparse_attention(q.to(s.device), s.cache, means, s.table, s.lens, top, first_pages=first, last_pages=last,
                                       cu_q=cu, return_pages=True, **kw)
    sparse_check(s, q, rows, y, pages, means, top, first, last, kw.get("scale"))
    return q, means, y, pages


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
def test_page_means(cuda_device, d, page):
    lengths = [1, 0, page - 1, page, page + 1, 5 * page + 3]
    s = Batch(lengths, 3, d, page, cuda_device, seed=page)
    means = pc.kv4_means(s.cache, d)
    means.fill_(9.0)
    pc.kv4_page_means(s.cache, means, s.table, s.lens, (sum(lengths),), cu_q=cu_of(lengths, cuda_device))
    used = set()
    for i, n in enumerate(lengths):
        if n:
            phys = s.table[i, :-(-n // page)].long()
            used |= set(phys.tolist())
            assert torch.equal(means[phys].cpu(), more.means(s.k[i], page))
    free = [p for p in range(means.shape[0]) if p not in used]
    assert (means[free] == 9).all()
    # only the pages of the rows
    means.fill_(9.0)
    rows = [1, 0, 2, 1, 1, page + 5]
    pc.kv4_page_means(s.cache, means, s.table, s.lens, (sum(rows),), cu_q=cu_of(rows, cuda_device))
    for i, (n, r) in enumerate(zip(lengths, rows)):
        for p in range(-(-n // page)):
            got = means[int(s.table[i, p])]
            if r and p >= (n - r) // page:
                assert torch.equal(got.cpu(), more.means(s.k[i], page)[p])
            else:
                assert (got == 9).all()
    # rows of one length, (B, L)
    again = torch.zeros_like(means)
    whole = Batch([70, 41], 2, d, 16, cuda_device)
    again = pc.kv4_means(whole.cache, d)
    pc.kv4_page_means(whole.cache, again, whole.table, whole.lens, (2, 41))
    for i, n in enumerate((70, 41)):
        for p in range((n - 41) // 16, -(-n // 16)):
            assert torch.equal(again[int(whole.table[i, p])].cpu(), more.means(whole.k[i], 16)[p])
    assert nat.device_status() == 0


@pytest.mark.parametrize("d,hk,G,page", [(64, 3, 1, 16), (64, 1, 16, 16), (128, 2, 4, 32), (128, 1, 8, 48)])
@pytest.mark.parametrize("top,first,last", [(3, 1, 2), (0, 1, 1), (1, 0, 1), (7, 2, 3), (40, 0, 2)])
def test_sparse(cuda_device, d, hk, G, page, top, first, last):
    """Single rows and chunks, rows before the start, sequences of no and of few pages."""
    lengths = [17 * page + 5, 1, 0, 4 * page, 9 * page - 1]
    rows = [3, 1, 1, 2, 20]
    s = Batch(lengths, hk, d, page, cuda_device, seed=d + G + top)
    sparse_call(s, rows, G, top, first, last)
    assert nat.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sparse_long(cuda_device, dtype):
    """Thousands of pages: several runs of scores to a row, more pages than threads."""
    s = Batch([16 * 2600 + 3, 16 * 301], 1, 64, 16, cuda_device, seed=3)
    for top in (5, 300, 2000):
        sparse_call(s, [1, 2], 2, top, 1, 2, dtype, seed=top)


def test_sparse_group_wider_than_a_tile(cuda_device):
    s = Batch([300, 150], 1, 64, 16, cuda_device, seed=8)
    for G in (17, 40, 70):
        sparse_call(s, [1, 3], G, 4, 1, 1, seed=G, scale=0.3)


def test_sparse_ties_and_nan(cuda_device):
    """Equal scores go to the lowest page; a NaN mean and a page that is none come last; all pages
    alike (also zero) are no trouble; scores of any size and sign."""
    page, hk, d = 16, 2, 64
    s = Batch([40 * page], hk, d, page, cuda_device, seed=5)
    q = torch.randn(1, 4, d, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(cuda_device)

    def pages(means, top, table=s.table):
        return pc.kv4_sparse_attention(q, s.cache, means, table, s.lens, top, 1, 2, return_pages=True)[1][0]

    zero = pc.kv4_means(s.cache, d)
    for top in (1, 5, 36, 37):
        want = [0] + list(range(1, 1 + min(top, 37))) + [38, 39]
        for m in (zero, zero - 0.0, torch.ones_like(zero), -torch.ones_like(zero)):
            assert pages(m, top).tolist() == [want] * hk
    mean = pc.kv4_means(s.cache, d)
    pc.kv4_page_means(s.cache, mean, s.table, s.lens, (40 * page,))
    total = q[0].double().view(hk, 2, d).sum(1).cpu()
    for power in (-60, 0, 60):  # far below and above the normal range of one digit
        m = (mean.double() * 2.0 ** power).to(torch.bfloat16)
        # pages 3 to 30 alternate between two means: ties among them
        for i in range(3, 31):
            m[int(s.table[0, i])] = m[int(s.table[0, 1 + i % 2])]
        m[int(s.table[0, 20])] = float("nan")
        logical = m[s.table[0].long()].cpu()
        for top in (1, 8, 14, 15, 36, 37):
            want = more.choose(q[0].cpu(), logical, 40 * page - 1, page, top, 1, 2)
            assert pages(m, top).tolist() == want, (power, top)
    assert nat.device_status() == 0
    lost = s.table.clone()
    lost[0, 7] = -1
    got = pages(mean, 36, lost)
    assert not (got == 7).any() and nat.device_status() == 0
    assert (pages(mean, 37, lost) == 7).any() and nat.device_status() == nat.PN_ERR_ARG


@pytest.mark.parametrize("B,pages,top", [(1, 1, 1), (3, 512, 40), (40, 500, 1), (1300, 77, 9), (1200, 512, 100), (2, 513, 64), (200, 520, 17),
                                         (2, 8300, 70), (160, 2100, 300)])
@pytest.mark.parametrize("scores", ["normal", "wide", "few", "not finite"])
def test_sparse_choice_over_many_pages(cuda_device, B, pages, top, scores):
    """The choice alone, for every kernel of it: up to 512 pages, more, more than the threads hold, few rows and
    many; scores that spread evenly, over many magnitudes, that are mostly equal, with infinities and NaN."""
    d, page, first, last = 64, 16, 1, 2
    gen = torch.Generator().manual_seed(B + pages + top)
    means = torch.zeros(pages, 1, d)
    q = torch.zeros(B, 1, d)
    if scores == "normal":
        means.normal_(generator=gen)
        q.normal_(generator=gen)
    else:
        q[..., 0] = 1
        x = torch.randn(pages, generator=gen)
        if scores == "wide":
            x = x.sign() * torch.exp2(x * 30)
        elif scores == "few":
            x = (x * 0.7).round()
        else:
            x[torch.rand(pages, generator=gen) < 0.3] = float("inf")
            x[torch.rand(pages, generator=gen) < 0.2] = -float("inf")
            x[torch.rand(pages, generator=gen) < 0.2] = float("nan")
        means[:, 0, 0] = x
    means = means.to(torch.bfloat16)
    cache = pc.kv4_cache(pages, 1, d, page, cuda_device)
    order = torch.stack([torch.randperm(pages, generator=gen) for _ in range(B)])
    lens = torch.randint(1, pages * page + 1, (B,), generator=gen)
    lens[0] = pages * page
    got = pc.kv4_sparse_attention(q.to(cuda_device), cache, means.to(cuda_device), order.int().to(cuda_device),
                                  lens.int().to(cuda_device), top, first, last, return_pages=True)[1].cpu()
    for b in range(B):
        seen = -(-int(lens[b]) // page)
        score = (means[order[b, :seen], 0].double() * q[b, 0].double()).sum(-1)
        score = torch.where(score.isnan(), torch.tensor(-torch.inf, dtype=torch.float64), score)
        nan = means[order[b, :seen], 0, 0].isnan()
        free = [i for i in range(first, seen - last)]
        free.sort(key=lambda i: (bool(nan[i]), -float(score[i]), i))
        want = sorted(set(range(min(first, seen))) | set(range(max(seen - last, 0), seen)) | set(free[:top]))
        assert got[b, 0].tolist() == want + [-1] * (first + top + last - len(want)), (b, seen)
    assert nat.device_status() == 0


def test_sparse_rows_of_a_projection(cuda_device):
    """(B, L) rows as views, with and without the choice; the same as the ragged form; in place of an out."""
    B, L, H, hk, d, page = 3, 4, 6, 2, 128, 16
    s = Batch([200, 97, 64], hk, d, page, cuda_device, seed=6)
    means = pc.kv4_means(s.cache, d)
    pc.kv4_page_means(s.cache, means, s.table, s.lens, (361,), cu_q=cu_of(s.lengths, cuda_device))
    g = torch.Generator().manual_seed(3)
    for off in (0, 1):
        q = torch.randn(B, L, H * d + off, generator=g).to(torch.bfloat16).to(cuda_device)[..., off:].view(B, L, H, d)
        y, pages = pc.kv4_sparse_attention(q, s.cache, means, s.table, s.lens, 3, return_pages=True)
        assert y.shape == q.shape and pages.shape == (B, L, hk, 6)
        sparse_check(s, q.cpu().reshape(-1, H, d), [L] * B, y.reshape(-1, H, d), pages.view(-1, hk, 6), means, 3, 1, 2)
        assert torch.equal(y, pc.kv4_sparse_attention(q, s.cache, means, s.table, s.lens, 3))
        turned = q.transpose(1, 2).contiguous().transpose(1, 2)  # strides of another order
        assert torch.equal(y, pc.kv4_sparse_attention(turned, s.cache, means, s.table, s.lens, 3))
        wide = torch.full((B * L + 3, H, d), 4.0, dtype=torch.bfloat16, device=cuda_device)
        x = torch.cat((q.reshape(-1, H, d), q.reshape(-1, H, d)[:3]))
        z, p = pc.kv4_sparse_attention(x, s.cache, means, s.table, s.lens, 3, cu_q=cu_of([L] * B, cuda_device), out=wide,
                                       return_pages=True)
        assert z is wide and torch.equal(z[:B * L].view(y.shape), y) and (z[B * L:] == 4).all() and (p[B * L:] == -1).all()
        # every page: what kv4_attention computes, but for the order of its sums
        full = pc.kv4_sparse_attention(q, s.cache, means, s.table, s.lens, 50)
        whole = pc.kv4_attention(q, s.cache, s.table, s.lens)
        assert (full.float() - whole.float()).abs().max() <= 2.0 ** -6 * whole.float().abs().max()


def test_sparse_edges(cuda_device):
    """Row starts that fall; no rows; no sequences; a table with no room for the rows."""
    s = Batch([100, 50], 2, 64, 16, cuda_device)
    means = pc.kv4_means(s.cache, 64)
    q = torch.randn(6, 4, 64, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda_device)
    out = torch.full_like(q, 3.0)
    y, p = pc.kv4_sparse_attention(q, s.cache, means, s.table, s.lens, 1, cu_q=ints([0, 5, 2], cuda_device), out=out, return_pages=True)
    assert (y == 3).all() and (p == -1).all() and nat.device_status() == nat.PN_ERR_ARG
    assert pc.kv4_sparse_attention(q[:0], s.cache, means, s.table, s.lens, 1).shape == (0, 4, 64)
    y, p = pc.kv4_sparse_attention(q, s.cache, means, s.table[:0], s.lens[:0], 1, cu_q=ints([0], cuda_device), return_pages=True)
    assert not y.any() and (p == -1).all()
    pc.kv4_page_means(s.cache, means, s.table[:0], s.lens[:0], (6,), cu_q=ints([0], cuda_device))
    assert nat.device_status() == 0
    y = pc.kv4_sparse_attention(q[:2], s.cache, means, s.table[:, :4], s.lens, 1)  # sequence 0 needs seven pages
    assert nat.device_status() == nat.PN_ERR_ARG and y.isfinite().all()
    none = torch.empty(2, 0, dtype=torch.int32, device=cuda_device)
    assert not pc.kv4_sparse_attention(q[:2], s.cache, means, none, s.lens, 1).any()
    nat.device_status()


def test_sparse_captured(cuda_device):
    """A captured step (rotate and append, means, choice, attention) follows lengths and inputs."""
    B, H, hk, d, page, R = 3, 4, 2, 64, 16, 64
    lengths = [150, 33, 260]
    s = Batch([n + 20 for n in lengths], hk, d, page, cuda_device, seed=4)
    cos, sin = tables(400, R, cuda_device)
    means = pc.kv4_means(s.cache, d)
    lens = ints(lengths, cuda_device)
    pc.kv4_page_means(s.cache, means, s.table, lens, (sum(lengths),), cu_q=cu_of(lengths, cuda_device))
    g = torch.Generator().manual_seed(6)
    x = torch.randn(20, B, 1, H + 2 * hk, d, generator=g).to(torch.bfloat16).to(cuda_device)
    static = x[0].clone()

    def step(cache, means, lens):
        q, k, v = static.split((H, hk, hk), dim=2)
        lens += 1
        q = pc.kv4_append_rotary(q, k, v, cos, sin, cache, s.table, lens)
        pc.kv4_page_means(cache, means, s.table, lens, (B, 1))
        return pc.kv4_sparse_attention(q, cache, means, s.table, lens, 4, return_pages=True)

    state = [t.clone() for t in (s.cache, means, lens)]
    held = [t.clone() for t in (s.cache, means, lens)]
    step(*[t.clone() for t in state])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, pages = step(*held)
    for a, b in zip(held, state):
        a.copy_(b)
    for i in range(20):
        static.copy_(x[i])
        graph.replay()
        want, chosen = step(*state)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(pages, chosen)
        assert all(torch.equal(a, b) for a, b in zip(held, state))


def test_a_decoder_with_all_of_them(cuda_device):
    """Prompt and steps of sequences behind a prefix: rotated keys stored behind offsets, attention
    behind the prefix as over whole sequences, and over chosen pages where all are chosen."""
    H, hk, d, page, R = 4, 2, 128, 16, 64
    m, prompts, steps = 96, [7, 20, 33], 3
    g = torch.Generator().manual_seed(9)
    cos, sin = tables(300, R, cuda_device)
    B = len(prompts)
    per = -(-(max(prompts) + steps) // page)
    pool = pc.kv4_cache(6 + 2 * B * (6 + per), hk, d, page, cuda_device)
    ptable = torch.arange(6, dtype=torch.int32, device=cuda_device)[None]
    table = 6 + torch.arange(B * per, dtype=torch.int32, device=cuda_device).view(B, per)
    whole = 6 + B * per + torch.arange(B * (6 + per), dtype=torch.int32, device=cuda_device).view(B, 6 + per)
    rnd = lambda n, h: torch.randn(n, h, d, generator=g).to(torch.bfloat16).to(cuda_device)
    head = [rnd(m, h) for h in (H, hk, hk)]
    pc.kv4_append_rotary(*head, cos, sin, pool, ptable, ints([m], cuda_device))
    for b in range(B):
        pc.kv4_append_rotary(*head, cos, sin, pool, whole[b:b + 1], ints([m], cuda_device))
    offsets = torch.full((B,), m, dtype=torch.int32, device=cuda_device)
    lens = ints([0] * B, cuda_device)
    means = pc.kv4_means(pool, d)
    pc.kv4_page_means(pool, means, whole, lens + m, (B * m,))
    for rows in [prompts] + [[1] * B] * steps:
        cu = cu_of(rows, cuda_device)
        lens = lens + ints(rows, cuda_device)
        q, k, v = (rnd(sum(rows), h) for h in (H, hk, hk))
        turned = pc.kv4_append_rotary(q, k, v, cos, sin, pool, table, lens, cu_q=cu, offsets=offsets)
        assert torch.equal(turned, pc.kv4_append_rotary(q, k, v, cos, sin, pool, whole, lens + m, cu_q=cu))
        y = pc.kv4_prefix_attention(turned, pool, table, lens, ptable, ints([m], cuda_device), cu_q=cu)
        pc.kv4_page_means(pool, means, whole, lens + m, (sum(rows),), cu_q=cu)
        z = pc.kv4_sparse_attention(turned, pool, means, whole, lens + m, 64, cu_q=cu)
        x = pc.kv4_attention(turned, pool, whole, lens + m, cu_q=cu)
        # three orders of the same sums: bf16 results within two steps of the largest
        for t in (y, z):
            assert (t.float() - x.float()).abs().max() <= 2.0 ** -6 * x.float().abs().max()
    assert nat.device_status() == 0
