"""Attention over long sequences of the 4-bit cache (penta_cache): its error must not grow with the
number of tokens that a block walks, whichever kernel does it."""
import pytest
import torch

import penta_cache as pc
import penta_native as nat

pytestmark = pytest.mark.gpu


def attend64(q, k, v):
    """q (rows, H, d), k and v (n, hk, d): every row sees all tokens; float64."""
    r, H, d = q.shape
    hk = k.shape[1]
    x = torch.einsum("rhgd,nhd->rhgn", q.double().view(r, hk, H // hk, d), k.double()) * d ** -0.5
    p = x.softmax(-1)
    return torch.einsum("rhgn,nhd->rhgd", p, v.double()).reshape(r, H, d)


class Long:
    """One sequence of n tokens, random keys and values, that any number of table rows share.
    values "skewed": of mean zero but mostly below it, as codes are then; "loud": a few dims are far above the others;
    "largest", "least": near the ends of the range that kv4_attention states."""

    def __init__(self, n, hk, d, device, page=64, values="normal"):
        g = torch.Generator(device=device).manual_seed(n + d)
        W = -(-n // page)
        self.n, self.hk, self.d, self.device = n, hk, d, device
        self.cache = pc.kv4_cache(W + 1, hk, d, page, device)
        self.table = torch.arange(W, dtype=torch.int32, device=device)[None]
        self.lens = torch.tensor([n], dtype=torch.int32, device=device)
        k, v = (torch.randn(n, hk, d, generator=g, device=device) for _ in range(2))
        if values == "skewed":
            v = v.abs().square() - 1
        elif values == "loud":
            v[..., :d // 2:d // 8] += 40
        elif values in ("largest", "least"):
            v = v * 2.0 ** (104 if values == "largest" else -48)
        self.quiet = torch.ones(d, dtype=torch.bool, device=device)
        if values == "loud":
            self.quiet[:d // 2:d // 8] = False
        pc.kv4_append(k, v, self.cache, self.table, self.lens)
        self.k, self.v = pc.kv4_gather(self.cache, d, self.table, self.lens, (n,), dtype=torch.float32)

    def queries(self, B, L, H):
        # (fp32, so that the results are not rounded; bf16 values, so that the queries are not either)
        g = torch.Generator(device=self.device).manual_seed(B)
        return torch.randn(B, L, H, self.d, generator=g, device=self.device).to(torch.bfloat16).float()

    def limit(self):
        """A weight times its value's scale is rounded to 11 bits, by at most 2^-11 of itself and independently
        from token to token, and meets a code: the error of a sum over the tokens is to the sum as that times
        the codes' root mean square, in the values' units v - z, is to the values'.  (Its own root mean square is
        at most 1 / sqrt 3 of this limit, and it is taken over thousands of dims.)  No length in it."""
        code, v = (self.v - self.v.amin(-1, keepdim=True))[..., self.quiet], self.v[..., self.quiet]
        return 2.0 ** -11 * float(code.square().mean().sqrt() / (v - v.mean((0, 1))).square().mean().sqrt())

    def check(self, q, y, rows, more=0.0):
        want = attend64(torch.stack([q[b, l] for b, l in rows]), self.k, self.v)
        want = want[..., self.quiet]
        got = torch.stack([y[b, l] for b, l in rows]).double()[..., self.quiet]
        err = float((got - want).norm() / want.norm())
        assert err <= self.limit() + more, (err, self.limit())
        assert nat.device_status() == 0


# sequences x rows x query heads, on eight kv heads: the 8-row, 16-row, chunk and tcgen05 kernels, with so many row
# tiles that a block walks a sequence alone, or half of it
SHAPES = [(64, 1, 8), (64, 1, 128), (20, 64, 8), (8, 512, 8)]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,L,H", SHAPES)
@pytest.mark.parametrize("n", [1000, 131072])
def test_attention(cuda_device, B, L, H, d, n):
    s = Long(n, 8, d, cuda_device)
    q = s.queries(B, L, H)
    y = pc.kv4_attention(q, s.cache, s.table.expand(B, -1).contiguous(), s.lens.expand(B).contiguous())
    s.check(q, y, [(0, L - 1), (B // 2, L - 1), (B - 1, L - 1)])


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,L,H", [(4, 1, 8), (16, 1, 8), (64, 1, 8), (64, 8, 8), (50, 1, 128)])
def test_prefix(cuda_device, B, L, H, d):
    """Rows without tokens of their own, behind 131072 that they share."""
    s = Long(131072, 8, d, cuda_device)
    q = s.queries(B, L, H)
    none = torch.zeros(B, dtype=torch.int32, device=cuda_device)
    y = pc.kv4_prefix_attention(q, s.cache, torch.zeros(B, 0, dtype=torch.int32, device=cuda_device), none, s.table, s.lens)
    s.check(q, y, [(0, 0), (B // 2, L - 1), (B - 1, L // 2)])


def test_a_million_tokens(cuda_device):
    """600 rows share a sequence, each a tile of its own."""
    s = Long(1 << 20, 1, 64, cuda_device)
    q = s.queries(600, 1, 4)
    y = pc.kv4_attention(q, s.cache, s.table.expand(600, -1).contiguous(), s.lens.expand(600).contiguous())
    s.check(q, y, [(0, 0), (300, 0), (599, 0)])


@pytest.mark.parametrize("values", ["skewed", "loud"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,L,H", SHAPES)
def test_values_to_one_side(cuda_device, B, L, H, d, values):
    """Codes whose mean is not the middle one; of the loud dims' neighbours, whose results are small beside theirs."""
    s = Long(131072, 8, d, cuda_device, values=values)
    q = s.queries(B, L, H)
    y = pc.kv4_attention(q, s.cache, s.table.expand(B, -1).contiguous(), s.lens.expand(B).contiguous())
    s.check(q, y, [(0, L - 1), (B // 2, L - 1), (B - 1, L - 1)])


@pytest.mark.parametrize("values", ["largest", "least"])
@pytest.mark.parametrize("B,L,H", SHAPES)
def test_values_of_any_size(cuda_device, B, L, H, values):
    """No sum on the way leaves fp32's range where the values are in theirs."""
    s = Long(3000, 8, 64, cuda_device, values=values)
    q = s.queries(B, L, H)
    y = pc.kv4_attention(q, s.cache, s.table.expand(B, -1).contiguous(), s.lens.expand(B).contiguous())
    up = 2.0 ** (-104 if values == "largest" else 48)
    s.v = s.v * up  # (the check squares)
    s.check(q, y * up, [(0, L - 1), (B // 2, L - 1), (B - 1, L - 1)])


@pytest.mark.parametrize("B,L,H", [(450, 1, 16), (450, 64, 1), (300, 128, 1)])
def test_a_million_tokens_in_every_kernel(cuda_device, B, L, H):
    """A block walks all of them.  Each product of 16 tokens may cut 2^-24 of the sum so far, which is the result's."""
    s = Long(1 << 20, 1, 64, cuda_device)
    q = s.queries(B, L, H)
    y = pc.kv4_attention(q, s.cache, s.table.expand(B, -1).contiguous(), s.lens.expand(B).contiguous())
    s.check(q, y, [(0, L - 1), (B // 2, L - 1), (B - 1, L - 1)], more=s.n / 16 * 2.0 ** -24)
