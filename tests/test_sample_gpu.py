"""sample_tokens against the definition in 64 bits, row by row.  The kernel's sums
are exact in 45-bit fractions, so tokens are compared for equality."""
import math

import numpy as np
import pytest
import torch

import penta_kernel as pk

pytestmark = pytest.mark.gpu


def oracle(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """One row: float64 numpy from the definition."""
    f32 = lambda v: float(np.float32(v))
    x = x.astype(np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1
    if not temperature > 0:
        return int(np.argmax(x))
    with np.errstate(invalid="ignore"):
        w = np.where(x == top, 1.0, 0.0 if math.isinf(top) else np.exp((x - top) / f32(temperature)))
    w[w < 2.0 ** -46] = 0
    order = np.argsort(-x, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    order = order[w[order] >= f32(min_p)]
    if top_p < 1:
        before = np.cumsum(w[order]) - w[order]
        order = order[(before < f32(top_p) * w[order].sum()) | (np.arange(len(order)) == 0)]  # never none
    kept = np.sort(order)
    c = np.cumsum(w[kept])
    return int(kept[min(int((c <= float(u) * c[-1]).sum()), int(np.nonzero(w[kept])[0][-1]))])


def check(x, u, **kw):
    got = pk.sample_tokens(x, u, **kw).cpu().tolist()
    xs, us = x.float().cpu().numpy(), u.cpu().numpy()
    at = lambda v, i: v[i].item() if isinstance(v, torch.Tensor) else v
    want = [oracle(xs[i], us[i], **{n: at(v, i) for n, v in kw.items()}) for i in range(len(us))]
    assert got == want
    return got


def inputs(B, V, dtype, seed, device, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, V, generator=g) * scale).to(dtype).to(device), torch.rand(B, generator=g).to(device)


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_p=0.9), dict(top_p=0.3), dict(min_p=0.1),
            dict(temperature=1.3, top_k=40, top_p=0.95, min_p=0.02), dict(top_k=1000, top_p=0.99), dict(temperature=0.0),
            dict(top_p=1e-6), dict(min_p=1.0), dict(temperature=0.05, top_p=0.5), dict(temperature=50.0, top_k=2000, top_p=0.7),
            dict(top_k=5, top_p=0.0)]


@pytest.mark.parametrize("V", [1, 2, 31, 257, 1023, 5000, 50257, 131071])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_settings(cuda_device, V, dtype):
    for n, kw in enumerate(SETTINGS):
        x, u = inputs(3 if V < 60000 else 2, V, dtype, V + n, cuda_device)
        check(x, u, **kw)


@pytest.mark.parametrize("B", [1, 2, 9, 40, 100, 200, 333])
def test_batches_with_settings_of_their_own(cuda_device, B):
    x, u = inputs(B, 4001, torch.float32, B, cuda_device)
    g = torch.Generator().manual_seed(B)
    rnd = lambda lo, hi: (lo + (hi - lo) * torch.rand(B, generator=g)).to(cuda_device)
    k = torch.randint(0, 100, (B,), generator=g, dtype=torch.int32).to(cuda_device)
    check(x, u, temperature=rnd(0.0, 2.0), top_k=k, top_p=rnd(0.3, 1.1), min_p=rnd(0.0, 0.2))


@pytest.mark.parametrize("V", [64, 3001, 50257])
def test_ties(cuda_device, V):
    """Equal logits: the lowest index first, a group cut in its middle by top-k and by top-p."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.999, 1.0 - 2.0 ** -24], device=cuda_device)
    flat = torch.zeros(5, V, device=cuda_device)
    for kw in (dict(), dict(top_k=7), dict(top_p=0.37), dict(top_k=11, top_p=0.5), dict(min_p=0.5), dict(temperature=0.0)):
        check(flat, u, **kw)
    few = torch.randint(0, 4, (5, V), generator=torch.Generator().manual_seed(V)).float().to(cuda_device)
    for kw in (dict(top_k=V // 3), dict(top_p=0.5), dict(top_p=0.9), dict(top_k=V // 2, top_p=0.8), dict(top_k=V // 3, min_p=0.2)):
        check(few, u, **kw)
        check(few.to(torch.bfloat16), u, **kw)


@pytest.mark.parametrize("V", [20, 1000, 50257])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("share", [0.03, 0.5, 0.97])
def test_zeros_of_both_signs(cuda_device, V, dtype, share):
    """-0 and +0 are equal logits, the lowest index first whatever their signs; the
    border among them lies in a short list, a long one and a row too long for it."""
    u = torch.tensor([0.0, 0.25, 0.5, 0.999, 1.0 - 2.0 ** -24], device=cuda_device)
    x = torch.rand(5, V, generator=torch.Generator().manual_seed(V)).to(cuda_device)
    x = torch.where(x < share, 0.0, -0.0).to(dtype)
    for rest in (0, 7):  # zeros alone; every seventh logit below them, one above
        if rest:
            x[:, ::rest] = -1.0
            x[:, V // 2] = 1.0
        for kw in (dict(top_k=V * 2 // 5), dict(top_p=0.37), dict(top_k=V // 2, top_p=0.6), dict(top_k=3), dict(temperature=0.0),
                   dict()):
            check(x, u, **kw)


def test_masked_and_special_logits(cuda_device):
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    x, u = inputs(12, 700, torch.float32, 3, cuda_device)
    x[0] = -inf                     # nothing left
    x[1] = nan
    x[2, 1:] = -inf                 # one token
    x[3, :650] = low                # masked by the type's lowest value
    x[4, ::2] = nan
    x[5, [7, 90, 400]] = inf        # these share all the weight
    x[6] = low                      # all masked alike: all alike
    x[7] = -inf
    x[7, 699] = low
    x[8] *= 1e30
    x[9] *= 1e-30
    x[10, 5] = 3e38
    x[11] = -0.0
    x[11, 100:] = 0.0
    for kw in (dict(), dict(top_k=3), dict(top_p=0.6), dict(min_p=0.01), dict(top_k=20, top_p=0.9, temperature=0.5),
               dict(temperature=0.0)):
        check(x, u, **kw)
    assert pk.sample_tokens(x[:2], u[:2]).tolist() == [-1, -1]


def test_ends_of_the_unit_interval(cuda_device):
    x, _ = inputs(4, 999, torch.float32, 5, cuda_device)
    x[:, 0] = -100
    x[:, 998] = -100
    u = torch.tensor([0.0, 2.0 ** -30, 1 - 2.0 ** -24, 1.0], device=cuda_device)
    check(x, u)
    check(x, u, top_k=10)
    check(x, u, top_p=0.8)


def test_extreme_temperatures(cuda_device):
    """Near zero the largest logit, at infinity every finite one alike, NaN as zero."""
    x, u = inputs(5, 3000, torch.float32, 11, cuda_device)
    x[1, ::3] = -float("inf")
    x[2] = x[2].round()
    for t in (1e-30, 1e-9, 1e-3, 1e6, 1e29, 1e30):
        check(x, u, temperature=t)
        check(x, u, temperature=t, top_p=0.5)
        check(x, u, temperature=t, top_k=17, top_p=0.9)
    hot = pk.sample_tokens(x, u, temperature=float("inf"))
    assert hot.tolist() == pk.sample_tokens(x, u, temperature=1e30).tolist()
    nan = torch.full((5,), float("nan"), device=cuda_device)
    assert pk.sample_tokens(x, u, temperature=nan).tolist() == x.argmax(-1).tolist()


def test_strided_logits_and_the_models_shape(cuda_device):
    wide, u = inputs(6, 2100, torch.bfloat16, 8, cuda_device)
    for x in (wide[:, 3:2050], wide[::2], wide[:, ::2], wide.t()[:6, :6]):
        check(x, u[:x.shape[0]], top_k=30, top_p=0.9)
    assert pk.sample_tokens(wide[:0], u[:0]).shape == (0,)


@pytest.mark.parametrize("V", [200000, 1 << 18])
def test_largest_vocabularies(cuda_device, V):
    x, u = inputs(2, V, torch.float32, V, cuda_device)
    for kw in (dict(), dict(top_p=0.9), dict(top_k=64)):
        check(x, u, **kw)
    check(x * 1e-4, u, top_p=0.5)  # nearly flat: a nucleus of half the vocabulary


def test_same_inputs_same_tokens_stream_and_graph(cuda_device):
    x, u = inputs(16, 50257, torch.bfloat16, 2, cuda_device, scale=1.0)
    kw = dict(top_p=0.95, temperature=0.9)
    want = check(x, u, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pk.sample_tokens(x, u, **kw)
    side.synchronize()
    assert got.tolist() == want
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pk.sample_tokens(x, u, **kw)
    x.copy_(x.flip(0))
    u.copy_(u.flip(0))
    for _ in range(2):
        graph.replay()
        assert got.tolist() == want[::-1]


def test_frequencies(cuda_device):
    """Evenly spread numbers give every token its share."""
    x = torch.log(torch.tensor([[0.5, 0.125, 0.25, 0.125]], device=cuda_device)).repeat(64, 1)
    u = (torch.arange(64, device=cuda_device) + 0.5) / 64
    assert torch.bincount(pk.sample_tokens(x, u), minlength=4).tolist() == [32, 8, 16, 8]
