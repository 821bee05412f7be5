"""RMS norm with the residual's addition (rms_norm, rms_norm_i8) against the
formula in 64 bits, and against the operators it joins.

Tolerances: y = (h * rstd) * w has three fp32 roundings (rstd and two products),
each within 2^-24 of its value, and one more where the output is bf16 (2^-8)."""
import ctypes

import pytest
import torch

import penta_kernel as pk
import penta_native as nat

pytestmark = pytest.mark.gpu

T32 = 3.01 * 2.0 ** -24


def _inputs(M, C, dtype, seed, device, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(M, C, generator=g) * spread).to(dtype).to(device)
    r = torch.randn(M, C, generator=g).to(dtype).to(device)
    w = (1 + 0.3 * torch.randn(C, generator=g)).to(device)
    return x, r, w


def _oracle(h, w, eps):
    h = h.double().cpu()
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    return y if w is None else y * w.double().cpu()


def _check(y, want, out_dtype):
    bound = want.abs() * (T32 if out_dtype == torch.float32 else T32 + 2.0 ** -8) + 1e-38
    assert ((y.double().cpu() - want).abs() <= bound).all()


SHAPES = [(1, 1), (2, 7), (3, 64), (5, 100), (1, 768), (257, 768), (1021, 1001), (33, 1024), (9, 4096), (148, 8192),
          (3, 8200), (4, 16384), (2, 16392), (3, 28672), (2, 65536), (1, 131080)]


@pytest.mark.parametrize("M,C", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
def test_matches_formula(cuda_device, M, C, dtype, residual):
    x, r, w = _inputs(M, C, dtype, M + C, cuda_device)
    h = (x.float() + r.float()).to(dtype) if residual else x
    want = _oracle(h, w, 1e-6)
    for out_dtype in (torch.float32, torch.bfloat16):
        got = pk.rms_norm(x, w, 1e-6, residual=r if residual else None, out_dtype=out_dtype)
        if residual:
            got, stream = got
            assert torch.equal(stream, h)
        assert got.dtype == out_dtype and got.shape == x.shape
        _check(got, want, out_dtype)


@pytest.mark.parametrize("M,C", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
def test_int8_is_the_quantiser_of_the_norm(cuda_device, M, C, dtype, residual):
    x, r, w = _inputs(M, C, dtype, 3 * M + C, cuda_device, spread=4.0)
    res = r if residual else None
    y = pk.rms_norm(x, w, 1e-5, residual=res, out_dtype=torch.float32)
    xq, s, total, *h = pk.rms_norm_i8(x, w, 1e-5, residual=res)
    if residual:
        y, stream = y
        assert torch.equal(h[0], stream)
    want_q, want_s, want_total = pk.quantize_activations_i8(y)
    assert torch.equal(xq, want_q) and torch.equal(s, want_s) and torch.equal(total, want_total)
    # and the codes are those of the formula: within half a step, and what two relative errors move
    exact = _oracle(h[0] if residual else x, w, 1e-5)
    q = xq[:, :C].double().cpu()
    step = exact.abs().amax(-1, keepdim=True) / 127
    assert ((q - exact / step).abs() <= 0.5 + 127 * 4 * T32).all()


@pytest.mark.parametrize("weight", ["none", "bf16"])
def test_weight_types(cuda_device, weight):
    x, _, w = _inputs(17, 512, torch.bfloat16, 5, cuda_device)
    w = None if weight == "none" else w.to(torch.bfloat16)
    _check(pk.rms_norm(x, w, 1e-6, out_dtype=torch.float32), _oracle(x, w, 1e-6), torch.float32)
    y = pk.rms_norm(x, w, 1e-6, out_dtype=torch.float32)
    assert torch.equal(pk.rms_norm_i8(x, w, 1e-6)[0], pk.quantize_activations_i8(y)[0])


def test_strides_and_alignment(cuda_device):
    """Views that start off a 16-byte boundary, transposed inputs, leading dimensions."""
    base = torch.randn(4, 6, 264, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(cuda_device)
    w = torch.randn(265, generator=torch.Generator().manual_seed(2)).to(cuda_device)
    for x, ww in ((base[..., 3:259], w[1:257]), (base.transpose(0, 1)[..., :256], w[:256]), (base[1:, :, 1:], w[2:265])):
        want = _oracle(x, ww, 1e-6)
        _check(pk.rms_norm(x, ww, 1e-6, out_dtype=torch.float32), want, torch.float32)
        flat = x.contiguous().reshape(-1)
        shifted = torch.cat((flat[:1], flat))[1:].view(x.shape)  # contiguous, two bytes off
        assert torch.equal(pk.rms_norm(shifted, ww, 1e-6), pk.rms_norm(x, ww, 1e-6))
        assert torch.equal(pk.rms_norm_i8(shifted, ww, 1e-6)[0], pk.rms_norm_i8(x, ww, 1e-6)[0])
    assert pk.rms_norm(base[:0], w[:264]).shape == (0, 6, 264)
    assert pk.rms_norm_i8(base[:0], w[:264])[0].shape == (0, 288)


@pytest.mark.parametrize("C", [768, 1001, 8192])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_zero_rows_and_rows_that_are_not_finite(cuda_device, C, dtype):
    x, r, w = _inputs(6, C, dtype, 9, cuda_device)
    clean = pk.rms_norm_i8(x, w, 1e-6, residual=r)
    x[1] = 0
    r[1] = 0
    x[2, C // 2] = float("nan")
    x[3, C - 1] = float("inf")
    r[4, 0] = -float("inf")
    xq, s, total, h = pk.rms_norm_i8(x, w, 1e-6, residual=r)
    assert s[1] == 1 and total[1] == 0 and not xq[1].any()
    for i in (2, 3, 4):
        assert torch.isnan(s[i]) and total[i] == 0 and not xq[i].any()
    for i in (0, 5):
        assert torch.equal(xq[i], clean[0][i]) and s[i] == clean[1][i]
    y, _ = pk.rms_norm(x, w, 1e-6, residual=r)
    assert not y[1].any() and torch.isnan(y[2]).all()
    assert torch.isfinite(y[0]).all() and torch.isfinite(y[5]).all()


@pytest.mark.parametrize("C", [512, 1001])
def test_tiny_values(cuda_device, C):
    """Rows whose scale is a subnormal number, or rounds to zero."""
    x, _, _ = _inputs(6, C, torch.float32, 2, cuda_device)
    w = torch.full((C,), 1e-38, device=cuda_device)
    for k, size in enumerate((1.0, 1e-3, 1e-5, 1e-6, 3e-7, 1e-8)):
        y = pk.rms_norm(x, w * size, 1e-6, out_dtype=torch.float32)
        xq, s, total = pk.rms_norm_i8(x, w * size, 1e-6)
        want = pk.quantize_activations_i8(y)
        assert torch.equal(xq, want[0]) and torch.equal(s, want[1]) and torch.equal(total, want[2]), size


def test_residual_stream_in_place(cuda_device):
    """The C ABI may write the stream over x or over the residual."""
    for dtype, C in ((torch.bfloat16, 1024), (torch.float32, 1001), (torch.bfloat16, 40000)):
        x, r, w = _inputs(7, C, dtype, 21, cuda_device)
        want, h = pk.rms_norm(x, w, 1e-6, residual=r)
        for over in (0, 1):
            a, b = x.clone(), r.clone()
            y = torch.empty(7, C, dtype=torch.bfloat16, device=cuda_device)
            dt = nat.PN_F32 if dtype == torch.float32 else nat.PN_BF16
            st = nat.load().pn_rms_norm(a.data_ptr(), dt, b.data_ptr(), 7, C, w.data_ptr(), nat.PN_F32,
                                        ctypes.c_double(1e-6), (a, b)[over].data_ptr(), y.data_ptr(), nat.PN_BF16,
                                        nat.stream_of(a))
            assert st == nat.PN_OK
            assert torch.equal((a, b)[over], h) and torch.equal(y, want)


def test_feeds_the_int8_product(cuda_device):
    """residual add + norm + quantise + int8 product, as a decoder block runs them."""
    x, r, w = _inputs(37, 1000, torch.bfloat16, 4, cuda_device)
    packed, K, gamma = pk.quantize_and_pack(torch.randn(300, 1000, generator=torch.Generator().manual_seed(6)).to(cuda_device))
    xq, s, total, h = pk.rms_norm_i8(x, w, 1e-6, residual=r)
    got = pk.penta_linear_i8_prequant(xq, s, total, K, packed, gamma)
    want = pk.penta_linear_i8(pk.rms_norm(h, w, 1e-6, out_dtype=torch.float32), packed, gamma, K)
    assert torch.equal(got, want)
    assert nat.device_status() == 0


def test_side_stream_and_graph(cuda_device):
    x, r, w = _inputs(64, 768, torch.bfloat16, 8, cuda_device)
    want = pk.rms_norm_i8(x, w, 1e-6, residual=r)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = pk.rms_norm_i8(x, w, 1e-6, residual=r)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = pk.rms_norm_i8(x, w, 1e-6, residual=r)
    x.copy_(x.flip(0))
    r.copy_(r.flip(0))
    graph.replay()
    assert all(torch.equal(a, b.flip(0)) for a, b in zip(got, want))


@pytest.mark.parametrize("M,C", [(0, 8), (1, 1), (3, 31), (5, 32), (2, 768), (17, 1001), (301, 1000), (4, 8200)])
@pytest.mark.parametrize("out_dtype", [torch.bfloat16, torch.float32])
def test_dequantize(cuda_device, M, C, out_dtype):
    """The values that codes stand for: one fp32 product, and one rounding where bf16 is asked for."""
    x, _, _ = _inputs(M, C, torch.bfloat16, C, cuda_device)
    xq, s, _ = pk.rms_norm_i8(x, None, 1e-6)
    if M > 2:
        s[1] = float("nan")
    want = (xq[:, :C].float() * s[:, None]).to(out_dtype)
    got = pk.dequantize_activations_i8(xq, s, C, out_dtype)
    assert got.dtype == out_dtype and torch.equal(torch.nan_to_num(got, nan=123.0), torch.nan_to_num(want, nan=123.0))
