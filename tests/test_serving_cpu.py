"""Refusals of the serving operators (norm, 4-bit cache, sampling): through the C
ABI with made-up pointers (every case fails before anything touches CUDA) and
through Python with CPU tensors."""
import ctypes

import pytest
import torch

import penta_cache as pc
import penta_kernel as pk
import penta_native as nat

P = 1 << 20
D = ctypes.c_double


def rms(**kw):
    a = dict(x=P, dt=nat.PN_BF16, r=None, M=4, C=64, w=None, wdt=nat.PN_F32, eps=1e-6, h=None, y=P, ydt=nat.PN_BF16)
    a.update(kw)
    return nat.load().pn_rms_norm(a["x"], a["dt"], a["r"], a["M"], a["C"], a["w"], a["wdt"], D(a["eps"]), a["h"], a["y"],
                                  a["ydt"], None)


def rms_i8(**kw):
    a = dict(x=P, dt=nat.PN_BF16, r=None, M=4, C=64, w=None, wdt=nat.PN_F32, eps=1e-6, h=None, q=P, pitch=64, s=P, t=P)
    a.update(kw)
    return nat.load().pn_rms_norm_i8(a["x"], a["dt"], a["r"], a["M"], a["C"], a["w"], a["wdt"], D(a["eps"]), a["h"],
                                     a["q"], a["pitch"], a["s"], a["t"], None)


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), nat.PN_ERR_ARG), (dict(dt=nat.PN_I8), nat.PN_ERR_DTYPE), (dict(w=P, wdt=nat.PN_I32), nat.PN_ERR_DTYPE),
    (dict(C=0), nat.PN_ERR_SHAPE), (dict(M=-1), nat.PN_ERR_SHAPE), (dict(eps=-1.0), nat.PN_ERR_ARG),
    (dict(eps=float("nan")), nat.PN_ERR_ARG), (dict(r=P), nat.PN_ERR_ARG), (dict(h=P), nat.PN_ERR_ARG),
    (dict(x=P + 1), nat.PN_ERR_ALIGN), (dict(r=P, h=P + 1), nat.PN_ERR_ALIGN), (dict(w=P + 2), nat.PN_ERR_ALIGN)])
def test_rms_refusals(kw, want):
    assert rms(**kw) == want
    assert rms_i8(**kw) == want


def test_rms_output_refusals():
    assert rms(y=None) == nat.PN_ERR_ARG
    assert rms(ydt=nat.PN_I8) == nat.PN_ERR_DTYPE
    assert rms(y=P + 1) == nat.PN_ERR_ALIGN
    assert rms_i8(q=None) == nat.PN_ERR_ARG and rms_i8(s=None) == nat.PN_ERR_ARG and rms_i8(t=None) == nat.PN_ERR_ARG
    assert rms_i8(pitch=63) == nat.PN_ERR_SHAPE and rms_i8(pitch=72) == nat.PN_ERR_SHAPE
    assert rms_i8(q=P + 8) == nat.PN_ERR_ALIGN and rms_i8(s=P + 2) == nat.PN_ERR_ALIGN


def test_dequantize_refusals():
    call = lambda q=P, pitch=64, s=P, M=4, K=60, y=P, dt=nat.PN_BF16: nat.load().pn_dequant_act_i8(q, pitch, s, M, K, y, dt, None)
    assert call(q=None) == call(s=None) == call(y=None) == nat.PN_ERR_ARG
    assert call(dt=nat.PN_I8) == nat.PN_ERR_DTYPE
    assert call(K=0) == call(K=65) == call(pitch=72) == call(M=-1) == nat.PN_ERR_SHAPE
    assert call(q=P + 8) == call(s=P + 2) == call(y=P + 1) == nat.PN_ERR_ALIGN


BASE = dict(cache=P, n_pages=8, hk=2, page=64, d=64, table=P, ld=4, w=4, lens=P, cu=None, B=2, T=2)


def append(**kw):
    a = dict(BASE, k=P, v=P, dt=nat.PN_BF16)
    a.update(kw)
    return nat.load().pn_kv4_append(a["k"], 1, 1, 1, a["v"], 1, 1, 1, a["dt"], a["cache"], a["n_pages"], a["hk"], a["page"],
                                    a["d"], a["table"], a["ld"], a["w"], a["lens"], a["cu"], a["B"], a["T"], None)


def gather(**kw):
    a = dict(BASE, k=P, v=P, dt=nat.PN_BF16)
    a.update(kw)
    return nat.load().pn_kv4_gather(a["cache"], a["n_pages"], a["hk"], a["page"], a["d"], a["table"], a["ld"], a["w"],
                                    a["lens"], a["cu"], a["B"], a["T"], a["k"], a["v"], a["dt"], None)


def attention(**kw):
    a = dict(BASE, k=P, v=P, dt=nat.PN_BF16, heads=4, ws=P, size=1 << 30, scale=1.0)
    a.update(kw)
    return nat.load().pn_kv4_attention(a["k"], 1, 1, 1, a["dt"], a["heads"], a["cache"], a["n_pages"], a["hk"], a["page"],
                                       a["d"], a["table"], a["ld"], a["w"], a["lens"], a["cu"], a["B"], a["T"],
                                       ctypes.c_float(a["scale"]), a["v"], a["ws"], a["size"], None)


@pytest.mark.parametrize("call", [append, gather, attention])
@pytest.mark.parametrize("kw,want", [
    (dict(d=32), nat.PN_ERR_SHAPE), (dict(d=96), nat.PN_ERR_SHAPE), (dict(d=0), nat.PN_ERR_SHAPE),
    (dict(page=8), nat.PN_ERR_SHAPE), (dict(page=40), nat.PN_ERR_SHAPE), (dict(page=0), nat.PN_ERR_SHAPE),
    (dict(page=1 << 20), nat.PN_ERR_SHAPE), (dict(hk=0), nat.PN_ERR_SHAPE), (dict(n_pages=-1), nat.PN_ERR_SHAPE),
    (dict(n_pages=1 << 32), nat.PN_ERR_SHAPE), (dict(ld=3), nat.PN_ERR_SHAPE), (dict(w=-1), nat.PN_ERR_SHAPE),
    (dict(w=1 << 25, ld=1 << 25), nat.PN_ERR_SHAPE), (dict(T=-2), nat.PN_ERR_SHAPE), (dict(T=3), nat.PN_ERR_SHAPE),
    (dict(B=-1), nat.PN_ERR_SHAPE), (dict(cache=None), nat.PN_ERR_ARG), (dict(table=None), nat.PN_ERR_ARG),
    (dict(lens=None), nat.PN_ERR_ARG), (dict(k=None), nat.PN_ERR_ARG), (dict(v=None), nat.PN_ERR_ARG),
    (dict(cache=P + 8), nat.PN_ERR_ALIGN), (dict(table=P + 2), nat.PN_ERR_ALIGN), (dict(lens=P + 1), nat.PN_ERR_ALIGN),
    (dict(cu=P + 2), nat.PN_ERR_ALIGN), (dict(dt=nat.PN_I8), nat.PN_ERR_DTYPE)])
def test_kv4_refusals(call, kw, want):
    assert call(**kw) == want


def test_kv4_attention_refusals():
    L = nat.load()
    for heads in (0, 1, 3, 1 << 20):
        assert attention(heads=heads) == nat.PN_ERR_SHAPE
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert attention(scale=scale) == nat.PN_ERR_ARG
    assert attention(v=P + 8) == nat.PN_ERR_ALIGN
    need = L.pn_kv4_attention_workspace_size(2, 2, 4, 2, 64)
    assert need > 0 and L.pn_kv4_attention_workspace_size(0, 0, 4, 2, 64) == 0
    assert L.pn_kv4_block_bytes(64, 64) == 64 * 36


def sample(**kw):
    a = dict(x=P, dt=nat.PN_F32, rows=4, V=100, ld=100, u=P, t=None, k=None, p=None, m=None, out=P)
    a.update(kw)
    F = ctypes.c_float
    return nat.load().pn_sample_tokens(a["x"], a["dt"], a["rows"], a["V"], a["ld"], a["u"], a["t"], F(1.0), a["k"], 0, a["p"],
                                       F(1.0), a["m"], F(0.0), a["out"], None)


@pytest.mark.parametrize("kw,want", [
    (dict(x=None), nat.PN_ERR_ARG), (dict(u=None), nat.PN_ERR_ARG), (dict(out=None), nat.PN_ERR_ARG),
    (dict(dt=nat.PN_I8), nat.PN_ERR_DTYPE), (dict(V=0), nat.PN_ERR_SHAPE), (dict(V=(1 << 18) + 1, ld=1 << 19), nat.PN_ERR_SHAPE),
    (dict(ld=99), nat.PN_ERR_SHAPE), (dict(rows=-1), nat.PN_ERR_SHAPE), (dict(x=P + 2), nat.PN_ERR_ALIGN),
    (dict(out=P + 4), nat.PN_ERR_ALIGN), (dict(t=P + 1), nat.PN_ERR_ALIGN), (dict(k=P + 2), nat.PN_ERR_ALIGN)])
def test_sample_refusals(kw, want):
    assert sample(**kw) == want


def test_python_refusals():
    """CPU tensors, wrong types and shapes raise AssertionError."""
    x = torch.randn(2, 64)
    with pytest.raises(AssertionError, match="CUDA"):
        pk.rms_norm(x)
    with pytest.raises(AssertionError, match="CUDA"):
        pk.rms_norm_i8(x)
    with pytest.raises(AssertionError, match="CUDA"):
        pk.sample_tokens(x, torch.zeros(2))
    with pytest.raises(AssertionError, match="logits"):
        pk.sample_tokens(x[0], torch.zeros(2))
    q = torch.randn(2, 1, 4, 64)
    cache = pc.kv4_cache(2, 2, 64, 16, "cpu")
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    with pytest.raises(AssertionError, match="CUDA"):
        pc.kv4_attention(q, cache, table, lens)
    with pytest.raises(AssertionError, match="CUDA"):
        pc.kv4_append(q[:, :, :2], q[:, :, :2], cache, table, lens)
    with pytest.raises(AssertionError, match="CUDA"):
        pc.kv4_gather(cache, 64, table, lens, (2, 1))
    with pytest.raises(AssertionError, match="head_dim"):
        pc.kv4_cache(2, 2, 80)
    with pytest.raises(AssertionError, match="page_size"):
        pc.kv4_cache(2, 2, 64, 24)


def test_cache_argument_checks():
    """The checks that the three cache calls share, on CPU tensors."""
    cache = pc.kv4_cache(2, 2, 64, 16, "cpu")
    table, lens, dev = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32), -1
    assert pc._cache_args(cache, 64, table, lens, None, dev) == (2, 2, 16)
    cu = torch.zeros(3, dtype=torch.int32)
    bad = [dict(cache=cache.float()), dict(cache=cache[..., :-4]), dict(cache=cache[:, :, :1]), dict(head_dim=128),
           dict(table=table.long()), dict(table=table[0]), dict(lens=lens.long()), dict(lens=lens[:1]), dict(cu=cu.long()),
           dict(cu=cu[:2]), dict(table=torch.zeros(2, 8, dtype=torch.int32)[:, ::2]),
           dict(table=torch.zeros(1, 8, dtype=torch.int32).expand(2, 8)), dict(dev=0)]
    for kw in bad:
        a = dict(cache=cache, head_dim=64, table=table, lens=lens, cu=cu, dev=dev, **{})
        a.update(kw)
        with pytest.raises(AssertionError):
            pc._cache_args(a["cache"], a["head_dim"], a["table"], a["lens"], a["cu"], a["dev"])
    q = torch.randn(2, 3, 4, 64)
    assert pc._rows(q, 2, None, "q") == (768, 256, 64, 6)
    assert pc._rows(q.view(6, 4, 64), 2, None, "q") == (768, 256, 64, 6)
    assert pc._rows(q.view(6, 4, 64), 4, cu, "q") == (0, 256, 64, 6)
    for x, B, c in ((q, 3, None), (q, 2, cu), (q[0, 0], 2, None), (q.view(6, 4, 64), 4, None), (q.view(6, 4, 64), 0, None)):
        with pytest.raises(AssertionError):
            pc._rows(x, B, c, "q")
