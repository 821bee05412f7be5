"""Refusals of rotated append, attention behind prefixes and attention over chosen
pages: through the C ABI with made-up pointers (every case fails before anything
touches CUDA) and through Python with CPU tensors."""
import ctypes

import pytest
import torch

import penta_cache as pc
import penta_native as nat

P = 1 << 20
F = ctypes.c_float
BASE = dict(q=P, k=P, v=P, dt=nat.PN_BF16, heads=4, cache=P, n_pages=8, hk=2, page=64, d=64, table=P, ld=4, w=4, lens=P, cu=None,
            B=2, T=2, scale=1.0, out=P, ws=P, size=1 << 40)


def rotary(**kw):
    a = dict(BASE, cos=P, sin=P, n=100, stride=32, R=64, offsets=None)
    a.update(kw)
    return nat.load().pn_kv4_append_rotary(a["q"], 1, 1, 1, a["heads"], a["k"], 1, 1, 1, a["v"], 1, 1, 1, a["dt"], a["cos"],
                                           a["sin"], a["n"], a["stride"], a["R"], 0, a["offsets"], a["cache"], a["n_pages"],
                                           a["hk"], a["page"], a["d"], a["table"], a["ld"], a["w"], a["lens"], a["cu"], a["B"],
                                           a["T"], a["out"], 0, None)


def prefix(**kw):
    a = dict(BASE, ptable=P, pld=4, pw=4, plens=P, cup=P, n=1)
    a.update(kw)
    return nat.load().pn_kv4_prefix_attention(a["q"], 1, 1, 1, a["dt"], a["heads"], a["cache"], a["n_pages"], a["hk"], a["page"],
                                              a["d"], a["table"], a["ld"], a["w"], a["lens"], a["cu"], a["B"], a["T"],
                                              a["ptable"], a["pld"], a["pw"], a["plens"], a["cup"], a["n"], F(a["scale"]),
                                              a["out"], a["ws"], a["size"], None)


def page_means(**kw):
    a = dict(BASE, means=P)
    a.update(kw)
    return nat.load().pn_kv4_page_means(a["cache"], a["n_pages"], a["hk"], a["page"], a["d"], a["table"], a["ld"], a["w"],
                                        a["lens"], a["cu"], a["B"], a["T"], a["means"], None)


def sparse(**kw):
    a = dict(BASE, means=P, first=1, last=1, top=1, chosen=None)
    a.update(kw)
    return nat.load().pn_kv4_sparse_attention(a["q"], 1, 1, 1, a["dt"], a["heads"], a["cache"], a["means"], a["n_pages"], a["hk"],
                                              a["page"], a["d"], a["table"], a["ld"], a["w"], a["lens"], a["cu"], a["B"], a["T"],
                                              a["first"], a["last"], a["top"], F(a["scale"]), a["out"], a["chosen"], a["ws"],
                                              a["size"], None)


@pytest.mark.parametrize("call", [rotary, prefix, page_means, sparse])
@pytest.mark.parametrize("kw,want", [
    (dict(d=32), nat.PN_ERR_SHAPE), (dict(d=96), nat.PN_ERR_SHAPE), (dict(page=8), nat.PN_ERR_SHAPE),
    (dict(page=40), nat.PN_ERR_SHAPE), (dict(page=1 << 20), nat.PN_ERR_SHAPE), (dict(hk=0), nat.PN_ERR_SHAPE),
    (dict(n_pages=-1), nat.PN_ERR_SHAPE), (dict(ld=3), nat.PN_ERR_SHAPE), (dict(w=-1), nat.PN_ERR_SHAPE),
    (dict(w=1 << 25, ld=1 << 25), nat.PN_ERR_SHAPE), (dict(T=-2), nat.PN_ERR_SHAPE), (dict(T=3), nat.PN_ERR_SHAPE),
    (dict(B=-1), nat.PN_ERR_SHAPE), (dict(cache=None), nat.PN_ERR_ARG), (dict(table=None), nat.PN_ERR_ARG),
    (dict(lens=None), nat.PN_ERR_ARG), (dict(cache=P + 8), nat.PN_ERR_ALIGN), (dict(table=P + 2), nat.PN_ERR_ALIGN),
    (dict(lens=P + 1), nat.PN_ERR_ALIGN), (dict(cu=P + 2), nat.PN_ERR_ALIGN)])
def test_cache_refusals(call, kw, want):
    assert call(**kw) == want


@pytest.mark.parametrize("call", [rotary, prefix, sparse])
@pytest.mark.parametrize("kw,want", [
    (dict(q=None), nat.PN_ERR_ARG), (dict(out=None), nat.PN_ERR_ARG), (dict(q=P + 1), nat.PN_ERR_ALIGN),
    (dict(out=P + 8), nat.PN_ERR_ALIGN), (dict(dt=nat.PN_I8), nat.PN_ERR_DTYPE), (dict(heads=0), nat.PN_ERR_SHAPE),
    (dict(heads=1 << 20), nat.PN_ERR_SHAPE)])
def test_query_refusals(call, kw, want):
    assert call(**kw) == want


@pytest.mark.parametrize("call", [prefix, sparse])
def test_attention_refusals(call):
    for heads in (1, 3):
        assert call(heads=heads) == nat.PN_ERR_SHAPE
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=scale) == nat.PN_ERR_ARG


@pytest.mark.parametrize("kw,want", [
    (dict(k=None), nat.PN_ERR_ARG), (dict(v=None), nat.PN_ERR_ARG), (dict(cos=None), nat.PN_ERR_ARG),
    (dict(sin=None), nat.PN_ERR_ARG), (dict(k=P + 1), nat.PN_ERR_ALIGN), (dict(v=P + 1), nat.PN_ERR_ALIGN),
    (dict(cos=P + 2), nat.PN_ERR_ALIGN), (dict(sin=P + 1), nat.PN_ERR_ALIGN), (dict(offsets=P + 2), nat.PN_ERR_ALIGN),
    (dict(R=0), nat.PN_ERR_SHAPE), (dict(R=8), nat.PN_ERR_SHAPE), (dict(R=40), nat.PN_ERR_SHAPE), (dict(R=80), nat.PN_ERR_SHAPE),
    (dict(R=-16), nat.PN_ERR_SHAPE), (dict(n=-1), nat.PN_ERR_SHAPE), (dict(stride=31), nat.PN_ERR_SHAPE),
    (dict(T=1 << 30), nat.PN_ERR_SHAPE)])
def test_rotary_refusals(kw, want):
    assert rotary(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(ptable=None), nat.PN_ERR_ARG), (dict(plens=None), nat.PN_ERR_ARG), (dict(ptable=P + 2), nat.PN_ERR_ALIGN),
    (dict(plens=P + 2), nat.PN_ERR_ALIGN), (dict(cup=P + 1), nat.PN_ERR_ALIGN), (dict(pld=3), nat.PN_ERR_SHAPE),
    (dict(pw=-1), nat.PN_ERR_SHAPE), (dict(pw=1 << 25, pld=1 << 25), nat.PN_ERR_SHAPE), (dict(n=-1), nat.PN_ERR_SHAPE),
    (dict(n=3, cup=None), nat.PN_ERR_SHAPE)])
def test_prefix_refusals(kw, want):
    assert prefix(**kw) == want


@pytest.mark.parametrize("kw,want", [
    (dict(means=None), nat.PN_ERR_ARG), (dict(means=P + 8), nat.PN_ERR_ALIGN), (dict(chosen=P + 2), nat.PN_ERR_ALIGN),
    (dict(first=-1), nat.PN_ERR_SHAPE), (dict(last=0), nat.PN_ERR_SHAPE), (dict(top=-1), nat.PN_ERR_SHAPE),
    (dict(top=1 << 31), nat.PN_ERR_SHAPE), (dict(top=1 << 24), nat.PN_ERR_SHAPE),
    # (a row of one query head is a tile of its own: 2^20 rows x 8 heads x 401 units of 128 tokens)
    (dict(T=1 << 20, B=1, heads=8, hk=8, page=128, top=398, w=401, ld=401), nat.PN_ERR_SHAPE)])
def test_sparse_refusals(kw, want):
    assert sparse(**kw) == want


def test_means_refusals():
    assert page_means(means=None) == nat.PN_ERR_ARG
    assert page_means(means=P + 8) == nat.PN_ERR_ALIGN


def test_python_refusals():
    """CPU tensors, wrong types and shapes raise AssertionError."""
    q = torch.randn(2, 1, 4, 64)
    cache = pc.kv4_cache(2, 2, 64, 16, "cpu")
    table, lens = torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32)
    means = pc.kv4_means(cache, 64)
    assert means.shape == (2, 2, 64) and means.dtype == torch.bfloat16
    cos = torch.zeros(10, 32)
    with pytest.raises(AssertionError, match="CUDA"):
        pc.kv4_append_rotary(q, q[:, :, :2], q[:, :, :2], cos, cos, cache, table, lens)
    with pytest.raises(AssertionError, match="CUDA"):
        pc.kv4_prefix_attention(q, cache, table, lens, table[:1], lens[:1])
    with pytest.raises(AssertionError, match="CUDA"):
        pc.kv4_page_means(cache, means, table, lens, (2, 1))
    with pytest.raises(AssertionError, match="CUDA"):
        pc.kv4_sparse_attention(q, cache, means, table, lens, 1)
    with pytest.raises(AssertionError, match="head_dim"):
        pc.kv4_means(cache, 80)
    for bad in (means.float(), means[:1], means[:, :1], means[0], means.transpose(0, 1)):
        with pytest.raises(AssertionError, match="means"):
            pc._means_args(bad, cache, -1)
    pc._means_args(means, cache, -1)
    cu = torch.zeros(3, dtype=torch.int32)
    assert pc._count((2, 5), 2, None) == 10 and pc._count((6,), 2, None) == 6 and pc._count((5,), 2, cu) == 5
    assert pc._count((0,), 0, None) == 0
    for rows, B, c in (((3, 5), 2, None), ((2, 5), 2, cu), ((5,), 2, None), ((1, 2, 3), 1, None), ((1,), 0, None)):
        with pytest.raises(AssertionError):
            pc._count(rows, B, c)
    for bad in (torch.zeros(2, 1, 4, 64, dtype=torch.float16), torch.zeros(2, 1, 4, 32), torch.zeros(2, 1, 64, 4).transpose(2, 3)):
        with pytest.raises(AssertionError, match="out must"):
            pc._out(q, bad, None)
    assert pc._out(q, None, None).shape == q.shape and not pc._out(q, None, cu).any()
