"""PentaGPT inference model (pentagpt.py): the packed model's logits against
the same network computed densely with torch (dequantised weights, bf16
activations), on a small configuration."""
import math

import pytest
import torch
import torch.nn.functional as F

import penta_kernel as pk
import penta_native as nat
from pentagpt import PentaGPTConfig, PentaGPTFast

pytestmark = pytest.mark.gpu


def _dense(lin):
    w = pk.unpack_weights(lin.packed_w, lin.K_orig).float() * lin.scale
    return w.to(torch.bfloat16)


def _dense_forward(model, idx):
    cfg = model.cfg
    B, T = idx.shape
    x = (model.wte(idx) + model.wpe(torch.arange(T, device=idx.device))).to(torch.bfloat16)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        for blk in model.h:
            C = cfg.n_embd
            q, k, v = F.linear(blk.ln_1(x).to(torch.bfloat16), _dense(blk.c_attn)).split(C, dim=2)
            sh = lambda t: t.view(B, T, cfg.n_head, C // cfg.n_head).transpose(1, 2)
            att = (sh(q).float() @ sh(k).float().transpose(-2, -1)) / math.sqrt(C // cfg.n_head)
            att = att.masked_fill(torch.ones(T, T, device=idx.device).tril() == 0, float("-inf")).softmax(-1)
            y = (att @ sh(v).float()).to(torch.bfloat16).transpose(1, 2).contiguous().view(B, T, C)
            x = x + F.linear(y, _dense(blk.attn_proj))
            h = F.linear(F.gelu(F.linear(blk.ln_2(x).to(torch.bfloat16), _dense(blk.c_fc))), _dense(blk.mlp_proj))
            x = x + h
        x = model.ln_f(x)
    return F.linear(x.to(torch.bfloat16), _dense(model.lm_head)).float()


def test_small_pentagpt_matches_dense(cuda_device):
    cfg = PentaGPTConfig(n_layer=2, n_head=4, n_embd=128, block_size=64, vocab_size=1000)
    model = PentaGPTFast.random(cfg, seed=42, device=cuda_device)
    idx = torch.randint(0, cfg.vocab_size, (3, 40), generator=torch.Generator().manual_seed(1)).to(cuda_device)
    got = model(idx, all_logits=True).float()
    want = _dense_forward(model, idx)
    assert got.shape == (3, 40, cfg.vocab_size)
    # bf16 activations through the whole network: agreement to bf16 precision
    err = (got - want).abs().max().item()
    assert err <= 2e-2 * want.abs().max().item() + 1e-3, err
    last = model(idx).float()
    assert last.shape == (3, 1, cfg.vocab_size)
    assert torch.allclose(last[:, 0], got[:, -1], rtol=0, atol=0)


def test_pentagpt_124m_shapes(cuda_device):
    model = PentaGPTFast.random(seed=42, device=cuda_device)
    # 12 x (2304 + 768 + 3072) x 768 + 768 x 3072 x 12 packed projection weights, plus the tied lm_head
    assert model.n_packed_params() == 12 * (768 * 2304 + 768 * 768 + 2 * 768 * 3072) + 50257 * 768
    idx = torch.randint(0, 50257, (2, 128), generator=torch.Generator().manual_seed(2)).to(cuda_device)
    out = model(idx)
    assert out.shape == (2, 1, 50257) and torch.isfinite(out.float()).all()


def _ref_fixture(name):
    import os
    import numpy as np
    from _util import GOLDEN_DIR
    R = np.load(os.path.join(GOLDEN_DIR, "pentagpt_ref.npz"))
    return (torch.from_numpy(R[f"{name}.logits_f32"]), torch.from_numpy(R[f"{name}.logits_bf16_autocast"]),
            float(R[f"{name}.loss_f32"][0]), R[f"{name}.gammas"])


def _rel(a, b):
    return ((a.double() - b.double()).norm() / b.double().norm()).item()


@pytest.mark.parametrize("name", ["small2", "large"])
def test_reference_model_converted_in_place(cuda_device, name):
    """The reference's own PentaGPT module tree (tests/refmodel.py restates
    train_pentagpt.py:16-176; the fixtures hold the logits the reference's code
    produced from the same weights), converted in place by
    convert_to_fast_inference and run as the reference runs inference: under
    bf16 autocast, last-position logits, and the targets path's loss.

    Bar: our logits are at least as close to the reference's fp32 logits as
    the reference's own bf16-autocast logits are (within 2x, relative L2 and
    max-abs), and the loss agrees within 0.02 (the loss is ~11.4)."""
    import refmodel as rm
    from pentanet_layer import PentaLinearFast, convert_to_fast_inference
    ref32, refbf, ref_loss, gammas = _ref_fixture(name)
    cfg, seed, batch, seq = rm.CONFIGS[name]
    model = rm.PentaGPT(cfg).eval()
    model.load_state_dict(rm.weights(model, seed))
    idx, tgt = rm.tokens(cfg, batch, seq, seed)
    # the restated module, with the gammas the reference computed, reproduces the
    # reference's fp32 logits (pins the restatement; the remaining difference is
    # the fp32 summation order of this machine's CPU kernels)
    qls = rm.quant_layers(model)
    assert len(qls) == len(gammas)
    for m, g in zip(qls, gammas):
        m.fixed_gamma = float(g)
    with torch.no_grad():
        l32, _ = model(idx)
    assert (l32[:, 0] - ref32).abs().max().item() < 1e-3
    for m in qls:
        m.fixed_gamma = None
    model = convert_to_fast_inference(model.to(cuda_device))
    fast = [m for m in model.modules() if isinstance(m, PentaLinearFast)]
    assert len(fast) == 4 * cfg.n_layer + 1
    assert not any(type(m).__name__ == "QuantLinear" for m in model.modules())
    with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
        logits, none = model(idx.to(cuda_device))
        _, loss = model(idx.to(cuda_device), tgt.to(cuda_device))
    assert none is None and logits.shape == (batch, 1, cfg.vocab_size)
    got = logits[:, 0].float().cpu()
    assert _rel(got, ref32) <= 2 * _rel(refbf, ref32), (_rel(got, ref32), _rel(refbf, ref32))
    assert (got - ref32).abs().max() <= 2 * (refbf - ref32).abs().max()
    assert abs(loss.item() - ref_loss) <= 0.02, (loss.item(), ref_loss)


@pytest.mark.parametrize("name", ["small2", "large"])
def test_pentagpt_fast_matches_reference(cuda_device, name):
    """pentagpt.PentaGPTFast (LayerNorm kernel, SDPA attention, packed
    projections and tied lm_head) built from the same weights as the
    reference model of the fixtures: last-position logits against the
    reference's fp32 logits.  Bar: within 3x the reference's own bf16-autocast
    error (relative L2 and max-abs).  The factor is 3, not 2 as for the
    converted module, because PentaGPTFast keeps the residual stream in bf16
    (each residual add rounds to bf16, as its fused epilogues do) where
    autocast keeps it in fp32."""
    import refmodel as rm
    from pentagpt import PentaGPTConfig, PentaGPTFast
    ref32, refbf, _, _ = _ref_fixture(name)
    cfg, seed, batch, seq = rm.CONFIGS[name]
    tmp = rm.PentaGPT(cfg)
    w = rm.weights(tmp, seed)
    p = "transformer.h.{}."
    weights = {"wte": w["transformer.wte.weight"], "wpe": w["transformer.wpe.weight"],
               "h": [{"c_attn": w[p.format(i) + "attn.c_attn.weight"], "attn_proj": w[p.format(i) + "attn.c_proj.weight"],
                      "c_fc": w[p.format(i) + "mlp.c_fc.weight"], "mlp_proj": w[p.format(i) + "mlp.c_proj.weight"]}
                     for i in range(cfg.n_layer)]}
    weights = {k: (v.to(cuda_device) if torch.is_tensor(v) else [{a: b.to(cuda_device) for a, b in d.items()}
                                                                 for d in v]) for k, v in weights.items()}
    fcfg = PentaGPTConfig(n_layer=cfg.n_layer, n_head=cfg.n_head, n_embd=cfg.n_embd, block_size=cfg.block_size,
                          vocab_size=cfg.vocab_size)
    model = PentaGPTFast(fcfg, weights).to(cuda_device)
    with torch.no_grad():
        for i, blk in enumerate(model.h):
            blk.ln_1.weight.copy_(w[p.format(i) + "ln_1.weight"])
            blk.ln_2.weight.copy_(w[p.format(i) + "ln_2.weight"])
        model.ln_f.weight.copy_(w["transformer.ln_f.weight"])
    idx, _ = rm.tokens(cfg, batch, seq, seed)
    got = model(idx.to(cuda_device))[:, 0].float().cpu()
    assert _rel(got, ref32) <= 3 * _rel(refbf, ref32), (_rel(got, ref32), _rel(refbf, ref32))
    assert (got - ref32).abs().max() <= 3 * (refbf - ref32).abs().max()


def _cached_forward_f64(model, idx):
    """The network with keys and values rounded to their 4-bit form, attention in float64."""
    import kv4_oracle
    cfg = model.cfg
    B, T = idx.shape
    C, H = cfg.n_embd, cfg.n_head
    x = (model.wte(idx) + model.wpe(torch.arange(T, device=idx.device))).to(torch.bfloat16)
    for blk in model.h:
        h = pk.layer_norm(x, blk.ln_1.weight, blk.ln_1.bias, blk.ln_1.eps)
        q, k, v = (t.view(B, T, H, C // H) for t in blk.c_attn(h).split(C, dim=2))
        y = torch.stack([kv4_oracle.attention(q[b], k[b], v[b])[0] for b in range(B)])
        x = x + blk.attn_proj(y.to(torch.bfloat16).to(idx.device).view(B, T, C))
        h = pk.layer_norm(x, blk.ln_2.weight, blk.ln_2.bias, blk.ln_2.eps)
        x = x + blk.mlp_proj(F.gelu(blk.c_fc(h)))
    return model.lm_head(pk.layer_norm(x, model.ln_f.weight, model.ln_f.bias, model.ln_f.eps))


@pytest.mark.parametrize("act_quant", [None, "int8"])
def test_cached_forward(cuda_device, act_quant):
    """A prompt at once, in pieces, and token by token over the 4-bit cache, against
    the same network with attention from the definition."""
    cfg = PentaGPTConfig(n_layer=2, n_head=2, n_embd=128, block_size=160, vocab_size=700)
    model = PentaGPTFast.random(cfg, seed=3, device=cuda_device, act_quant=act_quant)
    idx = torch.randint(0, cfg.vocab_size, (3, 83), generator=torch.Generator().manual_seed(1)).to(cuda_device)
    want = _cached_forward_f64(model, idx).float()
    tol = 2e-2 * want.abs().max().item() + 1e-3  # as the dense comparison above: bf16 through the whole network
    for cuts in ([83], [40, 43], [70] + [1] * 13, [64, 3, 16]):
        cache = model.new_cache(3, page_size=32)
        got = torch.cat([model(p, all_logits=True, cache=cache) for p in idx.split(cuts, dim=1)], 1).float()
        assert cache.seq_lens.tolist() == [83] * 3 and cache.length == 83
        assert (got - want).abs().max().item() <= tol, cuts
    cache.reset()
    assert (model(idx, cache=cache).float()[:, 0] - want[:, -1]).abs().max().item() <= tol


def test_generate(cuda_device):
    cfg = PentaGPTConfig(n_layer=2, n_head=2, n_embd=128, block_size=96, vocab_size=700)
    model = PentaGPTFast.random(cfg, seed=3, device=cuda_device)
    idx = torch.randint(0, cfg.vocab_size, (4, 20), generator=torch.Generator().manual_seed(5)).to(cuda_device)
    kw = dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.01)
    rng = lambda: torch.Generator(device=cuda_device).manual_seed(9)
    out = model.generate(idx, 30, generator=rng(), **kw)
    assert out.shape == (4, 50) and torch.equal(out[:, :20], idx) and 0 <= out.min() and out.max() < cfg.vocab_size
    assert torch.equal(out, model.generate(idx, 30, generator=rng(), **kw))
    # the steps by hand
    cache, u, step = model.new_cache(4, 50), torch.rand(30, 4, device=cuda_device, generator=rng()), idx
    for i in range(30):
        step = pk.sample_tokens(model(step, cache=cache)[:, 0], u[i], **kw)[:, None]
        assert torch.equal(step, out[:, 20 + i:21 + i])
    # greedy: the largest logit; and going on with the cache of an earlier call
    greedy = model.generate(idx, 12, temperature=0.0)
    cache = model.new_cache(4)
    first = model.generate(idx, 5, temperature=0.0, cache=cache)
    assert torch.equal(model.generate(first[:, -1:], 7, temperature=0.0, cache=cache)[:, 1:], greedy[:, 25:])
    assert model.generate(idx, 0).shape == (4, 20)
    with pytest.raises(AssertionError, match="do not fit"):
        model.generate(idx, 78)
    assert model.generate(idx, 77).shape == (4, 97)  # the last token is never fed back


def test_captured_decode_step(cuda_device):
    """One decode step (append, attention, products, sampling) captured once and
    replayed: the lengths on the GPU carry it on."""
    cfg = PentaGPTConfig(n_layer=2, n_head=2, n_embd=128, block_size=96, vocab_size=700)
    model = PentaGPTFast.random(cfg, seed=3, device=cuda_device)
    idx = torch.randint(0, cfg.vocab_size, (2, 15), generator=torch.Generator().manual_seed(5)).to(cuda_device)
    want = model.generate(idx, 20, temperature=0.0)
    cache = model.new_cache(2)
    tok, u = model.generate(idx, 2, temperature=0.0, cache=cache)[:, -1:].clone(), torch.zeros(2, device=cuda_device)
    got = [tok.clone()]
    keep = cache.seq_lens.clone()

    def step():
        tok.copy_(pk.sample_tokens(model(tok, cache=cache)[:, 0], u, temperature=0.0)[:, None])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    cache.seq_lens.copy_(keep)
    tok.copy_(got[0])
    for _ in range(18):
        graph.replay()
        got.append(tok.clone())
    assert torch.equal(torch.cat(got, 1), want[:, 16:])


def _small(device):
    cfg = PentaGPTConfig(n_layer=2, n_head=2, n_embd=128, block_size=96, vocab_size=700)
    return PentaGPTFast.random(cfg, seed=3, device=device)


def test_cache_after_replays(cuda_device):
    """Replays advance the lengths on the GPU alone; eager calls after them go on from
    there, and know when the cache is full."""
    model = _small(cuda_device)
    idx = torch.randint(0, 700, (2, 15), generator=torch.Generator().manual_seed(5)).to(cuda_device)
    want = model.generate(idx, 12, temperature=0.0)
    cache = model.new_cache(2, 24)
    tok, u = model.generate(idx, 1, temperature=0.0, cache=cache)[:, -1:].clone(), torch.zeros(2, device=cuda_device)
    first = tok.clone()

    def step():
        tok.copy_(pk.sample_tokens(model(tok, cache=cache)[:, 0], u, temperature=0.0)[:, None])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    assert cache.length == 16
    cache.rewind(15)
    assert cache.length == 15 and cache.seq_lens.tolist() == [15, 15]
    tok.copy_(first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    assert cache.length == 15  # nothing was stored
    got = [first]
    for _ in range(5):
        graph.replay()
        got.append(tok.clone())
    for i in range(4):  # eager
        step()
        got.append(tok.clone())
        assert cache.length == 21 + i and cache.seq_lens.tolist() == [21 + i] * 2
    assert torch.equal(torch.cat(got, 1), want[:, 15:25])
    with pytest.raises(AssertionError, match="do not fit"):
        model.generate(tok, 2, cache=cache)
    assert cache.length == 24
    with pytest.raises(AssertionError, match="full"):
        model(tok, cache=cache)
    assert cache.seq_lens.tolist() == [24, 24] and nat.device_status() == 0


def test_cache_of_another_batch(cuda_device):
    model = _small(cuda_device)
    idx = torch.randint(0, 700, (4, 5), generator=torch.Generator().manual_seed(5)).to(cuda_device)
    for batch, n in ((1, 4), (4, 1), (3, 2)):
        cache = model.new_cache(batch)
        for call in (lambda: model(idx[:n], cache=cache), lambda: model.generate(idx[:n], 3, cache=cache)):
            with pytest.raises(AssertionError, match="the cache holds"):
                call()
        assert cache.length == 0 and not cache.seq_lens.any()


def test_cache_after_a_block_that_raises(cuda_device, monkeypatch):
    """Tokens without keys are not counted."""
    model = _small(cuda_device)
    idx = torch.randint(0, 700, (2, 15), generator=torch.Generator().manual_seed(5)).to(cuda_device)
    cache = model.new_cache(2)
    want = model(idx, cache=cache), model(idx[:, :3], cache=cache)
    cache.reset()
    assert torch.equal(model(idx, cache=cache), want[0])

    def broken(*args):
        raise RuntimeError("out of something")

    with monkeypatch.context() as m:
        m.setattr(model.h[1], "forward", broken)
        with pytest.raises(RuntimeError, match="something"):
            model(idx[:, 3:9], cache=cache)
    assert cache.length == 15 and cache.seq_lens.tolist() == [15, 15]
    assert torch.equal(model(idx[:, :3], cache=cache), want[1])


def test_what_the_cache_costs(cuda_device):
    """Logits over the 4-bit cache against those of forward(idx), whose attention is bf16.

    Attention outputs move by 13 % in norm for keys and values without loud dims (see
    test_kv4_gpu.test_what_four_bits_cost), and with them what attention adds to the logits:
    bounded here by a fifth of the difference that leaving it out makes, plus 2^-7 of the
    logits for the bf16 roundings that differ (some ten per layer, 2^-9 each, as a root of
    their sum of squares)."""
    model = _small(cuda_device)
    idx = torch.randint(0, 700, (3, 83), generator=torch.Generator().manual_seed(1)).to(cuda_device)
    dense = model(idx, all_logits=True).double()
    cached = model(idx, all_logits=True, cache=model.new_cache(3)).double()
    hooks = [b.attn_proj.register_forward_hook(lambda m, args, y: torch.zeros_like(y)) for b in model.h]
    without = model(idx, all_logits=True).double()
    for h in hooks:
        h.remove()
    off, share = (cached - dense).norm() / dense.norm(), (without - dense).norm() / dense.norm()
    print(f"\nlogits over the 4-bit cache: {off:.4f} of their norm from forward(idx); attention adds {share:.4f}")
    assert off <= 0.2 * share + 2.0 ** -7
