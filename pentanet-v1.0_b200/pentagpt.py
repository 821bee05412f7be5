"""PentaGPT inference model on the packed sm_100a layers.

A GPT-2-style decoder with the architecture of the reference's PentaGPT
(train_pentagpt.py:46-136; GPTConfig size 'large': 12 layers, 12 heads,
d_model 768, MLP 3072, no biases, weight-tied lm_head) in which every
projection -- c_attn, attention c_proj, c_fc, MLP c_proj and the lm_head -- is
a PentaLinearFast (3-bit packed weights, fused dequant-matmul).  For
decode-sized batches the MLP's GELU and both residual adds run in the
epilogues of the projections that produce their inputs (c_fc, attention
c_proj, MLP c_proj), rounded as the separate bf16 ops round them; at prefill
sizes they stay separate torch ops, which are cheaper there (the product's
epilogue runs on the warps of its main loop: for c_fc at 32768 tokens a fused
GELU added ~180 us against ~110 us for F.gelu).  Each LayerNorm is one pass from bf16 to bf16
with fp32 statistics (penta_kernel.layer_norm: what nn.LayerNorm under bf16
autocast plus the cast in front of the projection compute, without the fp32
round trip).  Causal attention is torch's scaled_dot_product_attention, the
memory-efficient equivalent of the reference's masked softmax.

`PentaGPTFast.random(seed)` builds the model from random weights, as used for
throughput measurement; a trained reference model converts with
`pentanet_layer.convert_to_fast_inference`, which packs the same layers.
Forward without targets returns the logits of the last position only, as the
reference does (train_pentagpt.py:129-134).

`generate` continues prompts token by token.  Keys and values of past tokens are
kept in 4 bits (penta_cache), so a step computes the new tokens only:
`forward(idx, cache=...)` appends a chunk's keys and values and attends over the
cache, for prompts, for prompts in pieces and for single tokens alike; each
token is drawn by penta_kernel.sample_tokens.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch
import torch.nn as nn
import torch.nn.functional as F

try:
    from .pentanet_layer import PentaLinearFast
    from . import penta_cache as pc
    from . import penta_kernel as pk
except ImportError:
    from pentanet_layer import PentaLinearFast
    import penta_cache as pc
    import penta_kernel as pk


@dataclass
class PentaGPTConfig:
    n_layer: int = 12
    n_head: int = 12
    n_embd: int = 768
    block_size: int = 1024
    vocab_size: int = 50257


def _packed(w: torch.Tensor, act_quant: str | None) -> PentaLinearFast:
    packed, K, scale = pk.quantize_and_pack(w)
    return PentaLinearFast(packed, scale, K, None, act_quant=act_quant)


# Largest token count whose GELU and residual adds are fused into the products.
FUSE_MAX_TOKENS = 64


class _Block(nn.Module):
    def __init__(self, cfg: PentaGPTConfig, weights: dict, act_quant: str | None):
        super().__init__()
        self.n_head = cfg.n_head
        self.ln_1 = nn.LayerNorm(cfg.n_embd, bias=False)
        self.ln_2 = nn.LayerNorm(cfg.n_embd, bias=False)
        self.c_attn = _packed(weights["c_attn"], act_quant)
        self.attn_proj = _packed(weights["attn_proj"], act_quant)
        self.c_fc = _packed(weights["c_fc"], act_quant)
        self.mlp_proj = _packed(weights["mlp_proj"], act_quant)

    def forward(self, x: torch.Tensor, layer: torch.Tensor | None = None, cache: "PentaGPTCache | None" = None
                ) -> torch.Tensor:
        B, T, C = x.shape
        h = pk.layer_norm(x, self.ln_1.weight, self.ln_1.bias, self.ln_1.eps)
        q, k, v = self.c_attn(h).split(C, dim=2)
        q = q.view(B, T, self.n_head, C // self.n_head)
        k = k.view(B, T, self.n_head, C // self.n_head)
        v = v.view(B, T, self.n_head, C // self.n_head)
        if cache is None:
            y = F.scaled_dot_product_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), is_causal=True)
            y = y.transpose(1, 2).contiguous().view(B, T, C)
        else:
            pc.kv4_append(k, v, layer, cache.block_table, cache.seq_lens)
            y = pc.kv4_attention(q, layer, cache.block_table, cache.seq_lens).view(B, T, C)
        if B * T <= FUSE_MAX_TOKENS:
            x = self.attn_proj(y, residual=x)  # x + attn(ln_1(x)), train_pentagpt.py:100
            h = pk.layer_norm(x, self.ln_2.weight, self.ln_2.bias, self.ln_2.eps)
            return self.mlp_proj(self.c_fc(h, act="gelu"), residual=x)  # x + mlp(ln_2(x)), :101
        x = x + self.attn_proj(y)
        h = pk.layer_norm(x, self.ln_2.weight, self.ln_2.bias, self.ln_2.eps)
        return x + self.mlp_proj(F.gelu(self.c_fc(h)))


class PentaGPTCache:
    """The past tokens of a batch: a 4-bit cache per layer (penta_cache), their
    pages and the sequences' lengths.  The pages are handed out up front;
    seq_lens lives on the GPU, so a captured step goes on where it stands.

    A capture stores nothing, and replays advance seq_lens alone; so once a step
    was captured over the cache, eager calls read the length from there (a
    synchronisation each).  A replay past the capacity stores no more tokens and
    shows in penta_native.device_status()."""

    def __init__(self, cfg: PentaGPTConfig, batch: int, device, max_tokens: int | None = None, page_size: int = 64):
        self.capacity = cfg.block_size if max_tokens is None else max_tokens
        pages = -(-self.capacity // page_size)
        self.layers = [pc.kv4_cache(batch * pages, cfg.n_head, cfg.n_embd // cfg.n_head, page_size, device)
                       for _ in range(cfg.n_layer)]
        self.block_table = torch.arange(batch * pages, dtype=torch.int32, device=device).view(batch, pages)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.length = 0  # what the host knows: tokens appended so far (of the longest sequence)
        self.captured = False  # replays may have advanced seq_lens since

    def known_length(self) -> int:
        """length, brought up to what replays of captured steps left on the GPU (not
        while a step is being captured)."""
        if self.captured and self.seq_lens.numel() and not torch.cuda.is_current_stream_capturing():
            self.length = int(self.seq_lens.max())
        return self.length

    def rewind(self, length: int) -> None:
        """Forget the tokens behind the first `length` of each sequence (their pages
        are written over)."""
        assert length >= 0
        self.length = min(self.known_length(), length)
        self.seq_lens.clamp_(max=length)

    def reset(self) -> None:
        """Forget all tokens."""
        self.seq_lens.zero_()
        self.length = 0


class PentaGPTFast(nn.Module):
    """PentaGPT for inference with packed projections (bf16 activations, or the
    per-token int8 path with act_quant='int8')."""

    def __init__(self, cfg: PentaGPTConfig, weights: dict, act_quant: str | None = None):
        super().__init__()
        self.cfg = cfg
        self.wte = nn.Embedding(cfg.vocab_size, cfg.n_embd)
        self.wpe = nn.Embedding(cfg.block_size, cfg.n_embd)
        with torch.no_grad():
            self.wte.weight.copy_(weights["wte"])
            self.wpe.weight.copy_(weights["wpe"])
        self.h = nn.ModuleList([_Block(cfg, weights["h"][i], act_quant) for i in range(cfg.n_layer)])
        self.ln_f = nn.LayerNorm(cfg.n_embd, bias=False)
        # weight tying: the lm_head packs the token-embedding matrix
        self.lm_head = _packed(weights["wte"], act_quant)

    @classmethod
    def random(cls, cfg: PentaGPTConfig | None = None, seed: int = 42, device="cuda",
               act_quant: str | None = None) -> "PentaGPTFast":
        """Random N(0, 0.02) weights from `seed` (a throughput model)."""
        cfg = cfg or PentaGPTConfig()
        g = torch.Generator(device=device).manual_seed(seed)
        d = cfg.n_embd

        def rnd(*shape):
            return torch.randn(*shape, device=device, generator=g) * 0.02

        weights = {"wte": rnd(cfg.vocab_size, d), "wpe": rnd(cfg.block_size, d), "h": []}
        for _ in range(cfg.n_layer):
            weights["h"].append({"c_attn": rnd(3 * d, d), "attn_proj": rnd(d, d) / math.sqrt(2 * cfg.n_layer),
                                 "c_fc": rnd(4 * d, d), "mlp_proj": rnd(d, 4 * d) / math.sqrt(2 * cfg.n_layer)})
        model = cls(cfg, weights, act_quant).to(device)
        return model

    def n_packed_params(self) -> int:
        return sum(m.packed_w.shape[0] * m.K_orig for m in self.modules() if isinstance(m, PentaLinearFast))

    def new_cache(self, batch: int, max_tokens: int | None = None, page_size: int = 64) -> PentaGPTCache:
        """An empty cache for `batch` sequences of up to max_tokens (block_size)."""
        return PentaGPTCache(self.cfg, batch, self.wte.weight.device, max_tokens, page_size)

    @torch.no_grad()
    def forward(self, idx: torch.Tensor, all_logits: bool = False, cache: PentaGPTCache | None = None) -> torch.Tensor:
        """Logits of the last position (all with all_logits).  With a cache, idx
        holds the tokens that follow those in it; their keys and values are added
        and attention runs over the cache.  Where that raises, none were added."""
        B, T = idx.shape
        if cache is None:
            assert T <= self.cfg.block_size
            return self._logits(idx, torch.arange(T, device=idx.device), all_logits)
        assert B == cache.seq_lens.shape[0], f"{B} sequences, the cache holds {cache.seq_lens.shape[0]}"
        assert cache.known_length() + T <= min(cache.capacity, self.cfg.block_size), "the cache is full"
        capturing = torch.cuda.is_current_stream_capturing()
        # (a captured step replayed past the block stays at its last position)
        pos = (cache.seq_lens[:, None] + torch.arange(T, device=idx.device)).clamp(max=self.cfg.block_size - 1)
        cache.seq_lens += T
        try:
            logits = self._logits(idx, pos, all_logits, cache)
        except BaseException:
            if not capturing:
                cache.seq_lens -= T
            raise
        if capturing:
            cache.captured = True
        else:
            cache.length += T
        return logits

    def _logits(self, idx: torch.Tensor, pos: torch.Tensor, all_logits: bool, cache: PentaGPTCache | None = None
                ) -> torch.Tensor:
        x = (self.wte(idx) + self.wpe(pos)).to(torch.bfloat16)
        for i, block in enumerate(self.h):
            x = block(x) if cache is None else block(x, cache.layers[i], cache)
        if not all_logits:
            x = x[:, -1:, :]  # LayerNorm is per position: normalise only what the lm_head reads
        x = pk.layer_norm(x, self.ln_f.weight, self.ln_f.bias, self.ln_f.eps)
        return self.lm_head(x)

    @torch.no_grad()
    def generate(self, idx: torch.Tensor, max_new_tokens: int, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                 generator: torch.Generator | None = None, cache: PentaGPTCache | None = None) -> torch.Tensor:
        """idx (B, T) with max_new_tokens sampled tokens behind it: (B, T +
        max_new_tokens).  The settings are those of penta_kernel.sample_tokens
        (temperature=0: the most likely token), its uniform numbers come from
        `generator`.  With a cache from an earlier call, idx holds what follows
        the tokens in it (the last token returned is not in it yet).

        Past keys and values are held in 4 bits, which costs accuracy (attention
        outputs move by 13 % in norm and more; penta_cache says what that depends
        on): forward(idx) over the whole prefix is the way to bf16 attention.  Heads of
        64 or 128 dims."""
        B, T = idx.shape
        assert T >= 1 and max_new_tokens >= 0
        cache = cache if cache is not None else self.new_cache(B, min(T + max_new_tokens, self.cfg.block_size))
        held = cache.known_length()
        assert held + T + max(max_new_tokens - 1, 0) <= min(cache.capacity, self.cfg.block_size), \
            f"{held} + {T} + {max_new_tokens} tokens do not fit the model's block or the cache"
        out = [idx]
        u = torch.rand(max_new_tokens, B, device=idx.device, generator=generator)
        captured, cache.captured = cache.captured, False  # (nothing is replayed in between: one look at seq_lens will do)
        try:
            for i in range(max_new_tokens):
                logits = self(out[-1].clamp(min=0), cache=cache)  # -1: a row of NaN logits has no token
                out.append(pk.sample_tokens(logits[:, 0], u[i], temperature, top_k, top_p, min_p)[:, None])
        finally:
            cache.captured |= captured
        return torch.cat(out, dim=1)
