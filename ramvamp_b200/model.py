"""Whole-model Qwen3-30B-A3B decode on the GPU: the per-token step of
model/forward.rs:2548-2780 (embedding, 48 x (attention half + MoE block),
final norm, lm_head) and the greedy loop of generate/mod.rs (argmax, first
index wins ties), plus the KL / top-1 comparison the reference's
scripts/kl_vs_reference.py applies to two logit streams.

The step runs entirely on the device: the input token id, the position and
the sampled id live in device memory, so one CUDA graph captured once serves
every step (``Decoder.capture``), with no host work between tokens while
generating.  Every kernel on the step is this package's own; weights are
synthetic (seeded values through the reference's quantizers) or come from an
install.
"""
from __future__ import annotations

import math
from dataclasses import dataclass, field
from functools import wraps
from typing import List, Optional, Sequence

import numpy as np
import torch

from . import (AttnEngine, ExpertTable, KV_F16, KV_Q8, KvCache, MoeEngine, QuantFormat, QWEN3_Q6K_DOWN_LAYERS, _check,
               _p, _stream, attn_weights, dequantize_rows, gemv_q8_0_batched, gemv_q8_k, gemv_q8_k_batched, kv_append,
               kv_read, lib, prefix_attention, prefix_attention_scratch, qwen3_layer_layout, quantize_row_q8_0,
               quantize_row_q8_k, quantize_weights, rmsnorm, rmsnorm_quantize, rope_neox_heads, sample, synth_normal)

Q = QuantFormat


@dataclass
class ModelConfig:
    """model/shapes.rs:14-35 and the manifest's arch block; defaults are
    Qwen3-30B-A3B."""

    n_layers: int = 48
    hidden: int = 2048
    n_heads: int = 32
    n_kv_heads: int = 4
    head_dim: int = 128
    moe: int = 768
    n_experts: int = 128
    top_k: int = 8
    vocab: int = 151936
    rope_theta: float = 1e6
    eps: float = 1e-6
    norm_topk_prob: bool = True

    @property
    def q_dim(self):
        return self.n_heads * self.head_dim

    @property
    def kv_dim(self):
        return self.n_kv_heads * self.head_dim

    def q6k_layer(self, layer: int) -> bool:
        """attn_v and ffn_down are Q6_K on the pinned layer set of the
        48-layer model (model/shapes.rs:30-35), Q4_K elsewhere."""
        return layer in QWEN3_Q6K_DOWN_LAYERS if self.n_layers == 48 else layer % 2 == 0


@dataclass
class LayerWeights:
    attn_norm: torch.Tensor
    attn_q: torch.Tensor       # Q4_K [q_dim][hidden]
    attn_k: torch.Tensor       # Q8_0 [kv_dim][hidden]
    attn_v: torch.Tensor       # Q6_K or Q4_K [kv_dim][hidden]
    attn_v_format: int
    attn_output: torch.Tensor  # Q5_K [hidden][q_dim]
    attn_q_norm: torch.Tensor
    attn_k_norm: torch.Tensor
    ffn_norm: torch.Tensor
    router: torch.Tensor       # f32 [n_experts][hidden]


def _q8_0_weights(x: torch.Tensor) -> torch.Tensor:
    """Packed Q8_0 weight rows (34 B / 32 weights): the activation quantizer
    with d stored as f16, which is test_support.rs:221-234's recipe."""
    blocks = quantize_row_q8_0(x).view(-1, 36)
    d16 = blocks[:, :4].contiguous().view(torch.float32).half().view(torch.uint8)
    return torch.cat([d16, blocks[:, 4:]], dim=1).contiguous().view(-1)


@dataclass
class Qwen3Weights:
    cfg: ModelConfig
    token_embd: torch.Tensor   # Q4_K [vocab][hidden]
    output_norm: torch.Tensor
    lm_head: torch.Tensor      # Q6_K [vocab][hidden]
    layers: List[LayerWeights]
    experts: ExpertTable

    @classmethod
    def synthetic(cls, cfg: ModelConfig, seed: int = 1, device: int = 0, expert_sigma: float = 0.02):
        """Seeded random-init weights (config 1): every matrix N(0, 0.02)
        through the reference's quantizers (embedding N(0, 1)), norms
        1 + N(0, 0.05), router N(0, 0.02) f32."""
        dev = f"cuda:{device}"
        offset = [0]

        def normal(n, sigma):
            x = synth_normal(seed, offset[0], sigma, n, device=dev)
            offset[0] += n
            return x

        def norm_w(n):
            return 1.0 + normal(n, 0.05)

        H = cfg.hidden
        layers = []
        for l in range(cfg.n_layers):
            v_fmt = Q.Q6_K if cfg.q6k_layer(l) else Q.Q4_K
            layers.append(LayerWeights(
                attn_norm=norm_w(H),
                attn_q=quantize_weights(Q.Q4_K, normal(cfg.q_dim * H, 0.02)),
                attn_k=_q8_0_weights(normal(cfg.kv_dim * H, 0.02)),
                attn_v=quantize_weights(v_fmt, normal(cfg.kv_dim * H, 0.02)),
                attn_v_format=int(v_fmt),
                attn_output=quantize_weights(Q.Q5_K, normal(H * cfg.q_dim, 0.02)),
                attn_q_norm=norm_w(cfg.head_dim),
                attn_k_norm=norm_w(cfg.head_dim),
                ffn_norm=norm_w(H),
                router=normal(cfg.n_experts * H, 0.02),
            ))
        layouts = [qwen3_layer_layout(l, hidden=H, moe=cfg.moe, n_experts=cfg.n_experts,
                                      down_format=Q.Q6_K if cfg.q6k_layer(l) else Q.Q4_K)
                   for l in range(cfg.n_layers)]
        table = ExpertTable(layouts, device=device)
        for l in range(cfg.n_layers):
            table.fill_synthetic(l, seed * 1000 + l, expert_sigma)
        token_embd = quantize_weights(Q.Q4_K, normal(cfg.vocab * H, 1.0))
        output_norm = norm_w(H)
        lm_head = quantize_weights(Q.Q6_K, normal(cfg.vocab * H, 0.02))
        torch.cuda.synchronize(device)
        return cls(cfg, token_embd, output_norm, lm_head, layers, table)


class Decoder:
    """Batch-1 decoding over Qwen3Weights.  ``step`` runs one token of
    forward_token_traced (model/forward.rs:2548-2780) plus the greedy
    argmax; all state (token, position, caches) is on the device."""

    def __init__(self, weights: Qwen3Weights, max_positions: int = 1024, device: int = 0):
        cfg = weights.cfg
        self.w, self.cfg, self.device = weights, cfg, device
        self.max_positions = max_positions
        self.attn = AttnEngine(cfg.n_layers, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, max_positions,
                               cfg.rope_theta, cfg.eps, device, hidden=cfg.hidden)
        self.attn_w = [attn_weights(l.attn_norm, l.attn_q, l.attn_k, l.attn_v, l.attn_output, l.attn_q_norm,
                                    l.attn_k_norm, Q.Q4_K, l.attn_v_format, Q.Q5_K) for l in weights.layers]
        self.moe = MoeEngine(cfg.hidden, cfg.moe, cfg.n_experts, cfg.top_k, cfg.norm_topk_prob, cfg.eps,
                             max_tokens=1, device=device)
        d = f"cuda:{device}"
        f32 = lambda n: torch.zeros(n, dtype=torch.float32, device=d)
        H = cfg.hidden
        self.residual = f32(H)
        self.acts_k = torch.zeros(H // 256 * 292, dtype=torch.uint8, device=d)
        self.logits = f32(cfg.vocab)
        self.token = torch.zeros(1, dtype=torch.int32, device=d)
        self.next_token = torch.zeros(1, dtype=torch.int32, device=d)
        self.position = torch.zeros(1, dtype=torch.int32, device=d)
        self.ids = torch.zeros(max_positions, dtype=torch.int32, device=d)
        self.graph: Optional[torch.cuda.CUDAGraph] = None

    def reset(self):
        """KvCache::clear and position 0."""
        self.attn.clear()
        self.position.zero_()
        self.ids.zero_()

    def _launch_step(self):
        cfg, w, s = self.cfg, self.w, _stream()
        H = cfg.hidden
        dequantize_rows(Q.Q4_K, w.token_embd, H, cfg.vocab, rows=self.token, out=self.residual)
        for l, lw in enumerate(w.layers):
            # attention half (forward.rs:2572-2652), residual in place
            self.attn.block(l, self.attn_w[l], self.residual, position_dev=self.position)
            # MoE block (forward.rs:2654-2754), residual in place
            self.moe.forward(w.experts, l, lw.ffn_norm, lw.router, self.residual)
        rmsnorm_quantize(self.residual, w.output_norm, cfg.eps, self.acts_k)
        gemv_q8_k(Q.Q6_K, w.lm_head, H, cfg.vocab, self.acts_k, self.logits)
        _check(lib().rv_argmax(_p(self.logits), cfg.vocab, _p(self.next_token), s))
        _check(lib().rv_decode_advance(_p(self.position), _p(self.next_token), _p(self.token), _p(self.ids),
                                       self.ids.numel(), s))

    def capture(self):
        """Capture one step as a CUDA graph (replayed by ``step``)."""
        torch.cuda.synchronize(self.device)
        side = torch.cuda.Stream(self.device)
        saved = (self.token.clone(), self.position.clone(), self.ids.clone())
        with torch.cuda.stream(side):
            self._launch_step()  # warm-up outside capture (lazy set-up)
        torch.cuda.synchronize(self.device)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            self._launch_step()
        torch.cuda.synchronize(self.device)
        self.token.copy_(saved[0])
        self.position.copy_(saved[1])
        self.ids.copy_(saved[2])
        self.attn.clear()
        self.graph = g
        return g

    def step(self):
        """One token: reads self.token / self.position, writes self.logits,
        self.next_token (= self.token for the next step), self.ids[pos]."""
        if self.graph is not None:
            self.graph.replay()
        else:
            self._launch_step()

    def generate(self, prompt: Sequence[int], n_new: int, on_logits=None) -> List[int]:
        """Greedy continuation of `prompt` by n_new tokens (generate/mod.rs:
        the prompt is fed one token per step, then each argmax becomes the
        next input).  on_logits(step_index, logits) sees every step's logits
        (prompt steps included)."""
        if len(prompt) + n_new > self.max_positions:
            raise ValueError("prompt + new tokens exceed max_positions")
        self.reset()
        prompt_t = torch.tensor(list(prompt), dtype=torch.int32, device=self.token.device)
        self.token.copy_(prompt_t[:1])
        for i in range(len(prompt) + n_new - 1):
            self.step()
            if on_logits is not None:
                on_logits(i, self.logits)
            if i + 1 < len(prompt):
                self.token.copy_(prompt_t[i + 1:i + 2])
        torch.cuda.synchronize(self.device)
        ids = self.ids[:len(prompt) + n_new - 1].cpu().numpy()
        return [int(x) for x in ids[len(prompt) - 1:]]


def _on_its_device(method):
    """The method with its object's device current, where its kernels run."""

    @wraps(method)
    def run(self, *args, **kwargs):
        with torch.cuda.device(self.device):
            return method(self, *args, **kwargs)

    return run


class ParallelDecoder:
    """n continuations of one prompt, drawn together.  The prompt goes through
    ``Decoder`` once; its keys and values -- the engine's own f16 caches, or
    8-bit copies of them (``kv_format``) -- are the prefix that every
    continuation attends to, each beside its own rows, and a token of each is
    drawn per step.  No counterpart in the reference, whose generate/mod.rs
    draws one sequence."""

    def __init__(self, weights: Qwen3Weights, n: int, max_prompt: int = 1024, max_new: int = 1024,
                 kv_format: int = KV_Q8, device: int = 0):
        cfg = weights.cfg
        self.w, self.cfg, self.n, self.device, self.kv_format = weights, cfg, n, device, kv_format
        self.max_prompt, self.max_new = max_prompt, max_new
        self.prompt = Decoder(weights, max_prompt, device)
        self.prompt_len = self.new = 0
        d = f"cuda:{device}"
        caches = lambda n, rows: [KvCache(n, rows, cfg.n_kv_heads, cfg.head_dim, kv_format, device)  # noqa: E731
                                  for _ in range(cfg.n_layers)]
        self.suffix = caches(n, max_new)
        self.prefix = caches(1, max_prompt) if kv_format != KV_F16 else \
            [KvCache.of_engine(self.prompt.attn, l) for l in range(cfg.n_layers)]
        self.moe = MoeEngine(cfg.hidden, cfg.moe, cfg.n_experts, cfg.top_k, cfg.norm_topk_prob, cfg.eps,
                             max_tokens=n, device=device)
        f32 = lambda *shape: torch.zeros(shape, dtype=torch.float32, device=d)  # noqa: E731
        self.residual, self.normed = f32(n, cfg.hidden), f32(n, cfg.hidden)
        self.logits = f32(n, cfg.vocab)
        self.lens = torch.zeros(n, dtype=torch.int32, device=d)
        self.scratch = torch.empty(prefix_attention_scratch(n, 1, cfg.n_heads, cfg.n_kv_heads, cfg.head_dim),
                                   dtype=torch.uint8, device=d)

    @_on_its_device
    def prefill(self, prompt: Sequence[int]) -> torch.Tensor:
        """The prompt's rows into the prefix; the logits of its last token."""
        if not 0 < len(prompt) <= self.max_prompt:
            raise ValueError("the prompt must hold 1 to max_prompt tokens")
        dec = self.prompt
        dec.reset()
        ids = torch.tensor(list(prompt), dtype=torch.int32, device=dec.token.device)
        for i in range(len(prompt)):
            dec.token.copy_(ids[i:i + 1])
            dec.step()
        if self.kv_format != KV_F16:
            for l, cache in enumerate(self.prefix):
                k, v = kv_read(KvCache.of_engine(dec.attn, l), len(prompt))
                kv_append(cache, k, v)
        self.prompt_len, self.new = len(prompt), 0
        self.lens.zero_()
        return dec.logits

    def _rows(self, gemv, *args) -> torch.Tensor:
        """A batched GEMV's [out_dim][n] result as rows [n, out_dim]."""
        *head, in_dim, out_dim, acts = args
        out = torch.empty(out_dim, self.n, dtype=torch.float32, device=self.residual.device)
        gemv(*head, in_dim, out_dim, acts, self.n, range(out_dim), out)
        return out.t().contiguous()

    @_on_its_device
    def step(self, tokens: torch.Tensor) -> torch.Tensor:
        """One token of every continuation (int32 [n], on the device) through
        the model (model/forward.rs:2548-2780 for each row): logits [n, vocab]."""
        cfg, w, n = self.cfg, self.w, self.n
        H, hd, position = cfg.hidden, cfg.head_dim, self.prompt_len + self.new
        if self.prompt_len == 0 or self.new >= self.max_new:
            raise ValueError("no prompt yet, or max_new tokens drawn")
        self.new += 1
        self.lens.add_(1)
        dequantize_rows(Q.Q4_K, w.token_embd, H, cfg.vocab, rows=tokens, out=self.residual)
        for l, lw in enumerate(w.layers):
            rmsnorm(self.residual, lw.attn_norm, cfg.eps, self.normed)
            a = quantize_row_q8_k(self.normed)
            q = self._rows(gemv_q8_k_batched, Q.Q4_K, lw.attn_q, H, cfg.q_dim, a).view(n, 1, cfg.n_heads, hd)
            k = self._rows(gemv_q8_0_batched, lw.attn_k, H, cfg.kv_dim, quantize_row_q8_0(self.normed))
            k = k.view(n, 1, cfg.n_kv_heads, hd)
            v = self._rows(gemv_q8_k_batched, lw.attn_v_format, lw.attn_v, H, cfg.kv_dim, a).view_as(k)
            rmsnorm(q, lw.attn_q_norm, cfg.eps, q)
            rmsnorm(k, lw.attn_k_norm, cfg.eps, k)
            rope_neox_heads(q, n * cfg.n_heads, hd, position, cfg.rope_theta)
            rope_neox_heads(k, n * cfg.n_kv_heads, hd, position, cfg.rope_theta)
            kv_append(self.suffix[l], k, v, lens=self.lens)
            o = prefix_attention(q, self.prefix[l], self.prompt_len, self.suffix[l], self.lens, scratch=self.scratch)
            self.residual.add_(self._rows(gemv_q8_k_batched, Q.Q5_K, lw.attn_output, cfg.q_dim, H,
                                          quantize_row_q8_k(o)))
            self.moe.forward(w.experts, l, lw.ffn_norm, lw.router, self.residual)
        rmsnorm(self.residual, w.output_norm, cfg.eps, self.normed)
        self.logits.copy_(self._rows(gemv_q8_k_batched, Q.Q6_K, w.lm_head, H, cfg.vocab, quantize_row_q8_k(self.normed)))
        return self.logits

    @_on_its_device
    def generate(self, prompt: Sequence[int], n_new: int, seed: int = 0, temperature: float = 1.0, top_k: int = 0,
                 top_p: float = 1.0, min_p: float = 0.0):
        """n continuations of `prompt` by n_new tokens: (tokens int32, logprobs
        f32), both [n, n_new] on the device.  The uniforms come from `seed`."""
        d = self.residual.device
        g = torch.Generator(device=d)
        g.manual_seed(seed)
        u = torch.rand(n_new, self.n, device=d, generator=g)
        full = lambda v: torch.full((self.n,), v, dtype=torch.float32, device=d)  # noqa: E731
        filters = (full(temperature), torch.full((self.n,), top_k, dtype=torch.int32, device=d), full(top_p), full(min_p))
        tokens = torch.empty(n_new, self.n, dtype=torch.int32, device=d)
        logprobs = torch.empty(n_new, self.n, dtype=torch.float32, device=d)
        logits = self.prefill(prompt).expand(self.n, -1)
        for i in range(n_new):
            sample(logits, u[i], *filters, tokens=tokens[i], logprobs=logprobs[i])
            if i + 1 < n_new:
                logits = self.step(tokens[i])
        return tokens.t().contiguous(), logprobs.t().contiguous()


def kl_divergence(ref_logits, logits) -> float:
    """Full-vocab KL(p_ref || p) in f64 from two logit vectors (the
    comparison of scripts/kl_vs_reference.py)."""
    a = np.asarray(ref_logits, np.float64)
    b = np.asarray(logits, np.float64)
    la = a - a.max() - math.log(np.exp(a - a.max()).sum())
    lb = b - b.max() - math.log(np.exp(b - b.max()).sum())
    return float(np.sum(np.exp(la) * (la - lb)))


def top1(logits) -> int:
    """Sampler::argmax (generate/mod.rs:321-331): the first index of the
    largest value; NaN never wins; 0 when nothing beats -inf."""
    x = np.asarray(logits, np.float32)
    valid = x > -np.inf  # False for NaN
    if not valid.any():
        return 0
    return int(np.flatnonzero(valid & (x == x[valid].max()))[0])


def _main(argv=None):
    """python -m ramvamp_b200.model [--layers N] [--profile-step K]: build
    the synthetic Qwen3 model, run K eager steps, then one more inside the
    NVTX range "step" (for a profiler restricted to that range).  With
    --continuations C: draw C continuations of K tokens of a short prompt."""
    import argparse

    ap = argparse.ArgumentParser()
    ap.add_argument("--layers", type=int, default=48)
    ap.add_argument("--profile-step", type=int, default=8)
    ap.add_argument("--continuations", type=int, default=0)
    a = ap.parse_args(argv)
    w = Qwen3Weights.synthetic(ModelConfig(n_layers=a.layers), seed=1)
    if a.continuations:
        par = ParallelDecoder(w, a.continuations, max_prompt=16, max_new=a.profile_step)
        tokens, logprobs = par.generate([5, 17, 290, 4], a.profile_step, seed=1, temperature=0.8, top_k=50, top_p=0.95)
        for t, lp in zip(tokens.tolist(), logprobs.sum(1).tolist()):
            print(f"{lp:9.3f}", t)
        return
    dec = Decoder(w, max_positions=a.profile_step + 8)
    dec.reset()
    dec.token.fill_(5)
    for _ in range(a.profile_step):
        dec.step()
    torch.cuda.synchronize()
    torch.cuda.nvtx.range_push("step")
    dec.step()
    torch.cuda.nvtx.range_pop()
    torch.cuda.synchronize()
    print("next token", int(dec.next_token.item()))


if __name__ == "__main__":
    _main()
