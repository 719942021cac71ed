"""Qwen3 decoder on the gfx950 kernels (the model the attention path serves).

Follows the reference layer sequence (``src/models/qwen3/model.rs:155-534``):

    hidden = embed(ids)
    per layer:  (x, residual) = input_norm(hidden, residual)        rms_norm / add_rms_norm
                qkv = x W_qkv^T                                       packed [T, (Hq+2Hkv) D]
                q, k <- rope(qk_norm(q, k)); cache[write_loc] <- (k, v)   one fused pass here
                a = attention(q, k, v)                                 decode / prefill plan
                (x, residual) = add_rms_norm(a W_o^T, residual)
                hidden = (silu(x W_gate^T) * x W_up^T) W_down^T
    logits = add_rms_norm(hidden, residual)[logits_indices] W_lm^T

For decode batches (at most 256 rows) the QKV, o_proj and down projections run on this
library's projection kernel (QKV with its split-K partials summed inside the QK-norm/RoPE/
store pass, o_proj and down fused with the residual RMSNorm that follows them) and gate_up runs
fused with SiLU x mul, as does the lm_head of up to 64 rows; prefill-sized products and larger
heads are library GEMMs (torch -> hipBLASLt). Everything around them is this library's HIP code.
Configuration fields and defaults follow ``src/models/qwen3/config.rs:9-42``.

Two variants that the reference does not have: with ``num_experts`` every layer's MLP is one of
routed experts (``experts.route_experts``, ``experts.expert_mlp``) in place of the dense one, and
``Qwen3Model.quantize_int8`` turns the layers' matrices into 8-bit ones.
"""
from __future__ import annotations

import contextlib
import gc
import weakref
from dataclasses import dataclass

import torch
import torch.nn.functional as F

from . import experts, ops
from .backend import Attention, AttentionBatch, AttentionSpec
from .int8 import Int8Weight
from .kv_cache import BaseAttention, ModelError


@dataclass(frozen=True)
class Qwen3Config:
    hidden_size: int
    num_layers: int
    num_attention_heads: int
    num_kv_heads: int
    intermediate_size: int
    vocab_size: int
    head_dim: int = 128
    max_position_embeddings: int = 8192
    rope_theta: float = 10_000.0
    rms_norm_eps: float = 1e-6
    tie_word_embeddings: bool = False
    # Experts of every layer's MLP (0: a dense MLP of intermediate_size), how many of them a token
    # is routed to, their width, and whether the chosen weights are normalised to sum to 1. Experts
    # in 16 bits need hidden_size and their width to be multiples of 8, those in 8 bits do not.
    num_experts: int = 0
    num_experts_per_tok: int = 0
    moe_intermediate_size: int = 0
    norm_topk_prob: bool = True

    @staticmethod
    def qwen3_8b() -> "Qwen3Config":
        """Qwen3-8B dimensions (36 layers, hidden 4096, 32/8 heads, FFN 12288)."""
        return Qwen3Config(4096, 36, 32, 8, 12288, 151936, 128, 40960, 1_000_000.0, 1e-6, False)

    @staticmethod
    def qwen3_0_6b() -> "Qwen3Config":
        """Qwen3-0.6B dimensions (28 layers, hidden 1024, 16/8 heads, FFN 3072)."""
        return Qwen3Config(1024, 28, 16, 8, 3072, 151936, 128, 40960, 1_000_000.0, 1e-6, True)

    def validate(self) -> None:
        if min(self.hidden_size, self.num_layers, self.num_attention_heads, self.num_kv_heads,
               self.intermediate_size, self.vocab_size, self.head_dim) <= 0:
            raise ModelError("Qwen3 dimensions must be positive")
        if self.num_attention_heads % self.num_kv_heads:
            raise ModelError("num_attention_heads must be a multiple of num_kv_heads")
        if self.num_experts and not (
                0 < self.num_experts <= experts.MAX_EXPERTS and self.moe_intermediate_size > 0
                and 0 < self.num_experts_per_tok <= min(self.num_experts, experts.MAX_TOP_K)):
            raise ModelError("invalid expert count, experts per token or expert width")

    @property
    def qkv_width(self) -> int:
        return (self.num_attention_heads + 2 * self.num_kv_heads) * self.head_dim


class Qwen3Layer:
    def __init__(self, cfg: Qwen3Config, dtype: torch.dtype, device: torch.device):
        h, d = cfg.hidden_size, cfg.head_dim
        self.input_layernorm = torch.ones(h, dtype=dtype, device=device)
        self.qkv_proj = torch.empty(cfg.qkv_width, h, dtype=dtype, device=device)
        self.q_norm = torch.ones(d, dtype=dtype, device=device)
        self.k_norm = torch.ones(d, dtype=dtype, device=device)
        self.o_proj = torch.empty(h, cfg.num_attention_heads * d, dtype=dtype, device=device)
        self.post_attention_layernorm = torch.ones(h, dtype=dtype, device=device)
        # A dense MLP's matrices, or those of all experts ([E, 2 I, h], [E, h, I]) and their router.
        lead, f = (), cfg.intermediate_size
        self.router: torch.Tensor | None = None
        if cfg.num_experts:
            lead, f = (cfg.num_experts,), cfg.moe_intermediate_size
            self.router = torch.empty(cfg.num_experts, h, dtype=dtype, device=device)
        self.gate_up_proj = torch.empty(*lead, 2 * f, h, dtype=dtype, device=device)
        self.down_proj = torch.empty(*lead, h, f, dtype=dtype, device=device)
        self.base_attention = BaseAttention()

    def matrices(self) -> list[torch.Tensor]:
        router = [] if self.router is None else [self.router]
        return [self.qkv_proj, self.o_proj, *router, self.gate_up_proj, self.down_proj]


class Qwen3Model:
    """Weights plus forward; one ``Attention`` shared by all layers."""

    def __init__(self, cfg: Qwen3Config, dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda", attention_backend: str = "mi355x"):
        cfg.validate()
        device = torch.device(device)
        self.cfg = cfg
        self.dtype = dtype
        self.device = device
        self.embed_tokens = torch.empty(cfg.vocab_size, cfg.hidden_size, dtype=dtype,
                                        device=device)
        self.layers = [Qwen3Layer(cfg, dtype, device) for _ in range(cfg.num_layers)]
        self.norm = torch.ones(cfg.hidden_size, dtype=dtype, device=device)
        self.lm_head = (self.embed_tokens if cfg.tie_word_embeddings else
                        torch.empty(cfg.vocab_size, cfg.hidden_size, dtype=dtype, device=device))
        self.rope = ops.HalfSplitRope(cfg.max_position_embeddings, cfg.head_dim, cfg.rope_theta,
                                      device)
        self.attention = Attention.new(attention_backend, AttentionSpec(
            cfg.num_attention_heads, cfg.num_kv_heads, cfg.head_dim, dtype, device))
        # Who holds captured graphs that read the weights where they are now (see quantize_int8).
        self._graph_holders: weakref.WeakSet = weakref.WeakSet()
        self._captured_by_caller = False
        self._capturing = False

    # ------------------------------------------------------------------ weights
    def init_random(self, seed: int, std: float = 0.02) -> "Qwen3Model":
        """Seeded N(0, std) matrices and embeddings; norm weights stay 1 (synthetic weights)."""
        g = torch.Generator(device=self.device)
        g.manual_seed(seed)
        mats = [self.embed_tokens] + [m for layer in self.layers for m in layer.matrices()]
        if not self.cfg.tie_word_embeddings:
            mats.append(self.lm_head)
        if any(isinstance(m, Int8Weight) for m in mats):
            raise ModelError("weights are drawn before they are quantised")
        for m in mats:
            m.normal_(0.0, std, generator=g)
        return self

    def named_parameters(self) -> dict[str, torch.Tensor]:
        """Hugging Face parameter names (qkv and gate/up stay packed)."""
        out = {"model.embed_tokens.weight": self.embed_tokens, "model.norm.weight": self.norm}
        if not self.cfg.tie_word_embeddings:
            out["lm_head.weight"] = self.lm_head
        for i, layer in enumerate(self.layers):
            p = f"model.layers.{i}."
            out[p + "input_layernorm.weight"] = layer.input_layernorm
            out[p + "self_attn.qkv_proj.weight"] = layer.qkv_proj
            out[p + "self_attn.q_norm.weight"] = layer.q_norm
            out[p + "self_attn.k_norm.weight"] = layer.k_norm
            out[p + "self_attn.o_proj.weight"] = layer.o_proj
            out[p + "post_attention_layernorm.weight"] = layer.post_attention_layernorm
            if layer.router is None:
                out[p + "mlp.gate_up_proj.weight"] = layer.gate_up_proj
                out[p + "mlp.down_proj.weight"] = layer.down_proj
            else:
                out[p + "mlp.gate.weight"] = layer.router
                out[p + "mlp.experts.gate_up_proj"] = layer.gate_up_proj
                out[p + "mlp.experts.down_proj"] = layer.down_proj
        return out

    def quantize_int8(self) -> "Qwen3Model":
        """The layers' QKV, o, gate_up and down matrices (those of experts too) in 8 bits, one scale
        a row; embeddings, norms, routers and the head stay as they are. Done once, after the
        weights are loaded, and before a graph is captured over them: refused while an engine with
        captured graphs exists, and for good after any other capture of ``forward``, as a replay
        would read the memory of the 16-bit matrices that are let go here."""
        if len(self._graph_holders):
            gc.collect()  # engines that nothing refers to any more
        if self._captured_by_caller or len(self._graph_holders):
            raise ModelError("weights are quantised before a graph is captured over them")
        for layer in self.layers:
            for name in ("qkv_proj", "o_proj", "gate_up_proj", "down_proj"):
                weight = getattr(layer, name)
                if not isinstance(weight, Int8Weight):
                    setattr(layer, name, Int8Weight.quantize(weight))
        return self

    def load_weights(self, weights) -> int:
        """Copy tensors by Hugging Face name (``named_parameters`` names); every parameter must
        be supplied with its exact shape (src/models/qwen3/model.rs:231-300). Returns the count."""
        params = self.named_parameters()
        if any(isinstance(p, Int8Weight) for p in params.values()):
            raise ModelError("weights are loaded before they are quantised")
        loaded = 0
        for name, value in weights.items():
            if name not in params:
                raise ModelError(f"unexpected weight {name}")
            t = torch.as_tensor(value)
            if tuple(t.shape) != tuple(params[name].shape):
                raise ModelError(f"weight {name} has shape {tuple(t.shape)}, "
                                 f"expected {tuple(params[name].shape)}")
            params[name].copy_(t.to(params[name].dtype))
            loaded += 1
        if loaded != len(params):
            missing = sorted(set(params) - set(weights))
            raise ModelError(f"missing weights: {missing[:4]}")
        return loaded

    @contextlib.contextmanager
    def captured_for(self, holder):
        """Around captures of ``forward`` whose graphs live no longer than ``holder``."""
        self._graph_holders.add(holder)
        self._capturing = True
        try:
            yield
        finally:
            self._capturing = False

    def check_runnable(self) -> None:
        """Raise for weights that no forward takes: 16-bit experts of a width that is no multiple of
        8 (``quantize_int8`` makes them runnable)."""
        cfg = self.cfg
        if not cfg.num_experts or (cfg.hidden_size | cfg.moe_intermediate_size) % 8 == 0:
            return
        if any(not isinstance(m, Int8Weight) for layer in self.layers
               for m in (layer.gate_up_proj, layer.down_proj)):
            raise ModelError("16-bit experts need hidden_size and moe_intermediate_size to be "
                             "multiples of 8")

    def bind_kv_cache(self, pool, reserved_slot: int = 0) -> None:
        """Bind every layer to its views of a ``KVCachePool`` (page 0 reserved)."""
        if pool.layout.num_layers != self.cfg.num_layers:
            raise ModelError("KV pool layer count does not match the model")
        for i, layer in enumerate(self.layers):
            kc, vc = pool.layer(i)
            layer.base_attention.bind_kv_cache(kc, vc)
            layer.base_attention.set_reserved_write_slot(reserved_slot)
        self.attention.bind_cache_layout(pool.layout.page_size)

    def check_write_errors(self) -> None:
        for layer in self.layers:
            layer.base_attention.check_write_errors()

    # ------------------------------------------------------------------ forward
    def forward(self, input_ids: torch.Tensor, positions: torch.Tensor,
                attention_batch: AttentionBatch, write_loc: torch.Tensor | None,
                logits_indices: torch.Tensor | None = None,
                logits_out: torch.Tensor | None = None) -> torch.Tensor:
        """Logits ``[N, vocab]`` for the selected rows (all rows when ``logits_indices`` is
        None). Safe to capture in a HIP graph: no host synchronisation happens inside."""
        cfg = self.cfg
        if input_ids.dim() != 1 or positions.shape != input_ids.shape:
            raise ModelError("input_ids and positions must have identical lengths")
        self.check_runnable()
        if not self._capturing and torch.cuda.is_current_stream_capturing():
            self._captured_by_caller = True
        t = input_ids.size(0)
        hq, hkv, d = cfg.num_attention_heads, cfg.num_kv_heads, cfg.head_dim
        eps = cfg.rms_norm_eps
        hidden = F.embedding(input_ids, self.embed_tokens)
        residual = hidden
        x = ops.rms_norm(hidden, self.layers[0].input_layernorm, eps)
        n_layers = len(self.layers)
        for i, layer in enumerate(self.layers):
            qkv = ops.linear_qk_norm_rope_store(x, layer.qkv_proj, hq, hkv, layer.q_norm,
                                                layer.k_norm, eps, positions, self.rope,
                                                layer.base_attention, write_loc)
            q = qkv[:, : hq * d].view(t, hq, d)
            k = qkv[:, hq * d:(hq + hkv) * d].view(t, hkv, d)
            v = qkv[:, (hq + hkv) * d:].view(t, hkv, d)
            attn = attention_batch.forward(q, k, v, layer.base_attention)
            # o_proj + post-attention norm, down + the next layer's input norm (the final
            # norm after the last layer): each a projection fused with its residual RMSNorm.
            x, residual = ops.linear_add_rms_norm(attn, layer.o_proj, residual,
                                                  layer.post_attention_layernorm, eps)
            next_norm = self.layers[i + 1].input_layernorm if i + 1 < n_layers else self.norm
            if layer.router is not None:
                weights, ids = experts.route_experts(ops.linear(x, layer.router),
                                                     cfg.num_experts_per_tok, cfg.norm_topk_prob)
                x = experts.expert_mlp(x, ids, weights, layer.gate_up_proj, layer.down_proj)
                x, residual = ops.add_rms_norm(x, residual, next_norm, eps)
                continue
            # gate_up with SiLU x mul (one launch for decode batches)
            act = ops.linear_silu_mul(x, layer.gate_up_proj)
            x, residual = ops.linear_add_rms_norm(act, layer.down_proj, residual, next_norm, eps)
        hidden = x
        if logits_indices is not None:
            hidden = hidden.index_select(0, logits_indices)
        return ops.head_linear(hidden, self.lm_head, logits_out)


__all__ = ["Qwen3Config", "Qwen3Model", "Qwen3Layer"]
