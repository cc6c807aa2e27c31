"""Mixture-of-experts decoder: attention blocks whose FFN is a sparse top-k MoE of SwiGLU experts,
optionally with an always-on shared expert.

Covers the reference's MoEBlock / MoEModel (src/moe_model.cpp:17-53,115-212: attention + SparseMoE FFN
+ optional shared expert, presets, OIL save/load with the tensor names of :314-358) on the kernels of
``ops/moe.py``. ``forward`` returns the language-model loss plus the weighted auxiliary losses, which
carry gradients into the routers.
"""
from __future__ import annotations

import math

import torch
import torch.nn as nn

from .. import ops
from ..ops.int8 import Int8Weight
from ..ops.moe import FEW_TOKENS, moe_few_supported, moe_ffn, moe_ffn_few
from .config import TransformerConfig
from .dense import Attention, FFN, Norm, _ste, head_norm_state, load_head_norms


class MoELayer(nn.Module):
    """``ep_world`` > 1: only ``num_experts / ep_world`` experts are resident (expert parallelism); the model sets
    ``ep`` (the shared ``EPContext``) once the parameters are on their device."""

    # Prompts of up to that many times 64 tokens go through the form for a few, with experts in 8 bits: 80 us each for 8 experts of 2048 x 5632, 50 for 64 of 1024 x 704, 30 for 8
    # of 256 x 512, where widening all weights and the training form take 1.3 ms, 0.71 ms and 0.26 ms: even at 1050, 950 and 500 tokens.
    INT8_CHUNKS = 12

    def __init__(self, cfg: TransformerConfig, dtype, ep_world: int = 1):
        super().__init__()
        self.cfg = cfg
        E, D, Fh = cfg.num_experts, cfg.hidden_size, cfg.moe_ffn_hidden_size or cfg.ffn_hidden_size
        assert E % ep_world == 0
        self.router = nn.Linear(D, E, bias=False, dtype=dtype)
        self.w_gate_up = nn.Parameter(torch.empty(E // ep_world, 2 * Fh, D, dtype=dtype))
        self.w_down = nn.Parameter(torch.empty(E // ep_world, D, Fh, dtype=dtype))
        self.shared = FFN(cfg, dtype, hidden=Fh) if cfg.shared_expert else None
        self.last_counts = None
        self.ep = None

    def _experts(self, h, residual, w_gate_up, w_down):
        """(residual and weighted experts, auxiliary losses), as in training."""
        cfg = self.cfg
        if self.ep is not None:
            from ..parallel.expert_parallel import _EPMoEFn
            y, aux, self.last_counts = _EPMoEFn.apply(h, self.router.weight, w_gate_up, w_down, residual, self.ep, cfg.top_k, cfg.lb_coef, cfg.z_coef)
        else:
            y, aux, self.last_counts = moe_ffn(h, self.router.weight, w_gate_up, w_down, residual, cfg.top_k, cfg.lb_coef, cfg.z_coef)
        return y, aux

    def forward(self, h, residual):
        y, aux = self._experts(h, residual, _ste(self.w_gate_up, self.cfg), _ste(self.w_down, self.cfg))
        if self.shared is not None:
            y = self.shared(h, y)
        return y, aux

    def _plain_shared(self):
        """Whether the shared expert is one that the layer of a few tokens takes along: SwiGLU without biases and adapters."""
        s = self.shared
        return s is not None and s.gated and s.gate_up_proj.bias is None and s.adapter is None

    def _few_weights(self):
        """Experts, and a shared one or None, as a forward pass takes them."""
        s, cfg = self.shared, self.cfg
        return (_ste(self.w_gate_up, cfg), _ste(self.w_down, cfg),
                (_ste(s.gate_up_proj.weight, cfg), _ste(s.down_proj.weight, cfg)) if self._plain_shared() else None)

    @torch.no_grad()
    def int8_weights(self):
        """Experts, and a shared one of SwiGLU without biases and adapters, in 8-bit integers, for ``serve``."""
        if self.ep is not None:
            raise ValueError("experts that several ranks hold have no form in 8-bit integers")
        w_gate_up, w_down, shared = self._few_weights()
        return Int8Weight.quantize(w_gate_up), Int8Weight.quantize(w_down), shared and tuple(Int8Weight.quantize(w) for w in shared)

    @torch.no_grad()
    def serve(self, h, residual, int8=None):
        """The layer for generation, without the auxiliary losses: up to 64 tokens in two launches (``ops.moe.moe_ffn_few``), with experts in 8 bits where
        ``int8_weights`` are given. More tokens, experts on several ranks and what that form does not have run as in training; where ``int8_weights`` are given,
        on the values that these stand for, rounded to the model's type."""
        if int8 is not None:
            return self._serve_int8(h, residual, *int8)
        if self.ep is None and moe_few_supported(h, self.router.weight, self.w_gate_up, self.w_down, self.cfg.top_k):
            w_gate_up, w_down, shared = self._few_weights()
            y, self.last_counts = moe_ffn_few(h, self.router.weight, w_gate_up, w_down, residual, self.cfg.top_k, shared)
            return y if shared is not None or self.shared is None else self.shared(h, y)
        return self(h, residual)[0]

    def _serve_int8(self, h, residual, w_gate_up, w_down, shared):
        x, r = h.reshape(-1, h.shape[-1]), residual.reshape(-1, h.shape[-1])
        if len(x) <= self.INT8_CHUNKS * FEW_TOKENS and moe_few_supported(x[:FEW_TOKENS], self.router.weight, w_gate_up, w_down, self.cfg.top_k):
            parts = [moe_ffn_few(x[i:i + FEW_TOKENS], self.router.weight, w_gate_up, w_down, r[i:i + FEW_TOKENS], self.cfg.top_k, shared)
                     for i in range(0, max(1, len(x)), FEW_TOKENS)]              # a token's result depends on no other
            y, counts = parts[0] if len(parts) == 1 else (torch.cat([p[0] for p in parts]), torch.stack([p[1] for p in parts]).sum(0, dtype=torch.int32))
            y, self.last_counts = y.view(h.shape), counts
        else:
            y, _ = self._experts(h, residual, w_gate_up.dequantize(h.dtype), w_down.dequantize(h.dtype))
            if shared is not None:
                gate_up, down = (w.dequantize(h.dtype) for w in shared)
                y = ops.linear(ops.swiglu(ops.linear(h, gate_up)), down, residual=y, mode="add")
        return y if shared is not None or self.shared is None else self.shared(h, y)


class MoEBlock(nn.Module):
    def __init__(self, cfg: TransformerConfig, dtype, ep_world: int = 1):
        super().__init__()
        self.attention_norm = Norm(cfg.hidden_size, cfg.norm, cfg.norm_eps, dtype)
        self.attention = Attention(cfg, dtype)
        self.ffn_norm = Norm(cfg.hidden_size, cfg.norm, cfg.norm_eps, dtype)
        self.moe = MoELayer(cfg, dtype, ep_world)

    def forward(self, x, rope, positions=None):
        x = self.attention(self.attention_norm(x), x, rope, positions)
        return self.moe(self.ffn_norm(x), x)


class MoEModel(nn.Module):
    def __init__(self, cfg: TransformerConfig, dtype=torch.bfloat16, device=None, seed=42, ep_group=None, ep_max_tokens: int = 0,
                 ep_capacity_factor=None):
        """``ep_group``: process group over which the experts are sharded (expert e on rank e // (E / W)); tokens are
        exchanged over peer memory (parallel/expert_parallel.py). ``ep_max_tokens``: tokens per rank per step;
        ``ep_capacity_factor``: receive capacity per rank in units of its average load (None = dropless)."""
        super().__init__()
        assert cfg.num_experts > 0
        self.cfg = cfg
        import torch.distributed as dist
        self.ep_group = ep_group
        self.ep_world = dist.get_world_size(ep_group) if (ep_group is not None and dist.is_initialized()) else 1
        self.ep_rank = dist.get_rank(ep_group) if self.ep_world > 1 else 0
        Vp, E = cfg.padded_vocab, cfg.hidden_size
        self.tok_embeddings = nn.Embedding(Vp, E, dtype=dtype)
        self.pos_embeddings = nn.Embedding(cfg.max_seq_len, E, dtype=dtype) if cfg.positions == "learned" else None
        self.layers = nn.ModuleList([MoEBlock(cfg, dtype, self.ep_world) for _ in range(cfg.num_layers)])
        self.norm = Norm(E, cfg.norm, cfg.norm_eps, dtype)
        self.lm_head = nn.Linear(E, Vp, bias=False, dtype=dtype)
        self._rope = None
        self.reset_parameters(seed)
        if device is not None:
            self.to(device)
        if self.ep_world > 1:
            from ..parallel.expert_parallel import EPContext
            dev = next(self.parameters()).device
            ep = EPContext(ep_group, cfg.num_experts, cfg.hidden_size, ep_max_tokens or cfg.max_seq_len, cfg.top_k, dev, ep_capacity_factor)
            for blk in self.layers:
                blk.moe.ep = ep

    def expert_parameters(self):
        """Parameters that exist once per expert (sharded under expert parallelism, never all-reduced)."""
        return [p for n, p in self.named_parameters() if n.endswith("moe.w_gate_up") or n.endswith("moe.w_down")]

    @torch.no_grad()
    def reset_parameters(self, seed=42):
        g = torch.Generator().manual_seed(seed)
        g_local = torch.Generator().manual_seed(seed * 1000 + 17 + self.ep_rank)    # experts differ between ranks
        for name, p in self.named_parameters():
            if p.dim() >= 2:
                local = self.ep_world > 1 and (name.endswith("moe.w_gate_up") or name.endswith("moe.w_down"))
                w = torch.empty(p.shape, dtype=torch.float32).normal_(0.0, 0.02, generator=g_local if local else g)
                if name.endswith("o_proj.weight") or name.endswith("down_proj.weight") or name.endswith("w_down"):
                    w.mul_(1.0 / math.sqrt(2.0 * self.cfg.num_layers))
                p.copy_(w.to(p.dtype))
            elif name.endswith("bias"):
                p.zero_()
            else:
                p.fill_(1.0)

    def rope(self, device):
        if self.cfg.positions != "rope":
            return None
        if self._rope is None or self._rope[0].device != device:
            self._rope = ops.rope_tables(self.cfg.max_seq_len, self.cfg.head_dim, self.cfg.rope_theta, device)
        return self._rope

    def forward(self, ids, labels=None, positions=None, grad_scale=1.0):
        wpe = self.pos_embeddings.weight if self.pos_embeddings is not None else None
        x = ops.embedding(ids, self.tok_embeddings.weight, wpe)
        rope = self.rope(x.device)
        aux_total = None
        for blk in self.layers:
            x, aux = blk(x, rope, positions)
            aux_total = aux if aux_total is None else aux_total + aux
        h = self.norm(x)
        if labels is None:
            return ops.linear(h, self.lm_head.weight)[..., : self.cfg.vocab_size]
        loss = ops.lm_head_cross_entropy(h, self.lm_head.weight, labels, vocab=self.cfg.vocab_size, grad_scale=grad_scale)
        self.last_aux = aux_total.detach()
        return loss + aux_total

    def expert_utilisation(self):
        """Tokens routed to each expert in the last forward, per layer (MoEMetrics, include/oil/moe_trainer.h:40-57)."""
        return [blk.moe.last_counts for blk in self.layers]

    def num_params(self):
        return sum(p.numel() for p in self.parameters())

    # ------------------------------------------------------------------ reference tensor names
    def state_dict_reference(self):
        cfg = self.cfg
        H, Hkv, D = cfg.num_heads, cfg.kv_heads, cfg.head_dim
        out = {"tok_embeddings.weight": self.tok_embeddings.weight[: cfg.vocab_size]}
        for i, blk in enumerate(self.layers):
            pre = f"layers.{i}."
            out[pre + "attention_norm.weight"] = blk.attention_norm.weight
            out[pre + "ffn_norm.weight"] = blk.ffn_norm.weight
            q, k, v = blk.attention.qkv_proj.weight.split([H * D, Hkv * D, Hkv * D], dim=0)
            out[pre + "attention.q_proj.weight"], out[pre + "attention.k_proj.weight"], out[pre + "attention.v_proj.weight"] = q, k, v
            out[pre + "attention.o_proj.weight"] = blk.attention.o_proj.weight
            head_norm_state(out, pre, blk.attention)
            out[pre + "moe.router.weight"] = blk.moe.router.weight
            for e in range(cfg.num_experts):
                g, u = blk.moe.w_gate_up[e].chunk(2, dim=0)
                out[pre + f"moe.expert.{e}.gate_proj.weight"] = g
                out[pre + f"moe.expert.{e}.up_proj.weight"] = u
                out[pre + f"moe.expert.{e}.down_proj.weight"] = blk.moe.w_down[e]
            if blk.moe.shared is not None:
                g, u = blk.moe.shared.gate_up_proj.weight.chunk(2, dim=0)
                out[pre + "shared_expert.gate_proj.weight"], out[pre + "shared_expert.up_proj.weight"] = g, u
                out[pre + "shared_expert.down_proj.weight"] = blk.moe.shared.down_proj.weight
        out["norm.weight"] = self.norm.weight
        out["lm_head.weight"] = self.lm_head.weight[: cfg.vocab_size]
        return {k: v.detach().float().cpu().contiguous() for k, v in out.items()}

    @torch.no_grad()
    def load_reference_state(self, tensors: dict, ref_layout: bool = False):
        cfg = self.cfg
        H, Hkv, D, E = cfg.num_heads, cfg.kv_heads, cfg.head_dim, cfg.hidden_size
        Fh = cfg.moe_ffn_hidden_size or cfg.ffn_hidden_size

        def mat(name, out_f, in_f):
            t = tensors[name].reshape(-1)
            return t.view(in_f, out_f).t() if ref_layout else t.view(out_f, in_f)

        v = tensors["tok_embeddings.weight"].view(-1, E)
        self.tok_embeddings.weight[: v.shape[0]].copy_(v)
        for i, blk in enumerate(self.layers):
            pre = f"layers.{i}."
            blk.attention_norm.weight.copy_(tensors[pre + "attention_norm.weight"].view(-1))
            blk.ffn_norm.weight.copy_(tensors[pre + "ffn_norm.weight"].view(-1))
            blk.attention.qkv_proj.weight.copy_(torch.cat([mat(pre + "attention.q_proj.weight", H * D, E), mat(pre + "attention.k_proj.weight", Hkv * D, E),
                                                           mat(pre + "attention.v_proj.weight", Hkv * D, E)], dim=0))
            blk.attention.o_proj.weight.copy_(mat(pre + "attention.o_proj.weight", E, H * D))
            load_head_norms(tensors, pre, blk.attention)
            blk.moe.router.weight.copy_(mat(pre + "moe.router.weight", cfg.num_experts, E))
            for e in range(cfg.num_experts):
                blk.moe.w_gate_up[e].copy_(torch.cat([mat(pre + f"moe.expert.{e}.gate_proj.weight", Fh, E),
                                                      mat(pre + f"moe.expert.{e}.up_proj.weight", Fh, E)], dim=0))
                blk.moe.w_down[e].copy_(mat(pre + f"moe.expert.{e}.down_proj.weight", E, Fh))
            if blk.moe.shared is not None and pre + "shared_expert.gate_proj.weight" in tensors:
                blk.moe.shared.gate_up_proj.weight.copy_(torch.cat([mat(pre + "shared_expert.gate_proj.weight", Fh, E),
                                                                    mat(pre + "shared_expert.up_proj.weight", Fh, E)], dim=0))
                blk.moe.shared.down_proj.weight.copy_(mat(pre + "shared_expert.down_proj.weight", E, Fh))
        self.norm.weight.copy_(tensors["norm.weight"].view(-1))
        if "lm_head.weight" in tensors:
            v = mat("lm_head.weight", cfg.vocab_size, E)
            self.lm_head.weight[: v.shape[0]].copy_(v)
