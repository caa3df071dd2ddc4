"""One decoder layer of izwi-core's Qwen3 model at one token, and for whole prompts, composed from the library's calls.

Mirror of `Qwen3Layer::forward` (qwen3/core.rs:1863-1881) with `Qwen3Attention::forward`'s
single-token path (core.rs:1446-1575: q/k/v projections, per-head q/k norm, rotary embedding, cache
append, grouped-query attention, output projection) and `Qwen3Mlp::forward` (core.rs:1786-1798),
f32 activations.  Every arithmetic step is one library call; torch only appends the new key /
value rows to the caches in the unfused form and owns the tensors.  Per layer: 5 kernel launches, 6 where
the attention is split over the cache (the two RMSNorms ride in the projection launches behind them; q/k norm, rotary and the cache
append ride in the attention launch) behind one library call, or 11 to 12 with the reference's separate hooks and two copies,
where the reference's eager path issues one per operator.

`Qwen3PromptLayer` is the same layer for prompts of any lengths, packed one behind the other (the multi-token path of
core.rs:1446-1575 for a batch without padding): projections, rotary positions with the q/k norm, attention within each
prompt, output projection, MLP or experts (`SparseMlp`).
"""
from __future__ import annotations

import torch

from .capi import ERR_INVALID, QmmError, check, lib
from .decode_ops import (decode_attention_step, qk_norm_rope_append, try_fused_decode_gqa_attention_with_kv_len, try_fused_qk_rms_norm,
                         try_fused_rms_norm, try_fused_rope_pair_bshd)
from .prompt_ops import RotaryEmbedding, prompt_attention, rope_positions
from .qmatmul import MoeExperts, QMatMul, Qwen3GateUpProjection, _stream_ptr, forward_group, moe_route_scored, moe_sort


class Qwen3DecodeLayer:
    def __init__(self, input_layernorm: torch.Tensor, post_attention_layernorm: torch.Tensor, q_proj: QMatMul,
                 k_proj: QMatMul, v_proj: QMatMul, qk_norm_weight: torch.Tensor, o_proj: QMatMul, gate_proj: QMatMul,
                 up_proj: QMatMul, down_proj: QMatMul, num_heads: int, num_kv_heads: int, head_dim: int,
                 rms_norm_eps: float = 1e-6, fuse_prep: bool = True, fuse_norm: bool = True, fuse_step: bool = True):
        self.w_in, self.w_post, self.qk_w = input_layernorm, post_attention_layernorm, qk_norm_weight
        self.qkv = (q_proj, k_proj, v_proj)
        self.o_proj, self.down_proj = o_proj, down_proj
        self.gate_up = Qwen3GateUpProjection.new_separate(gate_proj, up_proj)
        self.heads, self.kv_heads, self.d, self.eps = num_heads, num_kv_heads, head_dim, rms_norm_eps
        self.fuse_prep = fuse_prep  # q/k norm, rotary and cache append as one launch instead of four
        self.fuse_norm = fuse_norm  # the two RMSNorms inside the projection launches that follow them
        self.fuse_step = fuse_step  # q/k norm, rotary and cache append inside the attention launch

    def forward(self, x: torch.Tensor, cos_sin: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                pos: int) -> torch.Tensor:
        """x [1, hidden] f32; cos_sin [1, head_dim] for position `pos`; caches [1, kv_heads, capacity,
        head_dim] holding positions < pos.  Returns the layer's output [1, hidden]; the caches gain
        position `pos`."""
        h, kv, d = self.heads, self.kv_heads, self.d
        if self.fuse_norm and self.fuse_prep and self.fuse_step:
            out = self._forward_one_call(x, cos_sin, k_cache, v_cache, pos)
            if out is not None:
                return out
        if self.fuse_norm:  # input_layernorm inside the q|k|v launch
            q, k, v = forward_group(self.qkv, x, norm_weight=self.w_in, eps=self.eps)
        else:
            q, k, v = forward_group(self.qkv, try_fused_rms_norm(x, self.w_in, self.eps))
        if self.fuse_prep and self.fuse_step:
            attn = decode_attention_step(q, k, v, self.qk_w, cos_sin, k_cache, v_cache, pos, self.eps, d ** -0.5)
        else:
            if self.fuse_prep:
                q4 = qk_norm_rope_append(q, k, v, self.qk_w, cos_sin, k_cache, v_cache, pos, self.eps)
            else:  # the same steps as the reference's separate hooks
                q4, k4 = try_fused_qk_rms_norm(q.view(1, 1, h, d), k.view(1, 1, kv, d), self.qk_w, self.eps)
                q4, k4 = try_fused_rope_pair_bshd(q4, k4, cos_sin)
                k_cache[0, :, pos] = k4.view(kv, d)
                v_cache[0, :, pos] = v.view(kv, d)
            attn = try_fused_decode_gqa_attention_with_kv_len(q4.view(1, h, 1, d), k_cache, v_cache, h, kv, d, pos + 1,
                                                              d ** -0.5)
        x = self.o_proj.forward_fused(attn.view(1, h * d), residual=x)       # x + o_proj(attn)
        if self.fuse_norm:  # post_attention_layernorm inside the gate|up launch
            hidden = self.gate_up.forward_silu_mul(x, norm_weight=self.w_post, eps=self.eps)
        else:
            hidden = self.gate_up.forward_silu_mul(try_fused_rms_norm(x, self.w_post, self.eps))  # silu(gate) * up
        return self.down_proj.forward_fused(hidden, residual=x)              # x + down_proj(hidden)

    def _forward_one_call(self, x, cos_sin, k_cache, v_cache, pos):
        """The fused form's five calls as one library call (the same kernels, the same results): the calls' own
        preparation, allocations and foreign-function overhead took 40 us of host time per layer, more than the
        launches of a 0.6B layer run for (28 layers and the head: 1850 us a token as calls, 855 this way).
        None for arguments it does not cover: those go call by call."""
        gate_up = self.gate_up._parts
        if gate_up is None:
            return None
        # (written out: every attribute and call here is paid once per layer and token; weights that do not fit together and a position
        # outside the caches are refused by the library before it launches anything, and then go call by call like everything else)
        w_in, w_post, qk_w = self.w_in, self.w_post, self.qk_w
        device = x.get_device()
        for t in (x, w_in, w_post, qk_w, cos_sin, k_cache, v_cache):
            if t.dtype is not torch.float32 or t.get_device() != device or not t.is_contiguous():
                return None
        qkv, h, kv, d = self.qkv, self.heads, self.kv_heads, self.d
        q, gate = qkv[0].qtensor, gate_up[0].qtensor
        hidden, cache = q._k, k_cache.shape
        if (device < 0 or x.shape != (1, hidden) or w_in.numel() != hidden or w_post.numel() != hidden or qk_w.numel() != 2 * d
                or cos_sin.numel() != d or len(cache) != 4 or cache[0] != 1 or cache[1] != kv or cache[3] != d or v_cache.shape != cache):
            return None
        floats = 2 * (h * d + 127 & -128) + 2 * (kv * d + 127 & -128) + (hidden + 127 & -128) + (gate._n + 127 & -128)
        workspace, y = x.new_empty(floats), x.new_empty((1, hidden))
        rc = lib().izwi_qmm_decode_layer_f32(q._h, qkv[1].qtensor._h, qkv[2].qtensor._h, self.o_proj.qtensor._h, gate._h,
                                             gate_up[1].qtensor._h, self.down_proj.qtensor._h, x.data_ptr(), w_in.data_ptr(),
                                             w_post.data_ptr(), qk_w.data_ptr(), cos_sin.data_ptr(), h, kv, d, self.eps,
                                             k_cache.data_ptr(), v_cache.data_ptr(), cache[2], pos, workspace.data_ptr(),
                                             4 * floats, y.data_ptr(), _stream_ptr(x))
        if rc == ERR_INVALID:
            return None
        check(rc)
        return y


class SparseMlp:
    """Experts behind a scored router: the router's product, `moe_route_scored` (whose arguments ``routing`` are), the sort by expert and the
    experts' products."""

    def __init__(self, router: QMatMul, experts: MoeExperts, top_k: int, **routing):
        n, hidden = router.qtensor.dims2()
        if (n, hidden) != (experts.gate.shape()[0], experts.gate.shape()[-1]) or len(experts.gate.shape()) != 3:
            raise QmmError(ERR_INVALID, f"SparseMlp: a router of {n} experts on {hidden} for experts of {experts.gate.shape()}")
        self.router, self.experts, self.top_k, self.routing = router, experts, top_k, routing

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() != 2 or x.dtype is not torch.float32 or x.shape[1] != self.router.qtensor.dims2()[1]:
            raise QmmError(ERR_INVALID, f"SparseMlp: x [tokens, {self.router.qtensor.dims2()[1]}] of f32 expected")
        if x.shape[0] == 0:
            return torch.empty_like(x)
        logits = self.router.forward(x)
        ids, weights = moe_route_scored(logits, self.top_k, **self.routing)
        perm, offsets = moe_sort(ids, logits.shape[1])
        return self.experts.forward(x, ids, weights, perm, offsets)


class Qwen3PromptLayer:
    """A decoder layer for whole prompts, f32 activations.  ``mlp``: (gate_proj, up_proj, down_proj), or a `SparseMlp`."""

    def __init__(self, input_layernorm: torch.Tensor, post_attention_layernorm: torch.Tensor, q_proj: QMatMul, k_proj: QMatMul, v_proj: QMatMul,
                 qk_norm_weight: torch.Tensor, o_proj: QMatMul, mlp, num_heads: int, num_kv_heads: int, head_dim: int, rotary: RotaryEmbedding,
                 rms_norm_eps: float = 1e-6):
        hidden = input_layernorm.numel()
        if num_heads <= 0 or num_kv_heads <= 0 or num_heads % num_kv_heads or rotary.head_dim != head_dim:
            raise QmmError(ERR_INVALID, f"Qwen3PromptLayer: {num_heads} heads of {head_dim} on {num_kv_heads}, rotary positions for heads of {rotary.head_dim}")
        if post_attention_layernorm.numel() != hidden or qk_norm_weight.numel() != 2 * head_dim:
            raise QmmError(ERR_INVALID, f"Qwen3PromptLayer: norms of {hidden}, {post_attention_layernorm.numel()} and {qk_norm_weight.numel()} (2 x {head_dim} expected)")
        q, kv = num_heads * head_dim, num_kv_heads * head_dim
        parts = [("q_proj", q_proj, (q, hidden)), ("k_proj", k_proj, (kv, hidden)), ("v_proj", v_proj, (kv, hidden)), ("o_proj", o_proj, (hidden, q))]
        if isinstance(mlp, SparseMlp):
            if mlp.router.qtensor.dims2()[1] != hidden:
                raise QmmError(ERR_INVALID, f"Qwen3PromptLayer: experts on {mlp.router.qtensor.dims2()[1]} in a layer of {hidden}")
        else:
            inner = mlp[0].qtensor.dims2()[0]
            parts += [("gate_proj", mlp[0], (inner, hidden)), ("up_proj", mlp[1], (inner, hidden)), ("down_proj", mlp[2], (hidden, inner))]
        for name, part, shape in parts:
            if tuple(part.qtensor.dims2()) != shape:
                raise QmmError(ERR_INVALID, f"Qwen3PromptLayer: {name} is {tuple(part.qtensor.dims2())}, {shape} expected")
        self.w_in, self.w_post, self.qk_w = input_layernorm, post_attention_layernorm, qk_norm_weight
        self.qkv, self.o_proj, self.rotary = (q_proj, k_proj, v_proj), o_proj, rotary
        self.sparse = mlp if isinstance(mlp, SparseMlp) else None
        if self.sparse is None:
            gate, up, self.down_proj = mlp
            self.gate_up = Qwen3GateUpProjection.new_separate(gate, up)
        self.heads, self.kv_heads, self.d, self.eps = num_heads, num_kv_heads, head_dim, rms_norm_eps

    def forward(self, x: torch.Tensor, positions: torch.Tensor, starts: torch.Tensor | None = None, max_len: int | None = None):
        """x [tokens, hidden] f32, positions int32 [tokens], starts int32 [prompts + 1] (None: one prompt) -> (the layer's output [tokens,
        hidden], keys, values [tokens, kv_heads, head_dim], which belong into the caches of the decode step).  ``max_len``: the longest
        prompt's tokens, where the caller knows them (else all tokens count); the attention's division of the work goes by it.  A token of no
        prompt, in front of, between or behind them, is one whose attention is zero."""
        if x.dim() != 2 or x.dtype is not torch.float32 or x.shape[1] != self.w_in.numel():
            raise QmmError(ERR_INVALID, f"Qwen3PromptLayer: x [tokens, {self.w_in.numel()}] of f32 expected")
        tokens, d = x.shape[0], self.d
        if tokens == 0:
            none = x.new_empty(0, self.kv_heads, d)
            return torch.empty_like(x), none, none.clone()
        q, k, v = forward_group(self.qkv, x, norm_weight=self.w_in, eps=self.eps)
        q, k, v = q.view(tokens, self.heads, d), k.view(tokens, self.kv_heads, d), v.view(tokens, self.kv_heads, d)
        rope_positions(q, k, positions, self.rotary, qk_weight=self.qk_w, eps=self.eps, out=(q, k))
        out = None if starts is None else torch.zeros_like(q)  # (rows of no prompt are not written: their attention is zero)
        attn = prompt_attention(q, k, v, starts, max_len_k=max_len, out=out)
        x = self.o_proj.forward_fused(attn.view(tokens, self.heads * d), residual=x)
        if self.sparse is not None:
            return x + self.sparse.forward(try_fused_rms_norm(x, self.w_post, self.eps)), k, v
        hidden = self.gate_up.forward_silu_mul(x, norm_weight=self.w_post, eps=self.eps)
        return self.down_proj.forward_fused(hidden, residual=x), k, v
