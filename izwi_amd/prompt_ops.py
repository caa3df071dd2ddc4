"""Whole prompts between the projections: rotary positions and attention of packed sequences, over the C ABI of
include/izwi_decode_ops.h.

Prompts of different lengths stand one behind the other as rows of tokens, f32, f16 or bf16; q, k and v may be parts of the rows of one
q|k|v product.  The reference rotates by tables of cosines and sines and attends over padded batches with eager operators
(qwen3/core.rs:1464-1575); here every token has its own position and nothing is padded.

    rotary = RotaryEmbedding(head_dim, base=1e6)                        # once
    starts = int32 [prompts + 1]: where each prompt begins, and the end
    q, k = rope_positions(q, k, positions, rotary, qk_weight, eps)       # the heads' norm with it
    out = prompt_attention(q, k, v, starts)

Everything runs on the current stream; nothing waits for the device.  Arguments that do not fit raise ``QmmError``."""
from __future__ import annotations

import ctypes as C
from typing import NamedTuple

import torch

from .capi import QmmError, check, lib
from .qmatmul import _current_device, _raw_stream

_NAMES = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}
_i32 = torch.int32
# (What a call checks and looks up is paid for once per layer: device numbers are compared instead of devices, and the library's functions are
# looked up once.)
_ropes, _attentions = {}, {}


def _fn(fns: dict, name: str, dtype):
    """The library's function for the type; None where there is none."""
    fn = fns.get(dtype)
    if fn is None and dtype in _NAMES:
        fn = fns[dtype] = getattr(lib(), f"{name}_{_NAMES[dtype]}")
    return fn


def _refuse(what: str):
    raise QmmError(-1, what)


def _stride(t, what: str) -> int:
    """Elements from one token to the next of [tokens, heads, d]; the heads of a token are contiguous."""
    tokens, heads, d = t.shape
    if t.is_contiguous():
        return heads * d
    s0, s1, s2 = t.stride()
    if (s2 != 1 and d > 1) or (s1 != d and heads > 1):
        _refuse(f"{what}: the heads of a token must be contiguous")
    return s0 if tokens > 1 else heads * d


class RopeScaling(NamedTuple):
    """How the frequencies of a context stretched to ``factor`` times its original length are scaled (izwi_rope_frequencies)."""
    kind: int
    factor: float
    original_len: float = 0.0
    low: float = 0.0
    high: float = 0.0
    attention_factor: float | None = None

    @classmethod
    def linear(cls, factor: float) -> "RopeScaling":
        """Every frequency divided by ``factor``."""
        return cls(1, factor)

    @classmethod
    def ntk(cls, factor: float) -> "RopeScaling":
        """The base times factor^(rotary_dim / (rotary_dim - 2))."""
        return cls(2, factor)

    @classmethod
    def llama3(cls, factor: float, original_len: float, low: float = 1.0, high: float = 4.0) -> "RopeScaling":
        """Frequencies that turn ``low`` times or less in ``original_len`` positions divided by ``factor``, those of ``high`` turns and more kept."""
        return cls(3, factor, original_len, low, high)

    @classmethod
    def yarn(cls, factor: float, original_len: float, low: float = 1.0, high: float = 32.0, attention_factor: float | None = None) -> "RopeScaling":
        """The same along the pairs' numbers; cosine and sine times ``attention_factor``, by default 0.1 ln(factor) + 1."""
        return cls(4, factor, original_len, low, high, attention_factor)


class RotaryEmbedding:
    """Frequencies of a model's rotary positions, made once: the first ``rotary_dim`` elements of a head (by default all) turn, in pairs
    (i, rotary_dim / 2 + i) or, ``interleaved``, (2 i, 2 i + 1).  ``frequencies`` (f64 [rotary_dim / 2] on the GPU) may be written to, but no other
    tensor put in its place; ``attention_factor`` may be set."""

    def __init__(self, head_dim: int, base: float = 10000.0, rotary_dim: int | None = None, interleaved: bool = False,
                 scaling: RopeScaling | None = None, device="cuda"):
        if torch.device(device).type != "cuda":
            _refuse(f"RotaryEmbedding: a GPU expected, not {device}")
        self.head_dim, self.rotary_dim, self.interleaved = head_dim, head_dim if rotary_dim is None else rotary_dim, bool(interleaved)
        if not 0 < self.rotary_dim <= head_dim:
            _refuse(f"RotaryEmbedding: {self.rotary_dim} of {head_dim} elements")
        values, self.attention_factor = rope_frequencies(self.rotary_dim, base, scaling)
        self._frequencies = torch.tensor(values, dtype=torch.float64, device=device)
        self._index = self._frequencies.get_device()

    @property
    def frequencies(self) -> torch.Tensor:
        return self._frequencies


def rope_frequencies(rotary_dim: int, base: float = 10000.0, scaling: RopeScaling | None = None):
    """([rotary_dim / 2] angles per position, factor on cosine and sine), on the host."""
    if not 0 < rotary_dim <= 1024:
        _refuse(f"rope_frequencies: rotary_dim {rotary_dim}")
    s = RopeScaling(0, 1.0) if scaling is None else scaling
    values, factor = (C.c_double * (rotary_dim // 2 + 1))(), C.c_double()
    check(lib().izwi_rope_frequencies(s.kind, rotary_dim, base, s.factor, s.original_len, s.low, s.high, values, C.byref(factor)))
    return list(values)[: rotary_dim // 2], factor.value if s.attention_factor is None else s.attention_factor


def rope_positions(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, rotary: RotaryEmbedding, qk_weight: torch.Tensor | None = None,
                   eps: float = 1e-6, out: tuple | None = None):
    """q [tokens, heads, head_dim] and k [tokens, kv_heads, head_dim] (None: q alone), rotated to ``positions`` (int32 [tokens]) -> (q, k).  With
    ``qk_weight`` [2 head_dim] (q's, then k's) every head is normed first.  ``out``: two tensors to write, which may be q and k themselves."""
    dtype, shape, index = q.dtype, q.shape, rotary._index
    fn = _ropes.get(dtype) or _fn(_ropes, "izwi_rope_positions", dtype)
    if fn is None or len(shape) != 3 or shape[2] != rotary.head_dim or q.get_device() != index:
        _refuse(f"rope_positions: q [tokens, heads, {rotary.head_dim}] of f32, f16 or bf16 on GPU {index} expected")
    tokens, heads, d = shape
    kv_heads = 0
    if k is not None:
        k_shape = k.shape
        if k.dtype is not dtype or len(k_shape) != 3 or k_shape[0] != tokens or k_shape[2] != d or k.get_device() != index:
            _refuse(f"rope_positions: k [{tokens}, kv_heads, {d}] of q's type and device expected")
        kv_heads = k_shape[1]
    if positions.dtype is not _i32 or positions.shape != (tokens,) or positions.get_device() != index or not positions.is_contiguous():
        _refuse(f"rope_positions: a contiguous int32 tensor of {tokens} positions on GPU {index} expected")
    weight = 0
    if qk_weight is not None:
        if qk_weight.dtype is not dtype or qk_weight.shape != (2 * d,) or qk_weight.get_device() != index or not qk_weight.is_contiguous():
            _refuse(f"rope_positions: a contiguous qk_weight of {2 * d} of q's type and device expected")
        weight = qk_weight.data_ptr()
    if index != _current_device():
        with torch.cuda.device(index):
            return rope_positions(q, k, positions, rotary, qk_weight, eps, out)
    q_step = heads * d if q.is_contiguous() else _stride(q, "rope_positions: q")
    k_ptr = k_step = k_to = k_to_step = 0
    if k is not None:
        k_ptr, k_step = k.data_ptr(), kv_heads * d if k.is_contiguous() else _stride(k, "rope_positions: k")
    if out is None:
        q_out, q_to_step, k_out = torch.empty_like(q), heads * d, None  # (contiguous, whether q is a part of wider rows or not)
        if k is not None:
            k_out, k_to_step = torch.empty_like(k), kv_heads * d
    else:
        q_out, k_out = out
        for x, y in ((q, q_out), (k, k_out)):
            if (x is None) != (y is None) or (x is not None and (y.dtype is not dtype or y.shape != x.shape or y.get_device() != index)):
                _refuse("rope_positions: out has to be as q and k are")
        q_to_step = _stride(q_out, "rope_positions: out")
        if k is not None:
            k_to_step = _stride(k_out, "rope_positions: out")
    if k is not None:
        k_to = k_out.data_ptr()
    rc = fn(q.data_ptr(), q_step, k_ptr, k_step, positions.data_ptr(), rotary._frequencies.data_ptr(), rotary.attention_factor, tokens, heads, kv_heads, d, rotary.rotary_dim,
            rotary.interleaved, weight, eps, q_out.data_ptr(), q_to_step, k_to, k_to_step, _raw_stream(index))
    if rc:
        check(rc)
    return q_out, k_out


def prompt_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor | None = None, starts_k: torch.Tensor | None = None,
                     causal: bool = True, scale: float | None = None, max_len_k: int | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of packed prompts: q [tokens, heads, head_dim], k and v [keys, kv_heads, head_dim] (f32, f16 or bf16, head_dim 64, 128 or 256) ->
    [tokens, heads, head_dim].  Prompt b has tokens starts[b] .. starts[b + 1] - 1 (int32 [prompts + 1] on the GPU; None: one prompt) and keys by
    ``starts_k`` (None: as its tokens).  ``causal``: the last query sees the last key, the one before it one key less, and so on, so that a
    prompt with more keys than tokens is a chunk behind a past.  A query without any key gives zeros; rows that belong to no prompt are not
    written (without ``out`` they hold anything).  ``max_len_k``: the longest prompt's keys where the caller knows them; only the division of the work goes by it."""
    dtype, shape, k_shape, index = q.dtype, q.shape, k.shape, q.get_device()
    fn = _attentions.get(dtype) or _fn(_attentions, "izwi_qmm_prompt_attention", dtype)
    if fn is None or len(shape) != 3 or index < 0:
        _refuse("prompt_attention: q [tokens, heads, head_dim] of f32, f16 or bf16 on a GPU expected")
    tokens, heads, d = shape
    if (len(k_shape) != 3 or v.shape != k_shape or k_shape[2] != d or k.dtype is not dtype or v.dtype is not dtype or k.get_device() != index
            or v.get_device() != index or not k_shape[1] or heads % k_shape[1]):
        _refuse(f"prompt_attention: k and v [keys, kv_heads, {d}] of q's type and device expected, {heads} heads a multiple of theirs")
    keys, kv_heads, _ = k_shape
    prompts, cu_q, cu_k = 1, 0, 0
    if starts is not None:
        prompts = len(starts) - 1 if starts.dim() == 1 else -1
        if starts.dtype is not _i32 or prompts < 0 or starts.get_device() != index or not starts.is_contiguous():
            _refuse(f"prompt_attention: starts as a contiguous int32 tensor of prompts + 1 on GPU {index} expected")
        cu_q = cu_k = starts.data_ptr()
        if starts_k is not None:
            if starts_k.dtype is not _i32 or starts_k.shape != (prompts + 1,) or starts_k.get_device() != index or not starts_k.is_contiguous():
                _refuse(f"prompt_attention: starts_k as a contiguous int32 tensor of {prompts + 1} on GPU {index} expected")
            cu_k = starts_k.data_ptr()
        elif keys != tokens:
            _refuse(f"prompt_attention: {keys} keys for {tokens} tokens need starts_k")
    elif starts_k is not None:
        _refuse("prompt_attention: starts_k comes with starts")
    if max_len_k is None:
        max_len_k = keys
    elif max_len_k < 0:
        _refuse(f"prompt_attention: max_len_k {max_len_k}")
    if index != _current_device():
        with torch.cuda.device(index):
            return prompt_attention(q, k, v, starts, starts_k, causal, scale, max_len_k, out)
    row = kv_heads * d
    q_step = heads * d if q.is_contiguous() else _stride(q, "prompt_attention: q")
    k_step = row if k.is_contiguous() else _stride(k, "prompt_attention: k")
    v_step = row if v.is_contiguous() else _stride(v, "prompt_attention: v")
    if out is None:
        out, out_step = torch.empty_like(q), heads * d  # (contiguous, whether q is a part of wider rows or not)
    else:
        if out.dtype is not dtype or out.shape != shape or out.get_device() != index:
            _refuse("prompt_attention: out has to be as q is")
        out_step = _stride(out, "prompt_attention: out")
    rc = fn(q.data_ptr(), q_step, k.data_ptr(), k_step, v.data_ptr(), v_step, cu_q, cu_k, prompts, tokens, keys, max_len_k, heads, kv_heads, d, bool(causal),
            d ** -0.5 if scale is None else scale, out.data_ptr(), out_step, _raw_stream(index))
    if rc:
        check(rc)
    return out
