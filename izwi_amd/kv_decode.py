"""Several continuations of one prompt: the quantized key / value cache, the attention that reads it and the step of
beam search, over the C ABI of include/izwi_decode_ops.h.

``prompts`` prompts of ``beams`` sequences each decode together, sequence b belongs to prompt b // beams.  What the sequences of a
prompt share stands once, in a cache with a slot per prompt; what each adds stands in a cache with a slot per sequence, and
a beam's *lineage* says for each of its positions which beam of the prompt wrote it, so that a beam that takes over another's
history copies a row of bytes instead of keys and values.  The reference keeps such caches as pages of 8- or 4-bit values
(models/shared/attention/paged.rs:160-342) and gathers them for its eager attention; here the attention reads them in place.

    prompt = QuantizedKvCache(KvCacheType.Q8_0, prompts, kv_heads, prompt_capacity, head_dim)
    answers = QuantizedKvCache(KvCacheType.Q8_0, prompts * beams, kv_heads, answer_capacity, head_dim)
    prompt.append(k, v, starts)                                   # once, k / v [prompts, tokens, kv_heads, head_dim]
    lineage, lens = answers.new_lineage(beams), zeros of int32    # every beam begins with positions of its own
    # a step: per layer append and attend, then pick (the lineage is every layer's)
    answers.append(k, v, lens)                                    # k / v [prompts * beams, 1, kv_heads, head_dim]
    out = shared_prefix_attention(q, answers, lens + 1, prefix=prompt, prefix_lens=prompt_lens, lineage=lineage)
    picked = beam_select(logits, scores, lineage=lineage, lens=lens + 1)

Everything runs on the current stream; nothing waits for the device.  Arguments that do not fit raise ``QmmError``."""
from __future__ import annotations

import enum
from typing import NamedTuple

import torch

from .capi import QmmError, check, lib
from .qmatmul import _current_device, _raw_stream

_PAD = 32  # positions of a cache, and bytes of a lineage row, come in multiples of this


class KvCacheType(enum.IntEnum):
    """Formats of a cache, by their ggml ids: blocks of 32 values with an f16 scale, 8 or 4 bits a value."""
    Q4_0 = 2
    Q8_0 = 8


def _refuse(what: str):
    raise QmmError(-1, what)


# (What a call checks and looks up is paid for once per layer and token: device numbers are compared instead of devices, and the
# library's functions are looked up once.)
_f32, _f16, _i32, _u8 = torch.float32, torch.float16, torch.int32, torch.uint8
_fns = {}


def _fn(name: str):
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(lib(), f"izwi_decode_{name}")
    return fn


def _ints(t, n: int, index: int, what: str) -> int:
    if t is None:
        return 0
    if t.dtype is not _i32 or t.get_device() != index or t.shape != (n,) or not t.is_contiguous():
        _refuse(f"{what}: a contiguous int32 tensor of {n} on GPU {index} expected")
    return t.data_ptr()


def _rows(t, what: str) -> int:
    """Elements from one row of heads to the next, rows being all leading dimensions taken together."""
    shape = t.shape
    heads, d = shape[-2:]
    stride = t.stride()
    if stride[-1] != 1 or (heads > 1 and stride[-2] != d):
        _refuse(f"{what}: heads of a row must be contiguous")
    step = None
    for size, at in zip(reversed(shape[:-2]), reversed(stride[:-2])):
        if size == 1:
            continue
        if step is None:
            step, count = at, size
        elif at != step * count:
            _refuse(f"{what}: rows must be equally far apart")
        else:
            count *= size
    if step is None:  # one row
        return heads * d
    if step < heads * d:
        _refuse(f"{what}: rows overlap")
    return step


class QuantizedKvCache:
    """Keys and values of ``slots`` sequences, up to ``capacity`` positions of ``kv_heads`` heads each, quantized as they
    are written.  head_dim 64, 128 or 256."""

    def __init__(self, dtype: KvCacheType, slots: int, kv_heads: int, capacity: int, head_dim: int, device="cuda"):
        self.dtype, self.slots, self.kv_heads, self.capacity, self.head_dim = KvCacheType(dtype), slots, kv_heads, capacity, head_dim
        if torch.device(device).type != "cuda":
            _refuse(f"QuantizedKvCache: a GPU expected, not {device}")
        nbytes = lib().izwi_decode_kv_cache_bytes(int(dtype), slots, kv_heads, capacity, head_dim)
        if nbytes == 0:
            raise QmmError(-1, lib().izwi_qmm_last_error().decode("utf-8", "replace"))
        self.buffer = torch.empty(nbytes, dtype=torch.uint8, device=device)
        self.device = self.buffer.device
        self._index, self._ptr, self._type, self._row = self.buffer.get_device(), self.buffer.data_ptr(), int(dtype), kv_heads * head_dim
        self._lineage_shape = (slots, -(-capacity // _PAD) * _PAD)

    def new_lineage(self, beams: int | None = None) -> torch.Tensor:
        """Lineage rows of all slots, [slots, capacity rounded up to 32] uint8.  With ``beams`` sequences a prompt every position is its
        own slot's, as it has to be for what is written before the first ``beam_select`` (which names the beams from then on).
        Without, zeros: every position is the first beam's of the prompt, which is right where that beam's first token is all beams'."""
        rows = torch.zeros(self._lineage_shape, dtype=torch.uint8, device=self.device)
        if beams is not None:
            if not 0 < beams <= 255 or self.slots % beams:
                _refuse(f"new_lineage: {beams} beams in {self.slots} slots (at most 255, a divisor)")
            rows += (torch.arange(self.slots, device=self.device) % beams).to(torch.uint8).unsqueeze(1)
        return rows

    def append(self, k: torch.Tensor, v: torch.Tensor, starts: torch.Tensor, counts: torch.Tensor | None = None, first_slot: int = 0) -> None:
        """k, v [sequences, tokens, kv_heads, head_dim] (f32 or f16; rows may be parts of wider ones): token t of
        sequence b goes to position starts[b] + t of slot first_slot + b, for t < counts[b].  What lies outside the
        capacity is left out."""
        dtype, shape, index = k.dtype, k.shape, self._index
        if (dtype is not _f32 and dtype is not _f16 or v.dtype is not dtype or len(shape) != 4 or v.shape != shape or shape[2] != self.kv_heads
                or shape[3] != self.head_dim or k.get_device() != index or v.get_device() != index):
            _refuse(f"append: k and v [sequences, tokens, {self.kv_heads}, {self.head_dim}] of f32 or f16 on {self.device} expected")
        if index != _current_device():
            with torch.cuda.device(index):
                return self.append(k, v, starts, counts, first_slot)
        batch = shape[0]
        rc = _fn("kv_append_f32" if dtype is _f32 else "kv_append_f16")(
            self._type, k.data_ptr(), v.data_ptr(), self._row if k.is_contiguous() else _rows(k, "append: k"),
            self._row if v.is_contiguous() else _rows(v, "append: v"), _ints(starts, batch, index, "append: starts"),
            _ints(counts, batch, index, "append: counts"), batch, shape[1], first_slot, self.slots, self.kv_heads, self.capacity, self.head_dim, self._ptr,
            _raw_stream(index))
        if rc:
            check(rc)

    def read(self, starts: torch.Tensor, tokens: int, counts: torch.Tensor | None = None, first_slot: int = 0, lineage: torch.Tensor | None = None,
             beams: int = 1, dtype: torch.dtype = torch.float32):
        """(k, v) [sequences, tokens, kv_heads, head_dim]: the values that positions starts[b] .. starts[b] + tokens - 1 of slots
        first_slot, .. stand for; zeros from counts[b] on and outside the capacity.  With ``lineage`` a position comes from
        the slot of the beam that wrote it (``beams`` slots a prompt)."""
        if dtype is not _f32 and dtype is not _f16 or tokens < 0:
            _refuse("read: f32 or f16, and a number of tokens, expected")
        index = self._index
        if index != _current_device():
            with torch.cuda.device(index):
                return self.read(starts, tokens, counts, first_slot, lineage, beams, dtype)
        batch = starts.shape[0]
        at, until = _ints(starts, batch, index, "read: starts"), _ints(counts, batch, index, "read: counts")
        k = torch.empty((batch, tokens, self.kv_heads, self.head_dim), dtype=dtype, device=self.device)
        v = torch.empty_like(k)
        rc = _fn("kv_read_f32" if dtype is _f32 else "kv_read_f16")(
            self._type, self._ptr, self.slots, self.kv_heads, self.capacity, self.head_dim, 0 if lineage is None else self._lineage(lineage, "read"), beams,
            at, until, batch, tokens, first_slot, k.data_ptr(), v.data_ptr(), _raw_stream(index))
        if rc:
            check(rc)
        return k, v

    def _lineage(self, lineage, what: str) -> int:
        if (lineage.dtype is not _u8 or lineage.get_device() != self._index or lineage.shape != self._lineage_shape or not lineage.is_contiguous()):
            _refuse(f"{what}: lineage as new_lineage() makes it expected")
        return lineage.data_ptr()


def shared_prefix_attention(q: torch.Tensor, cache: QuantizedKvCache | None, lens: torch.Tensor | None, prefix: QuantizedKvCache | None = None,
                            prefix_lens: torch.Tensor | None = None, lineage: torch.Tensor | None = None, beams: int | None = None,
                            scale: float | None = None, max_len: int | None = None, max_prefix_len: int | None = None) -> torch.Tensor:
    """Attention of one new token per sequence: q [sequences, heads, head_dim] (f32 or f16) over positions 0 ..
    prefix_lens[b // beams] - 1 of its prompt's slot of ``prefix`` and 0 .. lens[b] - 1 of its own slot of ``cache`` (found by ``lineage``
    if given).  Either cache may be None.  A sequence without any position gives zeros, a NaN that it reads NaN (a value's: in its block of
    32).  ``beams``: sequences per prompt,
    by default sequences // len(prefix_lens), or all of them without a prefix.  ``max_len`` and ``max_prefix_len`` bound the lengths where
    the caller knows them better than the capacities: the work is shared out by them.  Returns [sequences, heads, head_dim]."""
    dtype, shape = q.dtype, q.shape
    if dtype is not _f32 and dtype is not _f16 or len(shape) != 3:
        _refuse("shared_prefix_attention: q [sequences, heads, head_dim] of f32 or f16 expected")
    one = cache if cache is not None else prefix
    if one is None:
        _refuse("shared_prefix_attention: neither a cache nor a prefix")
    index = one._index
    if prefix is not None and cache is not None and (prefix._type != cache._type or prefix.kv_heads != cache.kv_heads or prefix.head_dim != cache.head_dim
                                                     or prefix._index != index):
        _refuse("shared_prefix_attention: the two caches differ in format, heads or device")
    batch, heads, d = shape
    if (prefix is None) != (prefix_lens is None) or (cache is None) != (lens is None) or (lineage is not None and cache is None):
        _refuse("shared_prefix_attention: a cache and its lengths come together, lineage with a cache")
    if beams is None:
        beams = (batch if prefix is None else batch // max(1, prefix_lens.shape[0])) or 1
    if beams <= 0 or batch % beams or d != one.head_dim or q.get_device() != index:
        _refuse(f"shared_prefix_attention: {batch} sequences of head_dim {d}, {beams} a prompt, on a cache of head_dim {one.head_dim} on {one.device}")
    if index != _current_device():
        with torch.cuda.device(index):
            return shared_prefix_attention(q, cache, lens, prefix, prefix_lens, lineage, beams, scale, max_len, max_prefix_len)
    p = p_slots = p_capacity = p_lens = c = c_slots = c_capacity = c_lens = c_lineage = 0
    if prefix is not None:
        p, p_slots, p_capacity = prefix._ptr, prefix.slots, prefix.capacity
        p_lens = _ints(prefix_lens, batch // beams, index, "shared_prefix_attention: prefix_lens")
    if cache is not None:
        c, c_slots, c_capacity, c_lens = cache._ptr, cache.slots, cache.capacity, _ints(lens, batch, index, "shared_prefix_attention: lens")
        if lineage is not None:
            c_lineage = cache._lineage(lineage, "shared_prefix_attention")
    whole = q.is_contiguous()
    out = torch.empty_like(q) if whole else torch.empty(shape, dtype=dtype, device=q.device)
    rc = _fn("shared_attention_f32" if dtype is _f32 else "shared_attention_f16")(
        one._type, q.data_ptr(), heads * d if whole else _rows(q, "shared_prefix_attention: q"), batch, beams, heads, one.kv_heads, d, p, p_slots, p_capacity,
        p_lens, p_capacity if max_prefix_len is None else max_prefix_len, c, c_slots, c_capacity, c_lens, c_capacity if max_len is None else max_len,
        c_lineage, d ** -0.5 if scale is None else scale, out.data_ptr(), _raw_stream(index))
    if rc:
        check(rc)
    return out


class BeamStep(NamedTuple):
    """What a step of beam search leaves, [prompts, beams] each, best first; lineage for the next step (None without)."""
    tokens: torch.Tensor    # int32
    parents: torch.Tensor   # int32: the beam that each new one continues
    scores: torch.Tensor    # f32: sums of log-probabilities
    finished: torch.Tensor  # uint8
    lineage: torch.Tensor | None


def beam_select(logits: torch.Tensor, scores: torch.Tensor, finished: torch.Tensor | None = None, eos_token: int | None = None,
                lineage: torch.Tensor | None = None, lens: torch.Tensor | None = None, out_lineage: torch.Tensor | None = None) -> BeamStep:
    """One step of beam search on the device: logits [prompts, beams, vocab] f32, scores [prompts, beams] f32 (a first step starts
    from 0, -inf, -inf, ..).  The best ``beams`` of beams * vocab candidates scores[w] + log_softmax(logits[w])[t], equal ones by
    rising w * vocab + t; a beam marked in ``finished`` (uint8) keeps its score and its one candidate ``eos_token``.  ``lineage``
    [prompts * beams, n] uint8 and ``lens`` int32 [prompts * beams]: the new beams' lineage is their parents', with their own index
    at position lens[parent], where their next key and value go; into ``out_lineage`` (it may be ``lineage``) or a new tensor."""
    shape = logits.shape
    if len(shape) != 3 or logits.dtype is not _f32 or not logits.is_contiguous() or not logits.is_cuda:
        _refuse("beam_select: contiguous f32 logits [prompts, beams, vocab] on a GPU expected")
    prompts, beams, vocab = shape
    rows, index = shape[:2], logits.get_device()
    if scores.dtype is not _f32 or scores.shape != rows or not scores.is_contiguous() or scores.get_device() != index:
        _refuse(f"beam_select: scores [{prompts}, {beams}] of f32 expected")
    if finished is not None:
        if eos_token is None:
            _refuse("beam_select: finished beams need an eos_token")
        if finished.dtype is not _u8 or finished.shape != rows or not finished.is_contiguous() or finished.get_device() != index:
            _refuse(f"beam_select: finished [{prompts}, {beams}] of uint8 expected")
    if (lineage is None) != (lens is None) or (lineage is None and out_lineage is not None):
        _refuse("beam_select: lineage and lens come together")
    if index != _current_device():
        with torch.cuda.device(index):
            return beam_select(logits, scores, finished, eos_token, lineage, lens, out_lineage)
    capacity = from_lineage = to_lineage = at = 0
    if lineage is not None:
        if out_lineage is None:
            out_lineage = torch.empty_like(lineage)
        capacity = lineage.shape[-1]
        for t in (lineage, out_lineage):
            if t.dtype is not _u8 or t.shape != (prompts * beams, capacity) or capacity % _PAD or not t.is_contiguous() or t.get_device() != index:
                _refuse("beam_select: lineage rows as QuantizedKvCache.new_lineage() makes them expected")
        from_lineage, to_lineage, at = lineage.data_ptr(), out_lineage.data_ptr(), _ints(lens, prompts * beams, index, "beam_select: lens")
    tokens = torch.empty_like(scores, dtype=_i32)
    parents, scores_out = torch.empty_like(tokens), torch.empty_like(scores)
    finished_out = torch.empty_like(scores, dtype=_u8)
    rc = _fn("beam_select_f32")(logits.data_ptr(), prompts, beams, vocab, scores.data_ptr(), 0 if finished is None else finished.data_ptr(),
                                -1 if eos_token is None else eos_token, tokens.data_ptr(), parents.data_ptr(), scores_out.data_ptr(), finished_out.data_ptr(),
                                from_lineage, capacity, at, to_lineage, _raw_stream(index))
    if rc:
        check(rc)
    return BeamStep(tokens, parents, scores_out, finished_out, out_lineage)
