"""The operators of decoding several continuations of one prompt, as cases that can be timed and compared.

``cache``   rows of new keys and values are quantized into a cache and read back from it: one decoded token, the
            tokens of a batch, a prompt (ragged: sequences of different lengths in one call).
``attend``  attention of one new token per sequence over the quantized cache: positions of a prompt that several
            sequences share, then each sequence's own positions, which beams find through their lineage (the beam
            that wrote each position).
``beam``    one step of beam search: log-probabilities of the whole vocabulary added to the beams' scores, the best
            of beams times vocabulary, the beams' lineage reordered to follow.

Heads are 16 or 32 on 8 of 128 elements (Qwen3-0.6B and Qwen3-8B), vocabulary 151936; other head sizes, odd
lengths and small vocabularies (codec books) are drawn.  Keys have a few channels of larger magnitude, as
trained models' keys have.
"""
from __future__ import annotations

import functools
import math
import random

import torch

own = False

TYPES = ("q8_0", "q4_0")
FLOATS = {"f32": torch.float32, "f16": torch.float16}
BLOCK = 32
PAD = 32  # positions of a lineage row: the capacity, rounded up


def listed():
    return [
        # one token of one sequence into the 8-bit cache and back: the smallest call, all latency
        {"name": "cache_q8_0_f32_token", "kind": "cache", "quant": "q8_0", "float": "f32", "batch": 1, "tokens": 1, "start": 299, "kv": 8, "d": 128},
        # a prompt of odd length, 4-bit cache, half precision
        {"name": "cache_q4_0_f16_prompt", "kind": "cache", "quant": "q4_0", "float": "f16", "batch": 1, "tokens": 2051, "start": 0, "kv": 8, "d": 128},
        # sixteen ragged prompts at once
        {"name": "cache_q8_0_f32_prompts", "kind": "cache", "quant": "q8_0", "float": "f32", "batch": 16, "tokens": 1024, "start": 77, "kv": 8, "d": 128},
        # one sequence, short context, nothing shared: speech decoding with the small model
        {"name": "attend_q8_0_f32_one", "kind": "attend", "quant": "q8_0", "float": "f32", "heads": 16, "kv": 8, "d": 128, "prompts": 1, "width": 1,
         "prefix": 0, "suffix": 300, "lineage": False},
        # eight beams on a chat prompt, 65 tokens into the answer
        {"name": "attend_q8_0_f32_beams8", "kind": "attend", "quant": "q8_0", "float": "f32", "heads": 32, "kv": 8, "d": 128, "prompts": 1, "width": 8,
         "prefix": 1501, "suffix": 65, "lineage": True},
        # 64 conversations behind one system prompt, each with its own ragged turn, 4-bit cache
        {"name": "attend_q4_0_f16_batch64", "kind": "attend", "quant": "q4_0", "float": "f16", "heads": 32, "kv": 8, "d": 128, "prompts": 1, "width": 64,
         "prefix": 8192, "suffix": 250, "lineage": False},
        # 32 unrelated sequences with long ragged histories: ordinary batched decode over the quantized cache
        {"name": "attend_q8_0_f32_batch32", "kind": "attend", "quant": "q8_0", "float": "f32", "heads": 32, "kv": 8, "d": 128, "prompts": 32, "width": 1,
         "prefix": 4001, "suffix": 0, "lineage": False},
        # one very long document, sixteen candidate answers: the largest
        {"name": "attend_q8_0_f32_long", "kind": "attend", "quant": "q8_0", "float": "f32", "heads": 32, "kv": 8, "d": 128, "prompts": 1, "width": 16,
         "prefix": 131072, "suffix": 40, "lineage": True},
        # one long sequence, 4-bit cache, nothing shared
        {"name": "attend_q4_0_f32_solo", "kind": "attend", "quant": "q4_0", "float": "f32", "heads": 32, "kv": 8, "d": 128, "prompts": 1, "width": 1,
         "prefix": 0, "suffix": 32700, "lineage": False},
        # two beams over a codec book of odd size: all latency
        {"name": "beam_w2_codec", "kind": "beam", "prompts": 1, "width": 2, "vocab": 2051, "suffix": 40},
        # four beams of one answer over the model's vocabulary
        {"name": "beam_w4_vocab", "kind": "beam", "prompts": 1, "width": 4, "vocab": 151936, "suffix": 120},
        # sixteen prompts of eight beams at once
        {"name": "beam_w8_prompts16", "kind": "beam", "prompts": 16, "width": 8, "vocab": 151936, "suffix": 500},
    ]


def _spread(rng, low, high):
    """A whole number, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    kind = rng.choice(("cache", "attend", "attend", "beam"))
    if kind == "beam":
        prompts, width = _spread(rng, 1, 16), _spread(rng, 1, 32)
        vocab = _spread(rng, max(64, width), min(151936, 128 * 151936 // (prompts * width)))
        return {"kind": kind, "prompts": prompts, "width": width, "vocab": vocab, "suffix": _spread(rng, 1, 1000)}
    quant, fl = rng.choice(TYPES), rng.choice(("f32", "f16"))
    kv, d = rng.choice((1, 2, 4, 8, 8)), rng.choice((64, 128, 128, 256))
    if kind == "cache":
        rows = max(1, _spread(rng, 1, 12000) * 1024 // max(1024, kv * d))
        batch = _spread(rng, 1, min(rows, 64))
        return {"kind": kind, "quant": quant, "float": fl, "batch": batch, "tokens": max(1, rows // batch), "start": rng.randrange(100), "kv": kv, "d": d}
    group, prompts = rng.choice((1, 2, 3, 4, 4, 8)), _spread(rng, 1, 32)
    width = _spread(rng, 1, 64)
    lineage = width <= 32 and rng.random() < 0.5
    # (no more query rows times positions, and no more cache, than the largest listed case)
    cache = 131072 * 8 * 128 // (kv * d)
    prefix = _spread(rng, 16, max(16, min(131072, cache // (2 * prompts), 131072 * 512 * 128 // (2 * prompts * width * kv * group * d))))
    suffix = _spread(rng, 1, max(1, min(1024, cache // (2 * prompts * width))))
    if rng.random() < 0.25:
        prefix = 0
    return {"kind": kind, "quant": quant, "float": fl, "heads": kv * group, "kv": kv, "d": d, "prompts": prompts, "width": width, "prefix": prefix,
            "suffix": suffix, "lineage": lineage}


# --- what a case's name stands for: lengths and lineages, the same for every seed ---------------------------


def _counts(case):
    """New rows per sequence of a cache call: the first takes all, the others fewer."""
    t = case["tokens"]
    return [t - (b * 37) % (t // 2 + 1) for b in range(case["batch"])]


def _prefix_lens(case):
    p = case["prefix"]
    return [p - (g * 101) % (p // 2 + 1) for g in range(case["prompts"])]


def _suffix_lens(case):
    """Beams of a prompt are equally long; other sequences are ragged, some of them still empty."""
    s, w = case["suffix"], case["width"]
    if case["lineage"]:
        return [s - g % (s // 2 + 1) for g in range(case["prompts"]) for _ in range(w)]
    return [s - (b * 53) % (s + 1) if case["prompts"] * w > 1 else s for b in range(case["prompts"] * w)]


@functools.lru_cache(maxsize=64)
def _lineage(prompts, width, length):
    """Beams [prompts][width][length] that wrote the positions of each beam, as that many steps of search leave them."""
    rng = random.Random(length)
    out = []
    for _ in range(prompts):
        parents = [[min(rng.randrange(width), rng.randrange(width)) for _ in range(width)] for _ in range(length)]
        beams, writers = [], list(range(width))
        for step in reversed(range(length)):  # beam w as it stands now: who wrote its last position, the one before, ..
            beams.append(writers)
            writers = [parents[step][w] for w in writers]
        out.append([[beams[length - 1 - p][w] for p in range(length)] for w in range(width)])
    return out


def _padded(n):
    return -(-n // PAD) * PAD


def _lineage_tensor(prompts, width, length, capacity):
    rows = torch.zeros(prompts * width, _padded(capacity), dtype=torch.uint8)
    if length:
        rows[:, :length] = torch.tensor(_lineage(prompts, width, length), dtype=torch.uint8).view(prompts * width, length)
    return rows.cuda()


# --- the cache in its plain form: whole numbers and half-precision scales, 32 values a block ------------------


def _quantize(x, quant):
    """[..., d] -> quants int8 [..., d], scales f16 [..., d / 32].  8 bits: scale = the block's largest magnitude / 127,
    quant = value * (1 / scale), halves away from zero.  4 bits: scale = the (first) value of largest magnitude / -8,
    quant = floor(value * (1 / scale) + 8.5), at most 15, less 8.  Every step is rounded to 32 bits, then the scale to 16; a
    block whose scale has no 16-bit value, or that holds an infinity or NaN, is NaN throughout.
    (Quotients and sums are taken in 64 bits and rounded once more, which gives the 32-bit results.)"""
    b = x.float().unflatten(-1, (-1, BLOCK))
    mag = b.abs()
    amax = mag.amax(-1, keepdim=True)
    if quant == "q8_0":
        scale = (amax.double() / torch.full_like(amax, 127.0).double()).float()
    else:
        far = b.gather(-1, mag.argmax(-1, keepdim=True))
        scale = far / -8.0
    half = scale.half()
    bad = ~torch.isfinite(amax) | ~torch.isfinite(half)
    dead = bad | (half == 0)
    inv = torch.where(dead, torch.zeros_like(scale), (1.0 / torch.where(dead, torch.ones_like(scale), scale).double()).float())
    v = torch.where(bad, torch.zeros_like(b), b) * inv
    if quant == "q8_0":
        q = torch.trunc(v.double() + torch.copysign(torch.full_like(v, 0.5), v).double())
    else:
        q = torch.trunc((v.double() + 8.5).float()).clamp(max=15.0) - 8.0
    q = torch.where(dead, torch.zeros_like(q), q.to(v.dtype))
    half = torch.where(bad, torch.full_like(half, math.nan), half)
    return q.to(torch.int8).flatten(-2), half.squeeze(-1)


def _values(quants, scales):
    return (quants.unflatten(-1, (-1, BLOCK)).float() * scales.float().unsqueeze(-1)).flatten(-2)


class _PlainCache:
    """Slots of positions of heads: [slots, capacity + 1, kv heads, d]; the last position takes what is not to be kept."""

    def __init__(self, quant, slots, kv, capacity, d):
        self.quant, self.capacity = quant, capacity
        self.quants = torch.zeros(2, slots, capacity + 1, kv, d, dtype=torch.int8, device="cuda")
        self.scales = torch.zeros(2, slots, capacity + 1, kv, d // BLOCK, dtype=torch.float16, device="cuda")

    def append(self, k, v, starts, counts):
        t = torch.arange(k.shape[1], device="cuda")
        at = starts.long().unsqueeze(1) + t
        at = torch.where((t < counts.unsqueeze(1)) & (at < self.capacity), at, self.capacity)
        slot = torch.arange(k.shape[0], device="cuda").unsqueeze(1)
        for i, x in enumerate((k, v)):
            self.quants[i][slot, at], self.scales[i][slot, at] = _quantize(x, self.quant)

    def read(self, starts, counts, tokens, dtype):
        t = torch.arange(tokens, device="cuda")
        at = starts.long().unsqueeze(1) + t
        there = (t < counts.unsqueeze(1)) & (at < self.capacity)
        slot = torch.arange(starts.shape[0], device="cuda").unsqueeze(1)
        at = torch.where(there, at, 0)
        return tuple(torch.where(there[..., None, None], _values(self.quants[i][slot, at], self.scales[i][slot, at]), 0.0).to(dtype) for i in range(2))


# --- states ---------------------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    s = {"case": case}
    if case["kind"] == "beam":
        g, w, n = case["prompts"], case["width"], case["vocab"]
        s["logits"] = randn(g, w, n, std=2.5)
        s["scores"] = (-torch.rand(g, w, device="cuda", generator=gen) * 8 - 0.3 * case["suffix"]).sort(1, descending=True).values
        s["finished"] = (torch.rand(g, w, device="cuda", generator=gen) < 0.1).to(torch.uint8)
        s["eos"] = n // 2
        s["lens"] = torch.full((g * w,), case["suffix"], dtype=torch.int32, device="cuda")
        s["lineage"] = _lineage_tensor(g, w, case["suffix"], case["suffix"] + 1)
        return s

    kv, d, dtype = case["kv"], case["d"], FLOATS[case["float"]]

    def keys_values(slots, length):
        gains = torch.exp(randn(2, kv, d, std=0.4))
        gains[0] *= 1 + 7 * (torch.rand(kv, d, device="cuda", generator=gen) < 0.03)
        return tuple((randn(slots, length, kv, d) * gains[i]).to(dtype) for i in range(2))

    def cache(slots, capacity):
        if not own:
            return _PlainCache(case["quant"], slots, kv, capacity, d)
        import izwi_amd
        return izwi_amd.QuantizedKvCache(getattr(izwi_amd.KvCacheType, case["quant"].upper()), slots, kv, capacity, d)

    def filled(slots, lens):
        """A cache whose slots hold `lens` positions each."""
        made = cache(slots, max(lens))
        step = max(1, (1 << 26) // (slots * kv * d))
        for at in range(0, max(lens), step):
            length = min(step, max(lens) - at)
            made.append(*keys_values(slots, length), ints([at] * slots), ints([max(0, min(length, n - at)) for n in lens]))
        return made

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["kind"] == "cache":
        s["cache"] = cache(case["batch"], case["start"] + case["tokens"])
        s["k"], s["v"] = keys_values(case["batch"], case["tokens"])
        s["starts"], s["counts"] = ints([case["start"]] * case["batch"]), ints(_counts(case))
        return s
    batch = case["prompts"] * case["width"]
    s["q"] = randn(batch, case["heads"], d).to(dtype)
    s["scale"] = d ** -0.5
    s["prefix"] = s["prefix_lens"] = s["lineage"] = s["cache"] = s["lens"] = None
    if case["prefix"]:
        lens = _prefix_lens(case)
        s["prefix"], s["prefix_lens"], s["max_prefix"] = filled(case["prompts"], lens), ints(lens), max(lens)
    if case["suffix"]:
        lens = _suffix_lens(case)
        s["cache"], s["lens"], s["max_len"] = filled(batch, lens), ints(lens), max(lens)
        if case["lineage"]:
            s["lineage"] = _lineage_tensor(case["prompts"], case["width"], case["suffix"], case["suffix"])
    return s


# --- passes ---------------------------------------------------------------------------------------------------


def run(state):
    return globals()["_run_" + state["case"]["kind"]](state)


def _run_cache(s):
    tokens, dtype = s["case"]["tokens"], s["k"].dtype
    s["cache"].append(s["k"], s["v"], s["starts"], s["counts"])
    if own:
        return s["cache"].read(s["starts"], tokens, s["counts"], dtype=dtype)
    return s["cache"].read(s["starts"], s["counts"], tokens, dtype)


def _run_attend(s):
    if own:
        import izwi_amd
        return izwi_amd.shared_prefix_attention(s["q"], s["cache"], s["lens"], prefix=s["prefix"], prefix_lens=s["prefix_lens"],
                                                lineage=s["lineage"], beams=s["case"]["width"], scale=s["scale"])
    case = s["case"]
    prompts, width, kv, d = case["prompts"], case["width"], case["kv"], case["d"]
    group = case["heads"] // kv
    q = s["q"].float().view(prompts, width, kv, group, d) * s["scale"]
    scores, values = [], []
    if s["prefix"] is not None:
        n = s["max_prefix"]
        k, v = (_values(s["prefix"].quants[i][:, :n], s["prefix"].scales[i][:, :n]).permute(0, 2, 1, 3) for i in range(2))
        rows = q.permute(0, 2, 1, 3, 4).reshape(prompts, kv, width * group, d)
        dots = (rows @ k.transpose(2, 3)).view(prompts, kv, width, group, n).permute(0, 2, 1, 3, 4)
        there = torch.arange(n, device="cuda") < s["prefix_lens"].view(prompts, 1, 1, 1, 1)
        scores.append(torch.where(there, dots, -math.inf))
        values.append(v)
    if s["cache"] is not None:
        n = s["max_len"]
        at = torch.arange(n, device="cuda")
        slot = torch.arange(prompts * width, device="cuda").unsqueeze(1)
        if s["lineage"] is not None:
            slot = slot // width * width + s["lineage"][:, :n].long()
        k, v = (_values(s["cache"].quants[i][slot, at], s["cache"].scales[i][slot, at]).view(prompts, width, n, kv, d).transpose(2, 3) for i in range(2))
        there = (at < s["lens"].unsqueeze(1)).view(prompts, width, 1, 1, n)
        scores.append(torch.where(there, q @ k.transpose(3, 4), -math.inf))
        values.append(v)
    best = functools.reduce(torch.maximum, [x.amax(-1, keepdim=True) for x in scores])
    best = torch.where(best == -math.inf, 0.0, best)
    weights = [torch.exp(x - best) for x in scores]
    total = functools.reduce(torch.add, [x.sum(-1, keepdim=True) for x in weights])
    out = 0.0
    for x, v in zip(weights, values):
        if v.dim() == 4:  # shared by the prompt's sequences
            rows = x.permute(0, 2, 1, 3, 4).reshape(prompts, kv, width * group, x.shape[-1])
            out = out + (rows @ v).view(prompts, kv, width, group, d).permute(0, 2, 1, 3, 4)
        else:
            out = out + x @ v
    out = torch.where(total > 0, out / total, 0.0)
    return out.reshape(prompts * width, case["heads"], d).to(s["q"].dtype)


def _run_beam(s):
    if own:
        import izwi_amd
        picked = izwi_amd.beam_select(s["logits"], s["scores"], finished=s["finished"], eos_token=s["eos"], lineage=s["lineage"], lens=s["lens"])
        return {"tokens": picked.tokens, "parents": picked.parents, "scores": picked.scores, "finished": picked.finished, "lineage": picked.lineage}
    # sums and order in 64 bits: neighbours among 10^6 candidates are closer than a 32-bit sum is exact
    logits, finished = s["logits"].double(), s["finished"].bool()
    prompts, width, n = logits.shape
    top = logits.amax(-1, keepdim=True)
    total = s["scores"].double().unsqueeze(-1) + logits - top - torch.log(torch.exp(logits - top).sum(-1, keepdim=True))
    ended = torch.where(torch.arange(n, device="cuda") == s["eos"], s["scores"].double().unsqueeze(-1), -math.inf)
    total = torch.where(finished.unsqueeze(-1), ended, total).view(prompts, width * n)
    at = torch.sort(total, dim=1, descending=True, stable=True).indices[:, :width]
    parents, tokens = at // n, at % n
    lineage = s["lineage"].view(prompts, width, -1).gather(1, parents.unsqueeze(-1).expand(-1, -1, s["lineage"].shape[1]))
    lens = s["lens"].view(prompts, width).gather(1, parents).long()
    lineage = lineage.scatter(2, lens.unsqueeze(-1), torch.arange(width, device="cuda", dtype=torch.uint8).view(1, width, 1).expand(prompts, width, 1))
    return {"tokens": tokens.int(), "parents": parents.int(), "scores": total.gather(1, at).float(),
            "finished": (finished.gather(1, parents) | (tokens == s["eos"])).to(torch.uint8), "lineage": lineage.view(prompts * width, -1)}


# --- the operators' definition in 64 bits -----------------------------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return globals()["_exact_" + case["kind"]](case, s)


def _exact_cache(case, s):
    """Block by block along the last dimension, after the formats' definition (see _quantize)."""
    out = []
    for x in (s["k"], s["v"]):
        blocks = x.double().reshape(-1, BLOCK)
        far = blocks.gather(1, blocks.abs().max(1).indices.view(-1, 1))
        step = ((far.abs() / 127) if case["quant"] == "q8_0" else far * -0.125).float()
        back = (1 / step.double()).float().double()
        scaled = (blocks * back).float().double()
        if case["quant"] == "q8_0":
            numbers = scaled.sign() * (scaled.abs() + 0.5).floor()
        else:
            numbers = (scaled + 8.5).float().double().floor().clamp(max=15) - 8
        values = torch.where(step.half() == 0, 0.0, numbers * step.half().double()).view(x.shape)
        for b, count in enumerate(_counts(case)):
            values[b, count:] = 0
        out.append(values)
    return tuple(out)


def _exact_attend(case, s):
    width, group, lineage = case["width"], case["heads"] // case["kv"], s["lineage"]
    out = torch.zeros(case["prompts"] * width, case["heads"], case["d"], dtype=torch.float64, device="cuda")
    suffix_lens = _suffix_lens(case) if case["suffix"] else [0] * len(out)
    prefix_lens = _prefix_lens(case) if case["prefix"] else [0] * case["prompts"]

    def rows(cache, i, slot, at, head):
        q, d = cache.quants[i][slot, at, head], cache.scales[i][slot, at, head]
        return q.double() * d.double().repeat_interleave(BLOCK, -1)

    for head in range(case["kv"]):
        for g in range(case["prompts"]):
            shared = [rows(s["prefix"], i, g, slice(0, prefix_lens[g]), head) for i in range(2)] if prefix_lens[g] else None
            for b in range(g * width, (g + 1) * width):
                n = suffix_lens[b]
                parts = [[], []]
                if shared is not None:
                    parts = [[shared[0]], [shared[1]]]
                if n:
                    slot = b if lineage is None else g * width + lineage[b, :n].long()
                    at = slice(0, n) if lineage is None else torch.arange(n, device="cuda")
                    for i in range(2):
                        parts[i].append(rows(s["cache"], i, slot, at, head))
                if parts[0]:
                    q = s["q"][b, head * group : (head + 1) * group].double()
                    p = torch.softmax(torch.cat([q @ k.T for k in parts[0]], 1) * s["scale"], 1).split([len(k) for k in parts[0]], 1)
                    out[b, head * group : (head + 1) * group] = sum(w @ v for w, v in zip(p, parts[1]))
    return out


def _exact_beam(case, s):
    prompts, width, n = case["prompts"], case["width"], case["vocab"]
    got = {"tokens": [], "parents": [], "scores": [], "finished": [], "lineage": []}
    for g in range(prompts):
        picks = []
        for w in range(width):
            score = float(s["scores"][g, w])
            if s["finished"][g, w]:
                picks.append((-score, w, s["eos"]))
                continue
            row = torch.log_softmax(s["logits"][g, w].double(), 0) + score
            # (a beam gives `width` at the most; equal values by index: the sort is stable)
            order = torch.sort(row, descending=True, stable=True)
            picks += [(-v, w, t) for v, t in zip(order.values[:width].tolist(), order.indices[:width].tolist())]
        picks.sort()
        for i, (score, w, token) in enumerate(picks[:width]):
            row = s["lineage"][g * width + w].clone()
            row[case["suffix"]] = i
            got["tokens"].append(token)
            got["parents"].append(w)
            got["scores"].append(-score)
            got["finished"].append(int(bool(s["finished"][g, w]) or token == s["eos"]))
            got["lineage"].append(row)
    types = {"tokens": torch.int32, "parents": torch.int32, "scores": torch.float64, "finished": torch.uint8}
    out = {name: torch.tensor(got[name], dtype=t, device="cuda").view(prompts, width) for name, t in types.items()}
    return {**out, "lineage": torch.stack(got["lineage"])}


# --- what a pass cannot do without --------------------------------------------------------------------------------


def work(case):
    if case["kind"] == "beam":
        rows = case["prompts"] * case["width"]
        # a logit is read, its exponential taken and summed (64 bits), compared
        return {"bytes": rows * (4 * case["vocab"] + 2 * _padded(case["suffix"] + 1) + 21), "flops": 20 * rows * case["vocab"]}
    size = FLOATS[case["float"]].itemsize
    per = case["kv"] * case["d"] * (34 / 32 if case["quant"] == "q8_0" else 18 / 32)  # bytes of the keys, or values, of a position
    if case["kind"] == "cache":
        rows = sum(_counts(case))
        out = case["batch"] * case["tokens"]
        return {"bytes": 4 * rows * per + 2 * size * case["kv"] * case["d"] * (rows + out), "flops": 10 * rows * case["kv"] * case["d"]}
    batch, width = case["prompts"] * case["width"], case["width"]
    prefix = _prefix_lens(case) if case["prefix"] else [0] * case["prompts"]
    suffix = _suffix_lens(case) if case["suffix"] else [0] * batch
    held = sum(prefix) + sum(suffix)
    if case["suffix"] and case["lineage"]:  # positions that beams have in common are read once
        beams = _lineage(case["prompts"], width, case["suffix"])
        held = sum(prefix) + sum(len({beams[g][w][p] for w in range(width)}) for g in range(case["prompts"]) for p in range(suffix[g * width]))
    pairs = case["heads"] * (width * sum(prefix) + sum(suffix))
    return {"bytes": 2 * per * held + 2 * size * batch * case["heads"] * case["d"] + (sum(suffix) if case["lineage"] else 0), "flops": 4 * case["d"] * pairs}
