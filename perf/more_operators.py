"""The operators of a prompt's decoder layer between its products, as cases that can be timed and compared.

``rope``    rotary positions of packed tokens, with the heads' RMSNorm in front where the model has one: both layouts,
            part of the head, frequencies scaled for long contexts, rows of their own or parts of a wider q|k|v row.
``attend``  attention over whole prompts: packed sequences of different lengths, causal or not, grouped heads, a chunk of
            new tokens behind a longer past.
``route``   routing of tokens to experts: softmax or sigmoid scores, a bias for the choice, groups of experts, the best
            ``top_k``, weights renormalised and scaled.

Heads are 16 or 32 on 8 of 128 elements (Qwen3-0.6B and Qwen3-8B), 128 experts with the best 8 (Qwen3-30B-A3B); other
head and expert numbers, ragged lengths and every float type are drawn.
"""
from __future__ import annotations

import functools
import math
import random

import torch

own = False

FLOATS = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = 1e-6
BASE = 1e6
SCALINGS = ("none", "linear", "ntk", "llama3", "yarn")
FACTOR, ORIGINAL = 4.0, 8192  # of the scaled frequencies: four times the context that the model was trained on


def listed():
    return [
        # one decoded token: the smallest call, all latency
        {"name": "rope_f32_token", "kind": "rope", "float": "f32", "tokens": 1, "heads": 16, "kv": 8, "d": 128, "rotary": 128, "interleaved": False, "scaling": "none", "norm": True, "packed": False, "far": 300},
        # a prompt's q and k inside the rows of the q|k|v product
        {"name": "rope_bf16_prompt", "kind": "rope", "float": "bf16", "tokens": 2051, "heads": 32, "kv": 8, "d": 128, "rotary": 128, "interleaved": False, "scaling": "none", "norm": True, "packed": True, "far": 2051},
        # half of small heads, interleaved, a context stretched by YaRN
        {"name": "rope_f16_part", "kind": "rope", "float": "f16", "tokens": 777, "heads": 12, "kv": 12, "d": 64, "rotary": 32, "interleaved": True, "scaling": "yarn", "norm": False, "packed": False, "far": 32000},
        # many prompts at once, positions up to a million
        {"name": "rope_f32_far", "kind": "rope", "float": "f32", "tokens": 16384, "heads": 32, "kv": 8, "d": 128, "rotary": 128, "interleaved": False, "scaling": "llama3", "norm": False, "packed": False, "far": 1000000},
        # a short question: latency
        {"name": "attend_f32_short", "kind": "attend", "float": "f32", "batch": 1, "tokens": 37, "past": 0, "heads": 16, "kv": 8, "d": 128, "causal": True, "packed": False},
        # ragged prompts in one call
        {"name": "attend_bf16_prompts", "kind": "attend", "float": "bf16", "batch": 9, "tokens": 1501, "past": 0, "heads": 32, "kv": 8, "d": 128, "causal": True, "packed": True},
        # a long chat history
        {"name": "attend_bf16_long", "kind": "attend", "float": "bf16", "batch": 1, "tokens": 8192, "past": 0, "heads": 32, "kv": 8, "d": 128, "causal": True, "packed": False},
        # clips of an audio encoder: every position sees every other
        {"name": "attend_f16_clips", "kind": "attend", "float": "f16", "batch": 4, "tokens": 1500, "past": 0, "heads": 16, "kv": 16, "d": 64, "causal": False, "packed": False},
        # a few new tokens behind a long past
        {"name": "attend_bf16_chunk", "kind": "attend", "float": "bf16", "batch": 1, "tokens": 17, "past": 30011, "heads": 32, "kv": 8, "d": 128, "causal": True, "packed": False},
        # one decoded token
        {"name": "route_f32_token", "kind": "route", "float": "f32", "tokens": 1, "experts": 128, "top_k": 8, "scoring": "softmax", "bias": False, "groups": 1, "top_groups": 1, "renormalize": False, "scale": 1.0},
        # a chunk of a prompt, experts in groups as on several devices
        {"name": "route_bf16_groups", "kind": "route", "float": "bf16", "tokens": 509, "experts": 256, "top_k": 8, "scoring": "sigmoid", "bias": True, "groups": 8, "top_groups": 4, "renormalize": True, "scale": 2.5},
        # a large batch of prompts
        {"name": "route_f32_many", "kind": "route", "float": "f32", "tokens": 16384, "experts": 128, "top_k": 8, "scoring": "softmax", "bias": True, "groups": 1, "top_groups": 1, "renormalize": True, "scale": 1.0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng: random.Random):
    kind = rng.choice(("rope", "attend", "attend", "route"))
    case = {"kind": kind, "float": rng.choice(tuple(FLOATS))}
    if kind == "rope":
        d = rng.choice((64, 128, 128, 256))
        kv = rng.choice((1, 2, 4, 8, 12))
        case.update(heads=kv * rng.choice((1, 2, 4, 5)), kv=kv, d=d, rotary=rng.choice((d, d, d // 2, d // 4)), interleaved=rng.random() < 0.4,
                    scaling=rng.choice(SCALINGS), norm=rng.random() < 0.5, packed=rng.random() < 0.5, far=_spread(rng, 300, 1000000))
        case["tokens"] = max(1, min(_spread(rng, 1, 16384), 16384 * 40 * 128 // ((case["heads"] + kv) * d)))
        return case
    if kind == "route":
        groups = rng.choice((1, 1, 4, 8))
        experts = groups * _spread(rng, 8, 512 // groups)
        top_groups = rng.randint(1, groups)
        case.update(tokens=max(1, min(_spread(rng, 1, 16384), 16384 * 128 // experts)), experts=experts, top_k=rng.randint(1, min(12, top_groups * experts // groups)),
                    scoring=rng.choice(("softmax", "sigmoid")), bias=rng.random() < 0.6, groups=groups, top_groups=top_groups,
                    renormalize=rng.random() < 0.6, scale=rng.choice((1.0, 2.5)))
        return case
    kv = rng.choice((1, 2, 4, 8))
    case.update(heads=kv * rng.choice((1, 2, 4, 7)), kv=kv, d=rng.choice((64, 128, 128, 256)), causal=rng.random() < 0.7, packed=rng.random() < 0.5,
                batch=_spread(rng, 1, 24))
    # at most a quarter of the longest listed prompt's pairs (f32 takes three times as long for them)
    most = 8192 * 8192 * 32 * 128 // 4 // (case["batch"] * case["heads"] * case["d"])
    case["tokens"] = min(_spread(rng, 1, 4096), int(math.sqrt(most)))
    case["past"] = 0 if rng.random() < 0.6 else _spread(rng, 1, max(2, min(30000, most // case["tokens"] - case["tokens"])))
    return case


def _lens(case):
    """(queries, keys) of each sequence: the first is the longest, the others shorter; a past is as ragged."""
    t, p = case["tokens"], case["past"]
    queries = [t - (b * 211) % (t // 2 + 1) for b in range(case["batch"])]
    return queries, [n + p - (b * 97) % (p // 3 + 1) for b, n in enumerate(queries)]


def _frequencies(case):
    """(angles per position in 64 bits, factor on cosine and sine)"""
    r, kind = case["rotary"], case["scaling"]
    i = torch.arange(r // 2, dtype=torch.float64)
    base = BASE * FACTOR ** (r / (r - 2)) if kind == "ntk" else BASE
    f = base ** (-2.0 * i / r)
    if kind == "linear":
        return f / FACTOR, 1.0
    if kind == "llama3":  # waves longer than the trained context are stretched, those of a quarter of it and less are not
        keep = ((ORIGINAL * f / (2 * math.pi) - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        return f * (keep + (1 - keep) / FACTOR), 1.0
    if kind == "yarn":  # those that turn 32 times in the trained context and more are kept, once and less are stretched
        low, high = (r * math.log(ORIGINAL / (turns * 2 * math.pi)) / (2 * math.log(BASE)) for turns in (32, 1))
        low, high = max(math.floor(low), 0), min(math.ceil(high), r - 1)
        stretch = ((i - low) / (high - low if high > low else 0.001)).clamp(0, 1)
        return f * (1 - stretch + stretch / FACTOR), 0.1 * math.log(FACTOR) + 1.0
    return f, 1.0


# --- states ---------------------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, std=1.0):
        return torch.randn(*shape, device="cuda", generator=gen) * std

    dtype, s = FLOATS[case["float"]], {"case": case}
    if case["kind"] == "route":
        # logits as a router's: of each token's own spread, some experts liked more
        t, n = case["tokens"], case["experts"]
        s["logits"] = (randn(t, n, std=1.5) * torch.exp(randn(t, 1, std=0.3)) + randn(n, std=0.7)).to(dtype)
        s["bias"] = randn(n, std=0.1 if case["scoring"] == "sigmoid" else 0.02) if case["bias"] else None
        return s
    heads, kv, d = case["heads"], case["kv"], case["d"]

    def rows(queries, keys):
        """q, k and v; packed: parts of rows q|k|v (where a sequence has as many of each)"""
        gains = torch.exp(randn(heads + 2 * kv, d, std=0.3))
        gains[: heads + kv] *= 1 + 4 * (torch.rand(heads + kv, d, device="cuda", generator=gen) < 0.03)
        if case["packed"] and queries == keys:
            return (randn(queries, heads + 2 * kv, d) * gains).to(dtype).split((heads, kv, kv), 1)
        return tuple((randn(n, g.shape[0], d) * g).to(dtype) for n, g in zip((queries, keys, keys), gains.split((heads, kv, kv))))

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if case["kind"] == "rope":
        s["q"], s["k"], _ = rows(case["tokens"], case["tokens"])
        first = torch.randint(0, max(1, case["far"] - case["tokens"]), (1,), device="cuda", generator=gen)
        s["positions"] = (first + torch.arange(case["tokens"], device="cuda")).int()
        s["weight"] = (1 + randn(2 * d, std=0.2)).to(dtype) if case["norm"] else None
        frequencies, s["factor"] = _frequencies(case)
        s["frequencies"] = frequencies.cuda()
        if own:
            import izwi_amd
            kinds = {"none": None, "linear": izwi_amd.RopeScaling.linear(FACTOR), "ntk": izwi_amd.RopeScaling.ntk(FACTOR),
                     "llama3": izwi_amd.RopeScaling.llama3(FACTOR, ORIGINAL), "yarn": izwi_amd.RopeScaling.yarn(FACTOR, ORIGINAL)}
            s["rotary"] = izwi_amd.RotaryEmbedding(d, base=BASE, rotary_dim=case["rotary"], interleaved=case["interleaved"], scaling=kinds[case["scaling"]])
        return s
    queries, keys = _lens(case)
    s["q"], s["k"], s["v"] = rows(sum(queries), sum(keys))
    s["cu_q"], s["cu_k"] = (ints([sum(n[:b]) for b in range(len(n) + 1)]) for n in (queries, keys))
    s["max_q"], s["max_k"] = max(queries), max(keys)
    s["scale"] = 1.5 * d ** -0.5  # (trained heads look at fewer positions than random ones)
    return s


# --- passes ---------------------------------------------------------------------------------------------------


def run(state):
    return globals()["_run_" + state["case"]["kind"]](state)


def _run_rope(s):
    if own:
        import izwi_amd
        return izwi_amd.rope_positions(s["q"], s["k"], s["positions"], s["rotary"], qk_weight=s["weight"], eps=EPS)
    case, d, r = s["case"], s["case"]["d"], s["case"]["rotary"]
    angles = s["positions"].double().unsqueeze(1) * s["frequencies"]
    cos, sin = ((t * s["factor"]).float().unsqueeze(1) for t in (torch.cos(angles), torch.sin(angles)))
    weights = (None, None) if s["weight"] is None else s["weight"].float().split(d)
    return tuple(_rotated(x.float(), cos, sin, w, r, case["interleaved"]).to(x.dtype) for x, w in zip((s["q"], s["k"]), weights))


def _rotated(x, cos, sin, weight, r, interleaved):
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    a, b = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., : r // 2], x[..., r // 2 : r])
    a, b = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((turned, x[..., r:]), -1)


def _run_attend(s):
    case = s["case"]
    if own:
        import izwi_amd
        return izwi_amd.prompt_attention(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=case["causal"], scale=s["scale"], max_len_k=s["max_k"])
    group = case["heads"] // case["kv"]
    lens_q, lens_k = s["cu_q"].diff().long(), s["cu_k"].diff().long()

    def padded(x, cu, lens, most):  # [sequences, heads, most, d], zeros behind a sequence's end
        at = torch.arange(most, device="cuda")
        there = at < lens.unsqueeze(1)
        rows = torch.where(there, cu[:-1].long().unsqueeze(1) + at, 0)
        return torch.where(there[..., None, None], x[rows].float(), 0.0).transpose(1, 2).contiguous(), there

    q, real = padded(s["q"], s["cu_q"], lens_q, s["max_q"])
    (k, there), (v, _) = (padded(x, s["cu_k"], lens_k, s["max_k"]) for x in (s["k"], s["v"]))
    k, v = (x.repeat_interleave(group, 1) for x in (k, v))
    seen = there[:, None, None, :]
    if case["causal"]:  # the last query sees the last key
        last = torch.arange(s["max_q"], device="cuda") + (lens_k - lens_q).unsqueeze(1)
        seen = seen & (torch.arange(s["max_k"], device="cuda") <= last[:, None, :, None])
    scores = (q * s["scale"]) @ k.transpose(2, 3).contiguous()
    scores.masked_fill_(~seen, -math.inf)
    best = scores.amax(-1, keepdim=True)
    weights = scores.sub_(torch.where(best == -math.inf, 0.0, best)).exp_()
    total = weights.sum(-1, keepdim=True)
    out = torch.where(total > 0, (weights @ v) / total, 0.0)
    return out.transpose(1, 2)[real].to(s["q"].dtype)


def _run_route(s):
    case = s["case"]
    if own:
        import izwi_amd
        return izwi_amd.moe_route_scored(s["logits"], case["top_k"], scoring=case["scoring"], bias=s["bias"], groups=case["groups"],
                                         top_groups=case["top_groups"], renormalize=case["renormalize"], scale=case["scale"])
    # in 64 bits: neighbours in the order may be closer than 32 bits tell apart
    logits = s["logits"].double()
    if case["scoring"] == "softmax":
        scores = torch.exp(logits - logits.amax(-1, keepdim=True))
        scores = scores / scores.sum(-1, keepdim=True)
    else:
        scores = 1 / (1 + torch.exp(-logits))
    choice = logits if s["bias"] is None else scores + s["bias"].double()  # (without a bias the logits' order is the scores')
    if case["groups"] > 1:
        t, n, g = case["tokens"], case["experts"], case["groups"]
        worth = choice.view(t, g, n // g).sort(dim=-1, descending=True).values[..., : 1 if s["bias"] is None else 2].sum(-1)
        kept = torch.zeros(t, g, dtype=torch.bool, device="cuda")
        kept.scatter_(1, worth.sort(dim=-1, descending=True, stable=True).indices[:, : case["top_groups"]], True)
        choice = torch.where(kept.repeat_interleave(n // g, 1), choice, -math.inf)
    ids = choice.sort(dim=-1, descending=True, stable=True).indices[:, : case["top_k"]]
    weights = scores.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return ids.int(), (weights * case["scale"]).float()


# --- the operators' definition in 64 bits -----------------------------------------------------------------------


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return globals()["_exact_" + case["kind"]](case, s)


def _exact_rope(case, s):
    """As products of complex numbers."""
    r, out = case["rotary"], []
    turn = torch.polar(torch.full_like(s["frequencies"], s["factor"]).expand(case["tokens"], -1), torch.outer(s["positions"].double(), s["frequencies"]))
    for i, x in enumerate((s["q"].double(), s["k"].double())):
        if case["norm"]:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * s["weight"].double()[i * case["d"] : (i + 1) * case["d"]]
        at = torch.arange(r, device="cuda").view(-1, 2) if case["interleaved"] else torch.arange(r, device="cuda").view(2, -1).T
        y, z = x.clone(), torch.complex(x[..., at[:, 0]], x[..., at[:, 1]]) * turn.unsqueeze(1)
        y[..., at[:, 0]], y[..., at[:, 1]] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_attend(case, s):
    """Sequence by sequence, head by head, some rows at a time."""
    group, out = case["heads"] // case["kv"], torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    queries, keys = _lens(case)
    at_q = at_k = 0
    for nq, nk in zip(queries, keys):
        for kv in range(case["kv"]):
            k, v = (x[at_k : at_k + nk, kv].double() for x in (s["k"], s["v"]))
            for head in range(kv * group, (kv + 1) * group):
                for i in range(0, nq, 4096):
                    rows = torch.arange(i, min(nq, i + 4096), device="cuda")
                    scores = s["q"][at_q + rows, head].double() @ k.T * s["scale"]
                    if case["causal"]:
                        scores[torch.arange(nk, device="cuda") > (rows + nk - nq).unsqueeze(1)] = -math.inf
                    out[at_q + rows, head] = torch.softmax(scores, 1) @ v
        at_q, at_k = at_q + nq, at_k + nk
    return out


def _exact_route(case, s):
    logits = s["logits"].double()
    scores = torch.softmax(logits, 1) if case["scoring"] == "softmax" else torch.sigmoid(logits)
    choice = logits.clone() if s["bias"] is None else scores + s["bias"].double()
    size = case["experts"] // case["groups"]
    if case["groups"] > 1:
        parts = choice.unfold(1, size, size)
        worth = parts.amax(-1) if s["bias"] is None else parts.topk(min(2, size), -1).values.sum(-1)
        left = worth.argsort(dim=1, descending=True, stable=True)[:, case["top_groups"] :]
        for column in left.T:
            choice.view(case["tokens"], -1, size)[torch.arange(case["tokens"], device="cuda"), column] = -math.inf
    ids = choice.argsort(dim=1, descending=True, stable=True)[:, : case["top_k"]]
    weights = torch.take_along_dim(scores, ids, 1) * case["scale"]
    return ids.int(), weights / (torch.take_along_dim(scores, ids, 1).sum(1, keepdim=True) if case["renormalize"] else 1.0)


# --- what a pass cannot do without --------------------------------------------------------------------------------


@functools.lru_cache(maxsize=256)
def _pairs(batch, tokens, past, causal):
    """Pairs of a query and a key that it sees, of one head."""
    queries, keys = _lens({"batch": batch, "tokens": tokens, "past": past})
    return sum(nq * nk - (nq * (nq - 1) // 2 if causal else 0) for nq, nk in zip(queries, keys))


def work(case):
    size = FLOATS[case["float"]].itemsize
    if case["kind"] == "rope":
        values = case["tokens"] * (case["heads"] + case["kv"]) * case["d"]
        return {"bytes": 2 * size * values + 4 * case["tokens"], "flops": values * (3 + 4 * case["norm"])}
    if case["kind"] == "route":
        return {"bytes": case["tokens"] * (size * case["experts"] + 8 * case["top_k"]), "flops": 20 * case["tokens"] * case["experts"]}
    queries, keys = _lens(case)
    rows = 2 * sum(queries) * case["heads"] + 2 * sum(keys) * case["kv"]
    return {"bytes": size * case["d"] * rows, "flops": 4 * case["d"] * case["heads"] * _pairs(case["batch"], case["tokens"], case["past"], case["causal"])}
