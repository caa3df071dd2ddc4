"""64-bit restatements of the operators on whole prompts: rotary positions, attention of packed sequences, scored routing."""
import math

import numpy as np


def frequencies(kind, r, base, factor=1.0, original=0.0, low=0.0, high=0.0):
    """Pair by pair, as the definitions go."""
    out, m = [], 1.0
    if kind == "ntk":
        base = base * factor ** (r / (r - 2))
    for i in range(r // 2):
        f = base ** (-2 * i / r)
        if kind == "linear":
            f /= factor
        elif kind == "llama3":
            wave = 2 * math.pi / f
            if wave >= original / low:
                f /= factor
            elif wave > original / high:
                keep = (original / wave - low) / (high - low)
                f = (1 - keep) * f / factor + keep * f
        elif kind == "yarn":
            first, last = (r * math.log(original / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (high, low))
            first, last = max(math.floor(first), 0), min(math.ceil(last), r - 1)
            if last <= first:
                last = first + 0.001
            ramp = min(max((i - first) / (last - first), 0), 1)
            f = f * (1 - ramp) + f / factor * ramp
        out.append(f)
    if kind == "yarn":
        m = 0.1 * math.log(factor) + 1
    return np.array(out), m


def rope(x, positions, freqs, factor, interleaved, weight=None, eps=0.0):
    """x [tokens, heads, d] of float64 -> the same."""
    x = np.asarray(x, np.float64)
    if weight is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * weight
    r = 2 * len(freqs)
    angle = np.asarray(positions, np.float64)[:, None] * freqs
    c, s = (factor * f(angle)[:, None] for f in (np.cos, np.sin))
    out = x.copy()
    ia, ib = (np.arange(0, r, 2), np.arange(1, r, 2)) if interleaved else (np.arange(r // 2), np.arange(r // 2, r))
    out[..., ia] = x[..., ia] * c - x[..., ib] * s
    out[..., ib] = x[..., ia] * s + x[..., ib] * c
    return out


def attention(q, k, v, starts, starts_k, causal, scale):
    """q [tokens, heads, d], k / v [keys, kv_heads, d] of float64 -> (out, seen keys per row, largest sum |q_i k_i| |scale| per row, largest seen |v|
    per row); rows of no sequence are NaN in out."""
    q, k, v = (np.asarray(x, np.float64) for x in (q, k, v))
    group = q.shape[1] // k.shape[1]
    out = np.full(q.shape, np.nan)
    seen = np.zeros(q.shape[:2], int)
    size, most = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    for b in range(len(starts) - 1):
        q0, q1, k0, k1 = starts[b], starts[b + 1], starts_k[b], starts_k[b + 1]
        n, m = q1 - q0, k1 - k0
        for h in range(q.shape[1]):
            keys, values = k[k0:k1, h // group], v[k0:k1, h // group]
            for i in range(n):
                upto = min(max(i + m - n + 1, 0), m) if causal else m
                seen[q0 + i, h] = upto
                if upto == 0:
                    out[q0 + i, h] = 0
                    continue
                with np.errstate(all="ignore"):
                    s = keys[:upto] @ q[q0 + i, h] * scale
                    size[q0 + i, h] = (np.abs(keys[:upto]) @ np.abs(q[q0 + i, h])).max() * abs(scale)
                    most[q0 + i, h] = np.abs(values[:upto]).max()
                    p = np.exp(s - s.max())
                    out[q0 + i, h] = p @ values[:upto] / p.sum()
    return out, seen, size, most


def route(logits, top_k, scoring, bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    """One token at a time; sorted() is stable, so ties go to the lower index."""
    logits = np.asarray(logits, np.float64)
    all_ids, all_weights = [], []
    for row in logits:
        bad = np.isnan(row)
        l = np.where(bad, -np.inf, np.minimum(row, np.finfo(np.float32).max))
        with np.errstate(all="ignore"):
            if scoring == "softmax":
                e = np.exp(l - l.max()) if l.max() > -np.inf else np.zeros_like(l)
                s = e / e.sum() if e.sum() else e
            else:
                s = 1 / (1 + np.exp(-l))
        c = l.copy() if bias is None else np.where(bad, -np.inf, s + np.asarray(bias, np.float64))
        c = np.where(np.isnan(c), -np.inf, c)
        n = len(row) // groups
        kept = list(range(len(row)))
        if groups > 1:
            worth = []
            for g in range(groups):
                best = sorted(c[g * n:(g + 1) * n], reverse=True)[:group_best]
                if bias is None and group_best > 1:
                    best = sorted(s[g * n:(g + 1) * n], reverse=True)[:group_best]
                worth.append(sum(best))
            chosen = sorted(range(groups), key=lambda g: -worth[g])[:top_groups]
            kept = [e for e in kept if e // n in chosen]
        ids = sorted(kept, key=lambda e: -c[e])[:top_k]
        w = s[ids]
        if renormalize:
            with np.errstate(all="ignore"):
                m = l[ids].max()
                if m == -np.inf:
                    w = np.zeros(len(ids))
                elif scoring == "softmax":
                    w = np.exp(l[ids] - m)
                else:  # relative to the largest, so that the quotient of tiny scores is there
                    x, top = l[ids], min(m, 0.0)
                    w = np.where(x <= 0, np.exp(x - top) / (1 + np.exp(np.minimum(x, 0))), np.exp(-top) / (1 + np.exp(-x)))
            w = w / w.sum() if w.sum() else w
        all_ids.append(ids)
        all_weights.append(w * scale)
    return np.array(all_ids, np.int32).reshape(len(logits), top_k), np.array(all_weights).reshape(len(logits), top_k)
