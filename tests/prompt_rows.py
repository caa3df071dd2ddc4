"""Attention of single tokens of packed prompts in 64 bits: the rows of long prompts that a test looks at, without all the others."""
import numpy as np


def attention_rows(q, k, v, starts, starts_k, causal, scale, tokens):
    """q [tokens, heads, d], k / v [keys, kv_heads, d] of float64 -> (out, keys seen, largest sum |q_i k_i| |scale|, largest seen |v|) of the named
    tokens, every head; a token of no sequence is NaN."""
    heads, kv, d = q.shape[1], k.shape[1], q.shape[2]
    group = heads // kv
    out = np.full((len(tokens), heads, d), np.nan)
    seen, size, most = (np.zeros((len(tokens), heads)) for _ in range(3))
    for at, token in enumerate(tokens):
        for b in range(len(starts) - 1):
            if starts[b] <= token < starts[b + 1]:
                m = starts_k[b + 1] - starts_k[b]
                upto = min(max(token - starts[b] + 1 + m - (starts[b + 1] - starts[b]), 0), m) if causal else m
                seen[at] = upto
                if upto == 0:
                    out[at] = 0
                    continue
                keys, values = (x[starts_k[b]:starts_k[b] + upto].transpose(1, 0, 2) for x in (k, v))  # [kv, keys, d]
                one = q[token].reshape(kv, group, d).transpose(0, 2, 1)  # [kv, d, group]
                s = keys @ one * scale
                size[at] = (np.abs(keys) @ np.abs(one)).max(1).reshape(-1) * abs(scale)
                p = np.exp(s - s.max(1, keepdims=True))
                most[at] = np.repeat(np.abs(values).max((1, 2)), group)
                out[at] = (p.transpose(0, 2, 1) @ values / p.sum(1)[:, :, None]).reshape(heads, d)
    return out, seen, size, most


def route_rows(logits, top_k, scoring, bias=None, groups=1, top_groups=1, group_best=1, renormalize=True, scale=1.0):
    """Scored routing of many tokens at once, in 64 bits: what prompt_ref.route gives token by token (its ties and missing numbers too) for scores that do
    not all vanish."""
    l = np.asarray(logits, np.float64)
    bad = np.isnan(l)
    l = np.where(bad, -np.inf, np.minimum(l, np.finfo(np.float32).max))
    t, n = l.shape
    with np.errstate(all="ignore"):
        if scoring == "softmax":
            top = l.max(1, keepdims=True)
            e = np.where(top > -np.inf, np.exp(l - np.where(top > -np.inf, top, 0)), 0)
            total = e.sum(1, keepdims=True)
            s = np.divide(e, total, out=np.zeros_like(e), where=total > 0)
        else:
            s = 1 / (1 + np.exp(-l))
        c = l if bias is None else np.where(bad, -np.inf, s + np.asarray(bias, np.float64))
        c = np.where(np.isnan(c), -np.inf, c)
        of = s if bias is None and group_best > 1 else c
        worth = np.sort(of.reshape(t, groups, -1), 2)[:, :, ::-1][:, :, :group_best].sum(2)
    order = np.argsort(-worth, 1, kind="stable")[:, :top_groups]
    kept = np.zeros((t, groups), bool)
    np.put_along_axis(kept, order, True, 1)
    kept = np.repeat(kept, n // groups, 1)
    ids = np.lexsort((np.broadcast_to(np.arange(n), (t, n)), -c, ~kept), 1)[:, :top_k]
    w = np.take_along_axis(s, ids, 1)
    if renormalize:
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    return ids.astype(np.int32), w * scale
