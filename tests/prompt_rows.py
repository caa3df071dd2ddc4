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
