"""Plain numpy restatements, in 64 bits, of the quantized cache, the attention over it and beam search's step
(include/izwi_decode_ops.h): what the kernels are tested against."""
import numpy as np

F32_MAX = np.float64(np.finfo(np.float32).max)


def quantize(x, bits):
    """x [..., d] f32 -> (quants int [..., d], scales f16 [..., d / 32]), every step rounded to f32 as the format asks."""
    x = np.asarray(x, np.float32)
    b = x.reshape(x.shape[:-1] + (-1, 32))
    with np.errstate(all="ignore"):
        amax = np.abs(b).max(-1)  # (a NaN stays one)
        if bits == 8:
            d = (amax / np.float32(127)).astype(np.float32)
        else:
            d = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1)[..., 0] * np.float32(-0.125)
        h = d.astype(np.float16)
        bad = ~np.isfinite(amax) | ~np.isfinite(h)
        dead = bad | (h == 0)
        inv = np.where(dead, np.float32(0), np.float32(1) / np.where(dead, np.float32(1), d))
        s = (np.where(bad[..., None], np.float32(0), b) * inv[..., None]).astype(np.float32)
        if bits == 8:
            q = np.trunc(s.astype(np.float64) + np.copysign(0.5, s))
        else:
            q = np.minimum(np.trunc((s + np.float32(8.5)).astype(np.float32)), 15) - 8
        q = np.where(dead[..., None], 0, q).astype(np.int64)
        h = np.where(bad, np.float16(np.nan), h)
    return q.reshape(x.shape), h


def values(q, h):
    b = q.reshape(q.shape[:-1] + (-1, 32)).astype(np.float64)
    return (b * h.astype(np.float64)[..., None]).reshape(q.shape)


class Cache:
    """values [2][slots][capacity][kv_heads][d] in 64 bits."""

    def __init__(self, bits, slots, kv_heads, capacity, d):
        self.bits, self.capacity = bits, capacity
        self.v = np.zeros((2, slots, capacity, kv_heads, d))

    def append(self, k, v, starts, counts=None, first_slot=0):
        for i, x in enumerate((k, v)):
            got = values(*quantize(x, self.bits))
            for b in range(x.shape[0]):
                for t in range(x.shape[1] if counts is None else min(x.shape[1], max(0, counts[b]))):
                    if 0 <= starts[b] + t < self.capacity:
                        self.v[i, first_slot + b, starts[b] + t] = got[b, t]

    def read(self, starts, tokens, counts=None, first_slot=0, lineage=None, beams=1):
        out = np.zeros((2, len(starts), tokens) + self.v.shape[3:])
        for b, start in enumerate(starts):
            for t in range(tokens if counts is None else min(tokens, max(0, counts[b]))):
                p, slot = start + t, first_slot + b
                if not 0 <= p < self.capacity:
                    continue
                if lineage is not None:
                    if lineage[slot, p] >= beams:
                        continue
                    slot = slot // beams * beams + lineage[slot, p]
                out[:, b, t] = self.v[:, slot, p]
        return out


def attention(q, cache, lens, prefix=None, prefix_lens=None, lineage=None, beams=1, scale=1.0):
    """q [batch, heads, d] -> (out, per row: largest sum of |q k| scale, largest |v|, positions) in 64 bits."""
    q = q.astype(np.float64)
    batch, heads, d = q.shape
    out, size, top, count = np.zeros(q.shape), np.zeros((batch, heads)), np.zeros((batch, heads)), np.zeros((batch, heads), int)
    for b in range(batch):
        parts = []
        if prefix is not None:
            parts.append(prefix.v[:, b // beams, :max(0, prefix_lens[b // beams])])
        if cache is not None:
            n = max(0, lens[b])
            if lineage is None:
                parts.append(cache.v[:, b, :n])
            else:
                at = [p for p in range(n) if lineage[b, p] < beams]
                parts.append(cache.v[:, [b // beams * beams + int(lineage[b, p]) for p in at], at])
        kv = np.concatenate(parts, 1)
        if kv.shape[1] == 0:
            continue
        kv_heads = kv.shape[2]
        for h in range(heads):
            k, v = kv[:, :, h // (heads // kv_heads)]
            s = (k @ q[b, h]) * scale
            w = np.exp(s - s.max())
            out[b, h] = (w @ v) / w.sum()
            size[b, h] = (np.abs(k) @ np.abs(q[b, h])).max() * abs(scale)
            top[b, h], count[b, h] = np.abs(v).max(), len(s)
    return out, size, top, count


def beam_select(logits, scores, finished=None, eos=-1):
    """logits [prompts, beams, vocab], scores [prompts, beams] -> (tokens, parents, scores in 64 bits, finished)."""
    prompts, beams, vocab = logits.shape
    clean = lambda x: np.where(np.isnan(x), -np.inf, np.minimum(x.astype(np.float64), F32_MAX))  # noqa: E731
    x, s = clean(np.asarray(logits)), clean(np.asarray(scores))
    tokens, parents, out, ended = [], [], [], []
    for g in range(prompts):
        total = np.full((beams, vocab), -np.inf)
        legal = np.ones((beams, vocab), bool)
        for w in range(beams):
            if finished is not None and finished[g, w]:
                legal[w] = np.arange(vocab) == eos
                total[w, eos] = s[g, w]
            elif s[g, w] != -np.inf and x[g, w].max() != -np.inf:
                m = x[g, w].max()
                with np.errstate(all="ignore"):
                    total[w] = s[g, w] - m - np.log(np.exp(x[g, w] - m).sum()) + x[g, w]
        flat = total.ravel()
        order = np.lexsort((np.arange(flat.size), -flat, ~legal.ravel()))[:beams]
        tokens.append(order % vocab)
        parents.append(order // vocab)
        out.append(flat[order])
        ended.append([(finished is not None and bool(finished[g, i // vocab])) or i % vocab == eos for i in order])
    return np.array(tokens), np.array(parents), np.array(out), np.array(ended)


def lineage_step(lineage, parents, lens):
    """lineage [prompts * beams, n], parents [prompts, beams], lens [prompts * beams]."""
    prompts, beams = parents.shape
    out = np.empty_like(lineage)
    for g in range(prompts):
        for i in range(beams):
            p = g * beams + parents[g, i]
            out[g * beams + i] = lineage[p]
            if 0 <= lens[p] < lineage.shape[1]:
                out[g * beams + i, lens[p]] = i
    return out
