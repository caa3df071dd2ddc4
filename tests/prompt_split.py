"""f32 attention whose results depend on every bit of its operands: inputs in which a single one of the six products of the three bf16 numbers of each
operand shows, the bound that a result has to keep, and the arithmetic restated with any of those products left out.

Of an f32 number the first bf16 number is its top 8 bits; what is left is below 2^-7 of the power of two, the second is that rounded to 8 bits,
the third what is left then, 2^-16 at most and exact.  The six products of weight 2^-16 and more leave out 2 2^-7 2^-16 + 2^-32, 2^-22 of a product.
Two elements of a head are not zero, so a score takes a few additions at its own size, u = 2^-24 each, six of them at most; a weight is as
far off as its score, 2^-22 for the exponential and 2^-21 for its argument (two roundings below 8).  A mean of values between -m and m is off by
that times m (their mean distance from it is m at most; 1 % more for what is of second order), one of equal values not at all; its products
leave out 2^-22, and their sums, few at the size of the result, 12 u."""
import numpy as np

U = 2.0 ** -24
PRODUCTS = [(2, 0), (1, 1), (0, 2), (1, 0), (0, 1), (0, 0)]


def split(x):
    """float32 -> three float64 arrays, bf16 numbers each."""
    x = np.asarray(x, np.float32)
    first = (x.view(np.uint32) & 0xffff0000).view(np.float32)
    rest = x - first
    bits = rest.view(np.uint32).astype(np.uint64)
    second = ((bits + 0x7fff + (bits >> 16 & 1)) & 0xffff0000).astype(np.uint32).view(np.float32)
    third = rest - second
    assert ((third.view(np.uint32) & 0xffff) == 0).all()
    return [n.astype(np.float64) for n in (first, second, third)]


def product(a, b, without=None):
    """a @ b of float32 matrices, by the six products but one."""
    a, b = split(a), split(b)
    return sum(a[i] @ b[j] for i, j in PRODUCTS if (i, j) != without)


def inputs(kind, rng, n, heads, keys, d):
    """(q [n, heads, d], k, v [keys, 1, d], scale) of float32.  "scores": two keys of scores of thousands that nearly agree, made of elements that
    do not; "values": three keys of different weights, each with the same value of 24 bits.  The other keys have no weight."""
    q, k, v = np.zeros((n, heads, d), np.float32), np.zeros((keys, 1, d), np.float32), np.zeros((keys, 1, d), np.float32)
    e, f = rng.choice(d, 2, replace=False)
    a, c = rng.uniform(1, 2, 2).astype(np.float32)
    real = rng.choice(keys, 2 if kind == "scores" else 3, replace=False)
    k[:, 0, e] = -40
    if kind == "scores":
        b = rng.uniform(1, 2, 2).astype(np.float32)
        scale, k[real, 0, e], k[real, 0, f] = 1024.0, b, (4 - a.astype(np.float64) * b) / c
        # every query its own numbers, as near to the first ones as keeps the scores together
        q[..., e] = a * (1 + rng.uniform(-1, 1, (n, heads)) * 2.0 ** -12)
        q[..., f] = c * (1 + rng.uniform(-1, 1, (n, heads)) * 2.0 ** -12)
        v[real[0], 0] = rng.choice([-1.0, 1.0], d)
        v[real[1], 0] = -v[real[0], 0]
    else:
        q[..., e] = rng.uniform(20, 40, (n, heads))
        k[real, 0, e] = rng.uniform(0, 1 / 40, 3)
        v[real, 0], scale = rng.uniform(1, 2, d), 1.0
    return q, k, v, scale


def bound(kind):
    """Of a result: scores are sums of two products, about 4 together, times 1024, and values 1 or -1; equal values are below 2."""
    if kind == "values":
        return 2 * (2.0 ** -22 + 12 * U)
    score = 4.1 * 1024 * (2.0 ** -22 + 6 * U)
    return 1.01 * (score + 2.0 ** -22 + 2.0 ** -21) + 2.0 ** -22 + 12 * U


def restated(q, k, v, scale, without_qk=None, without_pv=None):
    """[n, heads, d]: the two matrix products by bf16 numbers, sums and exponentials in 64 bits, weights rounded to f32."""
    n, heads, d = q.shape
    s = product(q.reshape(-1, d), k[:, 0].T.copy(), without_qk) * scale
    p = np.exp(s - s.max(1, keepdims=True)).astype(np.float32)
    p[p < 2.0 ** -90] = 0
    return (product(p, v[:, 0].copy(), without_pv) / p.astype(np.float64).sum(1, keepdims=True)).reshape(n, heads, d)
