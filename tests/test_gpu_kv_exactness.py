"""GPU tests (pytest -m gpu) of how exact the attention over the quantized cache is, in every division of its work, against the
plain 64-bit restatement of kv_ref.py.

The arithmetic that bounds it.  u = 2^-24; A the largest sum of |q_i k_i| scale of a row, p_i its softmax weights, v_i the values, n its positions.
  A score is off by A (2^-22 for an f32 query as two f16 numbers, d u for the sums of products, 4 u for the two scales and log2 e);
  a weight, relatively, by that + ln2 2^-21 (its exponent is a number below 16, rounded once) + 2^-22 (exponential) + 2^-22 (two f16 numbers);
  and by 5 2^-37 of the row's largest weight: where the largest is 2^12 or more, the second f16 number ends at 2^-24, half a step (2^-37) off; what
  its product with the value's scale d loses is made up for by two fused multiply-adds that end there too, 2^-25 / d each, d >= 1/2 for the largest value.
  A weighted mean is off by twice the weights' relative error times sum p|v|, its two sums by (n / 16 + 64) u sum p|v| each (a lane sums a
  sixteenth at the most; 64 for the joins of lanes, waves and parts), the quotient by 2 u, and by 5 2^-37 n of the largest |v|.
  An f16 result is rounded once more: 2^-11 of itself."""
import numpy as np
import pytest
import torch

import kv_ref
from test_gpu_kv_decode import BITS, DTYPES, dev, draw, ints, qa  # noqa: F401

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

# How a call is divided: sequences, beams a prompt, kv heads, positions of the own cache, of the prefix; what is tested stands `at` one of them
PLANS = {
    "one_launch": dict(batch=4, beams=1, kv=2, capacity=64),
    "four_parts": dict(batch=16, beams=1, kv=4, capacity=1200),
    "ten_parts": dict(batch=4, beams=1, kv=2, capacity=1200),
    "wave_each": dict(batch=512, beams=1, kv=2, capacity=64),
    "behind_prefix": dict(batch=4, beams=2, kv=2, capacity=64, prefix=40),
    "wave_each_behind_prefix": dict(batch=512, beams=4, kv=2, capacity=64, prefix=3),
    "lineage": dict(batch=6, beams=3, kv=2, capacity=64, lineage=True),
    "wave_each_by_lineage": dict(batch=512, beams=4, kv=2, capacity=64, lineage=True),
    "prompts": dict(batch=18, beams=9, kv=2, capacity=64, at="prefix"),
    "row_pairs": dict(batch=18, beams=9, kv=2, capacity=1 << 16, at="prefix"),
}
GROUP = 2  # query heads of a kv head


class Attend:
    """Keys and values [slots, n, kv heads, d] where the plan wants them, on the device and in 64 bits; everything else in the caches reads as
    NaN.  `of_prefix`, `prefix_len`: keys and values of the plan's prefix (zeros by default) and how many count."""

    def __init__(self, qa, plan, quant, dtype, k, v, lens, of_prefix=None, prefix_len=None):
        P = self.plan = PLANS[plan]
        self.qa, self.dtype, self.beams = qa, dtype, P["beams"]
        batch, kv, d, n = P["batch"], P["kv"], k.shape[-1], k.shape[1]
        prompts = batch // P["beams"]
        self.shape = (batch, GROUP * kv, d)
        self.own = self.pre = self.lens = self.plens = self.lineage = self.own_ref = self.pre_ref = None

        def cache(slots, capacity, k, v, lens):
            made, ref = qa.QuantizedKvCache(qa.KvCacheType[quant], slots, kv, capacity, d), kv_ref.Cache(BITS[quant], slots, kv, k.shape[1], d)
            made.buffer.fill_(0xff)
            made.append(dev(k, dtype), dev(v, dtype), ints([0] * slots), ints(lens))
            ref.append(k, v, [0] * slots)
            return made, ref

        if P.get("at") == "prefix":
            self.plens = lens
            self.pre, self.pre_ref = cache(prompts, P["capacity"], k, v, lens)
            return
        if "prefix" in P:
            k0, v0 = of_prefix or (np.zeros((prompts, P["prefix"], kv, d), np.float32),) * 2
            self.plens = [P["prefix"] if prefix_len is None else prefix_len] * prompts
            self.pre, self.pre_ref = cache(prompts, P["prefix"], k0, v0, self.plens)
        self.lens = lens
        if P.get("lineage"):  # beam w's position p stands in the slot of beam (w + p) % beams
            b, p = np.arange(batch)[:, None], np.arange(n)[None]
            slot = b // self.beams * self.beams + (b + p) % self.beams
            self.lineage = np.full((batch, -(-P["capacity"] // 32) * 32), 255, np.uint8)
            self.lineage[:, :n] = slot % self.beams
            here = np.empty_like(k), np.empty_like(v)
            here[0][slot, p], here[1][slot, p] = k[b, p], v[b, p]
            (k, v), lens = here, [n] * batch
        self.own, self.own_ref = cache(batch, P["capacity"], k, v, lens)

    def run(self, q, scale):
        return self.qa.shared_prefix_attention(dev(q, self.dtype), self.own, None if self.lens is None else ints(self.lens), prefix=self.pre,
                                               prefix_lens=None if self.plens is None else ints(self.plens), beams=self.beams, scale=scale,
                                               lineage=None if self.lineage is None else torch.from_numpy(self.lineage).cuda()).cpu().double().numpy()

    def exact(self, q, scale, own_ref=None, pre_ref=None):
        return kv_ref.attention(q, own_ref or self.own_ref, self.lens, pre_ref or self.pre_ref, self.plens, self.lineage, self.beams, scale)

    def magnitude(self, q, scale):
        """sum p|v| of every output"""
        refs = []
        for r in (self.own_ref, self.pre_ref):
            if r is not None:
                a = kv_ref.Cache(r.bits, 1, 1, r.capacity, 1)
                a.v = np.stack([r.v[0], np.abs(r.v[1])])
                r = a
            refs.append(r)
        return self.exact(q, scale, *refs)[0]


def slots_of(plan):
    P = PLANS[plan]
    return P["batch"] // P["beams"] if P.get("at") == "prefix" else P["batch"]


def rows_of(plan, d):
    return PLANS[plan]["batch"], GROUP * PLANS[plan]["kv"], d


def tolerance(dtype, d, want, size, count, mean, top):
    """The bound at the head of this file; `mean` = sum p|v| per element, `top` = the largest |v| of a row."""
    relative = size * (2.0 ** -22 + (d + 4) * U) + np.log(2) * 2.0 ** -21 + 2.0 ** -21
    tol = (2 * relative + 2 * (count / 16 + 64) * U + 2 * U)[..., None] * mean + (count * 5 * 2.0 ** -37 * top)[..., None]
    return tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25 if dtype == "f16" else tol


def check(call, q, scale, dtype, largest=None):
    """`largest`: of the values that count, where others have no weight."""
    want, size, top, count = call.exact(q, scale)
    if largest is not None:
        top = np.where(top > 0, largest, 0.0)
    tol = tolerance(dtype, q.shape[-1], want, size, count, call.magnitude(q, scale), top)
    got = call.run(q, scale)
    print(f"worst error / tolerance {np.max(np.abs(got - want) / np.maximum(tol, 1e-300)):.3f}", flush=True)
    assert (np.abs(got - want) <= tol).all()
    return want, tol


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quant,d", [("Q8_0", 64), ("Q4_0", 128), ("Q8_0", 128), ("Q4_0", 256)])
def test_weights_keep_more_bits_than_an_f16(qa, quant, d, dtype, plan):
    """Two positions with values 1 and -1 and nearly equal scores: what is left of the weights' difference.  Weights rounded to f16 leave an error
    that the bound does not allow."""
    print("weights", quant, d, dtype, plan, flush=True)
    rng = np.random.default_rng(d)
    k = np.zeros((slots_of(plan), 2, PLANS[plan]["kv"], d), np.float32)
    v = np.ones_like(k)
    k[:, 1, :, 0], v[:, 1] = -1, -1
    call = Attend(qa, plan, quant, dtype, k, v, [2] * len(k), prefix_len=0)
    q = np.zeros(rows_of(plan, d), np.float32)
    q[..., 0] = rng.uniform(0.002, 0.05, size=q.shape[:2]).astype(np.float16)
    want, tol = check(call, q, 1.0, dtype)
    # the bound resolves it: weights rounded to f16 (f16's own formula, in 64 bits) would break it
    r = (1 - want[..., 0]) / (1 + want[..., 0])  # the second weight relative to the first
    rounded = r.astype(np.float16).astype(np.float64)
    assert (np.abs((1 - rounded) / (1 + r) - want[..., 0]) > tol[..., 0]).any()


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("quant,d", [("Q8_0", 64), ("Q4_0", 64), ("Q8_0", 128), ("Q4_0", 128), ("Q8_0", 256), ("Q4_0", 256)])
def test_f32_queries_keep_more_bits_than_an_f16(qa, quant, d, plan):
    """Queries whose f16 part is orthogonal to the keys: the scores, and the result, are what is left of an f32 query behind its f16."""
    print("queries", quant, d, plan, flush=True)
    rng = np.random.default_rng(d + 1)
    k, v = np.zeros((slots_of(plan), 2, PLANS[plan]["kv"], d), np.float32), np.ones((slots_of(plan), 2, PLANS[plan]["kv"], d), np.float32)
    v[:, 1] = -1
    rows = rows_of(plan, d)
    q = np.zeros(rows, np.float32)
    for b in range(0, d, 32):  # of a block: its scale from a key that no query sees, then 15 pairs of keys 7/8, -7/8
        k[:, 0, :, b] = 1
        k[:, 0, :, b + 1:b + 31:2], k[:, 0, :, b + 2:b + 31:2] = 0.875, -0.875
        x = rng.integers(1024, 2048, size=rows[:2] + (15,)) / 1024.0
        t = rng.uniform(0.2, 0.45, size=x.shape) * 2.0 ** -10  # (less than half an f16's step from x)
        q[..., b + 1:b + 31:2], q[..., b + 2:b + 31:2] = x + t, x - t
    k[:, 1] = -k[:, 0]
    call = Attend(qa, plan, quant, "f32", k, v, [2] * len(k), prefix_len=0)
    scale = 8.0 / (d * 30 / 32 * 1.5)
    want, tol = check(call, q, scale, "f32")
    lost = call.exact(q.astype(np.float16).astype(np.float32), scale)[0]  # the result of f16 queries
    assert (np.abs(lost - want) > 2 * tol).all()  # (the bound resolves it)
