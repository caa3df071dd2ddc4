"""GPU tests (pytest -m gpu) of what small weights and small values add to the attention over the quantized cache: many positions far below a few
that dominate, and values of one size beside values of another.  Bounds: test_gpu_kv_exactness.py."""
import numpy as np
import pytest
import torch

from test_gpu_kv_decode import dev, ints, qa  # noqa: F401
from test_gpu_kv_exactness import PLANS, Attend, check, rows_of, slots_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("quant", ("Q8_0", "Q4_0"))
@pytest.mark.parametrize("beams", (1, 18))
def test_many_positions_behind_a_few(qa, beams, quant):
    """Four positions (values zero) take nearly all the weight, 2^15 others (values one) 2^-13 to 2^-27 of it each: their sum is the result, and a weight
    that is off is off for all of them.  As many sequences as there are compute units, so that every wave sees a dominating position; 18 beams on a
    prefix go two tiles of rows to a workgroup."""
    n, d, kv, slots = 1 << 15, 64, 8, 32
    cache = qa.QuantizedKvCache(qa.KvCacheType[quant], slots, kv, n, d)
    k, v = torch.zeros(1, n, kv, d, device="cuda"), torch.ones(1, n, kv, d, device="cuda")
    k[0, :128:32, :, 0], v[0, :128:32] = 1.0, 0.0
    for slot in range(slots):
        cache.append(k, v, ints([0]), first_slot=slot)
    got_k, got_v = (float(x.cpu()[0, i, 0, 0]) for x, i in zip(cache.read(ints([0]), 2), (0, 1)))
    q = np.zeros((slots * beams, kv, d), np.float32)
    q[..., 0] = np.linspace(13, 27, slots * beams * kv).reshape(slots * beams, kv) * np.log(2)
    lens = ints([n] * slots)
    out = qa.shared_prefix_attention(dev(q), cache, lens, beams=1, scale=1.0) if beams == 1 else qa.shared_prefix_attention(
        dev(q), None, None, prefix=cache, prefix_lens=lens, beams=beams, scale=1.0)
    size = q[..., 0].astype(np.float64) * got_k
    others = (n - 4) * np.exp(-size)
    want = (others / (4 + others)) * got_v
    # the bound of test_gpu_kv_exactness.py, for scores of a single product (four roundings); the four largest have a quarter each
    relative = size * (2.0 ** -22 + 4 * 2.0 ** -24) + np.log(2) * 2.0 ** -21 + 2.0 ** -21
    tol = (2 * relative + 2 * (n / 16 + 64) * 2.0 ** -24) * want + n / 4 * 5 * 2.0 ** -37
    got = out.cpu().double().numpy()
    print(f"worst error / tolerance {np.max(np.abs(got - want[..., None]) / tol[..., None]):.3f}", flush=True)
    assert (np.abs(got - want[..., None]) <= tol[..., None]).all()


@pytest.mark.parametrize("dtype", ("f32", "f16"))
@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("quant,d", [("Q8_0", 128), ("Q4_0", 64), ("Q4_0", 256)])
def test_values_beside_far_larger_ones(qa, quant, d, dtype, plan):
    """Values 2^10 larger than their neighbours in the tile of 32 positions, and a tile of values 2^19 larger in front of it or behind it, all under a
    weight that leaves nothing of them, cost the others no bits: the bound's largest value is that of the tile."""
    rng = np.random.default_rng(d)
    n, slots, kv = 45, slots_of(plan), PLANS[plan]["kv"]
    k, v = (rng.normal(size=(slots, n, kv, d)).astype(np.float16).astype(np.float32) for _ in range(2))
    k[..., 0] = 0.0
    v *= 2.0 ** -6
    for b in range(slots):
        far = np.arange(32, n) if b % 2 else np.arange(32)
        near = [33 + b % 5, 40] if b % 2 == 0 else [b % 16, 20]
        v[b, far] *= 2.0 ** 19
        v[b, near] *= 2.0 ** 10
        k[b, far, :, 0] = k[b, near, :, 0] = -1.0
    v = np.clip(v.astype(np.float16).astype(np.float32), -6e4, 6e4)
    call = Attend(qa, plan, quant, dtype, k, v, [n - b % 3 for b in range(slots)], prefix_len=0)
    q = rng.normal(size=rows_of(plan, d)).astype(np.float16).astype(np.float32)
    q[..., 0] = 200.0 * d ** 0.5 * 2  # positions with the large values: some 2^-290 and less of the largest weight
    check(call, q, 0.5 * d ** -0.5, dtype, largest=2.0 ** 10 * 5 * 2.0 ** -6)
