"""GPU tests (pytest -m gpu) of what small weights add to the attention over the quantized cache.  Bounds: test_gpu_kv_exactness.py."""
import numpy as np
import pytest
import torch

from test_gpu_kv_decode import dev, ints, qa  # noqa: F401

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
