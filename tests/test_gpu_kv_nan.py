"""GPU tests (pytest -m gpu): numbers that are none.  Whatever a row reads that is NaN, in its query, its keys or its values, makes its result NaN (in
the value's block of 32), as the definition in 64 bits does, however the work is divided; no other row sees it, and a row without positions is zero."""
import numpy as np
import pytest
import torch

from test_gpu_kv_decode import BITS, DTYPES, draw, qa  # noqa: F401
from test_gpu_kv_exactness import GROUP, PLANS, Attend, rows_of, slots_of, tolerance

pytestmark = pytest.mark.gpu


def check_nan(call, q, scale, dtype):
    with np.errstate(all="ignore"):
        want, size, top, count = call.exact(q, scale)
        mean = call.magnitude(q, scale)
    got = call.run(q, scale)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    # (rows with a NaN among their values are exact elsewhere; their largest value is taken from what is a number)
    tol = tolerance(dtype, q.shape[-1], want, size, count, mean, np.where(np.isnan(top), 100.0, top))
    assert (np.abs(got - want) <= tol)[~np.isnan(want)].all()
    assert (got[count == 0] == 0).all()
    return want


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quant,d", [("Q8_0", 128), ("Q4_0", 64), ("Q8_0", 256)])
def test_numbers_that_are_none(qa, quant, d, dtype, plan):
    print("none", quant, d, dtype, plan, flush=True)
    rng = np.random.default_rng(d + len(plan))
    n, slots, kv = 45, slots_of(plan), PLANS[plan]["kv"]
    k, v = draw(rng, slots, n, kv, d, dtype=dtype), draw(rng, slots, n, kv, d, dtype=dtype)
    # who has one position, more, none; whose key or value is NaN where
    lens = [n - (s * 7) % n for s in range(slots)]
    lens[0] = lens[-1] = 1
    k[0, 0, 0, 3] = np.nan           # the only position
    if slots > 3:
        lens[1], lens[2], lens[3] = 33, 33, 0
        k[1, 32, -1, 5] = np.inf     # the last, alone in its tile
        v[2, 32, 0, d - 1] = np.nan  # a value there
    if slots > 6:
        lens[4], lens[5], lens[6] = 40, 40, 20
        k[4, :32, 0, 40] = np.nan    # the first tile
        k[5, :, :, 0] = -np.inf      # every key
        v[6, 25, :, 0] = np.nan      # behind the end: not read
    pre = None
    if "prefix" in PLANS[plan]:
        shape = (slots // PLANS[plan]["beams"], PLANS[plan]["prefix"], kv, d)
        pre = draw(rng, *shape, dtype=dtype), draw(rng, *shape, dtype=dtype)
    call = Attend(qa, plan, quant, dtype, k, v, lens, pre)
    clean = draw(rng, *rows_of(plan, d), dtype=dtype, outliers=False)
    want = check_nan(call, clean, d ** -0.5, dtype)
    assert np.isnan(want).any() and not np.isnan(want).all()
    # queries: a NaN, infinities of both signs, among rows with positions and rows with none
    for bad in (np.nan, np.inf, -np.inf):
        q = clean.copy()
        q[1::3, 1, d // 2] = bad
        q[:, -1, 0] = bad
        assert np.isnan(check_nan(call, q, d ** -0.5, dtype)).any()


@pytest.mark.parametrize("plan", [p for p in PLANS if "prefix" in PLANS[p]])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_value_that_is_none_under_a_weight_of_zero(qa, dtype, plan):
    """0 * NaN is NaN in the part that holds it and where parts are joined."""
    n, d, kv, slots = 3, 64, 2, slots_of(plan)
    k = np.zeros((slots, n, kv, d), np.float32)
    k[..., 0] = -1.0
    v = np.ones_like(k)
    v[0, 1, 0, 40] = np.nan
    shape = (slots // PLANS[plan]["beams"], PLANS[plan]["prefix"], kv, d)
    call = Attend(qa, plan, "Q8_0", dtype, k, v, [n] * slots, (np.zeros(shape, np.float32), np.ones(shape, np.float32)))
    q = np.zeros(rows_of(plan, d), np.float32)
    q[..., 0] = 2000.0  # own positions score 2000 below the prefix
    want = check_nan(call, q, 1.0, dtype)
    assert np.isnan(want[0, :GROUP, 32:]).all() and not np.isnan(want[0, :GROUP, :32]).any() and not np.isnan(want[1:]).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch", (6, 512))
def test_no_position_by_lineage_stays_zero(qa, dtype, batch):
    """Positions that no beam wrote do not count, NaN query or not."""
    lens = torch.full((batch,), 20, dtype=torch.int32, device="cuda")
    cache = qa.QuantizedKvCache(qa.KvCacheType.Q8_0, batch, 2, 64, 64)
    cache.buffer.fill_(0xff)
    q = torch.full((batch, 4, 64), float("nan"), device="cuda", dtype=DTYPES[dtype])
    out = qa.shared_prefix_attention(q, cache, lens, beams=2, lineage=torch.full_like(cache.new_lineage(), 255))
    assert (out == 0).all()


@pytest.mark.parametrize("sign", (1.0, -1.0))
def test_scores_beyond_f32(qa, sign):
    """Scores that have no f32 take all the weight, or none, as in 64 bits: no infinity stands for them."""
    d, n = 64, 40
    k = np.zeros((4, n, 2, d), np.float32)
    k[..., 0] = 1.0
    k[:, 7, :, 0] = 3.0 if sign > 0 else 0.5  # the largest score
    v = np.random.default_rng(1).normal(size=k.shape).astype(np.float32)
    call = Attend(qa, "one_launch", "Q8_0", "f32", k, v, [n] * 4)
    q = np.zeros(rows_of("one_launch", d), np.float32)
    q[..., 0] = sign * 3e38
    for scale in (1e-3, 1.0, 1e10):
        want, _, top, _ = call.exact(q, scale)
        assert (np.abs(call.run(q, scale) - want) <= 200 * 2.0 ** -24 * top[..., None]).all()
