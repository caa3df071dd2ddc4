"""GPU tests (pytest -m gpu) of attention scores whose spacing in f32 grows from a fraction to thousands, in every division of the work: the largest
takes all the weight, equal ones share it, and no weight leaves f16."""
import numpy as np
import pytest

from test_gpu_kv_decode import DTYPES, qa  # noqa: F401
from test_gpu_kv_exactness import PLANS, Attend, rows_of, slots_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("plan", PLANS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_every_size(qa, dtype, plan):
    rng = np.random.default_rng(len(plan))
    n, d, slots, kv = 50, 64, slots_of(plan), PLANS[plan]["kv"]
    k = rng.integers(-126, 127, size=(slots, n, kv, d)).astype(np.float32)
    k[..., ::32] = 127  # scale 1: quants as they are
    v = rng.normal(size=k.shape).astype(np.float16).astype(np.float32)
    best = rng.integers(0, n, size=(slots, kv))
    for b in range(slots):
        for h in range(kv):
            k[b, best[b, h], h, 1:32] = 127  # the largest of all, by more than 30 times 1
    k[0, n - 1, 0] = k[0, best[0, 0], 0]  # (and once more at the end)
    call = Attend(qa, plan, "Q8_0", dtype, k, v, [n] * slots, prefix_len=0)
    # queries see the first block only; scores to 2^12 times these, the others 31 times these and more behind; signs as they fall
    reaches = 2.0 ** np.arange(3, 15 if dtype == "f16" else 60)
    for scale in (1.0, 2.0 ** 6):
        for start in range(0, len(reaches), 4):
            q = np.zeros(rows_of(plan, d), np.float32)
            q[..., :32] = np.resize(reaches[start:start + 4], q.shape[0])[:, None, None]
            want, _, top, _ = call.exact(q, scale)
            got = call.run(q, scale)
            tol = (2.0 ** -21 + 200 * 2.0 ** -24) * top[..., None] + (2.0 ** -11 * np.abs(want) if dtype == "f16" else 0)
            assert (np.abs(got - want) <= tol).all(), (scale, reaches[start])
