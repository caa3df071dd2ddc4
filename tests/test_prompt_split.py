"""The bound of prompt_split.py by itself: the six products keep it, any five of them do not."""
import numpy as np
import pytest

import prompt_split
from prompt_rows import attention_rows


@pytest.mark.parametrize("kind", ["scores", "values"])
@pytest.mark.parametrize("d,keys", [(64, 20), (128, 150), (256, 90)])
def test_the_bound_sees_every_product(kind, d, keys):
    seen = {}
    for seed in range(8):
        rng = np.random.default_rng(seed * 1000 + d)
        q, k, v, scale = prompt_split.inputs(kind, rng, 16, 2, keys, d)
        want = attention_rows(*(x.astype(np.float64) for x in (q, k, v)), [0, 16], [0, keys], False, scale, range(16))[0]
        tol = prompt_split.bound(kind)
        off = lambda **without: np.abs(prompt_split.restated(q, k, v, scale, **without) - want).max() / tol  # noqa: E731
        assert off() < 0.5
        for product in prompt_split.PRODUCTS:
            name = dict(scores="without_qk", values="without_pv")[kind]
            seen[product] = max(seen.get(product, 0), off(**{name: product}))
    assert min(seen.values()) > 1.5, seen


def test_what_is_left_out_is_below_its_bound():
    rng = np.random.default_rng(1)
    a, b = rng.uniform(1, 2, (2, 100000)).astype(np.float32)
    a[:3], b[:3] = 1 + 2.0 ** -7 - 2.0 ** -23, 1 + 2.0 ** -7 - 2.0 ** -23
    x, y = prompt_split.split(a), prompt_split.split(b)
    kept = sum(x[i] * y[j] for i, j in prompt_split.PRODUCTS)
    full = a.astype(np.float64) * b
    off = (full - kept) / full
    assert np.abs(off).max() <= 2.0 ** -22 and abs(off.mean()) <= 2.0 ** -27  # of either sign
    assert np.abs(off[:3]).max() <= 2.0 ** -28
    assert np.array_equal(sum(x), a.astype(np.float64))
