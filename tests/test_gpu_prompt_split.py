"""GPU tests (pytest -m gpu) of the bits that f32 prompt attention keeps: bounds and inputs of prompt_split.py, which fail with any one of the six
products of the three bf16 numbers left out (test_prompt_split.py)."""
import numpy as np
import pytest
import torch

import prompt_split
from prompt_rows import attention_rows

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def qa():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the HIP path cannot run (there is no fallback)")
    import izwi_amd
    izwi_amd.lib()
    torch.cuda.set_device(0)
    return izwi_amd


@pytest.mark.parametrize("kind", ["scores", "values"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,heads,keys", [(16, 2, 20), (16, 2, 90), (16, 2, 150), (16, 2, 1500), (3000, 16, 300)])
def test_no_product_is_missing(qa, kind, d, n, heads, keys):
    """One tile and several, one part and several, both sizes of workgroups."""
    print("split", kind, d, n, heads, keys, flush=True)
    for seed in range(8 if n < 100 else 1):
        rng = np.random.default_rng(seed * 1000 + d)
        q, k, v, scale = prompt_split.inputs(kind, rng, n, heads, keys, d)
        got = qa.prompt_attention(*(torch.from_numpy(x).cuda() for x in (q, k, v)), causal=False, scale=scale)
        tokens = sorted(set(np.linspace(0, n - 1, 16).astype(int).tolist()))
        want = attention_rows(*(x.astype(np.float64) for x in (q, k, v)), [0, n], [0, keys], False, scale, tokens)[0]
        off = np.abs(got[tokens].cpu().double().numpy() - want).max() / prompt_split.bound(kind)
        assert off <= 1, (seed, off)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,keys", [(40, 2), (40, 200), (2100, 200)])
def test_rests_of_the_value_s_own_sign(qa, d, n, keys):
    """a = 1 + 2^-7 - 2^-23 times itself, whose numbers cut off left out 2^-21 of the product, against a times 1 + 2^-7, which leaves out nothing.  Of a^2 2 2^-7 2^-23 =
    2^-29 is left out now; its sum is rounded when the last product is added (2^-23, whichever way the matrix core rounds) and when both
    halves are (2^-24); the two keys' weighted mean of 1 and -1 is off by half of that, and 2^-20 for exponentials and their arguments."""
    q, k, v = torch.zeros(n, 2, d), torch.zeros(keys, 1, d), torch.zeros(keys, 1, d)
    a = float(np.float32(1 + 2.0 ** -7 - 2.0 ** -23))
    e, one, two = 3 * d // 4, keys // 3, keys - 1
    q[:, :, e], k[:, :, e], scale = a, -1.0, 4096.0
    k[one, 0, e], k[two, 0, e], v[one], v[two] = a, 1 + 2.0 ** -7, 1.0, -1.0
    want = np.tanh((a * a - a * (1 + 2.0 ** -7)) * scale / 2)
    got = qa.prompt_attention(q.cuda(), k.cuda(), v.cuda(), causal=False, scale=scale).cpu().double().numpy()
    tol = 0.5 * a * a * scale * (2.0 ** -23 + 2.0 ** -24 + 2.0 ** -28) + 2.0 ** -20
    assert np.abs(got - want).max() <= tol, np.abs(got - want).max() / tol
