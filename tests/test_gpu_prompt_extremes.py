"""GPU tests (pytest -m gpu) of prompt attention on values of the largest size under weights that are zero in f32."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
CASES = [(40, 40, 4, 2), (40, 300, 4, 2), (5, 2500, 4, 1), (17, 8400, 32, 8), (2100, 2100, 32, 8), (700, 700, 16, 8)]


@pytest.fixture(scope="module")
def qa():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the HIP path cannot run (there is no fallback)")
    import izwi_amd
    izwi_amd.lib()
    torch.cuda.set_device(0)
    return izwi_amd


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,keys,heads,kv", CASES)
@pytest.mark.parametrize("causal", [True, False])
def test_large_values_under_no_weight(qa, dtype, d, n, keys, heads, kv, causal):
    """The first keys' scores are lower than the others' by 2000, and their values 10^37: rows that see another key are as if those values were zero, also where
    the two kinds stand in different tiles and parts, and the ones that see no other have them."""
    q, k = torch.ones(n, heads, d, device="cuda", dtype=dtype), torch.zeros(keys, kv, d, device="cuda", dtype=dtype)
    v = torch.randn(keys, kv, d, device="cuda").to(dtype)
    low = keys // 3
    k[:low, :, 0], k[low:, :, 0] = -1000, 1000
    v[:low] = 0
    want = qa.prompt_attention(q, k, v, causal=causal, scale=1.0)
    v[0] = 1e37
    got = qa.prompt_attention(q, k, v, causal=causal, scale=1.0)
    first = max(0, low - (keys - n)) if causal else 0  # the first row that sees one of the others
    assert torch.equal(got[first:], want[first:])
    if causal and first > 0:
        sees = torch.arange(first, device="cuda") + 1 + keys - n
        # equal weights w, not 1 as their scores of 1443 (base 2) have a reference of 24 bits: their sum takes an addition of 2^-24 for every key at most, the one product
        # that counts 12 of them (what three numbers leave out, 2^-22, and its sum), the quotient two; bf16 2^-16 for the weight and half a step
        off = (got[:first].double() * sees[:, None, None] / v[0, 0, 0].double() - 1).abs()
        tol = (sees + 14) * 2.0 ** -24 + (2.0 ** -16 + 2.0 ** -8 if dtype == torch.bfloat16 else 0)
        assert (off <= tol[:, None, None]).all(), float((off / tol[:, None, None]).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,keys,heads,kv", CASES)
@pytest.mark.parametrize("bad", [np.inf, -np.inf, np.nan])
def test_infinities_under_no_weight(qa, dtype, d, n, keys, heads, kv, bad):
    """An infinity that a row sees under a weight of zero, in a tile or part whose sums are scaled by zero: still that infinity, and NaN with another of the other
    sign."""
    q, k = torch.ones(n, heads, d, device="cuda", dtype=dtype), torch.zeros(keys, kv, d, device="cuda", dtype=dtype)
    v = torch.randn(keys, kv, d, device="cuda").to(dtype)
    k[:keys // 3, :, 0], k[keys // 3:, :, 0] = -1000, 1000
    want = qa.prompt_attention(q, k, v, causal=False, scale=1.0)
    v[1, :, 7], v[2, :, 9], v[keys - 1, :, 9] = bad, np.inf, -np.inf
    got = qa.prompt_attention(q, k, v, causal=False, scale=1.0)
    assert (torch.isnan(got[..., 7]) if bad != bad else got[..., 7] == bad).all() and torch.isnan(got[..., 9]).all()
    rest = [i for i in range(d) if i not in (7, 9)]
    assert torch.equal(got[..., rest], want[..., rest])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,keys,heads,kv", CASES + [(9, 8400, 16, 8)])
@pytest.mark.parametrize("causal", [True, False])
def test_means_of_the_largest_values(qa, dtype, d, n, keys, heads, kv, causal):
    """Values near the largest number of the type, whose weighted sums leave it and whose mean does not, in one element of every sixteen; the others are
    what they are beside ordinary values, to the bit (weights are scaled by a power of two)."""
    q, k, v = (torch.randn(rows, g, d, device="cuda").to(dtype) for rows, g in ((n, heads), (keys, kv), (keys, kv)))
    v[..., 3::16] = 1.0
    want = qa.prompt_attention(q, k, v, causal=causal)
    v[..., 3::16] = 3e38
    got = qa.prompt_attention(q, k, v, causal=causal)
    big = torch.arange(d, device="cuda") % 16 == 3
    sees = torch.ones(n, dtype=torch.bool, device="cuda")
    if causal and n > keys:
        sees[:n - keys] = False
    # a mean of equal values: what its products leave out (2^-22, bf16 weights 2^-16) and the sums of 17 and more terms at once, of f32 6 of each, 2^-24 an addition
    tol = (6 * keys / 16 + 64) * 2.0 ** -24 + 2.0 ** -22 + (2.0 ** -16 + 2.0 ** -8 if dtype == torch.bfloat16 else 0)
    off = (got[sees][..., big].double() / v[0, 0, 3].double() - 1).abs().max()
    assert off <= tol, float(off)
    assert torch.equal(got[..., ~big], want[..., ~big])
