"""GPU tests (pytest -m gpu) of what prompt attention keeps of its weights: f16 and bf16 results are as good as f32 weights make them, rounded once.

Tolerances, u = 2^-24.  A weight goes as two numbers of the type: the first is off by half a step, 2^-9 of the weight at most in bf16 and 2^-12 in f16
(relative to what it is rounded to, 2^-8 and 2^-11 relative to the power of two below), the second by as much of what is left: 2^-16, f16
2^-22 (or, far below the row's reference, 2^-32 of that).  Scores and exponentials are off as in test_gpu_prompt_ops.py, a mean by twice
that; the sums of n weighted values, two products of sixteen each at a time, by (2 n / 16 + 64) u V; the result by half a step."""
import numpy as np
import pytest
import torch

from prompt_rows import attention_rows

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
HALF = {name: torch.finfo(t).eps / 2 for name, t in DTYPES.items()}


@pytest.fixture(scope="module")
def qa():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the HIP path cannot run (there is no fallback)")
    import izwi_amd
    izwi_amd.lib()
    torch.cuda.set_device(0)
    return izwi_amd


def made(rng, *shape, dtype, std=1.0):
    x = torch.from_numpy((rng.normal(size=shape) * std).astype(np.float32)).to(DTYPES[dtype])
    return x.cuda(), x.double().numpy()


def check_rows(got, q64, k64, v64, starts, starts_k, causal, scale, dtype, tokens):
    want, n, size, most = attention_rows(q64, k64, v64, starts, starts_k, causal, scale, tokens)
    weight = 2 * (size * ((q64.shape[2] / 16 + 20) * U) + 2.0 ** -22) + (2.0 ** -16 if dtype == "bf16" else 2.0 ** -22 + n * 2.0 ** -32)
    tol = (most * (weight + (2 * n / 16 + 64) * U + 2.0 ** -23))[..., None] + HALF[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 1e-37)
    off = np.abs(got[tokens].cpu().double().numpy() - want) / tol
    assert (off <= 1).all(), float(np.nanmax(off))


SHAPES = [([40], [200], 8, 2), ([300], [300], 8, 2), ([2, 90, 1, 33], [150, 90, 400, 33], 4, 1), ([17], [1500], 16, 4), ([2100], [2100], 32, 8)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,lens_k,heads,kv", SHAPES)
def test_mean_of_values_of_both_signs(qa, dtype, d, causal, lens, lens_k, heads, kv):
    """Nearly equal weights on values of 1 and -1: what a weight loses stands beside a small result."""
    print("weights", dtype, d, causal, lens, heads, flush=True)
    rng = np.random.default_rng(d + sum(lens))
    starts, starts_k = np.cumsum([0] + lens), np.cumsum([0] + lens_k)
    (q, q64), (k, k64) = made(rng, starts[-1], heads, d, dtype=dtype), made(rng, starts_k[-1], kv, d, dtype=dtype)
    v64 = rng.choice([-1.0, 1.0], size=(starts_k[-1], kv, d))
    v = torch.from_numpy(v64.astype(np.float32)).to(DTYPES[dtype]).cuda()
    scale = 0.06 * d ** -0.5
    ints = lambda x: torch.tensor([int(i) for i in x], dtype=torch.int32, device="cuda")  # noqa: E731
    got = qa.prompt_attention(q, k, v, ints(starts), ints(starts_k), causal=causal, scale=scale)
    tokens = sorted(set(np.linspace(0, starts[-1] - 1, 12).astype(int).tolist()))
    check_rows(got, q64, k64, v64, starts, starts_k, causal, scale, dtype, tokens)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n,keys,heads,kv,causal", [(100, 100, 4, 2, True), (9, 1100, 4, 1, True), (2100, 2100, 32, 8, True), (1000, 800, 16, 8, False)])
def test_mean_of_equal_values_is_that_value(qa, dtype, d, n, keys, heads, kv, causal):
    """Keys of equal value give that value, whatever their weights and whether the row's reference has moved: the sum of the weights is that of the
    weights that the values meet.  (Off by less than 2^-14 the result still rounds to it: a step of either type is 2^-11 or more.)"""
    rng = np.random.default_rng(n + d)
    (q, _), (k, _) = made(rng, n, heads, d, dtype=dtype), made(rng, keys, kv, d, dtype=dtype)
    k = k * torch.linspace(0.2, 1.5, keys, device="cuda", dtype=torch.float32).to(k.dtype)[:, None, None]
    row, _ = made(rng, 1, kv, d, dtype=dtype)
    got = qa.prompt_attention(q, k, row.expand(keys, kv, d).contiguous(), causal=causal, scale=2.0 * d ** -0.5)
    first = n - keys if causal and keys < n else 0
    assert torch.equal(got[first:], row.repeat_interleave(heads // kv, 1).expand(n, heads, d)[first:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("d,n,keys,heads,kv,causal", [(64, 200, 200, 2, 1, True), (128, 130, 256, 2, 1, False), (128, 9, 1024, 4, 2, False), (256, 100, 128, 2, 1, False),
                                                      (256, 1100, 1100, 16, 8, True), (128, 2000, 2000, 32, 8, True)])
def test_a_value_that_is_no_number_that_every_row_sees(qa, dtype, bad, d, n, keys, heads, kv, causal):
    """The first key's value in one element, under weights that are a power of two, another number, or nothing: that element is no number for every
    row, an infinity the same infinity, and the others are as they were."""
    rng = np.random.default_rng(d + n)
    (q, _), (k, _), (v, _) = (made(rng, rows, g, d, dtype=dtype) for rows, g in ((n, heads), (keys, kv), (keys, kv)))
    k[0] *= 8
    clean = qa.prompt_attention(q, k, v, causal=causal)
    v[0, :, 5] = bad
    got = qa.prompt_attention(q, k, v, causal=causal)
    hit = got[..., 5]
    assert torch.isnan(hit).all() if bad != bad else (hit == bad).all()
    other = torch.arange(d, device="cuda") != 5
    assert torch.equal(got[..., other], clean[..., other])
