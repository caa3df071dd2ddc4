"""GPU tests (pytest -m gpu) of the bits of rotary positions: cosine, sine and factor in 64 bits, rounded to 32 once.

Tolerance, u = 2^-24: a rotated element is x c - y s (or x s + y c) with c and s rounded once, two products rounded and their sum: (|x c| + |y s|) 2 u
+ |out| u, 1 % more for the products of roundings and 2^-36 of the series; other types half a step more."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


@pytest.fixture(scope="module")
def qa():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the HIP path cannot run (there is no fallback)")
    import izwi_amd
    izwi_amd.lib()
    torch.cuda.set_device(0)
    return izwi_amd


def ints(values):
    return torch.tensor([int(v) for v in values], dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,r", [(128, 128), (64, 32), (70, 34)])
@pytest.mark.parametrize("yarn", [False, True])
def test_rotation_is_as_near_as_32_bits_are(qa, dtype, interleaved, d, r, yarn):
    rng = np.random.default_rng(d + r)
    tokens = 700
    rotary = qa.RotaryEmbedding(d, base=1e6, rotary_dim=r, interleaved=interleaved, scaling=qa.RopeScaling.yarn(4.0, 8192) if yarn else None)
    freqs, factor = rotary.frequencies.cpu().numpy(), rotary.attention_factor
    positions = np.concatenate([np.arange(200), rng.integers(-(2 ** 31), 2 ** 31, 250), rng.integers(0, 2 ** 20, 250)])
    x = torch.from_numpy(rng.normal(size=(tokens, 3, d)).astype(np.float32)).to(dtype)
    got = qa.rope_positions(x.cuda(), None, ints(positions), rotary)[0].cpu().double().numpy()
    x = x.double().numpy()
    angle = positions.astype(np.float64)[:, None, None] * freqs
    c, s = factor * np.cos(angle), factor * np.sin(angle)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
    half = torch.finfo(dtype).eps / 2
    for at, one, two, sign in ((a, x[..., a] * c, x[..., b] * s, -1), (b, x[..., a] * s, x[..., b] * c, 1)):
        want = one + sign * two
        tol = 1.01 * ((np.abs(one) + np.abs(two)) * 2 * U + np.abs(want) * U) + (half * np.abs(want) + 2.0 ** -25 if dtype != torch.float32 else 0)
        off = np.abs(got[..., at] - want) / tol
        assert off.max() <= 1, off.max()


def test_position_zero_is_the_factor_itself(qa):
    """c and s are the factor, rounded once, and 0."""
    x = torch.randn(5, 2, 128, device="cuda")
    assert torch.equal(qa.rope_positions(x, None, ints([0] * 5), qa.RotaryEmbedding(128))[0], x)
    rotary = qa.RotaryEmbedding(128, scaling=qa.RopeScaling.yarn(4.0, 4096))
    factor = float(np.float32(rotary.attention_factor))
    assert torch.equal(qa.rope_positions(x, None, ints([0] * 5), rotary)[0], x * factor)


def test_quarter_turns(qa):
    """Frequencies of whole quarter turns, in both directions: every branch of the reduction."""
    rotary = qa.RotaryEmbedding(64, rotary_dim=2)
    rotary.frequencies.fill_(np.pi / 2)
    x = torch.zeros(9, 1, 64, device="cuda")
    x[..., 0] = 1
    got = qa.rope_positions(x, None, ints(range(-4, 5)), rotary)[0][:, 0, :2].cpu()
    want = torch.tensor([[1, 0], [0, 1], [-1, 0], [0, -1], [1, 0], [0, 1], [-1, 0], [0, -1], [1, 0.0]])
    assert (got - want).abs().max() <= 2.0 ** -50


def test_other_frequencies(qa):
    """A call reads what the embedding holds then: values written to it count, and another tensor in its place, which a call would not look at, is
    refused."""
    x = torch.randn(9, 2, 64, device="cuda")
    one, other = qa.RotaryEmbedding(64, base=1e4), qa.RotaryEmbedding(64, base=1e6)
    want = qa.rope_positions(x, None, ints(range(9)), other)[0]
    kept = one.frequencies
    with pytest.raises(AttributeError):
        one.frequencies = other.frequencies
    assert one.frequencies is kept
    one.frequencies.copy_(other.frequencies)
    assert torch.equal(qa.rope_positions(x, None, ints(range(9)), one)[0], want)
