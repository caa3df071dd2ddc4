"""GPU tests (pytest -m gpu) of beam selection's sums of exponentials: right to 64 bits, which decides between beams that are close."""
import numpy as np
import pytest

from test_gpu_kv_decode import check_beam, dev, qa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", (1, 7, 9000))
def test_a_certain_token_costs_nothing(qa, vocab):
    """A beam whose other tokens are ruled out keeps its score, and ties with a finished one that has the same."""
    rng = np.random.default_rng(vocab)
    logits = np.full((3, 4, vocab), -np.inf, np.float32)
    at = rng.integers(0, vocab, size=(3, 4))
    np.put_along_axis(logits, at[..., None], rng.normal(size=(3, 4, 1)).astype(np.float32) * 10, -1)
    scores = np.broadcast_to(np.float32([-1.5, -1.5, -1.5, 0.0]), (3, 4)).copy()
    got = qa.beam_select(dev(logits), dev(scores))
    assert (got.scores.cpu().numpy()[:, :4] == np.float32([0.0, -1.5, -1.5, -1.5])).all()
    check_beam(qa, logits, scores)
    finished = np.zeros((3, 4), np.uint8)
    finished[:, 1] = 1
    check_beam(qa, logits, scores, finished, 0)


@pytest.mark.parametrize("beams,vocab", [(2, 40), (2, 2049), (2, 20000)])
def test_beams_closer_than_1e_11(qa, beams, vocab):
    """Two beams whose sums of exponentials are e^0 + e^a and e^0 + e^b + e^c, equal but for 2e-12 of them (a further logit makes up for the rounding of
    a, b and c): the order of their best tokens is the order of the sums.  The sums' own roundings are some 1e-15."""
    rng = np.random.default_rng(vocab)
    prompts = 32
    logits = np.full((prompts, beams, vocab), -np.inf, np.float32)
    ahead = rng.integers(0, 2, size=prompts)
    exp = lambda x: np.exp(np.longdouble(x))  # noqa: E731
    for g in range(prompts):
        a = np.float32(rng.uniform(-2, -0.1))
        b = np.float32(a + np.log(rng.uniform(0.2, 0.8)))
        c = np.float32(np.log(exp(a) - exp(b) - np.longdouble(1e-6)))
        rest = exp(a) - exp(b) - exp(c)
        # (the first beam's token is the likelier if the second's sum is the larger one)
        target = rest + np.longdouble(-2e-12 if ahead[g] else 2e-12)
        d = np.float32(np.log(target))  # an f32 logit takes the rest to 2^-24 of itself, one more the rest of that
        e = target - exp(d)
        extra = [d]
        if e > 0:
            extra.append(np.float32(np.log(e)))
        row = rng.permutation(vocab)[:6]
        logits[g, 0, row[:2]] = 0.0, a
        logits[g, 1, row[:4 + len(extra) - 1]] = [0.0, b, c] + extra
        sums = [float(sum(exp(x) for x in logits[g, w] if x > -np.inf) - 1 - exp(a)) for w in range(2)]
        assert 1e-12 < abs(sums[1] - sums[0]) < 4e-12 and (sums[1] < sums[0]) == bool(ahead[g])
    got = qa.beam_select(dev(logits), dev(np.zeros((prompts, beams), np.float32)))
    assert np.array_equal(got.parents.cpu().numpy()[:, 0], ahead)
