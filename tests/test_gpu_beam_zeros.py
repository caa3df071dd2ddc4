"""GPU tests (pytest -m gpu) of beam selection's order where scores are zeros of either sign: equal numbers, so the lower index first."""
import numpy as np
import pytest
import torch

from test_gpu_kv_decode import check_beam, qa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("beams,vocab", [(2, 1), (5, 1), (4, 300), (3, 9000)])
def test_zeros_of_either_sign_are_equal(qa, beams, vocab):
    for first in (0, 1):
        scores = np.where(np.arange(beams) % 2 == first, -0.0, 0.0).astype(np.float32)[None]
        logits = np.zeros((1, beams, vocab), np.float32)
        check_beam(qa, logits, scores, np.ones((1, beams), np.uint8), vocab // 2)  # all finished
        if vocab == 1:  # a beam with one token: a log-probability of zero
            check_beam(qa, logits, scores)
            check_beam(qa, -logits, scores, (np.arange(beams) % 2 == 0).astype(np.uint8)[None], 0)
