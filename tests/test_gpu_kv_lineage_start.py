"""GPU tests (pytest -m gpu) of where a lineage begins: what beams write before the first selection is their own."""
import numpy as np
import pytest
import torch

import kv_ref
from test_gpu_kv_decode import check_attention, dev, draw, ints, qa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("prompts,beams,own", [(1, 4, 1), (2, 3, 1), (3, 1, 2), (2, 5, 6)])
def test_beams_that_start_from_different_tokens(qa, prompts, beams, own):
    """The module's recipe: `own` positions a beam, written and attended to before any selection, then a selection and a position more."""
    rng = np.random.default_rng(prompts * 10 + beams)
    n, kv, heads, d, steps = prompts * beams, 2, 4, 64, 12
    cache, ref = qa.QuantizedKvCache(qa.KvCacheType.Q8_0, n, kv, steps, d), kv_ref.Cache(8, n, kv, steps, d)
    lineage, lens = cache.new_lineage(beams), torch.zeros(n, dtype=torch.int32, device="cuda")
    assert lineage.dtype == torch.uint8 and lineage.shape == (n, 32)
    scores = dev(np.sort(rng.normal(size=(prompts, beams)).astype(np.float32))[:, ::-1].copy())
    rows = np.repeat(np.arange(n)[:, None] % beams, 32, 1).astype(np.uint8)
    for step in range(3):
        tokens = own if step == 0 else 1
        k, v, q = draw(rng, n, tokens, kv, d), draw(rng, n, tokens, kv, d), draw(rng, n, heads, d)
        at = lens.tolist()
        cache.append(dev(k), dev(v), lens)
        ref.append(k, v, at)
        lens += tokens
        out = qa.shared_prefix_attention(dev(q), cache, lens, beams=beams, lineage=lineage)
        check_attention(out, kv_ref.attention(q, ref, lens.tolist(), lineage=rows, beams=beams, scale=d ** -0.5), "f32", d)
        picked = qa.beam_select(dev(rng.normal(size=(prompts, beams, 50)).astype(np.float32)), scores, lineage=lineage, lens=lens, out_lineage=lineage)
        rows = kv_ref.lineage_step(rows, picked.parents.cpu().numpy(), lens.tolist())
        assert np.array_equal(lineage.cpu().numpy(), rows)
        scores = picked.scores


def test_lineage_refusals(qa):
    cache = qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 6, 1, 8, 64)
    for beams in (0, -1, 4, 256):
        with pytest.raises(qa.QmmError):
            cache.new_lineage(beams)
    with pytest.raises(qa.QmmError):
        qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 256, 1, 8, 64).new_lineage(256)
    assert (cache.new_lineage() == 0).all()
    assert cache.new_lineage(3)[:, 0].tolist() == [0, 1, 2, 0, 1, 2]
