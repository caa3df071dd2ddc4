"""GPU tests (pytest -m gpu) of attention on parts of other tensors: query rows at odd addresses, a lineage at one, one cache as prefix and as own."""
import numpy as np
import pytest
import torch

import kv_ref
from test_gpu_kv_decode import check_attention, dev, draw, ints, make, qa  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", (64, 128, 256))
def test_f16_query_rows_at_odd_addresses(qa, d):
    rng = np.random.default_rng(d)
    cache, _ = make(qa, rng, "Q4_0", "f16", 5, 2, 50, d)
    wide = dev(draw(rng, 5, 4 * d + 9, dtype="f16"), "f16")
    for at in (0, 1, 2, 3, 8, 9):
        q = wide[:, at:at + 4 * d].unflatten(-1, (4, d))
        a, b = (qa.shared_prefix_attention(x, cache, ints([50, 3, 0, 1, 49]), beams=1) for x in (q, q.contiguous()))
        assert torch.equal(a, b)


def test_lineage_at_an_odd_address(qa):
    rng = np.random.default_rng(7)
    cache, ref = make(qa, rng, "Q8_0", "f32", 6, 2, 60, 128)
    rows = rng.integers(0, 3, size=(6, 64)).astype(np.uint8)
    q, lens = draw(rng, 6, 4, 128), [60, 59, 33, 32, 1, 0]
    for at in range(4):
        room = torch.zeros(6 * 64 + 4, dtype=torch.uint8, device="cuda")
        lineage = room[at:at + 6 * 64].view(6, 64)
        lineage.copy_(torch.from_numpy(rows))
        got = qa.shared_prefix_attention(dev(q), cache, ints(lens), beams=3, lineage=lineage)
        check_attention(got, kv_ref.attention(q, ref, lens, lineage=rows, beams=3, scale=128 ** -0.5), "f32", 128)
        k, v = cache.read(ints([0] * 6), 60, ints(lens), lineage=lineage, beams=3)
        for x, y in zip((k, v), ref.read([0] * 6, 60, lens, lineage=rows, beams=3)):
            assert np.array_equal(x.cpu().numpy(), y)


def test_one_cache_as_prefix_and_as_own(qa):
    """Positions that count twice."""
    rng = np.random.default_rng(8)
    cache, ref = make(qa, rng, "Q8_0", "f32", 4, 2, 70, 64)
    q, plens, lens = draw(rng, 4, 6, 64), [70, 5, 0, 33], [70, 0, 9, 32]
    got = qa.shared_prefix_attention(dev(q), cache, ints(lens), prefix=cache, prefix_lens=ints(plens), beams=1)
    check_attention(got, kv_ref.attention(q, ref, lens, ref, plens, beams=1, scale=64 ** -0.5), "f32", 64)
