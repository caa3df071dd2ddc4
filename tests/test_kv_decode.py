"""The quantized cache, shared-prefix attention and beam selection without a GPU: the restatements that the GPU tests
compare with, against the GGUF oracle and brute force, and the refusals of the C entry points."""
import numpy as np
import pytest

import kv_ref


@pytest.fixture(scope="module")
def L():
    from izwi_amd import capi
    return capi.lib()


def test_restated_q8_0_is_the_gguf_block_format(oracle):
    x = oracle.randn(3, (64, 256), std=1.3)
    q, h = kv_ref.quantize(x, 8)
    blocks = np.asarray(oracle.quantize(8, x)).reshape(64, 8, 34)
    assert np.array_equal(blocks[:, :, :2].copy().view(np.float16)[..., 0], h)
    assert np.array_equal(blocks[:, :, 2:].view(np.int8).reshape(64, 256), q)


def test_restated_q4_0_by_hand():
    x = np.zeros((1, 32), np.float32)
    x[0, :6] = [8.0, -8.0, 3.0, 0.49, -0.5, -7.6]  # the first of the two largest decides: scale 8 / -8 = -1
    q, h = kv_ref.quantize(x, 4)
    assert h[0, 0] == -1.0
    # floor(v / -1 + 8.5) - 8, at most 7
    assert q[0, :7].tolist() == [-8, 7, -3, 0, 1, 7, 0]
    assert (np.abs(kv_ref.values(q, h)[0, 2:] - x[0, 2:]) <= 0.5 + (x[0, 2:] < -7)).all()


def test_restated_blocks_that_hold_no_number():
    x = np.ones((5, 32), np.float32)
    x[0, 3], x[1, 5], x[2], x[3] = np.nan, -np.inf, 0.0, 1e-9
    x[4, 0] = 1e30
    for bits in (4, 8):
        q, h = kv_ref.quantize(x, bits)
        v = kv_ref.values(q, h)
        assert np.isnan(v[[0, 1, 4]]).all() and (v[[2, 3]] == 0).all()


def test_restated_beam_step_by_brute_force():
    rng = np.random.default_rng(5)
    logits, scores = rng.normal(size=(2, 3, 7)).astype(np.float32), rng.normal(size=(2, 3)).astype(np.float32)
    tokens, parents, out, _ = kv_ref.beam_select(logits, scores)
    for g in range(2):
        every = sorted((-(scores[g, w] + logits[g, w, t] - np.log(np.exp(logits[g, w].astype(np.float64)).sum())), w, t) for w in range(3) for t in range(7))
        assert [(w, t) for _, w, t in every[:3]] == list(zip(parents[g], tokens[g]))
        assert np.allclose([-s for s, _, _ in every[:3]], out[g], rtol=1e-6)


def test_cache_bytes(L):
    # 2 planes of quants (a byte, half a byte) and 2 of f16 scales, positions rounded up to 32
    assert L.izwi_decode_kv_cache_bytes(8, 2, 8, 33, 128) == 2 * (2 * 8 * 64 * (128 + 8))
    assert L.izwi_decode_kv_cache_bytes(2, 1, 4, 32, 64) == 2 * (4 * 32 * (32 + 4))
    assert L.izwi_decode_kv_cache_bytes(8, 1, 8, 1 << 29, 256) == 2 * (8 * (1 << 29) * (256 + 16))  # 2.3 TB: counted, not allocated
    for args, words in (((12, 1, 8, 32, 128), b"cache type 12"), ((8, 1, 8, 32, 96), b"head_dim 96"), ((8, 0, 8, 32, 128), b"slots 0"),
                        ((8, 1, 0, 32, 128), b"kv heads 0"), ((8, 1, 8, 0, 128), b"capacity 0"), ((8, 1, -1, 32, 128), b"kv heads -1"),
                        ((8, 0xfffff, 0xffff, 0x3fffffff, 256), b"bad cache shape")):
        assert L.izwi_decode_kv_cache_bytes(*args) == 0
        assert words in L.izwi_qmm_last_error()


P = 4096  # a pointer that is aligned and never followed: every call below is refused before any device work


@pytest.mark.parametrize("name", ["f32", "f16"])
def test_append_and_read_refusals(L, name):
    append, read = getattr(L, f"izwi_decode_kv_append_{name}"), getattr(L, f"izwi_decode_kv_read_{name}")
    good = dict(type=8, k=P, v=P, ks=1024, vs=1024, starts=P, counts=0, batch=1, tokens=1, first=0, slots=2, kv=8, cap=64, d=128, cache=P, stream=0)

    def call(**over):
        return append(*{**good, **over}.values())

    for over in (dict(batch=-1), dict(tokens=-1), dict(first=-1), dict(batch=3), dict(first=2), dict(k=0), dict(v=0), dict(starts=0), dict(cache=0),
                 dict(cache=P + 8), dict(ks=1023), dict(vs=0), dict(kv=0), dict(cap=0)):
        assert call(**over) == -1, over
        assert L.izwi_qmm_last_error()
    for over in (dict(type=12), dict(d=32), dict(tokens=1 << 30)):
        assert call(**over) == -2, over
    assert call(batch=0) == 0 and call(tokens=0) == 0

    good_read = dict(type=2, cache=P, slots=6, kv=8, cap=64, d=64, lineage=0, beams=0, starts=P, counts=0, batch=2, tokens=1, first=0, k=P, v=P, stream=0)

    def call_read(**over):
        return read(*{**good_read, **over}.values())

    for over in (dict(batch=7), dict(first=5), dict(starts=0), dict(k=0), dict(v=0), dict(cache=P + 4), dict(lineage=P, beams=0), dict(lineage=P, beams=4),
                 dict(lineage=P, beams=256, slots=256)):
        assert call_read(**over) == -1, over
    assert call_read(d=80) == -2 and call_read(batch=0) == 0


@pytest.mark.parametrize("name", ["f32", "f16"])
def test_attention_refusals(L, name):
    fn = getattr(L, f"izwi_decode_shared_attention_{name}")
    good = dict(type=8, q=P, q_stride=4096, batch=4, beams=2, heads=32, kv=8, d=128, prefix=P, pslots=2, pcap=64, plens=P, maxp=64, cache=P, slots=4,
                cap=32, lens=P, maxl=32, lineage=P, scale=1.0, out=P, stream=0)

    def call(**over):
        return fn(*{**good, **over}.values())

    for over in (dict(batch=-2), dict(beams=0), dict(batch=3), dict(heads=12), dict(heads=0), dict(kv=0), dict(q_stride=4095), dict(q=0), dict(out=0),
                 dict(plens=0), dict(lens=0), dict(pslots=1), dict(slots=3), dict(maxp=65), dict(maxl=33), dict(maxl=-1), dict(prefix=P + 8),
                 dict(cache=P + 2), dict(cache=0), dict(batch=512, beams=256, slots=512), dict(cap=0), dict(heads=65536 * 8)):
        assert call(**over) == -1, over
        assert L.izwi_qmm_last_error()
    assert call(type=14) == -2 and call(d=96, q_stride=1 << 20) == -2
    assert call(batch=0) == 0


def test_beam_select_refusals(L):
    good = dict(logits=P, prompts=2, beams=4, vocab=100, scores=P, finished=0, eos=-1, tokens=P, parents=P, scores_out=P, finished_out=0, lineage=P, cap=64,
                lens=P, lineage_out=P, stream=0)

    def call(**over):
        return L.izwi_decode_beam_select_f32(*{**good, **over}.values())

    for over in (dict(prompts=-1), dict(beams=0), dict(vocab=0), dict(logits=0), dict(scores=0), dict(tokens=0), dict(parents=0), dict(scores_out=0),
                 dict(eos=100), dict(eos=-2), dict(finished=P), dict(lineage=0), dict(lineage_out=0), dict(lens=0), dict(cap=0), dict(lineage=P + 1)):
        assert call(**over) == -1, over
        assert L.izwi_qmm_last_error()
    for over in (dict(beams=65), dict(vocab=1 << 30), dict(prompts=20000)):
        assert call(**over) == -2, over
    assert call(prompts=0) == 0


def test_refusals_of_shared_memory_and_sizes(L):
    for name in ("f32", "f16"):
        fn, size = getattr(L, f"izwi_decode_shared_attention_{name}"), 4 if name == "f32" else 2
        args = dict(type=8, q=P, q_stride=512, batch=2, beams=1, heads=4, kv=2, d=128, prefix=0, pslots=0, pcap=0, plens=0, maxp=0, cache=P, slots=2, cap=32,
                    lens=P, maxl=32, lineage=0, scale=1.0, out=P + 512 * size, stream=0)
        assert fn(*args.values()) == -1 and b"shares memory" in L.izwi_qmm_last_error()
        for scale in (float("nan"), float("inf"), -float("inf")):
            assert fn(*{**args, "out": 1 << 30, "scale": scale}.values()) == -1 and b"scale" in L.izwi_qmm_last_error()
        append = getattr(L, f"izwi_decode_kv_append_{name}")
        assert append(8, P, P, 128, 128, P, 0, 1, 1 << 28, 0, 1, 1, 64, 128, P, 0) == -2 and b"2^24" in L.izwi_qmm_last_error()
    assert L.izwi_decode_beam_select_f32(P, 2, 4, 100, P, 0, -1, P, P, P, 0, P, 64, P, P + 64, 0) == -1 and b"overlap" in L.izwi_qmm_last_error()
