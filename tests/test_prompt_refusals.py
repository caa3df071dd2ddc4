"""Calls of the operators on whole prompts that are refused before any device work: the pointers are aligned and never followed."""
import pytest

FAR = 1 << 32
NAMES = ["f32", "f16", "bf16"]


@pytest.fixture(scope="module")
def L():
    from izwi_amd import capi
    return capi.lib()


@pytest.mark.parametrize("name", NAMES)
def test_rope_positions_outputs_lie_apart_from_everything_else(L, name):
    """Positions, frequencies and weights are inputs as q and k are (which an output may be), up to their last byte."""
    fn, size = getattr(L, f"izwi_rope_positions_{name}"), 4 if name == "f32" else 2
    good = dict(q=FAR, qs=1024, k=2 * FAR, ks=512, positions=5 * FAR, frequencies=6 * FAR, factor=1.0, tokens=4, heads=8, kv=4, d=128, rotary=128, inter=0, weight=7 * FAR, eps=1e-6,
                qo=FAR, qos=1024, ko=2 * FAR, kos=512, stream=0)
    q_end, k_end = FAR + 4 * 1024 * size, 2 * FAR + 4 * 512 * size
    for over in (dict(positions=FAR), dict(positions=q_end - 4), dict(positions=FAR - 12), dict(positions=k_end - 4), dict(frequencies=FAR - 64 * 8 + 8), dict(frequencies=k_end - 8),
                 dict(weight=FAR - 256 * size + 16), dict(weight=q_end - 16), dict(weight=2 * FAR)):
        assert fn(*{**good, **over}.values()) == -1, over
        assert b"shares memory with positions" in L.izwi_qmm_last_error()


@pytest.mark.parametrize("name", NAMES)
def test_prompt_attention_out_lies_apart_from_the_offsets(L, name):
    fn, size = getattr(L, f"izwi_qmm_prompt_attention_{name}"), 4 if name == "f32" else 2
    good = dict(q=FAR, qs=1024, k=2 * FAR, ks=256, v=3 * FAR, vs=256, cu_q=4 * FAR, cu_k=5 * FAR, batch=2, tq=10, tk=20, mk=20, heads=8, kv=2, d=128, causal=1, scale=0.1, out=6 * FAR,
                os=1024, stream=0)
    end = 6 * FAR + 10 * 1024 * size
    for over in (dict(cu_q=6 * FAR), dict(cu_k=end - 4), dict(cu_q=6 * FAR - 8), dict(cu_k=6 * FAR + 512)):
        assert fn(*{**good, **over}.values()) == -1, over
        assert b"shares memory with the offsets" in L.izwi_qmm_last_error()


@pytest.mark.parametrize("name", NAMES)
def test_as_many_tokens_as_a_launch_takes(L, name):
    """Four tokens to a workgroup of 256 threads, below 2^32 threads: 2^26 - 4 tokens.  (That many pass this check and are refused for outputs that overlap.)"""
    rope, route = getattr(L, f"izwi_rope_positions_{name}"), getattr(L, f"izwi_moe_route_scored_{name}")
    for tokens, rc in ((2 ** 26 - 4, -1), (2 ** 26 - 3, -2), (2 ** 26 - 1, -2), (2 ** 26, -2)):
        assert rope(FAR, 64, 0, 0, FAR, FAR, 1.0, tokens, 1, 0, 64, 64, 0, 0, 1e-6, FAR + 64, 64, 0, 0, 0) == rc
        assert route(FAR, 512, 0, tokens, 512, 8, 0, 1, 1, 1, 1, 1.0, FAR, FAR, 0) == rc
