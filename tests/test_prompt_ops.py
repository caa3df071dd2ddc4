"""Rotary positions, prompt attention and scored routing without a GPU: the frequencies, the restatements that the GPU tests compare with
against other formulations, and the refusals of the C entry points."""
import ctypes as C
import math

import numpy as np
import pytest

import prompt_ref


@pytest.fixture(scope="module")
def L():
    from izwi_amd import capi
    return capi.lib()


CASES = [("none", {}), ("linear", dict(factor=4.0)), ("ntk", dict(factor=2.0)), ("llama3", dict(factor=8.0, original=8192, low=1, high=4)),
         ("llama3", dict(factor=32.0, original=777, low=1.5, high=2.5)), ("yarn", dict(factor=4.0, original=32768, low=1, high=32)),
         ("yarn", dict(factor=2.0, original=10, low=1, high=32))]


@pytest.mark.parametrize("kind,how", CASES)
@pytest.mark.parametrize("r,base", [(128, 1e6), (64, 1e4), (6, 5e5)])
def test_frequencies(kind, how, r, base):
    from izwi_amd import prompt_ops as ops
    S = ops.RopeScaling
    scaling = {"none": lambda: None, "linear": lambda: S.linear(how["factor"]), "ntk": lambda: S.ntk(how["factor"]),
               "llama3": lambda: S.llama3(how["factor"], how["original"], how["low"], how["high"]),
               "yarn": lambda: S.yarn(how["factor"], how["original"], how["low"], how["high"])}[kind]()
    got, factor = ops.rope_frequencies(r, base, scaling)
    want, m = prompt_ref.frequencies(kind, r, base, **how)
    assert np.allclose(got, want, rtol=1e-14, atol=0) and factor == pytest.approx(m, rel=1e-15)
    assert len(got) == r // 2


def test_frequencies_of_factor_one_are_the_plain_ones():
    from izwi_amd import prompt_ops as ops
    S = ops.RopeScaling
    plain, one = ops.rope_frequencies(96, 1e4)
    assert one == 1.0
    for scaling in (S.linear(1.0), S.ntk(1.0), S.llama3(1.0, 4096), S.yarn(1.0, 4096)):
        got, m = ops.rope_frequencies(96, 1e4, scaling)
        assert np.allclose(got, plain, rtol=1e-15) and m == 1.0
    assert ops.rope_frequencies(96, 1e4, S.yarn(4.0, 4096, attention_factor=0.75))[1] == 0.75


def test_restated_rope_is_a_turn_in_the_plane():
    rng = np.random.default_rng(1)
    x, f = rng.normal(size=(3, 2, 12)), np.array([1.0, 0.3, 0.01])
    for inter in (False, True):
        y = prompt_ref.rope(x, [0, 1, 9], f, 1.0, inter)
        assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 6:], x[..., 6:])
        pair = (lambda z: z[..., 0:6:2] + 1j * z[..., 1:6:2]) if inter else (lambda z: z[..., :3] + 1j * z[..., 3:6])
        assert np.allclose(pair(y), pair(x) * np.exp(1j * np.array([0, 1, 9])[:, None, None] * f))


def test_restated_attention_by_masks():
    rng = np.random.default_rng(2)
    q, k, v = rng.normal(size=(7, 4, 8)), rng.normal(size=(9, 2, 8)), rng.normal(size=(9, 2, 8))
    out, seen, _, _ = prompt_ref.attention(q, k, v, [0, 3, 7], [0, 5, 9], True, 0.5)
    for (a, b, c, d) in ((0, 3, 0, 5), (3, 7, 5, 9)):
        mask = np.tril(np.ones((b - a, d - c)), (d - c) - (b - a)) > 0
        for h in range(4):
            s = np.where(mask, q[a:b, h] @ k[c:d, h // 2].T * 0.5, -np.inf)
            p = np.exp(s) / np.exp(s).sum(1, keepdims=True)
            assert np.allclose(out[a:b, h], p @ v[c:d, h // 2])
            assert seen[a:b, h].tolist() == mask.sum(1).tolist()


def test_restated_routing_by_brute_force():
    rng = np.random.default_rng(3)
    logits, bias = rng.normal(size=(5, 12)), rng.normal(size=12) * 0.1
    ids, w = prompt_ref.route(logits, 3, "sigmoid", bias, 4, 2, 2, True, 2.5)
    for t in range(5):
        s = 1 / (1 + np.exp(-logits[t]))
        c = s + bias
        best = max(((sum(sorted(c[3 * g:3 * g + 3])[1:]), -g) for g in range(4)))
        assert -best[1] in {i // 3 for i in range(12) if i // 3 == -best[1]}
        worth = np.sort(c.reshape(4, 3), 1)[:, 1:].sum(1)
        allowed = np.isin(np.arange(12) // 3, np.argsort(-worth)[:2])
        want = np.argsort(-np.where(allowed, c, -9))[:3]
        assert ids[t].tolist() == want.tolist()
        assert np.allclose(w[t], s[want] / s[want].sum() * 2.5)


P = 4096  # a pointer that is aligned and never followed: every call below is refused before any device work
NAMES = ["f32", "f16", "bf16"]


@pytest.mark.parametrize("name", NAMES)
def test_rope_positions_refusals(L, name):
    fn, size = getattr(L, f"izwi_rope_positions_{name}"), 4 if name == "f32" else 2
    far = 1 << 30
    good = dict(q=P, qs=1024, k=far, ks=512, positions=P, frequencies=P, factor=1.0, tokens=4, heads=8, kv=4, d=128, rotary=128, inter=0, weight=0, eps=1e-6,
                qo=2 * far, qos=1024, ko=3 * far, kos=512, stream=0)

    def call(**over):
        return fn(*{**good, **over}.values())

    nan = float("nan")
    for over in (dict(tokens=-1), dict(heads=-1), dict(kv=-1), dict(d=0), dict(d=127), dict(d=1026, rotary=2, qs=1 << 20, ks=1 << 20, qos=1 << 20, kos=1 << 20),
                 dict(rotary=0), dict(rotary=3), dict(rotary=130), dict(qs=1023), dict(ks=511), dict(qos=1023), dict(kos=511), dict(inter=2), dict(factor=nan),
                 dict(eps=-1.0), dict(eps=nan), dict(q=0), dict(k=0), dict(positions=0), dict(frequencies=0), dict(qo=0), dict(ko=0),
                 dict(heads=65536, qs=1 << 24, qos=1 << 24),
                 dict(qo=P + 2 * size), dict(qo=P, qos=2048), dict(ko=P), dict(qo=far), dict(ko=2 * far), dict(ko=far + 512 * size)):
        assert call(**over) == -1, over
        assert L.izwi_qmm_last_error()
    assert call(tokens=1 << 30) == -2
    assert call(tokens=0) == 0 and call(heads=0, kv=0) == 0


def test_rope_frequencies_refusals(L):
    f, m = (C.c_double * 64)(), C.c_double()
    good = dict(kind=4, r=128, base=1e6, factor=4.0, original=8192.0, low=1.0, high=32.0, f=f, m=C.byref(m))
    assert L.izwi_rope_frequencies(*good.values()) == 0
    for over in (dict(kind=5), dict(kind=-1), dict(r=0), dict(r=7), dict(r=2048), dict(base=1.0), dict(base=math.inf), dict(factor=0.5), dict(factor=math.nan),
                 dict(original=0.0), dict(low=0.0), dict(low=32.0), dict(high=math.inf), dict(f=None), dict(m=None), dict(kind=2, r=2)):
        assert L.izwi_rope_frequencies(*{**good, **over}.values()) == -1, over


@pytest.mark.parametrize("name", NAMES)
def test_prompt_attention_refusals(L, name):
    fn, size = getattr(L, f"izwi_qmm_prompt_attention_{name}"), 4 if name == "f32" else 2
    far = 1 << 30
    good = dict(q=P, qs=1024, k=far, ks=256, v=2 * far, vs=256, cu_q=P, cu_k=P, batch=2, tq=10, tk=20, mk=20, heads=8, kv=2, d=128, causal=1, scale=0.1, out=3 * far,
                os=1024, stream=0)

    def call(**over):
        return fn(*{**good, **over}.values())

    for over in (dict(batch=-1), dict(tq=-1), dict(tk=-1), dict(mk=-1), dict(heads=0), dict(kv=0), dict(heads=7), dict(cu_q=0), dict(cu_k=0), dict(cu_q=0, cu_k=0),
                 dict(qs=1023), dict(qs=1016), dict(ks=255), dict(vs=128), dict(os=512), dict(scale=math.nan), dict(scale=-math.inf), dict(scale=3e38), dict(q=P + 8), dict(k=far + 2), dict(v=P + 4),
                 dict(out=far + 8), dict(qs=1025), dict(ks=257), dict(q=0), dict(k=0), dict(v=0), dict(out=0), dict(out=P), dict(out=P + 1024 * size * 9),
                 dict(out=far), dict(out=2 * far + 256 * size), dict(heads=65536 * 2, qs=1 << 28, os=1 << 28)):
        assert call(**over) == -1, over
        assert L.izwi_qmm_last_error()
    for over in (dict(d=96), dict(d=32), dict(tq=1 << 28), dict(tk=1 << 30), dict(ks=1 << 24), dict(vs=1 << 24), dict(batch=0xfffff, kv=8, ks=1024, vs=1024)):
        assert call(**over) == -2, over
    assert call(batch=0) == 0 and call(tq=0) == 0


@pytest.mark.parametrize("name", NAMES)
def test_route_scored_refusals(L, name):
    fn, size = getattr(L, f"izwi_moe_route_scored_{name}"), 4 if name == "f32" else 2
    far = 1 << 30
    good = dict(logits=P, stride=128, bias=far, t=3, n=128, k=8, scoring=1, groups=8, top=4, best=2, renorm=1, scale=1.0, ids=2 * far, w=3 * far, stream=0)

    def call(**over):
        return fn(*{**good, **over}.values())

    for over in (dict(t=-1), dict(n=0), dict(stride=127), dict(groups=0), dict(groups=7), dict(groups=65, n=130, stride=130), dict(top=0), dict(top=9), dict(best=0), dict(best=3),
                 dict(k=0), dict(k=65), dict(k=33, top=2), dict(scoring=2), dict(scoring=-1), dict(scale=math.nan), dict(logits=0), dict(ids=0), dict(w=0),
                 dict(ids=P), dict(w=P + 130 * size), dict(ids=3 * far + 4), dict(w=far), dict(ids=far + 508)):
        assert call(**over) == -1, over
        assert L.izwi_qmm_last_error()
    assert call(n=1032, stride=1032) == -2 and call(t=1 << 30) == -2
    assert call(t=0) == 0


def test_python_refusals_without_a_gpu():
    import torch

    import izwi_amd
    x = torch.zeros(4, 8, 64)
    for call in (lambda: izwi_amd.prompt_attention(x, x, x), lambda: izwi_amd.moe_route_scored(torch.zeros(3, 8), 2), lambda: izwi_amd.RotaryEmbedding(64, device="cpu"),
                 lambda: izwi_amd.RotaryEmbedding(64, rotary_dim=66), lambda: izwi_amd.prompt_ops.rope_frequencies(0)):
        with pytest.raises(izwi_amd.QmmError):
            call()
