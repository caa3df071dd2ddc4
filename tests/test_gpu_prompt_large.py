"""GPU tests (pytest -m gpu) of the kernels that large calls of the operators on whole prompts take: several tokens to a wave in routing, several sets of heads
to a wave in rotary positions, workgroups of 128 rows over tens of tiles in attention, whole and in parts, and their second pass over values
that are no numbers.  Tolerances: those of test_gpu_prompt_ops.py, of f16 and bf16 attention those of test_gpu_prompt_weights.py."""
import math

import numpy as np
import pytest
import torch

import prompt_ref
from gpu_streams import fresh_stream
from prompt_rows import attention_rows, route_rows
from test_gpu_prompt_ops import check_rope, ints, made, wide
from test_gpu_prompt_weights import check_rows

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def qa():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the HIP path cannot run (there is no fallback)")
    import izwi_amd
    izwi_amd.lib()
    torch.cuda.set_device(0)
    return izwi_amd


@pytest.fixture(scope="module")
def stream(qa):
    return fresh_stream()


# ---- routing ------------------------------------------------------------------------------------------------------------------


def check_route(qa, logits, l64, top_k, scoring, bias, groups, top_groups, group_best, renormalize, scale):
    ids, w = qa.moe_route_scored(logits, top_k, scoring, None if bias is None else torch.from_numpy(bias).cuda(), groups, top_groups, group_best, renormalize, scale)
    want_ids, want_w = route_rows(l64, top_k, scoring, bias, groups, top_groups, group_best, renormalize, scale)
    some = slice(0, 30)
    one_ids, one_w = prompt_ref.route(l64[some], top_k, scoring, bias, groups, top_groups, group_best, renormalize, scale)
    assert np.array_equal(want_ids[some], one_ids) and np.allclose(want_w[some], one_w, rtol=1e-12, atol=1e-300)
    ids, w = ids.cpu().numpy(), w.cpu().double().numpy()
    assert np.array_equal(ids, want_ids), np.flatnonzero((ids != want_ids).any(1))[:10]
    assert (np.abs(w - want_w) <= 2.0 ** -24 * np.abs(want_w) + 2.0 ** -50).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,n,top_k,groups,top_groups,group_best", [
    (1024, 64, 8, 1, 1, 1), (1025, 64, 16, 16, 9, 2), (2051, 65, 3, 5, 2, 2), (1026, 128, 16, 1, 1, 1), (2051, 128, 8, 8, 3, 1), (1027, 96, 8, 16, 8, 2), (4099, 7, 3, 7, 3, 1),
    (8193, 256, 8, 8, 4, 2), (8194, 256, 16, 16, 4, 1), (8195, 130, 5, 1, 1, 1), (1024, 100, 2, 2, 1, 2), (1030, 128, 17, 1, 1, 1), (1030, 128, 8, 32, 8, 2)])
def test_route_scored_of_many_tokens(qa, dtype, scoring, t, n, top_k, groups, top_groups, group_best):
    """As many tokens as get sixteen lanes each (four times, beyond 128 experts 32 times as many as compute units), the last wave with one to four of them; with seventeen
    experts a token or 32 groups sixteen lanes are too few."""
    print("route", dtype, scoring, t, n, top_k, groups, top_groups, group_best, flush=True)
    rng = np.random.default_rng(t + n)
    logits, l64 = made(rng, t, n + 1, dtype=dtype, std=2.0)
    logits, l64 = logits[:, :n], l64[:, :n]
    b = (rng.normal(size=n) * 0.1).astype(np.float32)
    for bias, renormalize, scale in ((None, True, 2.5), (None, False, 1.0), (b, True, 1.0), (b, False, 2.5)):
        check_route(qa, logits, l64, top_k, scoring, bias, groups, top_groups, group_best, renormalize, scale)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,n,groups,top_groups,group_best", [(1029, 24, 1, 1, 1), (2050, 96, 4, 2, 2), (2049, 128, 8, 3, 1), (8197, 256, 16, 5, 2)])
def test_route_scored_of_many_tokens_with_ties_and_no_numbers(qa, scoring, t, n, groups, top_groups, group_best):
    """Whole numbers as logits, so that most rows hold ties; rows of NaN, of -infinity and of zeros next to others of the same wave."""
    rng = np.random.default_rng(t)
    l = rng.integers(-2, 3, size=(t, n)).astype(np.float32)
    l[::7] = 0.0
    l[1::13] = np.nan
    l[2::17] = -np.inf
    l[3::11, ::3] = np.nan
    l[4::19, 5] = np.inf
    l[t - 1] = 1.0
    for bias in (None, (rng.integers(-1, 2, size=n) * 0.25).astype(np.float32)):
        for renormalize in (True, False):
            check_route(qa, torch.from_numpy(l).cuda(), l, 5, scoring, bias, groups, top_groups, group_best, renormalize, 1.0)


# ---- rotary positions -----------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv,d,r,inter,norm", [
    (2051, 32, 8, 128, 128, False, True), (1300, 32, 8, 128, 128, True, False), (5000, 32, 8, 128, 64, False, True), (4100, 17, 3, 128, 128, False, True), (2300, 40, 1, 64, 32, True, True),
    (9000, 5, 4, 64, 64, False, False), (4200, 6, 5, 256, 256, False, True)])
def test_rope_positions_of_several_sets_of_heads_a_wave(qa, dtype, tokens, heads, kv, d, r, inter, norm):
    """Two to ten sets a wave, more than are requested at once and numbers that do not divide by the waves of a token, as rows of their own, as parts of q|k|v rows and in
    place."""
    print("rope", dtype, tokens, heads, kv, d, r, inter, norm, flush=True)
    rng = np.random.default_rng(tokens + d)
    rotary = qa.RotaryEmbedding(d, base=1e6, rotary_dim=r, interleaved=inter)
    freqs = rotary.frequencies.cpu().numpy()
    positions = rng.integers(0, 2 ** 20, size=tokens)
    weight, w64 = made(rng, 2 * d, dtype=dtype) if norm else (None, None)
    (q, q64), (k, k64), _ = wide(rng, tokens, heads, kv, kv, d=d, dtype=dtype)
    some = np.unique(np.concatenate([np.arange(0, tokens, 97), np.arange(max(0, tokens - 9), tokens)]))
    got = qa.rope_positions(q, k, ints(positions), rotary, weight, 1e-5)
    for i, (g, x64) in enumerate(zip(got, (q64, k64))):
        check_rope(g[torch.from_numpy(some)], x64[some], positions[some], freqs, 1.0, inter, None if w64 is None else w64[i * d:(i + 1) * d], 1e-5, dtype)
    own = qa.rope_positions(q.contiguous(), k.contiguous(), ints(positions), rotary, weight, 1e-5)
    assert torch.equal(own[0], got[0]) and torch.equal(own[1], got[1])
    at = 1000  # (fewer tokens: the same kernel with one set a wave)
    few = qa.rope_positions(q[at:at + 3], k[at:at + 3], ints(positions[at:at + 3]), rotary, weight, 1e-5)
    assert torch.equal(few[0], got[0][at:at + 3]) and torch.equal(few[1], got[1][at:at + 3])
    qa.rope_positions(q, k, ints(positions), rotary, weight, 1e-5, out=(q, k))
    assert torch.equal(q, got[0]) and torch.equal(k, got[1])


# ---- attention --------------------------------------------------------------------------------------------------------------------


def check_f32(got, q64, k64, v64, starts, starts_k, causal, scale, tokens):
    want, n, size, most = attention_rows(q64, k64, v64, starts, starts_k, causal, scale, tokens)
    score = size * ((6 * q64.shape[2] / 16 + 20) * U + 2.0 ** -22)
    tol = (most * (2 * (score + 2.0 ** -22) + (6 * n / 16 + 64) * U + 2.0 ** -22))[..., None] + U * np.abs(want)
    off = np.abs(got[tokens].cpu().double().numpy() - want) / tol
    assert (off <= 1).all(), float(np.nanmax(off))


def sampled(starts, each):
    """The first, the last and some tokens between of every sequence."""
    return sorted({int(t) for a, b in zip(starts, starts[1:]) if b > a for t in np.linspace(a, b - 1, each)})


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,causal,lens,heads,kv", [
    (128, True, [1501, 775, 1, 1203, 999, 0, 1337, 1400, 1111, 1268], 32, 8), (64, True, [2500, 1500], 32, 8), (64, False, [1500, 867, 1200, 1333], 16, 16), (128, False, [1100, 2, 900], 32, 8),
    (256, True, [2000, 300], 16, 8), (256, False, [1000, 901], 16, 8), (128, True, [3300], 16, 8), (64, True, [4200], 16, 8)])
def test_prompt_attention_of_long_prompts(qa, dtype, d, causal, lens, heads, kv):
    """Tens of tiles to a workgroup of 128 rows, those that every row sees in front of a causal triangle; sequences by their offsets and by length."""
    print("attention", dtype, d, causal, lens, heads, kv, flush=True)
    rng = np.random.default_rng(d + sum(lens))
    starts = np.cumsum([0] + lens)
    (q, q64), (k, k64), (v, v64) = wide(rng, starts[-1], heads, kv, kv, d=d, dtype=dtype)
    scale = 1.5 * d ** -0.5
    got = qa.prompt_attention(q, k, v, ints(starts), causal=causal, scale=scale, max_len_k=max(lens))
    tokens = sampled(starts, 5 if len(lens) > 2 else 9)
    if dtype == "f32":
        check_f32(got, q64, k64, v64, starts, starts, causal, scale, tokens)
    else:
        check_rows(got, q64, k64, v64, starts, starts, causal, scale, dtype, tokens)
    assert torch.equal(got, qa.prompt_attention(q, k, v, ints(starts), causal=causal, scale=scale, max_len_k=max(lens)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,past,heads,kv", [([17], [8300], 32, 8), ([33, 20, 70], [8200, 0, 9100], 16, 4), ([9], [8300], 16, 8)])
def test_prompt_attention_of_a_chunk_behind_a_long_past(qa, stream, dtype, d, causal, lens, past, heads, kv):
    """More than 64 rows on more than 8192 keys, workgroups of 128 rows in parts, and fewer, in the smaller ones, also on a stream of its own and captured, replayed on new values."""
    print("chunk", dtype, d, causal, lens, past, flush=True)
    rng = np.random.default_rng(d + sum(past))
    starts, starts_k = np.cumsum([0] + lens), np.cumsum([0] + [a + b for a, b in zip(lens, past)])
    (q, q64), (k, k64), (v, v64) = (made(rng, n, g, d, dtype=dtype) for n, g in ((starts[-1], heads), (starts_k[-1], kv), (starts_k[-1], kv)))
    offsets, offsets_k, scale = ints(starts), ints(starts_k), 2.0 * d ** -0.5
    run = lambda **more: qa.prompt_attention(q, k, v, offsets, offsets_k, causal=causal, scale=scale, **more)  # noqa: E731
    check = lambda got, *x: check_f32(got, *x, starts, starts_k, causal, scale, tokens) if dtype == "f32" else check_rows(got, *x, starts, starts_k, causal, scale, dtype, tokens)  # noqa: E731
    tokens = sampled(starts, 4)
    check(run(), q64, k64, v64)
    out = torch.zeros_like(q)
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            run(out=out)
    torch.cuda.current_stream().wait_stream(stream)
    for _ in range(2):
        v2 = made(rng, *v.shape, dtype=dtype)
        v.copy_(v2[0]), out.fill_(3)
        graph.replay()
        check(out, q64, k64, v2[1])
        assert torch.equal(out, run())


@pytest.mark.parametrize("dtype,d,n,heads,kv", [(t, d, n, 32, 8) for t in ("f16", "bf16") for d in (64, 128, 256) for n in (150, 2100)] +
                         [("f32", 64, 4200, 16, 8), ("f32", 64, 900, 16, 8), ("f32", 128, 3000, 16, 8), ("f32", 128, 700, 16, 8), ("f32", 256, 1200, 16, 8), ("f32", 256, 100, 16, 8)])
@pytest.mark.parametrize("bad", [math.nan, -math.inf])
def test_prompt_attention_of_values_that_are_no_numbers_in_every_kernel(qa, dtype, d, n, heads, kv, bad):
    """A causal prompt and a second one behind it, a value that is no number early, in the middle and last: rows that do not see it are as they were to the bit, rows that do
    have it in its element alone."""
    rng = np.random.default_rng(n + d)
    (q, _), (k, _), (v, _) = (made(rng, n + 70, g, d, dtype=dtype) for g in (heads, kv, kv))
    starts = ints([0, n, n + 70])
    clean = qa.prompt_attention(q, k, v, starts)
    other = torch.arange(d, device="cuda") != d - 3
    for at in (1, n // 2, n - 1):
        values = v.clone()
        values[at, kv // 2, d - 3] = bad
        got = qa.prompt_attention(q, k, values, starts)
        sees = torch.zeros(n + 70, heads, dtype=torch.bool, device="cuda")
        sees[at:n, kv // 2 * (heads // kv):(kv // 2 + 1) * (heads // kv)] = True
        assert torch.equal(got[~sees], clean[~sees])
        assert torch.equal(got[..., other], clean[..., other])
        hit = got[..., d - 3][sees]
        assert torch.isnan(hit).all() if bad != bad else (~torch.isfinite(hit)).all() if dtype == "f32" else (hit == bad).all()


def test_route_scored_numbers_beyond_32_bits(qa):
    """Numbers that 32 bits would cut to ones that fit."""
    x = torch.zeros(4, 16, device="cuda")
    for over in (dict(top_k=2 ** 32 + 2), dict(groups=2 ** 32 + 1), dict(groups=4, top_groups=2 ** 32 + 2), dict(groups=4, top_groups=2, group_best=2 ** 32 + 1), dict(groups=-4), dict(group_best=0)):
        with pytest.raises(qa.QmmError):
            qa.moe_route_scored(**{**dict(logits=x, top_k=2), **over})
