"""GPU tests (pytest -m gpu) of rotary positions, prompt attention and scored routing against the 64-bit restatements of prompt_ref.py, through the
Python entry points.

Tolerances, u = 2^-24, h half a step of the type relative to the value (f32 2^-24, f16 2^-11, bf16 2^-8).
Rotary positions: the fraction of a turn is rounded once to 32 bits (at most 2^-26 turns: 2^-23.3 radians), cosine and sine are good to 4 u and
multiplied by the factor, the norm (sums of at most 64 terms a lane and six steps over lanes, a root, a quotient, two products) to 40 u with 32
for the longest heads: a result is off by at most (|a| + |b|) factor (2^-23 + 64 u) + h |out|, subnormal f16 by half a step of 2^-24.
Attention: with A the largest sum of |q_i k_i| scale of a row, V the largest |v| it sees, n its keys, N the products a value goes as (1, f32 6):
a score is off by at most A ((N d / 16 + 16) u for the f32 sum of 16-term steps + 4 u for scale and exponent, f32 2^-23 more for the products left out),
a weight relatively by that + 2^-22 and where weights are rounded h more (f16 ones below 2^-21 of the largest by 2^-32), a mean by twice the former
and once the rounding times V, its sums by (N n / 16 + 64) u V, the result by h |out| + 2^-23 V.
Routing: ids exactly, weights 2^-24 relatively + 2^-50."""
import math

import numpy as np
import pytest
import torch

import prompt_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {name: torch.finfo(t).eps / 2 for name, t in DTYPES.items()}  # 2^-24, 2^-11, 2^-8: in [1, 2) a step is eps


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


def made(rng, *shape, dtype="f32", std=1.0):
    """Values of the type, as a tensor on the GPU and in 64 bits."""
    x = torch.from_numpy((rng.normal(size=shape) * std).astype(np.float32)).to(DTYPES[dtype])
    return x.cuda(), x.double().numpy()


def wide(rng, tokens, *heads, d, dtype="f32", std=1.0):
    """Tensors [tokens, heads, d] as parts of one wider row."""
    x, x64 = made(rng, tokens, sum(heads), d, dtype=dtype, std=std)
    at = np.cumsum((0,) + heads)
    return [(x[:, a:b], x64[:, a:b]) for a, b in zip(at, at[1:])]


# ---- rotary positions ----------------------------------------------------------------------------------------------------


def check_rope(got, x64, positions, freqs, factor, inter, weight, eps, dtype):
    want = prompt_ref.rope(x64, positions, freqs, factor, inter, weight, eps)
    x = x64 if weight is None else x64 / np.sqrt((x64 * x64).mean(-1, keepdims=True) + eps) * weight
    r = 2 * len(freqs)
    near = np.abs(x)
    a, b = (slice(0, r, 2), slice(1, r, 2)) if inter else (slice(0, r // 2), slice(r // 2, r))
    pair = near[..., a] + near[..., b]
    near[..., a] = near[..., b] = pair
    got = got.cpu().double().numpy()
    tol = near * max(1.0, abs(factor)) * (2.0 ** -23 + 64 * U) + HALF[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 0)
    if weight is None:
        assert np.array_equal(got[..., r:], x64[..., r:])
    assert (np.abs(got - want) <= tol).all(), float((np.abs(got - want) / tol).max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,heads,kv,d,r,inter,norm", [
    (1, 16, 8, 128, 128, False, True), (1, 1, 1, 64, 64, True, False), (37, 32, 8, 128, 128, False, True), (5, 12, 12, 64, 32, True, True),
    (300, 4, 1, 256, 64, False, False), (9, 3, 2, 80, 80, False, True), (4, 5, 1, 96, 24, True, False), (3, 2, 2, 2, 2, False, True), (2, 3, 1, 1024, 1024, True, True),
    (700, 7, 1, 128, 32, False, True), (11, 2, 1, 70, 34, False, True), (1025, 2, 2, 64, 64, False, False), (6, 40, 8, 128, 64, True, True), (3, 1, 1, 512, 256, False, True)])
def test_rope_positions(qa, dtype, tokens, heads, kv, d, r, inter, norm):
    print("rope", dtype, tokens, heads, kv, d, r, inter, norm, flush=True)
    rng = np.random.default_rng(tokens * 100 + d)
    rotary = qa.RotaryEmbedding(d, base=1e6, rotary_dim=r, interleaved=inter, scaling=qa.RopeScaling.yarn(4.0, 8192) if tokens % 2 else None)
    freqs, factor = rotary.frequencies.cpu().numpy(), rotary.attention_factor
    positions = rng.integers(-3, 2 ** 20, size=tokens)
    positions[0] = 0
    if tokens > 2:
        positions[1], positions[2] = 2 ** 31 - 1, -2 ** 31
    weight, w64 = made(rng, 2 * d, dtype=dtype) if norm else (None, None)
    eps = 1e-5
    (q, q64), (k, k64) = made(rng, tokens, heads, d, dtype=dtype, std=2), made(rng, tokens, kv, d, dtype=dtype)
    for packed in (False, True):
        if packed:
            (q, q64), (k, k64), _ = wide(rng, tokens, heads, kv, kv, d=d, dtype=dtype)
        before = q.clone(), k.clone()
        got = qa.rope_positions(q, k, ints(positions), rotary, weight, eps)
        assert torch.equal(q, before[0]) and torch.equal(k, before[1])
        for i, (g, x64) in enumerate(zip(got, (q64, k64))):
            check_rope(g, x64, positions, freqs, factor, inter, None if w64 is None else w64[i * d:(i + 1) * d], eps, dtype)
        again = qa.rope_positions(q, k, ints(positions), rotary, weight, eps, out=(q, k))  # in place
        assert again[0] is q and torch.equal(q, got[0]) and torch.equal(k, got[1])
        alone, none = qa.rope_positions(before[0], None, ints(positions), rotary, weight, eps)
        assert none is None and torch.equal(alone, got[0])


def test_rope_positions_of_odd_addresses(qa):
    """Rows and outputs that begin anywhere, results as those of aligned ones."""
    rng = np.random.default_rng(5)
    rotary = qa.RotaryEmbedding(64, base=1e4)
    for dtype in DTYPES:
        room = made(rng, 7 * (5 * 64 + 3) + 8, dtype=dtype)[0]
        q = room[1:].as_strided((7, 4, 64), (5 * 64 + 3, 64, 1))
        k = room[1 + 4 * 64:].as_strided((7, 1, 64), (5 * 64 + 3, 64, 1))
        positions, weight = ints(range(100, 107)), made(rng, 128 + 1, dtype=dtype)[0][1:].contiguous()
        want = qa.rope_positions(q.contiguous(), k.contiguous(), positions, rotary, weight)
        kept = room.clone()
        out = qa.rope_positions(q, k, positions, rotary, weight, out=(q, k))
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        kept.as_strided((7, 5 * 64), (5 * 64 + 3, 1), 1).copy_(torch.cat((out[0].reshape(7, -1), out[1].reshape(7, -1)), 1))
        assert torch.equal(kept, room)  # nothing else was written


def test_rope_positions_of_far_offsets(qa):
    """Rows whose offsets pass 32 bits."""
    step = 1 << 21
    rotary = qa.RotaryEmbedding(128)
    room = torch.empty(2100 * step + 4096, dtype=torch.bfloat16, device="cuda")
    q = torch.randn(2100, 3, 128, device="cuda").bfloat16()
    view = room.as_strided(q.shape, (step, 128, 1))
    view.copy_(q)
    got, _ = qa.rope_positions(view, None, ints(range(2100)), rotary, out=(view, None))
    want, _ = qa.rope_positions(q, None, ints(range(2100)), rotary)
    assert torch.equal(got, want)
    odd = room[1:].as_strided(q.shape, (step, 128, 1))  # no row begins on 16 bytes
    odd.copy_(q)
    assert torch.equal(qa.rope_positions(odd, None, ints(range(2100)), rotary)[0], want)


def test_rope_positions_of_no_numbers(qa):
    """A NaN or infinity reaches its pair (with a norm its head) and nothing else; what does not turn is copied."""
    rotary = qa.RotaryEmbedding(128, rotary_dim=64)
    x = torch.ones(3, 2, 128, device="cuda")
    x[1, 0, 5], x[1, 1, 100], x[2, 0, 127] = math.nan, math.inf, -math.inf
    y, _ = qa.rope_positions(x, None, ints([3, 4, 5]), rotary)
    bad = ~torch.isfinite(y)
    assert bad.nonzero().tolist() == [[1, 0, 5], [1, 0, 37], [1, 1, 100], [2, 0, 127]]
    assert y[1, 1, 100] == math.inf and y[2, 0, 127] == -math.inf
    y, _ = qa.rope_positions(x, None, ints([3, 4, 5]), rotary, torch.ones(256, device="cuda"))
    assert torch.isfinite(y[0]).all() and torch.isnan(y[1, 0]).all() and (y[2, 0, :127] == 0).all()


# ---- attention ---------------------------------------------------------------------------------------------------------------


def check_attention(got, q64, k64, v64, starts, starts_k, causal, scale, dtype, untouched=None):
    want, n, a, big = prompt_ref.attention(q64, k64, v64, starts, starts_k, causal, scale)
    got = got.cpu().double().numpy()
    inside = np.zeros(got.shape[0], bool)
    for b in range(len(starts) - 1):
        inside[starts[b]:starts[b + 1]] = True
    if untouched is not None:
        assert (got[~inside] == untouched).all()
    terms = 6 if dtype == "f32" else 1
    score = a * ((terms * q64.shape[2] / 16 + 20) * U + (2.0 ** -23 if dtype == "f32" else 0))
    weight = 2 * (score + 2.0 ** -22) + (0 if dtype == "f32" else HALF[dtype]) + (n * 2.0 ** -32 if dtype == "f16" else 0)
    tol = (big * (weight + (terms * n / 16 + 64) * U + 2.0 ** -23))[..., None] + HALF[dtype] * np.abs(want) + (2.0 ** -25 if dtype == "f16" else 1e-37)
    off = (np.abs(got - want) / tol)[inside]
    assert not np.isnan(off).any() and (off <= 1).all(), float(np.nanmax(off))
    return off


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,lens_k,heads,kv", [
    ([1], [1], 1, 1), ([37], [37], 16, 8), ([65, 1, 0, 31, 200], [65, 1, 0, 31, 200], 4, 2), ([3, 40, 0, 5], [70, 33, 9, 0], 7, 1), ([130], [129], 2, 2),
    ([1], [1000], 8, 2), ([17, 1], [700, 300], 4, 1), ([33] * 70, [33] * 70, 2, 1), ([64, 128], [64, 128], 5, 1)])
def test_prompt_attention(qa, dtype, d, causal, lens, lens_k, heads, kv):
    print("attention", dtype, d, causal, lens[:6], lens_k[:6], heads, kv, flush=True)
    rng = np.random.default_rng(d + sum(lens) + heads)
    starts, starts_k = np.cumsum([0] + lens), np.cumsum([0] + lens_k)
    if lens == lens_k:  # parts of one row
        (q, q64), (k, k64), (v, v64) = wide(rng, sum(lens), heads, kv, kv, d=d, dtype=dtype)
    else:
        (q, q64), (k, k64), (v, v64) = (made(rng, n, g, d, dtype=dtype) for n, g in ((sum(lens), heads), (sum(lens_k), kv), (sum(lens_k), kv)))
    scale = 2.0 * d ** -0.5
    got = qa.prompt_attention(q, k, v, ints(starts), ints(starts_k), causal=causal, scale=scale)
    check_attention(got, q64, k64, v64, starts, starts_k, causal, scale, dtype)
    assert torch.equal(got, qa.prompt_attention(q, k, v, ints(starts), ints(starts_k), causal=causal, scale=scale))
    if len(lens) == 1:
        assert torch.equal(got, qa.prompt_attention(q, k, v, causal=causal, scale=scale))


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_attention_leaves_other_rows(qa, dtype):
    """Rows in front of, between and behind the sequences stay as they were, in an out whose rows are part of wider ones."""
    rng = np.random.default_rng(8)
    (q, q64), (k, k64), (v, v64) = (made(rng, 50, g, 64, dtype=dtype) for g in (4, 2, 2))
    starts, starts_k = [5, 20, 20, 41], [0, 15, 16, 37]
    for keys_hint in (None, 0, 1 << 20):
        room = torch.full((50, 6 * 64), 7.0, dtype=DTYPES[dtype], device="cuda")
        out = room[:, 64:5 * 64].unflatten(1, (4, 64))
        assert qa.prompt_attention(q, k, v, ints(starts), ints(starts_k), out=out, max_len_k=keys_hint) is out
        check_attention(out, q64, k64, v64, starts, starts_k, True, 64 ** -0.5, dtype, untouched=7.0)
        assert (room[:, :64] == 7).all() and (room[:, 5 * 64:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, -0.3, 1e-30, 40.0])
def test_prompt_attention_scales(qa, dtype, scale):
    rng = np.random.default_rng(9)
    (q, q64), (k, k64), (v, v64) = (made(rng, 70, g, 64, dtype=dtype) for g in (2, 1, 1))
    got = qa.prompt_attention(q, k, v, scale=scale)
    check_attention(got, q64, k64, v64, [0, 70], [0, 70], True, scale, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,keys", [(100, 100), (3, 900)])
def test_prompt_attention_of_large_and_small_scores(qa, dtype, n, keys):
    """Scores that rise and fall by hundreds along the keys, so that the running reference moves often; values of very different sizes."""
    rng = np.random.default_rng(10)
    q, q64 = made(rng, n, 2, 64, dtype=dtype)
    k64 = rng.normal(size=(keys, 1, 64)) * (1 + 12 * np.abs(np.sin(np.arange(keys) / 9.0)))[:, None, None]
    v64 = rng.normal(size=(keys, 1, 64)) * np.exp(rng.normal(size=(keys, 1, 64)) * 2)
    k, v = (torch.from_numpy(x.astype(np.float32)).to(DTYPES[dtype]) for x in (k64, v64))
    got = qa.prompt_attention(q, k.cuda(), v.cuda(), scale=1.0)
    check_attention(got, q64, k.double().numpy(), v.double().numpy(), [0, n], [0, keys], True, 1.0, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("n,keys", [(100, 100), (5, 800), (64, 64)])
def test_prompt_attention_of_no_numbers(qa, dtype, bad, n, keys):
    """What a row does not see has no influence whatever it holds, in this sequence or the next; what it sees makes the element (a value) or the
    row (a key, a query) no number.  (A key of one infinity gives scores of both infinities: NaN, or a weight of zero.)"""
    rng = np.random.default_rng(11)
    total, heads = n + 40, 2
    (q, q64), (k, k64), (v, v64) = (made(rng, rows, g, 64, dtype=dtype) for rows, g in ((total, heads), (keys + 40, 1), (keys + 40, 1)))
    starts, starts_k = ints([0, n, total]), ints([0, keys, keys + 40])
    clean = qa.prompt_attention(q, k, v, starts, starts_k)
    for at in (0, keys // 2, keys - 2, keys - 1):
        sees = torch.zeros(total, dtype=torch.bool, device="cuda")
        sees[max(0, at - (keys - n)):n] = True
        values = v.clone()
        values[at, 0, 17] = bad
        got = qa.prompt_attention(q, k, values, starts, starts_k)
        assert torch.equal(got[~sees], clean[~sees])
        other = torch.arange(64, device="cuda") != 17
        assert torch.equal(got[..., other], clean[..., other])
        hit = got[sees][..., 17]
        if math.isnan(bad):
            assert torch.isnan(hit).all()
        elif dtype == "f32":
            assert not torch.isfinite(hit).any()
        else:
            assert (hit == bad).all()
        keys_ = k.clone()
        keys_[at, 0, 3] = bad
        got = qa.prompt_attention(q, keys_, v, starts, starts_k)
        assert torch.equal(got[~sees], clean[~sees])
        if math.isnan(bad):
            assert torch.isnan(got[sees]).all()
    queries = q.clone()
    queries[2, 1, 5] = bad
    got = qa.prompt_attention(queries, k, v, starts, starts_k)
    rest = torch.ones(total, heads, dtype=torch.bool, device="cuda")
    rest[2, 1] = False
    assert torch.equal(got[rest], clean[rest]) and not torch.isfinite(got[2, 1]).any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_attention_of_offsets_that_do_not_fit(qa, dtype):
    """Offsets outside the tensors or falling read and write nothing outside; proper sequences among them are right."""
    rng = np.random.default_rng(12)
    (q, q64), (k, k64), (v, v64) = (made(rng, 30, g, 64, dtype=dtype) for g in (2, 1, 1))
    got = qa.prompt_attention(q, k, v, ints([0, 10, 2000000000]), ints([0, 10, 2000000000]))
    check_attention(got, q64, k64, v64, [0, 10, 30], [0, 10, 30], True, 0.125, dtype)
    got = qa.prompt_attention(q, k, v, ints([-5, 12, 30]), ints([-7, 12, 30]))
    check_attention(got, q64, k64, v64, [0, 12, 30], [0, 12, 30], True, 0.125, dtype)
    got = qa.prompt_attention(q, k, v, ints([0, 12, 3, 30]), ints([0, 12, 12, 12]), out=torch.zeros_like(q))
    check_attention(got[:3], q64[:3], k64[:12], v64[:12], [0, 3], [0, 3], True, 0.125, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_attention_of_offsets_that_fall_far(qa, dtype):
    """Sequences that overlap leave their rows in any state, and what is around the tensor as it was."""
    rng = np.random.default_rng(16)
    n = 3000
    (q, _), (k, _), (v, _) = (made(rng, n, g, 64, dtype=dtype) for g in (2, 1, 1))
    for starts in ([0, n, 100, n], [0, 2900, 64, 2800, 10, n], [n, 0, n, 0]):
        room = torch.full((n + 600, 2, 64), 3.0, dtype=DTYPES[dtype], device="cuda")
        qa.prompt_attention(q, k, v, ints(starts), out=room[300:300 + n])
        assert (room[:300] == 3.0).all() and (room[300 + n:] == 3.0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prompts,heads,kv", [(64, 3, 1), (65, 2, 2), (4097, 2, 1), (130, 40, 2)])
def test_prompt_attention_of_many_sequences(qa, dtype, prompts, heads, kv):
    """Short sequences, some empty, as many as need one, two and three looks at the offsets."""
    rng = np.random.default_rng(prompts)
    lens = rng.integers(0, 4, size=prompts)
    lens[prompts // 2] = 150
    lens_k = lens + rng.integers(0, 3, size=prompts) * (rng.random(prompts) < 0.3)
    starts, starts_k = np.cumsum([0, *lens]), np.cumsum([0, *lens_k])
    (q, q64), (k, k64), (v, v64) = (made(rng, n, g, 64, dtype=dtype) for n, g in ((starts[-1], heads), (starts_k[-1], kv), (starts_k[-1], kv)))
    got = qa.prompt_attention(q, k, v, ints(starts), ints(starts_k), max_len_k=int(lens_k.max()))
    check_attention(got, q64, k64, v64, starts, starts_k, True, 0.125, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d,causal", [(64, True), (128, True), (256, True), (64, False), (128, False)])
def test_prompt_attention_of_long_and_short_sequences(qa, dtype, d, causal):
    """Long sequences among short and empty ones, some with more keys than tokens and some with fewer: workgroups begin by length."""
    rng = np.random.default_rng(d)
    lens, lens_k = [0, 700, 1, 5, 900, 0, 330, 64], [3, 700, 250, 2, 1000, 0, 0, 1]
    starts, starts_k = np.cumsum([0, *lens]), np.cumsum([0, *lens_k])
    (q, q64), (k, k64), (v, v64) = (made(rng, n, g, d, dtype=dtype) for n, g in ((starts[-1], 24), (starts_k[-1], 8), (starts_k[-1], 8)))
    got = qa.prompt_attention(q, k, v, ints(starts), ints(starts_k), causal=causal)
    check_attention(got, q64, k64, v64, starts, starts_k, causal, d ** -0.5, dtype)
    room = torch.full((starts[-1] + 600, 24, d), 3.0, dtype=DTYPES[dtype], device="cuda")
    qa.prompt_attention(q, k, v, ints([2000, 0, 1700, 20, 1500, 1, 2000, 0, 1999]), ints(starts_k), causal=causal, out=room[300:300 + starts[-1]])
    assert (room[:300] == 3.0).all() and (room[300 + starts[-1]:] == 3.0).all()


@pytest.mark.parametrize("n,d", [(520, 256), (700, 128)])
def test_prompt_attention_of_one_prompt_in_parts(qa, n, d):
    """A causal f32 prompt whose tiles of rows are nearly as many as the compute units: tiles of unequal length in several parts."""
    rng = np.random.default_rng(n)
    (q, q64), (k, k64), (v, v64) = (made(rng, n, 16, d) for _ in range(3))
    check_attention(qa.prompt_attention(q, k, v), q64, k64, v64, [0, n], [0, n], True, d ** -0.5, "f32")


@pytest.mark.parametrize("d,lens,past,heads,kv", [(256, [28 - b % 9 for b in range(17)], 1000, 16, 4), (128, [128 - 7 * b for b in range(10)], 500, 8, 8)])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_attention_of_chunks_in_parts(qa, d, lens, past, heads, kv, causal):
    """f32 sequences of few rows on many keys each, as many workgroups as would leave a last turn nearly empty: in parts."""
    rng = np.random.default_rng(d)
    starts, starts_k = np.cumsum([0, *lens]), np.cumsum([0, *(n + past - 11 * b for b, n in enumerate(lens))])
    (q, q64), (k, k64), (v, v64) = (made(rng, n, g, d) for n, g in ((starts[-1], heads), (starts_k[-1], kv), (starts_k[-1], kv)))
    got = qa.prompt_attention(q, k, v, ints(starts), ints(starts_k), causal=causal, max_len_k=max(lens) + past)
    check_attention(got, q64, k64, v64, starts, starts_k, causal, d ** -0.5, "f32")


def test_prompt_attention_without_keys(qa):
    for dtype in DTYPES.values():
        q, none = torch.randn(5, 4, 128, device="cuda").to(dtype), torch.empty(0, 2, 128, device="cuda", dtype=dtype)
        assert (qa.prompt_attention(q, none, none) == 0).all()
        assert (qa.prompt_attention(q, none, none, ints([0, 3, 5]), ints([0, 0, 0]), causal=False) == 0).all()
        assert qa.prompt_attention(q[:0], none, none).shape == (0, 4, 128)


def test_prompt_attention_on_another_stream(qa):
    """Calls on two streams at once, split ones among them, each with the scratch of its own stream."""
    rng = np.random.default_rng(14)
    sets = []
    for i in range(2):
        (q, q64), (k, k64), (v, v64) = (made(rng, n, g, 128, dtype="bf16") for n, g in ((9, 8), (2000 + 300 * i, 2), (2000 + 300 * i, 2)))
        sets.append((q, k, v, q64, k64, v64, torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for s, out in zip(sets, outs):
            with torch.cuda.stream(s[6]):
                out.append(qa.prompt_attention(*s[:3]))
    torch.cuda.synchronize()
    for s, out in zip(sets, outs):
        check_attention(out[0], *s[3:6], [0, 9], [0, s[1].shape[0]], True, 128 ** -0.5, "bf16")
        assert all(torch.equal(out[0], o) for o in out)


def test_prompt_attention_of_far_offsets(qa):
    """Rows whose offsets in elements and bytes pass 32 bits: the last rows of keys of a wide stride, the last tokens of q and out."""
    rng = np.random.default_rng(15)
    for dtype in ("bf16", "f32"):
        step = 1 << 20
        tokens, keys = 2100, 2200
        room = torch.empty(keys * step + 4096, dtype=DTYPES[dtype], device="cuda")
        (q, q64), (k, k64), (v, v64) = (made(rng, n, g, 64, dtype=dtype) for n, g in ((tokens, 2), (keys, 1), (keys, 1)))
        views = []
        for i, x in enumerate((q, k, v)):
            view = room[i * 512:].as_strided(x.shape, (step, 64, 1))
            view.copy_(x)
            views.append(view)
        out = room[3 * 512:].as_strided(q.shape, (step, 64, 1))
        qa.prompt_attention(*views, ints([0, tokens - 5, tokens]), ints([0, 100, keys]), out=out)
        at, ak = tokens - 5, 100
        check_attention(out[at:], q64[at:], k64[ak:], v64[ak:], [0, 5], [0, keys - ak], True, 0.125, dtype)
        assert torch.equal(out, qa.prompt_attention(q, k, v, ints([0, tokens - 5, tokens]), ints([0, 100, keys])))
        del room, views, view, out
        torch.cuda.empty_cache()


def test_prompt_attention_in_a_graph(qa):
    """A captured call replayed with other lengths and values, eager work between the replays."""
    rng = np.random.default_rng(13)
    for dtype, shapes in (("f32", [([0, 20, 50], [0, 20, 50]), ([0, 1, 2], [0, 1, 2])]), ("bf16", [([0, 3, 4], [0, 600, 900]), ([0, 1, 3], [0, 800, 801]), ([0, 0, 4], [0, 0, 900])])):
        keys = 50 if dtype == "f32" else 900
        (q, _), (k, _), (v, _) = (made(rng, n, g, 128, dtype=dtype) for n, g in ((50 if dtype == "f32" else 4, 4), (keys, 2), (keys, 2)))
        starts, starts_k = ints(shapes[0][0]), ints(shapes[0][1])
        out = torch.zeros_like(q)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            qa.prompt_attention(q, k, v, starts, starts_k, out=out)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                qa.prompt_attention(q, k, v, starts, starts_k, out=out)
        torch.cuda.current_stream().wait_stream(stream)
        for a, b in shapes + shapes:
            (x, x64), (y, y64), (z, z64) = (made(rng, *t.shape, dtype=dtype) for t in (q, k, v))
            q.copy_(x), k.copy_(y), v.copy_(z), starts.copy_(ints(a)), starts_k.copy_(ints(b)), out.fill_(3)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            check_attention(out, x64, y64, z64, a, b, True, 128 ** -0.5, dtype, untouched=3.0)


def test_prompt_operators_in_one_graph(qa):
    """Rotation, attention of few rows on many keys and routing as one captured sequence, on new values, positions and lengths at every replay, with
    eager calls of other sizes on the same stream's scratch in between."""
    rng = np.random.default_rng(17)
    rotary = qa.RotaryEmbedding(128, base=1e6)
    for dtype in DTYPES:
        (q, k), (keys, values) = (torch.zeros(6, g, 128, dtype=DTYPES[dtype], device="cuda") for g in (4, 2)), (torch.zeros(1500, 2, 128, dtype=DTYPES[dtype], device="cuda") for _ in range(2))
        positions, starts, starts_k = ints([0] * 6), ints([0, 6, 6]), ints([0, 1500, 1500])
        mix = torch.from_numpy(rng.normal(size=(512, 32)).astype(np.float32)).cuda()
        logits = torch.zeros(6, 32, dtype=DTYPES[dtype], device="cuda")

        def run():
            a, _ = qa.rope_positions(q, k, positions, rotary)
            o = qa.prompt_attention(a, keys, values, starts, starts_k)
            return o, *qa.moe_route_scored(logits, 4, "sigmoid", groups=4, top_groups=2)

        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            run()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                kept = run()
            for step in range(4):
                for t in (q, k, keys, values, logits):
                    t.copy_(made(rng, *t.shape, dtype=dtype)[0])
                positions.copy_(ints(rng.integers(0, 100000, size=6)))
                cut, cut_k = int(rng.integers(0, 7)), int(rng.integers(0, 1501))
                starts.copy_(ints([0, cut, 6])), starts_k.copy_(ints([0, cut_k, 1500]))
                graph.replay()
                got = [t.clone() for t in kept]
                qa.prompt_attention(values[:9], values, keys)  # (split, too)
                want = run()
                stream.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(got, want)), step


def test_prompt_attention_by_two_threads(qa):
    """Calls of two host threads on one stream and on two, split ones, each as alone."""
    import threading
    rng = np.random.default_rng(18)
    sets = [[made(rng, n, g, 64, dtype="f16")[0] for n, g in ((5 + i, 4), (900 + 200 * i, 2), (900 + 200 * i, 2))] for i in range(2)]
    alone = [qa.prompt_attention(*s) for s in sets]
    torch.cuda.synchronize()
    for streams in ([torch.cuda.Stream()] * 2, [torch.cuda.Stream(), torch.cuda.Stream()]):
        outs = [[], []]

        def work(i):
            with torch.cuda.stream(streams[i]):
                for _ in range(50):
                    outs[i].append(qa.prompt_attention(*sets[i]))

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        [t.start() for t in threads], [t.join() for t in threads]
        torch.cuda.synchronize()
        for i in range(2):
            assert len(outs[i]) == 50 and all(torch.equal(o, alone[i]) for o in outs[i])


def test_prompt_attention_python_refusals(qa):
    x = torch.zeros(4, 8, 64, device="cuda")
    kv = torch.zeros(4, 2, 64, device="cuda")
    bad = [dict(q=x.double()), dict(q=x[0]), dict(k=kv.half()), dict(v=kv[:3]), dict(k=kv.cpu()), dict(k=torch.zeros(4, 3, 64, device="cuda"), v=torch.zeros(4, 3, 64, device="cuda")),
           dict(starts=ints([0, 4]).long()), dict(starts=ints([0, 4]).cpu()), dict(starts_k=ints([0, 4])), dict(starts=ints([0, 4]), starts_k=ints([0, 2, 4])),
           dict(starts=ints([0, 4]), k=kv[:2], v=kv[:2]), dict(out=torch.zeros(4, 8, 64)), dict(out=x), dict(q=x.transpose(0, 1)), dict(max_len_k=-1), dict(scale=math.nan),
           dict(q=torch.zeros(4 * 512 + 1, device="cuda")[1:].view(4, 8, 64)), dict(starts=ints([]))]
    good = dict(q=x, k=kv, v=kv)
    qa.prompt_attention(**good)
    for over in bad:
        with pytest.raises(qa.QmmError):
            qa.prompt_attention(**{**good, **over})
    rotary = qa.RotaryEmbedding(64)
    good = dict(q=x, k=kv, positions=ints(range(4)), rotary=rotary)
    qa.rope_positions(**good)
    for over in (dict(q=x.double()), dict(k=kv.half()), dict(k=kv[:3]), dict(positions=ints(range(3))), dict(positions=ints(range(4)).long()), dict(qk_weight=x.new_zeros(64)),
                 dict(qk_weight=x.new_zeros(128).half()), dict(out=(x, None)), dict(out=(x, kv.half())), dict(rotary=qa.RotaryEmbedding(128)), dict(eps=-1.0), dict(q=x.cpu()), dict(out=(x, x[:, :2]))):
        with pytest.raises(qa.QmmError):
            qa.rope_positions(**{**good, **over})


# ---- routing ------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,n,top_k,groups,top_groups,group_best", [
    (1, 128, 8, 1, 1, 1), (1, 1, 1, 1, 1, 1), (70, 256, 8, 8, 4, 2), (33, 64, 6, 1, 1, 1), (17, 40, 40, 4, 4, 1), (9, 1024, 64, 64, 5, 2), (21, 160, 6, 8, 3, 1), (300, 65, 1, 5, 1, 2),
    (50, 512, 10, 16, 16, 2), (13, 7, 3, 7, 3, 2), (5, 1000, 5, 1, 1, 2)])
def test_route_scored(qa, dtype, scoring, t, n, top_k, groups, top_groups, group_best):
    print("route", dtype, scoring, t, n, top_k, groups, top_groups, group_best, flush=True)
    rng = np.random.default_rng(t * 7 + n)
    logits, l64 = made(rng, t, n + 3, dtype=dtype, std=3.0)
    logits, l64 = logits[:, 1:n + 1], l64[:, 1:n + 1]  # parts of wider rows
    b = (rng.normal(size=n) * 0.1).astype(np.float32)
    for bias in (None, b):
        for renormalize, scale in ((True, 2.5), (False, 1.0)):
            ids, w = qa.moe_route_scored(logits, top_k, scoring, None if bias is None else torch.from_numpy(bias).cuda(), groups, top_groups, group_best, renormalize, scale)
            want_ids, want_w = prompt_ref.route(l64, top_k, scoring, bias, groups, top_groups, group_best, renormalize, scale)
            assert np.array_equal(ids.cpu().numpy(), want_ids)
            assert (np.abs(w.cpu().double().numpy() - want_w) <= 2.0 ** -24 * np.abs(want_w) + 2.0 ** -50).all()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups,group_best", [(1, 1, 1), (4, 2, 1), (4, 3, 2)])
def test_route_scored_of_ties_and_no_numbers(qa, scoring, groups, top_groups, group_best):
    """Equal logits and biases, rows of NaN, infinities of both signs, logits far below the others."""
    rng = np.random.default_rng(3)
    l = rng.integers(-2, 3, size=(40, 24)).astype(np.float32)
    l[0], l[1], l[2] = 0.0, -np.inf, np.nan
    l[3, ::2], l[4, 3], l[5, :20], l[6, 5], l[7, 1:3] = np.nan, np.inf, -np.inf, -np.inf, np.inf
    l[8] = -0.0
    l[9], l[10], l[11, 4:] = -2000.0 - np.arange(24), -1e30 * (1 + np.arange(24) % 5), -1e38
    l[12] = 3e38 * np.where(np.arange(24) % 3, 1, -1)
    l[13] = 800.0 + np.arange(24)[::-1]
    biases = [None, np.zeros(24, np.float32), (rng.integers(-1, 2, size=24) * 0.25).astype(np.float32)]
    odd = biases[2].copy()
    odd[[3, 9, 14]] = np.nan, np.inf, -np.inf
    for bias in biases + [odd]:
        for renormalize in (True, False):
            ids, w = qa.moe_route_scored(torch.from_numpy(l).cuda(), 5, scoring, None if bias is None else torch.from_numpy(bias).cuda(), groups, top_groups, group_best, renormalize)
            want_ids, want_w = prompt_ref.route(l, 5, scoring, bias, groups, top_groups, group_best, renormalize)
            assert np.array_equal(ids.cpu().numpy(), want_ids), np.flatnonzero((ids.cpu().numpy() != want_ids).any(1))
            assert (np.abs(w.cpu().double().numpy() - want_w) <= 2.0 ** -24 * np.abs(want_w) + 2.0 ** -50).all()


def test_route_scored_with_the_plain_settings_is_the_plain_router(qa):
    rng = np.random.default_rng(4)
    logits, _ = made(rng, 200, 128)
    ids, w = qa.moe_route(logits, 8)
    got, v = qa.moe_route_scored(logits, 8)
    assert torch.equal(ids, got) and (w - v).abs().max() <= 1e-6


def test_route_scored_python_refusals(qa):
    x = torch.zeros(4, 16, device="cuda")
    good = dict(logits=x, top_k=2)
    qa.moe_route_scored(**good)
    for over in (dict(logits=x.double()), dict(logits=x[0]), dict(logits=x.T), dict(top_k=0), dict(top_k=17), dict(top_k=65), dict(scoring="tanh"), dict(bias=x[0].half()), dict(bias=x[0, :8]),
                 dict(groups=3), dict(groups=4, top_groups=5), dict(groups=4, top_groups=0), dict(group_best=3), dict(scale=math.inf), dict(bias=x[0].cpu())):
        with pytest.raises(qa.QmmError):
            qa.moe_route_scored(**{**good, **over})
