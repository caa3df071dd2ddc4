"""GPU tests (pytest -m gpu) of the quantized cache, shared-prefix attention and beam selection against the plain 64-bit
restatements of kv_ref.py, through the Python entry points.

Tolerances.  The cache's values are the format's, exactly (f16 outputs: half a step, 2^-11).  Attention: with A the largest sum of |q_i k_i| scale
of a row, V the largest |v|, n its positions, u = 2^-24:
  a score is off by at most A (2^-22 for the two-part f16 split of an f32 query + d u for sums of d terms) + A 2u (scale, log2 e),
  a weight relatively by that + 2^-22 (exponential) and, split into two f16 parts, 2^-22 more,
  a weighted mean by twice its weights' relative error times V, its two sums by (n / 16 + 64) u V each, the quotient by 2u V,
f16 outputs by 2^-11 |out| more, and where f16 inputs let weights be single f16 numbers by 2^-11 V (they are rounded twice, to f16 and under the
value's scale, each by at most that relatively; both at their worst with one sign would be twice this: what is asked is the half)."""
import numpy as np
import pytest
import torch

import kv_ref

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "f16": torch.float16}
BITS = {"Q8_0": 8, "Q4_0": 4}


@pytest.fixture(scope="module")
def qa():
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the HIP path cannot run (there is no fallback)")
    import izwi_amd
    izwi_amd.lib()
    torch.cuda.set_device(0)
    return izwi_amd


def ints(values):
    return torch.tensor(list(values), dtype=torch.int32, device="cuda")


def draw(rng, *shape, dtype="f32", outliers=True):
    x = rng.normal(size=shape).astype(np.float32)
    if outliers:
        x *= np.exp(rng.normal(size=shape[-1]) * 0.7).astype(np.float32)
    return x.astype(np.float16).astype(np.float32) if dtype == "f16" else x


def dev(x, dtype="f32"):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda().to(DTYPES[dtype])


def same_values(got, want, dtype):
    got, want = got.cpu().double().numpy(), np.asarray(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    ok = ~np.isnan(want)
    if dtype == "f32":
        assert np.array_equal(got[ok], want[ok])  # scale times quant has 19 bits
    else:
        assert (np.abs(got[ok] - want[ok]) <= 2.0 ** -11 * np.abs(want[ok]) + 2.0 ** -25).all()


# ---- the cache -----------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quant", BITS)
@pytest.mark.parametrize("batch,tokens,kv_heads,d,capacity,first", [
    (1, 1, 8, 128, 33, 0), (3, 5, 1, 64, 32, 1), (2, 37, 3, 256, 50, 2), (5, 1, 7, 128, 1, 0), (1, 300, 2, 64, 257, 0), (4, 9, 5, 128, 20, 3)])
def test_cache_round_trip(qa, quant, dtype, batch, tokens, kv_heads, d, capacity, first):
    """Ragged rows go to their places bit for bit, what lies outside is left out, the rest stays as it was."""
    print("round trip", quant, dtype, batch, tokens, kv_heads, d, capacity, flush=True)
    rng = np.random.default_rng(batch * 1000 + tokens)
    slots = first + batch + 1
    cache, want = qa.QuantizedKvCache(qa.KvCacheType[quant], slots, kv_heads, capacity, d), kv_ref.Cache(BITS[quant], slots, kv_heads, capacity, d)
    every = [draw(rng, slots, capacity, kv_heads, d, dtype=dtype) for _ in range(2)]
    cache.append(dev(every[0], dtype), dev(every[1], dtype), ints([0] * slots))
    want.append(*every, [0] * slots)
    starts = [int(rng.integers(-2, capacity)) for _ in range(batch)]
    counts = [tokens - (b * 3) % (tokens + 1) for b in range(batch)]
    counts[-1] = tokens + 5  # more than there are
    for c in (counts, None):
        k, v = (draw(rng, batch, tokens, kv_heads, d, dtype=dtype) for _ in range(2))
        cache.append(dev(k, dtype), dev(v, dtype), ints(starts), None if c is None else ints(c), first_slot=first)
        want.append(k, v, starts, c, first)
        got = cache.read(ints([0] * slots), capacity, dtype=DTYPES[dtype])
        for g, w in zip(got, want.v):
            same_values(g, w, dtype)
        got = cache.read(ints(starts), tokens + 2, None if c is None else ints(c), first_slot=first, dtype=DTYPES[dtype])
        for g, w in zip(got, want.read(starts, tokens + 2, c, first)):
            same_values(g, w, dtype)


@pytest.mark.parametrize("quant", BITS)
def test_cache_of_odd_values(qa, quant):
    """Zeros, ties of both signs, exact halves, tiny and huge blocks, infinities and NaN, per block of 32."""
    rng = np.random.default_rng(9)
    x = draw(rng, 1, 24, 2, 64)
    x[0, 0] = 0.0
    x[0, 1, 0] = np.where(np.arange(64) % 2, 2.0, -2.0)
    x[0, 2, 0] = np.where(np.arange(64) % 2, -2.0, 2.0)
    x[0, 3, 0, :32] = (np.arange(32) - 16) * 0.5 + 0.5
    x[0, 3, 0, 31] = 127.0 / 2
    x[0, 4] *= 1e-5
    x[0, 5] *= 1e-7
    x[0, 6] *= 1e-30
    x[0, 7, 0, 3] = 1e-42
    x[0, 8, 1, 40] = np.inf
    x[0, 9, 0, 7] = -np.inf
    x[0, 10, 1, 0] = np.nan
    x[0, 11, 0, 33] = np.nan
    x[0, 11, 0, 35] = np.inf
    x[0, 12] *= 1e7
    x[0, 13, 0, 5] = 3e38
    x[0, 14, 0, :32] = np.arange(32) - 15.5
    x[0, 15, 0, :32] = -(np.arange(32) - 15.5)
    x[0, 16] = np.float32(1e-40)
    x[0, 17, 1, 31] = -0.0
    cache = qa.QuantizedKvCache(qa.KvCacheType[quant], 1, 2, 24, 64)
    cache.append(dev(x), dev(x[:, ::-1]), ints([0]))
    k, v = cache.read(ints([0]), 24)
    same_values(k, kv_ref.values(*kv_ref.quantize(x, BITS[quant])), "f32")
    same_values(v, kv_ref.values(*kv_ref.quantize(x[:, ::-1], BITS[quant])), "f32")


def test_cache_equals_gguf_blocks(qa, oracle):
    """Q8_0 rows read back as the GGUF quantizer's blocks dequantize."""
    x = oracle.randn(11, (40, 1024), std=0.7)
    want = oracle.dequantize(8, oracle.quantize(8, x), 40, 1024)
    cache = qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 1, 8, 40, 128)
    t = dev(x).view(1, 40, 8, 128)
    cache.append(t, t, ints([0]))
    for got in cache.read(ints([0]), 40):
        assert np.array_equal(got.cpu().numpy().reshape(40, 1024), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cache_rows_inside_wider_ones(qa, dtype):
    """k and v as parts of a packed q|k|v result, and rows at odd addresses."""
    rng = np.random.default_rng(2)
    for d, kv in ((128, 2), (64, 3)):
        wide = dev(draw(rng, 3, 5, 4 * kv * d + 6, dtype=dtype), dtype)
        for at in (0, kv * d, 2 * kv * d + 1, 2 * kv * d + 6):
            k, v = (wide[:, :, a:a + kv * d].unflatten(-1, (kv, d)) for a in (at, kv * d + 3))
            a, b = (qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 3, kv, 8, d) for _ in range(2))
            a.append(k, v, ints([0, 1, 2]))
            b.append(k.contiguous(), v.contiguous(), ints([0, 1, 2]))
            for x, y in zip(a.read(ints([0, 1, 2]), 5), b.read(ints([0, 1, 2]), 5)):
                assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quant", BITS)
@pytest.mark.parametrize("batch,tokens,kv_heads,d,capacity,first", [
    (3, 500, 3, 256, 510, 1), (70, 50, 5, 64, 57, 0), (9, 40, 24, 128, 33, 2), (700, 9, 2, 128, 12, 0), (1, 2200, 4, 128, 2201, 0), (300, 8, 8, 64, 9, 0)])
def test_cache_round_trip_of_many_rows(qa, quant, dtype, batch, tokens, kv_heads, d, capacity, first):
    """Calls of more than 2^20 values, of which more than 8 tokens of a sequence go sixteen positions to a wave (8: one by one)."""
    test_cache_round_trip(qa, quant, dtype, batch, tokens, kv_heads, d, capacity, first)


@pytest.mark.parametrize("dtype", DTYPES)
def test_cache_of_many_rows_inside_wider_ones_and_by_lineage(qa, dtype):
    """Sixteen positions to a wave from rows at odd addresses, and read through a lineage."""
    rng = np.random.default_rng(21)
    kv, d, prompts, beams, capacity = 6, 64, 4, 8, 110
    n = prompts * beams
    wide = dev(draw(rng, n, capacity, 2 * kv * d + 3, dtype=dtype), dtype)
    a, b = (qa.QuantizedKvCache(qa.KvCacheType.Q4_0, n, kv, capacity, d) for _ in range(2))
    k, v = (wide[:, :, at:at + kv * d].unflatten(-1, (kv, d)) for at in (1, kv * d + 3))
    a.append(k, v, ints([0] * n))
    b.append(k.contiguous(), v.contiguous(), ints([0] * n))
    every = a.read(ints([0] * n), capacity, dtype=DTYPES[dtype])
    for x, y in zip(every, b.read(ints([0] * n), capacity, dtype=DTYPES[dtype])):
        assert torch.equal(x, y)
    rows = torch.from_numpy(rng.integers(0, beams + 1, size=tuple(a.new_lineage().shape)).astype(np.uint8)).cuda()
    at = torch.arange(n, device="cuda").view(n, 1) // beams * beams + rows[:, :capacity].long()
    there = rows[:, :capacity] < beams
    for got, x in zip(a.read(ints([0] * n), capacity, lineage=rows, beams=beams, dtype=DTYPES[dtype]), every):
        want = x[at.clamp(max=n - 1), torch.arange(capacity, device="cuda").view(1, -1)] * there[..., None, None].to(x.dtype)
        assert torch.equal(got, want)


@pytest.mark.parametrize("quant", BITS)
def test_cache_and_attention_past_32_bits(qa, quant):
    """A slot that begins, and a position that stands, more than 2^32 bytes into its plane (2^33 values of keys)."""
    rng = np.random.default_rng(13)
    d, far = 256, 1 << 25
    for slots, capacity, slot, start in ((40, far // 32, 39, 5), (1, far, 0, far - 37)):
        cache = qa.QuantizedKvCache(qa.KvCacheType[quant], slots, 1, capacity, d)
        cache.buffer.zero_()  # scales of zero: keys and values of zero
        x = draw(rng, 2, 1, 30, 1, d)
        cache.append(dev(x[0]), dev(x[1]), ints([start]), first_slot=slot)
        ref = [kv_ref.values(*kv_ref.quantize(x[i], BITS[quant])) for i in range(2)]
        got = cache.read(ints([start - 2]), 35, first_slot=slot)
        for g, w in zip(got, ref):
            same_values(g, np.pad(w, ((0, 0), (2, 3), (0, 0), (0, 0))), "f32")
        # zeros, then scores of about 20 among them: the softmax by hand
        k, v = (r[0, :, 0] for r in ref)
        q, lens = draw(rng, slots, 2, d), [0] * slots
        lens[slot] = n = start + 30
        q *= np.float32(20) / np.abs(q[slot] @ k.T).max()
        got = qa.shared_prefix_attention(dev(q), cache, ints(lens), beams=1, scale=1.0).cpu().double().numpy()
        assert (got[:slot] == 0).all()
        s = q[slot].astype(np.float64) @ k.T
        want = (np.exp(s) @ v) / (np.exp(s).sum(1) + start)[:, None]
        size, top = (np.abs(q[slot].astype(np.float64)) @ np.abs(k).T).max(1), np.abs(v).max()
        tol = (2 * (size * (2.0 ** -22 + (d + 2) * U) + 2.0 ** -21) + 2 * (n / 16 / 256 + 64 + 30) * U + 2 * U) * top  # (a split of 256, a wave of four, a lane of four sums its share)
        assert (np.abs(got[slot] - want) <= tol[:, None]).all()
        del cache


def test_cache_read_by_lineage(qa):
    rng = np.random.default_rng(4)
    prompts, beams, capacity = 2, 3, 45
    cache, want = qa.QuantizedKvCache(qa.KvCacheType.Q4_0, 6, 2, capacity, 128), kv_ref.Cache(4, 6, 2, capacity, 128)
    k, v = draw(rng, 6, capacity, 2, 128), draw(rng, 6, capacity, 2, 128)
    cache.append(dev(k), dev(v), ints([0] * 6))
    want.append(k, v, [0] * 6)
    lineage = cache.new_lineage()
    assert lineage.shape == (6, 64)
    rows = rng.integers(0, beams + 1, size=(6, 64)).astype(np.uint8)  # (3 and 255 are no beams)
    rows[0, 3] = 255
    lineage.copy_(torch.from_numpy(rows))
    starts, counts = [0, 3, 44, -1, 0, 10], [45, 45, 45, 9, 0, 1]
    got = cache.read(ints(starts), 45, ints(counts), lineage=lineage, beams=beams)
    for g, w in zip(got, want.read(starts, 45, counts, lineage=rows, beams=beams)):
        same_values(g, w, "f32")
    got = cache.read(ints([2]), 8, first_slot=4, lineage=lineage, beams=beams, dtype=torch.float16)
    for g, w in zip(got, want.read([2], 8, first_slot=4, lineage=rows, beams=beams)):
        same_values(g, w, "f16")


# ---- attention ---------------------------------------------------------------------------------------------------


def make(qa, rng, quant, dtype, slots, kv_heads, capacity, d, gain=1.0):
    cache, want = qa.QuantizedKvCache(qa.KvCacheType[quant], slots, kv_heads, capacity, d), kv_ref.Cache(BITS[quant], slots, kv_heads, capacity, d)
    cache.buffer.fill_(0xff)  # NaN scales wherever nothing is written
    k, v = draw(rng, slots, capacity, kv_heads, d, dtype=dtype), draw(rng, slots, capacity, kv_heads, d, dtype=dtype) * np.float32(gain)
    cache.append(dev(k, dtype), dev(v, dtype), ints([0] * slots))
    want.append(k, v if dtype == "f32" else v.astype(np.float16).astype(np.float32), [0] * slots)
    return cache, want


def check_attention(got, ref, dtype, d):
    out, size, top, n = (np.asarray(x) for x in ref)
    got = got.cpu().double().numpy()
    score = size * (2.0 ** -22 + (d + 2) * U)
    weight = 2 * (score + 2.0 ** -22 + 2.0 ** -22) + 2 * (n / 16 + 64) * U + 2 * U
    tol = (weight * top)[..., None] * np.ones(d)
    if dtype == "f16":
        tol = tol + 2.0 ** -11 * (top[..., None] + np.abs(out)) + 2.0 ** -25
    worst = np.max(np.abs(got - out) / np.maximum(tol, 1e-300), initial=0)
    print(f"worst error / tolerance {worst:.3f}", flush=True)
    assert (np.abs(got - out) <= tol).all()
    assert (got[n == 0] == 0).all()


SHAPES = [  # heads, kv heads, d, prompts, beams, prefix, suffix
    (16, 8, 128, 1, 1, 0, 1), (16, 8, 128, 1, 1, 0, 300), (32, 8, 128, 1, 4, 70, 9), (4, 4, 64, 2, 3, 33, 40), (6, 2, 256, 3, 1, 129, 0), (8, 1, 64, 1, 5, 31, 32),
    (10, 2, 128, 1, 17, 64, 1), (40, 1, 128, 2, 2, 200, 35), (7, 7, 256, 1, 2, 16, 95), (32, 8, 128, 2, 32, 100, 3), (3, 1, 64, 1, 70, 257, 11), (5, 5, 128, 1, 1, 1000, 0),
    (8, 2, 128, 1, 1, 0, 4100), (16, 8, 64, 1, 16, 2100, 20)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("quant", BITS)
@pytest.mark.parametrize("heads,kv_heads,d,prompts,beams,prefix,suffix", SHAPES)
def test_attention(qa, quant, dtype, heads, kv_heads, d, prompts, beams, prefix, suffix):
    print("attention", quant, dtype, heads, kv_heads, d, prompts, beams, prefix, suffix, flush=True)
    rng = np.random.default_rng(heads * 7919 + prefix + suffix)
    batch = prompts * beams
    q = draw(rng, batch, heads, d, dtype=dtype)
    pre = own = pre_ref = own_ref = plens = lens = None
    if prefix:
        pre, pre_ref = make(qa, rng, quant, dtype, prompts, kv_heads, prefix, d)
        plens = [prefix - (g * 29) % (prefix + 1) for g in range(prompts)]
    if suffix:
        own, own_ref = make(qa, rng, quant, dtype, batch, kv_heads, suffix, d)
        lens = [suffix - (b * 13) % (suffix + 1) for b in range(batch)]
    got = qa.shared_prefix_attention(dev(q, dtype), own, None if lens is None else ints(lens), prefix=pre, prefix_lens=None if plens is None else ints(plens),
                                     beams=beams, scale=d ** -0.5)
    check_attention(got, kv_ref.attention(q, own_ref, lens, pre_ref, plens, None, beams, d ** -0.5), dtype, d)


@pytest.mark.parametrize("quant,dtype", [("Q8_0", "f32"), ("Q4_0", "f16")])
@pytest.mark.parametrize("heads,kv_heads,d,prompts,beams,prefix,suffix", [(32, 8, 128, 2, 4, 90, 65), (4, 2, 64, 1, 3, 0, 130), (2, 1, 256, 3, 2, 40, 33), (8, 8, 128, 1, 32, 7, 70)])
def test_attention_by_lineage(qa, quant, dtype, heads, kv_heads, d, prompts, beams, prefix, suffix):
    """Positions of a beam stand in the slots of the beams that wrote them; an entry that is no beam is no position."""
    rng = np.random.default_rng(suffix)
    batch = prompts * beams
    q = draw(rng, batch, heads, d, dtype=dtype)
    own, own_ref = make(qa, rng, quant, dtype, batch, kv_heads, suffix, d)
    pre = pre_ref = plens = None
    if prefix:
        pre, pre_ref = make(qa, rng, quant, dtype, prompts, kv_heads, prefix, d)
        plens = [prefix - g for g in range(prompts)]
    rows = rng.integers(0, beams, size=tuple(own.new_lineage().shape)).astype(np.uint8)
    rows[1, ::5] = 255
    rows[0, 2] = beams
    if not prefix:
        rows[2, :] = 200  # no position at all
    lens = [suffix - b % 7 for b in range(batch)]
    got = qa.shared_prefix_attention(dev(q, dtype), own, ints(lens), prefix=pre, prefix_lens=None if plens is None else ints(plens), beams=beams,
                                     lineage=torch.from_numpy(rows).cuda())
    check_attention(got, kv_ref.attention(q, own_ref, lens, pre_ref, plens, rows, beams, d ** -0.5), dtype, d)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_scales_and_lengths(qa, dtype):
    """Large and tiny values and queries, scores far apart, lengths that are zero, negative or above the bound."""
    rng = np.random.default_rng(31)
    big, small = (3e4, 1e-3) if dtype == "f16" else (1e6, 1e-6)
    for gain, reach, scale in ((big / 8, 1.0, 0.1), (small, 1.0, 0.1), (1.0, 30.0, 1.0), (1.0, small, 1 / small), (2.0, 0.0, 1.0), (1.0, 1.0, -0.3)):
        pre, pre_ref = make(qa, rng, "Q8_0", dtype, 2, 2, 100, 128, gain if dtype == "f32" else min(gain, 1000.0))
        own, own_ref = make(qa, rng, "Q8_0", dtype, 6, 2, 40, 128, 1.0)
        q = draw(rng, 6, 4, 128, dtype=dtype) * np.float32(reach)
        q = q.astype(np.float16).astype(np.float32) if dtype == "f16" else q
        plens, lens = [100, -3], [0, 40, 45, -1, 0, 17]
        got = qa.shared_prefix_attention(dev(q, dtype), own, ints(lens), prefix=pre, prefix_lens=ints(plens), scale=scale)
        ref = kv_ref.attention(q, own_ref, [min(x, 40) for x in lens], pre_ref, plens, None, 3, scale)
        check_attention(got, ref, dtype, 128)
        got = qa.shared_prefix_attention(dev(q, dtype), own, ints(lens), prefix=pre, prefix_lens=ints(plens), scale=scale, max_len=16, max_prefix_len=70)
        ref = kv_ref.attention(q, own_ref, [min(x, 16) for x in lens], pre_ref, [70, 0], None, 3, scale)
        check_attention(got, ref, dtype, 128)


def test_attention_of_nan_positions(qa):
    """A NaN block inside a sequence makes the heads that read it NaN, and no others; behind the sequence it is never seen."""
    rng = np.random.default_rng(8)
    k, v = draw(rng, 2, 70, 2, 128), draw(rng, 2, 70, 2, 128)
    k[0, 20, 0, 5] = np.nan
    v[1, 60, 1, 100] = np.inf
    cache = qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 2, 2, 70, 128)
    cache.append(dev(k), dev(v), ints([0, 0]))
    q = dev(draw(rng, 2, 4, 128))
    out = qa.shared_prefix_attention(q, cache, ints([70, 70]), beams=1)
    bad = torch.isnan(out)
    assert bad[0, :2].all() and not bad[0, 2:].any() and not bad[1, :2].any()
    assert bad[1, 2:, 96:128].all() and not bad[1, 2:, :96].any()
    assert not torch.isnan(qa.shared_prefix_attention(q, cache, ints([20, 60]), beams=1)).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads,kv_heads,d,prompts,beams,prefix,suffix", [
    (8, 2, 64, 130, 4, 0, 20), (8, 2, 64, 130, 4, 40, 9), (4, 4, 128, 70, 4, 33, 5), (24, 1, 64, 128, 5, 20, 33), (32, 1, 64, 2, 9, 2200, 40),
    (32, 1, 64, 1, 33, 9000, 1), (16, 4, 256, 40, 7, 30, 8)])
def test_attention_of_many_sequences(qa, dtype, heads, kv_heads, d, prompts, beams, prefix, suffix):
    """So many short sequences that a wave has one, alone or behind a prefix, by lineage too; many rows on one long prefix."""
    rng = np.random.default_rng(heads * suffix)
    batch = prompts * beams
    print("many", dtype, heads, kv_heads, d, prompts, beams, prefix, suffix, flush=True)
    q = draw(rng, batch, heads, d, dtype=dtype)
    own, own_ref = make(qa, rng, "Q4_0", dtype, batch, kv_heads, suffix, d)
    lens = [suffix - b % (suffix + 1) for b in range(batch)]
    pre = pre_ref = plens = None
    if prefix:
        pre, pre_ref = make(qa, rng, "Q4_0", dtype, prompts, kv_heads, prefix, d)
        plens = [prefix - g % (prefix + 1) if prefix < 100 else prefix - 31 * g for g in range(prompts)]
    rows = rng.integers(0, beams + 1, size=tuple(own.new_lineage().shape)).astype(np.uint8)
    for lineage in (None, rows):
        got = qa.shared_prefix_attention(dev(q, dtype), own, ints(lens), prefix=pre, prefix_lens=None if plens is None else ints(plens), beams=beams,
                                         lineage=None if lineage is None else torch.from_numpy(lineage).cuda())
        check_attention(got, kv_ref.attention(q, own_ref, lens, pre_ref, plens, lineage, beams, d ** -0.5), dtype, d)


@pytest.mark.parametrize("quant", BITS)
@pytest.mark.parametrize("d", (64, 128, 256))
def test_attention_of_blocks_of_every_size(qa, quant, d):
    """Blocks of the head that are 2^24 smaller than their neighbours are no less exact: the bound by the largest value holds with each
    block's own."""
    rng = np.random.default_rng(d)
    gain = np.repeat(2.0 ** rng.permutation(np.linspace(-14, 10, d // 32).astype(int)), 32).astype(np.float32)
    k, v = draw(rng, 3, 90, 2, d), rng.normal(size=(3, 90, 2, d)).astype(np.float32) * gain
    v[:, 50:] *= 4  # so that the largest rises late
    cache, ref = qa.QuantizedKvCache(qa.KvCacheType[quant], 3, 2, 90, d), kv_ref.Cache(BITS[quant], 3, 2, 90, d)
    cache.append(dev(k), dev(v), ints([0] * 3))
    ref.append(k, v, [0] * 3)
    q, lens = draw(rng, 3, 4, d), [90, 51, 1]
    got = qa.shared_prefix_attention(dev(q), cache, ints(lens), beams=1).cpu().double().numpy()
    want, size, _, count = kv_ref.attention(q, ref, lens, beams=1, scale=d ** -0.5)
    for b in range(3):
        for h in range(4):
            top = np.abs(ref.v[1, b, :lens[b], h // 2]).max(0).reshape(-1, 32).max(1).repeat(32)
            tol = (2 * (size[b, h] * (2.0 ** -22 + (d + 2) * U) + 2.0 ** -21) + 2 * (count[b, h] / 16 + 64) * U + 2 * U) * top
            assert (np.abs(got[b, h] - want[b, h]) <= tol).all()


@pytest.mark.parametrize("reach", (1e5, 1e7, 1e9, 1e12, 1e20))
def test_attention_of_huge_scores(qa, reach):
    """Scores whose spacing in f32 is far above 1: one position, or equal ones, take all the weight, and nothing overflows."""
    rng = np.random.default_rng(4)
    k, v = rng.integers(-127, 128, size=(2, 300, 2, 64)).astype(np.float32), draw(rng, 2, 300, 2, 64)
    k[..., ::32] = 127  # scale 1: quants as they are
    best = rng.integers(0, 300, size=(2, 2))
    for b in range(2):
        for h in range(2):
            k[b, best[b, h], h, 1:32] = 127  # the largest product of all with queries that see the first block only
    k[0, 299, 0] = k[0, best[0, 0], 0]  # (and once more at the end)
    cache, ref = qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 2, 2, 300, 64), kv_ref.Cache(8, 2, 2, 300, 64)
    cache.append(dev(k), dev(v), ints([0, 0]))
    ref.append(k, v, [0, 0])
    q = np.zeros((2, 2, 64), np.float32)
    q[..., :32] = reach
    got = qa.shared_prefix_attention(dev(q), cache, ints([300, 300]), beams=1, scale=1.0).cpu().double().numpy()
    want, _, top, _ = kv_ref.attention(q, ref, [300, 300], beams=1, scale=1.0)
    # (a product with quants is a whole number times the query: next to the best the others are 2^16 or more behind)
    assert (np.abs(got - want) <= (2.0 ** -21 + 200 * U) * top[..., None]).all()


def test_attention_query_rows_inside_wider_ones(qa):
    rng = np.random.default_rng(3)
    cache, _ = make(qa, rng, "Q8_0", "f32", 5, 2, 50, 64)
    wide = dev(draw(rng, 5, 4 * 64 + 7))
    for at in (0, 3, 7):
        q = wide[:, at:at + 256].unflatten(-1, (4, 64))
        a, b = (qa.shared_prefix_attention(x, cache, ints([50, 3, 0, 1, 49]), beams=1) for x in (q, q.contiguous()))
        assert torch.equal(a, b)


# ---- beam search -------------------------------------------------------------------------------------------------


def check_beam(qa, logits, scores, finished=None, eos=None):
    got = qa.beam_select(dev(logits), dev(scores), None if finished is None else torch.from_numpy(finished).cuda(), eos)
    tokens, parents, out, ended = kv_ref.beam_select(logits, scores, finished, -1 if eos is None else eos)
    assert np.array_equal(got.parents.cpu().numpy(), parents)
    assert np.array_equal(got.tokens.cpu().numpy(), tokens)
    assert np.array_equal(got.finished.cpu().numpy().astype(bool), ended)
    have = got.scores.cpu().double().numpy()
    with np.errstate(invalid="ignore"):  # one rounding to f32 of a sum that is right to 1e-9
        ok = (have == out.astype(np.float32)) | (np.abs(have - out) <= U * np.abs(out) + 1e-9)
    assert ok.all()
    return got


@pytest.mark.parametrize("prompts,beams,vocab", [(1, 1, 1), (1, 1, 5000), (1, 2, 2051), (3, 4, 32001), (1, 64, 64), (2, 64, 9000), (5, 3, 2), (1, 33, 151936), (7, 8, 4096), (2, 5, 4097)])
def test_beam_select(qa, prompts, beams, vocab):
    print("beams", prompts, beams, vocab, flush=True)
    rng = np.random.default_rng(vocab + beams)
    logits = (rng.normal(size=(prompts, beams, vocab)) * 2.5).astype(np.float32)
    scores = -np.sort(rng.random((prompts, beams)).astype(np.float32) * 8, 1)
    check_beam(qa, logits, scores)
    finished = (rng.random((prompts, beams)) < 0.3).astype(np.uint8) * 7
    check_beam(qa, logits, scores, finished, vocab // 2)
    finished[:] = 1
    check_beam(qa, logits, scores, finished, vocab - 1)
    check_beam(qa, logits, scores, None, int(logits[0, 0].argmax()))


def test_beam_select_of_equal_and_missing_numbers(qa):
    """Ties, first steps, constant rows, masked rows, NaN and infinities: equal ones by rising beam * vocab + token."""
    rng = np.random.default_rng(6)
    for beams, vocab in ((4, 5000), (8, 20000), (64, 8200)):
        base = (rng.normal(size=(2, beams, vocab)) * 2).astype(np.float32)
        zero = np.zeros((2, beams), np.float32)
        first = np.full((2, beams), -np.inf, np.float32)
        first[:, 0] = 0
        check_beam(qa, base, first)                                   # first step
        check_beam(qa, np.zeros_like(base), zero)                     # everything equal
        check_beam(qa, np.broadcast_to(base[:, :1], base.shape).copy(), zero)  # beams equal
        x = np.round(base * 4) / 4                                    # many ties within a beam
        check_beam(qa, np.broadcast_to(x[:, :1], x.shape).copy(), zero)
        x = np.where(rng.random(base.shape) < 0.99, -np.inf, base).astype(np.float32)
        x[0, 1] = -np.inf                                             # a beam that may say nothing
        check_beam(qa, x, zero)
        x = np.full_like(base, -np.inf)
        x[:, 2, 7] = 1.0                                              # one token in all
        check_beam(qa, x, zero)
        x = base.copy()
        x[0, 0, ::3] = np.nan
        x[1, 1] = np.nan
        check_beam(qa, x, zero)
        x = base.copy()
        x[0, 0, 5] = np.inf
        s = zero.copy()
        s[0, 2], s[1, 0] = np.nan, -np.inf
        check_beam(qa, x, s)
        x = base.copy()
        x[:, :, 10] = -0.0
        x[:, :, 11] = 0.0
        x[x > 0] = -1.0
        x[:, :, 11], x[:, :, 10] = 0.0, -0.0
        check_beam(qa, np.broadcast_to(x[:, :1], x.shape).copy(), zero)
    check_beam(qa, base, first * 0 - np.inf)                          # no beam has a score


@pytest.mark.parametrize("prompts,beams,capacity", [(1, 1, 1), (2, 3, 50), (1, 8, 33), (3, 64, 700), (1, 5, 5000)])
def test_beam_lineage(qa, prompts, beams, capacity):
    rng = np.random.default_rng(capacity)
    width = -(-capacity // 32) * 32
    logits, scores = rng.normal(size=(prompts, beams, 100)).astype(np.float32), rng.normal(size=(prompts, beams)).astype(np.float32)
    rows = rng.integers(0, 256, size=(prompts * beams, width)).astype(np.uint8)
    lens = rng.integers(0, capacity, size=prompts * beams).astype(np.int32)
    lens[-1] = width + 3  # outside: left out
    if len(lens) > 2:
        lens[1] = -1
    lineage = torch.from_numpy(rows).cuda()
    got = qa.beam_select(dev(logits), dev(scores), lineage=lineage, lens=ints(lens))
    want = kv_ref.lineage_step(rows, got.parents.cpu().numpy(), lens)
    assert np.array_equal(got.lineage.cpu().numpy(), want)
    assert np.array_equal(lineage.cpu().numpy(), rows)
    again = qa.beam_select(dev(logits), dev(scores), lineage=lineage, lens=ints(lens), out_lineage=lineage)  # in place
    assert again.lineage is lineage and np.array_equal(lineage.cpu().numpy(), want)


# ---- together ------------------------------------------------------------------------------------------------------


def search(qa, rng, prompts, beams, steps, quant, capture):
    """A tiny model decodes `steps` tokens: keys, values and queries from a token's embedding, one attention, logits.  Returns what
    the library picks and what a plain search in 64 bits that copies whole histories would."""
    heads, kv, d, vocab, prefix = 4, 2, 64, 333, 45
    embed = rng.normal(size=(vocab, (heads + 2 * kv) * d)).astype(np.float32)
    head = (rng.normal(size=(heads * d, vocab)) * 0.2).astype(np.float32)
    pk, pv = draw(rng, prompts, prefix, kv, d), draw(rng, prompts, prefix, kv, d)
    plens = [prefix - 7 * g for g in range(prompts)]
    pre = qa.QuantizedKvCache(qa.KvCacheType[quant], prompts, kv, prefix, d)
    pre.append(dev(pk), dev(pv), ints([0] * prompts), ints(plens))
    pre_ref = kv_ref.Cache(BITS[quant], prompts, kv, prefix, d)
    pre_ref.append(pk, pv, [0] * prompts, plens)
    own = qa.QuantizedKvCache(qa.KvCacheType[quant], prompts * beams, kv, steps, d)
    n = prompts * beams
    E, H, plens_t = dev(embed), dev(head), ints(plens)
    tokens = torch.arange(n, dtype=torch.int32, device="cuda")
    scores = torch.full((prompts, beams), -np.inf, device="cuda")
    scores[:, 0] = 0
    finished = torch.zeros(prompts, beams, dtype=torch.uint8, device="cuda")
    lineage, lens = own.new_lineage(), torch.zeros(n, dtype=torch.int32, device="cuda")
    lineage += torch.arange(n, dtype=torch.uint8, device="cuda").remainder(beams).view(n, 1)  # the first step writes position 0

    def step():
        x = E[tokens.long()]
        q = x[:, :heads * d].unflatten(1, (heads, d))
        k, v = (x[:, at:at + kv * d].reshape(n, 1, kv, d) for at in (heads * d, (heads + kv) * d))
        own.append(k, v, lens)
        out = qa.shared_prefix_attention(q, own, lens + 1, prefix=pre, prefix_lens=plens_t, lineage=lineage)
        logits = (out.view(n, heads * d) @ H).view(prompts, beams, vocab).contiguous()
        picked = qa.beam_select(logits, scores, finished, 5, lineage=lineage, lens=lens + 1, out_lineage=lineage)
        tokens.copy_(picked.tokens.view(-1))
        scores.copy_(picked.scores)
        finished.copy_(picked.finished)
        lens.add_(1)
        return picked, logits

    if capture:
        keep = [t.clone() for t in (tokens, scores, finished, lens, lineage)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            result = step()
        for t, was in zip((tokens, scores, finished, lens, lineage), keep):
            t.copy_(was)
    trace = []
    for _ in range(steps):
        if capture:
            graph.replay()
            torch.zeros(100, device="cuda").sum().item()  # the program's own work between replays
            picked, logits = result
        else:
            picked, logits = step()
        trace.append([x.clone() for x in picked[:4]] + [logits.clone()])
    return trace, (embed, pre_ref, plens, heads, kv, d, head, lineage)


@pytest.mark.parametrize("quant,prompts,beams,steps", [("Q8_0", 1, 4, 40), ("Q4_0", 2, 3, 35), ("Q8_0", 2, 1, 10)])
def test_search_from_the_cache_and_lineage(qa, quant, prompts, beams, steps):
    """Append, attend, pick and reorder for many steps: each step's logits against the whole histories of the beams that
    the picks so far leave, each step's picks against its logits."""
    rng = np.random.default_rng(17)
    trace, (embed, pre_ref, plens, heads, kv, d, head, _) = search(qa, rng, prompts, beams, steps, quant, False)
    n = prompts * beams
    history, scores, finished = [[] for _ in range(n)], np.full((prompts, beams), -np.inf, np.float32), np.zeros((prompts, beams), np.uint8)
    scores[:, 0] = 0
    tokens = np.arange(n)
    for tk, pa, sc, fi, logits in trace:
        history = [h + [embed[t]] for h, t in zip(history, tokens)]
        rows = np.array(history)  # [n, positions, ..]
        own = kv_ref.Cache(BITS[quant], n, kv, rows.shape[1], d)
        own.append(rows[..., heads * d:(heads + kv) * d].reshape(n, -1, kv, d), rows[..., (heads + kv) * d:].reshape(n, -1, kv, d), [0] * n)
        q = np.array([embed[t][:heads * d].reshape(heads, d) for t in tokens])
        out, size, top, count = kv_ref.attention(q, own, [rows.shape[1]] * n, pre_ref, plens, None, beams, d ** -0.5)
        want = out.reshape(n, -1) @ head
        # each attention value by test_attention's bound, then the f32 product's own sum of heads * d terms
        tol = (2 * (size * (2.0 ** -22 + (d + 2) * U) + 2.0 ** -21) + 2 * (count / 16 + 64) * U + 2 * U) * top
        bound = np.repeat(tol, d, 1) @ np.abs(head) + heads * d * U * (np.abs(out.reshape(n, -1)) @ np.abs(head))
        assert (np.abs(logits.cpu().numpy().reshape(n, -1) - want) <= bound).all()
        w_tokens, w_parents, w_scores, w_finished = kv_ref.beam_select(logits.cpu().numpy(), scores, finished, 5)
        assert np.array_equal(w_tokens, tk.cpu().numpy()) and np.array_equal(w_parents, pa.cpu().numpy())
        assert np.array_equal(w_finished, fi.cpu().numpy().astype(bool))
        scores, finished = sc.cpu().numpy(), fi.cpu().numpy()
        tokens = w_tokens.ravel()
        history = [list(history[g * beams + p]) for g in range(prompts) for p in w_parents[g]]


def test_search_captured_and_replayed(qa):
    """The whole step in a graph, lengths growing on the device: every replay equals the eager step bit for bit."""
    a, _ = search(qa, np.random.default_rng(3), 2, 4, 36, "Q8_0", False)
    b, _ = search(qa, np.random.default_rng(3), 2, 4, 36, "Q8_0", True)
    for x, y in zip(a, b):
        for s, t in zip(x, y):
            assert torch.equal(s, t)


def test_other_streams_and_scratch(qa):
    """Two streams at once, each with its own scratch: the results of one call after the other."""
    rng = np.random.default_rng(12)
    own, _ = make(qa, rng, "Q8_0", "f32", 4, 2, 700, 128)
    q = [dev(draw(rng, 4, 8, 128)) for _ in range(2)]
    logits = [dev(draw(rng, 2, 4, 30000)) for _ in range(2)]
    scores, lens = torch.zeros(2, 4, device="cuda"), ints([700, 500, 1, 0])

    def work(i):
        out = [qa.shared_prefix_attention(q[i], own, lens, beams=1) for _ in range(3)]
        return out + [t for _ in range(3) for t in qa.beam_select(logits[i], scores)[:4]]

    want = [work(0), work(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            got.append(work(i))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_more_python_refusals(qa):
    cache, q = qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 2, 2, 32, 64), torch.zeros(2, 4, 64, device="cuda")
    lineage = torch.zeros(64 * 3, dtype=torch.uint8, device="cuda")
    for call in (lambda: cache.read(ints([0]), -1), lambda: qa.shared_prefix_attention(q, cache, ints([1, 1]), beams=0),
                 lambda: qa.shared_prefix_attention(q, cache, ints([1, 1]), scale=float("inf")), lambda: qa.shared_prefix_attention(q, cache, ints([1, 1]), beams=-1),
                 lambda: qa.shared_prefix_attention(q, cache, ints([1, 1]), prefix=qa.QuantizedKvCache(qa.KvCacheType.Q4_0, 1, 2, 32, 64), prefix_lens=ints([1])),
                 lambda: qa.beam_select(torch.zeros(1, 2, 9, device="cuda"), torch.zeros(1, 2, device="cuda"), lineage=lineage[:64].view(2, 32), lens=ints([0, 0]),
                                        out_lineage=lineage[32:96].view(2, 32))):
        with pytest.raises(qa.QmmError):
            call()


def test_captured_on_two_streams(qa):
    """Attention and selection captured on two streams, each with its own scratch, replayed at once and in turn."""
    rng = np.random.default_rng(5)
    own, _ = make(qa, rng, "Q4_0", "f32", 6, 2, 900, 64)
    lens, scores = ints([900, 7, 0, 500, 333, 64]), torch.zeros(2, 3, device="cuda")
    qs, logits = [dev(draw(rng, 6, 4, 64)) for _ in range(2)], [dev(draw(rng, 2, 3, 20000)) for _ in range(2)]

    def work(i):
        return [qa.shared_prefix_attention(qs[i], own, lens, beams=1), *qa.beam_select(logits[i], scores)[:4]]

    want, streams, graphs, results = [work(0), work(1)], [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for i, s in enumerate(streams):
        with torch.cuda.stream(s):
            work(i)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            results.append(work(i))
        graphs.append(graph)
    for turn in range(4):
        for t in results[0] + results[1]:
            t.zero_()
        torch.cuda.synchronize()
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
            if turn % 2:
                torch.cuda.synchronize()
                work(0)  # the program's own
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(x, y) for x, y in zip(want[i], results[i]))


def test_python_refusals(qa):
    cache = qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 2, 2, 32, 64)
    good = torch.zeros(1, 1, 2, 64, device="cuda")
    bad = [lambda: qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 1, 1, 8, 48), lambda: qa.QuantizedKvCache(qa.KvCacheType.Q8_0, 1, 1, 8, 64, device="cpu"),
           lambda: cache.append(good.double(), good.double(), ints([0])),
           lambda: cache.append(good, good.half(), ints([0])), lambda: cache.append(good, good, torch.zeros(1, dtype=torch.int64, device="cuda")),
           lambda: cache.append(good.cpu(), good, ints([0])), lambda: cache.append(good, good, ints([0, 0])), lambda: cache.append(good, good, ints([0]), first_slot=2),
           lambda: cache.append(good.transpose(2, 3), good, ints([0])), lambda: cache.append(good.expand(2, 1, 2, 64), good.expand(2, 1, 2, 64), ints([0, 0])),
           lambda: cache.read(ints([0, 0, 0]), 1), lambda: cache.read(ints([0]), 1, dtype=torch.float64),
           lambda: cache.read(ints([0]), 1, lineage=cache.new_lineage()[:1], beams=2), lambda: cache.read(ints([0]), 1, lineage=cache.new_lineage(), beams=3),
           lambda: qa.shared_prefix_attention(torch.zeros(2, 4, 64, device="cuda"), None, None), lambda: qa.shared_prefix_attention(torch.zeros(2, 4, 128, device="cuda"), cache, ints([1, 1])),
           lambda: qa.shared_prefix_attention(torch.zeros(2, 3, 64, device="cuda"), cache, ints([1, 1])), lambda: qa.shared_prefix_attention(torch.zeros(3, 4, 64, device="cuda"), cache, ints([1, 1, 1])),
           lambda: qa.shared_prefix_attention(torch.zeros(2, 4, 64, device="cuda"), cache, ints([1, 1]), max_len=33),
           lambda: qa.shared_prefix_attention(torch.zeros(2, 4, 64, device="cuda"), cache, ints([1, 1]), scale=float("nan")), lambda: qa.shared_prefix_attention(torch.zeros(2, 4, 64, device="cuda"), cache, None),
           lambda: qa.beam_select(torch.zeros(1, 2, 9, device="cuda").half(), torch.zeros(1, 2, device="cuda")), lambda: qa.beam_select(torch.zeros(1, 2, 9), torch.zeros(1, 2)),
           lambda: qa.beam_select(torch.zeros(1, 2, 9, device="cuda"), torch.zeros(2, 1, device="cuda")), lambda: qa.beam_select(torch.zeros(1, 65, 9, device="cuda"), torch.zeros(1, 65, device="cuda")),
           lambda: qa.beam_select(torch.zeros(1, 2, 9, device="cuda"), torch.zeros(1, 2, device="cuda"), torch.zeros(1, 2, dtype=torch.uint8, device="cuda")),
           lambda: qa.beam_select(torch.zeros(1, 2, 9, device="cuda"), torch.zeros(1, 2, device="cuda"), lineage=torch.zeros(2, 31, dtype=torch.uint8, device="cuda"), lens=ints([0, 0]))]
    for i, call in enumerate(bad):
        with pytest.raises(qa.QmmError):
            call()
            print("not refused:", i)
    assert qa.shared_prefix_attention(torch.zeros(0, 4, 64, device="cuda"), cache, ints([])).shape == (0, 4, 64)
    cache.append(good[:0], good[:0], ints([]))
    assert cache.read(ints([]), 5)[0].shape == (0, 5, 2, 64)
