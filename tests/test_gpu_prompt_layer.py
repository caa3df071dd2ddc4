"""The operators on whole prompts as they are used together (pytest -m gpu): a prompt's layer against the decode layer token by token, the
decode step that goes on from its keys and values, the quantized cache behind it, a layer of experts behind a scored router."""
import numpy as np
import pytest
import torch

import prompt_ref

pytestmark = pytest.mark.gpu


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


def parts(qa, oracle, hidden, heads, kv_heads, d, inter, quant=8):
    shapes = {"q": (heads * d, hidden), "k": (kv_heads * d, hidden), "v": (kv_heads * d, hidden), "o": (hidden, heads * d), "gate": (inter, hidden),
              "up": (inter, hidden), "down": (hidden, inter)}
    mm = {n: qa.QMatMul.from_qtensor(qa.QTensor.from_blocks(qa.GgmlDType(quant), oracle.quantize(quant, oracle.randn(10 + i, s, std=0.03)), s)) for i, (n, s) in enumerate(shapes.items())}
    dev = lambda seed, n: torch.from_numpy(oracle.randn(seed, (n,), mean=1.0, std=0.1)).cuda()  # noqa: E731
    return mm, dev(30, hidden), dev(31, hidden), dev(32, 2 * d)


@pytest.mark.parametrize("hidden,heads,kv_heads,d,inter", [(512, 8, 2, 64, 1024), (1024, 8, 4, 128, 1024)])
def test_prompt_layer_is_the_decode_layer_token_by_token(qa, oracle, hidden, heads, kv_heads, d, inter):
    """Prompts of 13, 1 and 7 tokens in one call, each against its tokens one after the other through the decode layer; then a decode step on
    the prompt layer's keys and values.

    Tolerances.  One row has its norm folded into the product, several have it in front: of Q8_0 activation blocks the f16 scale is rounded at
    another magnitude, 2^-11 a block in either form.  B blocks with contributions c_b differ by at most 2^-10 sum |c_b| <= 2^-10 sqrt(B)
    sqrt(sum c_b^2), so keys and values (B = hidden / 32, at most 32) by 5.5e-3 of their size in the root mean square, which is a third of the
    largest or less among some hundred: 2e-3 of the largest, asked is twice that.  What follows is quantized again: rows that differ by
    more than a fraction of a step (the largest of 32 values / 127, 2 % of their root mean square) are rounded independently, and two
    such roundings leave sqrt(2 / 12) of a step, 0.8 %, of the root mean square of the row, and of a product of it.  Three products in a row
    (o; gate and up; down) make 1.6 %, of which the largest of some hundred outputs sees three and a half times, being itself three
    times the root mean square: 2e-2 of the largest output."""
    from izwi_amd.qwen3_layer import Qwen3DecodeLayer, Qwen3PromptLayer
    mm, w_in, w_post, qk_w = parts(qa, oracle, hidden, heads, kv_heads, d, inter)
    rotary = qa.RotaryEmbedding(d, base=1e4)
    decode = Qwen3DecodeLayer(w_in, w_post, mm["q"], mm["k"], mm["v"], qk_w, mm["o"], mm["gate"], mm["up"], mm["down"], heads, kv_heads, d, 1e-6)
    prompt = Qwen3PromptLayer(w_in, w_post, mm["q"], mm["k"], mm["v"], qk_w, mm["o"], (mm["gate"], mm["up"], mm["down"]), heads, kv_heads, d, rotary, 1e-6)
    lens = [13, 1, 7]
    starts = np.cumsum([0] + lens)
    x = torch.from_numpy(oracle.randn(40, (sum(lens), hidden))).cuda()
    y, keys, values = prompt.forward(x, ints(np.concatenate([np.arange(n) for n in lens])), ints(starts))
    freqs = rotary.frequencies.cpu().numpy()
    for a, b in zip(starts, starts[1:]):
        caches = [torch.zeros(1, kv_heads, 32, d, device="cuda") for _ in range(2)]
        cos_sin = [torch.from_numpy(np.concatenate([f(pos * freqs) for f in (np.cos, np.sin)]).astype(np.float32)[None]).cuda() for pos in range(b - a + 1)]
        for pos in range(b - a):
            want = decode.forward(x[a + pos:a + pos + 1], cos_sin[pos], caches[0], caches[1], pos)
            got = y[a + pos:a + pos + 1]
            assert (got - want).abs().max() <= 2e-2 * want.abs().max(), (a, pos)
        for cache, rows in zip(caches, (keys, values)):
            have = rows[a:b].transpose(0, 1)
            assert (have - cache[0, :, :b - a]).abs().max() <= 4e-3 * cache.abs().max()
        # one more token, on the decode layer's own caches and on the prompt layer's keys and values
        mine = [torch.zeros_like(c) for c in caches]
        for cache, rows in zip(mine, (keys, values)):
            cache[0, :, :b - a] = rows[a:b].transpose(0, 1)
        new = torch.from_numpy(oracle.randn(50 + int(a), (1, hidden))).cuda()
        want, got = (decode.forward(new, cos_sin[b - a], c[0], c[1], int(b - a)) for c in (caches, mine))
        assert (got - want).abs().max() <= 2e-2 * want.abs().max()


@pytest.mark.parametrize("quant", ["Q8_0", "Q4_0"])
def test_prompt_into_the_quantized_cache_and_on(qa, quant):
    """A prompt's rotated keys and values go into the quantized cache; the attention over it agrees with the prompt attention of the new
    token over the values that the cache stands for.  Both are within 1e-5 of the largest value of 64 bits here (scores up to 30)."""
    rng = np.random.default_rng(2)
    heads, kv, d, lens = 8, 2, 128, [50, 33]
    rotary = qa.RotaryEmbedding(d, base=1e6, scaling=qa.RopeScaling.llama3(8.0, 4096))
    row = torch.from_numpy(rng.normal(size=(sum(lens), heads + 2 * kv, d)).astype(np.float32)).cuda()
    q, k, v = row.split((heads, kv, kv), 1)
    positions = ints(np.concatenate([np.arange(n) for n in lens]))
    rope_q, rope_k = qa.rope_positions(q, k, positions, rotary)
    cache = qa.QuantizedKvCache(qa.KvCacheType[quant], 2, kv, 64, d)
    at = 0
    for slot, n in enumerate(lens):
        cache.append(rope_k[None, at:at + n], v[None, at:at + n], ints([0]), first_slot=slot)
        at += n
    new = rope_q[[lens[0] - 1, sum(lens) - 1]].contiguous()
    got = qa.shared_prefix_attention(new, cache, ints(lens))
    have_k, have_v = (t.reshape(-1, kv, d) for t in cache.read(ints([0, 0]), 64, ints(lens)))
    want = qa.prompt_attention(new, have_k, have_v, ints([0, 1, 2]), ints([0, lens[0], 64]), max_len_k=64)  # of the second all 64: zeros behind
    assert (got[0] - want[0]).abs().max() <= 2e-5 * have_v.abs().max()
    want = qa.prompt_attention(new[1:], have_k[64:64 + lens[1]], have_v[64:64 + lens[1]])
    assert (got[1] - want[0]).abs().max() <= 2e-5 * have_v.abs().max()


@pytest.mark.parametrize("routing", [dict(), dict(scoring="sigmoid", groups=4, top_groups=2, scale=2.5)])
def test_sparse_mlp_is_its_experts(qa, oracle, routing):
    """Tokens through the router, the sort and the experts' products, against the experts one by one by the restated routing of the router's logits."""
    from izwi_amd.qwen3_layer import SparseMlp
    n, hidden, inter, top_k, tokens = 16, 512, 256, 4, 37
    rng = np.random.default_rng(6)
    router_w = oracle.randn(1, (n, hidden), std=0.06)
    router = qa.QMatMul.from_qtensor(qa.QTensor.from_blocks(qa.GgmlDType.Q8_0, oracle.quantize(8, router_w), (n, hidden)))
    blocks = {name: oracle.quantize(12, oracle.randn(2 + i, (n * s[0], s[1]), std=0.05)) for i, (name, s) in enumerate((("gate", (inter, hidden)), ("up", (inter, hidden)), ("down", (hidden, inter))))}
    stack = {name: qa.QTensor.from_blocks(qa.GgmlDType.Q4K, b, (n, hidden, inter) if name == "down" else (n, inter, hidden)) for name, b in blocks.items()}
    if routing:
        routing = dict(routing, bias=torch.from_numpy((rng.normal(size=n) * 0.1).astype(np.float32)).cuda())
    mlp = SparseMlp(router, qa.MoeExperts(stack["gate"], stack["up"], stack["down"]), top_k, **routing)
    x = torch.from_numpy(oracle.randn(9, (tokens, hidden))).cuda()
    got = mlp.forward(x).cpu().numpy()
    logits = router.forward(x).cpu().numpy()
    bias = routing["bias"].cpu().numpy() if routing else None
    ids, weights = prompt_ref.route(logits, top_k, routing.get("scoring", "softmax"), bias, routing.get("groups", 1), routing.get("top_groups", 1), 2 if routing else 1, True, routing.get("scale", 1.0))
    one = {name: [qa.QMatMul.from_qtensor(qa.QTensor.from_blocks(qa.GgmlDType.Q4K, np.asarray(b).reshape(n, -1)[e], (hidden, inter) if name == "down" else (inter, hidden))) for e in range(n)]
           for name, b in blocks.items()}
    want = np.zeros((tokens, hidden))
    for t in range(tokens):
        row = x[t:t + 1].contiguous()
        for e, w in zip(ids[t], weights[t]):
            g, u = one["gate"][e].forward(row), one["up"][e].forward(row)
            want[t] += w * one["down"][e].forward((torch.nn.functional.silu(g) * u).contiguous()).double().cpu().numpy()[0]
    assert np.abs(got - want).max() <= 2e-3 * np.abs(want).max()


def test_prompt_layer_of_experts_and_its_refusals(qa, oracle):
    """A layer with experts: no token, one token, several prompts as alone; a router of another size and activations of another width are refused.
    (Up to two rows have their norm folded into the products, so the prompts are compared among themselves: 5 and 3 tokens in one call and in two.
    What a row meets is the same then, up to the order of f32 sums where kernels go by the number of rows: 2e-5.)"""
    from izwi_amd.qwen3_layer import Qwen3PromptLayer, SparseMlp
    n, hidden, inter, heads, kv_heads, d = 8, 512, 256, 8, 2, 64
    mm, w_in, w_post, qk_w = parts(qa, oracle, hidden, heads, kv_heads, d, inter)

    def stack(seed, rows, cols, quant=12):
        return qa.QTensor.from_blocks(qa.GgmlDType(quant), oracle.quantize(quant, oracle.randn(seed, (n * rows, cols), std=0.05)), (n, rows, cols))

    experts = qa.MoeExperts(stack(60, inter, hidden), stack(61, inter, hidden), stack(62, hidden, inter))
    router = lambda rows: qa.QMatMul.from_qtensor(qa.QTensor.from_blocks(qa.GgmlDType.Q8_0, oracle.quantize(8, oracle.randn(63, (rows, hidden), std=0.06)), (rows, hidden)))  # noqa: E731
    for rows in (4, 16):
        with pytest.raises(qa.QmmError):
            SparseMlp(router(rows), experts, 2)
    layer = Qwen3PromptLayer(w_in, w_post, mm["q"], mm["k"], mm["v"], qk_w, mm["o"], SparseMlp(router(n), experts, 2), heads, kv_heads, d, qa.RotaryEmbedding(d), 1e-6)
    x = torch.from_numpy(oracle.randn(64, (8, hidden))).cuda()
    for bad in (x[:, :256].contiguous(), x.half(), x[0]):
        with pytest.raises(qa.QmmError):
            layer.forward(bad, ints(range(8)))
    with pytest.raises(qa.QmmError):
        layer.sparse.forward(x[:, :256].contiguous())
    y, k, v = layer.forward(x[:0], ints([]))
    assert y.shape == (0, hidden) and k.shape == v.shape == (0, kv_heads, d)
    y, k, v = layer.forward(x[:1], ints([0]))
    assert y.shape == (1, hidden) and torch.isfinite(y).all()
    y, k, v = layer.forward(x, ints([0, 1, 2, 3, 4, 0, 1, 2]), ints([0, 5, 8]))
    for a, b in ((0, 5), (5, 8)):
        one = layer.forward(x[a:b].contiguous(), ints(range(b - a)))
        for got, want in zip((y, k, v), one):
            assert (got[a:b] - want).abs().max() <= 2e-5 * want.abs().max()
