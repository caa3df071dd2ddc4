"""GPU tests (pytest -m gpu) of the prompt layer's arguments: what it hands on, leaves alone and refuses."""
import numpy as np
import pytest
import torch

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


HIDDEN, HEADS, KV, D, INTER = 512, 8, 2, 64, 1024


def arguments(qa, oracle, **shapes):
    """What a layer of the sizes above is made of, its products of other shapes where they are named."""
    shapes = {**dict(q=(HEADS * D, HIDDEN), k=(KV * D, HIDDEN), v=(KV * D, HIDDEN), o=(HIDDEN, HEADS * D), gate=(INTER, HIDDEN), up=(INTER, HIDDEN), down=(HIDDEN, INTER)), **shapes}
    mm = {n: qa.QMatMul.from_qtensor(qa.QTensor.from_blocks(qa.GgmlDType.Q8_0, oracle.quantize(8, oracle.randn(10 + i, s, std=0.03)), s)) for i, (n, s) in enumerate(shapes.items())}
    dev = lambda seed, n: torch.from_numpy(oracle.randn(seed, (n,), mean=1.0, std=0.1)).cuda()  # noqa: E731
    return dict(input_layernorm=dev(30, HIDDEN), post_attention_layernorm=dev(31, HIDDEN), q_proj=mm["q"], k_proj=mm["k"], v_proj=mm["v"], qk_norm_weight=dev(32, 2 * D), o_proj=mm["o"],
                mlp=(mm["gate"], mm["up"], mm["down"]), num_heads=HEADS, num_kv_heads=KV, head_dim=D, rotary=qa.RotaryEmbedding(D))


def test_the_longest_prompt_is_handed_on(qa, oracle, monkeypatch):
    """Four prompts of 100 tokens: the attention hears of 100 keys (or of nothing), and the result is the same up to the order of f32 sums in front of
    products that quantize (the tolerance of test_gpu_prompt_layer.py)."""
    from izwi_amd import qwen3_layer
    heard = []

    def listen(*args, **how):
        heard.append(how.get("max_len_k"))
        return attention(*args, **how)

    attention = qwen3_layer.prompt_attention
    monkeypatch.setattr(qwen3_layer, "prompt_attention", listen)
    layer = qwen3_layer.Qwen3PromptLayer(**arguments(qa, oracle))
    x = torch.from_numpy(oracle.randn(40, (400, HIDDEN))).cuda()
    positions, starts = ints(np.tile(np.arange(100), 4)), ints(range(0, 401, 100))
    want = layer.forward(x, positions, starts)
    got = layer.forward(x, positions, starts, max_len=100)
    assert heard == [None, 100]
    for a, b in zip(got, want):
        assert (a - b).abs().max() <= 2e-2 * b.abs().max()


def test_tokens_of_no_prompt_have_no_attention(qa, oracle):
    """A padded batch: tokens in front of, between and behind the prompts come out as the rest of the layer makes them of their own activations,
    whatever the memory held that the attention's result stands in; the prompts' own tokens do not notice."""
    from izwi_amd.qwen3_layer import Qwen3PromptLayer
    layer = Qwen3PromptLayer(**arguments(qa, oracle))
    tokens, starts = 90, [5, 45, 70]
    x = torch.from_numpy(oracle.randn(41, (tokens, HIDDEN))).cuda()
    positions = ints(range(tokens))
    outside = torch.ones(tokens, dtype=torch.bool)
    outside[5:70] = False
    results = []
    for poison in (float("nan"), 3e38, 0.0):
        for n in (tokens * HEADS * D, tokens * HIDDEN, tokens * INTER, tokens * KV * D):  # what the allocator hands out next
            kept = [torch.full((n,), poison, device="cuda") for _ in range(8)]
            del kept
        results.append(layer.forward(x, positions, ints(starts))[0])
    for got in results:
        assert torch.isfinite(got).all() and torch.equal(got, results[0])
    alone = x + 0
    hidden = layer.gate_up.forward_silu_mul(alone, norm_weight=layer.w_post, eps=layer.eps)
    want = layer.down_proj.forward_fused(hidden, residual=alone)
    assert torch.equal(results[0][outside], want[outside])


def test_parts_that_do_not_fit_are_refused(qa, oracle):
    """Head numbers that the projections do not have (in any product that comes to the same number of elements, too), norms and products of other sizes."""
    from izwi_amd.qwen3_layer import Qwen3PromptLayer
    good = arguments(qa, oracle)
    Qwen3PromptLayer(**good)
    ones = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    for over in (dict(num_heads=4), dict(num_kv_heads=4), dict(num_kv_heads=0), dict(num_heads=9, num_kv_heads=2), dict(num_heads=4, num_kv_heads=1, head_dim=128),
                 dict(num_heads=4, num_kv_heads=1, head_dim=128, rotary=qa.RotaryEmbedding(128)), dict(rotary=qa.RotaryEmbedding(128)), dict(qk_norm_weight=ones(D)),
                 dict(post_attention_layernorm=ones(HIDDEN // 2)), dict(input_layernorm=ones(2 * HIDDEN)), dict(k_proj=good["q_proj"]), dict(v_proj=good["q_proj"]),
                 dict(o_proj=good["k_proj"]), dict(mlp=(good["mlp"][0], good["q_proj"], good["mlp"][2])), dict(mlp=(good["mlp"][0], good["mlp"][1], good["o_proj"]))):
        with pytest.raises(qa.QmmError):
            Qwen3PromptLayer(**{**good, **over})
