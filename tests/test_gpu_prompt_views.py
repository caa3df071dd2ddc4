"""GPU tests (pytest -m gpu): outputs in wide rows, whose gaps hold the call's own small inputs."""
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


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_small_inputs_between_the_rows_of_an_output(qa, dtype):
    tokens, heads, d, step = 6, 2, 64, 512
    q, weight = torch.randn(tokens, heads, d, device="cuda").to(dtype), torch.randn(2 * d, device="cuda").to(dtype)
    positions, starts = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in (range(6), [0, 2, 6]))
    room = torch.zeros(tokens * step, dtype=dtype, device="cuda")
    out = room.as_strided((tokens, heads, d), (step, d, 1))
    gap = lambda row, n, kind: room[row * step + heads * d: row * step + heads * d + n * kind.itemsize // dtype.itemsize].view(kind)  # noqa: E731
    w, p, s = gap(0, 2 * d, dtype), gap(1, tokens, torch.int32), gap(2, 3, torch.int32)
    w.copy_(weight), p.copy_(positions), s.copy_(starts)
    rotary = qa.RotaryEmbedding(d)
    assert torch.equal(qa.rope_positions(q, None, p, rotary, w, out=(out, None))[0], qa.rope_positions(q, None, positions, rotary, weight)[0])
    assert torch.equal(qa.prompt_attention(q, q, q, s, out=out), qa.prompt_attention(q, q, q, starts))
    assert torch.equal(w, weight) and torch.equal(p, positions) and torch.equal(s, starts)
    with pytest.raises(qa.QmmError):
        qa.rope_positions(q, None, room[4 * step:4 * step + 24].view(torch.int32)[:tokens], rotary, out=(out, None))
    with pytest.raises(qa.QmmError):
        qa.prompt_attention(q, q, q, room[4 * step:4 * step + 12].view(torch.int32)[:3], out=out)
