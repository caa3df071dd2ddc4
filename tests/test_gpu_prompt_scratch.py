"""GPU test (pytest -m gpu) of what prompt attention allocates: a stream's scratch grows to 256 MiB at most, sums and statistics of all parts together."""
import pytest
import torch

from gpu_streams import fresh_stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,heads,kv,d", [(2683, 32, 8, 256), (2572, 32, 8, 256), (1400, 16, 8, 128), (12, 32, 8, 128)])
def test_scratch_stays_within_its_bound(tokens, heads, kv, d):
    if not torch.cuda.is_available():
        pytest.fail("no GPU visible: the HIP path cannot run (there is no fallback)")
    import izwi_amd
    keys = max(tokens, 1000)
    q, k, v = (torch.randn(n, g, d, device="cuda") for n, g in ((tokens, heads), (keys, kv), (keys, kv)))
    out = izwi_amd.prompt_attention(q, k, v, causal=False)  # (code and the default stream's scratch)
    stream = fresh_stream()
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    with torch.cuda.stream(stream):
        izwi_amd.prompt_attention(q, k, v, causal=False, out=out)
    torch.cuda.synchronize()
    assert before - torch.cuda.mem_get_info()[0] <= 256 << 20
