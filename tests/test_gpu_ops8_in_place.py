"""Outputs in the memory of inputs: what the 8-bit serving operators allow gives the bits that it gives elsewhere."""
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m", [1, 2, 3, 33])
@pytest.mark.parametrize("n,k", [(896, 896), (2048, 2048), (100, 896), (896, 100)])
def test_matmul_over_its_tokens(dtype, m, n, k):
    """One token and two are quantized by every CTA of the product for itself elsewhere, but not here."""
    from e2e_browser_voice_agent_b200 import int8
    gen = torch.Generator(device=DEV)
    gen.manual_seed(m + n + k)
    w = torch.randint(-127, 128, (n, (k + 15) // 16 * 16), generator=gen, device=DEV).to(torch.int8)
    ws = 0.001 * torch.exp(torch.randn(n, generator=gen, device=DEV))
    for _ in range(20):
        buf = torch.randn(m, max(n, k) + 7, generator=gen, device=DEV).to(dtype)
        want = int8.matmul(buf[:, :k].clone(), w, ws)
        for at in (0, 3):
            z = buf.clone()
            got = int8.matmul(z[:, :k], w, ws, out=z[:, at:at + n])
            assert torch.equal(got, want)
            assert torch.equal(z[:, at + n:], buf[:, at + n:]) and torch.equal(z[:, :at], buf[:, :at])


def test_columns_of_one_buffer_stay_one_launch():
    """Tokens and outputs side by side share no memory, although their ranges interleave."""
    from e2e_browser_voice_agent_b200 import int8
    x = torch.randn(2, 900, device=DEV)
    w, ws = int8.quantize(torch.randn(128, 400, device=DEV))
    want = int8.matmul(x[:, :400].contiguous(), w, ws)
    assert torch.equal(int8.matmul(x[:, :400], w, ws, out=x[:, 450:578]), want)
