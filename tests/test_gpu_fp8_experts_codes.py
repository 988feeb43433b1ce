"""The hidden activations' codes are the block quantizer's: at scales whose
reciprocal is rounded and activations that are the scale times the middle
between two codes, where a product with the reciprocal takes the other
neighbour in about 1 of 15."""
import pytest
import torch

from test_gpu_fp8_blocks import dev, say

pytestmark = pytest.mark.gpu


def _activations(g, e, u):
    """[e, u]: in each block of 128 the first is 448 s, the others s times
    (2 m + 1) / 16 * 2^j, m in [8, 16): exact in f32 (s has 19 bits)."""
    s = torch.randint(1 << 18, 1 << 19, (e, u // 128, 1), generator=g).double() / (1 << 18)
    m = torch.randint(8, 16, (e, u // 128, 128), generator=g).double()
    j = torch.randint(3, 8, (e, u // 128, 128), generator=g).double()
    a = s * (2 * m + 1) / 16 * 2.0 ** j
    a[:, :, 0] = 448.0 * s[:, :, 0]
    a = torch.minimum(a, a[:, :, :1])
    assert torch.equal(a.float().double(), a)
    return a.float().view(e, u)


@pytest.mark.parametrize("n", [4, 40, 600, 2100])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_hidden_activations_take_the_quantizers_codes(dtype, n):
    """GELU of a bias of at least 8 is the bias itself; the down weights hand on
    one channel each, so that the delta is code times scale, the bits of
    quantize_fp8_blocks (few tokens, then tiles of rows)."""
    from spider_moe_amd import (Fp8BlockExperts, dequantize_fp8_blocks, quantize_fp8_blocks,
                                sparse_expert_delta_fp8_blocks)
    say("activation codes", dtype, n)
    g = torch.Generator().manual_seed(n)
    e, h, u = 8, 512, 512
    act = _activations(g, e, u)
    eye = torch.eye(u).expand(e, h, u).contiguous().to(torch.float8_e4m3fn).to(dev)
    zero = torch.zeros(e, u, h).to(torch.float8_e4m3fn).to(dev)
    one = torch.ones(e, 4, 4, device=dev)
    ex = Fp8BlockExperts(zero, one, eye, one, b_up=act.to(dev))
    msg = torch.randn(n, h, generator=g).to(dtype).to(dev)
    idx = torch.randint(0, e, (n, 1), generator=g)
    got = sparse_expert_delta_fp8_blocks(msg, idx.int().to(dev), torch.ones(n, 1, device=dev), ex)
    q, s = quantize_fp8_blocks(act, block_rows=1)
    want = dequantize_fp8_blocks(q, s, block_rows=1)[idx.view(-1)].to(dtype)
    assert torch.equal(got.cpu(), want), int((got.cpu() != want).sum())


@pytest.mark.parametrize("n", [4, 40, 600])
def test_gated_activations_take_the_quantizers_codes(n):
    """SwiGLU with a gate of 32, which SiLU hands on as it is."""
    from spider_moe_amd import (Fp8BlockExperts, dequantize_fp8_blocks, quantize_fp8_blocks,
                                sparse_expert_delta_fp8_blocks)
    say("gated activation codes", n)
    g = torch.Generator().manual_seed(n)
    e, h, u = 4, 512, 512
    act = _activations(g, e, u)
    w_up = torch.zeros(e, 2 * u, h)
    w_up[:, :u, 0] = 32.0
    eye = torch.eye(u).expand(e, h, u).contiguous().to(torch.float8_e4m3fn).to(dev)
    ex = Fp8BlockExperts(w_up.to(torch.float8_e4m3fn).to(dev), torch.ones(e, 8, 4, device=dev), eye,
                         torch.ones(e, 4, 4, device=dev), b_up=(act / 32).to(dev), activation="swiglu")
    msg = torch.zeros(n, h, device=dev)
    msg[:, 0], msg[:, 1] = 1.0, 448.0  # a block of scale 1
    idx = torch.randint(0, e, (n, 1), generator=g)
    got = sparse_expert_delta_fp8_blocks(msg, idx.int().to(dev), torch.ones(n, 1, device=dev), ex)
    q, s = quantize_fp8_blocks(act, block_rows=1)
    want = dequantize_fp8_blocks(q, s, block_rows=1)[idx.view(-1)]
    assert torch.equal(got.cpu(), want), int((got.cpu() != want).sum())
