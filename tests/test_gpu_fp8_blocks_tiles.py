"""Block-scaled fp8 products with more tiles than the card has CUs, where a
workgroup walks from tile to tile: ragged rows, channels and K, one to four
stages of K (an odd number swaps the ring's slots from tile to tile), channels
that cannot leave in whole 16-byte chunks, more groups than a wave has lanes,
groups without rows.  Tolerances: those of tests/test_gpu_fp8_blocks.py."""
import pytest
import torch

from oracle import fp8_blocks as O
from test_gpu_fp8_blocks import _check_delta, _experts, _routing, _tol, _weights, dev, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k,n_out", [(4300, 300, 5000), (4610, 100, 4111), (5000, 256, 4608), (2600, 390, 7180),
                                       (4096, 512, 5632)])
def test_linear_over_many_tiles(dtype, n, k, n_out):
    from spider_moe_amd import ForgeGEMM
    say("linear, many tiles", dtype, n, k, n_out)
    g = torch.Generator().manual_seed(n + k + n_out)
    x = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(dtype)
    q, s = _weights(g, n_out, k)
    b = torch.randn(n_out, generator=g)
    for bias, act in ((None, None), (b, "gelu")):
        got = ForgeGEMM().linear_fp8_blocks(x.to(dev), q, s, None if bias is None else bias.to(dev), act=act)
        again = ForgeGEMM().linear_fp8_blocks(x.to(dev), q, s, None if bias is None else bias.to(dev), act=act)
        assert torch.equal(got, again)
        y, mag, top = O.linear(x, q, s, bias, act)
        tol = _tol(y, mag + (0 if bias is None else b.abs().double()), top, k, dtype, act == "gelu")
        err = (got.cpu().double() - y).abs()
        assert bool((err <= tol + 1e-30).all()), (act, float((err / (tol + 1e-30)).max()))


@pytest.mark.parametrize("activation,bias", [("gelu", True), ("swiglu", True), ("swiglu", False)])
@pytest.mark.parametrize("n,e,k,h,u", [(5000, 16, 2, 1312, 1296), (8400, 65, 4, 272, 272), (6000, 9, 2, 112, 2064)])
def test_expert_delta_over_many_tiles(activation, bias, n, e, k, h, u):
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("expert delta, many tiles", activation, bias, n, e, k, h, u)
    g = torch.Generator().manual_seed(n + e + h)
    ex = _experts(g, e, h, u, activation, bias)
    msg = torch.randn(n, 1, h, generator=g).bfloat16()
    idx, w = _routing(g, n, e, k)
    idx[idx == 1] = -1  # an expert without rows
    got = sparse_expert_delta_fp8_blocks(msg.to(dev), idx.view(n, 1, k).to(dev), w.view(n, 1, k).to(dev), ex)
    again = sparse_expert_delta_fp8_blocks(msg.to(dev), idx.view(n, 1, k).to(dev), w.view(n, 1, k).to(dev), ex)
    assert torch.equal(got, again)
    _check_delta(got, O.expert_delta(msg.view(n, h), idx, w, ex.w_up, ex.s_up, ex.w_down, ex.s_down, ex.b_up, ex.b_down,
                                     activation))
