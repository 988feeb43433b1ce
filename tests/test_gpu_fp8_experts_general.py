"""The expert step on the general dispatch plan and the separate quantizer
(more tokens or choices than the plan by bit masks takes), captured; and a
prompt of messages wider than 4096 channels."""
import pytest
import torch

from oracle import fp8_blocks as O
from test_gpu_fp8_blocks import _check_delta, _experts, _routing, dev, say

pytestmark = pytest.mark.gpu


def test_captured_steps_of_the_general_plan():
    """More than 4096 tokens; more than 16 choices a token; more than 8192
    choices: captured, replayed in turn on new inputs with eager calls and
    another stream's between them."""
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("captured general plans")
    g = torch.Generator().manual_seed(31)
    ex = _experts(g, 24, 144, 80, "swiglu", True)
    held = []
    for n, k in ((4200, 1), (300, 20), (1700, 5)):
        x = torch.randn(n, 144, generator=g).bfloat16().to(dev)
        idx, w = _routing(g, n, 24, k)
        idx, w = idx.to(dev), w.to(dev)
        sparse_expert_delta_fp8_blocks(x, idx, w, ex)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = sparse_expert_delta_fp8_blocks(x, idx, w, ex)
        held.append((x, idx, w, out, gr))
    side = torch.cuda.Stream()
    for r in range(3):
        for x, idx, w, out, gr in held:
            i2, w2 = _routing(g, *(x.shape[0], 24, idx.shape[1]))
            if r == 2:
                i2[::3] = -1  # tokens without experts
            x.copy_(torch.randn(x.shape, generator=g).bfloat16())
            idx.copy_(i2)
            w.copy_(w2)
            torch.cuda.synchronize()
            gr.replay()
            with torch.cuda.stream(side):  # at the same time
                beside = sparse_expert_delta_fp8_blocks(x, idx, w, ex)
            torch.cuda.synchronize()
            assert torch.equal(out, sparse_expert_delta_fp8_blocks(x, idx, w, ex)) and torch.equal(beside, out), (r, len(x))
            if r == 2:
                assert not bool(out[::3].any())
                _check_delta(out, O.expert_delta(x.cpu(), idx, w, ex.w_up, ex.s_up, ex.w_down, ex.s_down, ex.b_up,
                                                 ex.b_down, "swiglu"))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k,h", [(1, 2, 4112), (2, 3, 7168), (70, 2, 4112), (300, 3, 5136), (9000, 1, 4224)])
def test_wide_messages(dtype, n, k, h):
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("wide messages", dtype, n, k, h)
    g = torch.Generator().manual_seed(n + h)
    ex = _experts(g, 4, h, 48, "gelu", True)
    msg = torch.randn(n, h, generator=g).to(dtype)
    idx, w = _routing(g, n, 4, k)
    got = sparse_expert_delta_fp8_blocks(msg.to(dev), idx.to(dev), w.to(dev), ex)
    m = min(n, 400)  # the oracle on the first and the last rows
    for at in (slice(0, m), slice(n - m, n)):
        _check_delta(got[at], O.expert_delta(msg[at], idx[at], w[at], ex.w_up, ex.s_up, ex.w_down, ex.s_down, ex.b_up,
                                             ex.b_down, "gelu", f32_sums=dtype == torch.float32))
