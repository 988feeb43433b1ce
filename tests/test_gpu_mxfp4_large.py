"""Microscaled 4-bit products on large tiles: ends of K and of the output, special
values, other streams and captured graphs, against oracle/mxfp4.py in 64 bits
with the bounds of test_gpu_mxfp4.py (the products' error bounds that the oracle
returns, and half a step of the output's type)."""
import pytest
import torch

from test_gpu_mxfp4 import check_experts, check_linear, dev, experts_of, routing, say, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("k", [1, 33, 250, 257, 511, 777])
def test_ends_of_k_and_rows_of_any_alignment(dtype, k):
    say("large linear", dtype, k)
    g = torch.Generator().manual_seed(k)
    n, n_out = 2561, 4099  # 11 x 17 tiles of 256 x 256, neither whole; output rows of odd pitch
    x = torch.randn(n, k + 5, generator=g).to(dtype).to(dev)[:, 3:3 + k]
    codes, scale = weight(n_out, k)
    check_linear(x, codes, scale)
    check_linear(x, codes, scale, torch.randn(n_out, generator=g).to(dev), "gelu")


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
@pytest.mark.parametrize("h,u", [(32, 32), (288, 544), (544, 96)])
def test_experts_unevenly_loaded(act, h, u):
    say("large experts", act, h, u)
    ex = experts_of(5, h, u, act, True)
    g = torch.Generator().manual_seed(h + u)
    n = 1700
    x = torch.randn(n, h, generator=g).bfloat16().to(dev)
    idx, w = routing(n, 5, 2, skew=3.0)
    check_experts(x, idx, w, ex)
    idx[:] = torch.tensor([3, 1], dtype=torch.int32, device=dev)  # three experts without rows
    check_experts(x, idx, w, ex)


def test_nan_and_infinity_stay_in_their_token():
    from spider_moe_amd import sparse_expert_delta_mxfp4
    say("large NaN")
    ex = experts_of(4, 64, 96, "swiglu", False)
    n = 1500
    x = torch.randn(n, 64, generator=torch.Generator().manual_seed(1)).to(dev)
    idx, w = routing(n, 4, 2)
    want = sparse_expert_delta_mxfp4(x, idx, w, ex)
    bad = [0, 127, 128, 777, n - 1]
    y = x.clone()
    for i, r in enumerate(bad):
        y[r, 7 * i] = float("nan") if i % 2 else float("inf")
    got = sparse_expert_delta_mxfp4(y, idx, w, ex)
    keep = torch.ones(n, dtype=torch.bool, device=dev)
    keep[bad] = False
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[~keep]).all()


def test_other_stream_and_graph():
    from spider_moe_amd import ForgeGEMM, sparse_expert_delta_mxfp4
    say("large graph")
    ex = experts_of(4, 96, 160, "gelu", True)
    codes, scale = weight(4096, 96)
    g = torch.Generator().manual_seed(3)
    n = 2600
    x = torch.randn(n, 96, generator=g).bfloat16().to(dev)
    idx, w = routing(n, 4, 2)

    def step(a):
        d = sparse_expert_delta_mxfp4(a, idx, w, ex)
        return d, ForgeGEMM().linear_mxfp4(a + d, codes, scale)

    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    held = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(held)
    for i in range(4):
        new = torch.randn(n, 96, generator=g).bfloat16().to(dev)
        held.copy_(new)
        graph.replay()
        want = step(new)
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b), i
