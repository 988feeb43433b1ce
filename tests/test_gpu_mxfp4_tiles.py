"""Microscaled 4-bit products at the sizes that the middle kernel's taller tiles
take (256 CUs): 64 rows at 57 to 112 rows an expert, 128 at 113 to 511, both
where that leaves 256 tiles or more of 128 channels (SwiGLU: 64); dense 128 x 128
past 1024 tiles of 64 x 64 and below the large kernel's sizes.  Against
oracle/mxfp4.py in 64 bits with the bounds of test_gpu_mxfp4.py."""
import pytest
import torch

from test_gpu_mxfp4 import check_experts, check_linear, dev, experts_of, routing, say, weight

pytestmark = pytest.mark.gpu


def tiles(rows, groups, bm, channels, ch):
    """Row tiles over groups as evenly filled as may be, times strips."""
    per = -(-rows // groups)
    return groups * -(-per // bm) * -(-channels // ch)


def height(rows, groups, channels, ch):
    """Rows of a grouped tile by the rule that the header states."""
    per = -(-rows // groups)
    bm = 32 if per <= 56 else 64 if per <= 112 else 128
    while bm > 32 and tiles(rows, groups, bm, channels, ch) < 256:
        bm //= 2
    return bm


# --------------------------------------------------------------------- dense ----
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("k", [1, 31, 96, 250, 257, 512, 777, 1024])
def test_dense_128_by_128(dtype, k):
    """2000 x 2800 whole chunks, 1999 x 2797 ends inside a tile and an odd pitch."""
    g = torch.Generator().manual_seed(k)
    for n, n_out in ((2000, 2800), (1999, 2797)):
        say("dense", dtype, n, k, n_out)
        assert tiles(n, 1, 64, n_out, 64) > 1024 and tiles(n, 1, 256, n_out, 256) < 160
        x = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(dtype).to(dev)
        codes, scale = weight(n_out, k)
        check_linear(x, codes, scale)
        check_linear(x, codes, scale, (torch.randn(n_out, generator=g) * 0.1).to(dev), "gelu")


def test_dense_nan_and_what_lies_behind():
    from spider_moe_amd import ForgeGEMM
    say("dense nan")
    n, k, n_out = 2000, 290, 2800
    x = torch.randn(n, k, generator=torch.Generator().manual_seed(5)).to(dev)
    codes, scale = weight(n_out, k)
    nb = -(-k // 32)
    wide = torch.full((n_out, 20), 0xFF, dtype=torch.uint8, device=dev)
    wide[:, :nb] = scale
    want = check_linear(x, codes, scale)
    assert torch.equal(ForgeGEMM().linear_mxfp4(x, codes, wide[:, :nb]), want)
    wide[9, 3] = 255
    x[130, 7] = float("nan")
    nan = torch.isnan(check_linear(x, codes, wide[:, :nb]))
    assert nan[130].all() and nan[:, 9].all() and int(nan.sum()) == n + n_out - 1


# ------------------------------------------------------------------- grouped ----
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act,bias", [("gelu", True), ("swiglu", False), ("swiglu", True)])
@pytest.mark.parametrize("rows,n,e,k,h,u", [
    (64, 800, 32, 4, 512, 1408), (64, 777, 32, 4, 1024, 1408), (64, 1101, 48, 3, 544, 1184), (64, 1399, 28, 2, 864, 928),
    (128, 1600, 32, 4, 512, 1408), (128, 1500, 16, 2, 1056, 2080), (128, 4000, 24, 2, 736, 1184)])
def test_grouped(dtype, act, bias, rows, n, e, k, h, u):
    say("grouped", dtype, act, bias, n, e, k, h, u)
    assert height(n * k, e, u, 64 if act == "swiglu" else 128) == rows and height(n * k, e, h, 128) == rows
    ex = experts_of(e, h, u, act, bias)
    x = torch.randn(n, h, generator=torch.Generator().manual_seed(n + h)).to(dtype).to(dev)
    check_experts(x, *routing(n, e, k), ex)


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
@pytest.mark.parametrize("n,e,h,u", [(800, 32, 544, 1184), (1600, 32, 544, 1184)])
def test_grouped_unevenly(act, n, e, h, u):
    """A few experts with most of the rows, some with one or none; choices left
    out; every row on one expert."""
    say("uneven", act, n)
    ex = experts_of(e, h, u, act, True)
    x = torch.randn(n, h, generator=torch.Generator().manual_seed(n)).bfloat16().to(dev)
    idx, w = routing(n, e, 4, skew=3.0)
    idx[idx == 3] = 4
    idx[5], w[6] = -1, 0.0
    idx[7, 1], w[8, 2] = e, -1.0
    got = check_experts(x, idx, w, ex)
    assert (got[5] == 0).all() and (got[6] == 0).all()
    check_experts(x, torch.full_like(idx, e - 1), w, ex)


@pytest.mark.parametrize("n", [800, 1600])
def test_grouped_nan_stays_in_its_token(n):
    from spider_moe_amd import sparse_expert_delta_mxfp4
    say("grouped nan", n)
    ex = experts_of(32, 544, 1184, "swiglu", False)
    x = torch.randn(n, 544, generator=torch.Generator().manual_seed(n)).to(dev)
    idx, w = routing(n, 32, 4)
    want = sparse_expert_delta_mxfp4(x, idx, w, ex)
    y, bad = x.clone(), [0, 63, 64, 500, n - 1]
    for i, r in enumerate(bad):
        y[r, 100 * i] = float("nan") if i % 2 else float("inf")
    got = sparse_expert_delta_mxfp4(y, idx, w, ex)
    keep = torch.ones(n, dtype=torch.bool, device=dev)
    keep[bad] = False
    assert torch.equal(got[keep], want[keep]) and torch.isnan(got[~keep]).all()


@pytest.mark.parametrize("n", [800, 1600])
def test_grouped_in_a_graph(n):
    from spider_moe_amd import sparse_expert_delta_mxfp4
    say("grouped graph", n)
    ex = experts_of(32, 544, 1184, "gelu", True)
    g = torch.Generator().manual_seed(n)
    xs = [torch.randn(n, 544, generator=g).bfloat16().to(dev) for _ in range(3)]
    idx, w = routing(n, 32, 4)
    held = xs[0].clone()
    want = [sparse_expert_delta_mxfp4(x, idx, w, ex) for x in xs]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse_expert_delta_mxfp4(held, idx, w, ex)
    for i in range(4):
        held.copy_(xs[i % 3])
        graph.replay()
        again = sparse_expert_delta_mxfp4(xs[i % 3], idx, w, ex)
        torch.cuda.synchronize()
        assert torch.equal(out, want[i % 3]) and torch.equal(again, want[i % 3])
