"""Block-scaled fp8 products with more tiles than the card has CUs: ragged
rows, channels and K, one to four stages of K, channels that cannot leave in
whole 16-byte chunks, more groups than a wave has lanes, groups without rows;
every kind of dispatch plan; captured steps.  Tolerances: those of
tests/test_gpu_fp8_blocks.py."""
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


@pytest.mark.parametrize("n,e,k", [(3, 70, 4), (300, 70, 6), (300, 5, 20), (1300, 70, 6), (1300, 24, 20), (1024, 256, 16),
                                   (1025, 3, 1), (2048, 190, 8), (2048, 200, 4), (2049, 90, 4), (4096, 96, 2),
                                   (4095, 97, 2), (4097, 8, 2), (3000, 40, 5)])
def test_expert_delta_every_plan(n, e, k):
    """The few-token step, the plan by bit masks (one, two and four tokens a
    thread, up to its limits) and the general one: more experts than a wave
    has lanes, more choices than the bit masks take (k > 16), the same id several times in a row of choices, int64 ids past 32
    bits (outside [0, E), as any other id there)."""
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("expert delta, plans", n, e, k)
    g = torch.Generator().manual_seed(n + e + k)
    ex = _experts(g, e, 144, 80, "swiglu", True)
    msg = torch.randn(n, 144, generator=g)
    idx = torch.randint(0, e, (n, k), generator=g)
    w = torch.rand(n, k, generator=g)
    idx[0] = e - 1
    idx[1, :2] = torch.tensor([1 << 32, -(1 << 32)])[:k]
    got = sparse_expert_delta_fp8_blocks(msg.to(dev), idx.to(dev), w.to(dev), ex)
    ids = torch.where((idx >= 0) & (idx < e), idx, torch.full_like(idx, -1))
    _check_delta(got, O.expert_delta(msg, ids, w, ex.w_up, ex.s_up, ex.w_down, ex.s_down, ex.b_up, ex.b_down, "swiglu"))


def test_captured_steps_beside_eager_ones():
    """Two captured steps of different sizes replayed in turn with eager calls
    and another stream's between them: each replay gives the eager result."""
    from spider_moe_amd import ForgeSelect, sparse_expert_delta_fp8_blocks
    say("captured steps")
    g = torch.Generator().manual_seed(21)
    ex = _experts(g, 16, 272, 144, "swiglu", True)
    select = ForgeSelect()

    def step(x, z):
        w, idx = select.route_groups(z, top_k=2, num_groups=4, top_groups=2)
        return sparse_expert_delta_fp8_blocks(x, idx, w, ex)

    held, graphs = [], []
    for n in (5, 300, 1100):  # few tokens, plan by bit masks, general plan
        x = torch.randn(n, 272, generator=g).bfloat16().to(dev)
        z = torch.randn(n, 16, generator=g).to(dev)
        step(x, z)
        torch.cuda.synchronize()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = step(x, z)
        held.append((x, z, out))
        graphs.append(gr)
    side = torch.cuda.Stream()
    for r in range(3):
        for (x, z, out), gr in zip(held, graphs):
            x.copy_(torch.randn(x.shape, generator=g).bfloat16())
            z.copy_(torch.randn(z.shape, generator=g))
            torch.cuda.synchronize()
            gr.replay()
            with torch.cuda.stream(side):  # at the same time
                beside = step(x, z)
            torch.cuda.synchronize()
            assert torch.equal(out, step(x, z)) and torch.equal(beside, out), (r, len(x))
