"""Group-limited routing (ForgeSelect.route_groups) and its gradient against
oracle/fp8_blocks.py in 64 bits.

The choice is that of the 64-bit scores on both sides, so indices are equal.
The weights are f32 arithmetic, relative to the value: expf (1 ulp = 2 * 2^-24
at most), for softmax its argument's rounding (|z - max| 2^-24) and a sum of 10
levels, a division, the sum of up to 64 chosen scores (6 levels, each score with
the errors before), a division and the scale: below (24 + |z - max|) * 2^-24.
The gradient is f32 arithmetic of about 20 operations on
terms whose magnitudes the bound below adds up (|ds| s and the softmax's sum),
rounded once more to the logits' type."""
import numpy as np
import pytest
import torch

from oracle import fp8_blocks as O

pytestmark = pytest.mark.gpu

dev = "cuda"
INF = float("inf")


def say(*a):
    print("[case]", *a, flush=True)


def _route(z, k, **kw):
    from spider_moe_amd import ForgeSelect
    args = dict(score=kw.get("score", "sigmoid"), bias=kw.get("bias"), num_groups=kw.get("groups", 1),
                top_groups=kw.get("top_groups", 1), renormalize=kw.get("renorm", True),
                scale=kw.get("scale", 1.0))
    return ForgeSelect().route_groups(z, top_k=k, **args)


def _check(z, k, **kw):
    bias = kw.get("bias")
    w, idx = _route(z.to(dev), k, **{**kw, "bias": None if bias is None else bias.to(dev)})
    assert w.dtype == torch.float32 and idx.dtype == torch.int32
    assert w.shape == idx.shape == (*z.shape[:-1], k)
    ww, wi = O.select_groups(z.reshape(-1, z.shape[-1]), k, **{"score": "sigmoid", **kw})
    got = idx.cpu().long().view(-1, k)
    assert torch.equal(got, wi), torch.nonzero((got != wi).any(-1)).flatten()[:5]
    err = (w.cpu().double().view(-1, k) - ww).abs()
    nan = torch.isnan(ww)
    assert torch.equal(torch.isnan(w.cpu()).view(-1, k), nan)
    z2 = z.reshape(-1, z.shape[-1]).double()
    far = (z2.nan_to_num(neginf=0.0).amax(-1, keepdim=True) - z2.gather(1, wi)).abs() if kw.get("score") == "softmax" \
        else torch.zeros_like(ww)
    tol = (24 + far.nan_to_num(posinf=0.0)) * 2.0 ** -24 * ww.abs() + 1e-38
    assert bool((err <= tol)[~nan].all()), float((err / tol)[~nan].max())


CASES = [  # E, K, groups, top_groups
    (1, 1, 1, 1), (2, 1, 2, 1), (3, 2, 1, 1), (8, 2, 1, 1), (16, 4, 4, 2), (16, 2, 16, 2), (33, 5, 1, 1),
    (48, 6, 6, 1), (60, 8, 6, 3), (64, 8, 8, 4), (65, 7, 5, 2), (128, 8, 1, 1), (160, 6, 8, 3),
    (192, 16, 64, 32), (255, 9, 85, 40), (256, 8, 8, 4), (256, 8, 1, 1), (256, 64, 8, 2), (256, 1, 256, 3),
    (255, 64, 3, 1), (256, 32, 128, 16), (64, 64, 1, 1),
]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("e,k,groups,top_groups", CASES)
def test_choice_and_weights(score, e, k, groups, top_groups):
    say("select groups", score, e, k, groups, top_groups)
    g = torch.Generator().manual_seed(e * 64 + k)
    for n, dtype, bias, renorm, scale in ((1, torch.float32, True, True, 2.5), (3, torch.bfloat16, True, False, 1.0),
                                          (66, torch.float32, False, True, 1.0), (257, torch.float16, True, True, 0.5)):
        z = (torch.randn(n, e, generator=g) * 1.5).to(dtype)
        b = torch.randn(e, generator=g) * 0.05 if bias else None
        _check(z, k, score=score, bias=b, groups=groups, top_groups=top_groups, renorm=renorm, scale=scale)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_many_near_scores(score):
    """20000 tokens of 256 experts whose scores lie close together: some pairs
    are nearer than f32 tells apart, and are still ordered as in 64 bits."""
    say("near scores", score)
    g = torch.Generator().manual_seed(3)
    z = torch.randn(20000, 256, generator=g) * 1e-3
    b = torch.randn(256, generator=g) * 1e-4
    _check(z, 8, score=score, bias=b, groups=8, top_groups=4)
    _check(z, 8, score=score, groups=8, top_groups=4)


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (8, 3)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_ties_go_to_the_lower_index(score, groups, top_groups):
    say("ties", score, groups)
    g = torch.Generator().manual_seed(4)
    z = torch.randint(-2, 3, (300, 64), generator=g).float()
    z[0] = 0.0
    z[1, :] = 1e-30
    _check(z, 6, score=score, groups=groups, top_groups=top_groups)
    _check(z.to(torch.bfloat16), 6, score=score, groups=groups, top_groups=top_groups, bias=torch.zeros(64))


@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2), (8, 3)])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_masked_experts(score, groups, top_groups):
    """-inf logits: single experts, all but one, whole groups, all of them; a
    bias does not bring a masked expert back."""
    say("masked", score, groups)
    g = torch.Generator().manual_seed(5)
    z = torch.randn(64, 32, generator=g)
    z[torch.rand(64, 32, generator=g) < 0.5] = -INF
    z[0] = -INF
    z[1, :] = -INF
    z[1, 17] = 0.3
    z[2, :16] = -INF
    z[3, 16:] = -INF
    z[4] = torch.finfo(torch.float32).min
    b = torch.randn(32, generator=g)
    for bias in (None, b):
        _check(z, 5, score=score, groups=groups, top_groups=top_groups, bias=bias)
    w, idx = _route(z[:1].to(dev), 5, score=score, groups=groups, top_groups=top_groups, bias=b.to(dev))
    assert not bool(w.any()) and len(set(idx.view(-1).tolist())) == 5


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_extreme_and_nan_logits(score):
    say("extreme", score)
    z = torch.zeros(8, 40)
    z[0, 3], z[0, 30] = 80.0, -80.0
    z[1] = torch.linspace(-100, 100, 40)
    z[2, 5] = float("nan")
    z[3, 5] = INF
    z[4] = 3e38
    z[5] = -3e38
    z[6, :20] = -INF
    z[6, 25] = float("nan")
    for groups, top_groups in ((1, 1), (4, 2)):
        _check(z, 4, score=score, groups=groups, top_groups=top_groups)
        w, idx = _route(z.to(dev), 4, score=score, groups=groups, top_groups=top_groups)
        assert all(len(set(r)) == 4 for r in idx.tolist())


def test_strides_streams_and_leading_dimensions():
    """A transposed and a sliced input, [B,T,E], an odd storage offset, and a
    stream of the caller's own."""
    say("strides")
    g = torch.Generator().manual_seed(6)
    z = torch.randn(5, 7, 48, generator=g)
    _check(z, 3, groups=4, top_groups=2)
    zt = torch.randn(48, 35, generator=g)
    w, idx = _route(zt.to(dev).t(), 3, groups=4, top_groups=2)
    ww, wi = _route(zt.t().contiguous().to(dev), 3, groups=4, top_groups=2)
    assert torch.equal(w, ww) and torch.equal(idx, wi)
    buf = torch.randn(1 + 35 * 50, generator=g)
    v = buf.to(dev)[1:].view(35, 50)[:, :48]
    w, idx = _route(v, 3, groups=4, top_groups=2)
    ww, wi = _route(v.contiguous(), 3, groups=4, top_groups=2)
    assert torch.equal(w, ww) and torch.equal(idx, wi)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        w2, i2 = _route(v, 3, groups=4, top_groups=2)
    s.synchronize()
    assert torch.equal(w2, ww) and torch.equal(i2, wi)
    w, idx = _route(torch.empty(0, 48, device=dev), 3)
    assert w.shape == idx.shape == (0, 3)


def _grad_bound(z, idx, d_w, score, renorm, scale):
    """Sum of the magnitudes that the gradient's f32 terms have."""
    z = z.double()
    s = torch.softmax(z, -1) if score == "softmax" else torch.sigmoid(z)
    sel = s.gather(1, idx)
    total = sel.sum(-1, keepdim=True).clamp_min(1e-9)
    q = sel / total
    g = d_w.double().abs()
    ds = (g + (g * q).sum(-1, keepdim=True)) / total if renorm else g
    ds = torch.zeros_like(s).scatter_add_(1, idx, ds * abs(scale))
    if score == "softmax":
        return s * (ds + (s * ds).sum(-1, keepdim=True))
    return ds * s * (1 - s)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("n,e,k,groups,top_groups", [(1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (5, 48, 6, 6, 2),
                                                     (777, 64, 2, 1, 1), (131, 255, 64, 3, 1), (64, 16, 1, 4, 1)])
def test_gradient(dtype, renorm, score, n, e, k, groups, top_groups):
    """Against autograd through the 64-bit formula at the chosen experts."""
    say("gradient", dtype, renorm, score, n, e, k)
    g = torch.Generator().manual_seed(n + e)
    z = (torch.randn(n, e, generator=g) * 2).to(dtype)
    b = torch.randn(e, generator=g) * 0.1
    d_w = torch.randn(n, k, generator=g)
    zg = z.to(dev).requires_grad_(True)
    w, idx = _route(zg, k, score=score, bias=b.to(dev), groups=groups, top_groups=top_groups, renorm=renorm, scale=1.7)
    assert w.requires_grad and not idx.requires_grad
    w.backward(d_w.to(dev))
    got = zg.grad
    assert got.dtype == dtype and got.shape == z.shape
    z64 = z.double().requires_grad_(True)
    O.select_groups_weights(z64, idx.cpu().long(), score=score, renorm=renorm, scale=1.7).backward(d_w.double())
    want = z64.grad
    bound = _grad_bound(z, idx.cpu().long(), d_w, score, renorm, 1.7)
    tiny = {torch.float32: 1e-37, torch.bfloat16: 1e-37, torch.float16: 2.0 ** -24}[dtype]
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    # ~20 f32 roundings, a sum over up to 64 slots, and expf's argument error |z| 2^-24
    tol = (64 + 2 * z.double().abs().max()) * 2.0 ** -24 * bound + half * want.abs() + tiny
    err = (got.cpu().double() - want).abs()
    assert bool((err <= tol).all()), (float((err / tol.clamp_min(1e-300)).max()))


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_gradient_against_differences(score):
    """Central differences of the operator's own forward pass, h = 2^-6 in f32:
    off by h^2 / 6 of the third derivative (below |w| <= 1.5 here) and the
    weights' rounding 8 * 2^-24 over h."""
    say("differences", score)
    g = torch.Generator().manual_seed(8)
    n, e, k = 6, 24, 4
    z = torch.randn(n, e, generator=g)
    for t in range(n):  # gaps of more than 2 h, so the choice stays
        z[t] = torch.linspace(-1.5, 1.5, e)[torch.randperm(e, generator=g)]
    d_w = torch.randn(n, k, generator=g).to(dev)
    zg = z.to(dev).requires_grad_(True)
    w, idx = _route(zg, k, score=score, scale=1.5)
    (got,) = torch.autograd.grad(w, zg, d_w)
    h = 2.0 ** -6
    for j in range(e):
        zp, zm = z.clone(), z.clone()
        zp[:, j] += h
        zm[:, j] -= h
        wp, ip = _route(zp.to(dev), k, score=score, scale=1.5)
        wm, im = _route(zm.to(dev), k, score=score, scale=1.5)
        assert torch.equal(ip, idx) and torch.equal(im, idx)
        diff = ((wp - wm) / (2 * h) * d_w).sum(-1)
        err = (diff - got[:, j]).abs()
        assert bool((err <= (h * h + 16 * 2.0 ** -24 / h) * 1.5 * d_w.abs().sum(-1)).all()), (j, float(err.max()))


def test_gradient_with_masks_repeats_and_ids_outside():
    """The backward entry on choices that a program wrote itself: an id twice,
    ids outside [0, E); masked experts and fully masked rows get exact zeros."""
    say("gradient: masks, repeats")
    from spider_moe_amd import _native as nat
    g = torch.Generator().manual_seed(9)
    n, e, k = 5, 20, 4
    z = torch.randn(n, e, generator=g)
    z[1, :10] = -INF
    z[2] = -INF
    idx = torch.tensor([[3, 3, 5, 1], [12, 13, 2, 19], [0, 1, 2, 3], [7, -1, 20, 8], [4, 4, 4, 4]], dtype=torch.int32)
    d_w = torch.randn(n, k, generator=g)
    for score in ("softmax", "sigmoid"):
        for renorm in (False, True):
            d = torch.full((n, e), 7.0, device=dev)
            zd, idd, dd = z.to(dev), idx.to(dev), d_w.to(dev)
            nat.check(nat.lib().smoe_select_groups_backward(
                zd.data_ptr(), nat.F32, n, e, k, nat.SCORES[score], int(renorm), 1.0, idd.data_ptr(),
                dd.data_ptr(), d.data_ptr(), nat.stream_of(zd.device)), "backward")
            d = d.cpu()
            assert not bool(torch.isnan(d).any())
            assert not bool(d[2].any()) and not bool(d[1, :10].any())
            for t in (0, 3, 4):  # the formula, slot by slot, on the valid ids
                zt = z[t].double().requires_grad_(True)
                s = torch.softmax(zt, 0) if score == "softmax" else torch.sigmoid(zt)
                ok = (idx[t] >= 0) & (idx[t] < e)
                sel = s[idx[t][ok].long()]
                w = sel / sel.sum() if renorm else sel
                w.backward(d_w[t][ok].double())
                assert torch.allclose(d[t].double(), zt.grad, rtol=1e-5, atol=1e-6), (score, renorm, t)


def test_captured_forward_and_backward():
    """Forward and gradient captured in a graph and replayed on new logits,
    with eager calls of the same operator between the replays."""
    say("graph")
    from spider_moe_amd.forge import _SelectGroups  # noqa: F401
    g = torch.Generator().manual_seed(10)
    z = torch.randn(65, 64, generator=g).to(dev)
    d_w = torch.randn(65, 6, generator=g).to(dev)

    def step(x):
        x = x.detach().requires_grad_(True)
        w, idx = _route(x, 6, groups=8, top_groups=4)
        (d,) = torch.autograd.grad(w, x, d_w)
        return w.detach(), idx, d

    static = z.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for i in range(4):
        new = torch.randn(65, 64, generator=g).to(dev)
        static.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in out]
        want = step(new)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_routes_into_the_dispatch_plan():
    """The routing's outputs go into the dispatch plan as they are: masked
    experts' zero weights are dropped."""
    say("route -> plan")
    from oracle import plan as P
    from spider_moe_amd import build_dispatch_plan
    g = torch.Generator().manual_seed(11)
    z = torch.randn(300, 32, generator=g)
    z[torch.rand(300, 32, generator=g) < 0.9] = -INF
    w, idx = _route(z.to(dev), 4, groups=4, top_groups=2, scale=2.5)
    plan = build_dispatch_plan(idx, w, num_experts=32)
    _, cnt, perm, pw, _ = P.dispatch_plan(idx.cpu().numpy(), w.cpu().numpy(), 32)
    assert plan.counts.cpu().numpy().tolist() == cnt.tolist()
    assert plan.rows.cpu().numpy().tolist() == perm.tolist()
    assert np.array_equal(plan.row_weights.cpu().numpy(), pw)


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("n,e,k", [(597, 16, 1), (40, 255, 7)])
def test_gradient_is_zero_where_the_weights_cannot_matter(score, n, e, k):
    """Renormalised weights add up to the scale: one slot, or slots of equal
    gradients, cannot change the loss, and the gradient is 0, not a rounding."""
    say("zero gradient", score, n, e, k)
    g = torch.Generator().manual_seed(n)
    zg = (torch.randn(n, e, generator=g) * 2).to(dev).requires_grad_(True)
    w, _ = _route(zg, k, score=score, scale=2.5)
    (d,) = torch.autograd.grad(w, zg, torch.randn(n, 1, generator=g).expand(n, k).to(dev))
    assert not bool(d.any())
