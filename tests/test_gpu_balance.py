"""The router's balance loss on the GPU against oracle/mxfp4.py in 64 bits.

Tolerances.  A share p of a token comes from an exponential (2 ulp with its
argument's rounding, |z - max| 2^-24, which for the logits here stays below
2^-19), a sum of at most 10 levels and a product: within 2^-18 of its value.
The loss adds shares over tokens in f32 (at most 256 a lane and 64 partial
sums, 2^-24 each of the sum) and then in 64 bits: within 2^-16 of its value, and
rounded to f32.  A gradient entry p (u - sum p u) dloss has the share's error,
the slope's rounding and the sum's, 2^-18 of p (|u| + sum p |u|) |dloss| each:
2^-16 of that, and half a step of its type.  A share below the smallest normal
number may be 0: 2^-126 of |u| < E <= 256 and dloss <= 1.5."""
import pytest
import torch

from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu

dev = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def say(*a):
    print("[case]", *a, flush=True)


def inputs(s, t, e, k, dtype=torch.float32, seed=0, spread=2.0):
    g = torch.Generator().manual_seed(seed + 7 * s + t + 3 * e + k)
    z = (torch.randn(s, t, e, generator=g) * spread + torch.randn(e, generator=g)).to(dtype)
    idx = torch.topk(z.float() + 0.5 * torch.randn(s, t, e, generator=g), k, dim=-1).indices.to(torch.int32)
    return z.to(dev), idx.to(dev), g


def check(z, idx, *, score, mask=None, per_sequence=True, seed=0):
    from spider_moe_amd import ForgeSelect
    s, t, e = z.shape
    leaf = z.detach().clone().requires_grad_()
    loss, counts = ForgeSelect().balance_loss(leaf, idx, score=score, mask=mask, per_sequence=per_sequence)
    zo = z.detach().double().requires_grad_()
    if per_sequence:
        want, wc, u, p = O.balance(zo, idx, score=score, mask=mask)
    else:
        want, wc, u, p = O.balance(zo.view(1, s * t, e), idx.view(1, s * t, -1), score=score,
                                   mask=None if mask is None else mask.view(1, s * t))
        want, wc = want[0], wc[0]
    assert loss.shape == want.shape and loss.dtype == torch.float32
    assert counts.dtype == torch.int32 and torch.equal(counts.cpu(), wc.cpu())
    assert ((loss.detach().double() - want.detach()).abs() <= (2.0 ** -16 + 2.0 ** -24) * want.detach().abs()).all()
    gen = torch.Generator().manual_seed(seed)
    d = (0.5 + torch.rand(want.shape, generator=gen)).to(dev)
    (got,) = torch.autograd.grad(loss, leaf, d)
    (ref,) = torch.autograd.grad(want, zo, d.double())
    p, u = p.detach().view(-1, *p.shape[-2:]), u.detach().unsqueeze(1)
    bound = p * (u.abs() + (p * u.abs()).sum(-1, keepdim=True)) * d.double().view(-1, 1, 1)
    tol = 2.0 ** -16 * bound.view(z.shape) + HALF[z.dtype] * ref.abs() + {torch.float16: 2.0 ** -25}.get(z.dtype, 2.0 ** -117)
    assert got.dtype == z.dtype and got.shape == z.shape
    assert ((got.double() - ref).abs() <= tol).all(), float(((got.double() - ref).abs() / tol).max())
    with torch.no_grad():  # without a gradient: the same bits
        l2, c2 = ForgeSelect().balance_loss(z, idx, score=score, mask=mask, per_sequence=per_sequence)
    assert torch.equal(l2, loss.detach()) and torch.equal(c2, counts)
    return got


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (1, 1, 8, 2), (3, 5, 7, 3), (2, 127, 16, 2), (1, 128, 17, 4),
                                   (4, 129, 48, 2), (1, 777, 64, 2), (5, 300, 65, 8), (2, 1000, 128, 8),
                                   (3, 257, 129, 5), (2, 700, 256, 8), (1, 4099, 253, 6), (40, 3, 60, 4)])
def test_loss_counts_and_gradient(score, shape):
    say(score, shape)
    z, idx, _ = inputs(*shape)
    check(z, idx, score=score)
    check(z, idx, score=score, per_sequence=False)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(2, 9, 12, 2), (1, 300, 64, 2), (3, 200, 255, 8), (2, 513, 256, 8)])
def test_narrow_logits(score, dtype, shape):
    say(score, dtype, shape)
    z, idx, _ = inputs(*shape, dtype=dtype)
    check(z, idx, score=score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("per_sequence", [True, False])
def test_padding_plays_no_part(score, per_sequence):
    """Masked tokens with NaN, infinities and the lowest value in their
    logits; a sequence of padding alone; ids outside the experts."""
    say("padding", score, per_sequence)
    z, idx, g = inputs(4, 200, 24, 3)
    length = torch.tensor([200, 0, 1, 131])
    mask = (torch.arange(200) < length.unsqueeze(1)).to(dev)
    for i, v in enumerate((float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min)):
        z[:, i::4][~mask[:, i::4]] = v
    idx[~mask] = 5
    idx[0, 3, 0], idx[0, 4, 1], idx[3, 9, 2] = -1, 24, 1 << 30
    idx[0, 7] = 2  # the same expert three times
    got = check(z, idx, score=score, mask=mask, per_sequence=per_sequence)
    assert (got[~mask] == 0).all()
    # another mask type, and a strided one
    from spider_moe_amd import ForgeSelect
    sel = ForgeSelect()
    a = sel.balance_loss(z, idx, score=score, mask=mask, per_sequence=per_sequence)
    wide = torch.zeros(4, 400, dtype=torch.int64, device=dev)
    wide[:, ::2] = mask
    b = sel.balance_loss(z, idx, score=score, mask=wide[:, ::2], per_sequence=per_sequence)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masked_experts_and_far_logits(score):
    """Experts at -inf or the type's lowest value, a token with every expert at
    -inf, logits far below and above 0 (where sigmoids underflow, their shares
    do not)."""
    say("masked experts", score)
    z, idx, _ = inputs(2, 40, 20, 2)
    z[:, :, 3] = -float("inf")
    z[0, :, 4] = torch.finfo(torch.float32).min
    z[1, 5] = -float("inf")
    z[1, 6] -= 300.0
    z[1, 7] += 300.0
    z[1, 8, 10:] -= 150.0
    got = check(z, idx, score=score)
    assert (got[:, :, 3] == 0).all() and (got[1, 5] == 0).all()


def test_nan_and_infinite_logits_stay_with_their_token():
    from spider_moe_amd import ForgeSelect
    say("nan")
    for score in ("softmax", "sigmoid"):
        z, idx, _ = inputs(2, 30, 10, 2)
        z[1, 4, 2] = float("nan")
        leaf = z.clone().requires_grad_()
        loss, counts = ForgeSelect().balance_loss(leaf, idx, score=score, per_sequence=True)
        assert torch.isfinite(loss[0]) and torch.isnan(loss[1]) and int(counts.sum()) == 2 * 30 * 2
        (d,) = torch.autograd.grad(loss.sum(), leaf)
        bad = torch.isnan(d).any(-1)
        assert bad[1, 4] and int(bad.sum()) == 1


def test_even_load_has_no_gradient():
    from spider_moe_amd import ForgeSelect
    say("even")
    z = torch.randn(1, 64, 16, device=dev, requires_grad=True)
    idx = (torch.arange(128, device=dev) % 16).view(1, 64, 2)
    loss, counts = ForgeSelect().balance_loss(z, idx, per_sequence=True)
    (d,) = torch.autograd.grad(loss.sum(), z)
    assert (counts == 8).all() and (d == 0).all() and abs(loss.item() - 1.0) < 2.0 ** -16


def test_empty_batches():
    from spider_moe_amd import ForgeSelect
    say("empty")
    sel = ForgeSelect()
    for shape, per, want in (((0, 8), False, ()), ((3, 0, 8), True, (3,)), ((0, 5, 8), True, (0,))):
        z = torch.randn(*shape, device=dev, requires_grad=True)
        idx = torch.zeros(*shape[:-1], 2, dtype=torch.int32, device=dev)
        loss, counts = sel.balance_loss(z, idx, per_sequence=per)
        assert loss.shape == want and counts.shape == (*want, 8) and (loss == 0).all() and (counts == 0).all()
        (d,) = torch.autograd.grad(loss.sum(), z)
        assert d.shape == z.shape


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_gradient_against_differences(score):
    """(L(z + h v) - L(z - h v)) / 2h along random directions v, |v| <= 1: off by
    h^2 / 6 of the third derivative (at most 8 E max|u|... below 8 E for shares,
    whose derivatives of third order are at most 2 in sum along |v| <= 1) and by
    2 * 2^-16 L / 2h of the loss's error."""
    from spider_moe_amd import ForgeSelect
    say("differences", score)
    z, idx, g = inputs(1, 6, 9, 2)
    leaf = z.clone().requires_grad_()
    loss, _ = ForgeSelect().balance_loss(leaf, idx, score=score)
    (d,) = torch.autograd.grad(loss, leaf)
    h = 2.0 ** -4
    for i in range(6):
        v = (torch.rand(z.shape, generator=g) * 2 - 1).to(dev)
        a = ForgeSelect().balance_loss(z + h * v, idx, score=score)[0].double()
        b = ForgeSelect().balance_loss(z - h * v, idx, score=score)[0].double()
        assert abs(((a - b) / (2 * h) - (d.double() * v.double()).sum()).item()) <= h * h / 6 * 8 * 9 + 2.0 ** -16 * 9 / h


def test_other_layouts():
    """Views, int64 and narrow ids, a leading shape of several dimensions, a
    base that keeps no vector's alignment."""
    from spider_moe_amd import ForgeSelect
    say("layouts")
    sel = ForgeSelect()
    z, idx, _ = inputs(6, 50, 12, 2)
    want = sel.balance_loss(z, idx, per_sequence=True)
    t = sel.balance_loss(z.transpose(0, 1).contiguous().transpose(0, 1), idx.long(), per_sequence=True)
    u = sel.balance_loss(z.view(2, 3, 50, 12), idx.view(2, 3, 50, 2).to(torch.uint8), per_sequence=True)
    off = torch.empty(z.numel() + 1, device=dev)[1:].view_as(z).copy_(z)
    o = sel.balance_loss(off, idx, per_sequence=True)
    assert torch.equal(want[0], t[0]) and torch.equal(want[1], t[1])
    assert u[0].shape == (2, 3) and u[1].shape == (2, 3, 12) and torch.equal(u[0].view(-1), want[0])
    assert torch.equal(o[0], want[0]) and torch.equal(o[1], want[1])


def test_other_stream_and_graph():
    from spider_moe_amd import ForgeSelect
    say("stream and graph")
    sel = ForgeSelect()
    z, idx, _ = inputs(3, 900, 64, 4)
    leaf = z.clone().requires_grad_()
    want = sel.balance_loss(leaf, idx, per_sequence=True)
    (dw,) = torch.autograd.grad(want[0].sum(), leaf)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sel.balance_loss(z, idx, per_sequence=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0].detach()) and torch.equal(got[1], want[1])
    buf = torch.zeros_like(z)
    one = torch.ones(3, device=dev)
    with torch.cuda.stream(side):
        own = buf.detach().requires_grad_()
        torch.autograd.grad(sel.balance_loss(own, idx, per_sequence=True)[0], own, one)
    torch.cuda.current_stream().wait_stream(side)
    del own
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        own = buf.detach().requires_grad_()
        loss, counts = sel.balance_loss(own, idx, per_sequence=True)
        (d,) = torch.autograd.grad(loss, own, one)
    for k in range(3):
        buf.copy_(z if k != 1 else z * 0.5)
        graph.replay()
        ref = z if k != 1 else z * 0.5
        leaf = ref.clone().requires_grad_()
        want = sel.balance_loss(leaf, idx, per_sequence=True)
        (dw,) = torch.autograd.grad(want[0], leaf, one)
        torch.cuda.synchronize()
        assert torch.equal(loss, want[0].detach()) and torch.equal(counts, want[1]) and torch.equal(d, dw)


def test_python_refusals():
    from spider_moe_amd import ForgeSelect
    from torch.autograd import forward_ad
    say("refusals")
    sel = ForgeSelect()
    z, idx, _ = inputs(2, 5, 8, 2)
    for bad in (dict(score="relu"), dict(mask=torch.ones(2, 4, device=dev)), dict(mask=torch.ones(2, 5))):
        with pytest.raises((ValueError, RuntimeError)):
            sel.balance_loss(z, idx, **bad)
    with pytest.raises(ValueError):
        sel.balance_loss(z, idx[:, :4])
    with pytest.raises(ValueError):
        sel.balance_loss(z[0, 0], idx[0, 0], per_sequence=True)
    with pytest.raises(RuntimeError):
        sel.balance_loss(z.double(), idx)
    with pytest.raises(RuntimeError):
        sel.balance_loss(torch.randn(2, 300, device=dev), idx[0, :2])
    leaf = z.clone().requires_grad_()
    loss, _ = sel.balance_loss(leaf, idx)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, leaf, create_graph=True)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError):
            sel.balance_loss(forward_ad.make_dual(z, z), idx)


def test_the_layers_statistic():
    """SpiderMoELayer's aux_loss is the softmax form over the whole batch."""
    from spider_moe_amd import ForgeSelect
    from spider_moe_amd.workloads import make_block
    say("aux_loss")
    wl = make_block("c1", tokens=96, hidden_size=128, num_experts=16, expert_ffn_size=256, experts="bf16")
    with torch.no_grad():
        _, stats = wl.layer(wl.h, wl.x0, 0, return_stats=True)
    r = wl.layer.last_routing()
    loss, counts = ForgeSelect().balance_loss(r["logits"], r["top_idx"])
    assert abs(loss.item() - float(stats["aux_loss"])) <= 2.0 ** -15 * abs(loss.item())
    load = counts.float() / counts.sum()
    assert torch.allclose(load, stats["expert_load"], rtol=2.0 ** -22, atol=0)
