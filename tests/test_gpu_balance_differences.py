"""The balance loss's gradient against differences that a wrong gradient, or one
of 0, cannot pass: entry by entry against 64-bit differences of the definition,
and along one expert's logits against differences of the kernel's own losses."""
import pytest
import torch

from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu

dev = "cuda"


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_every_entry_against_64_bit_differences(score):
    """(L(z + h) - L(z - h)) / 2h in one entry, h = 2^-16: off by h^2 / 6 of the
    third derivative, at most E / 8 (a share is a scaled logistic function of one
    logit), 2^-35 of E = 9, and by 2^-52 L / h = 2^-33 of the values; the kernel's
    shares as in test_gpu_balance.py."""
    from spider_moe_amd import ForgeSelect
    print("[case] 64-bit differences", score, flush=True)
    t, e = 6, 9
    g = torch.Generator().manual_seed(4)
    z = torch.randn(1, t, e, generator=g).to(dev)
    idx = torch.tensor([0, 1, 0, 2, 0, 0, 1, 0, 3, 0, 0, 4], dtype=torch.int32, device=dev).view(1, t, 2)
    mask = torch.tensor([[1, 1, 0, 1, 1, 1]], dtype=torch.bool, device=dev)
    leaf = z.clone().requires_grad_()
    loss, _ = ForgeSelect().balance_loss(leaf, idx, score=score, mask=mask)
    (got,) = torch.autograd.grad(loss, leaf)
    h, m = 2.0 ** -16, t * e
    step = h * torch.eye(m, dtype=torch.float64, device=dev).view(m, t, e)
    every = [O.balance(z.double() + sign * step, idx.expand(m, t, 2), score=score, mask=mask.expand(m, t))[0]
             for sign in (1, -1)]
    want = ((every[0] - every[1]) / (2 * h)).view(t, e)
    _, _, u, p = O.balance(z, idx, score=score, mask=mask)
    p, u = p[0], u[0].abs()
    tol = 2.0 ** -16 * p * (u + (p * u).sum(-1, keepdim=True)) + 2.0 ** -24 * want.abs() + 2.0 ** -30
    assert ((got[0].double() - want).abs() <= tol).all()
    assert (want[mask[0]].abs() > 100 * tol[mask[0]]).double().mean() > 0.9  # a gradient of 0 would fail
    assert (got[0, 2] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("s,t,e", [(1, 40, 9), (3, 200, 33), (2, 700, 200)])
def test_one_experts_logits_against_differences(score, dtype, s, t, e):
    """Every choice on expert 3, whose logits all move by h = 2^-6 (kept by every
    type: they are multiples of 2^-6 up to 2): off by h^2 / 6 * E / 8 and by
    (2^-16 + 2^-24) of each of the two losses over 2h.  The derivative is about 1
    (softmax) or 1/2, so that a wrong one fails."""
    from spider_moe_amd import ForgeSelect
    print("[case] differences", score, dtype, s, t, e, flush=True)
    sel = ForgeSelect()
    g = torch.Generator().manual_seed(s + t + e)
    z = (torch.randint(-64, 65, (s, t, e), generator=g) / 64.0).to(dtype).to(dev)
    idx = torch.full((s, t, 2), 3, dtype=torch.int32, device=dev)
    leaf = z.clone().requires_grad_()
    loss, _ = sel.balance_loss(leaf, idx, score=score, per_sequence=True)
    (d,) = torch.autograd.grad(loss.sum(), leaf)
    h = 2.0 ** -6
    step = torch.zeros_like(z)
    step[..., 3] = h
    a = sel.balance_loss(z + step, idx, score=score, per_sequence=True)[0].double()
    b = sel.balance_loss(z - step, idx, score=score, per_sequence=True)[0].double()
    half = torch.finfo(dtype).eps / 2
    along = d.double()[..., 3].sum(-1)
    tol = h * h / 6 * e / 8 + (2.0 ** -16 + 2.0 ** -24) * (a + b) / (2 * h) + (half + 2.0 ** -16) * along.abs() + 2.0 ** -25 * t
    assert ((a - b) / (2 * h) - along).abs().le(tol).all()
    assert (along > 0.25).all() and (tol < 0.1 * along).all()
