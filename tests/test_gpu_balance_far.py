"""Shares of logits far below a token's largest, by the gradient that they get,
against 64 bits, within what include/smoe.h states: 2^-17 + 2.3 d 2^-24 of a
share d below the largest logit (sigmoid: or of a logit of magnitude d), the
same of the token's others in the gradient's sum, at most 2^-126 where a share
may be 0, and half a step of the gradient's f32."""
import pytest
import torch

from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu

dev = "cuda"


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("shift", [0.0, 30.0, -40.0])
def test_far_shares(score, shift):
    from spider_moe_amd import ForgeSelect
    print("[case] far", score, shift, flush=True)
    t, e = 64, 40
    g = torch.Generator().manual_seed(int(shift) + 50)
    z = (torch.randn(1, t, e, generator=g) - torch.linspace(0, 84, e) + shift).to(dev)
    idx = torch.zeros(1, t, 1, dtype=torch.int32, device=dev)
    idx[:, ::4] = 7
    leaf, ref = z.clone().requires_grad_(), z.double().requires_grad_()
    loss, _ = ForgeSelect().balance_loss(leaf, idx, score=score, per_sequence=True)
    want, _, u, p = O.balance(ref, idx, score=score)
    (got,) = torch.autograd.grad(loss.sum(), leaf)
    (grad,) = torch.autograd.grad(want.sum(), ref)
    p, u = p.detach(), u.detach().unsqueeze(1).abs()
    d = z.double().amax(-1, keepdim=True) - z.double()
    if score == "sigmoid":
        d = torch.maximum(d, z.double().abs())
    rel = 2.0 ** -17 + 2.3 * 2.0 ** -24 * d
    # p (u - sum p u) [times 1 - sigmoid(z), an exponential of its own]
    tol = p * rel * (u + (p * u).sum(-1, keepdim=True)) + p * ((p * u) * rel).sum(-1, keepdim=True)
    if score == "sigmoid":
        rest = torch.sigmoid(-z.double())
        tol = tol * rest + grad.abs() * rel
    tol = tol + 2.0 ** -22 * grad.abs() + 2.0 ** -126 * (u + 1)
    assert ((got.double() - grad).abs() <= tol).all(), float(((got.double() - grad).abs() / tol).max())
    near = (p > 0) & (p * u > 2.0 ** -100)
    assert near.any() and (got[near] != 0).any()
