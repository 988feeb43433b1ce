"""Where the choices are spread evenly the balance loss has no gradient, exactly,
at every number of experts (E (1 / E) is not 1 in 64 bits for 49, 98, 103, ..)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_even_choices_at_every_number_of_experts(score):
    from spider_moe_amd import ForgeSelect
    sel = ForgeSelect()
    g = torch.Generator(device=dev).manual_seed(1)
    for e in range(1, 257):
        print("[case] even", score, e, flush=True)
        for t in (e, 3 * e):  # one token an expert, three; 3 * 256 tokens take several workgroups
            z = torch.randn(2, t, e, device=dev, generator=g).requires_grad_()
            idx = (torch.arange(t, device=dev) % e).view(1, t, 1).expand(2, t, 1)
            loss, counts = sel.balance_loss(z, idx, score=score, per_sequence=True)
            (d,) = torch.autograd.grad(loss.sum(), z)
            assert (counts == t // e).all()
            assert (d == 0).all(), e
