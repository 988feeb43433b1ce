"""Forward-mode derivatives of grouped routing are refused, not left out."""
import pytest
import torch

from test_gpu_fp8_blocks import dev, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(requires_grad):
    from spider_moe_amd import ForgeSelect
    say("forward mode", requires_grad)
    z = torch.randn(5, 16, device=dev, requires_grad=requires_grad)
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(z, torch.ones_like(z))
        with pytest.raises(RuntimeError, match="forward"):
            ForgeSelect().route_groups(dual, top_k=2)
        w, _ = ForgeSelect().route_groups(z, top_k=2)  # no tangent: as ever
        assert w.requires_grad == requires_grad
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: ForgeSelect().route_groups(a, top_k=2)[0], (z.detach(),), (torch.ones_like(z),))
