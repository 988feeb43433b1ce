"""Inputs of the expert step on block-scaled fp8 weights in the forms that
programs hand on: ids of every integer type."""
import pytest
import torch

from test_gpu_fp8_blocks import _experts, dev, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.uint8, torch.int8, torch.int16, torch.int64])
@pytest.mark.parametrize("n,e,k", [(2, 6, 2), (40, 130, 3), (40, 256, 3)])
def test_ids_of_every_integer_type(dtype, n, e, k):
    """The result with int32 ids, bit for bit; as many experts as uint8 has
    values, and more than int8 has."""
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("ids", dtype, n, e, k)
    g = torch.Generator().manual_seed(n + e)
    ex = _experts(g, e, 64, 32, "gelu", True)
    msg = torch.randn(n, 64, generator=g).bfloat16().to(dev)
    idx = torch.randint(0, min(e, torch.iinfo(dtype).max + 1), (n, k), generator=g)
    w = torch.rand(n, k, generator=g).to(dev) + 0.1
    want = sparse_expert_delta_fp8_blocks(msg, idx.to(torch.int32).to(dev), w, ex)
    assert bool(want.any())
    assert torch.equal(sparse_expert_delta_fp8_blocks(msg, idx.to(dtype).to(dev), w, ex), want)
