"""The balance loss over millions of tokens against 64 bits.

Tolerance.  A share is within 2^-18 of its value (test_gpu_balance.py).  A lane
adds at most 128 shares in f32 before they go to 64 bits, each addition off by
at most 2^-24 of the sum: 2^-17.  Up to 16 lanes' and waves' sums follow in f32,
2^-20, and one rounding each of a workgroup's sum and of the loss: below 2^-16
of the loss together, whatever the number of tokens."""
import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"


@pytest.fixture(autouse=True)
def room():
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("t,e", [(1 << 22, 155), ((1 << 24) - 3, 133), (1 << 24, 53), (1 << 25, 11)])
def test_even_shares(score, t, e):
    """Logits of 0: every share is 1 / e, every mean of them too, and the loss 1
    wherever the choices went."""
    from spider_moe_amd import ForgeSelect
    print("[case] even shares", score, t, e, flush=True)
    z = torch.zeros(t, e, dtype=torch.bfloat16, device=dev)
    idx = torch.full((t, 1), e - 2, dtype=torch.int32, device=dev)
    loss, counts = ForgeSelect().balance_loss(z, idx, score=score)
    assert counts[e - 2].item() == t and counts.sum().item() == t
    assert abs(loss.double().item() - 1.0) <= 2.0 ** -16


def test_drawn_shares():
    """Two sequences of drawn logits; the oracle's sums in parts."""
    from spider_moe_amd import ForgeSelect
    s, t, e = 2, (1 << 21) + 77, 160
    print("[case] drawn shares", s, t, e, flush=True)
    g = torch.Generator(device=dev).manual_seed(3)
    z = torch.randn(s, t, e, dtype=torch.bfloat16, device=dev, generator=g)
    idx = torch.randint(0, e, (s, t, 2), dtype=torch.int32, device=dev, generator=g)
    mask = torch.rand(s, t, device=dev, generator=g) < 0.9
    loss, counts = ForgeSelect().balance_loss(z, idx, mask=mask, per_sequence=True)
    for i in range(s):
        p = torch.zeros(e, dtype=torch.float64, device=dev)
        for a in range(0, t, 1 << 18):
            part = torch.softmax(z[i, a:a + (1 << 18)].double(), -1)
            p += part[mask[i, a:a + (1 << 18)]].sum(0)
        want = torch.bincount(idx[i][mask[i]].view(-1), minlength=e)
        assert torch.equal(counts[i].long(), want)
        ref = (e * (want.double() / want.sum() * p).sum() / mask[i].sum()).item()
        assert abs(loss[i].double().item() - ref) <= 2.0 ** -16 * ref
