"""Kept experts whose tensors get another shape where they lie: the next call
takes them as they are then, or refuses what does not fit together."""
import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"
NAMES = ("w_up", "s_up", "w_down", "s_down", "b_up", "b_down")


def made(kind, bias, e=5, h=160, u=288):
    import spider_moe_amd as s
    g = torch.Generator().manual_seed(e + h)
    r = lambda *shape: (torch.randn(*shape, generator=g) * 0.1).to(dev)
    return getattr(s, kind).quantize(r(e, u, h), r(e, h, u), b_up=r(e, u) if bias else None,
                                     b_down=r(e, h) if bias else None)


def delta(kind, *args):
    import spider_moe_amd as s
    return {"Fp8BlockExperts": s.sparse_expert_delta_fp8_blocks,
            "MxFp4Experts": s.sparse_expert_delta_mxfp4}[kind](*args)


@pytest.mark.parametrize("kind", ["Fp8BlockExperts", "MxFp4Experts"])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("n", [2, 60])
def test_fewer_experts_in_place(kind, bias, n):
    print("[case] fewer experts", kind, bias, n, flush=True)
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, 160, generator=g).bfloat16().to(dev)
    idx = torch.randint(0, 5, (n, 2), generator=g).to(dev)
    idx[0] = torch.tensor([4, 1])
    w = torch.rand(n, 2, generator=g).to(dev) + 0.1
    ex = made(kind, bias)
    all_of = delta(kind, x, idx, w, ex)
    want = delta(kind, x, torch.where(idx < 3, idx, -1), w, ex)
    assert not torch.equal(all_of, want)
    for name in NAMES:
        t = getattr(ex, name)
        if t is not None:
            t.data = t.data[:3]
    assert torch.equal(delta(kind, x, idx, w, ex), want) and ex.num_experts == 3
    ex.w_down.data = ex.w_down.data[:2]  # the others still hold three
    with pytest.raises(ValueError):
        delta(kind, x, idx, w, ex)
