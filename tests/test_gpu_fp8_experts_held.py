"""Fp8BlockExperts kept over changes of the tensors it was made from: biases
of other types, tensors whose memory was exchanged (as Module.to and a loaded
state exchange it), attributes set anew."""
import pytest
import torch

from test_gpu_fp8_blocks import _routing, dev, say

pytestmark = pytest.mark.gpu


def _parts(g, e=4, h=144, u=272):
    from spider_moe_amd import quantize_fp8_blocks
    up, s_up = quantize_fp8_blocks((torch.randn(e, u, h, generator=g) * h ** -0.5).to(dev))
    down, s_down = quantize_fp8_blocks((torch.randn(e, h, u, generator=g) * u ** -0.5).to(dev))
    return dict(w_up=up.contiguous(), s_up=s_up, w_down=down.contiguous(), s_down=s_down,
                b_up=torch.randn(e, u, generator=g).to(dev), b_down=torch.randn(e, h, generator=g).to(dev))


def _make(p):
    from spider_moe_amd import Fp8BlockExperts
    return Fp8BlockExperts(p["w_up"], p["s_up"], p["w_down"], p["s_down"], b_up=p["b_up"], b_down=p["b_down"])


def _inputs(g, n, e=4, h=144):
    idx, w = _routing(g, n, e, 2)
    return torch.randn(n, h, generator=g).bfloat16().to(dev), idx.to(dev), w.to(dev)


@pytest.mark.parametrize("n", [3, 50])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64])
def test_biases_changed_in_place(dtype, n):
    """The next call, and the next replay of a captured one, take the biases
    as they are then, whatever their type."""
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("biases in place", dtype, n)
    g = torch.Generator().manual_seed(n)
    p = _parts(g)
    p["b_up"], p["b_down"] = p["b_up"].to(dtype), p["b_down"].to(dtype)
    ex, x = _make(p), _inputs(g, n)
    before = sparse_expert_delta_fp8_blocks(*x, ex)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = sparse_expert_delta_fp8_blocks(*x, ex)
    for i in range(3):
        p["b_up"].mul_(-1.5)
        p["b_down"].add_(1.0)
        want = sparse_expert_delta_fp8_blocks(*x, _make(p))
        assert not torch.equal(before, want)
        assert torch.equal(sparse_expert_delta_fp8_blocks(*x, ex), want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


@pytest.mark.parametrize("name", ["w_up", "s_up", "w_down", "s_down", "b_up", "b_down"])
def test_exchanged_memory(name):
    """`t.data = other` on a kept tensor (its old memory is kept alive here)."""
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("exchanged memory", name)
    g = torch.Generator().manual_seed(5)
    p, q = _parts(g), _parts(g)
    ex, x = _make(p), _inputs(g, 20)
    sparse_expert_delta_fp8_blocks(*x, ex)
    want = sparse_expert_delta_fp8_blocks(*x, _make({**p, name: q[name]}))
    old = p[name].data
    p[name].data = q[name]
    assert torch.equal(sparse_expert_delta_fp8_blocks(*x, ex), want)
    del old


@pytest.mark.parametrize("name", ["w_up", "s_up", "w_down", "s_down", "b_up", "b_down"])
def test_attributes_set_anew(name):
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("attributes", name)
    g = torch.Generator().manual_seed(6)
    p, q = _parts(g), _parts(g)
    ex, x = _make(p), _inputs(g, 20)
    want = sparse_expert_delta_fp8_blocks(*x, _make({**p, name: q[name]}))
    setattr(ex, name, q[name])
    assert torch.equal(sparse_expert_delta_fp8_blocks(*x, ex), want)


@pytest.mark.parametrize("name", ["w_up", "s_down", "b_up"])
def test_tensors_that_left_are_refused(name):
    """A kept tensor moved to the host, or whose memory was released."""
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("tensors that left", name)
    g = torch.Generator().manual_seed(7)
    p = _parts(g)
    ex, x = _make(p), _inputs(g, 20)
    want = sparse_expert_delta_fp8_blocks(*x, ex)
    there = p[name].data
    p[name].data = there.cpu()
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        sparse_expert_delta_fp8_blocks(*x, ex)
    p[name].data = there
    assert torch.equal(sparse_expert_delta_fp8_blocks(*x, ex), want)
    with pytest.raises(ValueError):
        setattr(ex, name, torch.zeros(3, 5, device=dev))
        sparse_expert_delta_fp8_blocks(*x, ex)
    setattr(ex, name, p[name])
    size = there.untyped_storage().nbytes()
    p[name].untyped_storage().resize_(0)
    with pytest.raises(ValueError, match="released"):
        sparse_expert_delta_fp8_blocks(*x, ex)
    p[name].untyped_storage().resize_(size)


def test_strided_scales_and_biases_follow():
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("strided scales and biases")
    g = torch.Generator().manual_seed(8)
    p = _parts(g)
    x = _inputs(g, 20)
    t = {**p, **{n: p[n].transpose(0, -1).contiguous().transpose(0, -1) for n in ("s_up", "s_down", "b_up", "b_down")}}
    assert not any(t[n].is_contiguous() for n in ("s_up", "s_down", "b_up", "b_down"))
    ex = _make(t)
    assert torch.equal(sparse_expert_delta_fp8_blocks(*x, ex), sparse_expert_delta_fp8_blocks(*x, _make(p)))
    for n in ("s_up", "s_down", "b_up", "b_down"):
        t[n].mul_(2.0)
        p[n].mul_(2.0)
        assert torch.equal(sparse_expert_delta_fp8_blocks(*x, ex), sparse_expert_delta_fp8_blocks(*x, _make(p))), n
