"""Grouped routing and block-scaled fp8 past 32-bit offsets: more than 2^31
logits, codes, outputs, activations.  The last rows (or the last experts) give
what a call on them alone gives, bit for bit: a token's choice and a block's
scale do not depend on the others, and every tile adds the blocks of K in the
same order."""
import pytest
import torch

pytestmark = pytest.mark.gpu

dev = "cuda"


@pytest.fixture(autouse=True)
def room():
    yield
    torch.cuda.empty_cache()


def _codes(g, *shape):
    c = torch.randint(0, 120, shape, dtype=torch.uint8, device=dev, generator=g)  # finite, up to 240
    return (c | torch.randint(0, 2, shape, dtype=torch.uint8, device=dev, generator=g) * 128).view(torch.float8_e4m3fn)


def _gen(seed):
    return torch.Generator(device=dev).manual_seed(seed)


def test_routing_and_quantizer_past_2_31_elements():
    from spider_moe_amd import ForgeSelect, quantize_fp8_blocks
    n, e = (1 << 23) + 300, 256
    print("[case] route", n, e, flush=True)
    z = torch.randn(n, e, dtype=torch.bfloat16, device=dev, generator=_gen(1)).requires_grad_(True)
    select = ForgeSelect()

    def route(z):
        w, idx = select.route_groups(z, top_k=8, num_groups=8, top_groups=4)
        (d,) = torch.autograd.grad(w, z, torch.arange(8, device=dev).float().expand_as(w))
        return w.detach(), idx, d

    all_of, last = route(z), route(z.detach()[-500:].requires_grad_(True))
    for a, b in zip(all_of, last):
        assert torch.equal(a[-500:], b)
    del all_of
    q, s = quantize_fp8_blocks(z, block_rows=1)
    ql, sl = quantize_fp8_blocks(z[-500:], block_rows=1)
    assert torch.equal(q[-500:].view(torch.uint8), ql.view(torch.uint8)) and torch.equal(s[-500:], sl)
    first = n // 128 * 128 - 256
    q, s = quantize_fp8_blocks(z)
    ql, sl = quantize_fp8_blocks(z[first:])
    assert torch.equal(q[first:].view(torch.uint8), ql.view(torch.uint8)) and torch.equal(s[-len(sl):], sl)


def test_linear_past_2_31_codes_and_outputs():
    from spider_moe_amd import ForgeGEMM
    gemm = ForgeGEMM()
    g = _gen(2)
    for n, k, n_out, rows in ((40, 16384, 140032, 1024), (7, 16384, 140032, 1024)):  # weights
        print("[case] linear weights", n, k, n_out, flush=True)
        q, s = _codes(g, n_out, k), torch.rand(n_out // 128, k // 128, device=dev, generator=g) * 1e-4
        x = torch.randn(n, k, device=dev, generator=g).bfloat16()
        y = gemm.linear_fp8_blocks(x, q, s)
        assert torch.equal(y[:, -rows:], gemm.linear_fp8_blocks(x, q[-rows:], s[-rows // 128:]))
    del q, s, x, y
    n, k, n_out = 300100, 144, 8192  # outputs
    print("[case] linear outputs", n, k, n_out, flush=True)
    q, s = _codes(g, n_out, k), torch.rand(n_out // 128, 2, device=dev, generator=g) * 1e-3
    x = torch.randn(n, k, device=dev, generator=g).bfloat16()
    y = gemm.linear_fp8_blocks(x, q, s)
    assert torch.equal(y[-300:], gemm.linear_fp8_blocks(x[-300:], q, s))


def test_experts_past_2_31_codes_and_activations():
    from spider_moe_amd import Fp8BlockExperts, sparse_expert_delta_fp8_blocks
    g = _gen(3)

    def experts(e, h, u):
        return Fp8BlockExperts(_codes(g, e, u, h), torch.rand(e, u // 128, h // 128, device=dev, generator=g) * 1e-4,
                               _codes(g, e, h, u), torch.rand(e, h // 128, u // 128, device=dev, generator=g) * 1e-4)

    print("[case] experts' weights", flush=True)
    ex = experts(256, 4096, 4096)
    last = Fp8BlockExperts(ex.w_up[-2:], ex.s_up[-2:], ex.w_down[-2:], ex.s_down[-2:])
    for n in (4, 100):
        x = torch.randn(n, 4096, device=dev, generator=g).bfloat16()
        idx = torch.randint(0, 2, (n, 2), dtype=torch.int32, device=dev, generator=g)
        w = torch.rand(n, 2, device=dev, generator=g)
        assert torch.equal(sparse_expert_delta_fp8_blocks(x, idx + 254, w, ex),
                           sparse_expert_delta_fp8_blocks(x, idx, w, last))
    del ex, last
    n, h, u = 300000, 1024, 4096  # 2.4e9 activations
    print("[case] experts' activations", n, h, u, flush=True)
    ex = experts(4, h, u)
    x = torch.randn(n, h, device=dev, generator=g).bfloat16()
    idx = torch.rand(n, 4, device=dev, generator=g).topk(2, dim=1).indices.int()
    w = torch.rand(n, 2, device=dev, generator=g)
    got = sparse_expert_delta_fp8_blocks(x, idx, w, ex)
    assert torch.equal(got[-700:], sparse_expert_delta_fp8_blocks(x[-700:], idx[-700:], w[-700:], ex))
