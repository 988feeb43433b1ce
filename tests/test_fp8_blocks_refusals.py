"""CPU checks of group-limited routing and block-scaled fp8: what the entry
points refuse before any launch, the CPU form of the quantizer, and the pins
of oracle/fp8_blocks.py (known answers, autograd, the framework's other
formats)."""
import ctypes

import pytest
import torch

from oracle import fp8_blocks as O

FAKE = 0x1000  # never dereferenced: every call below is refused, or has no rows


@pytest.fixture(scope="module")
def lib():
    from spider_moe_amd import _native
    return _native.lib()


def test_select_groups_refusals(lib):
    from spider_moe_amd import _native as nat

    def go(dt=nat.F32, n=4, e=16, k=2, score=1, groups=4, top=2, z=FAKE, w=FAKE, i=FAKE):
        return lib.smoe_select_groups(z, dt, n, e, k, score, None, groups, top, 1, 1.0, w, i, None)

    assert go(dt=nat.FP8_E4M3) == -2
    for bad in (dict(n=-1), dict(e=0), dict(e=257), dict(k=0), dict(k=17), dict(e=256, k=65), dict(score=2),
                dict(groups=0), dict(groups=3), dict(groups=32), dict(top=0), dict(top=5), dict(groups=8, top=1, k=3),
                dict(z=None), dict(w=None), dict(i=None)):
        assert go(**bad) == 1, bad
    assert go(n=0, z=None, w=None, i=None) == 0
    assert go(n=1 << 26) == 1

    def back(dt=nat.F32, n=4, e=16, k=2, score=0, z=FAKE, i=FAKE, g=FAKE, d=FAKE):
        return lib.smoe_select_groups_backward(z, dt, n, e, k, score, 1, 1.0, i, g, d, None)

    assert back(dt=7) == -2
    for bad in (dict(n=-1), dict(e=300), dict(k=0), dict(k=17), dict(score=-1), dict(z=None), dict(i=None),
                dict(g=None), dict(d=None)):
        assert back(**bad) == 1, bad
    assert back(n=0) == 0


def test_quantizer_refusals(lib):
    from spider_moe_amd import _native as nat

    def go(dt=nat.BF16, g=1, r=4, c=100, ldx=100, br=1, q=FAKE, ld=112, s=FAKE, x=FAKE):
        return lib.smoe_quantize_fp8_blocks(x, dt, g, r, c, ldx, br, q, ld, s, None)

    assert go(dt=nat.INT4) == -2
    for bad in (dict(g=-1), dict(r=-1), dict(c=0), dict(ldx=99), dict(br=64), dict(ld=100), dict(ld=96), dict(ld=144),
                dict(q=FAKE + 8), dict(q=None), dict(s=None), dict(x=None)):
        assert go(**bad) == 1, bad
    assert go(r=0) == 0 and go(g=0) == 0
    assert go(g=1 << 15, r=1 << 13, c=129, ldx=129, ld=144) == 1  # 2^28 rows of two blocks
    assert go(g=1 << 24, r=129, br=128) == 1


def test_linear_refusals(lib):
    from spider_moe_amd import _native as nat

    def go(x=FAKE, dt=nat.BF16, ldx=100, xs=None, n=40, k=100, w=FAKE, ldw=112, ws=FAKE, no=30, act=0, out=FAKE,
           od=nat.BF16, wk=FAKE, wb=1 << 20):
        return lib.smoe_linear_fp8_blocks(x, dt, ldx, xs, n, k, w, ldw, ws, None, no, act, out, od, wk, wb, None)

    assert go(dt=nat.INT4) == -2 and go(od=nat.F16) == -2
    for bad in (dict(n=-1), dict(k=0), dict(no=0), dict(ldx=99), dict(ldw=99), dict(ldw=104), dict(act=2), dict(x=None),
                dict(w=None), dict(ws=None), dict(out=None), dict(wk=None), dict(xs=FAKE), dict(w=FAKE + 4),
                dict(wk=FAKE + 1), dict(dt=nat.FP8_E4M3, ldx=112), dict(dt=nat.FP8_E4M3, ldx=100, xs=FAKE),
                dict(dt=nat.FP8_E4M3, ldx=112, xs=FAKE, x=FAKE + 2)):
        assert go(**bad) == 1, bad
    need = lib.smoe_linear_fp8_blocks_workspace_bytes(40, 100)
    assert need >= 40 * 112 + 40 * 4 and go(wb=need - 1) == 3
    assert go(n=0) == 0
    # a few rows are quantized by the product itself
    assert lib.smoe_linear_fp8_blocks_workspace_bytes(4, 100) == 0
    assert lib.smoe_linear_fp8_blocks_workspace_bytes(0, 100) == 0


def test_expert_refusals(lib):
    from spider_moe_amd import _native as nat

    def desc(**kw):
        d = nat.SmoeExpertsFp8Blocks()
        d.act, d.E, d.H, d.U = nat.ACT_GELU, 4, 64, 96
        d.w_up = d.w_down = d.s_up = d.s_down = FAKE
        for a, b in kw.items():
            setattr(d, a, b)
        return d

    def go(d, msg=FAKE, dt=nat.BF16, idx=FAKE, w=FAKE, n=4, k=2, out=FAKE, od=nat.BF16, ws=FAKE, wb=1 << 30):
        return lib.smoe_expert_delta_fp8_blocks(ctypes.byref(d), msg, dt, idx, w, n, k, out, od, ws, wb, None)

    size = lib.smoe_expert_delta_fp8_blocks_workspace_bytes
    for bad in (dict(act=2), dict(E=0), dict(E=257), dict(H=0), dict(H=72), dict(U=100), dict(w_up=None),
                dict(w_down=None), dict(s_up=None), dict(s_down=None), dict(w_up=FAKE + 8), dict(w_down=FAKE + 1)):
        assert go(desc(**bad)) == 1, bad
        assert size(ctypes.byref(desc(**bad)), 4, 2) == 0
    ok = desc()
    for bad in (dict(n=-1), dict(k=0), dict(k=65), dict(n=1 << 30), dict(msg=None), dict(idx=None), dict(w=None),
                dict(out=None), dict(ws=None), dict(ws=FAKE + 8)):
        assert go(ok, **bad) == 1, bad
    assert go(ok, dt=nat.F16) == -2 and go(ok, od=nat.FP8_E4M3) == -2
    assert go(desc(H=8192), n=70000) == 1 and go(ok, n=65535 * 64 + 1) == 1
    assert size(ctypes.byref(ok), 65535 * 64 + 1, 2) == 0
    need = size(ctypes.byref(ok), 4, 2)
    assert need > 0 and go(ok, wb=need - 1) == 3
    assert go(ok, n=0) == 0
    assert lib.smoe_expert_delta_fp8_blocks(None, FAKE, 1, FAKE, FAKE, 4, 2, FAKE, 1, FAKE, 1, None) == 1


def test_python_refusals():
    """No CPU fallback, and shape errors that name the argument."""
    from spider_moe_amd import ForgeGEMM, ForgeSelect, Fp8BlockExperts, quantize_fp8_blocks
    z = torch.zeros(2, 8)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ForgeSelect().route_groups(z, top_k=2)
    q, s = quantize_fp8_blocks(torch.zeros(32, 64))
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ForgeGEMM().linear_fp8_blocks(torch.zeros(3, 64), q, s)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        Fp8BlockExperts.quantize(torch.zeros(2, 32, 64), torch.zeros(2, 64, 32))
    with pytest.raises(ValueError, match="block_rows"):
        quantize_fp8_blocks(torch.zeros(4, 4), block_rows=64)
    with pytest.raises(ValueError, match="rows, cols"):
        quantize_fp8_blocks(torch.zeros(4))


@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_cpu_quantizer_and_oracle(block_rows, dtype):
    """The product's CPU form and the oracle agree (different code: torch's
    cast against rounding by hand); a value is within half a code's step."""
    from spider_moe_amd import dequantize_fp8_blocks, quantize_fp8_blocks
    g = torch.Generator().manual_seed(1)
    for rows, cols in ((1, 1), (3, 127), (130, 300), (256, 128)):
        x = (torch.randn(rows, cols, generator=g) * 3).to(dtype)
        q, s = quantize_fp8_blocks(x, block_rows=block_rows)
        oq, os_ = O.quantize(x, block_rows)
        assert torch.equal(q.double(), oq) and torch.equal(s.double(), os_)
        v = dequantize_fp8_blocks(q, s, block_rows=block_rows)
        full = O.values(torch.ones(rows, cols), s, block_rows)
        assert bool(((v.double() - x.double()).abs() <= 2.0 ** -4 * x.double().abs() * (1 + 1e-6) + 2.0 ** -10 * full).all())


def test_quantizer_known_answer():
    """amax 896 -> scale 2: 3 -> 1.5 (code 0x3c), 17 -> 8.5 -> 8 (ties to even),
    19 -> 9.5 -> 10; the second block has its own scale."""
    from spider_moe_amd import quantize_fp8_blocks
    x = torch.zeros(1, 130)
    x[0, :4] = torch.tensor([896.0, 3.0, 17.0, -19.0])
    x[0, 128:] = torch.tensor([448.0, 1.0])
    q, s = quantize_fp8_blocks(x, block_rows=1)
    assert s.tolist() == [[2.0, 1.0]]
    assert q[0, :4].float().tolist() == [448.0, 1.5, 8.0, -10.0]
    assert q[0, 128:].float().tolist() == [448.0, 1.0]
    assert q.view(-1)[1:2].contiguous().view(torch.uint8).item() == 0x3c


def test_oracle_select_known_answer():
    """8 experts in 4 groups.  Scores after sigmoid: group values decide first
    (group 1 holds the single best expert, but groups 0 and 3 are the better
    pairs); the bias moves the choice, not the weights."""
    p = torch.tensor([[0.6, 0.5, 0.9, 0.05, 0.1, 0.2, 0.7, 0.45]], dtype=torch.float64)
    z = torch.log(p / (1 - p))
    w, i = O.select_groups(z, 3, score="sigmoid", groups=4, top_groups=2, renorm=False)
    assert i.tolist() == [[6, 0, 1]]
    assert torch.allclose(w, torch.tensor([[0.7, 0.6, 0.5]], dtype=torch.float64))
    b = torch.zeros(8)
    b[3] = 0.5
    w, i = O.select_groups(z, 3, score="sigmoid", bias=b, groups=4, top_groups=2, renorm=True, scale=2.0)
    assert i.tolist() == [[2, 6, 3]]
    assert torch.allclose(w, 2 * torch.tensor([[0.9, 0.7, 0.05]], dtype=torch.float64) / 1.65)
    z[0, :7] = -float("inf")
    w, i = O.select_groups(z, 3, score="softmax", groups=4, top_groups=2)
    assert i.tolist() == [[7, 0, 1]] and w.tolist() == [[1.0, 0.0, 0.0]]


def test_oracle_experts_against_the_frameworks_float_experts():
    """With scales of 1 and small integers nothing is rounded: the block
    oracle is the plain expert FFN (relu-free check through GELU on values
    whose activations quantize within the 2^-4 of a code)."""
    g = torch.Generator().manual_seed(2)
    e, h, u, n, k = 3, 32, 48, 6, 2
    w_up = torch.randint(-3, 4, (e, u, h), generator=g).float() / 16
    w_dn = torch.randint(-3, 4, (e, h, u), generator=g).float() / 16
    one = torch.ones(e, 1, 1)
    x = torch.randint(-4, 5, (n, h), generator=g).float()
    x[:, 0] = 7.0
    idx = torch.tensor([[0, 1], [2, 2], [1, 5], [0, 2], [1, 0], [2, 1]])
    w = torch.rand(n, k, generator=g) + 0.1
    got, tol = O.expert_delta(x, idx, w, w_up, one, w_dn, one)
    want = torch.zeros(n, h, dtype=torch.float64)
    for t in range(n):
        for j in range(k):
            i = int(idx[t, j])
            if 0 <= i < e:
                a = O.gelu(w_up[i].double() @ x[t].double())
                want[t] += w[t, j].double() * (w_dn[i].double() @ a)
    assert float((got - want).norm() / want.norm()) < 2.0 ** -4
    assert bool((tol < 0.2 * want.pow(2).mean().sqrt()).all())


def test_oracle_code_distance():
    """An activation in the middle between two codes may take either; one a
    quarter of a step away may not."""
    a = torch.full((1, 128), 448.0, dtype=torch.float64)
    a[0, 1], a[0, 2] = 17.0, 16.5
    v, d = O._act_codes(a, torch.full_like(a, 1e-3))
    assert v[0, :3].tolist() == [448.0, 16.0, 16.0]
    assert abs(float(d[0, 1]) - 2.0) < 1e-3 and float(d[0, 2]) < 1e-3


def test_route_gradient_oracle_against_differences():
    g = torch.Generator().manual_seed(3)
    z = torch.randn(4, 12, generator=g, dtype=torch.float64)
    idx = torch.topk(z, 3).indices
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            f = lambda a: O.select_groups_weights(a, idx, score=score, renorm=renorm, scale=1.3)  # noqa: E731
            assert torch.autograd.gradcheck(f, (z.clone().requires_grad_(True),))
