"""Microscaled 4-bit floats on the GPU: the quantizer bit for bit against the
CPU formula, the linear product and the expert FFN against oracle/mxfp4.py in
64 bits.

The oracle returns each output's error bound beside it: the f32 sums'
(oracle.mxfp4.sum_error), and in the expert FFN what hidden activations whose
f32 error reaches a border between two codes, or takes their block's largest
over a power of two, can move.  The output's own rounding, 2^-8 of a bf16 and
2^-24 of an f32, comes on top."""
import pytest
import torch

from oracle import mxfp4 as O

pytestmark = pytest.mark.gpu

dev = "cuda"
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def say(*a):
    print("[case]", *a, flush=True)


def assert_within(got, want, err):
    tol = err + HALF[got.dtype] * (want.abs() + err) + 2.0 ** -120
    off = (got.double() - want).abs()
    assert got.shape == want.shape
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    ok = (off <= tol) | torch.isnan(want)
    assert ok.all(), (float((off / tol).nan_to_num().max()), int((~ok).sum()))


# ---------------------------------------------------------------- quantizer ----
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1,), (1, 1), (1, 32), (3, 31), (5, 33), (17, 16), (127, 200), (128, 256), (2, 1, 7),
                                   (130, 1000), (2, 3, 70, 136), (4, 1, 40), (300, 1408), (1, 4099), (513, 96)])
def test_quantizer_is_the_cpu_formula(dtype, shape):
    from spider_moe_amd import dequantize_mxfp4, quantize_mxfp4
    say("quantize", dtype, shape)
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(*shape, generator=g) * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=g))).to(dtype)
    q, s = quantize_mxfp4(x.to(dev))
    cq, cs = quantize_mxfp4(x)
    assert torch.equal(q.cpu(), cq) and torch.equal(s.cpu(), cs)
    for out in (torch.float32, torch.bfloat16, torch.float16, torch.float64):
        a = dequantize_mxfp4(q, s, cols=shape[-1], dtype=out)
        b = dequantize_mxfp4(cq, cs, cols=shape[-1], dtype=out)
        assert a.dtype == out and torch.equal(a.cpu(), b)


def test_every_exponent_tie_and_special_value():
    """Blocks of every exponent that f32 has, with the seven ties, the values
    between them and both neighbours of each; zeros of both signs; subnormal,
    infinite and NaN entries."""
    from spider_moe_amd import dequantize_mxfp4, quantize_mxfp4
    say("exponents")
    base = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, 7.9, 0.1, 4.0], dtype=torch.float64)
    rows = []
    for e in range(-149, 126):
        v = (base * 2.0 ** e).clamp_max(3.4e38).float()
        near = torch.cat([v, torch.nextafter(v, torch.tensor(0.0)), torch.nextafter(v, torch.tensor(3.4e38))])[:31]
        rows.append(torch.cat([near * torch.where(torch.arange(31) % 3 == 0, -1.0, 1.0), torch.tensor([-0.0])]))
    x = torch.stack(rows)
    bad = torch.randn(6, 32)
    bad[0, 5], bad[1, 31], bad[2, 0], bad[3, 7] = float("inf"), -float("inf"), float("nan"), 1e-45
    bad[4], bad[5] = 0.0, -0.0
    x = torch.cat([x, bad])
    q, s = quantize_mxfp4(x.to(dev))
    cq, cs = quantize_mxfp4(x)
    assert torch.equal(s.cpu(), cs) and torch.equal(q.cpu(), cq)
    a, b = dequantize_mxfp4(q, s).cpu(), dequantize_mxfp4(cq, cs)
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a.nan_to_num(), b.nan_to_num())
    fin = torch.isfinite(x).all(-1)
    assert torch.equal(a[fin].double(), O.quantize(x[fin])[0])


def test_strides_of_the_quantizer():
    from spider_moe_amd import dequantize_mxfp4, quantize_mxfp4
    say("strides")
    big = torch.randn(40, 300, device=dev)
    for x in (big[:, :100], big[:, 3:103], big[::2, :96], big.t(), big[:, ::2], big.view(4, 10, 300)[:, ::2, 7:77],
              big.bfloat16()[:, 1:130], big[5, :50], big[:, :1].t(), big.view(2, 20, 300).transpose(0, 1)):
        q, s = quantize_mxfp4(x)
        cq, cs = quantize_mxfp4(x.cpu().contiguous())
        assert torch.equal(q.cpu(), cq) and torch.equal(s.cpu(), cs)
    x = torch.randn(12, 6, 70, device=dev)  # codes and scales read at other pitches and alignments
    q, s = quantize_mxfp4(x)
    want = dequantize_mxfp4(q, s, cols=70)
    tight = torch.empty(q.numel() + 1, dtype=torch.uint8, device=dev)[1:].view(q.shape).copy_(q)
    assert torch.equal(dequantize_mxfp4(tight, s.contiguous(), cols=70), want)
    assert torch.equal(dequantize_mxfp4(q.transpose(0, 1), s.transpose(0, 1), cols=70), want.transpose(0, 1))
    for shape in ((0, 64), (3, 0, 64)):
        q, s = quantize_mxfp4(torch.zeros(shape, device=dev))
        assert dequantize_mxfp4(q, s).shape == shape


# ------------------------------------------------------------------- linear ----
def weight(n_out, k, seed=0, std=0.05):
    from spider_moe_amd import quantize_mxfp4
    g = torch.Generator().manual_seed(seed + n_out + k)
    return quantize_mxfp4((torch.randn(n_out, k, generator=g) * std).to(dev))


def check_linear(x, codes, scale, bias=None, act=None):
    from spider_moe_amd import ForgeGEMM
    got = ForgeGEMM().linear_mxfp4(x, codes, scale, bias, act=act)
    want, err = O.linear(x.reshape(-1, x.shape[-1]), codes, scale, bias, act)
    assert got.dtype == x.dtype
    assert_within(got.reshape(want.shape), want, err)
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("shape", [
    (1, 1, 1), (1, 32, 16), (1, 2048, 1408), (2, 31, 33), (5, 1000, 70), (16, 257, 48), (16, 1024, 64),   # quantized inside
    (9, 2816, 40), (17, 96, 100), (24, 2048, 130),                                                   # a few rows of codes
    (25, 64, 60), (33, 300, 65), (40, 1000, 2800), (64, 256, 512),                                    # 32 x 64 tiles
    (200, 1000, 2800), (257, 288, 1300), (1000, 544, 2000), (515, 96, 5632),                          # 64 x 64
    (2000, 96, 5000), (4000, 352, 2500),                                                              # 128 x 128
    (2100, 352, 5632), (4096, 64, 2816)])                                                             # 256 x 256
def test_linear(dtype, shape):
    n, k, n_out = shape
    say("linear", dtype, shape)
    g = torch.Generator().manual_seed(n + k)
    x = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(dtype).to(dev)
    codes, scale = weight(n_out, k)
    bias = torch.randn(n_out, generator=g).to(dev) * 0.1
    check_linear(x, codes, scale)
    check_linear(x, codes, scale, bias, "gelu")


@pytest.mark.parametrize("k", [1, 16, 32, 33, 64, 95, 96, 97, 128, 160, 224, 256, 257, 288, 352, 480, 511, 512, 513, 608, 800])
@pytest.mark.parametrize("n", [3, 20, 50, 300])
def test_linear_at_every_end_of_k(n, k):
    say("k", n, k)
    g = torch.Generator().manual_seed(k)
    x = torch.randn(n, k, generator=g).bfloat16().to(dev)
    codes, scale = weight(77, k)
    check_linear(x, codes, scale)


@pytest.mark.parametrize("n", [1, 20, 40, 300, 2500])
def test_what_lies_behind_a_row_plays_no_part(n):
    """Weight rows in wider storage whose bytes past K, codes and scales, are
    anything: other codes, NaN scales."""
    from spider_moe_amd import ForgeGEMM
    say("behind", n)
    g = torch.Generator().manual_seed(n)
    for k in (33, 100, 130, 290, 420):
        codes, scale = weight(600, k)
        nb = -(-k // 32)
        wc = torch.full((600, 16 * nb + 48), 0xFF, dtype=torch.uint8, device=dev)
        wsc = torch.full((600, -(-nb // 4) * 4 + 8), 0xFF, dtype=torch.uint8, device=dev)
        wc[:, :codes.shape[1]] = codes
        if k % 2:  # the half of the last byte
            wc[:, codes.shape[1] - 1] |= 0xF0
        wsc[:, :nb] = scale
        x = torch.randn(n, k, generator=g).bfloat16().to(dev)
        a = check_linear(x, codes, scale)
        b = ForgeGEMM().linear_mxfp4(x, wc[:, :codes.shape[1]], wsc[:, :nb])
        assert torch.equal(a, b)
        tight = torch.empty(codes.numel() + 3, dtype=torch.uint8, device=dev)[3:].view(codes.shape).copy_(codes)
        c = ForgeGEMM().linear_mxfp4(x, tight, scale.contiguous())
        assert torch.equal(a, c)


@pytest.mark.parametrize("n", [2, 20, 70, 400])
def test_nan_and_infinity_stay_in_their_row_and_channel(n):
    say("nan", n)
    x = torch.randn(n, 200, device=dev)
    codes, scale = weight(50, 200)
    x[1, 7] = float("nan")
    scale = scale.clone()
    scale[9, 3] = 255
    got = check_linear(x, codes, scale)
    nan = torch.isnan(got)
    assert nan[1].all() and nan[:, 9].all() and int(nan.sum()) == 50 + n - 1
    x[1, 7] = -float("inf")
    assert torch.equal(torch.isnan(check_linear(x, codes, scale)), nan)


def test_extreme_magnitudes():
    """Rows near both ends of f32 beside ordinary ones, weights of 2^-127."""
    say("magnitudes")
    for n in (4, 40, 300):
        x = torch.randn(n, 96, device=dev)
        x[0] *= 2.0 ** 100
        x[1] *= 2.0 ** -100
        x[2] *= 0
        codes, scale = weight(40, 96)
        scale = scale.clone()
        scale[3] = 0
        check_linear(x, codes, scale)


def test_leading_shapes_views_and_empty():
    from spider_moe_amd import ForgeGEMM
    say("views")
    gemm = ForgeGEMM()
    codes, scale = weight(64, 96)
    x = torch.randn(6, 7, 96, device=dev).bfloat16()
    want = check_linear(x.view(42, 96), codes, scale)
    assert torch.equal(gemm.linear_mxfp4(x, codes, scale), want.view(6, 7, 64))
    wide = torch.randn(42, 130, device=dev).bfloat16()
    wide[:, 5:101] = x.view(42, 96)
    assert torch.equal(gemm.linear_mxfp4(wide[:, 5:101], codes, scale), want)
    assert torch.equal(gemm.linear_mxfp4(x.view(42, 96)[::2], codes, scale), want[::2])
    assert gemm.linear_mxfp4(x[0, 0], codes, scale).shape == (64,)
    assert gemm.linear_mxfp4(x[:0], codes, scale).shape == (0, 7, 64)
    # an output base and width that keep no 16-byte chunks
    codes, scale = weight(37, 96)
    for n in (30, 300, 1500):
        check_linear(torch.randn(n, 96, device=dev).bfloat16(), codes, scale)
    for bad in (dict(act="relu"), dict(bias=torch.zeros(5, device=dev))):
        with pytest.raises(ValueError):
            gemm.linear_mxfp4(x, *weight(64, 96), **bad)
    with pytest.raises(ValueError):
        gemm.linear_mxfp4(x[..., :90], *weight(64, 96))
    with pytest.raises(RuntimeError):
        gemm.linear_mxfp4(x.double(), *weight(64, 96))


# ------------------------------------------------------------------ experts ----
def experts_of(e, h, u, act, bias, seed=0):
    from spider_moe_amd import MxFp4Experts
    g = torch.Generator().manual_seed(seed + e + h + u)
    halves = 2 if act == "swiglu" else 1
    w_up = (torch.randn(e, halves * u, h, generator=g) * 0.06).to(dev)
    w_down = (torch.randn(e, h, u, generator=g) * 0.06).to(dev)
    b_up = (torch.randn(e, u, generator=g) * 0.1).to(dev) if bias else None
    b_down = (torch.randn(e, h, generator=g) * 0.1).to(dev) if bias else None
    return MxFp4Experts.quantize(w_up, w_down, b_up=b_up, b_down=b_down, activation=act)


def routing(n, e, k, seed=0, skew=0.5):
    g = torch.Generator().manual_seed(seed + n + e + k)
    z = torch.randn(n, e, generator=g) + skew * torch.randn(e, generator=g)
    z, idx = torch.topk(z, k, dim=-1)
    return idx.to(torch.int32).to(dev), torch.softmax(z, -1).to(dev)


def check_experts(x, idx, w, ex):
    from spider_moe_amd import sparse_expert_delta_mxfp4
    got = sparse_expert_delta_mxfp4(x, idx, w, ex)
    want, err = O.expert_delta(x, idx, w, ex.w_up, ex.s_up, ex.w_down, ex.s_down, ex.b_up, ex.b_down, ex.activation)
    assert got.dtype == x.dtype and got.shape == x.shape
    assert_within(got, want, err)
    # the bound is no licence: where it allows more than ten roundings it is rarely used
    free = (got.double() - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -8 * want.abs().mean()
    assert free.double().mean() >= 0.99
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("act,bias", [("gelu", True), ("swiglu", False), ("swiglu", True), ("gelu", False)])
@pytest.mark.parametrize("n,e,k,h,u", [
    (1, 8, 2, 256, 512), (1, 64, 2, 2048, 1408), (4, 4, 4, 96, 32), (16, 3, 1, 544, 224), (5, 6, 3, 32, 1184),  # a few entries
    (9, 5, 2, 64, 96), (64, 16, 2, 256, 288), (150, 12, 3, 544, 1184),                                     # 32 rows an expert
    (600, 8, 2, 256, 512), (1024, 32, 4, 160, 160),                                                        # 64 to 128
    (4000, 6, 3, 96, 320), (2000, 2, 1, 64, 64)])
def test_experts(dtype, act, bias, n, e, k, h, u):
    say("experts", dtype, act, bias, n, e, k, h, u)
    ex = experts_of(e, h, u, act, bias)
    g = torch.Generator().manual_seed(n + h)
    x = torch.randn(n, h, generator=g).to(dtype).to(dev)
    check_experts(x, *routing(n, e, k), ex)


@pytest.mark.parametrize("act", ["gelu", "swiglu"])
def test_large_groups(act):
    """Past 512 rows an expert, 256-row tiles; more than 8192 choices, the
    general plan."""
    say("large groups", act)
    ex = experts_of(4, 96, 2112, act, act == "gelu")
    x = torch.randn(9000, 96, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    check_experts(x, *routing(9000, 4, 2), ex)


@pytest.mark.parametrize("n", [3, 40, 700, 5000])
def test_dropped_merged_and_missing_choices(n):
    """Ids outside the experts, weights of 0 and below, one id in two slots, an
    expert that nobody wants, tokens without experts, NaN messages."""
    from spider_moe_amd import sparse_expert_delta_mxfp4
    say("dropped", n)
    e, k, h, u = 7, 3, 96, 160
    ex = experts_of(e, h, u, "gelu", True)
    idx, w = routing(n, e, k)
    idx[idx == 4] = 5  # nobody wants 4; some want 5 twice
    idx[0, 1], w[1, 0] = -1, 0.0
    idx[2, 0], w[2, 1], w[2, 2] = e, -0.5, 0.0
    if n > 6:
        idx[4] = idx[4, 0]
        w[5] = 0.0
    x = torch.randn(n, h, device=dev)
    want = check_experts(x, idx, w, ex)
    assert (want[2] == 0).all()
    y = x.clone()
    y[1, 50] = float("nan")
    y[0, 3] = float("inf")
    got = sparse_expert_delta_mxfp4(y, idx, w, ex)
    assert torch.isnan(got[:2]).all() and torch.equal(got[2:], want[2:])
    assert torch.equal(sparse_expert_delta_mxfp4(x, idx.long(), w.double(), ex), want)
    none = sparse_expert_delta_mxfp4(x, torch.full_like(idx, -1), w, ex)
    assert (none == 0).all()


@pytest.mark.parametrize("n", [2, 30, 600])
def test_hidden_activations_past_f32_make_nan(n):
    """Biases that make some hidden blocks infinite; the other tokens' rows and
    other experts stay."""
    say("overflow", n)
    ex = experts_of(4, 64, 96, "gelu", True)
    ex.b_up = ex.b_up.clone()
    ex.b_up[2, 40] = float("inf")
    x = torch.randn(n, 64, device=dev)
    idx, w = routing(n, 4, 2)
    from spider_moe_amd import sparse_expert_delta_mxfp4
    got = sparse_expert_delta_mxfp4(x, idx, w, ex)
    hit = (idx == 2).any(-1)
    assert torch.isnan(got[hit]).all() and torch.isfinite(got[~hit]).all()


@pytest.mark.parametrize("n", [4, 60, 900])
def test_scales_of_any_layout_and_held_tensors(n):
    """Scales in tight rows are copied once, codes that are laid out well stay;
    what changes in place afterwards, in the attributes, counts."""
    from spider_moe_amd import MxFp4Experts, sparse_expert_delta_mxfp4
    say("held", n)
    q = experts_of(5, 96, 160, "swiglu", True)
    idx, w = routing(n, 5, 2)
    x = torch.randn(n, 96, device=dev).bfloat16()
    want = check_experts(x, idx, w, q)
    tight = MxFp4Experts(q.w_up, q.s_up.contiguous(), q.w_down, q.s_down.contiguous(), b_up=q.b_up.bfloat16().float(),
                         b_down=q.b_down, activation="swiglu")
    assert tight.w_up.data_ptr() == q.w_up.data_ptr()
    tight.b_up = q.b_up
    assert torch.equal(sparse_expert_delta_mxfp4(x, idx, w, tight), want)
    off = torch.empty(q.w_up.numel() + 5, dtype=torch.uint8, device=dev)[5:].view(q.w_up.shape).copy_(q.w_up)
    assert torch.equal(sparse_expert_delta_mxfp4(x, idx, w, MxFp4Experts(
        off, q.s_up, q.w_down.transpose(0, 1).contiguous().transpose(0, 1), q.s_down, b_up=q.b_up, b_down=q.b_down,
        activation="swiglu")), want)
    if hasattr(torch, "float8_e8m0fnu"):
        named = MxFp4Experts(q.w_up, q.s_up.contiguous().view(torch.float8_e8m0fnu), q.w_down, q.s_down, b_up=q.b_up,
                             b_down=q.b_down, activation="swiglu")
        assert torch.equal(sparse_expert_delta_mxfp4(x, idx, w, named), want)
    other = experts_of(5, 96, 160, "swiglu", True, seed=9)
    for name in ("w_up", "s_up", "w_down", "s_down"):
        getattr(tight, name).copy_(getattr(other, name))
    tight.b_up, tight.b_down = other.b_up, other.b_down
    assert torch.equal(sparse_expert_delta_mxfp4(x, idx, w, tight), check_experts(x, idx, w, other))


def test_expert_refusals():
    from spider_moe_amd import Fp8BlockExperts, MxFp4Experts, sparse_expert_delta_fp8_blocks, sparse_expert_delta_mxfp4
    say("refusals")
    ex = experts_of(3, 64, 96, "gelu", False)
    idx, w = routing(5, 3, 2)
    x = torch.randn(5, 64, device=dev)
    for bad in ((x[:, :32], idx, w), (x, idx[:4], w), (x, idx, w[:, :1])):
        with pytest.raises(ValueError):
            sparse_expert_delta_mxfp4(*bad, ex)
    with pytest.raises(RuntimeError):
        sparse_expert_delta_mxfp4(x.half(), idx, w, ex)
    f8 = Fp8BlockExperts.quantize(torch.randn(3, 96, 64, device=dev), torch.randn(3, 64, 96, device=dev))
    with pytest.raises(TypeError):
        sparse_expert_delta_mxfp4(x, idx, w, f8)
    with pytest.raises(TypeError):
        sparse_expert_delta_fp8_blocks(x, idx, w, ex)
    for bad in (dict(w_up=ex.w_up[:, :64]), dict(s_up=ex.s_up[..., :1]), dict(w_up=ex.w_up.float()),
                dict(w_down=ex.w_down[..., :40]), dict(s_down=ex.s_down.cpu())):
        args = {**dict(w_up=ex.w_up, s_up=ex.s_up, w_down=ex.w_down, s_down=ex.s_down), **bad}
        with pytest.raises((ValueError, RuntimeError)):
            MxFp4Experts(**args)
    with pytest.raises(ValueError):
        MxFp4Experts.quantize(torch.randn(3, 96, 48, device=dev), torch.randn(3, 48, 96, device=dev))
    assert sparse_expert_delta_mxfp4(x[:0], idx[:0], w[:0], ex).shape == (0, 64)


# ------------------------------------------------------------ used together ----
@pytest.mark.parametrize("n", [1, 33, 300])
def test_route_balance_and_experts_in_a_graph(n):
    """A router's step as it is used: grouped routing, its balance loss, the
    experts and a projection, on another stream and captured; every replay
    against the eager results."""
    from spider_moe_amd import ForgeGEMM, ForgeSelect, sparse_expert_delta_mxfp4
    say("graph", n)
    ex = experts_of(16, 128, 192, "swiglu", True)
    codes, scale = weight(200, 128)
    sel, gemm = ForgeSelect(), ForgeGEMM()

    def step(x, z):
        w, i = sel.route_groups(z, top_k=4, score="sigmoid", num_groups=4, top_groups=2)
        loss, counts = sel.balance_loss(z, i, score="sigmoid")
        d = sparse_expert_delta_mxfp4(x, i, w, ex)
        return w, i, loss, counts, d, gemm.linear_mxfp4(x + d, codes, scale, act="gelu")

    g = torch.Generator().manual_seed(n)
    xs = [torch.randn(n, 128, generator=g).bfloat16().to(dev) for _ in range(3)]
    zs = [torch.randn(n, 16, generator=g).to(dev) for _ in range(3)]
    eager = [step(x, z) for x, z in zip(xs, zs)]
    bx, bz = xs[0].clone(), zs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(bx, bz)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(other, eager[0]):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(bx, bz)
    for r in range(4):
        bx.copy_(xs[r % 3])
        bz.copy_(zs[r % 3])
        graph.replay()
        again = step(xs[r % 3], zs[r % 3])
        torch.cuda.synchronize()
        for a, b, c in zip(out, eager[r % 3], again):
            assert torch.equal(a, b) and torch.equal(c, b)
