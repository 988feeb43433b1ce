"""Block-scaled fp8 on the GPU: the quantizer bit for bit against the CPU
formula, the linear product and the expert FFN against oracle/fp8_blocks.py in
64 bits.

Tolerances of a product (per output): bf16 outputs are off by half a step,
2^-8 of the value, and by the matrix unit's sums of e4m3 products, which are
cut at 2^-18 of a block's largest product each: 128 of them, 2^-11 of the
largest product, block by block (`top`).  f32 outputs are summed in f32:
2^-24 per operation, K + K / 128 + 4 of them, of the products' magnitudes
(`mag`).

The expert FFN quantizes its hidden activations, and one that lies as near as
the up product's error to a border between two codes may take the other code:
the oracle returns how far that lets each output be off
(oracle/fp8_blocks.py, expert_delta); a bf16 output's own rounding, 2^-8 of it,
comes on top."""
import pytest
import torch

from oracle import fp8_blocks as O

pytestmark = pytest.mark.gpu

dev = "cuda"


def say(*a):
    print("[case]", *a, flush=True)


def bits(codes):
    return codes.contiguous().view(torch.uint8).cpu()


def same_codes(a, b):
    """Equal codes; NaN codes of either sign are one."""
    a, b = bits(a), bits(b)
    return torch.equal(torch.where((a & 127) == 127, torch.full_like(a, 127), a),
                       torch.where((b & 127) == 127, torch.full_like(b, 127), b))


# ---------------------------------------------------------------- quantizer ----
@pytest.mark.parametrize("block_rows", [1, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", [(1, 1), (1, 128), (3, 127), (5, 129), (17, 16), (127, 200), (128, 256),
                                   (130, 1000), (2, 3, 70, 136), (4, 1, 40), (300, 1408), (1, 4099)])
def test_quantizer_is_the_cpu_formula(block_rows, dtype, shape):
    from spider_moe_amd import dequantize_fp8_blocks, quantize_fp8_blocks
    say("quantize", block_rows, dtype, shape)
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(*shape, generator=g) * torch.exp(2 * torch.randn(*shape[:-1], 1, generator=g))).to(dtype)
    q, s = quantize_fp8_blocks(x.to(dev), block_rows=block_rows)
    cq, cs = quantize_fp8_blocks(x, block_rows=block_rows)
    assert q.dtype == torch.float8_e4m3fn and q.shape == x.shape and s.dtype == torch.float32
    assert s.shape == (*shape[:-2], -(-shape[-2] // block_rows), -(-shape[-1] // 128))
    assert torch.equal(s.cpu(), cs)
    assert same_codes(q, cq)
    assert torch.equal(dequantize_fp8_blocks(q, s, block_rows=block_rows).cpu(),
                       dequantize_fp8_blocks(cq, cs, block_rows=block_rows))


@pytest.mark.parametrize("block_rows", [1, 128])
def test_quantizer_special_values(block_rows):
    """Zero blocks, values below the smallest scale, subnormals, the largest
    floats, NaN and infinities (as the f32 formula gives them)."""
    from spider_moe_amd import quantize_fp8_blocks
    say("quantize special", block_rows)
    x = torch.zeros(block_rows * 8, 256)
    r = block_rows
    x[r, 5], x[r, 130] = 1e-30, 1e-12
    x[2 * r, :3] = torch.tensor([1e-40, 2e-40, -1e-39])
    x[3 * r, :4] = torch.tensor([3.4e38, -3.4e38, 1.0, 1e30])
    x[4 * r, 7], x[4 * r, 8] = float("nan"), 2.0
    x[5 * r, 7], x[5 * r, 8] = float("inf"), 2.0
    x[6 * r, 200] = float("-inf")
    x[7 * r] = torch.linspace(-448, 448, 256)
    q, s = quantize_fp8_blocks(x.to(dev), block_rows=block_rows)
    cq, cs = quantize_fp8_blocks(x, block_rows=block_rows)
    assert torch.equal(torch.isnan(s.cpu()), torch.isnan(cs))
    assert torch.equal(torch.nan_to_num(s.cpu(), nan=-1.0), torch.nan_to_num(cs, nan=-1.0))
    assert same_codes(q, cq)


def test_quantizer_codes_on_every_border():
    """Quotients on, and one f32 step around, the middle between each two
    neighbouring codes and the codes themselves (scale exactly 1)."""
    from spider_moe_amd import quantize_fp8_blocks
    say("quantize borders")
    v = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
    mid = (v[1:] + v[:-1]) / 2
    pts = torch.cat([v, mid])
    up = torch.nextafter(pts, torch.full_like(pts, 1e9))
    dn = torch.nextafter(pts, torch.full_like(pts, -1e9))
    pts = torch.cat([pts, up, dn])
    pts = torch.cat([pts, -pts])
    pts = pts[pts.abs() <= 448]
    x = torch.zeros(-(-pts.numel() // 127), 128)
    x[:, 0] = 448.0
    flat = torch.zeros(x.shape[0] * 127)
    flat[:pts.numel()] = pts
    x[:, 1:] = flat.view(-1, 127)
    q, s = quantize_fp8_blocks(x.to(dev), block_rows=1)
    assert bool((s == 1).all())
    assert torch.equal(bits(q), bits(x.to(torch.float8_e4m3fn)))


def test_quantizer_strides():
    """Column slices, every second row, a transposed input, an odd offset: the
    codes of the same values laid out densely."""
    from spider_moe_amd import quantize_fp8_blocks
    say("quantize strides")
    g = torch.Generator().manual_seed(1)
    base = torch.randn(64, 700, generator=g).to(dev)
    for v in (base[:, 3:403], base[::2, 8:300], base.t()[:200], base[:, :1], base[5:6, 11:140],
              base.view(8, 8, 700)[:, :, 100:260], base.view(8, 8, 700)[:, 2:3, 40:168],
              base.view(8, 8, 700)[:, ::2, 40:168], base[0].expand(5, 700), base.view(-1)[1:1 + 60 * 700].view(60, 700)):
        for br in (1, 128):
            q, s = quantize_fp8_blocks(v, block_rows=br)
            cq, cs = quantize_fp8_blocks(v.contiguous().cpu(), block_rows=br)
            assert torch.equal(s.cpu(), cs) and same_codes(q, cq), (v.shape, v.stride(), br)


def test_quantizer_empty():
    from spider_moe_amd import quantize_fp8_blocks
    q, s = quantize_fp8_blocks(torch.empty(0, 40, device=dev), block_rows=1)
    assert q.shape == (0, 40) and s.shape == (0, 1)
    q, s = quantize_fp8_blocks(torch.empty(0, 5, 40, device=dev))
    assert q.shape == (0, 5, 40) and s.shape == (0, 1, 1)


# ------------------------------------------------------------------- linear ----
def _tol(y, mag, top, k, dtype, gelu):
    """GELU's slope is at most 1.13, its erf's own error 1.5e-7 of x."""
    slope = 1.13 if gelu else 1.0
    extra = 2e-7 * (y.abs() + mag) if gelu else 0.0
    if dtype == torch.bfloat16:
        return 2.0 ** -8 * y.abs() + slope * 2.0 ** -11 * top + extra + 2.0 ** -24 * mag
    return slope * (k + k / 128 + 8) * 2.0 ** -24 * mag + 2.0 ** -23 * y.abs() + extra + (
        2.0 ** -11 * y.abs() if dtype == torch.float16 else 0.0)


def _weights(g, *shape):
    from spider_moe_amd import quantize_fp8_blocks
    return quantize_fp8_blocks((torch.randn(*shape, generator=g) * 0.05).to(dev))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32, torch.float16])
@pytest.mark.parametrize("n,k,n_out", [(1, 128, 16), (1, 2048, 1408), (2, 1, 1), (3, 16, 5), (7, 100, 130),
                                       (16, 129, 128), (17, 1000, 300), (33, 256, 257), (64, 1408, 64),
                                       (65, 130, 1000), (127, 512, 129), (129, 384, 384), (200, 1000, 700),
                                       (257, 2816, 256), (300, 272, 2800), (600, 200, 520),
                                       (1029, 384, 300)])
def test_linear(dtype, n, k, n_out):
    from spider_moe_amd import ForgeGEMM
    say("linear", dtype, n, k, n_out)
    g = torch.Generator().manual_seed(n + k + n_out)
    x = (torch.randn(n, k, generator=g) * torch.exp(torch.randn(n, 1, generator=g))).to(dtype)
    q, s = _weights(g, n_out, k)
    b = torch.randn(n_out, generator=g)
    for bias, act in ((None, None), (b, None), (b, "gelu")):
        got = ForgeGEMM().linear_fp8_blocks(x.to(dev), q, s, None if bias is None else bias.to(dev), act=act)
        assert got.dtype == dtype and got.shape == (n, n_out)
        y, mag, top = O.linear(x, q, s, bias, act)
        tol = _tol(y, mag + (0 if bias is None else b.abs().double()), top, k, dtype, act == "gelu")
        err = (got.cpu().double() - y).abs()
        assert bool((err <= tol + 1e-30).all()), (bias is not None, act, float((err / (tol + 1e-30)).max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n,k,n_out", [(1, 384, 260), (5, 640, 512), (40, 640, 260), (130, 640, 515), (300, 1100, 200),
                                       (777, 400, 700)])
def test_linear_is_exact_on_small_integers(dtype, n, k, n_out):
    """One nonzero element a block and row, of value 448 times a power of two:
    every code is +-448, every product a power of two times the weight's
    small integer, every sum an integer that bf16 holds.  A block taken with
    another's scale, or a pair of wrong k, misses by whole numbers."""
    from spider_moe_amd import ForgeGEMM
    say("linear exact", dtype, n, k, n_out)
    g = torch.Generator().manual_seed(k)
    kb, nb = -(-k // 128), -(-n_out // 128)
    x = torch.zeros(n, k)
    for b in range(kb):
        width = min(128, k - 128 * b)
        at = 128 * b + torch.randint(0, width, (n,), generator=g)
        x[torch.arange(n), at] = (2.0 ** torch.randint(0, 2, (n,), generator=g)) * (
            2.0 * torch.randint(0, 2, (n,), generator=g) - 1)
    codes = torch.randint(-4, 5, (n_out, k), generator=g).float()
    scale = 2.0 ** torch.randint(0, 2, (nb, kb), generator=g).float()
    q = torch.zeros(n_out, -(-k // 16) * 16, dtype=torch.uint8)
    q[:, :k] = codes.to(torch.float8_e4m3fn).view(torch.uint8)
    q = q.view(torch.float8_e4m3fn)[:, :k].to(dev)
    got = ForgeGEMM().linear_fp8_blocks(x.to(dtype).to(dev), q, scale.to(dev)).cpu().double()
    want = x.double() @ O.values(codes, scale).t()
    # scale = 2^j / 448 is off by its rounding, 2^-24 of it, in every product, and
    # each of the (at most 9) blocks' sums by another 2^-24: within 16 * 2^-24 of
    # the magnitudes.  Rounding to bf16 takes a value that near to a whole number
    # below 256 to that number; where products cancel to 0 the difference stays
    assert bool(((got - want).abs() <= 2.0 ** -20 * (x.double().abs() @ O.values(codes, scale).abs().t())).all())


def test_linear_ignores_what_lies_behind_the_rows():
    """K that ends inside a block and a 16-byte chunk, weights in wider rows
    whose rest holds NaN codes; a column slice as input."""
    from spider_moe_amd import ForgeGEMM
    say("linear rests")
    g = torch.Generator().manual_seed(2)
    for n, k, n_out in ((3, 72, 40), (140, 200, 260), (1, 1000, 130)):
        q, s = _weights(g, n_out, k)
        wide = torch.full((n_out, 16 * (k // 16 + 3)), 0x7f, dtype=torch.uint8, device=dev)
        wide[:, :k] = q.contiguous().view(torch.uint8)
        x = torch.randn(n, k + 37, generator=g).to(torch.bfloat16).to(dev)
        x[:, :5] = float("nan")
        x[:, 5 + k:] = float("nan")
        a = ForgeGEMM().linear_fp8_blocks(x[:, 5:5 + k], wide.view(torch.float8_e4m3fn)[:, :k], s)
        b = ForgeGEMM().linear_fp8_blocks(x[:, 5:5 + k].contiguous(), q, s)
        assert torch.equal(a, b) and not bool(torch.isnan(a).any())
        # codes in rows that the kernels do not read: copied on the way
        c = ForgeGEMM().linear_fp8_blocks(x[:, 5:5 + k].contiguous(), q.contiguous(), s)
        d = ForgeGEMM().linear_fp8_blocks(x[:, 5:5 + k].contiguous().view(n, 1, k),
                                          q.contiguous().view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn), s)
        assert torch.equal(c, b) and torch.equal(d.view(n, n_out), b)


def test_linear_special_rows():
    """A row of zeros gives the bias; a NaN or infinite element makes its row
    NaN and no other."""
    from spider_moe_amd import ForgeGEMM
    say("linear special rows")
    g = torch.Generator().manual_seed(3)
    q, s = _weights(g, 200, 300)
    b = torch.randn(200, generator=g).to(dev)
    for n in (4, 150):
        x = torch.randn(n, 300, generator=g).to(torch.bfloat16).to(dev)
        clean = ForgeGEMM().linear_fp8_blocks(x, q, s, b)
        x[1] = 0
        x[2, 290] = float("nan")
        x[3, 7] = float("inf")
        got = ForgeGEMM().linear_fp8_blocks(x, q, s, b)
        assert torch.equal(got[0], clean[0]) and torch.equal(got[4:], clean[4:])
        assert torch.equal(got[1], b.to(torch.bfloat16))
        assert bool(torch.isnan(got[2:4]).all())


def test_linear_takes_codes():
    """Input quantized by the caller: the same result as quantizing on the way."""
    from spider_moe_amd import ForgeGEMM, quantize_fp8_blocks
    from spider_moe_amd import _native as nat
    say("linear codes")
    g = torch.Generator().manual_seed(4)
    for n, k, n_out in ((1, 200, 48), (20, 1000, 130), (150, 384, 256)):
        x = torch.randn(n, k, generator=g).to(torch.bfloat16).to(dev)
        q, s = _weights(g, n_out, k)
        xq, xs = quantize_fp8_blocks(x, block_rows=1)
        out = torch.empty(n, n_out, dtype=torch.bfloat16, device=dev)
        ldx = xq.stride(0) if n > 1 else -(-k // 16) * 16
        nat.check(nat.lib().smoe_linear_fp8_blocks(
            xq.data_ptr(), nat.FP8_E4M3, ldx, xs.data_ptr(), n, k, q.data_ptr(), q.stride(0), s.data_ptr(),
            None, n_out, 0, out.data_ptr(), nat.BF16, None, 0, nat.stream_of(x.device)), "linear")
        assert torch.equal(out, ForgeGEMM().linear_fp8_blocks(x, q, s))


def test_linear_empty_and_streams():
    from spider_moe_amd import ForgeGEMM
    say("linear empty, streams")
    g = torch.Generator().manual_seed(5)
    q, s = _weights(g, 200, 300)
    assert ForgeGEMM().linear_fp8_blocks(torch.empty(0, 300, device=dev), q, s).shape == (0, 200)
    x = torch.randn(70, 300, generator=g).to(torch.bfloat16).to(dev)
    want = ForgeGEMM().linear_fp8_blocks(x, q, s)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for st in streams:
        with torch.cuda.stream(st):
            outs.append([ForgeGEMM().linear_fp8_blocks(x, q, s) for _ in range(3)])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for group in outs for o in group)


# ------------------------------------------------------------------ experts ----
def _experts(g, e, h, u, activation, bias):
    from spider_moe_amd import Fp8BlockExperts
    halves = 2 if activation == "swiglu" else 1
    up = torch.randn(e, halves * u, h, generator=g) * h ** -0.5
    down = torch.randn(e, h, u, generator=g) * u ** -0.5
    bu = torch.randn(e, u, generator=g) * 0.1 if bias else None
    bd = torch.randn(e, h, generator=g) * 0.1 if bias else None
    to = lambda t: None if t is None else t.to(dev)  # noqa: E731
    return Fp8BlockExperts.quantize(to(up), to(down), b_up=to(bu), b_down=to(bd), activation=activation)


def _routing(g, n, e, k):
    z, idx = torch.topk(torch.randn(n, e, generator=g), k, dim=-1)
    return idx.to(torch.int32), torch.softmax(z, -1)


def _check_delta(got, ref):
    want, tol = ref
    tol = tol * (1 + 2.0 ** -8) + 2.0 ** -8 * want.abs() if got.dtype == torch.bfloat16 else tol
    err = (got.cpu().double().view_as(want) - want).abs()
    print("  largest share of the tolerance", float((err / (tol + 1e-30)).max()), "tolerance / rms",
          float(tol.mean() / want.pow(2).mean().sqrt().clamp_min(1e-30)), flush=True)
    assert bool((err <= tol + 1e-30).all()), float((err / (tol + 1e-30)).max())


SHAPES = [  # n, e, k, h, u
    (1, 1, 1, 16, 16), (1, 8, 2, 256, 512), (1, 64, 2, 2048, 1408), (2, 4, 3, 144, 208), (5, 12, 3, 528, 1200),
    (16, 8, 2, 256, 384), (33, 16, 4, 512, 272), (64, 16, 2, 1024, 256), (100, 3, 2, 128, 128),
    (260, 5, 2, 400, 336), (300, 2, 1, 1024, 640), (515, 33, 6, 272, 144),
    (1100, 2, 1, 272, 400), (1300, 3, 2, 128, 272),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("activation,bias", [("gelu", True), ("gelu", False), ("swiglu", False), ("swiglu", True)])
@pytest.mark.parametrize("n,e,k,h,u", SHAPES)
def test_expert_delta(dtype, activation, bias, n, e, k, h, u):
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("expert delta", dtype, activation, bias, n, e, k, h, u)
    g = torch.Generator().manual_seed(n + e + h)
    ex = _experts(g, e, h, u, activation, bias)
    msg = torch.randn(n, 1, h, generator=g).to(dtype)
    idx, w = _routing(g, n, e, k)
    got = sparse_expert_delta_fp8_blocks(msg.to(dev), idx.view(n, 1, k).to(dev), w.view(n, 1, k).to(dev), ex)
    assert got.dtype == dtype and got.shape == msg.shape
    want = O.expert_delta(msg.view(n, h), idx, w, ex.w_up, ex.s_up, ex.w_down, ex.s_down, ex.b_up, ex.b_down,
                          activation)
    _check_delta(got, want)
    again = sparse_expert_delta_fp8_blocks(msg.to(dev), idx.view(n, 1, k).to(dev), w.view(n, 1, k).to(dev), ex)
    assert torch.equal(got, again)


@pytest.mark.parametrize("n", [9, 70, 400])
def test_expert_delta_uneven_routing(n):
    """All tokens on one expert; ids outside [0, E), repeated ids, weights of
    0, below 0 and NaN; tokens left without experts get exact zeros."""
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("expert delta uneven", n)
    g = torch.Generator().manual_seed(n)
    e, k, h, u = 6, 3, 256, 192
    ex = _experts(g, e, h, u, "swiglu", False)
    msg = torch.randn(n, h, generator=g).to(torch.bfloat16)
    idx, w = _routing(g, n, e, k)
    idx[:, 0], idx[:, 1], idx[:, 2] = 4, 4, torch.randint(-2, e + 2, (n,), generator=g).int()
    w[0], w[1, 0], w[2] = 0.0, -1.0, -0.5
    idx[3] = torch.tensor([-1, e, 1 << 30])
    got = sparse_expert_delta_fp8_blocks(msg.to(dev), idx.to(dev), w.to(dev), ex)
    want = O.expert_delta(msg, idx, w, ex.w_up, ex.s_up, ex.w_down, ex.s_down, activation="swiglu")
    _check_delta(got, want)
    assert not bool(got[0].any()) and not bool(got[2].any()) and not bool(got[3].any())
    none = sparse_expert_delta_fp8_blocks(msg.to(dev), torch.full_like(idx, -1).to(dev), w.to(dev), ex)
    assert not bool(none.any())
    assert sparse_expert_delta_fp8_blocks(msg[:0].to(dev), idx[:0].to(dev), w[:0].to(dev), ex).shape == (0, h)


def test_expert_delta_special_messages():
    """A NaN, an infinite and a zero message: each token's own result only."""
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("expert delta special")
    g = torch.Generator().manual_seed(12)
    for n in (5, 200):
        ex = _experts(g, 8, 256, 320, "gelu", True)
        msg = torch.randn(n, 256, generator=g).to(torch.bfloat16).to(dev)
        idx, w = _routing(g, n, 8, 2)
        idx, w = idx.to(dev), w.to(dev)
        clean = sparse_expert_delta_fp8_blocks(msg, idx, w, ex)
        msg[1, 3], msg[2, 255], msg[3] = float("nan"), float("inf"), 0.0
        got = sparse_expert_delta_fp8_blocks(msg, idx, w, ex)
        assert bool(torch.isnan(got[1]).all()) and bool(torch.isnan(got[2]).all())
        assert torch.equal(got[0], clean[0]) and torch.equal(got[4:], clean[4:])
        want = O.expert_delta(msg[3:4].cpu(), idx[3:4], w[3:4], ex.w_up, ex.s_up, ex.w_down, ex.s_down, ex.b_up,
                              ex.b_down)
        _check_delta(got[3:4], want)


def test_a_tokens_result_in_batches_of_every_size():
    """One token alone, in a decode batch and in a prompt: each within the
    oracle's distance."""
    from spider_moe_amd import sparse_expert_delta_fp8_blocks
    say("expert delta batch")
    g = torch.Generator().manual_seed(13)
    ex = _experts(g, 8, 512, 640, "swiglu", False)
    msg = torch.randn(600, 512, generator=g).to(torch.bfloat16)
    idx, w = _routing(g, 600, 8, 2)
    want, tol = O.expert_delta(msg, idx, w, ex.w_up, ex.s_up, ex.w_down, ex.s_down, activation="swiglu")
    for n in (1, 7, 30, 100, 600):
        got = sparse_expert_delta_fp8_blocks(msg[:n].to(dev), idx[:n].to(dev), w[:n].to(dev), ex)
        _check_delta(got, (want[:n], tol[:n]))


def test_a_step_of_them_together():
    """Router logits -> grouped routing -> experts on block-scaled weights,
    and a projection on them: a decode step's and a prompt's sizes, captured
    in a graph, replayed on new inputs, against the eager calls and the
    oracle."""
    from spider_moe_amd import ForgeGEMM, ForgeSelect, quantize_fp8_blocks, sparse_expert_delta_fp8_blocks
    say("together")
    g = torch.Generator().manual_seed(14)
    e, k, h, u = 16, 4, 256, 384
    ex = _experts(g, e, h, u, "swiglu", False)
    router = (torch.randn(e, h, generator=g) * h ** -0.5).to(dev)
    bias = (torch.randn(e, generator=g) * 0.05).to(dev)
    wq, ws = quantize_fp8_blocks((torch.randn(200, h, generator=g) * h ** -0.5).to(dev))
    sel, gemm = ForgeSelect(), ForgeGEMM()

    def step(x):
        w, idx = sel.route_groups(x.float() @ router.t(), top_k=k, bias=bias, num_groups=4, top_groups=2, scale=2.5)
        d = sparse_expert_delta_fp8_blocks(x, idx, w, ex)
        return w, idx, d, gemm.linear_fp8_blocks(x + d, wq, ws)

    for n in (1, 6, 64, 300):
        static = torch.randn(n, h, generator=g).to(torch.bfloat16).to(dev)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(static)
        for i in range(3):
            new = torch.randn(n, h, generator=g).to(torch.bfloat16).to(dev)
            static.copy_(new)
            graph.replay()
            torch.cuda.synchronize()
            got = [o.clone() for o in out]
            want = step(new)
            assert all(torch.equal(a, b) for a, b in zip(got, want)), (n, i)
        w, idx, d, y = got
        ww, wi = O.select_groups((new.float() @ router.t()).cpu(), k, score="sigmoid", bias=bias, groups=4,
                                 top_groups=2, scale=2.5)
        assert torch.equal(idx.cpu().long(), wi)
        _check_delta(d, O.expert_delta(new, idx, w, ex.w_up, ex.s_up, ex.w_down, ex.s_down, activation="swiglu"))
        ref, mag, top = O.linear(new + d, wq, ws)
        assert bool(((y.cpu().double() - ref).abs() <= _tol(ref, mag, top, h, torch.bfloat16, False)).all())
