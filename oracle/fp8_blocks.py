"""64-bit oracles of group-limited routing and of block-scaled fp8.

Routing: s = softmax(z) or sigmoid(z), 0 where z = -inf; c = s + bias, masked
experts below every other; a group's value is the sum of its two largest
unmasked c; the K largest c of the best groups, ties to the lower index, NaN
as +infinity; weights scale * s / max(sum, 1e-9) or scale * s.

Block-scaled fp8: per block scale = max(amax / 448, 1e-12) and code =
e4m3(x / scale), both quotients rounded to f32 first (the format's
definition); everything after the codes is exact in 64 bits.
"""
from __future__ import annotations

import numpy as np
import torch

B = 128


def select_groups(z: torch.Tensor, k: int, *, score: str, bias=None, groups: int = 1,
                  top_groups: int = 1, renorm: bool = True, scale: float = 1.0):
    """z [N,E] -> (weights f64 [N,K], indices [N,K])."""
    z = z.detach().cpu().double()
    n, e = z.shape
    masked = z == -np.inf
    if score == "softmax":
        m = torch.where(masked, -np.inf, z).amax(-1, keepdim=True)
        p = torch.where(masked, 0.0, torch.exp(z - m))
        s = p / p.sum(-1, keepdim=True)
    else:
        s = torch.sigmoid(z)
    s = torch.where(masked, 0.0, s)
    c = s if bias is None else s + bias.detach().cpu().double()
    c = torch.where(masked, -np.inf, c)
    c = torch.where(torch.isnan(c), np.inf, c).numpy()
    idx = np.zeros((n, k), dtype=np.int64)
    per = e // groups
    for t in range(n):
        order = np.argsort(-c[t], kind="stable")
        if groups > 1:
            value = []
            for g in range(groups):
                v = np.sort(c[t, g * per:(g + 1) * per])[::-1][:2]
                u = v[v > -np.inf]
                value.append(u.sum() if u.size else -np.inf)
            kept = set(np.argsort(-np.array(value), kind="stable")[:top_groups].tolist())
            order = np.array([i for i in order if i // per in kept])
        idx[t] = order[:k]
    idx = torch.from_numpy(idx)
    w = s.gather(1, idx)
    if renorm:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total < 1e-9, 1e-9, total)
    return w * scale, idx


def select_groups_weights(z: torch.Tensor, idx: torch.Tensor, *, score: str, renorm: bool, scale: float):
    """The weights of a fixed choice as a differentiable function of z (f64)."""
    masked = z == -np.inf
    if score == "softmax":
        m = z.detach().amax(-1, keepdim=True)
        p = torch.where(masked, torch.zeros((), dtype=z.dtype), torch.exp(torch.where(masked, m, z) - m))
        s = p / p.sum(-1, keepdim=True)
    else:
        s = torch.sigmoid(z)
    w = s.gather(1, idx)
    if renorm:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-9)
    return w * scale


def quantize(x: torch.Tensor, block_rows: int):
    """x [rows, cols] -> (code values f64 [rows, cols], scales f64)."""
    x = x.detach().cpu().double().numpy()
    rows, cols = x.shape
    rb, cb = -(-rows // block_rows), -(-cols // B)
    p = np.zeros((rb * block_rows, cb * B))
    p[:rows, :cols] = x
    p = p.reshape(rb, block_rows, cb, B)
    s = np.maximum((np.abs(p).max(axis=(1, 3)) / 448.0).astype(np.float32).astype(np.float64), np.float64(np.float32(1e-12)))
    v = (p / s[:, None, :, None]).astype(np.float32).astype(np.float64)
    step = np.exp2(np.floor(np.log2(np.maximum(np.abs(v), 2.0 ** -6))) - 3)
    v = np.rint(v / step) * step
    return torch.from_numpy(v.reshape(rb * block_rows, cb * B)[:rows, :cols].copy()), torch.from_numpy(s)


def values(codes: torch.Tensor, scale: torch.Tensor, block_rows: int = B):
    """codes [rows, cols] (values) times the scales of their blocks, f64."""
    rows, cols = codes.shape
    r = torch.arange(rows) // block_rows
    c = torch.arange(cols) // B
    return codes.cpu().double() * scale.cpu().double()[r][:, c]


def gelu(y):
    return 0.5 * y * (1.0 + torch.erf(y * 0.5 ** 0.5))


def linear(x, codes, scale, bias=None, act=None):
    """x [N,K] quantized in 1 x 128 blocks, times W^T; also the sum of the
    products' magnitudes (what rounding errors scale with) and, summed over
    the blocks, the largest product of each."""
    xv = values(*quantize(x, 1), 1)
    wv = values(codes, scale)
    y = xv @ wv.t()
    mag = xv.abs() @ wv.abs().t()
    top = torch.zeros_like(y)
    for k in range(0, xv.shape[1], B):
        a, b = xv[:, k:k + B].abs(), wv[:, k:k + B].abs()
        top += (a.amax(1, keepdim=True) * b.amax(1)[None])
    if bias is not None:
        y = y + bias.cpu().double()
    return (gelu(y) if act == "gelu" else y), mag, top


def _round_code(q: torch.Tensor) -> torch.Tensor:
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(q / step) * step).clamp(-448.0, 448.0)


def _spread(s, cols):
    return s.repeat_interleave(B, dim=1)[:, :cols]


def _act_codes(a, d):
    """Activations a [rows, U], each off by at most d: their quantized values
    and how far those may be off, as the codes at both ends of each interval
    (the block's scale moves with its largest element)."""
    rows, u = a.shape
    pad = -u % B
    blocks = lambda t: torch.nn.functional.pad(t, (0, pad)).view(rows, -1, B).amax(-1)  # noqa: E731
    c, s = quantize(a, 1)
    amax, damax = blocks(a.abs()), blocks(d)
    rel = damax / amax.clamp_min(1e-300) + 2.0 ** -22
    sf = _spread(s, u)
    q = a / sf
    dq = d / sf + (q.abs() + d / sf) * _spread(rel, u)
    off = torch.maximum((_round_code(q + dq) - c).abs(), (_round_code(q - dq) - c).abs())
    return c * sf, off * sf + c.abs() * sf * _spread(rel, u)


# What the matrix unit's e4m3 x e4m3 sums of a block are off by on codes of
# random data: 2^-11 of the block's largest product.  At worst (7 of each eight
# products cut by 2^-13 of the eight's largest) it is 7 * 16 * 2^-13 of it:
# tests/test_gpu_fp8_block_sums.py.
BLOCK_CUT = 2.0 ** -11


def expert_delta(msg, idx, w, w_up, s_up, w_down, s_down, b_up=None, b_down=None, activation="gelu",
                 f32_sums=False):
    """msg [N,H], idx / w [N,K] -> (delta f64 [N,H], how far a right result
    may be off before its last rounding); slots of one expert merged, weights
    <= 0 and ids outside [0, E) dropped.

    The distance: each pre-activation is off by BLOCK_CUT of its blocks'
    largest products; the activation function carries that on (GELU's slope is
    at most 1.13, SiLU's 1.1; their own errors in f32 3e-7 of the argument and
    2e-6 of the value); where a border between two codes lies that near, the
    other code is as right; the down product carries on the codes' distance
    and adds its own cut.

    f32_sums: both products summed in f32, with no cut: off by 2^-24 of the
    magnitudes for each of a sum's K + K / 128 + 8 operations."""
    n, h = msg.shape
    e, u = w_down.shape[0], w_down.shape[2]
    ub = -(-u // B)
    x = values(*quantize(msg, 1), 1)
    out, tol = torch.zeros(n, h, dtype=torch.float64), torch.zeros(n, h, dtype=torch.float64)
    idx, w = idx.cpu().long(), w.cpu().float()

    def product(a, codes, scale, bias):
        wv = values(codes, scale)
        y = a @ wv.t()
        mag = a.abs() @ wv.abs().t()
        if f32_sums:
            d = (a.shape[1] * (1 + 1 / B) + 8) * 2.0 ** -24 * mag
            if bias is not None:
                d = d + 2.0 ** -24 * (y + bias.cpu().double()).abs()
            return (y if bias is None else y + bias.cpu().double()), d, wv
        d = 2.0 ** -20 * mag
        for k in range(0, a.shape[1], B):
            d += BLOCK_CUT * a[:, k:k + B].abs().amax(1, keepdim=True) * wv[:, k:k + B].abs().amax(1)[None]
        return (y if bias is None else y + bias.cpu().double()), d, wv

    for i in range(e):
        wt = torch.zeros(n, dtype=torch.float32)
        for j in range(idx.shape[1]):  # slot order, in f32, as the plan merges
            wt = wt + torch.where(idx[:, j] == i, w[:, j], torch.zeros(()))
        at = torch.nonzero(wt > 0).flatten()
        if not at.numel():
            continue
        bu = None if b_up is None else b_up[i]
        if activation == "swiglu":
            gate, dg, _ = product(x[at], w_up[i, :u], s_up[i, :ub], None)
            up, du, _ = product(x[at], w_up[i, u:], s_up[i, ub:], bu)
            sg = gate * torch.sigmoid(gate)
            a = sg * up
            d = 1.1 * dg * (up.abs() + du) + sg.abs() * du + 2e-6 * a.abs()
        else:
            up, du, _ = product(x[at], w_up[i], s_up[i], bu)
            a = gelu(up)
            d = 1.13 * du + 3e-7 * up.abs()
        v, dv = _act_codes(a, d)
        y, dy, wv = product(v, w_down[i], s_down[i], None if b_down is None else b_down[i])
        wt = wt[at].double().unsqueeze(1)
        out[at] += y * wt
        tol[at] += (dy + dv @ wv.abs().t() + 2.0 ** -22 * y.abs()) * wt
    return out, tol
