"""64-bit oracles of microscaled 4-bit floats (MXFP4) and of a router's balance
loss.

A block of 32 along a row: power of two 2^(floor(log2 amax) - 2), at least
2^-127, and the nearest of the e2m1 values to x / power, ties to the even code,
past 6 to 6; a block with an infinity or a NaN is NaN.  Everything runs where
its inputs are, in float64.
"""
from __future__ import annotations

import torch

B = 32


def blocks(x: torch.Tensor) -> torch.Tensor:
    """[rows, cols] -> [rows, blocks, 32], zeros past cols."""
    return torch.nn.functional.pad(x, (0, -x.shape[-1] % B)).unflatten(-1, (-1, B))


def exponent(amax: torch.Tensor) -> torch.Tensor:
    """Of the block's power of two, for finite amax."""
    return (torch.frexp(amax).exponent - 3).clamp(-127, 127).double()


def nearest(v: torch.Tensor) -> torch.Tensor:
    """v >= 0 to the nearest e2m1 value: multiples of 1/2 below 2, of 1 below
    4, of 2 up to 6 (torch.round takes ties to the even multiple, which is the
    even code)."""
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    return (torch.round(v / step) * step).clamp_max(6.0)


def quantize(x: torch.Tensor):
    """x [rows, cols] -> (values f64 [rows, cols], biased exponents [rows, blocks])."""
    p = blocks(x.double())
    bad = ~torch.isfinite(p).all(-1)
    p = torch.where(bad.unsqueeze(-1), 0.0, p)
    e = exponent(p.abs().amax(-1))
    two = torch.exp2(e).unsqueeze(-1)
    v = torch.copysign(nearest(p.abs() / two) * two, p)
    v = torch.where(bad.unsqueeze(-1), float("nan"), v)
    return v.flatten(-2)[..., :x.shape[-1]], torch.where(bad, 255.0, e + 127.0)


def spread(x: torch.Tensor, err: torch.Tensor) -> torch.Tensor:
    """How far the quantized value of anything within err of x can be from
    x's: the value grows with x at a fixed power, so the ends decide, at every
    power that the block's amax can have."""
    p, d = blocks(x.double()), blocks(err.double())
    base = nearest(p.abs() / torch.exp2(exponent(p.abs().amax(-1))).unsqueeze(-1))
    base = base * torch.exp2(exponent(p.abs().amax(-1))).unsqueeze(-1)
    lo, hi = (p.abs() - d).clamp_min(0.0), p.abs() + d
    far = torch.zeros_like(p)
    for amax in (lo.amax(-1), p.abs().amax(-1), hi.amax(-1)):
        two = torch.exp2(exponent(amax)).unsqueeze(-1)
        for v in (lo, hi):
            q = nearest(v / two) * two
            far = torch.maximum(far, (q - base).abs())
    far = torch.where((p.abs() < d) & (far > 0), far + base, far)  # the sign may turn
    return far.flatten(-2)[..., :x.shape[-1]]


def values(codes: torch.Tensor, scale: torch.Tensor, cols: int) -> torch.Tensor:
    """What stored codes [rows, ceil(cols / 2)] and scales [rows, blocks] stand for."""
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=codes.device)
    table = torch.cat([table, -table])
    c = torch.stack([codes % 16, codes // 16], -1).flatten(-2)[..., :cols].long()
    two = torch.where(scale == 255, float("nan"), torch.exp2(scale.double() - 127.0))
    return table[c] * two.repeat_interleave(B, -1)[..., :cols]


def gelu(y: torch.Tensor) -> torch.Tensor:
    return 0.5 * y * torch.special.erfc(-y * 0.5 ** 0.5)


def sum_error(k: int, mag: torch.Tensor) -> torch.Tensor:
    """Bound of an f32 sum of k products in steps of 128: each step adds exact
    sums of 32 and its accumulator, and is off by at most 4 * 2^-24 of the
    magnitudes; up to 8 partial sums and 3 more operations follow."""
    return (4 * (-(-k // 128) + 1) + 11) * 2.0 ** -24 * mag


def linear(x, codes, scale, bias=None, act=None):
    """(act(q(x) . W^T + bias), its error bound in f32) of x [N, K]."""
    k = x.shape[-1]
    xv, w = quantize(x)[0], values(codes, scale, k)
    y, mag = xv @ w.t(), xv.abs() @ w.abs().t()
    if bias is not None:
        y, mag = y + bias.double(), mag + bias.double().abs()
    err = sum_error(k, mag)
    if act == "gelu":
        z = gelu(y)
        return z, 1.13 * err + 2.0 ** -17.8 * z.abs() + 2.0 ** -23 * y.clamp_min(0.0)
    return y, err


def expert_delta(msg, idx, w, w_up, s_up, w_down, s_down, b_up=None, b_down=None, activation="gelu"):
    """(delta [N,H] f64, error bound [N,H] of an f32 computation, output
    rounding left out): the hidden activations' f32 errors may take them over
    a border between two codes, and a block's largest over a power of two."""
    n, h = msg.shape
    e, u = w_down.shape[0], 2 * w_down.shape[2]
    xv = quantize(msg)[0]
    delta = torch.zeros(n, h, dtype=torch.float64, device=msg.device)
    bound = torch.zeros_like(delta)
    for j in range(e):
        wt = torch.where(idx == j, w.double(), 0.0).sum(-1)
        at = torch.nonzero((idx == j).any(-1) & (wt > 0)).view(-1)
        if not at.numel():
            continue
        x, wv = xv[at], values(w_up[j], s_up[j], h)
        y, mag = x @ wv.t(), x.abs() @ wv.abs().t()
        b = torch.zeros(u, dtype=torch.float64, device=msg.device) if b_up is None else b_up[j].double()
        if activation == "swiglu":
            gate, up = y[:, :u], y[:, u:] + b
            eg, eu = sum_error(h, mag[:, :u]), sum_error(h, mag[:, u:] + b.abs())
            s = gate * torch.sigmoid(gate)
            a = s * up
            # silu's slope is below 1.1; its own error: |x| 2^-23 in the exponent, a reciprocal, a product
            err = 1.1 * eg * (up.abs() + eu) + s.abs() * eu + a.abs() * (gate.abs() + 6) * 2.0 ** -22
        else:
            y = y + b
            a = gelu(y)
            err = 1.13 * sum_error(h, mag + b.abs()) + 2.0 ** -17.8 * a.abs() + 2.0 ** -23 * y.clamp_min(0.0)
        q, far = quantize(a)[0], spread(a, err)
        d = values(w_down[j], s_down[j], u)
        o, omag = q @ d.t(), (q.abs() + far) @ d.abs().t()
        if b_down is not None:
            o, omag = o + b_down[j].double(), omag + b_down[j].double().abs()
        k = wt[at].unsqueeze(-1)
        delta[at] += k * o
        # the products' sums, the weight (merged slots) and the sum over experts
        bound[at] += k * (far @ d.abs().t() + sum_error(u, omag) + (4 + idx.shape[-1] * 2) * 2.0 ** -24 * omag)
    return delta, bound


def balance(z, idx, *, score="softmax", mask=None):
    """(loss [S], counts [S,E], u / n [S,E], p [S,T,E]) of z [S,T,E], idx
    [S,T,K] in f64, differentiable in z through loss."""
    s, t, e = z.shape
    z = z.double()
    on = torch.ones(s, t, dtype=torch.bool, device=z.device) if mask is None else mask.bool()
    dead = z == -float("inf")
    every = dead.all(-1, keepdim=True)
    safe = torch.where(on.unsqueeze(-1) & ~every, torch.where(dead, -1e30, z), torch.zeros_like(z))
    p = torch.softmax(safe if score == "softmax" else torch.nn.functional.logsigmoid(safe), -1)
    p = torch.where(on.unsqueeze(-1) & ~every & ~dead, p, torch.zeros_like(p))
    hot = ((idx.unsqueeze(-1) == torch.arange(e, device=z.device)).sum(2) * on.unsqueeze(-1)).double()
    counts = hot.sum(1)
    n = on.sum(1).double().clamp_min(1.0).unsqueeze(-1)
    load = counts / counts.sum(-1, keepdim=True).clamp_min(1.0)
    loss = e * (load * p.sum(1) / n).sum(-1)
    u = torch.where(counts.sum(-1, keepdim=True) > 0, (e * load - 1.0) / n, torch.zeros_like(load))
    return loss, counts.to(torch.int32), u, p
