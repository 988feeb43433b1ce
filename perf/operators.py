"""Routed experts on block-scaled fp8 weights, operator by operator, as measurable cases.

Four operators, in the order a step runs them:

  route    ForgeSelect.route_groups: softmax or sigmoid scores of the router's
           logits, a balance bias that counts in the choice only, the choice
           limited to the best groups of experts, top-k, renormalised weights;
           with its gradient in a training step
  quant    quantize_fp8_blocks: e4m3 codes with one scale for each 1 x 128
           block (activations) or 128 x 128 block (weights)
  linear   ForgeGEMM.linear_fp8_blocks: activations quantized in 1 x 128
           blocks on the way, times weights held in 128 x 128 blocks
  experts  sparse_expert_delta_fp8_blocks: dispatch, both products of every
           token's experts on such weights, and the weighted combine

Hidden states are N(0, 1), weights N(0, 0.02), router logits N(0, 1.5), as
the seeded workloads of spider_moe_amd.workloads have them; everything is
drawn on the GPU from the seed alone.  exact() restates each operator in 64
bits.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
EXPONENT_MIN = -6  # of e4m3's normal numbers

# The expert shapes of the framework's benchmark and of its default
# ModelConfig, and one whose sizes are no multiples of a block.
MODELS = {
    "swiglu16": dict(H=1024, E=16, K=2, U=2816, act="swiglu"),
    "gelu32": dict(H=1024, E=32, K=4, U=1408, act="gelu"),
    "gelu64": dict(H=2048, E=64, K=2, U=1408, act="gelu"),
    "default": dict(H=256, E=8, K=2, U=512, act="gelu"),
    "ragged12": dict(H=528, E=12, K=3, U=1200, act="swiglu"),
}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ cases ----
def _route(name, n, e, k, *, score, dtype="f32", bias=True, groups=1, top_groups=1, renorm=True,
           scale=1.0, train=False):
    return {"name": name, "kind": "route", "N": n, "E": e, "K": k, "score": score, "dtype": dtype,
            "bias": bias, "groups": groups, "top_groups": top_groups, "renorm": renorm,
            "scale": scale, "train": train}


def _quant(name, rows, cols, *, block_rows, dtype="bf16"):
    return {"name": name, "kind": "quant", "rows": rows, "cols": cols, "block_rows": block_rows,
            "dtype": dtype}


def _linear(name, n, k, n_out, *, act="none", bias=False):
    return {"name": name, "kind": "linear", "N": n, "K": k, "N_out": n_out, "act": act, "bias": bias}


def _experts(name, model, tokens, *, skew=0.0):
    return {"name": name, "kind": "experts", "model": model, "tokens": tokens, "skew": skew}


def listed():
    return [
        # one user's next token over 256 grouped experts: all latency
        _route("route-1-sigmoid-256", 1, 256, 8, score="sigmoid", groups=8, top_groups=4, scale=2.5),
        # a training step of a small router on bf16 logits, odd length, with the gradient
        _route("route-777-softmax-64-train", 777, 64, 2, score="softmax", dtype="bf16", bias=False,
               train=True),
        # a large training step of grouped sigmoid routing, with the gradient
        _route("route-16384-sigmoid-256-train", 16384, 256, 8, score="sigmoid", groups=8,
               top_groups=4, scale=2.5, train=True),
        # the activations of an ordinary prompt with rows that end inside a block
        _quant("quant-777x1000", 777, 1000, block_rows=1),
        # a stack of 16 experts' down projections when a model is loaded
        _quant("quant-weights-16384x2816", 16384, 2816, block_rows=128),
        # one token through a projection: weight streaming
        _linear("linear-1x2048x1408", 1, 2048, 1408),
        # a ragged chunk with bias and GELU, K and N_out that end inside a block
        _linear("linear-200x1000x2800-gelu", 200, 1000, 2800, act="gelu", bias=True),
        # a large prefill batch through a gate and up projection
        _linear("linear-16384x1024x5632", 16384, 1024, 5632),
        # one user's next token over 64 experts, 2 of which are read
        _experts("experts-1-gelu64", "gelu64", 1),
        # a full decode batch: every expert's weights, a few rows each
        _experts("experts-64-swiglu16", "swiglu16", 64),
        # one ordinary prompt of odd length over 32 experts, unevenly loaded
        _experts("experts-777-gelu32", "gelu32", 777, skew=0.5),
        # a large prefill batch (8 prompts of 2048)
        _experts("experts-16384-swiglu16", "swiglu16", 16384),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["route", "route", "quant", "linear", "linear", "experts", "experts", "experts"])
    if kind == "route":
        e, groups = rng.choice([(8, 1), (16, 1), (16, 4), (48, 1), (60, 6), (64, 8), (128, 1), (160, 8),
                                (256, 8), (256, 1)])
        top_groups = rng.randint(max(1, groups // 4), groups)
        k = rng.randint(1, min(8, top_groups * (e // groups)))
        c = _route("", _log_int(rng, 1, 16384), e, k, score=rng.choice(["softmax", "sigmoid"]),
                   dtype=rng.choice(["f32", "f32", "bf16"]), bias=rng.random() < 0.6, groups=groups,
                   top_groups=top_groups, renorm=rng.random() < 0.7,
                   scale=rng.choice([1.0, 2.5]), train=rng.random() < 0.5)
    elif kind == "quant":
        rows = _log_int(rng, 1, 16384)
        c = _quant("", rows, _log_int(rng, 64, 4096), block_rows=rng.choice([1, 1, 128]),
                   dtype=rng.choice(["bf16", "bf16", "f32"]))
    elif kind == "linear":
        k = rng.choice([256, 1000, 1024, 1408, 2048, 2816, _log_int(rng, 64, 2816)])
        n_out = rng.choice([256, 1024, 1408, 2048, 2800, 5632, _log_int(rng, 16, 5632)])
        most = min(16384, 16384 * 1024 * 5632 // (k * n_out))
        c = _linear("", _log_int(rng, 1, most), k, n_out, act=rng.choice(["none", "none", "gelu"]),
                    bias=rng.random() < 0.5)
    else:
        model = rng.choice(["swiglu16", "gelu32", "gelu64", "default", "ragged12"])
        most = 8192 if model == "gelu64" else 16384
        c = _experts("", model, rng.choice([_log_int(rng, 1, 64), _log_int(rng, 65, most)]),
                     skew=round(rng.uniform(0.0, 0.6), 2))
    c.pop("name", None)
    return c


# ----------------------------------------------------------------- inputs ----
def _blocks_of(n):
    return -(-n // BLOCK)


def _weight(gen, groups, rows, cols):
    """Codes [groups, rows, cols] and scales [groups, row blocks, col blocks] of N(0, 0.02)
    weights: what a loaded checkpoint holds."""
    w = torch.randn(groups, rows, cols, generator=gen, device="cuda") * 0.02
    rb, cb = _blocks_of(rows), _blocks_of(cols)
    p = torch.zeros(groups, rb * BLOCK, cb * BLOCK, device="cuda")
    p[:, :rows, :cols] = w
    amax = p.view(groups, rb, BLOCK, cb, BLOCK).abs().amax(dim=(2, 4))
    scale = (amax / FP8_MAX).clamp_min(1e-12)
    q = (w / _spread(scale, rows, cols)).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return q, scale


def _spread(scale, rows, cols, block_rows=BLOCK):
    """Each block's scale at every one of its elements."""
    s = scale.repeat_interleave(BLOCK, dim=-1)[..., :cols]
    return s.repeat_interleave(block_rows, dim=-2)[..., :rows, :] if block_rows > 1 else s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if kind == "route":
        n, e = case["N"], case["E"]
        # experts differ in how often they are wanted; the bias works against it
        tilt = normal(e) * 0.5
        st["logits"] = (normal(n, e) * 1.5 + tilt).to(DTYPES[case["dtype"]])
        st["balance"] = -0.05 * tilt if case["bias"] else None
        st["d_weights"] = normal(n, case["K"])
        st["logits"].requires_grad_(case["train"])
    elif kind == "quant":
        # rows and a few columns of other magnitudes, as hidden states have them
        x = normal(case["rows"], case["cols"]) * torch.exp(normal(case["rows"], 1))
        x[:, ::97] *= 20.0
        st["x"] = x.to(DTYPES[case["dtype"]])
    elif kind == "linear":
        st["x"] = normal(case["N"], case["K"]).to(torch.bfloat16)
        q, s = _weight(gen, 1, case["N_out"], case["K"])
        st["codes"], st["scale"] = _rows_of_16(q[0]), s[0]
        st["b"] = normal(case["N_out"]) * 0.1 if case["bias"] else None
    else:
        m = MODELS[case["model"]]
        e, h, u, k, n = m["E"], m["H"], m["U"], m["K"], case["tokens"]
        halves = 2 if m["act"] == "swiglu" else 1
        st.update(m)
        st["x"] = normal(n, 1, h).to(torch.bfloat16)
        # gate and up projections are matrices of their own: neither shares a block with the other
        q, s = _weight(gen, e * halves, u, h)
        st["w_up"] = q.view(e, halves * u, h)
        st["s_up"] = s.view(e, halves * _blocks_of(u), _blocks_of(h))
        st["w_down"], st["s_down"] = _weight(gen, e, h, u)
        st["b_up"] = normal(e, u) * 0.1 if m["act"] == "gelu" else None
        st["b_down"] = normal(e, h) * 0.1 if m["act"] == "gelu" else None
        # the routing a router hands on: k distinct experts, weights that add up to 1
        z = normal(n, 1, e) + normal(e) * case["skew"]
        z, idx = torch.topk(z, k, dim=-1)
        st["idx"], st["w"] = idx.to(torch.int32), torch.softmax(z, dim=-1)
    if own:
        _handles(st)
    return st


def _rows_of_16(q):
    """The codes with rows that start 16 bytes apart or a multiple of it, as
    quantize_fp8_blocks lays them out."""
    rows, cols = q.shape
    p = torch.zeros(rows, -(-cols // 16) * 16, dtype=torch.uint8, device=q.device)
    p[:, :cols] = q.view(torch.uint8)
    return p.view(torch.float8_e4m3fn)[:, :cols]


def _handles(st):
    """What a program keeps between its calls: the Forge pillars, and the experts' weights as one
    object."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "spider-web-moe_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import spider_moe_amd as smoe
    st["smoe"] = smoe
    if st["kind"] == "route":
        st["select"] = smoe.ForgeSelect()
    elif st["kind"] == "linear":
        st["gemm"] = smoe.ForgeGEMM()
    elif st["kind"] == "experts":
        st["experts"] = smoe.Fp8BlockExperts(st["w_up"], st["s_up"], st["w_down"], st["s_down"],
                                             b_up=st["b_up"], b_down=st["b_down"],
                                             activation=st["act"])


# ------------------------------------------------------------------- runs ----
def run(st):
    kind = st["kind"]
    if kind == "route":
        return _run_route(st) if own else _plain_route(st)
    if kind == "quant":
        if own:
            return st["smoe"].quantize_fp8_blocks(st["x"], block_rows=st["block_rows"])
        return _plain_quant(st["x"], st["block_rows"])
    act = None if st.get("act") == "none" else st["act"]
    if kind == "linear":
        if own:
            return st["gemm"].linear_fp8_blocks(st["x"], st["codes"], st["scale"], st["b"], act=act)
        return _plain_linear(st["x"], st["codes"], st["scale"], st["b"], act)
    if own:
        return st["smoe"].sparse_expert_delta_fp8_blocks(st["x"], st["idx"], st["w"], st["experts"])
    return _plain_experts(st)


def _run_route(st):
    w, idx = st["select"].route_groups(st["logits"], top_k=st["K"], score=st["score"],
                                       bias=st["balance"], num_groups=st["groups"],
                                       top_groups=st["top_groups"], renormalize=st["renorm"],
                                       scale=st["scale"])
    if not st["train"]:
        return w, idx
    (d,) = torch.autograd.grad(w, st["logits"], st["d_weights"])
    return w.detach(), idx, d


def _plain_route(st):
    """In 64 bits: which of two near scores is the larger decides whole outputs."""
    n, e, k, g = st["N"], st["E"], st["K"], st["groups"]
    z = st["logits"].detach().double()
    if st["score"] == "softmax":
        s = torch.exp(z - z.amax(dim=-1, keepdim=True))
        s = s / s.sum(dim=-1, keepdim=True)
    else:
        s = 1.0 / (1.0 + torch.exp(-z))
    c = s if st["balance"] is None else s + st["balance"].double()
    if g > 1:
        best = torch.sort(c.view(n, g, e // g), dim=-1, descending=True).values[..., :2].sum(dim=-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, :st["top_groups"]]
        open_ = torch.zeros(n, g, dtype=torch.bool, device=z.device).scatter_(1, kept, True)
        c = torch.where(open_.repeat_interleave(e // g, dim=1), c, float("-inf"))
    idx = torch.sort(c, dim=-1, descending=True, stable=True).indices[:, :k]
    chosen = s.gather(1, idx)
    total = chosen.sum(dim=-1, keepdim=True).clamp_min(1e-9) if st["renorm"] else 1.0
    w = (st["scale"] * chosen / total).float()
    if not st["train"]:
        return w, idx.to(torch.int32)
    d = st["d_weights"].double()
    if st["renorm"]:
        d = (d - (d * chosen / total).sum(dim=-1, keepdim=True)) / total
    ds = torch.zeros_like(s).scatter_(1, idx, st["scale"] * d)
    if st["score"] == "softmax":
        dz = s * (ds - (s * ds).sum(dim=-1, keepdim=True))
    else:
        dz = ds * s * (1.0 - s)
    return w, idx.to(torch.int32), dz.to(st["logits"].dtype)


def _plain_quant(x, block_rows):
    """The division in 64 bits, rounded to 32: the quotient of a 32-bit division, whose neighbours
    are other codes."""
    rows, cols = x.shape[-2:]
    lead = x.shape[:-2]
    rb, cb = -(-rows // block_rows), _blocks_of(cols)
    p = torch.zeros(*lead, rb * block_rows, cb * BLOCK, dtype=torch.float32, device=x.device)
    p[..., :rows, :cols] = x.float()
    amax = p.view(*lead, rb, block_rows, cb, BLOCK).abs().amax(dim=(-3, -1))
    scale = (amax.double() / FP8_MAX).float().clamp_min(1e-12)
    full = _spread(scale, rows, cols, block_rows)
    return (x.double() / full.double()).float().to(torch.float8_e4m3fn), scale


def _plain_values(q, scale, block_rows=BLOCK):
    return q.float() * _spread(scale, q.shape[-2], q.shape[-1], block_rows)


def _plain_gelu(y):
    return 0.5 * y * (1.0 + torch.erf(y * math.sqrt(0.5)))


def _plain_linear(x, codes, scale, b, act):
    y = _plain_values(*_plain_quant(x, 1), 1) @ _plain_values(codes, scale).t()
    if b is not None:
        y = y + b
    return (_plain_gelu(y) if act == "gelu" else y).to(x.dtype)


def _plain_experts(st):
    """Each expert's tokens side by side, padded to the fullest expert: two batched products over
    the experts that have tokens."""
    n, k, e, h, u = st["x"].shape[0], st["K"], st["E"], st["H"], st["U"]
    x = _plain_values(*_plain_quant(st["x"].view(n, h), 1), 1)
    flat = st["idx"].view(-1).long()
    count = torch.bincount(flat, minlength=e)
    order = torch.sort(flat, stable=True).indices
    first = torch.cumsum(count, 0) - count
    here = torch.nonzero(count).view(-1)
    place = torch.full((e,), -1, dtype=torch.long, device=x.device)
    place[here] = torch.arange(here.numel(), device=x.device)
    most = int(count.max())
    ge = flat[order]
    slot = place[ge] * most + torch.arange(n * k, device=x.device) - first[ge]
    rows = torch.zeros(here.numel() * most, h, device=x.device)
    rows[slot] = x[order // k]
    halves = 2 if st["act"] == "swiglu" else 1
    up = _plain_values(st["w_up"].view(torch.uint8).view(e, halves, u, h)[here].view(torch.float8_e4m3fn),
                       st["s_up"].view(e, halves, -1, st["s_up"].shape[-1])[here])
    y = torch.bmm(rows.view(here.numel(), most, h), up.view(here.numel(), halves * u, h).transpose(1, 2))
    if halves == 2:
        gate, y = y[..., :u], y[..., u:]
        y = y * gate / (1.0 + torch.exp(-gate))
    else:
        y = _plain_gelu(y + st["b_up"][here].unsqueeze(1))
    y = _plain_values(*_plain_quant(y.reshape(-1, u), 1), 1).view(here.numel(), most, u)
    down = _plain_values(st["w_down"].view(torch.uint8)[here].view(torch.float8_e4m3fn), st["s_down"][here])
    y = torch.bmm(y, down.transpose(1, 2))
    if st["b_down"] is not None:
        y = y + st["b_down"][here].unsqueeze(1)
    back = torch.empty_like(slot)
    back[order] = slot
    y = y.view(-1, h)[back].view(n, k, h) * st["w"].view(n, k, 1)
    return y.sum(dim=1).to(st["x"].dtype).view_as(st["x"])


# ------------------------------------------------------------------- work ----
def work(case):
    if case["kind"] == "route":
        n, e, k = case["N"], case["E"], case["K"]
        b = 2 if case["dtype"] == "bf16" else 4
        moved = n * e * b + n * k * 8 + (e * 4 if case["bias"] else 0)
        if case["train"]:  # the gradient of every logit, from that of the weights
            moved += n * k * 4 + n * e * b
        return {"bytes": moved, "flops": n * e * (12 if case["train"] else 6)}
    if case["kind"] == "quant":
        r, c = case["rows"], case["cols"]
        b = 2 if case["dtype"] == "bf16" else 4
        return {"bytes": r * c * (b + 1) + -(-r // case["block_rows"]) * _blocks_of(c) * 4,
                "flops": 3 * r * c}
    if case["kind"] == "linear":
        n, k, o = case["N"], case["K"], case["N_out"]
        return {"bytes": 2 * n * (k + o) + o * k + _blocks_of(o) * _blocks_of(k) * 4,
                "flops": 2 * n * k * o}
    m = MODELS[case["model"]]
    n, e, k, h, u = case["tokens"], m["E"], m["K"], m["H"], m["U"]
    mats = 3 if m["act"] == "swiglu" else 2
    read = e * (1.0 - (1.0 - k / e) ** n)  # the experts that some token wants
    return {"bytes": read * mats * (h * u + _blocks_of(h) * _blocks_of(u) * 4) + 4 * n * h + 8 * n * k,
            "flops": 2.0 * n * k * mats * h * u}


# ------------------------------------------------------------------ exact ----
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "route":
        return _exact_route(st)
    if case["kind"] == "quant":
        q, s = _exact_quant(st["x"], case["block_rows"])
        return q, s
    if case["kind"] == "linear":
        y = _exact_product(st["x"].double(), st["codes"], st["scale"])
        if st["b"] is not None:
            y = y + st["b"].double()
        return torch.nn.functional.gelu(y) if case["act"] == "gelu" else y
    return _exact_experts(st)


def _exact_route(st):
    n, e, g = st["N"], st["E"], st["groups"]
    z = st["logits"].detach().double().requires_grad_(True)
    s = torch.softmax(z, dim=-1) if st["score"] == "softmax" else torch.sigmoid(z)
    with torch.no_grad():
        c = s.clone() if st["balance"] is None else s + st["balance"].double()
        per = c.reshape(n, g, e // g)
        value = torch.topk(per, min(2, e // g), dim=-1).values.sum(-1)
        per[_places(value) >= st["top_groups"]] = float("-inf")
        idx = torch.argsort(_places(per.reshape(n, e)), dim=-1)[:, :st["K"]]
    w = torch.gather(s, 1, idx)
    if st["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    w = w * st["scale"]
    if not st["train"]:
        return w.detach(), None
    (d,) = torch.autograd.grad(w, z, st["d_weights"].double())
    return w.detach(), None, d


def _places(c):
    """Each entry's place in its row: the larger ones, and equal ones before it, come first."""
    at = torch.arange(c.shape[-1], device=c.device)
    out = []
    for part in c.split(1024):
        a, b = part.unsqueeze(-1), part.unsqueeze(-2)
        out.append(((b > a) | ((b == a) & (at < at.unsqueeze(-1)))).sum(-1))
    return torch.cat(out)


def _exact_quant(x, block_rows):
    """Codes as values: the quotients of a 32-bit division (elements of few bits divide to values
    within its last place of halfway between two codes), rounded by hand to four significant bits."""
    x = x.detach().double()
    rows, cols = x.shape[-2:]
    p = torch.nn.functional.pad(x, (0, -cols % BLOCK, 0, -rows % block_rows))
    p = p.unflatten(-1, (-1, BLOCK)).unflatten(-3, (-1, block_rows))  # [.., rb, br, cb, 128]
    s = (p.abs().amax(dim=(-3, -1), keepdim=True) / FP8_MAX).float().double().clamp_min(1e-12)
    v = (p / s).float().double()
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0 ** EXPONENT_MIN))) - 3.0)
    v = (torch.round(v / step) * step).clamp(-FP8_MAX, FP8_MAX)
    v = v.flatten(-4, -3).flatten(-2, -1)[..., :rows, :cols]
    return v, s[..., 0, :, 0]


def _exact_values(codes, scale):
    o, k = codes.shape
    r = torch.arange(o, device=codes.device) // BLOCK
    c = torch.arange(k, device=codes.device) // BLOCK
    return codes.double() * scale.double()[r][:, c]


def _exact_product(x, codes, scale):
    q, s = _exact_quant(x, 1)
    c = torch.arange(x.shape[-1], device=x.device) // BLOCK
    return (q * s[:, c]) @ _exact_values(codes, scale).t()


def _exact_experts(st):
    n, h, u = st["x"].shape[0], st["H"], st["U"]
    x = st["x"].view(n, h).double()
    idx, w = st["idx"].view(n, -1), st["w"].view(n, -1).double()
    blocks = _blocks_of(u)
    out = torch.zeros(n, h, dtype=torch.float64, device=x.device)
    for e in range(st["E"]):
        at, j = torch.nonzero(idx == e, as_tuple=True)
        if not at.numel():
            continue
        if st["act"] == "swiglu":
            gate = _exact_product(x[at], st["w_up"][e, :u], st["s_up"][e, :blocks])
            y = _exact_product(x[at], st["w_up"][e, u:], st["s_up"][e, blocks:])
            y = torch.nn.functional.silu(gate) * y
        else:
            y = torch.nn.functional.gelu(_exact_product(x[at], st["w_up"][e], st["s_up"][e])
                                         + st["b_up"][e].double())
        y = _exact_product(y, st["w_down"][e], st["s_down"][e])
        if st["b_down"] is not None:
            y = y + st["b_down"][e].double()
        out.index_add_(0, at, y * w[at, j].unsqueeze(-1))
    return out.view_as(st["x"])
