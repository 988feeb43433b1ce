"""Routed experts on microscaled 4-bit weights and the router's balance, as measurable cases.

Four operators, which a mixture-of-experts step runs together:

  balance  ForgeSelect.balance_loss: how evenly a router spreads its tokens,
           E * sum_e load_e * P_e with the tokens each expert got and its mean
           score, over the whole batch or sequence by sequence, padding left
           out; the counts, and the gradient in the logits
  quant    quantize_mxfp4 and dequantize_mxfp4: blocks of 32 values as e2m1
           codes (4 bits) with one power of two, and the values they stand for
  linear   ForgeGEMM.linear_mxfp4: activations quantized in such blocks on the
           way, times weights held in them
  experts  sparse_expert_delta_mxfp4: dispatch, both products of every token's
           experts on such weights, and the weighted combine

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

BLOCK = 32
CODE_MAX = 6.0    # of e2m1
CODE_EXP = 2      # exponent of its largest values
SCALE_EXP = 127   # bias, and largest exponent, of a block's power of two
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)

# The expert shapes of the framework's benchmark and of its default
# ModelConfig, and one whose sizes are multiples of 32 but of no larger tile.
MODELS = {
    "swiglu16": dict(H=1024, E=16, K=2, U=2816, act="swiglu"),
    "gelu32": dict(H=1024, E=32, K=4, U=1408, act="gelu"),
    "gelu64": dict(H=2048, E=64, K=2, U=1408, act="gelu"),
    "default": dict(H=256, E=8, K=2, U=512, act="gelu"),
    "ragged12": dict(H=544, E=12, K=3, U=1184, act="swiglu"),
}
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ cases ----
def _balance(name, seqs, tokens, e, k, *, score, dtype="f32", padded=False, per_sequence=False,
             train=True):
    return {"name": name, "kind": "balance", "B": seqs, "T": tokens, "E": e, "K": k, "score": score,
            "dtype": dtype, "padded": padded, "per_sequence": per_sequence, "train": train}


def _quant(name, rows, cols, *, dtype="bf16"):
    return {"name": name, "kind": "quant", "rows": rows, "cols": cols, "dtype": dtype}


def _linear(name, n, k, n_out, *, act="none", bias=False, dtype="bf16"):
    return {"name": name, "kind": "linear", "N": n, "K": k, "N_out": n_out, "act": act, "bias": bias,
            "dtype": dtype}


def _experts(name, model, tokens, *, skew=0.0, dtype="bf16"):
    return {"name": name, "kind": "experts", "model": model, "tokens": tokens, "skew": skew,
            "dtype": dtype}


def listed():
    return [
        # the load of a decode batch over a small model's experts, watched while it serves: latency
        _balance("balance-1x64-softmax-8", 1, 64, 8, 2, score="softmax", train=False),
        # a padded batch of odd length, bf16 logits, the whole batch's loss with its gradient
        _balance("balance-4x777-softmax-64-train", 4, 777, 64, 2, score="softmax", dtype="bf16",
                 padded=True),
        # a large training step over 256 experts, balanced sequence by sequence, with the gradient
        _balance("balance-8x2048-sigmoid-256-train", 8, 2048, 256, 8, score="sigmoid",
                 per_sequence=True),
        # the activations of an ordinary prompt with rows that end inside a block
        _quant("quant-777x1000", 777, 1000),
        # a stack of 16 experts' down projections when a model is loaded, and what it then holds
        _quant("quant-weights-16384x2816", 16384, 2816),
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
    kind = rng.choice(["balance", "balance", "quant", "linear", "linear", "experts", "experts", "experts"])
    if kind == "balance":
        e = rng.choice([8, 16, 48, 60, 64, 128, 160, 256])
        seqs = _log_int(rng, 1, 16)
        c = _balance("", seqs, _log_int(rng, 1, 16384 // seqs), e, rng.randint(1, min(8, e)),
                     score=rng.choice(["softmax", "sigmoid"]), dtype=rng.choice(["f32", "f32", "bf16"]),
                     padded=rng.random() < 0.5, per_sequence=rng.random() < 0.5,
                     train=rng.random() < 0.7)
    elif kind == "quant":
        c = _quant("", _log_int(rng, 1, 16384), _log_int(rng, 1, 2816),
                   dtype=rng.choice(["bf16", "bf16", "f32"]))
    elif kind == "linear":
        k = rng.choice([256, 1000, 1024, 1408, 2048, 2816, _log_int(rng, 16, 2816)])
        n_out = rng.choice([256, 1024, 1408, 2048, 2800, 5632, _log_int(rng, 16, 5632)])
        most = min(16384, 16384 * 1024 * 5632 // (k * n_out))
        c = _linear("", _log_int(rng, 1, most), k, n_out, act=rng.choice(["none", "none", "gelu"]),
                    bias=rng.random() < 0.5, dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))
    else:
        model = rng.choice(["swiglu16", "gelu32", "gelu64", "default", "ragged12"])
        most = 8192 if model == "gelu64" else 16384
        c = _experts("", model, rng.choice([_log_int(rng, 1, 64), _log_int(rng, 65, most)]),
                     skew=round(rng.uniform(0.0, 0.6), 2),
                     dtype=rng.choice(["bf16", "bf16", "bf16", "f32"]))
    c.pop("name", None)
    return c


# ----------------------------------------------------------------- inputs ----
def _blocks_of(n):
    return -(-n // BLOCK)


def _in_blocks(x):
    """[.., blocks, 32], the last block filled up with zeros."""
    cols = x.shape[-1]
    p = torch.zeros(*x.shape[:-1], _blocks_of(cols) * BLOCK, dtype=x.dtype, device=x.device)
    p[..., :cols] = x
    return p.view(*x.shape[:-1], -1, BLOCK)


def _plain_codes(x):
    """Nibbles 0 .. 15 [.., blocks, 32] and biased scale exponents [.., blocks] of float32 x: the
    exponent of the block's largest magnitude less 2, and the nearest of the sixteen values, ties
    to the even code."""
    p = _in_blocks(x)
    exponent = (p.abs().amax(dim=-1).view(torch.int32) >> 23) - CODE_EXP
    exponent = exponent.clamp_min(0)
    v = p.double().abs() * torch.exp2((SCALE_EXP - exponent).double()).unsqueeze(-1)
    code = torch.zeros_like(p, dtype=torch.int32)
    for i in range(1, len(CODES)):
        middle = 0.5 * (CODES[i - 1] + CODES[i])
        code += (v > middle) | ((v == middle) & (i % 2 == 0))
    return torch.where(torch.signbit(p), code + 8, code), exponent


def _plain_pack(x):
    """Codes two a byte (the first in the low half) [.., ceil(cols / 2)], whose rows lie a multiple
    of 16 bytes apart, and scale bytes [.., blocks], whose rows lie a multiple of 4 apart: as
    quantize_mxfp4 lays them out."""
    code, exponent = _plain_codes(x.float())
    code = code.to(torch.uint8).flatten(-2)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    blocks = exponent.shape[-1]
    scale = torch.full((*exponent.shape[:-1], -(-blocks // 4) * 4), SCALE_EXP, dtype=torch.uint8,
                       device=x.device)
    scale[..., :blocks] = exponent.to(torch.uint8)
    return packed[..., :-(-x.shape[-1] // 2)], scale[..., :blocks]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    kind = case["kind"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if kind == "balance":
        b, t, e, k = case["B"], case["T"], case["E"], case["K"]
        # experts differ in how often they are wanted, and so do they from text to text
        z = normal(b, t, e) * 1.5 + normal(b, 1, e) * 0.3 + normal(e) * 0.5
        z = z.to(DTYPES[case["dtype"]])
        st["idx"] = torch.topk(z.float(), k, dim=-1).indices.to(torch.int32)
        st["mask"] = None
        if case["padded"]:  # texts of any length, behind them padding; now and then none at all
            length = torch.rand(b, generator=gen, device="cuda") * (t + 1)
            if b > 2:
                length[torch.randint(b, (1,), generator=gen, device="cuda")] = 0
            st["mask"] = torch.arange(t, device="cuda") < length.long().unsqueeze(1)
        st["logits"] = z.requires_grad_(case["train"])
        # what the rest of a step makes of the loss: its coefficient, over the sequences
        st["d_loss"] = 0.01 + 0.001 * normal(b) if case["per_sequence"] else 0.01 + 0.001 * normal()
    elif kind == "quant":
        # rows and a few columns of other magnitudes, as hidden states have them
        x = normal(case["rows"], case["cols"]) * torch.exp(normal(case["rows"], 1))
        x[:, ::97] *= 20.0
        st["x"] = x.to(DTYPES[case["dtype"]])
    elif kind == "linear":
        st["x"] = normal(case["N"], case["K"]).to(DTYPES[case["dtype"]])
        st["codes"], st["scale"] = _plain_pack(normal(case["N_out"], case["K"]) * 0.02)
        st["b"] = normal(case["N_out"]) * 0.1 if case["bias"] else None
    else:
        m = MODELS[case["model"]]
        e, h, u, k, n = m["E"], m["H"], m["U"], m["K"], case["tokens"]
        halves = 2 if m["act"] == "swiglu" else 1
        st.update(m)
        st["x"] = normal(n, 1, h).to(DTYPES[case["dtype"]])
        up = [_plain_pack(normal(halves * u, h) * 0.02) for _ in range(e)]
        down = [_plain_pack(normal(h, u) * 0.02) for _ in range(e)]
        st["w_up"], st["s_up"] = (torch.stack(t) for t in zip(*up))
        st["w_down"], st["s_down"] = (torch.stack(t) for t in zip(*down))
        st["b_up"] = normal(e, u) * 0.1 if m["act"] == "gelu" else None
        st["b_down"] = normal(e, h) * 0.1 if m["act"] == "gelu" else None
        # the routing a router hands on: k distinct experts, weights that add up to 1
        z = normal(n, 1, e) + normal(e) * case["skew"]
        z, idx = torch.topk(z, k, dim=-1)
        st["idx"], st["w"] = idx.to(torch.int32), torch.softmax(z, dim=-1)
    if own:
        _handles(st)
    return st


def _handles(st):
    """What a program keeps between its calls: the Forge pillars, and the experts' weights as one
    object."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "spider-web-moe_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import spider_moe_amd as smoe
    st["smoe"] = smoe
    if st["kind"] == "balance":
        st["select"] = smoe.ForgeSelect()
    elif st["kind"] == "linear":
        st["gemm"] = smoe.ForgeGEMM()
    elif st["kind"] == "experts":
        st["experts"] = smoe.MxFp4Experts(st["w_up"], st["s_up"], st["w_down"], st["s_down"],
                                          b_up=st["b_up"], b_down=st["b_down"],
                                          activation=st["act"])


# ------------------------------------------------------------------- runs ----
def run(st):
    kind = st["kind"]
    if kind == "balance":
        return _run_balance(st) if own else _plain_balance(st)
    if kind == "quant":
        if own:
            codes, scale = st["smoe"].quantize_mxfp4(st["x"])
            return st["smoe"].dequantize_mxfp4(codes, scale, cols=st["cols"], dtype=torch.bfloat16), scale
        codes, scale = _plain_pack(st["x"])
        return _plain_values(codes, scale, st["cols"]).to(torch.bfloat16), scale
    act = None if st.get("act") == "none" else st["act"]
    if kind == "linear":
        if own:
            return st["gemm"].linear_mxfp4(st["x"], st["codes"], st["scale"], st["b"], act=act)
        return _plain_linear(st["x"], st["codes"], st["scale"], st["b"], act)
    if own:
        return st["smoe"].sparse_expert_delta_mxfp4(st["x"], st["idx"], st["w"], st["experts"])
    return _plain_experts(st)


def _run_balance(st):
    loss, counts = st["select"].balance_loss(st["logits"], st["idx"], score=st["score"], mask=st["mask"],
                                             per_sequence=st["per_sequence"])
    if not st["train"]:
        return loss, counts
    (d,) = torch.autograd.grad(loss, st["logits"], st["d_loss"])
    return loss.detach(), counts, d


def _plain_balance(st):
    """Sums over the tokens in 64 bits: there are thousands of them."""
    b, t, e = st["B"], st["T"], st["E"]
    z = st["logits"].detach().float()
    here = torch.ones(b, t, device=z.device) if st["mask"] is None else st["mask"].float()
    # sigmoid: its logarithm, so that the shares of far negative logits still add up
    s = z if st["score"] == "softmax" else torch.clamp_max(z, 0.0) - torch.log1p(torch.exp(-z.abs()))
    p = torch.exp(s - s.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True) * here.unsqueeze(-1)
    hot = torch.zeros(b, t, e, device=z.device).scatter_add_(
        2, st["idx"].long(), torch.ones(st["idx"].shape, device=z.device))
    hot = hot * here.unsqueeze(-1)
    dims = (1,) if st["per_sequence"] else (0, 1)
    n = here.sum(dim=dims).clamp_min(1.0).double()
    counts = hot.double().sum(dim=dims)
    load = counts / counts.sum(dim=-1, keepdim=True).clamp_min(1.0)
    mean = p.double().sum(dim=dims) / n.unsqueeze(-1)
    loss = (e * (load * mean).sum(dim=-1)).float()
    counts = counts.to(torch.int32)
    if not st["train"]:
        return loss, counts
    g = (e * load * (st["d_loss"].double() / n).unsqueeze(-1)).float()
    g = g.view(b, 1, e) if st["per_sequence"] else g.view(1, 1, e)
    d = p * (g - (p * g).sum(dim=-1, keepdim=True))
    if st["score"] == "sigmoid":
        d = d / (1.0 + torch.exp(z))
    return loss, counts, d.to(st["logits"].dtype)


def _plain_values(codes, scale, cols):
    """What codes [.., ceil(cols / 2)] and scale [.., blocks] stand for, in float32."""
    table = torch.tensor(CODES + tuple(-c for c in CODES), device=codes.device)
    nibbles = torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)[..., :cols]
    two = torch.ldexp(torch.ones((), dtype=torch.float64, device=codes.device),
                      scale.int() - SCALE_EXP).float()
    return table[nibbles.long()] * two.repeat_interleave(BLOCK, dim=-1)[..., :cols]


def _plain_round(x):
    """x as the values that its codes stand for."""
    codes, scale = _plain_pack(x)
    return _plain_values(codes, scale, x.shape[-1])


def _plain_gelu(y):
    """With erf's complement for negative y: 1 + erf(y) would lose what a block of small values is
    measured by."""
    return 0.5 * y * torch.where(y < 0, torch.special.erfc(-y * math.sqrt(0.5)),
                                 1.0 + torch.erf(y * math.sqrt(0.5)))


def _plain_linear(x, codes, scale, b, act):
    y = _plain_round(x.float()) @ _plain_values(codes, scale, x.shape[-1]).t()
    if b is not None:
        y = y + b
    return (_plain_gelu(y) if act == "gelu" else y).to(x.dtype)


def _plain_experts(st):
    """Each expert's tokens side by side, padded to the fullest expert: two batched products over
    the experts that have tokens."""
    n, k, e, h, u = st["x"].shape[0], st["K"], st["E"], st["H"], st["U"]
    x = _plain_round(st["x"].view(n, h).float())
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
    up = _plain_values(st["w_up"][here], st["s_up"][here], h)
    y = torch.bmm(rows.view(here.numel(), most, h), up.transpose(1, 2).contiguous())
    if st["act"] == "swiglu":
        gate, y = y[..., :u], y[..., u:]
        y = y * gate / (1.0 + torch.exp(-gate))
    else:
        y = _plain_gelu(y + st["b_up"][here].unsqueeze(1))
    y = _plain_round(y)
    down = _plain_values(st["w_down"][here], st["s_down"][here], u)
    y = torch.bmm(y, down.transpose(1, 2).contiguous())
    if st["b_down"] is not None:
        y = y + st["b_down"][here].unsqueeze(1)
    back = torch.empty_like(slot)
    back[order] = slot
    y = y.view(-1, h)[back].view(n, k, h) * st["w"].view(n, k, 1)
    return y.sum(dim=1).to(st["x"].dtype).view_as(st["x"])


# ------------------------------------------------------------------- work ----
def work(case):
    b = 2 if case.get("dtype") == "bf16" else 4
    if case["kind"] == "balance":
        n, e, k = case["B"] * case["T"], case["E"], case["K"]
        moved = n * e * b + n * k * 4 + (n if case["padded"] else 0)
        if case["train"]:  # the gradient of every logit
            moved += n * e * b
        return {"bytes": moved, "flops": n * e * (12 if case["train"] else 6)}
    if case["kind"] == "quant":
        r, c = case["rows"], case["cols"]
        return {"bytes": r * c * (b + 2) + r * _blocks_of(c), "flops": 3 * r * c}
    if case["kind"] == "linear":
        n, k, o = case["N"], case["K"], case["N_out"]
        return {"bytes": b * n * (k + o) + o * (k / 2 + _blocks_of(k)) + (4 * o if case["bias"] else 0),
                "flops": 2 * n * k * o}
    m = MODELS[case["model"]]
    n, e, k, h, u = case["tokens"], m["E"], m["K"], m["H"], m["U"]
    mats = 3 if m["act"] == "swiglu" else 2
    read = e * (1.0 - (1.0 - k / e) ** n)  # the experts that some token wants
    return {"bytes": read * mats * h * u * (1 / 2 + 1 / BLOCK) + 2 * b * n * h + 8 * n * k,
            "flops": 2.0 * n * k * mats * h * u}


# ------------------------------------------------------------------ exact ----
def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "balance":
        return _exact_balance(st)
    if case["kind"] == "quant":
        return _exact_round(st["x"].double()), None
    if case["kind"] == "linear":
        y = _exact_round(st["x"].double()) @ _exact_values(st["codes"], st["scale"], case["K"]).t()
        if st["b"] is not None:
            y = y + st["b"].double()
        return torch.nn.functional.gelu(y) if case["act"] == "gelu" else y
    return _exact_experts(st)


def _exact_balance(st):
    z = st["logits"].detach().double().requires_grad_(True)
    e = st["E"]
    s = torch.softmax(z if st["score"] == "softmax" else torch.nn.functional.logsigmoid(z), dim=-1)
    total = []
    for i in range(st["B"]):
        at = slice(None) if st["mask"] is None else st["mask"][i]
        total.append((s[i][at].sum(0), torch.bincount(st["idx"][i][at].flatten().long(), minlength=e),
                      s[i][at].shape[0]))
    if not st["per_sequence"]:
        total = [tuple(sum(part) for part in zip(*total))]
    loss = torch.stack([e * (p * c).sum() / max(int(c.sum()), 1) / max(n, 1) for p, c, n in total])
    if not st["per_sequence"]:
        loss = loss[0]
    if not st["train"]:
        return loss.detach(), None
    (d,) = torch.autograd.grad(loss, z, st["d_loss"].double())
    return loss.detach(), None, d


def _exact_round(x):
    """x (in 64 bits) as the values of its codes: quotients rounded by hand to one significant bit
    behind the leading one."""
    cols = x.shape[-1]
    p = torch.nn.functional.pad(x, (0, -cols % BLOCK)).unflatten(-1, (-1, BLOCK))
    power = torch.frexp(p.abs().amax(dim=-1, keepdim=True)).exponent - 1 - CODE_EXP
    two = torch.exp2(power.clamp(-SCALE_EXP, SCALE_EXP).double())
    v = p / two
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(1.0, CODE_MAX))) - 1.0)
    v = (torch.round(v / step) * step).clamp(-CODE_MAX, CODE_MAX)
    return (v * two).flatten(-2)[..., :cols]


def _exact_values(codes, scale, cols):
    low, high = (codes % 16).double(), (codes // 16).double()
    c = torch.stack([low, high], dim=-1).flatten(-2)[..., :cols]
    sign, c = 1.0 - 2.0 * (c >= 8), c % 8
    v = torch.where(c < 2, c / 2, torch.exp2(torch.floor(c / 2) - 1.0) * (1.0 + (c % 2) / 2))
    at = torch.arange(cols, device=codes.device) // BLOCK
    return sign * v * torch.exp2(scale.double() - SCALE_EXP)[..., at]


def _exact_experts(st):
    n, h, u = st["x"].shape[0], st["H"], st["U"]
    x = _exact_round(st["x"].view(n, h).double())
    idx, w = st["idx"].view(n, -1), st["w"].view(n, -1).double()
    out = torch.zeros(n, h, dtype=torch.float64, device=x.device)
    for e in range(st["E"]):
        at, j = torch.nonzero(idx == e, as_tuple=True)
        if not at.numel():
            continue
        y = x[at] @ _exact_values(st["w_up"][e], st["s_up"][e], h).t()
        if st["act"] == "swiglu":
            y = torch.nn.functional.silu(y[:, :u]) * y[:, u:]
        else:
            y = torch.nn.functional.gelu(y + st["b_up"][e].double())
        y = _exact_round(y) @ _exact_values(st["w_down"][e], st["s_down"][e], u).t()
        if st["b_down"] is not None:
            y = y + st["b_down"][e].double()
        out.index_add_(0, at, y * w[at, j].unsqueeze(-1))
    return out.view_as(st["x"])
