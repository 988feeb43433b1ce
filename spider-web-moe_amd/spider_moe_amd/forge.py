"""Forge surfaces (spider_infer/forge/*) on the block's HIP kernels.

The reference's kernel fabric exposes three of the block's operations with
its own call surface and slightly different semantics (forge/select,
forge/gemm, forge/ep).  Here they run on libsmoe.so:

  ForgeSelect.route    top-k on the logits, softmax over the k values
                       (forge/select/api.py:28-40) -> smoe_select_topk
  ForgeGEMM.linear / linear_fp8 / expert_ffn, fp8_linear /
  fp8_expert_ffn       (forge/gemm/api.py:34-74, fp8.py:22-78,
                       triton_kernels.py:65-123) -> smoe_linear; fp8
                       weights use the reference's per-tensor scale
                       (quantize_fp8), cached per weight version;
                       quantize_input -> smoe_quantize_fp8_tensor +
                       smoe_linear_fp8fp8 (e4m3 x e4m3 MFMA)
  ForgeEP.dispatch_plan / run_dispatched_ffn / combine
                       (forge/ep/api.py:46-104) -> the dispatch plan
                       kernels, sparse_expert_delta, or an expert_fn
                       callback per assignment with the weighted combine
                       on the GPU (dispatch.dispatch_expert_ffn)

Beside them, without a counterpart in the reference:

  ForgeSelect.route_groups   softmax or sigmoid scores, a balance bias,
                       top-k within the best groups of experts, with its
                       gradient -> smoe_select_groups(_backward)
  ForgeSelect.balance_loss   how evenly the choices spread, with its gradient,
                       and the experts' counts -> smoe_balance_loss(_backward)
  ForgeGEMM.linear_fp8_blocks   fp8 with a scale per block of 128 ->
                       smoe_linear_fp8_blocks
  ForgeGEMM.linear_mxfp4   4-bit floats with a power of two per 32 ->
                       smoe_linear_mxfp4

One GPU: the cross-rank combine is the identity (no process group), as
the reference's combine_across_ranks is at world size 1.
"""
from __future__ import annotations

import ctypes
import math
from dataclasses import dataclass
from enum import Enum
from typing import Any, Callable

import torch
from torch.autograd import forward_ad

from . import _native as nat
from .dispatch import DispatchPlan, build_dispatch_plan, dispatch_expert_ffn
from .quant import FP8_BLOCK, MX_BLOCK, _as_bytes, _pitched, mx_pitches, quantize_fp8_per_tensor
from .sparse_experts import _expert_ids


class ForgeBackend(str, Enum):
    """forge/config.py:8-16; this build has one backend."""
    HIP = "hip"


@dataclass
class ForgeConfig:
    """The fields of forge/config.py:19-51 that these surfaces read."""
    gemm_fp8: bool = False
    ep_enabled: bool = True
    ep_async: bool = False
    select_top_k: int = 2
    select_top_dobu: int = 4

    def to_dict(self) -> dict:
        return {"gemm_fp8": self.gemm_fp8, "ep": self.ep_enabled, "ep_async": self.ep_async,
                "select_top_k": self.select_top_k, "select_top_dobu": self.select_top_dobu,
                "backend": ForgeBackend.HIP.value}


# ---------------------------------------------------------------- select ----
class ForgeSelect:
    """Router selection with explicit top_k (compute) vs top_dobu (the Dobu
    residency budget, reported, not used as k)."""

    def __init__(self, config: ForgeConfig | None = None):
        self.config = config or ForgeConfig()
        self.calls = 0

    @torch.no_grad()
    def route(self, logits: torch.Tensor, *, top_k: int | None = None):
        """logits [..., E] -> (top_weights, top_indices) [..., k]: top-k on
        the logits, softmax over the k values; weights in the logits'
        dtype (computed in fp32), indices int64 as torch.topk returns."""
        self.calls += 1
        e = logits.shape[-1]
        k = int(top_k if top_k is not None else self.config.select_top_k)
        k = max(1, min(k, e))
        return select_topk(logits, k, nat.SMOE_SELECT_TOPK_SOFTMAX)

    def route_groups(self, logits: torch.Tensor, *, top_k: int | None = None,
                     score: str = "sigmoid", bias: torch.Tensor | None = None,
                     num_groups: int = 1, top_groups: int = 1, renormalize: bool = True,
                     scale: float = 1.0):
        """logits [..., E] (float32, bfloat16 or float16) -> (weights float32,
        indices int32) [..., k], as the dispatch plan and the experts read
        them.

        s = softmax(logits) or sigmoid(logits); s + bias (bias [E], taken as
        float32, which evens out the experts' load) decides the choice, s alone the weights.
        With num_groups > 1 consecutive experts form groups, a group's value
        is the sum of its two largest s + bias, and only the top_groups best
        groups take part.  The k largest are chosen, ties to the lower index,
        and weigh scale * s, divided by the chosen scores' sum (at least 1e-9)
        with renormalize.  Experts whose logit is -inf are chosen last, with
        weight 0.

        Differentiable in logits, once and in reverse mode (the choice held
        fixed; the bias gets no gradient); a tangent of forward mode is
        refused."""
        self.calls += 1
        k = int(top_k if top_k is not None else self.config.select_top_k)
        return select_groups(logits, k, score=score, bias=bias, num_groups=num_groups,
                             top_groups=top_groups, renormalize=renormalize, scale=scale)

    def balance_loss(self, logits: torch.Tensor, top_indices: torch.Tensor, *, score: str = "softmax",
                     mask: torch.Tensor | None = None, per_sequence: bool = False):
        """(loss float32, counts int32 [.., E]) of a router's logits [.., E]
        (float32, bfloat16 or float16) and its choices top_indices [.., k]:

          p = softmax(logits), or sigmoid(logits) over its sum
          load_e = share of the choices that went to expert e
          loss = E * sum_e load_e * (mean over tokens of p_e)

        1 where both are even; the aux_loss of SpiderMoELayer's statistics
        (model.py:330-337) over all tokens.  mask [..] (bool, or 0 / 1): tokens
        that count; what the others' logits hold plays no part.  per_sequence:
        logits [.., T, E], a loss and counts for each sequence of T tokens
        (loss [..], counts [.., E]).  Ids outside [0, E) count nowhere; a
        sequence without tokens or choices has loss 0.  An expert with logit
        -inf has p = 0.

        Differentiable in logits, once and in reverse mode (the counts held
        fixed)."""
        self.calls += 1
        return balance_loss(logits, top_indices, score=score, mask=mask, per_sequence=per_sequence)

    def top_dobu_budget(self) -> int:
        return int(self.config.select_top_dobu)

    def stats(self) -> dict[str, Any]:
        return {"pillar": "select", "impl": "hip_select_topk", "backend": ForgeBackend.HIP.value,
                "calls": self.calls, "top_k": self.config.select_top_k,
                "top_dobu": self.config.select_top_dobu}


def select_topk(logits: torch.Tensor, k: int, mode: int):
    """smoe_select_topk over the last dimension (E <= 64)."""
    dev = nat.require_gpu(logits)
    e = logits.shape[-1]
    lead = logits.shape[:-1]
    x = logits.reshape(-1, e).to(torch.float32).contiguous()
    n = x.shape[0]
    w = torch.empty(n, k, dtype=torch.float32, device=dev)
    idx = torch.empty(n, k, dtype=torch.int32, device=dev)
    nat.check(nat.lib().smoe_select_topk(x.data_ptr(), n, e, k, mode, w.data_ptr(), idx.data_ptr(),
                                         nat.stream_of(dev)), "smoe_select_topk")
    out_dtype = logits.dtype if logits.dtype.is_floating_point else torch.float32
    return w.view(*lead, k).to(out_dtype), idx.view(*lead, k).long()


def _select_groups_fwd(x, n, e, idx, k, score, bias, num_groups, top_groups, renormalize, scale):
    """x: contiguous logits, n rows of e; fills idx, returns the weights."""
    w = torch.empty(idx.shape, dtype=torch.float32, device=x.device)
    nat.launch(x.device, "smoe_select_groups", x.data_ptr(), nat.float_code(x.dtype), n, e, k, score,
               None if bias is None else bias.data_ptr(), num_groups, top_groups, renormalize, scale,
               w.data_ptr(), idx.data_ptr())
    return w


class _SelectGroups(torch.autograd.Function):
    # idx is filled, not returned: a second output and its bookkeeping cost the
    # host 4 us of a step's 86
    @staticmethod
    def forward(ctx, logits, n, e, idx, how):
        x = logits.contiguous()
        ctx.save_for_backward(x, idx)
        ctx.how = n, e, how
        return _select_groups_fwd(x, n, e, idx, *how)

    @staticmethod
    def backward(ctx, d_w):
        if torch.is_grad_enabled():
            raise RuntimeError("route_groups is not twice differentiable")
        x, idx = ctx.saved_tensors
        n, e, (k, score, _, _, _, renormalize, scale) = ctx.how
        d = torch.empty_like(x)
        d_w = d_w.contiguous()
        nat.launch(x.device, "smoe_select_groups_backward", x.data_ptr(), nat.float_code(x.dtype), n, e, k,
                   score, renormalize, scale, idx.data_ptr(), d_w.data_ptr(), d.data_ptr())
        return d, None, None, None, None


def select_groups(logits: torch.Tensor, k: int, *, score: str = "sigmoid", bias=None,
                  num_groups: int = 1, top_groups: int = 1, renormalize: bool = True,
                  scale: float = 1.0):
    """smoe_select_groups over the last dimension (ForgeSelect.route_groups)."""
    dev = nat.require_gpu(logits, bias)
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise RuntimeError("route_groups has no forward-mode derivative")
    shape = logits.shape
    e = shape[-1] if shape else 0
    n = logits.numel() // e if e else 0
    if not shape or n > 0x7fffffff:
        raise ValueError(f"logits must be [.., E], got {tuple(shape)}")
    if score not in nat.SCORES:
        raise ValueError("score must be 'softmax' or 'sigmoid'")
    if bias is not None:
        if bias.shape != shape[-1:]:
            raise ValueError(f"bias must be [{e}], got {tuple(bias.shape)}")
        if bias.dtype != torch.float32:
            bias = bias.float()
        bias = bias.contiguous()
    idx = torch.empty((*shape[:-1], k), dtype=torch.int32, device=dev)
    how = (k, nat.SCORES[score], bias, num_groups, top_groups, renormalize, scale)
    if logits.requires_grad and torch.is_grad_enabled():
        return _SelectGroups.apply(logits, n, e, idx, how), idx
    return _select_groups_fwd(logits.contiguous(), n, e, idx, *how), idx


def _balance_fwd(x, idx, mask, how, slope):
    """x: contiguous logits of s sequences of t tokens -> (loss [s], counts [s, e])."""
    s, t, e, k, score = how
    dev = x.device
    loss = torch.empty(s, dtype=torch.float32, device=dev)
    counts = torch.empty(s, e, dtype=torch.int32, device=dev)
    need = nat.lib().smoe_balance_loss_workspace_bytes(s, t, e)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    nat.launch(dev, "smoe_balance_loss", x.data_ptr(), nat.float_code(x.dtype), s, t, e, k, score,
               idx.data_ptr(), nat.ptr(mask), loss.data_ptr(), counts.data_ptr(), nat.ptr(slope),
               nat.ptr(ws), need)
    return loss, counts


class _BalanceLoss(torch.autograd.Function):
    # the counts are kept on ctx's holder, not returned: no bookkeeping for them
    @staticmethod
    def forward(ctx, logits, idx, mask, how, shape, out):
        x = logits.contiguous()
        slope = torch.empty(how[0], how[2], dtype=torch.float32, device=x.device)
        loss, counts = _balance_fwd(x, idx, mask, how, slope)
        out.append(counts)
        ctx.save_for_backward(x, mask, slope)
        ctx.how = how
        return loss.view(shape)

    @staticmethod
    def backward(ctx, d_loss):
        if torch.is_grad_enabled():
            raise RuntimeError("balance_loss is not twice differentiable")
        x, mask, slope = ctx.saved_tensors
        s, t, e, _, score = ctx.how
        d = torch.empty_like(x)
        d_loss = d_loss.contiguous()
        nat.launch(x.device, "smoe_balance_loss_backward", x.data_ptr(), nat.float_code(x.dtype), s, t, e,
                   score, nat.ptr(mask), slope.data_ptr(), d_loss.data_ptr(), d.data_ptr())
        return d, None, None, None, None, None


def balance_loss(logits: torch.Tensor, top_indices: torch.Tensor, *, score: str = "softmax", mask=None,
                 per_sequence: bool = False):
    """smoe_balance_loss over the last dimension (ForgeSelect.balance_loss)."""
    nat.require_gpu(logits, top_indices, mask)
    if forward_ad.unpack_dual(logits).tangent is not None:
        raise RuntimeError("balance_loss has no forward-mode derivative")
    if score not in nat.SCORES:
        raise ValueError("score must be 'softmax' or 'sigmoid'")
    shape = logits.shape
    if len(shape) < (2 if per_sequence else 1):
        raise ValueError(f"logits must be [.., {'T, ' if per_sequence else ''}E], got {tuple(shape)}")
    if top_indices.ndim != len(shape) or top_indices.shape[:-1] != shape[:-1]:
        raise ValueError("top_indices must be logits' shape with k last")
    e, k = shape[-1], top_indices.shape[-1]
    lead = tuple(shape[:-2]) if per_sequence else ()
    s = math.prod(lead)
    t = shape[-2] if per_sequence else math.prod(shape[:-1])
    if mask is not None:
        if mask.shape != shape[:-1]:
            raise ValueError(f"mask must be {tuple(shape[:-1])}, got {tuple(mask.shape)}")
        mask = (mask if mask.dtype == torch.bool else mask != 0).contiguous()
    if max(s, t) > 0x7fffffff:
        raise ValueError("more than 2^31 - 1 tokens")
    idx = _expert_ids(top_indices, e).contiguous()
    how = (s, t, e, k, nat.SCORES[score])
    if logits.requires_grad and torch.is_grad_enabled():
        out = []
        loss = _BalanceLoss.apply(logits, idx, mask, how, lead, out)
        counts = out[0]
    else:
        loss, counts = _balance_fwd(logits.contiguous(), idx, mask, how, None)
        loss = loss.view(lead)
    return loss, counts.view(*lead, e)


# ------------------------------------------------------------------ gemm ----
_ACT = {None: 0, "gelu": 1}


def _linear(x: torch.Tensor, w: torch.Tensor, w_format: int, scale, bias, act, out_dtype):
    """smoe_linear: x [..., K] . w^T (+ bias, act) -> [..., N_out]."""
    dev = nat.require_gpu(x, w)
    k = x.shape[-1]
    lead = x.shape[:-1]
    xa = x.reshape(-1, k).to(torch.float32 if w_format == nat.F32 else torch.bfloat16).contiguous()
    n = xa.shape[0]
    n_out = w.shape[0]
    out = torch.empty(n, n_out, dtype=out_dtype, device=dev)
    b = None if bias is None else bias.detach().float().contiguous()
    nat.check(nat.lib().smoe_linear(xa.data_ptr(), n, k, w.data_ptr(), w_format, nat.ptr(scale),
                                    nat.ptr(b), n_out, _ACT[act], out.data_ptr(),
                                    nat.dtype_code(out_dtype), nat.stream_of(dev)), "smoe_linear")
    return out.view(*lead, n_out)


def _linear_fp8_blocks(x, codes, scale, bias, act):
    dev = nat.require_gpu(x, codes, scale, bias)
    k, lead = x.shape[-1], x.shape[:-1]
    if codes.dtype != torch.float8_e4m3fn or codes.ndim != 2 or codes.shape[1] != k:
        raise ValueError(f"codes must be float8_e4m3fn [N_out, {k}], got {codes.dtype} {tuple(codes.shape)}")
    n_out = codes.shape[0]
    if scale.dtype != torch.float32 or scale.shape != (-(-n_out // FP8_BLOCK), -(-k // FP8_BLOCK)):
        raise ValueError("scale must be float32 [ceil(N_out / 128), ceil(K / 128)], "
                         f"got {scale.dtype} {tuple(scale.shape)}")
    if act not in _ACT:
        raise ValueError("act must be None or 'gelu'")
    if max(k, n_out) > 0x7fffff00 or x.numel() > 0x7fffff00 * k:
        raise ValueError("more than 2^31 - 256 rows, K or N_out")
    if bias is not None:
        if bias.shape != (n_out,):
            raise ValueError(f"bias must be [{n_out}], got {tuple(bias.shape)}")
        bias = bias.float().contiguous()
    if x.ndim == 2 and x.stride(1) == 1 and x.stride(0) >= k:
        ldx = x.stride(0)
    else:
        x, ldx = x.contiguous(), k
    codes, ldw = _rows16(codes)
    scale = scale.contiguous()
    out_dtype = torch.bfloat16 if x.dtype == torch.bfloat16 else torch.float32
    out = torch.empty(*lead, n_out, dtype=out_dtype, device=dev)
    n = out.numel() // n_out if n_out else 0
    lib = nat.lib()
    need = lib.smoe_linear_fp8_blocks_workspace_bytes(n, k)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    nat.launch(dev, "smoe_linear_fp8_blocks", x.data_ptr(), nat.float_code(x.dtype), ldx, None, n, k,
               codes.data_ptr(), ldw, scale.data_ptr(), nat.ptr(bias), n_out, _ACT[act],
               out.data_ptr(), nat.dtype_code(out_dtype), nat.ptr(ws), need)
    return out if out_dtype == x.dtype else out.to(x.dtype)


def _rows16(codes):
    """Codes [rows, cols] in rows that start a multiple of 16 bytes apart,
    each whole in memory, and that distance: the tensor itself where it is
    laid out so, else a copy."""
    rows, cols = codes.shape
    ld = codes.stride(0) if rows > 1 else -(-cols // 16) * 16
    if (codes.stride(1) == 1 or cols == 1) and ld >= cols and ld % 16 == 0 and \
            codes.data_ptr() % 16 == 0 and (cols % 16 == 0 or codes.untyped_storage().nbytes() -
                                            codes.storage_offset() >= rows * ld):
        return codes, ld
    ld = -(-cols // 16) * 16
    c = torch.zeros(rows, ld, dtype=torch.uint8, device=codes.device)
    c[:, :cols] = codes.view(torch.uint8)
    return c, ld


def _linear_mxfp4(x, codes, scale, bias, act):
    dev = nat.require_gpu(x, codes, scale, bias)
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("x must be [.., K] with K >= 1")
    k, lead = x.shape[-1], x.shape[:-1]
    codes, scale = _as_bytes(codes, "codes"), _as_bytes(scale, "scale")
    if codes.ndim != 2 or codes.shape[1] != -(-k // 2):
        raise ValueError(f"codes must be [N_out, {-(-k // 2)}], got {tuple(codes.shape)}")
    n_out = codes.shape[0]
    if scale.shape != (n_out, -(-k // MX_BLOCK)):
        raise ValueError(f"scale must be {(n_out, -(-k // MX_BLOCK))}, got {tuple(scale.shape)}")
    if act not in _ACT:
        raise ValueError("act must be None or 'gelu'")
    if max(k, n_out) > 0x7fffff00 or x.numel() > 0x7fffff00 * k:
        raise ValueError("more than 2^31 - 256 rows, K or N_out")
    if bias is not None:
        if bias.shape != (n_out,):
            raise ValueError(f"bias must be [{n_out}], got {tuple(bias.shape)}")
        bias = bias.float().contiguous()
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise RuntimeError(f"unsupported activation dtype {x.dtype} (float32, bfloat16 or float16)")
    if x.ndim == 2 and x.stride(1) == 1 and x.stride(0) >= k:
        ldx = x.stride(0)
    else:
        x, ldx = x.contiguous(), k
    ldc, lds = mx_pitches(k)
    codes, ldw = _pitched(codes, ldc, 16, most=1 << 22)
    scale, ld_ws = _pitched(scale, lds, 4)
    out_dtype = torch.bfloat16 if x.dtype == torch.bfloat16 else torch.float32
    out = torch.empty(*lead, n_out, dtype=out_dtype, device=dev)
    n = out.numel() // n_out if n_out else 0
    if n:
        need = nat.lib().smoe_linear_mxfp4_workspace_bytes(n, k, n_out)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
        nat.launch(dev, "smoe_linear_mxfp4", x.data_ptr(), nat.float_code(x.dtype), ldx, n, k,
                   codes.data_ptr(), ldw, scale.data_ptr(), ld_ws, nat.ptr(bias), n_out, _ACT[act],
                   out.data_ptr(), nat.dtype_code(out_dtype), nat.ptr(ws), need)
    return out if out_dtype == x.dtype else out.to(x.dtype)


class _Fp8Cache:
    """Per-tensor fp8 codes of a weight, re-quantized when the weight
    changes (the reference quantizes on every call, fp8.py:46), in the
    forms the kernels read: the codes [N_out, K] with the scale repeated per
    channel (weight-only GEMM), the codes zero-padded to K % 256 == 0 with
    the scale as one f32 (fp8 x fp8 GEMM), and the dequantized f32 weight
    codes * scale (fp32 inputs, which the reference multiplies in fp32)."""

    def __init__(self):
        self._c: dict = {}

    def _entry(self, w: torch.Tensor) -> dict:
        key = (w.data_ptr(), w._version, tuple(w.shape), w.dtype)
        hit = self._c.get(id(w))
        if hit is not None and hit[0] == key:
            return hit[1]
        codes, scale = quantize_fp8_per_tensor(w)
        ent = {"codes": codes.view(torch.uint8), "scale": scale.reshape(1).to(w.device)}
        self._c[id(w)] = (key, ent)
        return ent

    def get(self, w: torch.Tensor):
        ent = self._entry(w)
        if "scale_vec" not in ent:
            ent["scale_vec"] = ent["scale"].expand(w.shape[0]).contiguous()
        return ent["codes"], ent["scale_vec"]

    def get_padded(self, w: torch.Tensor):
        ent = self._entry(w)
        if "padded" not in ent:
            k = w.shape[1]
            kp = -(-k // 256) * 256
            pad = torch.zeros(w.shape[0], kp, dtype=torch.uint8, device=w.device)
            pad[:, :k] = ent["codes"]
            ent["padded"] = pad
        return ent["padded"], ent["scale"]

    def get_dequant(self, w: torch.Tensor):
        ent = self._entry(w)
        if "deq" not in ent:
            ent["deq"] = (ent["codes"].view(torch.float8_e4m3fn).float() * ent["scale"]).contiguous()
        return ent["deq"]


def quantize_fp8_input(x: torch.Tensor, k_pad: int):
    """Per-tensor e4m3 codes of x [..., K] on the device (smoe_quantize_fp8_tensor:
    quant.py:30-56's scale and round-to-nearest-even cast) as [rows, k_pad]
    u8 with zero codes past K, and the scale (f32 [1])."""
    dev = nat.require_gpu(x)
    k = x.shape[-1]
    xa = x.reshape(-1, k)
    if xa.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        xa = xa.float()
    xa = xa.contiguous()
    rows = xa.shape[0]
    codes = torch.empty(rows, k_pad, dtype=torch.uint8, device=dev)
    scale = torch.empty(1, dtype=torch.float32, device=dev)
    lib = nat.lib()
    ws = torch.empty(lib.smoe_quantize_fp8_workspace_bytes(), dtype=torch.uint8, device=dev)
    code = nat.F16 if xa.dtype == torch.float16 else nat.dtype_code(xa.dtype)
    nat.check(lib.smoe_quantize_fp8_tensor(xa.data_ptr(), code, rows, k, k_pad, 0,
                                           codes.data_ptr(), scale.data_ptr(), ws.data_ptr(),
                                           ws.numel(), nat.stream_of(dev)),
              "smoe_quantize_fp8_tensor")
    return codes, scale


class ForgeGEMM:
    """ForgeGEMM (forge/gemm/api.py:22-87) on the block's GEMM kernels.

    linear: x . w^T + b in fp32 on the values of x / w (bf16 inputs run
    the bf16 MFMA path with fp32 accumulation, f32 inputs the fp32 path),
    result in x's dtype.  With config.gemm_fp8 (or linear_fp8) the weight is
    quantized to e4m3 with one per-tensor scale (quantize_fp8): bf16 / f16
    inputs run the GEMM on the codes (activations read as bf16, the scale
    in the epilogue), f32 inputs the fp32 GEMM on the dequantized weight
    (the reference's fp32 compute dtype, fp8.py:41-54).  quantize_input:
    x is quantized per tensor too (smoe_quantize_fp8_tensor) and the GEMM
    multiplies e4m3 by e4m3 (smoe_linear_fp8fp8, the f8f6f4 MFMA), both
    scales applied in f32.  expert_ffn: linear, GELU (erf), linear."""

    def __init__(self, config: ForgeConfig | None = None):
        self.config = config or ForgeConfig()
        self.calls = 0
        self._fp8 = _Fp8Cache()
        self.last_fp8_backend = "not_run"

    def _run(self, x, w, bias, act, fp8, quantize_input=False):
        """fp8: e4m3 weight codes; else fp32 when x or w is fp32 (exact
        products of their values), bf16 x bf16 otherwise."""
        if fp8 and quantize_input:
            return self._run_fp8fp8(x, w, bias, act)
        if fp8 and x.dtype == torch.float32:
            wt, fmt, scale = self._fp8.get_dequant(w), nat.F32, None
            self.last_fp8_backend = "hip_fp8_weight_dequant_f32"
        elif fp8:
            wt, scale = self._fp8.get(w)
            fmt = nat.FP8_E4M3
            self.last_fp8_backend = "hip_fp8_weight_bf16_mfma"
        elif x.dtype == torch.float32 or w.dtype == torch.float32:
            wt, fmt, scale = w.detach().float().contiguous(), nat.F32, None
        else:
            wt, fmt, scale = w.detach().to(torch.bfloat16).contiguous(), nat.BF16, None
        out_dtype = torch.float32 if (act is None or fmt == nat.F32) else torch.bfloat16
        return _linear(x, wt, fmt, scale, bias, act, out_dtype)

    def _run_fp8fp8(self, x, w, bias, act):
        dev = nat.require_gpu(x, w)
        wq, ws = self._fp8.get_padded(w)
        k_pad = wq.shape[1]
        xq, xs = quantize_fp8_input(x, k_pad)
        n, n_out = xq.shape[0], wq.shape[0]
        out_dtype = torch.bfloat16 if (act is not None and x.dtype != torch.float32) else torch.float32
        out = torch.empty(n, n_out, dtype=out_dtype, device=dev)
        b = None if bias is None else bias.detach().float().contiguous()
        nat.check(nat.lib().smoe_linear_fp8fp8(xq.data_ptr(), xs.data_ptr(), n, k_pad, wq.data_ptr(),
                                               ws.data_ptr(), nat.ptr(b), n_out, _ACT[act],
                                               out.data_ptr(), nat.dtype_code(out_dtype),
                                               nat.stream_of(dev)), "smoe_linear_fp8fp8")
        self.last_fp8_backend = "hip_fp8xfp8_mfma_f8f6f4"
        return out.view(*x.shape[:-1], n_out)

    @torch.no_grad()
    def linear(self, x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None):
        self.calls += 1
        return self._run(x, weight, bias, None, self.config.gemm_fp8).to(x.dtype)

    @torch.no_grad()
    def linear_fp8(self, x, weight, bias=None, *, quantize_input: bool = False):
        """Explicit fp8 path regardless of config.gemm_fp8 (fp8.py:22-62)."""
        self.calls += 1
        return self._run(x, weight, bias, None, True, quantize_input).to(x.dtype)

    def linear_fp8_blocks(self, x, codes, scale, bias=None, *, act: str | None = None):
        """act(x . W^T + bias) with W held as e4m3 codes [N_out, K] and one
        scale per 128 x 128 block (quantize_fp8_blocks), x [..., K] quantized
        in 1 x 128 blocks on the way (smoe_linear_fp8_blocks); act None or
        "gelu" (erf).  Result in x's dtype: bfloat16 from e4m3 x e4m3
        products, each cut by less than 2^-13 of the largest of its eight
        neighbours; float32 (and float16) from the same values' products with
        f32 sums throughout.  No gradient."""
        self.calls += 1
        return _linear_fp8_blocks(x, codes, scale, bias, act)

    def linear_mxfp4(self, x, codes, scale, bias=None, *, act: str | None = None):
        """act(x . W^T + bias) with W held as quantize_mxfp4 gives it: e2m1
        codes [N_out, ceil(K / 2)] and a power of two per 32 along K
        [N_out, ceil(K / 32)]; x [..., K] is quantized the same way on the way
        (smoe_linear_mxfp4).  act None or "gelu" (erf).  Products of the two
        operands' values, summed in f32; result in x's dtype.  No gradient."""
        self.calls += 1
        return _linear_mxfp4(x, codes, scale, bias, act)

    @torch.no_grad()
    def expert_ffn(self, x, w_up, b_up, w_down, b_down):
        self.calls += 1
        fp8 = self.config.gemm_fp8
        h = self._run(x, w_up, b_up, "gelu", fp8)
        return self._run(h.to(x.dtype), w_down, b_down, None, fp8).to(x.dtype)

    @torch.no_grad()
    def fp8_expert_ffn(self, x, w_up, b_up, w_down, b_down, *, quantize_input: bool = False):
        """fp8.py:65-76: the up projection (input quantized when asked) with
        its GELU, then the down projection on fp8 weights only."""
        self.calls += 1
        h = self._run(x, w_up, b_up, "gelu", True, quantize_input)
        return self._run(h.to(x.dtype), w_down, b_down, None, True).to(x.dtype)

    def stats(self) -> dict[str, Any]:
        return {"pillar": "gemm", "impl": "hip_grouped_gemm", "backend": ForgeBackend.HIP.value,
                "calls": self.calls, "fp8": self.config.gemm_fp8,
                "last_fp8_kernel": self.last_fp8_backend}


_FP8_GEMM = None


def _fp8_gemm() -> "ForgeGEMM":
    global _FP8_GEMM
    if _FP8_GEMM is None:
        _FP8_GEMM = ForgeGEMM(ForgeConfig(gemm_fp8=True))
    return _FP8_GEMM


def fp8_linear(x, weight, bias=None, *, quantize_input: bool = False, compute_dtype=None):
    """forge/gemm/fp8.py:22-62 on the HIP kernels: per-tensor e4m3 weights
    (and, with quantize_input, activations); F.linear's shape, result in
    x's dtype.  compute_dtype is accepted for the reference's signature:
    the kernels accumulate in f32 whatever it says."""
    return _fp8_gemm().linear_fp8(x, weight, bias, quantize_input=quantize_input)


def fp8_expert_ffn(x, w_up, b_up, w_down, b_down, *, quantize_input: bool = False):
    """forge/gemm/fp8.py:65-76 on the HIP kernels."""
    return _fp8_gemm().fp8_expert_ffn(x, w_up, b_up, w_down, b_down, quantize_input=quantize_input)


def get_last_fp8_gemm_backend():
    """(kernel, error) of the last fp8 call (fp8.py:79-80); errors raise
    here instead of falling back."""
    return _fp8_gemm().last_fp8_backend, None


# -------------------------------------------------------------------- ep ----
class ForgeEP:
    """Token dispatch + combine (forge/ep/api.py:21-117) at world size 1."""

    def __init__(self, config: ForgeConfig | None = None):
        self.config = config or ForgeConfig()
        self.calls = 0

    def enabled(self) -> bool:
        return False  # one GPU: no expert-parallel group

    def rank_world(self) -> tuple[int, int]:
        return 0, 1

    def owns(self, expert_id: int) -> bool:
        return True  # expert_id % 1 == 0 (expert_parallel.py:29)

    def combine(self, delta: torch.Tensor) -> torch.Tensor:
        self.calls += 1
        return delta

    def dispatch_meta(self, top_indices: torch.Tensor, num_experts: int) -> dict:
        self.calls += 1
        plan = build_dispatch_plan(top_indices, torch.ones_like(top_indices, dtype=torch.float32),
                                   num_experts=num_experts, local_only=True)
        return {"rank": 0, "world": 1, "local_experts": plan.local_expert_ids,
                "assignments": len(plan.assignments), "top_indices_shape": list(top_indices.shape)}

    def dispatch_plan(self, top_indices, top_weights, num_experts: int) -> DispatchPlan:
        self.calls += 1
        return build_dispatch_plan(top_indices, top_weights, num_experts=num_experts,
                                   local_only=True)

    def run_dispatched_ffn(self, messages, top_indices, top_weights, *, w_up, b_up, w_down,
                           b_down, num_experts: int, expert_fn: Callable | None = None):
        self.calls += 1
        return dispatch_expert_ffn(messages, top_indices, top_weights, w_up=w_up, b_up=b_up,
                                   w_down=w_down, b_down=b_down, num_experts=num_experts,
                                   expert_fn=expert_fn)

    def stats(self) -> dict[str, Any]:
        return {"pillar": "ep", "impl": "hip_dispatch_plan", "backend": ForgeBackend.HIP.value,
                "calls": self.calls, "rank": 0, "world": 1, "async": self.config.ep_async}


# --------------------------------------------------------------- runtime ----
class ForgeRuntime:
    """The object init_forge returns (forge/registry.py:20-56): the pillars
    this build provides."""

    def __init__(self, config: ForgeConfig | None = None):
        self.config = config or ForgeConfig()
        self.select = ForgeSelect(self.config)
        self.gemm = ForgeGEMM(self.config)
        self.ep = ForgeEP(self.config)

    def stats(self) -> dict[str, Any]:
        return {"config": self.config.to_dict(), "select": self.select.stats(),
                "gemm": self.gemm.stats(), "ep": self.ep.stats()}


_RUNTIME: ForgeRuntime | None = None


def init_forge(config: ForgeConfig | None = None) -> ForgeRuntime:
    """forge/registry.py:58-88."""
    global _RUNTIME
    _RUNTIME = ForgeRuntime(config)
    return _RUNTIME


def get_forge() -> ForgeRuntime:
    """forge/registry.py:91-95: the runtime, created with defaults on first use."""
    return _RUNTIME if _RUNTIME is not None else init_forge()


__all__ = ["ForgeBackend", "ForgeConfig", "ForgeSelect", "ForgeGEMM", "ForgeEP", "ForgeRuntime",
           "init_forge", "get_forge", "select_topk", "select_groups", "balance_loss", "fp8_linear", "fp8_expert_ffn",
           "get_last_fp8_gemm_backend", "quantize_fp8_input"]
