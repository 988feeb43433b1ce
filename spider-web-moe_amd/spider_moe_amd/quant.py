"""Expert weight formats (host-side packing; runs once, not per call).

int4: spider_moe/quant.py:76-143 — same function names, argument meaning and
bytes: symmetric per-group along the last dim, scale = max(amax, 1e-8) / 7,
q = clamp(round_half_even(w / scale), -8, 7), element 2i in the low nibble.
``scale_dtype=torch.float16`` stores the (identical) scales as fp16 — the
layout of the int4 decode/prefill configuration; the packed bytes do not
change.

fp8: per-output-channel e4m3 — scale = max(amax_K / 448, 1e-12) and
codes = (w / scale).to(float8_e4m3fn), as quantize_fp8_with_scale_tensor
(quant.py:146-158) with a [.., N] scale; dequant = code * scale
(quant.py:161-169).

fp8 in blocks: e4m3 codes with one f32 scale per 128 x 128 block of a weight
or per 1 x 128 block of activations (no counterpart in the reference):
quantize_fp8_blocks / dequantize_fp8_blocks.

microscaled 4-bit floating point (OCP MXFP4, no counterpart in the reference):
e2m1 codes with one power of two per 32 elements of a row: quantize_mxfp4 /
dequantize_mxfp4.
"""
from __future__ import annotations

import math
from dataclasses import dataclass

import torch

FP8_E4M3_MAX = 448.0


@dataclass
class Int4Tensor:
    """Packed INT4 weights with per-group scales (quant.py:76-86)."""

    packed: torch.Tensor
    scales: torch.Tensor
    shape: tuple
    group_size: int

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        return dequantize_int4(self.packed, self.scales, self.shape, self.group_size, dtype=dtype)


def quantize_int4(weight: torch.Tensor, group_size: int = 64,
                  scale_dtype: torch.dtype = torch.float32) -> Int4Tensor:
    """quant.py:89-117 (plus an optional fp16 scale storage)."""
    if weight.ndim < 1:
        raise ValueError("weight must be at least 1D")
    *lead, n = weight.shape
    if n % 2 != 0:
        raise ValueError("last dimension must be even for INT4 packing")
    if group_size <= 0 or n % group_size != 0:
        group_size = n
    g = group_size
    w = weight.detach().float().reshape(-1, n // g, g)
    scales = w.abs().amax(dim=-1).clamp_min(1e-8) / 7.0
    q = torch.round(w / scales.unsqueeze(-1)).clamp(-8, 7).to(torch.int8).reshape(-1, n)
    lo = (q[:, 0::2] & 0x0F).to(torch.uint8)
    hi = (q[:, 1::2] & 0x0F).to(torch.uint8)
    packed = (lo | (hi << 4)).reshape(*lead, n // 2).contiguous()
    return Int4Tensor(packed=packed, scales=scales.to(scale_dtype).reshape(*lead, n // g).contiguous(),
                      shape=tuple(weight.shape), group_size=g)


def dequantize_int4(packed, scales, shape, group_size, dtype=None):
    """quant.py:120-143."""
    *lead, half = packed.shape
    n = half * 2
    flat = packed.reshape(-1, half)
    lo = (flat & 0x0F).to(torch.int8)
    hi = ((flat >> 4) & 0x0F).to(torch.int8)
    lo = torch.where(lo >= 8, lo - 16, lo)
    hi = torch.where(hi >= 8, hi - 16, hi)
    q = torch.empty(flat.shape[0], n, device=packed.device, dtype=torch.int8)
    q[:, 0::2] = lo
    q[:, 1::2] = hi
    g = group_size
    w = (q.view(q.shape[0], n // g, g).float() * scales.float().reshape(q.shape[0], n // g, 1))
    w = w.view(*lead, n)
    if dtype is not None:
        w = w.to(dtype)
    return w.view(shape)


def _quantize_fp8_device(weight: torch.Tensor, per_row: bool):
    """smoe_quantize_fp8_tensor: the reference's scale and cast with IEEE
    divisions, the bits torch computes on the CPU (torch's GPU kernels
    divide by a reciprocal: an ulp off in the scale and, rarely, one code
    step off)."""
    from . import _native as nat
    w = weight.detach()
    if w.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        w = w.float()
    w = w.contiguous()
    k = w.shape[-1]
    rows = w.numel() // k if k else 0
    kp = -(-k // 4) * 4
    codes = torch.empty(rows, kp, dtype=torch.uint8, device=w.device)
    scale = torch.empty(rows if per_row else 1, dtype=torch.float32, device=w.device)
    lib = nat.lib()
    wsp = None if per_row else torch.empty(lib.smoe_quantize_fp8_workspace_bytes(),
                                           dtype=torch.uint8, device=w.device)
    code = nat.F16 if w.dtype == torch.float16 else nat.dtype_code(w.dtype)
    with torch.cuda.device(w.device):
        nat.check(lib.smoe_quantize_fp8_tensor(w.data_ptr(), code, rows, k, kp, int(per_row),
                                               codes.data_ptr(), scale.data_ptr(), nat.ptr(wsp),
                                               0 if wsp is None else wsp.numel(),
                                               nat.stream_of(w.device)),
                  "smoe_quantize_fp8_tensor")
    if kp != k:
        codes = codes[:, :k].contiguous()
    return codes.view(torch.float8_e4m3fn).view(w.shape), scale


def quantize_fp8_per_channel(weight: torch.Tensor):
    """[..., N, K] -> (float8_e4m3fn codes [..., N, K], float32 scale [..., N]).
    On a GPU: the HIP quantizer (same bits as the CPU formula)."""
    if weight.is_cuda and weight.numel():
        codes, scale = _quantize_fp8_device(weight, per_row=True)
        return codes, scale.view(weight.shape[:-1])
    w = weight.detach().float()
    scale = (w.abs().amax(dim=-1) / FP8_E4M3_MAX).clamp_min(1e-12)
    codes = (w / scale.unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes.contiguous(), scale.contiguous()


def dequantize_fp8_per_channel(codes: torch.Tensor, scale: torch.Tensor,
                               dtype: torch.dtype = torch.float32) -> torch.Tensor:
    return (codes.float() * scale.float().unsqueeze(-1)).to(dtype)


def quantize_fp8_per_tensor(weight: torch.Tensor):
    """One scale for the whole tensor, the format of the reference's
    quantize_fp8 / compute_fp8_scale (quant.py:30-56): scale = max(amax / 448,
    1e-12) (fp32, a 0-dim tensor), codes = (w.float() / scale) cast to
    float8_e4m3fn (round to nearest even).  On a GPU: the HIP quantizer
    (same bits as the CPU formula)."""
    if weight.is_cuda and weight.numel():
        codes, scale = _quantize_fp8_device(weight, per_row=False)
        return codes, scale.reshape(())
    w = weight.detach().float()
    scale = (w.abs().amax() / FP8_E4M3_MAX).clamp_min(1e-12)
    return (w / scale).to(torch.float8_e4m3fn).contiguous(), scale


# ------------------------------------------------------- fp8 in blocks ----
FP8_BLOCK = 128


def _row_stride(x: torch.Tensor):
    """Elements between rows when x [.., rows, cols] is rows of contiguous
    elements at one distance throughout, else None."""
    if x.ndim < 2 or (x.shape[-1] > 1 and x.stride(-1) != 1):
        return None
    ld = x.stride(-2) if x.shape[-2] > 1 else x.shape[-1]
    if x.shape[-2] == 1 and x.ndim > 2:  # the rows of the leading dimension
        for n, st in zip(reversed(x.shape[:-2]), reversed(x.stride()[:-2])):
            if n > 1:
                ld = st
                break
    step = ld * x.shape[-2]
    for n, st in zip(reversed(x.shape[:-2]), reversed(x.stride()[:-2])):
        if n > 1 and st != step:
            return None
        step *= n
    return ld if ld >= x.shape[-1] else None


def quantize_fp8_blocks(x: torch.Tensor, *, block_rows: int = FP8_BLOCK):
    """x [.., rows, cols] -> (float8_e4m3fn codes of that shape, float32 scale
    [.., ceil(rows / block_rows), ceil(cols / 128)]): one scale for each block
    of block_rows x 128 elements, block_rows 128 (weights) or 1 (activations).
    scale = max(amax|block| / 448, 1e-12), code = x / scale rounded to nearest
    even, both divisions in f32 (a NaN makes its block's scale and codes NaN).
    The codes' rows start a multiple of 16 bytes apart, as the GEMMs read
    them (a view where cols % 16 != 0).  On a GPU: the HIP quantizer (same
    bits as the CPU formula)."""
    if block_rows not in (1, FP8_BLOCK):
        raise ValueError("block_rows must be 1 or 128")
    if x.ndim < 2 or x.shape[-1] < 1:
        raise ValueError("x must be [.., rows, cols] with cols >= 1")
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        x = x.float()
    *lead, rows, cols = x.shape
    cb, ld = -(-cols // FP8_BLOCK), -(-cols // 16) * 16
    rb = -(-rows // block_rows)
    if x.is_cuda:
        from . import _native as nat
        ldx = cols if x.is_contiguous() else _row_stride(x)
        if ldx is None:
            x, ldx = x.contiguous(), cols
        g = math.prod(lead)
        if max(g, rows, cols) > 0x7fffffff:
            raise ValueError("more than 2^31 - 1 rows, columns or matrices")
        codes = torch.empty(*lead, rows, ld, dtype=torch.float8_e4m3fn, device=x.device)
        scale = torch.empty(*lead, rb, cb, dtype=torch.float32, device=x.device)
        nat.launch(x.device, "smoe_quantize_fp8_blocks", x.data_ptr(), nat.float_code(x.dtype), g, rows,
                   cols, ldx, block_rows, codes.data_ptr(), ld, scale.data_ptr())
        return (codes if ld == cols else codes.narrow(-1, 0, cols)), scale
    x = x.detach()
    p = torch.zeros(*lead, rb * block_rows, cb * FP8_BLOCK)
    p[..., :rows, :cols] = x
    p = p.view(*lead, rb, block_rows, cb, FP8_BLOCK)
    scale = (p.abs().amax(dim=(-3, -1)) / FP8_E4M3_MAX).clamp_min(1e-12)
    q = (p / scale[..., :, None, :, None]).view(*lead, rb * block_rows, cb * FP8_BLOCK)
    codes = torch.zeros(*lead, rows, ld, dtype=torch.uint8)
    codes[..., :cols] = q[..., :rows, :cols].to(torch.float8_e4m3fn).view(torch.uint8)
    return codes.view(torch.float8_e4m3fn)[..., :cols], scale


def dequantize_fp8_blocks(codes: torch.Tensor, scale: torch.Tensor, *, block_rows: int = FP8_BLOCK,
                          dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """code * scale of its block, in f32, as dtype."""
    rows, cols = codes.shape[-2:]
    if scale.shape != (*codes.shape[:-2], -(-rows // block_rows), -(-cols // FP8_BLOCK)):
        raise ValueError("scale does not match the codes' blocks")
    s = scale.float().repeat_interleave(FP8_BLOCK, dim=-1)[..., :cols]
    if block_rows > 1:
        s = s.repeat_interleave(block_rows, dim=-2)[..., :rows, :]
    return (codes.float() * s).to(dtype)


# -------------------------------------------- microscaled 4-bit floats ----
MX_BLOCK = 32
_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_BYTES = tuple(getattr(torch, n) for n in ("uint8", "float4_e2m1fn_x2", "float8_e8m0fnu") if hasattr(torch, n))


def _as_bytes(t: torch.Tensor, name: str) -> torch.Tensor:
    """Codes or scales as uint8, whichever of torch's names for them they
    carry."""
    if t.dtype not in _BYTES:
        raise ValueError(f"{name} must be uint8 (or float4_e2m1fn_x2 codes, float8_e8m0fnu scales), got {t.dtype}")
    return t if t.dtype == torch.uint8 else t.view(torch.uint8)


def mx_pitches(cols: int):
    """Bytes from row to row that the kernels want at least: codes (whole
    blocks) and scales (whole words)."""
    nb = -(-cols // MX_BLOCK)
    return 16 * nb, -(-nb // 4) * 4


def _pitched(t: torch.Tensor, pitch: int, align: int, most: int | None = None):
    """t [rows, n] bytes with rows `ld` apart, ld a multiple of `align`, at most
    `most`, and every row's `pitch` bytes inside the storage: t itself, else a
    copy.  Returns it and ld."""
    rows, n = t.shape
    ld = t.stride(0) if rows > 1 else pitch
    if (t.stride(1) == 1 or n == 1) and pitch <= ld <= (most or ld) and ld % align == 0 and t.data_ptr() % align == 0 and \
            t.untyped_storage().nbytes() - t.storage_offset() >= (rows - 1) * ld + pitch:
        return t, ld
    c = torch.zeros(rows, pitch, dtype=torch.uint8, device=t.device)
    c[:, :n] = t
    return c[:, :n], pitch


def _flat_rows(t: torch.Tensor):
    """t [.., n] as (tensor, elements from row to row): t itself where its rows
    lie at one distance, else a contiguous copy."""
    t2 = t if t.ndim > 1 else t.unsqueeze(0)
    ld = t2.shape[-1] if t2.is_contiguous() else _row_stride(t2)
    return (t2, ld) if ld is not None else (t2.contiguous(), t2.shape[-1])


def quantize_mxfp4(x: torch.Tensor):
    """x [.., cols] -> (codes uint8 [.., ceil(cols / 2)], scale uint8
    [.., ceil(cols / 32)]): blocks of 32 along the last dimension (the last one
    may be shorter), each a power of two 2^(scale - 127) = 2^(floor(log2 amax)
    - 2), at least 2^-127, times e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a
    sign) rounded to nearest even, past 6 to 6; element 2i in the low half of
    byte i.  An infinity or a NaN makes its block NaN (scale 255, codes 0).
    The codes' rows start a multiple of 16 bytes apart and the scales' a
    multiple of 4, as the products read them (views where cols does not fill
    them).  On a GPU: the HIP quantizer (same bits as the CPU formula)."""
    if x.ndim < 1 or x.shape[-1] < 1:
        raise ValueError("x must be [.., cols] with cols >= 1")
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        x = x.float()
    *lead, cols = x.shape
    nb = -(-cols // MX_BLOCK)
    ldc, lds = mx_pitches(cols)
    if x.is_cuda:
        from . import _native as nat
        rows = math.prod(lead)
        if max(rows, cols) > 0x7fffffff:
            raise ValueError("more than 2^31 - 1 rows or columns")
        x, ldx = _flat_rows(x)
        codes = torch.empty(*lead, ldc, dtype=torch.uint8, device=x.device)
        scale = torch.empty(*lead, lds, dtype=torch.uint8, device=x.device)
        nat.launch(x.device, "smoe_quantize_mxfp4", x.data_ptr(), nat.float_code(x.dtype), rows, cols, ldx,
                   codes.data_ptr(), ldc, scale.data_ptr(), lds)
    else:
        p = torch.zeros(*lead, nb * MX_BLOCK)
        p[..., :cols] = x.detach()
        p = p.view(*lead, nb, MX_BLOCK)
        biased = p.abs().amax(dim=-1).view(torch.int32) >> 23  # NaN is the largest magnitude
        biased = torch.where(torch.isfinite(p).all(dim=-1), (biased - 2).clamp_min(0), 255)
        v = p.double().abs() * torch.exp2(127.0 - biased.double()).unsqueeze(-1)
        c = torch.zeros(p.shape, dtype=torch.uint8)
        for i in range(1, 8):  # a tie goes to the even code
            middle = (_E2M1[i - 1] + _E2M1[i]) / 2
            c += (v >= middle) if i % 2 == 0 else (v > middle)
        c = torch.where(biased.unsqueeze(-1) == 255, 0, c + 8 * torch.signbit(p).to(torch.uint8))
        c = c.to(torch.uint8).view(*lead, -1)
        codes = c[..., 0::2] | (c[..., 1::2] << 4)
        scale = torch.zeros(*lead, lds, dtype=torch.uint8)
        scale[..., :nb] = biased.to(torch.uint8)
    if ldc != -(-cols // 2):
        codes = codes.narrow(-1, 0, -(-cols // 2))
    return codes, (scale if lds == nb else scale.narrow(-1, 0, nb))


def dequantize_mxfp4(codes: torch.Tensor, scale: torch.Tensor, *, cols: int | None = None,
                     dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """The values [.., cols] of quantize_mxfp4's codes and scale, as dtype
    (float32 and bfloat16 hold them exactly); cols: 2 * codes.shape[-1] by
    default, one less where the last byte holds one code."""
    codes, scale = _as_bytes(codes, "codes"), _as_bytes(scale, "scale")
    if codes.ndim < 1 or codes.shape[-1] < 1:
        raise ValueError("codes must be [.., ceil(cols / 2)] with cols >= 1")
    cols = 2 * codes.shape[-1] if cols is None else int(cols)
    lead = codes.shape[:-1]
    if codes.shape[-1] != -(-cols // 2):
        raise ValueError(f"{cols} columns take {-(-cols // 2)} bytes of codes, got {codes.shape[-1]}")
    if scale.shape != (*lead, -(-cols // MX_BLOCK)):
        raise ValueError(f"scale must be {(*lead, -(-cols // MX_BLOCK))}, got {tuple(scale.shape)}")
    if codes.is_cuda:
        from . import _native as nat
        nat.require_gpu(codes, scale)
        rows = math.prod(lead)
        if max(rows, cols) > 0x7fffffff:
            raise ValueError("more than 2^31 - 1 rows or columns")
        out = torch.empty(*lead, cols, device=codes.device,
                          dtype=dtype if dtype in (torch.float32, torch.bfloat16, torch.float16) else torch.float32)
        (c, ldc), (s, lds) = _flat_rows(codes), _flat_rows(scale)
        nat.launch(codes.device, "smoe_dequantize_mxfp4", c.data_ptr(), ldc, s.data_ptr(), lds, rows, cols,
                   out.data_ptr(), nat.float_code(out.dtype))
        return out if out.dtype == dtype else out.to(dtype)
    table = torch.tensor(_E2M1 + tuple(-v for v in _E2M1))
    v = table[torch.stack([codes & 15, codes >> 4], dim=-1).flatten(-2)[..., :cols].long()]
    two = torch.exp2(scale.double() - 127.0)
    two = torch.where(scale == 255, float("nan"), two).float()
    return (v * two.repeat_interleave(MX_BLOCK, dim=-1)[..., :cols]).to(dtype)


# ------------------------------------------------------ SwiGLU layout ----
SWIGLU_BLOCK = 32


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """[..., U, X] gate and up -> [..., 2U, X] with 32-row blocks alternating
    gate / up: rows [64j, 64j+32) = gate[32j:32j+32], rows [64j+32, 64j+64) =
    up[32j:32j+32] (the order the up-GEMM epilogue pairs them in)."""
    *lead, u, x = gate.shape
    if u % SWIGLU_BLOCK:
        raise ValueError("SwiGLU hidden size must be a multiple of 32")
    gb = gate.reshape(*lead, u // SWIGLU_BLOCK, SWIGLU_BLOCK, x)
    ub = up.reshape(*lead, u // SWIGLU_BLOCK, SWIGLU_BLOCK, x)
    return torch.stack([gb, ub], dim=-3).reshape(*lead, 2 * u, x).contiguous()


def interleave_gate_up_rows(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """Same interleave for per-row vectors [..., U] (fp8 scales)."""
    return interleave_gate_up(gate.unsqueeze(-1), up.unsqueeze(-1)).squeeze(-1)
