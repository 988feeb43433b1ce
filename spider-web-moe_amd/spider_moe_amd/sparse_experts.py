"""sparse_expert_delta with the reference signature (spider_moe/sparse_experts.py:11-68),
computed by libsmoe.so: slot merge -> stable dispatch plan -> grouped up
GEMM + GELU -> grouped down GEMM (+ bias, x routing weight) -> per-token
combine in ascending expert order.

Duplicate expert ids across slots add their weights; a token whose merged
weight is <= 0 is dropped for that expert (sparse_experts.py:52-56); ids
outside [0, E) match no expert.  Weights may be float32 or bfloat16
(messages are cast to bfloat16 for bf16 weights, the MFMA path).

With expert parallelism active (torch.distributed world > 1) the reference
computes its local experts and SUM-all-reduces; this single-GPU module
computes every expert on every rank, which yields the same delta.

sparse_expert_delta_fp8_blocks is the same step on experts whose weights are
e4m3 codes with a scale per 128 x 128 block (Fp8BlockExperts).
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as nat
from .quant import FP8_BLOCK, quantize_fp8_blocks


def _experts_desc(w_up, b_up, w_down, b_down, act=nat.ACT_GELU):
    e, u, h = w_up.shape
    ex = nat.SmoeExperts()
    ex.format = nat.dtype_code(w_up.dtype)
    ex.act = act
    ex.E, ex.H, ex.U = e, h, u
    keep = [w_up.contiguous(), w_down.to(w_up.dtype).contiguous()]
    ex.w_up, ex.w_down = keep[0].data_ptr(), keep[1].data_ptr()
    for name, b in (("b_up", b_up), ("b_down", b_down)):
        if b is not None:
            bb = b.detach().float().contiguous()
            keep.append(bb)
            setattr(ex, name, bb.data_ptr())
    return ex, keep


@torch.no_grad()
def sparse_expert_delta(
    messages: torch.Tensor,
    top_indices: torch.Tensor,
    top_weights: torch.Tensor,
    w_up: torch.Tensor,
    b_up: torch.Tensor,
    w_down: torch.Tensor,
    b_down: torch.Tensor,
    num_experts: int,
    top_k: int,
    expert_parallel: bool = True,
) -> torch.Tensor:
    """messages [B,T,H]; top_indices / top_weights [B,T,K]; w_up [E,U,H];
    b_up [E,U]; w_down [E,H,U]; b_down [E,H] -> delta [B,T,H] (messages.dtype)."""
    dev = nat.require_gpu(messages, top_indices, top_weights, w_up, b_up, w_down, b_down)
    b, t, width = messages.shape
    if w_up.shape[0] != num_experts or top_indices.shape[-1] != top_k:
        raise ValueError("num_experts / top_k do not match the tensors")
    n = b * t
    ex, keep = _experts_desc(w_up, b_up, w_down, b_down)
    ffn_dtype = torch.float32 if ex.format == nat.F32 else torch.bfloat16
    msg = messages.reshape(n, width).to(ffn_dtype).contiguous()
    idx = top_indices.reshape(n, top_k).to(torch.int32).contiguous()
    wts = top_weights.reshape(n, top_k).to(torch.float32).contiguous()
    out_dtype = messages.dtype if messages.dtype in (torch.float32, torch.bfloat16) else torch.float32
    delta = torch.empty(n, width, dtype=out_dtype, device=dev)
    lib = nat.lib()
    need = lib.smoe_expert_delta_workspace_bytes(ctypes.byref(ex), n, top_k)
    if need == 0:
        raise RuntimeError(f"smoe_expert_delta: unsupported expert shapes ({lib.smoe_last_error().decode()})")
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    nat.check(lib.smoe_expert_delta(ctypes.byref(ex), msg.data_ptr(), idx.data_ptr(), wts.data_ptr(),
                                    n, top_k, delta.data_ptr(), nat.dtype_code(out_dtype),
                                    ws.data_ptr(), need, nat.stream_of(dev)),
              "smoe_expert_delta")
    del keep
    return delta.view(b, t, width).to(messages.dtype)


class Fp8BlockExperts:
    """Expert FFN weights as e4m3 codes with one f32 scale per 128 x 128 block.

    w_up [E,U,H] codes and s_up [E, ceil(U/128), ceil(H/128)]; for
    activation "swiglu" [E,2U,H], the gate's rows first, and s_up
    [E, 2 ceil(U/128), ceil(H/128)] (gate and up projection are quantized
    each on its own).  w_down [E,H,U], s_down [E, ceil(H/128), ceil(U/128)].
    b_up [E,U] (swiglu: added to the up projection) and b_down [E,H] or None.
    H % 16 == 0 and U % 16 == 0.

    The tensors are kept, not copied, and every call takes them as they are
    then: changed in place, with other memory (`t.data = ..`, Module.to) or set
    anew as an attribute.  Scales that are not contiguous and biases that are
    not contiguous float32 are converted in each call.  Only codes that are not
    contiguous or not 16-byte aligned are copied once and no longer followed.
    Fp8BlockExperts.quantize makes one from float weights."""

    _TENSORS = ("w_up", "s_up", "w_down", "s_down", "b_up", "b_down")

    def __init__(self, w_up, s_up, w_down, s_down, *, b_up=None, b_down=None,
                 activation: str = "gelu"):
        self.w_up, self.s_up, self.w_down, self.s_down = w_up, s_up, w_down, s_down
        self.b_up, self.b_down = b_up, b_down
        self.activation = activation
        self._bind()

    def __setattr__(self, name, value):
        super().__setattr__(name, value)
        if name in self._TENSORS or name == "activation":
            super().__setattr__("_at", None)  # the next call looks at it

    def _bind(self):
        """Checks the tensors and describes them to the library."""
        w_up, s_up, w_down, s_down, b_up, b_down = (getattr(self, n) for n in self._TENSORS)
        if self.activation not in ("gelu", "swiglu"):
            raise ValueError("activation must be 'gelu' or 'swiglu'")
        device = nat.require_gpu(w_up, s_up, w_down, s_down, b_up, b_down)
        if w_up.ndim != 3 or w_down.ndim != 3:
            raise ValueError("w_up and w_down must be stacked over experts: [E, .., ..]")
        halves = 2 if self.activation == "swiglu" else 1
        e, h, u = w_down.shape
        hb, ub = -(-h // FP8_BLOCK), -(-u // FP8_BLOCK)
        if w_up.shape != (e, halves * u, h):
            raise ValueError(f"w_up must be {(e, halves * u, h)}, got {tuple(w_up.shape)}")
        for name, t, shape in (("s_up", s_up, (e, halves * ub, hb)), ("s_down", s_down, (e, hb, ub))):
            if t.shape != shape or t.dtype != torch.float32:
                raise ValueError(f"{name} must be float32 {shape}, got {t.dtype} {tuple(t.shape)}")
        for name, t in (("w_up", w_up), ("w_down", w_down)):
            if t.dtype != torch.float8_e4m3fn:
                raise ValueError(f"{name} must be float8_e4m3fn codes, got {t.dtype}")
        for name, t, shape in (("b_up", b_up, (e, u)), ("b_down", b_down, (e, h))):
            if t is not None and t.shape != shape:
                raise ValueError(f"{name} must be {shape}, got {tuple(t.shape)}")
        if h % 16 or u % 16 or not 1 <= e <= 256:
            raise ValueError("Fp8BlockExperts: H % 16 == 0, U % 16 == 0, 1 <= E <= 256")
        self.device = device
        self.num_experts, self.hidden_size, self.expert_ffn_size = e, h, u
        for name, t in (("w_up", w_up), ("w_down", w_down)):
            if not t.is_contiguous():
                setattr(self, name, t.contiguous())
            elif t.data_ptr() % 16:
                setattr(self, name, t.clone())
        at = self._addresses()
        if 0 in at:
            raise ValueError("Fp8BlockExperts: a tensor's memory was released")
        d = nat.SmoeExpertsFp8Blocks()
        d.act = nat.ACT_SWIGLU if halves == 2 else nat.ACT_GELU
        d.E, d.H, d.U = e, h, u
        d.w_up, d.s_up, d.w_down, d.s_down, d.b_up, d.b_down = at
        self._desc = d
        self._ref = ctypes.byref(d)
        self._convert = [n for n, t in zip(self._TENSORS, (w_up, s_up, w_down, s_down, b_up, b_down))
                         if n not in ("w_up", "w_down") and t is not None and
                         not (t.dtype == torch.float32 and t.is_contiguous())]
        self._at = at

    def _addresses(self):
        u, d = self.b_up, self.b_down
        return (self.w_up.data_ptr(), self.s_up.data_ptr(), self.w_down.data_ptr(), self.s_down.data_ptr(),
                None if u is None else u.data_ptr(), None if d is None else d.data_ptr())

    def _descriptor(self):
        """The C descriptor of the tensors as they are now, and what has to
        live until the call on it is made."""
        if self._at is None or self._at != self._addresses():
            self._bind()
        if not self._convert:
            return self._ref, None
        d = nat.SmoeExpertsFp8Blocks.from_buffer_copy(self._desc)
        keep = [getattr(self, n).detach().float().contiguous() for n in self._convert]
        for n, t in zip(self._convert, keep):
            setattr(d, n, t.data_ptr())
        return ctypes.byref(d), keep

    @classmethod
    def quantize(cls, w_up, w_down, *, b_up=None, b_down=None, activation: str = "gelu"):
        """From float weights w_up [E, U or 2U, H] and w_down [E,H,U]."""
        e, _, u = w_down.shape
        if activation == "swiglu":
            if w_up.shape[1] != 2 * u:
                raise ValueError("swiglu: w_up must hold the gate's and the up projection's rows, [E,2U,H]")
            q, s = quantize_fp8_blocks(w_up.reshape(2 * e, u, w_up.shape[-1]))
            q = q.contiguous().view(e, 2 * u, w_up.shape[-1])
            s = s.view(e, -1, s.shape[-1])
        else:
            q, s = quantize_fp8_blocks(w_up)
        qd, sd = quantize_fp8_blocks(w_down)
        return cls(q, s, qd, sd, b_up=b_up, b_down=b_down, activation=activation)


def _expert_ids(idx: torch.Tensor, num_experts: int) -> torch.Tensor:
    """idx as int32, ids outside [0, num_experts) still outside.  Narrow types
    go straight to int32: they need not hold the limits of a clamp (-1 in
    uint8 is 255)."""
    if idx.dtype == torch.int32:
        return idx
    if idx.dtype not in (torch.uint8, torch.int8, torch.int16):
        idx = idx.clamp(-1, num_experts)
    return idx.to(torch.int32)


def sparse_expert_delta_fp8_blocks(messages: torch.Tensor, top_indices: torch.Tensor,
                                   top_weights: torch.Tensor, experts: Fp8BlockExperts) -> torch.Tensor:
    """sparse_expert_delta on Fp8BlockExperts: messages [..,H] (float32 or
    bfloat16), top_indices / top_weights [..,K] -> delta [..,H] in messages'
    dtype.  Messages and hidden activations are quantized in 1 x 128 blocks on
    the way into the two products.  float32: both products and all that
    follows are summed in f32; bfloat16: the products by the e4m3 x e4m3 matrix
    instruction, which cuts each one by less than 2^-13 of the largest of its
    eight neighbours, the rest in f32.  No gradient."""
    ref, keep = experts._descriptor()
    dev = nat.require_gpu(messages, top_indices, top_weights, experts.w_up)
    h, k = messages.shape[-1], top_indices.shape[-1]
    if h != experts.hidden_size:
        raise ValueError(f"messages have {h} channels, the experts {experts.hidden_size}")
    if top_indices.shape[:-1] != messages.shape[:-1] or top_weights.shape != top_indices.shape:
        raise ValueError("top_indices and top_weights must be messages' shape with K last")
    code = nat.dtype_code(messages.dtype)
    idx, wts = _expert_ids(top_indices, experts.num_experts), top_weights
    if wts.dtype != torch.float32:
        wts = wts.float()
    msg, idx, wts = messages.contiguous(), idx.contiguous(), wts.contiguous()
    n = idx.numel() // k if k else 0
    if n > 0x7fffffff:
        raise ValueError("more than 2^31 - 1 tokens")
    delta = torch.empty(messages.shape, dtype=messages.dtype, device=dev)
    lib = nat.lib()
    need = lib.smoe_expert_delta_fp8_blocks_workspace_bytes(ref, n, k)
    if need == 0:
        raise RuntimeError("smoe_expert_delta_fp8_blocks: "
                           f"unsupported shapes ({lib.smoe_last_error().decode()})")
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    nat.launch(dev, "smoe_expert_delta_fp8_blocks", ref, msg.data_ptr(), code,
               idx.data_ptr(), wts.data_ptr(), n, k, delta.data_ptr(), code, ws.data_ptr(), need)
    del keep
    return delta
