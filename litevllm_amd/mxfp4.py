"""Microscaled 4-bit floating point (MXFP4): quantisation, linear layers and mixture-of-experts stacks whose
two operands the matrix cores multiply in that format.

The format (OCP Microscaling Formats 1.0): 32 consecutive values along the last dimension share a scale
``2 ** (byte - 127)``; a value is an e2m1 code.  A ``[..., K]`` tensor is ``codes`` uint8 ``[..., K/2]`` (the even
index in the low four bits) and ``scales`` uint8 ``[..., K/32]``, as MXFP4 checkpoints hold weights; the kernels
read that layout as it is, so no copy of a weight is built.  Activations are quantised on the way in.  None of these
operators is differentiable: where an input requires a gradient, a backward through the result raises, and so does the
call where the result cannot carry that (codes, ``out``, forward-mode derivatives).

Every byte of the arithmetic runs in ``libawq_w4a16.so``; there is no CPU fallback.  Scratch memory comes from
PyTorch's allocator for each call, so calls on different streams and captured graphs share none.
"""
from __future__ import annotations

import torch
import torch.nn as nn
from torch.autograd import forward_ad

from . import _lib as L
from . import ops
from .tensor import QuantizedLinearWeight

BLOCK = 32


def _call(dev: torch.device, name: str, *args) -> None:
    """One C call on ``dev``'s current stream; a launch needs its stream's device to be the current one."""
    fn = getattr(L._lib or L.load(), name)
    index = dev.index
    if torch._C._cuda_getDevice() == index:
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        raise L.AWQKernelError(name, rc)


class _Refused(torch.autograd.Function):
    """A result unchanged, whose derivative is refused: a backward that reaches it on its way to any of ``inputs`` raises."""

    @staticmethod
    def forward(ctx, why, result, *inputs):
        ctx.why = why
        ctx.mark_dirty(result)  # the result itself, no view of it
        return result

    @staticmethod
    def backward(ctx, *upstream):
        raise RuntimeError(ctx.why)


def _derivative_asked(name: str, out: torch.Tensor | None, *inputs: torch.Tensor | None) -> bool:
    """Whether a backward may ask for a derivative in ``inputs``, which the result has to refuse.  Raises where it cannot: for
    a caller's ``out``, and for an input with a tangent of forward mode."""
    if forward_ad._current_level >= 0:
        for t in inputs:
            if t is not None and t.is_floating_point() and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError(f"{name} has no forward-mode derivative")
    if not torch.is_grad_enabled():
        return False
    for t in inputs:
        if t is not None and t.requires_grad:
            if out is not None:
                raise RuntimeError(f"{name} with out= takes no inputs that require a gradient")
            return True
    return False


def _check_codes(what: str, codes: torch.Tensor, scales: torch.Tensor) -> int:
    """K of a quantised tensor, after its types and shapes."""
    if codes.dtype is not torch.uint8 or scales.dtype is not torch.uint8:
        raise TypeError(f"{what}: codes and scales must be uint8, got {codes.dtype} and {scales.dtype}")
    cs, ss = codes.shape, scales.shape
    k = cs[-1] * 2 if cs else -1
    if k < 0 or k % BLOCK or not ss or ss[-1] * BLOCK != k or cs[:-1] != ss[:-1]:
        raise ValueError(f"{what}: codes [..., K/2] and scales [..., K/{BLOCK}] do not match: "
                         f"{tuple(codes.shape)} and {tuple(scales.shape)}")
    return k


def _dense(t: torch.Tensor) -> torch.Tensor:
    """``t``, or a copy, contiguous on a 16-byte boundary."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """A 2-D ``x`` (or a copy) whose rows the kernels can read, and its row stride."""
    m, k = x.shape
    ld = x.stride(0) if m > 1 else k
    if (x.stride(1) != 1 and k > 1) or ld < k or ld % 8 or x.data_ptr() % 16:
        return _dense(x), k
    return x, ld


def _meet(x: torch.Tensor, y: torch.Tensor) -> bool:
    """Whether the addresses from first to last of two tensors (not empty) overlap."""
    (x0, x1), (y0, y1) = ((t.data_ptr(), t.data_ptr() + t.element_size() * (1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride()))))
                          for t in (x, y))
    return x0 < y1 and y0 < x1


def mxfp4_quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """``(codes, scales)`` of ``x [..., K]`` (fp16, bf16 or fp32; K a multiple of 32).

    A block with the largest magnitude ``m`` takes the scale ``2 ** (floor(log2(m)) - 2)`` (at least ``2 ** -127``);
    values are rounded to the nearest code, ties to even, and those past 6 scales to 6.  A block that holds a
    NaN or an infinity takes the NaN scale (byte 255): all of it stands for NaN."""
    dev = ops._require_device(x)
    dt = ops.dtype_code(x.dtype)
    if _derivative_asked("mxfp4_quantize", None, x):
        raise RuntimeError("mxfp4_quantize is not differentiable, and codes cannot carry that to a backward: detach the input or "
                           "call it under torch.no_grad()")
    if x.dim() == 0 or x.shape[-1] % BLOCK:
        raise ValueError(f"the last dimension must be a multiple of {BLOCK}, got {tuple(x.shape)}")
    k = x.shape[-1]
    codes = torch.empty(x.shape[:-1] + (k // 2,), dtype=torch.uint8, device=dev)
    scales = torch.empty(x.shape[:-1] + (k // BLOCK,), dtype=torch.uint8, device=dev)
    if codes.numel():
        flat, ld = _rows(x if x.dim() == 2 else x.reshape(-1, k))
        _call(dev, "awq_w4a16_mxfp4_quantize", flat.data_ptr(), ld, codes.data_ptr(), scales.data_ptr(), flat.shape[0], k, dt)
    return codes, scales


def mxfp4_dequantize(codes: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = torch.float16) -> torch.Tensor:
    """The values ``[..., K]`` that codes and scales stand for, each rounded once to ``out_dtype``."""
    dev = ops._require_device(codes, scales)
    k = _check_codes("mxfp4_dequantize", codes, scales)
    dt = ops.dtype_code(out_dtype)
    out = torch.empty(codes.shape[:-1] + (k,), dtype=out_dtype, device=dev)
    if out.numel():
        codes, scales = _dense(codes), scales.contiguous()
        _call(dev, "awq_w4a16_mxfp4_dequantize", codes.data_ptr(), scales.data_ptr(), out.data_ptr(), out.numel() // k, k, dt)
    return out


def mxfp4_gemm(a: torch.Tensor, qweight: torch.Tensor, scales: torch.Tensor, a_scales: torch.Tensor | None = None,
               bias: torch.Tensor | None = None, out: torch.Tensor | None = None,
               out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``out[M, N] = Q(a) @ W^T (+ bias)`` with MXFP4 operands, sums in fp32, one rounding.

    ``qweight`` uint8 ``[N, K/2]``, ``scales`` uint8 ``[N, K/32]``.  ``a``: fp16 or bf16 ``[M, K]``, quantised in the
    call, the result in its type; or, with ``a_scales``, codes that :func:`mxfp4_quantize` made (once for
    several projections of one input), the result in ``out_dtype`` (fp16 or bf16).  Other activations than
    quantised ones are not provided.  ``out`` may lie over a 16-bit ``a``, over no other operand.  Results are bitwise
    reproducible."""
    dev = ops._require_device(a, qweight, scales, a_scales, bias, out)
    if a.dim() != 2 or qweight.dim() != 2:
        raise ValueError(f"a and qweight must be 2-D, got {tuple(a.shape)} and {tuple(qweight.shape)}")
    k = _check_codes("mxfp4_gemm: weight", qweight, scales)
    m, n = a.shape[0], qweight.shape[0]
    if a_scales is None:
        ka, dtype = a.shape[1], a.dtype
        if out_dtype is not None and out_dtype != dtype:
            raise ValueError(f"out_dtype {out_dtype} with an unquantised a of {dtype}: the result has a's type")
    else:
        ka, dtype = _check_codes("mxfp4_gemm: a", a, a_scales), out_dtype
        if dtype is None:
            raise ValueError("a quantised a needs out_dtype")
    if ka != k or k == 0:
        raise ValueError(f"K mismatch: a has {ka}, weight has {k}")
    if dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported dtype {dtype}: fp16 or bf16")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"bias must be [{n}], got {tuple(bias.shape)}")
    asked, inputs = _derivative_asked("mxfp4_gemm", out, a, bias), (a, bias)
    if out is None:
        out = torch.empty((m, n), dtype=dtype, device=dev)
    elif out.dtype != dtype:
        raise ValueError(f"bad_output: out must be {dtype}, got {out.dtype}")
    else:
        ops.check_out(out, m, n, out)
        if a_scales is None and m and n and _meet(a, out):
            # few rows are read by every block, also while others write: a, which out may lie over, first
            a, a_scales = mxfp4_quantize(a)
    if m == 0 or n == 0:
        return out
    lib = L.load()
    qweight, scales = _dense(qweight), scales.contiguous()
    ws, ws_bytes, ld = None, 0, k
    if a_scales is None:
        a, ld = _rows(a)
        ws_bytes = lib.awq_w4a16_mxfp4_gemm_workspace_bytes(m, n, k)
        if ws_bytes:
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    else:
        a, a_scales = _dense(a), a_scales.contiguous()
    if bias is not None:
        bias = bias.contiguous()
    _call(dev, "awq_w4a16_mxfp4_gemm", a.data_ptr(), ld, ops._ptr(a_scales), qweight.data_ptr(), scales.data_ptr(),
          ops._ptr(bias), out.data_ptr(), out.stride(0) if m > 1 else n, m, n, k, ops.dtype_code(dtype),
          L.DTYPE_NONE if bias is None else ops.dtype_code(bias.dtype), ops._ptr(ws), ws_bytes)
    return _Refused.apply("mxfp4_gemm is not differentiable", out, *inputs) if asked else out


def is_mxfp4(qweight: torch.Tensor, scales: torch.Tensor) -> bool:
    """Whether a layer's tensors are MXFP4's: both uint8 (the scales of int4 weights are floating point)."""
    return qweight.dtype is torch.uint8 and scales.dtype is torch.uint8


class MXFP4Weight(QuantizedLinearWeight):
    """A linear layer's MXFP4 weight, beside :class:`AWQWeight` and used as it is: ``qweight`` uint8 ``[N, K/2]``,
    ``scales`` uint8 ``[N, K/32]``."""

    def __init__(self, qweight: torch.Tensor, scales: torch.Tensor, prefix: str = ""):
        super().__init__()
        if qweight.dim() != 2:
            raise ValueError(f"qweight must be [N, K/2], got {tuple(qweight.shape)}")
        _check_codes("MXFP4Weight", qweight, scales)
        self.qweight = nn.Parameter(qweight, requires_grad=False)
        self.scales = nn.Parameter(scales, requires_grad=False)
        self.prefix = prefix

    @classmethod
    def from_dense(cls, weight: torch.Tensor, prefix: str = "") -> "MXFP4Weight":
        """Quantises the values of a dense ``[N, K]`` weight."""
        return cls(*mxfp4_quantize(weight.detach()), prefix=prefix)

    def dense_weight(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """The ``[N, K]`` values."""
        return mxfp4_dequantize(self.qweight, self.scales, dtype)

    def matmul(self, x: torch.Tensor, bias: torch.Tensor | None = None, *, config: object | None = None) -> torch.Tensor:
        """``x [..., K] @ W^T (+ bias)``, in ``x``'s type (:func:`mxfp4_gemm`).  Of the policies in ``config`` none applies:
        there is one path."""
        y = mxfp4_gemm(x.reshape(-1, x.shape[-1]), self.qweight, self.scales, bias=bias)
        return y.view(x.shape[:-1] + (y.shape[-1],))


class MXFP4Experts:
    """An MXFP4 expert stack ``[E, N, K]``: ``qweight`` uint8 ``[E, N, K/2]``, ``scales`` uint8 ``[E, N, K/32]``."""

    __slots__ = ("qweight", "scales")

    def __init__(self, qweight: torch.Tensor, scales: torch.Tensor):
        self.qweight, self.scales = qweight, scales

    def dims(self) -> tuple[int, int, int]:
        """(E, K, N) of the stack."""
        e, n, kb = self.qweight.shape
        return e, kb * 2, n


def mxfp4_moe(x: torch.Tensor, topk_weights: torch.Tensor, topk_ids: torch.Tensor, gate_up: MXFP4Experts, down: MXFP4Experts,
              *, activation: str = "silu", out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[t] = sum_j w[t, j] * (Q(act(g) * u) @ W2_e^T)``, ``g, u = Q(x[t]) @ W1_e^T``, ``e = topk_ids[t, j]``.

    ``gate_up`` is the ``[E, 2I, H]`` stack (rows 0 .. I-1 gate, I .. 2I-1 up), ``down`` the ``[E, H, I]`` one; H and I
    are multiples of 32.  Sums are fp32 in slot order with one rounding; the routing weights enter in fp32.
    Ids outside ``[0, E)`` contribute nothing.  ``out`` may lie over ``x``, over no other operand.  Results are bitwise
    reproducible.  Scratch of ``T * top_k * (4 H + 17 I / 32)`` bytes and more is allocated for the call (7.8 GB for 32768
    tokens, top 8, H = 7168, I = 2048): cut long prompts into calls."""
    dev = ops._require_device(x, topk_weights, topk_ids, gate_up.qweight, gate_up.scales, down.qweight, down.scales, out)
    if x.dim() != 2 or gate_up.qweight.dim() != 3 or down.qweight.dim() != 3:
        raise ValueError("x must be [T, H] and the stacks [E, N, K/2]")
    if x.dtype not in (torch.float16, torch.bfloat16):
        raise TypeError(f"unsupported dtype {x.dtype}: fp16 or bf16")
    act = ops.MOE_ACTIVATIONS.get(str(activation).strip().lower())
    if act is None:
        raise ValueError(f"unsupported activation {activation!r}")
    t, h = x.shape
    if _check_codes("mxfp4_moe: gate_up", gate_up.qweight, gate_up.scales) != h:
        raise ValueError(f"gate_up has K = {gate_up.qweight.shape[2] * 2}, x has {h}")
    inter = _check_codes("mxfp4_moe: down", down.qweight, down.scales)
    e = gate_up.qweight.shape[0]
    if gate_up.qweight.shape[1] != 2 * inter or down.qweight.shape[:2] != (e, h):
        raise ValueError(f"gate_up [E, 2I, H/2] {tuple(gate_up.qweight.shape)} and down [E, H, I/2] "
                         f"{tuple(down.qweight.shape)} do not match")
    if topk_ids.dim() != 2 or topk_ids.shape[0] != t or topk_weights.shape != topk_ids.shape:
        raise ValueError(f"topk_weights and topk_ids must be [{t}, top_k], got {tuple(topk_weights.shape)} and "
                         f"{tuple(topk_ids.shape)}")
    if topk_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"topk_ids must be int32 or int64, got {topk_ids.dtype}")
    wdt, k = ops.dtype_code(topk_weights.dtype), topk_ids.shape[1]
    asked, inputs = _derivative_asked("mxfp4_moe", out, x, topk_weights), (x, topk_weights)
    if out is None:
        out = torch.empty((t, h), dtype=x.dtype, device=dev)
    else:
        ops.check_out(out, t, h, x)
    if t == 0 or h == 0:
        return out
    if k == 0 or e == 0 or inter == 0:
        return out.zero_()
    lib = L.load()
    x, ld = _rows(x)
    topk_ids, topk_weights = topk_ids.contiguous(), topk_weights.contiguous()
    w1, s1, w2, s2 = _dense(gate_up.qweight), gate_up.scales.contiguous(), _dense(down.qweight), down.scales.contiguous()
    ws_bytes = lib.awq_w4a16_mxfp4_moe_workspace_bytes(t, h, inter, e, k)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
    _call(dev, "awq_w4a16_mxfp4_moe", x.data_ptr(), ld, topk_ids.data_ptr(), 64 if topk_ids.dtype == torch.int64 else 32,
          topk_weights.data_ptr(), wdt, w1.data_ptr(), s1.data_ptr(), w2.data_ptr(), s2.data_ptr(), out.data_ptr(),
          out.stride(0) if t > 1 else h, t, h, inter, e, k, act, ops.dtype_code(x.dtype), ws.data_ptr(), ws_bytes)
    return _Refused.apply("mxfp4_moe is not differentiable", out, *inputs) if asked else out
