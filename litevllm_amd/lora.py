"""Low-rank adapters of many requests beside a shared projection: what the reference adds behind a layer's product
(``lite_linear.py:65-78``), each row with its own adapter, in one call."""
from __future__ import annotations

from collections.abc import Sequence

import torch
import torch.nn as nn

from . import _lib as L
from . import ops
from .mxfp4 import _call, _derivative_asked, _meet, _Refused
from .moe_sort import _rows

MAX_RANK = 256
_DTYPES = {torch.float16: L.DTYPE_F16, torch.bfloat16: L.DTYPE_BF16}


def _stack(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """An adapter stack, or a copy, dense but for the elements between adapters, and their number."""
    count, rows, cols = t.shape
    dense = rows * cols
    if (cols > 1 and t.stride(2) != 1) or (rows > 1 and t.stride(1) != cols) or (count > 1 and t.stride(0) < dense):
        t = t.contiguous()
    return t, t.stride(0) if count > 1 else dense


def lora_add(base: torch.Tensor | None, x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, ids: torch.Tensor,
             scales: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """``out[m] = base[m] + scales[l] * (x[m] @ lora_a[l].T) @ lora_b[l].T`` with ``l = ids[m]``; ``base[m]`` where ``ids[m]`` is
    outside ``[0, L)`` (a request without an adapter).

    ``x [..., K]``, ``base [..., N]`` (None: zeros), fp16 or bf16; ``lora_a [L, R, K]`` and ``lora_b [L, N, R]`` in their type, R up
    to 256 (adapters of lower ranks: zeros, :meth:`LoRAAdapters.stack`); ``ids [...]`` int32 or int64; ``scales`` fp32 ``[L]`` or
    None (1).  Sums in fp32, one rounding of the result; ``x @ A^T`` enters the second product off by at most 2^-17 of itself
    (bf16), or 2^-22 of itself or 2^-38 of the row's largest of 32 neighbouring ranks, whichever is more (fp16).
    ``out`` may be ``base`` itself, and lie over ``x`` or parts of ``base`` (which are copied first), over no other operand.
    Rows of the same adapter are cheapest next to each other, as a request's tokens are.  The same call gives the same bits; the
    order of a row's fp32 sums, and so its last bit, may follow how many rows the call has and which adapters they name.
    Not differentiable: a backward through the result raises, and so does a call with ``out`` where an input or ``out``
    requires a gradient."""
    dev = ops._require_device(base, x, lora_a, lora_b, ids, scales, out)
    a_shape, b_shape, x_shape, dtype = lora_a.shape, lora_b.shape, x.shape, x.dtype
    if len(a_shape) != 3 or len(b_shape) != 3 or a_shape[0] != b_shape[0] or a_shape[1] != b_shape[2]:
        raise ValueError(f"lora_a must be [L, R, K] and lora_b [L, N, R], got {tuple(a_shape)} and {tuple(b_shape)}")
    adapters, rank, k = a_shape
    n = b_shape[1]
    if adapters < 1 or not 1 <= rank <= MAX_RANK or k < 1:
        raise ValueError(f"at least one adapter and input, a rank of 1 to {MAX_RANK}, got lora_a {tuple(a_shape)}")
    if not x_shape or x_shape[-1] != k:
        raise ValueError(f"K mismatch: x is {tuple(x_shape)}, lora_a has {k}")
    code = _DTYPES.get(dtype)
    if code is None:
        raise TypeError(f"unsupported dtype {dtype}: fp16 or bf16")
    lead = x_shape[:-1]
    shape = lead + (n,)
    if lora_a.dtype is not dtype or lora_b.dtype is not dtype or (base is not None and base.dtype is not dtype) or (
            out is not None and out.dtype is not dtype):
        raise TypeError(f"base, lora_a, lora_b and out must be of x's type {dtype}, got "
                        f"{[None if t is None else t.dtype for t in (base, lora_a, lora_b, out)]}")
    if (base is not None and base.shape != shape) or (out is not None and out.shape != shape):
        raise ValueError(f"base and out must be {tuple(shape)}, got {[None if t is None else tuple(t.shape) for t in (base, out)]}")
    wide = ids.dtype is torch.int64
    if not wide and ids.dtype is not torch.int32:
        raise TypeError(f"ids must be int32 or int64, got {ids.dtype}")
    if ids.shape != lead:
        raise ValueError(f"ids must be {tuple(lead)}, got {tuple(ids.shape)}")
    if scales is not None and (scales.dtype is not torch.float32 or scales.shape != (adapters,)):
        raise ValueError(f"scales must be fp32 [{adapters}], got {scales.dtype} {tuple(scales.shape)}")
    asked = _derivative_asked("lora_add", out, base, x, lora_a, lora_b, scales, out)  # out's graph would not hear of the call
    m = ids.numel()
    given = out is not None
    if not given:
        out = torch.empty(shape, dtype=dtype, device=dev) if base is None or not base.is_contiguous() else torch.empty_like(base)
        to, ldo = out, n
    else:
        to = out
        if out.dim() != 2:
            try:
                to = out.view(-1, n) if n else out
            except RuntimeError:
                raise ValueError(f"bad_output: out's rows must be those of a matrix, got strides {out.stride()}") from None
        ldo = to.stride(0) if m > 1 else n
        if m and n and ((n > 1 and to.stride(-1) != 1) or ldo < n):
            raise ValueError(f"bad_output: out must have dense rows apart from each other, got strides {out.stride()}")
    if m == 0 or n == 0:
        return out
    if x.is_contiguous():
        ldx = k
    else:
        x, ldx = _rows(x if x.dim() == 2 else x.reshape(-1, k))
    at, ldb = None, n
    if base is out:
        at, ldb = to.data_ptr(), ldo
    elif base is not None:
        flat = base
        if not base.is_contiguous():
            flat, ldb = _rows(base if base.dim() == 2 else base.reshape(-1, n))
        if given and (flat.data_ptr() != to.data_ptr() or ldb != ldo) and _meet(flat, to):
            flat, ldb = flat.clone(memory_format=torch.contiguous_format), n  # other elements of the same memory
        at = flat.data_ptr()
    if given and _meet(x, to):
        x, ldx = x.clone(memory_format=torch.contiguous_format), k  # read by blocks while others write
    a_stride, b_stride = rank * k, n * rank
    if not lora_a.is_contiguous():
        lora_a, a_stride = _stack(lora_a)
    if not lora_b.is_contiguous():
        lora_b, b_stride = _stack(lora_b)
    ids = ids.contiguous()
    if scales is not None:
        scales = scales.contiguous()
    ws_bytes = (L._lib or L.load()).awq_w4a16_lora_workspace_bytes(m, k, rank)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    _call(dev, "awq_w4a16_lora_add", at, ldb, x.data_ptr(), ldx, lora_a.data_ptr(), a_stride, lora_b.data_ptr(), b_stride,
          ids.data_ptr(), 64 if wide else 32, None if scales is None else scales.data_ptr(), to.data_ptr(), ldo, m, n, k, rank,
          adapters, code, None if ws is None else ws.data_ptr(), ws_bytes)
    if given:
        torch.autograd.graph.increment_version(out)  # a backward that has saved it would take other values
    return _Refused.apply("lora_add is not differentiable", out, base, x, lora_a, lora_b, scales) if asked else out


class LoRAAdapters(nn.Module):
    """The adapters of a linear layer: ``lora_a [L, R, K]``, ``lora_b [L, N, R]`` and ``scales`` fp32 ``[L]`` (alpha / rank; None:
    1).  As ``layer.lora_adapters`` :meth:`AWQConfig.apply` adds them to the layer's product for the ids that a call names; the
    rows are of the adapters' type, fp16 or bf16.  The scales stay fp32 when the module is cast."""

    def __init__(self, lora_a: torch.Tensor, lora_b: torch.Tensor, scales: torch.Tensor | None = None):
        super().__init__()
        self.lora_a = nn.Parameter(lora_a, requires_grad=False)
        self.lora_b = nn.Parameter(lora_b, requires_grad=False)
        self.scales = None if scales is None else nn.Parameter(scales, requires_grad=False)

    def _apply(self, fn, recurse=True):
        """A cast of the module is one of the adapters: the scales keep their 32 bits, as 16 / 12 in bf16 would be off by 2^-9 in
        every value that they weight, and go along to another device."""
        before = None if self.scales is None else self.scales.data
        super()._apply(fn, recurse)
        if before is not None and self.scales.dtype is not before.dtype:
            self.scales.data = before.to(self.scales.device)
        return self

    @classmethod
    def stack(cls, adapters: Sequence[tuple[torch.Tensor, torch.Tensor, float]]) -> "LoRAAdapters":
        """Of ``(A [r, K], B [N, r], scale)`` of any ranks, zeros behind the lower ones."""
        if not adapters:
            raise ValueError("no adapters to stack")
        first_a, first_b, _ = adapters[0]
        rank = max(a.shape[0] for a, _, _ in adapters)
        lora_a = first_a.new_zeros(len(adapters), rank, first_a.shape[1])
        lora_b = first_b.new_zeros(len(adapters), first_b.shape[0], rank)
        for i, (a, b, _) in enumerate(adapters):
            if a.shape[0] != b.shape[1] or a.shape[1] != first_a.shape[1] or b.shape[0] != first_b.shape[0]:
                raise ValueError(f"adapter {i}: A {tuple(a.shape)} and B {tuple(b.shape)} do not match or differ from the first's")
            lora_a[i, :a.shape[0]] = a.detach()
            lora_b[i, :, :a.shape[0]] = b.detach()
        return cls(lora_a, lora_b, torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32, device=lora_a.device))

    def add(self, base: torch.Tensor | None, x: torch.Tensor, ids: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """:func:`lora_add` with these adapters."""
        scales = self.scales
        if scales is not None and scales.dtype is not torch.float32:
            scales = scales.float()  # given so
        return lora_add(base, x, self.lora_a, self.lora_b, ids, scales, out)
