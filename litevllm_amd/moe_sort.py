"""The tokens' rows in the order of the experts that :func:`moe_route` chose, and back at the tokens with the routing's weights,
for experts whose products the grouped kernels do not take: dense ones, ones that are trained, and, where nothing is trained,
experts with low-rank adapters of their own (:func:`lora_add`, which has no derivative)."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib as L
from . import ops
from .mxfp4 import _call, _derivative_asked, _Refused


class MoERoutes(NamedTuple):
    """Where the routes went.  ``offsets`` int32 ``[E + 1]``: the places ``offsets[e] .. offsets[e + 1] - 1`` are expert ``e``'s;
    ``experts`` int32 ``[T * top_k]``: the expert of a place, -1 behind the last; ``places`` int32 ``[T, top_k]``: the place of a
    route, -1 for one without an expert."""

    offsets: torch.Tensor
    experts: torch.Tensor
    places: torch.Tensor


def _rows(x: torch.Tensor) -> tuple[torch.Tensor, int]:
    """A 2-D ``x``, or a copy, whose rows are dense, and its row stride."""
    n, h = x.shape
    if x.is_contiguous():
        return x, h
    if (h > 1 and x.stride(1) != 1) or (n > 1 and x.stride(0) < h):
        return x.contiguous(), h
    return x, x.stride(0) if n > 1 else h


def _elsewhere(name: str):
    return RuntimeError(f"{name}: saved tensors came back elsewhere, or with other shapes or types")


def _index(ids, experts):
    """(offsets, experts, places), still to be written; no views of one tensor, since a backward would take what a user writes
    over one of them for a change of those that it has saved."""
    places = torch.empty_like(ids, dtype=torch.int32)
    return places.new_empty(experts + 1), places.new_empty(ids.numel()), places


def _sorted(x, ids, experts, index):
    (t, k), h, dev = ids.shape, x.shape[1], x.device
    rows = torch.empty((t * k, h), dtype=x.dtype, device=dev)
    need = (L._lib or L.load()).awq_w4a16_moe_sort_workspace_bytes(t, experts, k)
    ws = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    x, ld = _rows(x)
    offsets, of, places = index
    _call(dev, "awq_w4a16_moe_sort", x.data_ptr(), ld, ids.data_ptr(), 64 if ids.dtype is torch.int64 else 32, rows.data_ptr(),
          offsets.data_ptr(), of.data_ptr(), places.data_ptr(), t, h, experts, k, ops.dtype_code(x.dtype), ops._ptr(ws), need)
    return rows


def _unsorted(rows, weights, places):
    (t, k), h, dtype = places.shape, rows.shape[1], rows.dtype
    out = torch.empty((t, h), dtype=dtype, device=rows.device)
    _call(rows.device, "awq_w4a16_moe_unsort", rows.data_ptr(), places.data_ptr(), None if weights is None else weights.data_ptr(),
          L.DTYPE_NONE if weights is None else ops.dtype_code(weights.dtype), out.data_ptr(), h, t, h, k, ops.dtype_code(dtype))
    return out


# The backward passes run on a thread of the engine's, where each object that they touch comes from another core: they keep to
# few.  Saved-tensor hooks may give back other tensors, so each is checked again.
class _Sort(torch.autograd.Function):
    """The rows; the index, which is no function of x, is written on the way and comes from outside."""

    @staticmethod
    def forward(ctx, x, ids, experts, index):
        ctx.save_for_backward(index[2])
        ctx.of = x.shape, ids.shape, ops.dtype_code(x.dtype)
        return _sorted(x, ids, experts, index)

    @staticmethod
    def backward(ctx, upstream):
        places, = ctx.saved_tensors
        shape, routes, code = ctx.of
        if places.shape != routes or places.dtype is not torch.int32 or places.get_device() != upstream.get_device():
            raise _elsewhere("moe_sort")
        upstream, places = upstream.contiguous(), places.contiguous()
        grad = upstream.new_empty(shape)
        h = shape[1]
        _call(upstream.device, "awq_w4a16_moe_unsort", upstream.data_ptr(), places.data_ptr(), None, L.DTYPE_NONE, grad.data_ptr(), h,
              shape[0], h, routes[1], code)
        if torch.is_grad_enabled():  # create_graph: a second derivative is refused, not taken as zero
            grad = _Refused.apply("moe_sort is not differentiable twice", grad, upstream)
        return grad, None, None, None


class _Unsort(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, places, offsets):
        of_rows, of_weights, _, _ = ctx.needs_input_grad  # what each gradient reads, so that the rest may change
        ctx.save_for_backward(rows if of_weights else None, weights if of_rows else None, places, offsets if of_rows else None)
        ctx.of = (rows.shape, rows.dtype, places.shape, None if weights is None else weights.dtype, offsets.shape,
                  ops.dtype_code(rows.dtype), L.DTYPE_NONE if weights is None else ops.dtype_code(weights.dtype))
        return _unsorted(rows, weights, places)

    @staticmethod
    def backward(ctx, upstream):
        rows, weights, places, offsets = ctx.saved_tensors
        shape, dtype, routes, wdtype, experts, code, wcode = ctx.of
        on = upstream.get_device()
        if places.shape != routes or places.dtype is not torch.int32 or places.get_device() != on or (
                offsets is not None and (offsets.shape != experts or offsets.dtype is not torch.int32 or offsets.get_device() != on)) or (
                rows is not None and (rows.shape != shape or rows.dtype is not dtype or rows.get_device() != on)) or (
                weights is not None and (weights.shape != routes or weights.dtype is not wdtype or weights.get_device() != on)):
            raise _elsewhere("moe_unsort")
        want_rows, want_weights, _, _ = ctx.needs_input_grad
        flat, ld = (upstream, shape[1]) if upstream.is_contiguous() else _rows(upstream)
        grad_rows = upstream.new_empty(shape) if want_rows else None
        grad_weights = upstream.new_empty(routes, dtype=wdtype) if want_weights else None
        read, w, places, offsets = (None if t is None else t.contiguous() for t in (rows, weights, places, offsets))
        _call(upstream.device, "awq_w4a16_moe_unsort_grad", flat.data_ptr(), ld, ops._ptr(read), places.data_ptr(),
              None if offsets is None else offsets.data_ptr() + 4 * (experts[0] - 1), ops._ptr(w), wcode, ops._ptr(grad_rows),
              ops._ptr(grad_weights), routes[0], shape[1], routes[1], code)
        if torch.is_grad_enabled():
            inputs = upstream, rows, weights
            grad_rows, grad_weights = (None if g is None else _Refused.apply("moe_unsort is not differentiable twice", g, *inputs)
                                       for g in (grad_rows, grad_weights))
        return grad_rows, grad_weights, None, None


def moe_sort(x: torch.Tensor, topk_ids: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, MoERoutes]:
    """``(rows, routes)``: the rows ``[T * top_k, H]`` of ``x [T, H]`` (fp16, bf16 or fp32), one for every route, expert after
    expert and an expert's in the order of the tokens (:class:`MoERoutes`); differentiable in ``x``.

    ``topk_ids``: int32 or int64 ``[T, top_k]``; routes whose id is outside ``[0, num_experts)`` (dropped ones, experts of other
    devices) get no row, and as many rows behind the last are 0 (what a gradient holds there is not read).  1 to 1024 experts and
    routes a token.
    ``routes.offsets`` stays on the device; a loop over experts that needs it on the host reads it there itself.  The gradient
    is not differentiable again.  As for any operation, a backward is captured into a graph only while no graph recorded
    outside the capture over the same leaves is alive."""
    ops._require_device(x, topk_ids)
    ops.dtype_code(x.dtype)
    if x.dim() != 2 or topk_ids.dim() != 2 or topk_ids.shape[0] != x.shape[0]:
        raise ValueError(f"x must be [T, H] and topk_ids [T, top_k], got {tuple(x.shape)} and {tuple(topk_ids.shape)}")
    num_experts = int(num_experts)
    if not 1 <= num_experts <= 1024 or not 1 <= topk_ids.shape[1] <= 1024:
        raise ValueError(f"1 to 1024 experts and 1 to 1024 routes a token, got {num_experts} and {topk_ids.shape[1]}")
    if topk_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"topk_ids must be int32 or int64, got {topk_ids.dtype}")
    topk_ids = topk_ids.contiguous()
    index = _index(topk_ids, num_experts)
    run = _Sort.apply if _derivative_asked("moe_sort", None, x) else _sorted
    return run(x, topk_ids, num_experts, index), MoERoutes(*index)


def moe_unsort(rows: torch.Tensor, topk_weights: torch.Tensor | None, routes: MoERoutes) -> torch.Tensor:
    """``out[t] = sum_j topk_weights[t, j] * rows[routes.places[t, j]]``, ``[T, H]`` in ``rows``' type: fp32 sums in slot order,
    one rounding; differentiable in ``rows`` and ``topk_weights``.

    ``rows [T * top_k, H]`` (fp16, bf16 or fp32) in the order of ``routes``, which :func:`moe_sort` gave; ``topk_weights``: fp16,
    bf16 or fp32 ``[T, top_k]``, all 1 where it is None.  A route without a place adds nothing, its weight's gradient is 0;
    what rows behind the last hold is not read, their gradient is 0.  The gradients are not differentiable again.  As for any
    operation, a backward is captured into a graph only while no graph recorded outside the capture over the same leaves is alive."""
    offsets, _, places = routes
    ops._require_device(rows, topk_weights, offsets, places)
    ops.dtype_code(rows.dtype)
    if places.dtype != torch.int32 or offsets.dtype != torch.int32:
        raise TypeError(f"routes must be int32, got {places.dtype} and {offsets.dtype}")
    if places.dim() != 2 or places.shape[1] < 1 or offsets.dim() != 1 or offsets.shape[0] < 2:
        raise ValueError(f"routes must hold places [T, top_k] and offsets [E + 1], got {tuple(places.shape)} and {tuple(offsets.shape)}")
    if rows.dim() != 2 or rows.shape[0] != places.numel():
        raise ValueError(f"rows must be [{places.numel()}, H], got {tuple(rows.shape)}")
    if topk_weights is not None:
        ops.dtype_code(topk_weights.dtype)
        if topk_weights.shape != places.shape:
            raise ValueError(f"topk_weights must be {tuple(places.shape)}, got {tuple(topk_weights.shape)}")
        topk_weights = topk_weights.contiguous()
    rows, places = rows.contiguous(), places.contiguous()
    if _derivative_asked("moe_unsort", None, rows, topk_weights):
        return _Unsort.apply(rows, topk_weights, places, offsets)
    return _unsorted(rows, topk_weights, places)
