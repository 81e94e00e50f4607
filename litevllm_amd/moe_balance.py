"""The load-balancing loss of a mixture of experts and the routes per expert, beside :func:`moe_route`, whose
logits and ids it takes."""
from __future__ import annotations

import torch

from . import _lib as L
from . import ops
from .mxfp4 import _call, _derivative_asked, _Refused


def _rows(logits: torch.Tensor) -> torch.Tensor:
    """``logits``, or a copy, as rows that the kernels can read."""
    t, e = logits.shape
    if (logits.stride(1) != 1 and e > 1) or (t > 1 and logits.stride(0) < e):
        return logits.contiguous()
    return logits


def _forward(logits, ids, mask, experts):
    """(loss, counts, buf): the gradient's factors are the first ``experts`` floats of ``buf``, scratch the rest."""
    dev, t = logits.device, logits.shape[0]
    ws_bytes = L.load().awq_w4a16_moe_balance_workspace_bytes(t, experts)
    start = -(-experts // 4) * 4  # scratch on a 16-byte boundary
    buf = torch.empty(start + ws_bytes // 4, dtype=torch.float32, device=dev)
    loss = torch.empty((), dtype=torch.float32, device=dev)
    counts = torch.empty(experts, dtype=torch.int32, device=dev)
    at = buf.data_ptr()
    _call(dev, "awq_w4a16_moe_balance", logits.data_ptr(), logits.stride(0) if t > 1 else experts, ops.dtype_code(logits.dtype),
          ids.data_ptr(), 64 if ids.dtype == torch.int64 else 32, ops._ptr(mask), t, experts, ids.shape[1], loss.data_ptr(),
          counts.data_ptr(), at, at + 4 * start, ws_bytes)
    return loss, counts, buf


class _BalanceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, ids, mask, experts):
        loss, counts, buf = _forward(logits, ids, mask, experts)
        ctx.save_for_backward(logits, mask, buf)
        ctx.mark_non_differentiable(counts)
        ctx.set_materialize_grads(False)  # no zeros in place of the counts' gradient
        ctx.shape = logits.shape
        return loss, counts

    @staticmethod
    def backward(ctx, upstream, _):
        if upstream is None:
            return None, None, None, None
        # saved-tensor hooks may give back copies with other strides
        logits, mask, buf = ctx.saved_tensors
        inputs = logits, upstream
        on, (t, experts) = upstream.get_device(), ctx.shape
        if logits.get_device() != on or buf.get_device() != on or logits.shape != ctx.shape or (
                buf.dtype is not torch.float32 or buf.numel() < experts) or (
                mask is not None and (mask.get_device() != on or mask.dtype is not torch.bool or mask.shape != (t,))):
            raise RuntimeError("moe_balance_loss: saved tensors came back elsewhere, or with other shapes or types")
        ld = experts
        if not logits.is_contiguous():
            logits = _rows(logits)
            ld = logits.stride(0)
        mask, buf = None if mask is None else mask.contiguous(), buf.contiguous()
        grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
        _call(logits.device, "awq_w4a16_moe_balance_grad", logits.data_ptr(), ld,
              ops.dtype_code(logits.dtype), ops._ptr(mask), buf.data_ptr(), upstream.data_ptr(), grad.data_ptr(), t, experts)
        if torch.is_grad_enabled():  # create_graph: a second derivative is refused, not taken as zero
            grad = _Refused.apply("moe_balance_loss is not differentiable twice", grad, *inputs)
        return grad, None, None, None


def moe_balance_loss(router_logits: torch.Tensor, topk_ids: torch.Tensor,
                     mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``(loss, counts)`` of a router: ``loss`` an fp32 scalar, differentiable in ``router_logits``, ``counts`` int32
    ``[E]``, the routes of every expert.

    With ``n`` kept tokens (``mask [T]`` bool, True keeps; all without one), ``p = softmax(router_logits)`` in fp32::

        loss = E * sum_e (counts[e] / (n * top_k)) * (sum over kept t of p[t, e] / n)

    which is 1 for an even load.  ``router_logits``: fp16, bf16 or fp32 ``[T, E]`` (E up to 1024); ``topk_ids``: int32 or
    int64 ``[T, top_k]``; ids outside ``[0, E)`` count nowhere.  What a masked row holds is not read and its
    gradient is 0; without a kept token loss and gradient are 0.  A row of nothing but ``-inf`` has no
    probabilities.  The gradient takes the counts as constants; it is not differentiable again.  As for any operation, a backward is
    captured into a graph only while no graph recorded outside the capture over the same leaves is alive."""
    ops._require_device(router_logits, topk_ids, mask)
    ops.dtype_code(router_logits.dtype)
    if router_logits.dim() != 2 or topk_ids.dim() != 2 or topk_ids.shape[0] != router_logits.shape[0]:
        raise ValueError(f"router_logits must be [T, E] and topk_ids [T, top_k], got {tuple(router_logits.shape)} and "
                         f"{tuple(topk_ids.shape)}")
    experts = router_logits.shape[1]
    if not 1 <= experts <= 1024 or topk_ids.shape[1] < 1:
        raise ValueError(f"1 to 1024 experts and at least one route a token, got {experts} and {topk_ids.shape[1]}")
    if topk_ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"topk_ids must be int32 or int64, got {topk_ids.dtype}")
    if mask is not None:
        if mask.dtype != torch.bool or mask.shape != router_logits.shape[:1]:
            raise ValueError(f"mask must be bool [{router_logits.shape[0]}], got {mask.dtype} {tuple(mask.shape)}")
        mask = mask.contiguous()
    router_logits, topk_ids = _rows(router_logits), topk_ids.contiguous()
    if _derivative_asked("moe_balance_loss", None, router_logits):
        return _BalanceLoss.apply(router_logits, topk_ids, mask, experts)
    return _forward(router_logits, topk_ids, mask, experts)[:2]
