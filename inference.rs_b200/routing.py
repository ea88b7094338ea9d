"""Tokens sorted by expert and back: what a layer of experts does before and after its products, with the gradients of both.

A router gives every token a few experts (`ids`) and a weight for each. `TokenRouting` sorts the slots by expert once; `dispatch` brings
the tokens into that order, one row per slot, `combine` adds a token's rows up again with the weights applied. Both can be
differentiated in reverse mode (what carries a tangent of forward mode is refused); their sums run in slot order and in 32 bits, so
that results and gradients are the same bits every time.
"""
from __future__ import annotations

import math

import torch

from . import kernel_library as kl
from . import ops


def _no_tangent(*tensors: torch.Tensor) -> None:
    if ops.has_tangent(*tensors):
        raise NotImplementedError("the routing of tokens has no derivatives in forward mode, nor do its gradients")


class _Once(torch.autograd.Function):
    """Passes a gradient on that is not to be differentiated again."""

    @staticmethod
    def forward(ctx, grad):
        return grad

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("the gradients of token routing cannot be differentiated again")


def _once(grad: torch.Tensor | None, *sources: torch.Tensor) -> torch.Tensor | None:
    """A gradient made of `sources`: under create_graph one that raises if it is differentiated, towards whichever of them."""
    if grad is None or not torch.is_grad_enabled() or not any(t.requires_grad for t in sources):
        return grad
    return _Once.apply(grad.requires_grad_())


class _Dispatch(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, position, offsets):
        ctx.save_for_backward(position)
        ctx.dtype = x.dtype
        return ops.route_dispatch(x, position, offsets)

    @staticmethod
    def backward(ctx, grad):
        (position,) = ctx.saved_tensors
        _no_tangent(grad)
        return _once(ops.route_combine(grad, position, None, ctx.dtype), grad), None, None


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, rows, weights, position, offsets, out_dtype):
        ctx.save_for_backward(rows, weights, position, offsets)
        return ops.route_combine(rows, position, weights, out_dtype)

    @staticmethod
    def backward(ctx, grad):
        rows, weights, position, offsets = ctx.saved_tensors
        _no_tangent(grad)
        need_rows, need_weights = ctx.needs_input_grad[:2]
        grad_rows, grad_weights = ops.route_combine_grad(grad, rows, position, offsets, weights, need_rows, need_weights)
        return _once(grad_rows, grad, weights), _once(grad_weights, grad, rows), None, None, None


class TokenRouting:
    """The slots of `ids` [..., slots per token] (int32 or int64) sorted by expert.

    order [slots]: the slot of each row, -1 behind the last; offsets [experts + 1]: where each expert's rows start; position
    [*ids.shape]: the row of each slot, -1 where its id is not one of 0..experts - 1 (an expert of another rank, a dropped token). Slots
    of one expert keep their order. All int32, on the device of `ids`; nothing is copied to the host."""

    def __init__(self, ids: torch.Tensor, experts: int):
        if ids.dim() < 2:
            raise ValueError(f"expert ids have a dimension for the tokens and one for their slots, got {tuple(ids.shape)}")
        if ids.shape[-1] == 0:
            raise ValueError(f"tokens with no slots: {tuple(ids.shape)}")
        self.experts = int(experts)
        sorted_slots = kl.host().route_sort(ids, self.experts)
        self.order, self.offsets, self.position = ops.route_sort(ids, self.experts) if sorted_slots is None else sorted_slots

    def _position2d(self) -> torch.Tensor:
        return self.position.view(math.prod(self.position.shape[:-1]), self.position.shape[-1])

    def dispatch(self, x: torch.Tensor) -> torch.Tensor:
        """x [..., h], a row per token -> [slots, h], a row per slot in the order of the experts; rows behind the last expert's are zeros."""
        if tuple(x.shape[:-1]) != tuple(self.position.shape[:-1]):
            raise ValueError(f"tokens {tuple(x.shape)} for expert ids {tuple(self.position.shape)}")
        rows = kl.host().route_dispatch(x, self.position, self.offsets) if x.dim() == 2 == self.position.dim() else None
        if rows is not None:
            return rows
        _no_tangent(x)
        position = self._position2d()
        x2 = x.reshape(position.shape[0], x.shape[-1])
        if torch.is_grad_enabled() and x2.requires_grad:
            return _Dispatch.apply(x2, position, self.offsets)
        return ops.route_dispatch(x2, position, self.offsets)

    def combine(self, rows: torch.Tensor, weights: torch.Tensor, out_dtype: torch.dtype | None = None) -> torch.Tensor:
        """rows [slots, h] as `dispatch` orders them, weights [..., slots per token] -> [..., h] in `out_dtype` (that of the rows): each
        token's rows times its weights. Slots without an expert count for nothing, whatever their weight; rows behind the last
        expert's are not read."""
        if tuple(weights.shape) != tuple(self.position.shape):
            raise ValueError(f"weights {tuple(weights.shape)} for expert ids {tuple(self.position.shape)}")
        out_dtype = rows.dtype if out_dtype is None else out_dtype
        w = weights.to(torch.float32).contiguous()
        out = kl.host().route_combine(rows, w, self.position, self.offsets, ops.elem_of(out_dtype))
        if out is not None:
            return out if weights.dim() == 2 else out.view(*weights.shape[:-1], rows.shape[-1])
        _no_tangent(rows, w)
        position = self._position2d()
        w = w.view(position.shape)
        if torch.is_grad_enabled() and (rows.requires_grad or w.requires_grad):
            out = _Combine.apply(rows, w, position, self.offsets, out_dtype)
        else:
            out = ops.route_combine(rows, position, w, out_dtype)
        return out.view(*weights.shape[:-1], rows.shape[-1])
