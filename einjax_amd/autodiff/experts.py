"""Differentiable expert operators.

``route_experts``, ``grouped_matmul`` and ``combine_experts`` are
``torch.autograd`` functions over the library's kernels; their backward
kernels are also callable directly (``*_vjp``).  Gradients are first order,
as ``sparse_einsum_raw``'s.  The reference has no such operators.
"""

from __future__ import annotations

import torch

from ..kernels import experts as K
from ..kernels.experts import ExpertRouting

__all__ = ["route_experts", "route_experts_vjp", "grouped_matmul", "grouped_matmul_vjp",
           "combine_experts", "combine_experts_vjp"]


class _Route(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k, renormalize, made):
        r = K.route(logits, k, renormalize)
        made.append(r)
        ctx.renormalize = renormalize
        ctx.save_for_backward(logits, r.experts)
        return r.weights

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        logits, experts = ctx.saved_tensors
        return K.route_vjp(logits, experts, g, ctx.renormalize), None, None, None


def route_experts(logits, k: int, *, renormalize: bool = True) -> ExpertRouting:
    """Each token's k experts and their weights, grouped by expert.

    logits [T, E] (float32, bfloat16 or float16; at most 1024 experts, k at
    most 16).  A token's picks are its k largest logits, equal ones in the
    order of their experts; weights are the softmax over the picks, or over all
    logits with ``renormalize=False``.  A logit of -inf excludes its expert: a
    token with fewer than k experts left has experts -1 and weights 0 for the
    rest (a padding token: all logits -inf).  NaN and +inf logits give NaN
    weights.  ``weights`` carries the gradient to the logits; the picks are
    constants."""
    if not (isinstance(logits, torch.Tensor) and logits.requires_grad and torch.is_grad_enabled()):
        return K.route(logits, k, renormalize)
    made = []  # the routing with its integers, which autograd need not see
    weights = _Route.apply(logits, k, renormalize, made)
    r = made[0]
    return ExpertRouting(weights, r.experts, r.offsets, r.rows, r.slots)


def route_experts_vjp(logits, experts, grad_weights, *, renormalize: bool = True):
    """Gradient of ``route_experts``' weights to the logits, for the picks
    ``experts`` that it returned."""
    K.on_gpu(logits, "logits")
    K.on_gpu(experts, "experts")
    if logits.dim() != 2 or experts.dim() != 2 or experts.shape[0] != logits.shape[0]:
        raise ValueError(f"logits {tuple(logits.shape)} and experts {tuple(experts.shape)} must "
                         "be [tokens, experts] and [tokens, k]")
    return K.route_vjp(logits, experts, grad_weights, renormalize)


def _check_product(x, w, out_dtype) -> torch.dtype:
    K.on_gpu(x, "x")
    K.on_gpu(w, "w")
    if x.dim() != 2 or w.dim() != 3 or x.shape[1] != w.shape[1]:
        raise ValueError(f"x {tuple(x.shape)} and w {tuple(w.shape)} must be [rows, k] and "
                         "[groups, k, n]")
    if x.dtype != w.dtype or x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"x and w must share float32, bfloat16 or float16, got {x.dtype} and "
                        f"{w.dtype}")
    if x.device != w.device:
        raise ValueError(f"w is on {w.device}, expected {x.device}")
    dt = x.dtype if out_dtype is None else out_dtype
    if dt not in (torch.float32, x.dtype):
        raise TypeError(f"out_dtype must be float32 or {x.dtype}, got {dt}")
    return dt


class _GroupedMatmul(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, groups, out_dtype):
        ctx.groups = groups
        ctx.save_for_backward(x, w)
        return K.grouped_product(x, w, groups, out_dtype)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, w = ctx.saved_tensors
        return (*_product_vjp(x, w, ctx.groups, g, ctx.needs_input_grad[0],
                              ctx.needs_input_grad[1]), None, None)


def _product_vjp(x, w, groups, grad, need_x, need_w):
    # an fp32 cotangent of 16-bit operands is rounded to their type: both
    # gradients are 16-bit products with fp32 sums
    if grad.dtype is not x.dtype:
        grad = grad.to(x.dtype)
    gx = gw = None
    if need_x:
        # gathered rows: each slot's gradient stays in fp32 until a token's
        # slots are summed, so that the sum is rounded once
        slots = K.Groups(groups.offsets, None, None, groups.n_slots)
        summed = groups.rows is not None
        gx = K.grouped_product(grad, w.transpose(1, 2), slots, torch.float32 if summed else x.dtype)
        if summed:
            gx = K.combine(gx, groups.slots, None, x.dtype)
    if need_w:
        gw = K.grouped_weight_gradient(x, w, groups, grad)
    return gx, gw


def grouped_matmul(x, w, groups, *, gather: bool = False, out_dtype=None):
    """Products grouped by expert: out[s] = x[s] @ w[e] for the slots s of
    group e.

    w [E, k, n], n- or k-contiguous (``weight.transpose(1, 2)`` of linear
    weights [E, n, k] is taken as it lies).  groups: an ``ExpertRouting``, or
    offsets [E + 1] (non-decreasing, int32 or int64, on the GPU) of rows that
    are already grouped.  x [slots, k]; with ``gather=True`` x [tokens, k] and
    slot s takes its token's row, without a copy.  Rows of no group are zero.
    float32, bfloat16 or float16, summed in fp32; the result has x's dtype
    unless ``out_dtype=torch.float32``.  Differentiable in x and w; the
    gradient to w lies as w does."""
    dt = _check_product(x, w, out_dtype)
    g = K.groups_of(x, w.shape[0], groups, gather)
    if not ((x.requires_grad or w.requires_grad) and torch.is_grad_enabled()):
        return K.grouped_product(x, w, g, dt)
    return _GroupedMatmul.apply(x, w, g, dt)


def grouped_matmul_vjp(x, w, groups, grad_out, *, gather: bool = False, need_x: bool = True,
                       need_w: bool = True):
    """(grad_x, grad_w) of ``grouped_matmul`` for the cotangent grad_out
    [slots, n]; None where not needed."""
    _check_product(x, w, None)
    g = K.groups_of(x, w.shape[0], groups, gather)
    K.on_gpu(grad_out, "grad_out")
    if tuple(grad_out.shape) != (g.n_slots, w.shape[2]):
        raise ValueError(f"grad_out has shape {tuple(grad_out.shape)}, expected "
                         f"{(g.n_slots, w.shape[2])}")
    return _product_vjp(x.detach(), w.detach(), g, grad_out, need_x, need_w)


class _Combine(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, slots, offsets):
        ctx.save_for_backward(y, weights, slots, offsets)
        return K.combine(y, slots, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        y, weights, slots, offsets = ctx.saved_tensors
        return (*K.combine_vjp(y, slots, offsets, weights, g, ctx.needs_input_grad[0],
                               ctx.needs_input_grad[1]), None, None)


def _check_combine(y, routing, weights):
    K.on_gpu(y, "y")
    if not isinstance(routing, ExpertRouting):
        raise TypeError("routing must be an ExpertRouting")
    if y.dim() != 2 or y.shape[0] != routing.n_slots:
        raise ValueError(f"y has shape {tuple(y.shape)}, expected [{routing.n_slots}, n]: a row "
                         "for each slot of the routing")
    if y.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"y must be float32, bfloat16 or float16, got {y.dtype}")
    weights = routing.weights if weights is None else weights
    K._same_device(y, weights=weights, slots=routing.slots, offsets=routing.offsets)
    if weights.dtype != torch.float32 or weights.shape != routing.slots.shape:
        raise ValueError(f"weights must be float32 {tuple(routing.slots.shape)}, got "
                         f"{weights.dtype} {tuple(weights.shape)}")
    return (weights if weights.is_contiguous() else weights.contiguous(), K._index(routing.slots, routing.slots.shape, "slots"),
            K._index(routing.offsets, (routing.n_experts + 1,), "offsets"))


def combine_experts(y, routing: ExpertRouting, weights=None):
    """Back to tokens: out[t] = sum over j of weights[t, j] y[slots[t, j]].

    y [slots, n] (float32, bfloat16 or float16), a row for each slot; weights
    float32 [T, k], by default the routing's own.  Summed in fp32 in the order
    of the picks and rounded once to y's dtype; pairs without a slot are left
    out (a token without any gets zeros).  Differentiable in y and weights."""
    weights, slots, offsets = _check_combine(y, routing, weights)
    if not ((y.requires_grad or weights.requires_grad) and torch.is_grad_enabled()):
        return K.combine(y, slots, weights)
    return _Combine.apply(y, weights, slots, offsets)


def combine_experts_vjp(y, routing: ExpertRouting, grad_out, weights=None, *, need_y: bool = True,
                        need_weights: bool = True):
    """(grad_y, grad_weights) of ``combine_experts`` for the cotangent
    grad_out [T, n]; None where not needed."""
    weights, slots, offsets = _check_combine(y, routing, weights)
    K.on_gpu(grad_out, "grad_out")
    if tuple(grad_out.shape) != (slots.shape[0], y.shape[1]):
        raise ValueError(f"grad_out has shape {tuple(grad_out.shape)}, expected "
                         f"{(slots.shape[0], y.shape[1])}")
    return K.combine_vjp(y.detach(), slots, offsets, weights.detach(), grad_out.to(y.dtype),
                         need_y, need_weights)
