"""Differentiable expert operators.

``route_experts``, ``grouped_matmul`` and ``combine_experts`` carry gradients
through torch.autograd; their backward kernels are also callable directly
(``*_vjp``).  Gradients are first order, as ``sparse_einsum_raw``'s, and
reverse mode only: dual tensors are refused.  The reference has no such
operators.
"""

from __future__ import annotations

from .. import _lib
from ..kernels.experts import ExpertRouting, group_args

__all__ = ["route_experts", "route_experts_vjp", "grouped_matmul", "grouped_matmul_vjp",
           "combine_experts", "combine_experts_vjp"]


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
    return ExpertRouting(*_lib.experts().route(logits, k, renormalize))


def route_experts_vjp(logits, experts, grad_weights, *, renormalize: bool = True):
    """Gradient of ``route_experts``' weights to the logits, for the picks
    ``experts`` that it returned."""
    return _lib.experts().route_vjp(logits, experts, grad_weights, renormalize)


def grouped_matmul(x, w, groups, *, gather: bool = False, out_dtype=None):
    """Products grouped by expert: out[s] = x[s] @ w[e] for the slots s of
    group e.

    w [E, k, n], n- or k-contiguous (``weight.transpose(1, 2)`` of linear
    weights [E, n, k] is taken as it lies).  groups: an ``ExpertRouting``, or
    offsets [E + 1] (non-decreasing, int32 or int64, on the GPU) of rows that
    are already grouped.  x [slots, k]; with ``gather=True`` x [tokens, k] and
    slot s takes its token's row, without a copy (the gradient to x is the sum
    over routing.slots, see ``ExpertRouting`` on pairs taken out).  Rows of no
    group are zero.
    float32, bfloat16 or float16, summed in fp32; the result has x's dtype
    unless ``out_dtype=torch.float32``.  Differentiable in x and w (in gathered
    x for routings of 1 to 16 picks); the gradient to w lies as w does.  Both
    gradients are products in x's dtype, summed in fp32: the float32 cotangent of
    an ``out_dtype=torch.float32`` product is rounded to x's dtype before them
    (in float16 beyond 65504 to infinity)."""
    offsets, rows, slots = group_args(groups)
    return _lib.experts().grouped_matmul(x, w, offsets, rows, slots, gather, out_dtype)


def grouped_matmul_vjp(x, w, groups, grad_out, *, gather: bool = False, need_x: bool = True,
                       need_w: bool = True):
    """(grad_x, grad_w) of ``grouped_matmul`` for the cotangent grad_out
    [slots, n], which is rounded to x's dtype; None where not needed."""
    offsets, rows, slots = group_args(groups)
    return _lib.experts().grouped_matmul_vjp(x, w, offsets, rows, slots, gather, grad_out, need_x,
                                             need_w)


def _combine_args(y, routing, weights) -> tuple:
    if not isinstance(routing, ExpertRouting):
        raise TypeError("routing must be an ExpertRouting")
    return (y, routing.weights if weights is None else weights, routing.slots, routing.offsets)


def combine_experts(y, routing: ExpertRouting, weights=None):
    """Back to tokens: out[t] = sum over j of weights[t, j] y[slots[t, j]].

    y [slots, n] (float32, bfloat16 or float16), a row for each slot; weights
    float32 [T, k], by default the routing's own.  Summed in fp32 in the order
    of the picks and rounded once to y's dtype; pairs without a slot are left
    out (a token without any gets zeros).  Differentiable in y (rows that no
    pair holds have a gradient of zero) and weights."""
    return _lib.experts().combine(*_combine_args(y, routing, weights))


def combine_experts_vjp(y, routing: ExpertRouting, grad_out, weights=None, *, need_y: bool = True,
                        need_weights: bool = True):
    """(grad_y, grad_weights) of ``combine_experts`` for the cotangent
    grad_out [T, n], which is rounded to y's dtype; None where not needed."""
    return _lib.experts().combine_vjp(*_combine_args(y, routing, weights), grad_out, need_y,
                                      need_weights)
