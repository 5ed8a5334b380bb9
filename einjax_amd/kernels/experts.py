"""Expert operators on the GPU: the routing relation, and rows and products in
8-bit integers.

A mixture of experts is a relation between tokens and experts that every call
makes anew: ``route_experts`` (or ``group_by_expert``, for picks that the caller
made) makes it, the grouped products contract over it and ``combine_experts``
takes their rows back to the tokens.  The sizes of the groups stay on the
device: no call waits for the GPU.  The differentiable operators are in
``autodiff/experts.py``.

All tensors are on the GPU; work runs on torch's current stream of their
device.  Arguments are checked, and the library called, by the compiled binding
(``csrc/experts_torch.cpp``).
"""

from __future__ import annotations

from dataclasses import dataclass

import torch

from .. import _lib


@dataclass
class ExpertRouting:
    """The relation of T tokens to their k experts, grouped by expert.

    A slot is one (token, expert) pair; slots of one expert follow each other,
    in token order.

    weights: float32 [T, k], what each expert's result counts for the token;
    experts: int32 [T, k], -1 where a token has fewer than k experts;
    offsets: int32 [E + 1], slots [offsets[e], offsets[e + 1]) are expert e's;
    rows: int32 [T * k], the token of each slot (0 past the last slot in use);
    slots: int32 [T, k], the slot of each pair (-1 where there is none); no two
    pairs have the same slot, and rows[slots[t, j]] = t.

    A caller may take single pairs out by setting their slot to -1 (an expert's
    capacity, say) before the relation is used.  ``combine_experts`` then leaves them out, and the gradient
    to their rows is zero.  The products, which go by offsets and rows, still
    compute those rows and take them into the gradient to the weights; the
    gradient to gathered rows, which adds up a token's slots, does not.  The two
    agree where the rows are used through ``combine_experts`` alone.
    """

    weights: torch.Tensor
    experts: torch.Tensor
    offsets: torch.Tensor
    rows: torch.Tensor
    slots: torch.Tensor

    @property
    def n_experts(self) -> int:
        return self.offsets.shape[0] - 1

    @property
    def n_tokens(self) -> int:
        return self.slots.shape[0]

    @property
    def n_slots(self) -> int:
        return self.rows.shape[0]


def group_args(groups) -> tuple:
    """(offsets, rows, slots) of an ``ExpertRouting``, or of offsets alone."""
    if isinstance(groups, ExpertRouting):
        return groups.offsets, groups.rows, groups.slots
    return groups, None, None


def group_by_expert(experts, n_experts: int, weights=None) -> ExpertRouting:
    """The routing of picks that the caller made: experts [T, k], int32 or
    int64, distinct for each token, -1 (or anything outside [0, n_experts), such
    as experts held elsewhere) for none; weights float32 [T, k], 1 for every pair
    if not given.  At most 1024 experts and 16 picks; there may be more picks
    than experts."""
    return ExpertRouting(*_lib.experts().group(experts, n_experts, weights))


def quantize_rows(x) -> tuple:
    """x [..., n] in 8-bit integers with a scale for each row: (q int8 of x's
    shape, scale float32 of x's shape without the last extent), x ~ q scale.

    scale = max |row| / 127, q rounded to nearest (ties to even).  A row of
    zeros has scale 0; a row that holds a NaN or an infinity has scale NaN, so
    that every product with it is NaN.  Rows of activations give a scale for
    each token, rows of [experts, n_out, n_in] weights one for each channel.
    Not differentiable: q and scale are constants to torch.autograd."""
    return _lib.experts().quantize_rows(x)


def int8_matmul(q, q_scale, w, w_scale, groups=None, *, gather: bool = False,
                out_dtype: torch.dtype = torch.bfloat16):
    """Product of 8-bit rows and 8-bit weights with their scales.

    q int8 [m, k] and q_scale float32 [m] are rows and their scales
    (``quantize_rows``); w int8 holds one row of k for each output channel,
    w_scale float32 their scales.  The integer sum is exact (k < 131072), times
    both scales in float32 (whose own product may pass its range), rounded once to
    out_dtype (float32, bfloat16 or float16).

    Without groups: w [n, k] or [1, n, k], w_scale [n] or [1, n], the dense
    product [m, n].  With groups (an ``ExpertRouting`` or offsets [E + 1]):
    w [E, n, k], w_scale [E, n]; slot s of group e is q's row s, or with
    ``gather`` the row of its token, times w[e]; zero in slots of no group.

    Not differentiable, in the scales either: the result is a constant to
    torch.autograd."""
    offsets, rows, slots = group_args(groups)
    return _lib.experts().int8_matmul(q, q_scale, w, w_scale, offsets, rows, slots, gather,
                                      out_dtype)
