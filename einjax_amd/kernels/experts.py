"""Expert operators on the GPU: routing, products grouped by expert, the
weighted sum back to tokens, rows in 8-bit integers.

A mixture of experts is a relation between tokens and experts that every call
makes anew: ``route`` makes it (``ExpertRouting``), the grouped products
contract over it and ``combine`` takes their rows back to the tokens.  The
sizes of the groups stay on the device: no call waits for the GPU.  These
functions compute without gradients; the differentiable forms, under the names
the package exports, are in ``autodiff/experts.py``.

All tensors are on the GPU and work runs on torch's current stream.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass
from math import prod

import torch

from .. import _device, _lib
from .._lib import check

_DTYPES = {torch.float32: _lib.EJ_F32, torch.bfloat16: _lib.EJ_BF16, torch.float16: _lib.EJ_F16}


@dataclass
class ExpertRouting:
    """The relation of T tokens to their k experts, grouped by expert.

    A slot is one (token, expert) pair; slots of one expert follow each other,
    in token order.

    weights: float32 [T, k], what each expert's result counts for the token;
    experts: int32 [T, k], -1 where a token has fewer than k experts;
    offsets: int32 [E + 1], slots [offsets[e], offsets[e + 1]) are expert e's;
    rows: int32 [T * k], the token of each slot (0 past the last slot in use);
    slots: int32 [T, k], the slot of each pair (-1 where there is none).
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


def on_gpu(t, what: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{what} must be a torch tensor on the GPU")
    return t


def _same_device(ref: torch.Tensor, **tensors) -> None:
    dev = ref.get_device()
    for name, t in tensors.items():
        if t is not None and on_gpu(t, name).get_device() != dev:
            raise ValueError(f"{name} is on {t.device}, expected {ref.device}")


def _value_code(t: torch.Tensor, what: str) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _index(t: torch.Tensor, shape: tuple, what: str) -> torch.Tensor:
    if t.shape != shape:
        raise ValueError(f"{what} has shape {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype is not torch.int32:
        if t.dtype is not torch.int64:
            raise TypeError(f"{what} must be int32 or int64, got {t.dtype}")
        t = t.to(torch.int32)
    return t if t.is_contiguous() else t.contiguous()


def rows_of(t: torch.Tensor) -> torch.Tensor:
    """t [n, m] with unit stride along its rows and rows that do not overlap
    (itself if it is so already)."""
    if t.is_contiguous():
        return t
    n, m = t.shape
    if (m <= 1 or t.stride(1) == 1) and (n <= 1 or t.stride(0) >= m):
        return t
    return t.contiguous()


def _row_stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _ptr(t: torch.Tensor | None):
    return None if t is None else t.data_ptr()


_entry_points: dict = {}


def _call(ref: torch.Tensor, name: str, *args) -> None:
    """The library's `name` on the device of ref, on that device's current
    stream of torch.  Pointers are plain integers: these calls last a few
    microseconds, of which building ctypes objects would be a good part."""
    fn = _entry_points.get(name)
    if fn is None:
        fn = _entry_points[name] = getattr(_lib.load(), name)
    dev = ref.get_device()
    if dev == _device.current_device_index():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if status:
        check(status, name)


def _route_workspace(ref: torch.Tensor, n_tokens: int, n_experts: int):
    """(workspace tensor or None, its size)."""
    nbytes = ctypes.c_size_t()
    check(_lib.load().ej_expert_route_workspace_size(n_tokens, n_experts, ctypes.byref(nbytes)),
          "ej_expert_route_workspace_size")
    n = nbytes.value
    return (_device.workspace(n, ref.device) if n else None), n


def _empty_routing(ref: torch.Tensor, n_tokens: int, k: int, n_experts: int):
    """offsets, rows, slots [T, k] and a spare int32 [T, k] in one allocation."""
    n = n_tokens * k
    buf = torch.empty(3 * n + n_experts + 1, dtype=torch.int32, device=ref.device)
    rows, slots, spare, offsets = buf.split((n, n, n, n_experts + 1))
    return offsets, rows, slots.view(n_tokens, k), spare.view(n_tokens, k)


def route(logits: torch.Tensor, k: int, renormalize: bool) -> ExpertRouting:
    on_gpu(logits, "logits")
    if logits.dim() != 2:
        raise ValueError(f"logits must be [tokens, experts], got shape {tuple(logits.shape)}")
    code = _value_code(logits, "logits")
    T, E = logits.shape
    k = int(k)
    if not 1 <= k <= max(E, 1):
        raise ValueError(f"k = {k}, expected 1 to the number of experts, {E}")
    logits = rows_of(logits)
    ws, ws_bytes = _route_workspace(logits, T, E)
    weights = torch.empty((T, k), dtype=torch.float32, device=logits.device)
    offsets, rows, slots, experts = _empty_routing(logits, T, k, E)
    p = _ptr
    _call(logits, "ej_expert_route", p(logits), code, T, E, max(_row_stride(logits), E), k,
          1 if renormalize else 0, p(weights), p(experts), p(offsets), p(rows), p(slots), p(ws),
          ws_bytes)
    return ExpertRouting(weights, experts, offsets, rows, slots)


def group_by_expert(experts: torch.Tensor, n_experts: int,
                    weights: torch.Tensor | None = None) -> ExpertRouting:
    """The routing of picks that the caller made: experts [T, k], int32 or
    int64, distinct for each token, -1 (or anything outside [0, n_experts))
    for none; weights float32 [T, k], 1 for every pair if not given."""
    on_gpu(experts, "experts")
    if experts.dim() != 2:
        raise ValueError(f"experts must be [tokens, k], got shape {tuple(experts.shape)}")
    T, k = experts.shape
    E = int(n_experts)
    if weights is None:
        weights = torch.ones((T, k), dtype=torch.float32, device=experts.device)
    _same_device(experts, weights=weights)
    if tuple(weights.shape) != (T, k) or weights.dtype != torch.float32:
        raise ValueError(f"weights must be float32 {(T, k)}, got {weights.dtype} "
                         f"{tuple(weights.shape)}")
    if experts.dtype == torch.int64:  # no wrapping of values past 32 bits into the range
        experts = experts.clamp(-1, E)
    experts = _index(experts, (T, k), "experts")
    ws, ws_bytes = _route_workspace(experts, T, E)
    offsets, rows, slots, _ = _empty_routing(experts, T, k, E)
    p = _ptr
    _call(experts, "ej_expert_group", p(experts), T, k, E, p(offsets), p(rows), p(slots), p(ws),
          ws_bytes)
    return ExpertRouting(weights, experts, offsets, rows, slots)


def route_vjp(logits: torch.Tensor, experts: torch.Tensor, grad_weights: torch.Tensor,
              renormalize: bool) -> torch.Tensor:
    on_gpu(logits, "logits")
    T, E = logits.shape
    k = experts.shape[1]
    _same_device(logits, experts=experts, grad_weights=grad_weights)
    if tuple(grad_weights.shape) != (T, k):
        raise ValueError(f"grad_weights has shape {tuple(grad_weights.shape)}, expected {(T, k)}")
    code = _value_code(logits, "logits")
    experts = _index(experts, (T, k), "experts")
    grad_weights = grad_weights.to(torch.float32).contiguous()
    logits = rows_of(logits)
    out = torch.empty((T, E), dtype=logits.dtype, device=logits.device)
    p = _ptr
    _call(logits, "ej_expert_route_vjp", p(logits), code, T, E, max(_row_stride(logits), E), k,
          1 if renormalize else 0, p(experts), p(grad_weights), p(out))
    return out


def combine(y: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor | None,
            out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Sum over j of weights[t, j] y[slots[t, j]]; no weights: 1.  In y's
    dtype, or from float32 in out_dtype."""
    y = rows_of(y)
    T, k = slots.shape
    out_dtype = out_dtype or y.dtype
    out = torch.empty((T, y.shape[1]), dtype=out_dtype, device=y.device)
    p = _ptr
    _call(y, "ej_expert_combine", p(y), _value_code(y, "y"), y.shape[0], _row_stride(y),
          p(weights), p(slots), T, k, y.shape[1], p(out), _DTYPES[out_dtype])
    return out


def combine_vjp(y, slots, offsets, weights, grad, need_y: bool, need_weights: bool):
    y, grad = rows_of(y), rows_of(grad)
    T, k = slots.shape
    gy = torch.empty((y.shape[0], y.shape[1]), dtype=y.dtype, device=y.device) if need_y else None
    gw = torch.empty((T, k), dtype=torch.float32, device=y.device) if need_weights else None
    p = _ptr
    _call(y, "ej_expert_combine_vjp", p(y), _value_code(y, "y"), y.shape[0], _row_stride(y),
          p(weights), p(slots), p(offsets), offsets.shape[0] - 1, T, k, y.shape[1], p(grad),
          _row_stride(grad), p(gy), p(gw))
    return gy, gw


def quantize_rows(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., n] in 8-bit integers with a scale for each row: (q int8 of x's
    shape, scale float32 of x's shape without the last extent), x ~ q scale.

    scale = max |row| / 127, q rounded to nearest (ties to even).  A row of
    zeros has scale 0; a row that holds a NaN or an infinity has scale NaN, so
    that every product with it is NaN.  Rows of activations give a scale for
    each token, rows of [experts, n_out, n_in] weights one for each channel."""
    on_gpu(x, "x")
    code = _value_code(x, "x")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    lead, n = x.shape[:-1], x.shape[-1]
    m = prod(lead)
    flat = rows_of(x if x.dim() == 2 else x.reshape(m, n))
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(lead, dtype=torch.float32, device=x.device)
    p = _ptr
    _call(x, "ej_quantize_rows", p(flat), code, m, max(_row_stride(flat), n), n, p(q), p(scale))
    return q, scale


# ---------------------------------------------------------------------------
# Grouped products.


@dataclass
class Groups:
    """What a grouped product reads of its groups: offsets int32 [E + 1]
    (None: one group of every slot), rows (the row of x for each slot, None:
    the slot itself) and, where rows are gathered, the slots of each row for
    the gradient."""

    offsets: torch.Tensor | None
    rows: torch.Tensor | None
    slots: torch.Tensor | None
    n_slots: int


def groups_of(x: torch.Tensor, n_groups: int, groups, gather: bool) -> Groups:
    """Checks x, the number of weight groups and the grouping of a call."""
    if isinstance(groups, ExpertRouting):
        if groups.n_experts != n_groups:
            raise ValueError(f"the routing has {groups.n_experts} experts, the weights have "
                             f"{n_groups}")
        n_slots, n_tokens = groups.n_slots, groups.n_tokens
        want = n_tokens if gather else n_slots
        if x.shape[0] != want:
            raise ValueError(f"x has {x.shape[0]} rows, expected {want} "
                             f"({'tokens' if gather else 'slots'} of the routing)")
        _same_device(x, offsets=groups.offsets, rows=groups.rows, slots=groups.slots)
        offsets = _index(groups.offsets, (n_groups + 1,), "offsets")
        if not gather:
            return Groups(offsets, None, None, n_slots)
        if groups.slots.numel() != n_slots:
            raise ValueError(f"the routing has {groups.slots.numel()} pairs and {n_slots} slots")
        return Groups(offsets, _index(groups.rows, (n_slots,), "rows"),
                      _index(groups.slots, groups.slots.shape, "slots"), n_slots)
    if gather:
        raise ValueError("gather=True needs an ExpertRouting: offsets alone do not say which "
                         "rows the slots take")
    _same_device(x, offsets=groups)
    return Groups(_index(groups, (n_groups + 1,), "offsets"), None, None, x.shape[0])


def weight_order(w: torch.Tensor) -> tuple[torch.Tensor, int, int, int]:
    """(w, order, group stride, row stride) of w [E, k, n] as it lies in
    memory; a copy if neither k nor n is contiguous."""
    E, k, n = w.shape
    if w.is_contiguous():
        return w, _lib.EJ_W_KN, k * n, n
    for _ in range(2):
        for order, rows, cols, rs, cs in ((_lib.EJ_W_KN, k, n, w.stride(1), w.stride(2)),
                                          (_lib.EJ_W_NK, n, k, w.stride(2), w.stride(1))):
            if cols > 1 and cs != 1:
                continue
            rs = rs if rows > 1 else max(cols, 1)
            gs = w.stride(0) if E > 1 else rows * rs
            if rs >= cols and gs >= rows * rs:
                return w, order, gs, rs
        w = w.contiguous()
    raise AssertionError("a contiguous tensor has an order")


def _desc(x, code, out_code, order, E, k, n, n_slots, w_group, w_stride, out_stride):
    return _lib.GroupedDesc(code, out_code, order, E, k, n, n_slots, x.shape[0],
                            max(_row_stride(x), k), w_group, w_stride, out_stride)


def _product_workspace(ref: torch.Tensor, query: str, d):
    """(workspace tensor or None, its size) of a grouped product."""
    nbytes = ctypes.c_size_t()
    check(getattr(_lib.load(), query)(ctypes.byref(d), ctypes.byref(nbytes)), query)
    n = nbytes.value
    return (_device.workspace(n, ref.device) if n else None), n


def grouped_product(x: torch.Tensor, w: torch.Tensor, g: Groups, out_dtype) -> torch.Tensor:
    """out[s] = x[row of s] w[group of s], zero in slots of no group."""
    x = rows_of(x)
    w, order, gs, rs = weight_order(w)
    E, k, n = w.shape
    out = torch.empty((g.n_slots, n), dtype=out_dtype, device=x.device)
    d = _desc(x, _value_code(x, "x"), _DTYPES[out_dtype], order, E, k, n, g.n_slots, gs, rs, n)
    p = _ptr
    ws, ws_bytes = _product_workspace(x, "ej_grouped_gemm_workspace_size", d)
    _call(x, "ej_grouped_gemm", ctypes.byref(d), p(x), p(g.rows), p(g.offsets), p(w), None, None,
          p(out), p(ws), ws_bytes)
    return out


def grouped_weight_gradient(x: torch.Tensor, w: torch.Tensor, g: Groups,
                            grad: torch.Tensor) -> torch.Tensor:
    """Gradient to w [E, k, n] in the order w lies in."""
    x, grad = rows_of(x), rows_of(grad)
    E, k, n = w.shape
    _, order, _, _ = weight_order(w)
    if order == _lib.EJ_W_KN:
        gw = torch.empty((E, k, n), dtype=w.dtype, device=w.device)
        rs = n
    else:
        gw = torch.empty((E, n, k), dtype=w.dtype, device=w.device).transpose(1, 2)
        rs = k
    code = _value_code(x, "x")
    d = _desc(x, code, code, order, E, k, n, g.n_slots, k * n, rs, max(_row_stride(grad), n))
    p = _ptr
    ws, ws_bytes = _product_workspace(x, "ej_grouped_gemm_dw_workspace_size", d)
    _call(x, "ej_grouped_gemm_dw", ctypes.byref(d), p(x), p(g.rows), p(g.offsets), p(grad), p(gw),
          p(ws), ws_bytes)
    return gw


def int8_matmul(q: torch.Tensor, q_scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                groups=None, *, gather: bool = False,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Product of 8-bit rows and 8-bit weights with their scales.

    q int8 [m, k] and q_scale float32 [m] are rows and their scales
    (``quantize_rows``); w int8 holds one row of k for each output channel,
    w_scale float32 their scales.  The integer sum is exact (k < 131072), times
    both scales in float32, rounded once to out_dtype (float32, bfloat16 or
    float16).

    Without groups: w [n, k] or [1, n, k], w_scale [n] or [1, n], the dense
    product [m, n].  With groups (an ``ExpertRouting`` or offsets [E + 1]):
    w [E, n, k], w_scale [E, n]; slot s of group e is q's row s, or with
    ``gather`` the row of its token, times w[e]; zero in slots of no group."""
    on_gpu(q, "q")
    _same_device(q, q_scale=q_scale, w=w, w_scale=w_scale)
    if q.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError(f"q and w must be int8, got {q.dtype} and {w.dtype}")
    if q_scale.dtype != torch.float32 or w_scale.dtype != torch.float32:
        raise TypeError(f"scales must be float32, got {q_scale.dtype} and {w_scale.dtype}")
    if out_dtype not in _DTYPES:
        raise TypeError(f"out_dtype must be float32, bfloat16 or float16, got {out_dtype}")
    if q.dim() != 2:
        raise ValueError(f"q must be [rows, k], got shape {tuple(q.shape)}")
    if groups is None and w.dim() == 2:
        w, w_scale = w[None], w_scale[None]
    if w.dim() != 3:
        raise ValueError(f"w must be [groups, n, k] (or [n, k] without groups), got shape "
                         f"{tuple(w.shape)}")
    E, n, k = w.shape
    if q.shape[1] != k:
        raise ValueError(f"q has rows of {q.shape[1]}, w of {k}")
    if q_scale.shape != (q.shape[0],) or w_scale.shape != (E, n):
        raise ValueError(f"scales have shapes {tuple(q_scale.shape)} and {tuple(w_scale.shape)}, "
                         f"expected {(q.shape[0],)} and {(E, n)}")
    if groups is None:
        if gather or E != 1:
            raise ValueError("more than one weight matrix, or gather=True, needs groups")
        g = Groups(None, None, None, q.shape[0])
    else:
        g = groups_of(q, E, groups, gather)
    q = rows_of(q)
    if not w.is_contiguous() and (
            (k > 1 and w.stride(2) != 1) or (n > 1 and w.stride(1) < k) or
            (E > 1 and w.stride(0) < n * (w.stride(1) if n > 1 else k))):
        w = w.contiguous()
    rs = w.stride(1) if n > 1 else max(k, 1)
    gs = w.stride(0) if E > 1 else n * rs
    out = torch.empty((g.n_slots, n), dtype=out_dtype, device=q.device)
    d = _desc(q, _lib.EJ_I8, _DTYPES[out_dtype], _lib.EJ_W_NK, E, k, n, g.n_slots, gs, rs, n)
    p = _ptr
    q_scale, w_scale = q_scale.contiguous(), w_scale.contiguous()
    _call(q, "ej_grouped_gemm", ctypes.byref(d), p(q), p(g.rows), p(g.offsets), p(w), p(q_scale),
          p(w_scale), p(out), None, 0)
    return out

