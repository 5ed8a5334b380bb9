"""Expert operators: what they refuse, and what is decided without a GPU."""

import ctypes

import pytest
import torch

import einjax_amd as ej
from einjax_amd import _lib

FAKE = ctypes.c_void_p(16)  # never dereferenced: checks come first


def desc(**kw):
    d = dict(dtype=_lib.EJ_BF16, out_dtype=_lib.EJ_BF16, w_order=_lib.EJ_W_KN, n_groups=2, k=64,
             n=32, n_slots=10, n_rows=10, x_stride=64, w_group=64 * 32, w_stride=32,
             out_stride=32)
    d.update(kw)
    return _lib.GroupedDesc(*(d[f] for f, _ in _lib.GroupedDesc._fields_))


def gemm(d, x=FAKE, rows=None, offsets=FAKE, w=FAKE, xs=None, ws=None, out=FAKE):
    return _lib.load().ej_grouped_gemm(ctypes.byref(d), x, rows, offsets, w, xs, ws, out, None, 0,
                                      None)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=_lib.EJ_F64), _lib.EJ_E_INVAL),
    (dict(out_dtype=_lib.EJ_F16), _lib.EJ_E_INVAL),
    (dict(w_order=2), _lib.EJ_E_INVAL),
    (dict(n=-1), _lib.EJ_E_INVAL),
    (dict(x_stride=63), _lib.EJ_E_INVAL),
    (dict(w_stride=31), _lib.EJ_E_INVAL),
    (dict(out_stride=31), _lib.EJ_E_INVAL),
    (dict(w_group=100), _lib.EJ_E_INVAL),
    (dict(n_rows=9), _lib.EJ_E_INVAL),
    (dict(n_slots=1 << 31), _lib.EJ_E_UNSUPPORTED),
    (dict(dtype=_lib.EJ_I8), _lib.EJ_E_INVAL),                     # 8-bit weights are [n][k]
    (dict(dtype=_lib.EJ_I8, w_order=_lib.EJ_W_NK, w_stride=64), _lib.EJ_E_INVAL),  # no scales
    (dict(dtype=_lib.EJ_I8, out_dtype=_lib.EJ_I8, w_order=_lib.EJ_W_NK, w_stride=64),
     _lib.EJ_E_INVAL),
    (dict(dtype=_lib.EJ_I8, w_order=_lib.EJ_W_NK, k=1 << 17, x_stride=1 << 17, w_stride=1 << 17,
          w_group=1 << 23), _lib.EJ_E_INVAL),                      # sums past 32 bits
])
def test_product_refusals(change, status):
    assert gemm(desc(**change)) == status
    assert _lib.load().ej_last_error()


def test_product_null_arguments():
    assert gemm(desc(), x=None) == _lib.EJ_E_INVAL
    assert gemm(desc(), w=None) == _lib.EJ_E_INVAL
    assert gemm(desc(), out=None) == _lib.EJ_E_INVAL
    assert gemm(desc(), offsets=None) == _lib.EJ_E_INVAL  # two groups need offsets
    lib = _lib.load()
    assert lib.ej_grouped_gemm(None, FAKE, None, FAKE, FAKE, None, None, FAKE, None, 0, None) == \
        _lib.EJ_E_INVAL
    # nothing to write: no launch
    assert gemm(desc(n_slots=0), x=None, w=None, out=None, offsets=None) == 0
    assert gemm(desc(n=0), x=None, w=None, out=None, offsets=None) == 0
    assert lib.ej_grouped_gemm_dw(ctypes.byref(desc(n_groups=0)), None, None, None, None, None,
                                  None, 0, None) == 0
    assert lib.ej_grouped_gemm_dw(ctypes.byref(desc(dtype=_lib.EJ_I8)), FAKE, None, FAKE, FAKE,
                                  FAKE, None, 0, None) == _lib.EJ_E_INVAL


def test_split_products_need_their_workspace():
    lib, n = _lib.load(), ctypes.c_size_t()
    few = desc(n_groups=1, k=4096, n_slots=512, n_rows=512, x_stride=4096, w_group=4096 * 32)
    assert lib.ej_grouped_gemm_workspace_size(ctypes.byref(few), ctypes.byref(n)) == 0
    assert n.value > 0 and n.value % (4 * 512 * 32) == 0
    assert gemm(few) == _lib.EJ_E_INVAL and b"workspace" in lib.ej_last_error()
    tall = desc(n_groups=1, n_slots=8192, n_rows=8192)
    assert lib.ej_grouped_gemm_dw_workspace_size(ctypes.byref(tall), ctypes.byref(n)) == 0
    assert n.value > 0 and n.value % (4 * 64 * 32) == 0
    assert lib.ej_grouped_gemm_dw(ctypes.byref(tall), FAKE, None, FAKE, FAKE, FAKE, None, 0,
                                  None) == _lib.EJ_E_INVAL
    for d in (desc(), desc(n_groups=0), desc(n_slots=0)):
        assert lib.ej_grouped_gemm_workspace_size(ctypes.byref(d), ctypes.byref(n)) == 0
        assert n.value == 0
        assert lib.ej_grouped_gemm_dw_workspace_size(ctypes.byref(d), ctypes.byref(n)) == 0
        assert n.value == 0
    assert lib.ej_grouped_gemm_workspace_size(None, ctypes.byref(n)) == _lib.EJ_E_INVAL


@pytest.mark.parametrize("t,e,k,status", [
    (-1, 4, 1, _lib.EJ_E_INVAL), (4, 0, 1, _lib.EJ_E_INVAL), (4, 4, 0, _lib.EJ_E_INVAL),
    (4, 4, 5, _lib.EJ_E_INVAL), (4, 2000, 1, _lib.EJ_E_UNSUPPORTED),
    (4, 100, 17, _lib.EJ_E_UNSUPPORTED), (1 << 26, 4, 1, _lib.EJ_E_UNSUPPORTED),
])
def test_route_refusals(t, e, k, status):
    lib = _lib.load()
    args = (FAKE, FAKE, FAKE, FAKE, FAKE, None, 0, None)
    assert lib.ej_expert_route(FAKE, _lib.EJ_F32, t, e, e, k, 1, *args) == status
    assert lib.ej_expert_group(FAKE, t, k, e, FAKE, FAKE, FAKE, None, 0, None) == status
    assert lib.ej_expert_route_vjp(FAKE, _lib.EJ_F32, t, e, e, k, 1, FAKE, FAKE, FAKE,
                                   None) == status


def test_route_argument_checks():
    lib = _lib.load()
    args = (FAKE, FAKE, FAKE, FAKE, FAKE, None, 0, None)
    assert lib.ej_expert_route(FAKE, _lib.EJ_I32, 4, 4, 4, 1, 1, *args) == _lib.EJ_E_INVAL
    assert lib.ej_expert_route(FAKE, _lib.EJ_F32, 4, 4, 3, 1, 1, *args) == _lib.EJ_E_INVAL
    assert lib.ej_expert_route(None, _lib.EJ_F32, 4, 4, 4, 1, 1, *args) == _lib.EJ_E_INVAL
    # a large batch needs its workspace
    n = ctypes.c_size_t()
    assert lib.ej_expert_route_workspace_size(100_000, 64, ctypes.byref(n)) == 0 and n.value > 0
    assert lib.ej_expert_route(FAKE, _lib.EJ_F32, 100_000, 64, 64, 1, 1, *args) == \
        _lib.EJ_E_INVAL
    assert b"workspace" in lib.ej_last_error()
    assert lib.ej_expert_route_workspace_size(1, 64, ctypes.byref(n)) == 0 and n.value == 0


def test_combine_and_quantize_refusals():
    lib = _lib.load()
    f32, bf16 = _lib.EJ_F32, _lib.EJ_BF16

    def combine(dtype=f32, stride=8, slots=FAKE, t=2, k=2, out_dtype=f32):
        return lib.ej_expert_combine(FAKE, dtype, 4, stride, None, slots, t, k, 8, FAKE, out_dtype,
                                     None)

    assert combine(dtype=_lib.EJ_I32) == _lib.EJ_E_INVAL
    assert combine(stride=7) == _lib.EJ_E_INVAL
    assert combine(slots=None) == _lib.EJ_E_INVAL
    assert combine(k=17) == _lib.EJ_E_UNSUPPORTED
    assert combine(dtype=bf16) == _lib.EJ_E_INVAL  # 16-bit values keep their dtype
    assert combine(out_dtype=_lib.EJ_I8) == _lib.EJ_E_INVAL
    assert combine(t=0) == 0
    assert lib.ej_expert_combine_vjp(FAKE, _lib.EJ_F32, 4, 8, None, FAKE, None, 2, 2, 2, 8, FAKE,
                                     8, FAKE, FAKE, None) == _lib.EJ_E_INVAL
    assert lib.ej_quantize_rows(FAKE, _lib.EJ_F64, 4, 8, 8, FAKE, FAKE, None) == _lib.EJ_E_INVAL
    assert lib.ej_quantize_rows(FAKE, _lib.EJ_F32, 4, 7, 8, FAKE, FAKE, None) == _lib.EJ_E_INVAL
    assert lib.ej_quantize_rows(FAKE, _lib.EJ_F32, 4, 8, 8, None, FAKE, None) == _lib.EJ_E_INVAL
    assert lib.ej_quantize_rows(FAKE, _lib.EJ_F32, -1, 8, 8, FAKE, FAKE, None) == _lib.EJ_E_INVAL


def test_operands_must_be_on_the_gpu():
    t = torch.zeros(4, 4)
    for call in (lambda: ej.route_experts(t, 2), lambda: ej.route_experts(t.numpy(), 2),
                 lambda: ej.group_by_expert(t.int(), 4), lambda: ej.quantize_rows(t),
                 lambda: ej.grouped_matmul(t, t[None], t.int()),
                 lambda: ej.int8_matmul(t, t, t, t),
                 lambda: ej.combine_experts(t, ej.ExpertRouting(t, t, t, t, t)),
                 lambda: ej.route_experts_vjp(t, t, t)):
        with pytest.raises(TypeError, match="on the GPU"):
            call()
    with pytest.raises(TypeError, match="ExpertRouting"):
        ej.combine_experts(t, None)


def test_weight_order_reads_strides():
    w = torch.zeros(3, 5, 7)
    same, order, gs, rs = _lib.experts().weight_order(w)
    assert same.data_ptr() == w.data_ptr() and (order, gs, rs) == (_lib.EJ_W_KN, 35, 7)
    v = torch.zeros(3, 7, 5).transpose(1, 2)
    same, order, gs, rs = _lib.experts().weight_order(v)
    assert same.data_ptr() == v.data_ptr() and (order, gs, rs) == (_lib.EJ_W_NK, 35, 5)
    part = torch.zeros(3, 9, 20)[:, 2:7, 4:11]
    same, order, gs, rs = _lib.experts().weight_order(part)
    assert same.data_ptr() == part.data_ptr() and (order, gs, rs) == (_lib.EJ_W_KN, 180, 20)
    for odd in (torch.zeros(3, 5, 14)[:, :, ::2], torch.zeros(1, 5, 7).expand(3, 5, 7)):
        copy, order, gs, rs = _lib.experts().weight_order(odd)
        assert copy.is_contiguous() and (order, gs, rs) == (_lib.EJ_W_KN, 35, 7)
    for shape in ((1, 1, 1), (2, 1, 4), (2, 4, 1), (0, 3, 3)):
        _, order, gs, rs = _lib.experts().weight_order(torch.zeros(shape))
        assert order in (_lib.EJ_W_KN, _lib.EJ_W_NK)


def test_rows_of_copies_only_what_it_must():
    t = torch.zeros(6, 8)
    assert _lib.experts().rows_of(t).data_ptr() == t.data_ptr()
    assert _lib.experts().rows_of(t[:, 2:5]).data_ptr() == t[:, 2:5].data_ptr()
    assert _lib.experts().rows_of(t.t()).is_contiguous()
    assert _lib.experts().rows_of(t[:1].expand(4, 8)).is_contiguous()


def test_routing_takes_no_more_tokens_than_its_gradient():
    """A token of more than 256 experts is a wave of the gradient; a launch holds
    fewer than 2^32 threads."""
    lib, n = _lib.load(), ctypes.c_size_t()
    for t, status in (((1 << 26) - 3, _lib.EJ_E_UNSUPPORTED), ((1 << 26) - 4, 0)):
        assert lib.ej_expert_route_workspace_size(t, 300, ctypes.byref(n)) == status
        # null operands are noticed after the sizes
        refused = status or _lib.EJ_E_INVAL
        assert lib.ej_expert_route_vjp(None, _lib.EJ_F32, t, 300, 300, 1, 1, None, None, None,
                                       None) == refused


def test_slots_that_32_bits_do_not_count():
    """Blocks and stages end past the last slot, by less than 512."""
    lib, n = _lib.load(), ctypes.c_size_t()
    for slots, status in (((1 << 31) - 1, _lib.EJ_E_UNSUPPORTED),
                          ((1 << 31) - 511, _lib.EJ_E_UNSUPPORTED), ((1 << 31) - 512, 0)):
        d = desc(n_slots=slots, n_rows=slots)
        assert lib.ej_grouped_gemm_workspace_size(ctypes.byref(d), ctypes.byref(n)) == status
        assert lib.ej_grouped_gemm_dw_workspace_size(ctypes.byref(d), ctypes.byref(n)) == status
