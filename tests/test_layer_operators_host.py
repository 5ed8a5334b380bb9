"""Gated products, block-scaled 8-bit products and token rows: what they refuse,
and what is decided without a GPU."""

import ctypes

import pytest
import torch

import einjax_amd as ej
from einjax_amd import _lib
from test_experts_host import FAKE, desc

INVAL, UNSUPPORTED = _lib.EJ_E_INVAL, _lib.EJ_E_UNSUPPORTED


def gated_desc(**kw):
    """k = 64, n = 32 results of 64 columns of w."""
    return desc(**{**dict(w_group=64 * 64, w_stride=64), **kw})


def gated(d, act=_lib.EJ_SILU, x=FAKE, rows=None, offsets=FAKE, w=FAKE, out=FAKE, gate_up=None):
    return _lib.load().ej_gated_gemm(ctypes.byref(d), act, x, rows, offsets, w, out, gate_up, None,
                                     0, None)


@pytest.mark.parametrize("change,status", [
    (dict(dtype=_lib.EJ_F64), INVAL), (dict(dtype=_lib.EJ_I8), INVAL),
    (dict(out_dtype=_lib.EJ_F16), INVAL), (dict(w_order=2), INVAL), (dict(k=-1), INVAL),
    (dict(x_stride=63), INVAL), (dict(w_stride=63), INVAL), (dict(out_stride=31), INVAL),
    (dict(w_group=64 * 64 - 1), INVAL), (dict(n_rows=9), INVAL),
    (dict(w_order=_lib.EJ_W_NK, w_group=64 * 64 - 1), INVAL),
    (dict(n_slots=(1 << 31) - 511), UNSUPPORTED),
    (dict(n=1 << 30, w_stride=1 << 31, out_stride=1 << 30, w_group=1 << 40), UNSUPPORTED),
])
def test_gated_refusals(change, status):
    assert gated(gated_desc(**change)) == status
    assert _lib.load().ej_last_error()


def test_gated_arguments():
    lib, n = _lib.load(), ctypes.c_size_t()
    assert gated(gated_desc(), act=3) == INVAL
    assert gated(gated_desc(), x=None) == INVAL
    assert gated(gated_desc(), w=None) == INVAL
    assert gated(gated_desc(), out=None) == INVAL
    assert gated(gated_desc(), offsets=None) == INVAL
    assert lib.ej_gated_gemm(None, 0, FAKE, None, FAKE, FAKE, FAKE, None, None, 0, None) == INVAL
    # nothing to write: no launch
    assert gated(gated_desc(n_slots=0), x=None, w=None, out=None, offsets=None) == 0
    assert gated(gated_desc(n=0), x=None, w=None, out=None, offsets=None) == 0
    # a contraction in parts needs room for the sums of both projections
    few = gated_desc(n_groups=1, k=4096, n_slots=512, n_rows=512, x_stride=4096,
                     w_group=4096 * 64)
    assert lib.ej_gated_gemm_workspace_size(ctypes.byref(few), ctypes.byref(n)) == 0
    assert n.value > 0 and n.value % (4 * 512 * 64) == 0
    assert gated(few) == INVAL and b"workspace" in lib.ej_last_error()
    for d in (gated_desc(), gated_desc(n_groups=0), gated_desc(n_slots=0)):
        assert lib.ej_gated_gemm_workspace_size(ctypes.byref(d), ctypes.byref(n)) == 0
        assert n.value == 0
    assert lib.ej_gated_gemm_workspace_size(None, ctypes.byref(n)) == INVAL


def test_gated_vjp_arguments():
    def vjp(both=FAKE, grad=FAKE, dtype=_lib.EJ_BF16, rows=4, n=8, stride=8, act=0, out=FAKE):
        return _lib.load().ej_gated_vjp(both, grad, dtype, rows, n, stride, act, out, None)

    assert vjp(dtype=_lib.EJ_I8) == INVAL
    assert vjp(stride=7) == INVAL
    assert vjp(rows=-1) == INVAL
    assert vjp(act=-1) == INVAL
    assert vjp(both=None) == INVAL and vjp(grad=None) == INVAL and vjp(out=None) == INVAL
    assert vjp(rows=0, both=None, grad=None, out=None) == 0
    assert vjp(n=0, stride=0, both=None, grad=None, out=None) == 0
    assert vjp(rows=1 << 40) == UNSUPPORTED
    assert vjp(rows=1 << 62) == UNSUPPORTED
    assert vjp(n=1 << 30, stride=1 << 30) == UNSUPPORTED


def test_operands_must_be_on_the_gpu():
    t = torch.zeros(4, 4)
    for call in (lambda: ej.gated_matmul(t, t), lambda: ej.gated_matmul(t, t[None], t.int()),
                 lambda: ej.gated_matmul_vjp(t, t, None, t)):
        with pytest.raises(TypeError, match="on the GPU"):
            call()


@pytest.mark.parametrize("change,status", [
    (dict(w_order=_lib.EJ_W_KN, w_stride=64), INVAL), (dict(out_dtype=_lib.EJ_E4M3), INVAL),
    (dict(out_dtype=_lib.EJ_I8), INVAL), (dict(x_stride=63), INVAL), (dict(w_stride=63), INVAL),
])
def test_block_product_refusals(change, status):
    d = desc(**{**dict(dtype=_lib.EJ_E4M3, w_order=_lib.EJ_W_NK, w_stride=64), **change})
    lib = _lib.load()
    args = (ctypes.byref(d), FAKE, None, FAKE, FAKE)
    assert lib.ej_grouped_gemm(*args, FAKE, FAKE, FAKE, None, 0, None) == status
    assert lib.ej_last_error()


def test_block_product_arguments():
    lib, n = _lib.load(), ctypes.c_size_t()
    d = desc(dtype=_lib.EJ_E4M3, w_order=_lib.EJ_W_NK, w_stride=64)
    args = (ctypes.byref(d), FAKE, None, FAKE, FAKE)
    assert lib.ej_grouped_gemm(*args, None, FAKE, FAKE, None, 0, None) == INVAL
    assert lib.ej_grouped_gemm(*args, FAKE, None, FAKE, None, 0, None) == INVAL
    assert lib.ej_grouped_gemm_dw(*args, FAKE, None, 0, None) == INVAL
    assert lib.ej_grouped_gemm_workspace_size(ctypes.byref(d), ctypes.byref(n)) == 0


def test_quantize_blocks_arguments():
    def quantize(x=FAKE, dtype=_lib.EJ_BF16, mats=1, rows=4, ld=8, n=8, block=1, q=FAKE, s=FAKE):
        return _lib.load().ej_quantize_blocks(x, dtype, mats, 0, rows, ld, n, block, q, s, None)

    assert quantize(dtype=_lib.EJ_I8) == INVAL
    assert quantize(block=64) == INVAL
    assert quantize(ld=7) == INVAL
    assert quantize(rows=-1) == INVAL and quantize(mats=-1) == INVAL and quantize(n=-1) == INVAL
    assert quantize(x=None) == INVAL and quantize(q=None) == INVAL and quantize(s=None) == INVAL
    for empty in (dict(rows=0), dict(mats=0), dict(n=0)):
        assert quantize(x=None, q=None, s=None, **empty) == 0
    for large in (dict(rows=1 << 40), dict(mats=1 << 62), dict(mats=1 << 20, rows=1 << 20),
                  dict(mats=1 << 40, rows=1 << 40), dict(rows=1 << 31, block=128),
                  dict(n=(1 << 31) - 1, ld=1 << 31)):
        assert quantize(**large) == UNSUPPORTED


def test_8_bit_operands_must_be_on_the_gpu():
    t = torch.zeros(4, 128)
    q, s = t.to(torch.float8_e4m3fn), torch.zeros(4, 1)
    for call in (lambda: ej.quantize_blocks(t), lambda: ej.fp8_matmul(q, s, q, s[:1])):
        with pytest.raises(TypeError, match="on the GPU"):
            call()


def test_embed_arguments():
    lib, n = _lib.load(), ctypes.c_size_t()

    def embed(table=FAKE, dtype=_lib.EJ_BF16, rows=9, ld=8, n=8, tokens=FAKE, kind=_lib.EJ_I64,
              t=4, out=FAKE):
        return lib.ej_embed(table, dtype, rows, ld, n, tokens, kind, t, 1.0, out, None)

    def vjp(tokens=FAKE, kind=_lib.EJ_I64, t=4, grad=FAKE, dtype=_lib.EJ_BF16, ld=8, rows=9, n=8,
            out=FAKE, ws=FAKE, size=1 << 20):
        return lib.ej_embed_vjp(tokens, kind, t, grad, dtype, ld, rows, n, 1.0, out, ws, size,
                                None)

    for call in (embed, vjp):
        assert call(dtype=_lib.EJ_I32) == INVAL and call(kind=_lib.EJ_F32) == INVAL
        assert call(ld=7) == INVAL
        assert call(t=-1) == INVAL and call(rows=-1) == INVAL and call(n=-1) == INVAL
        assert call(tokens=None) == INVAL and call(out=None) == INVAL
        assert call(rows=1 << 31) == UNSUPPORTED and call(t=1 << 31) == UNSUPPORTED
        assert call(n=(1 << 31) - 1, ld=1 << 31) == UNSUPPORTED
        assert call(n=0, ld=0, tokens=None, out=None) == 0
    assert embed(table=None) == INVAL and vjp(grad=None) == INVAL
    assert embed(t=0, tokens=None, out=None, table=None) == 0
    assert vjp(rows=0, tokens=None, grad=None, out=None, ws=None, size=0) == 0
    assert vjp(ws=None) == INVAL and vjp(size=1) == INVAL
    assert b"workspace" in lib.ej_last_error()
    # keys, places and the parts of long sums; above 16384 tokens the sort's room
    sizes = []
    for t in (0, 1, 16384, 16385):
        assert lib.ej_embed_vjp_workspace_size(t, 9, 8, ctypes.byref(n)) == 0
        sizes.append(n.value)
    assert sizes[0] == 0 and 0 < sizes[1] < sizes[2] < sizes[3] - 16 * 16384
    assert lib.ej_embed_vjp_workspace_size(4, 9, 8, None) == INVAL


def test_tokens_must_be_on_the_gpu():
    t, i = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    for call in (lambda: ej.embed_tokens(i, t), lambda: ej.embed_tokens_vjp(i, t, t)):
        with pytest.raises(TypeError, match="on the GPU"):
            call()
