"""Grouped products of rows that begin anywhere: every offset of the bases from 4
and 16 bytes, odd lengths of rows and of columns, in the larger tiles too.

A product is a sum of k products in fp32, off by 2 (k + 2) 2^-24 of the sum of their
magnitudes, and rounded once (``sum_bound`` of the aligned products' tests); 8-bit
ones as in the tests of theirs.
"""

import pytest
import torch

import einjax_amd as ej
from test_gpu_experts import BF16, F16, F32, TINY, UNIT, assert_within, randn, rng
from test_gpu_fp8 import assert_product, blocks, fp8_64, operands, scales
from test_gpu_gated import gated64

pytestmark = pytest.mark.gpu

SIZES = [700, 0, 650, 150]
SLOTS, LIVE = 1507, 1500


def at_offset(t, shift):
    """The same values, `shift` elements behind an aligned address."""
    flat = torch.empty(t.numel() + 64, dtype=t.dtype, device=t.device)
    view = flat[shift:shift + t.numel()].view(t.shape)
    view.copy_(t)
    return view


def relation(seed):
    """Slots of each group in a shuffled order of the rows."""
    g = torch.Generator().manual_seed(seed)
    picks = torch.repeat_interleave(torch.arange(len(SIZES)), torch.tensor(SIZES))
    picks = torch.cat([picks, torch.full((SLOTS - LIVE,), -1)])
    return ej.group_by_expert(picks[torch.randperm(SLOTS, generator=g)].cuda()[:, None],
                              len(SIZES))


def weights(g, k, n, dtype, order, shift):
    if order == "kn":
        return at_offset(randn(g, len(SIZES), k, n, dtype=dtype, scale=k ** -0.5), shift)
    return at_offset(randn(g, len(SIZES), n, k, dtype=dtype, scale=k ** -0.5),
                     shift).transpose(1, 2)


@pytest.mark.parametrize("shift", [0, 1, 2, 3, 5])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k,n", [(259, 1347), (260, 1346), (7, 1411), (64, 2050), (131, 1350)])
def test_products_of_unaligned_rows(gpu, k, n, dtype, shift):
    g, r = rng(k + shift), relation(k)
    ends = [0] + torch.tensor(SIZES).cumsum(0).tolist()
    for order in ("kn", "nk"):
        x = at_offset(randn(g, SLOTS, k, dtype=dtype), shift)
        w = weights(g, k, n, dtype, order, (shift + 1) % 4)
        for gather in (False, True):
            got = ej.grouped_matmul(x, w, r, gather=gather)
            for e, (a, b) in enumerate(zip(ends, ends[1:])):
                xe = (x[r.rows[a:b].long()] if gather else x[a:b]).double()
                want, size = xe @ w[e].double(), xe.abs() @ w[e].double().abs()
                off = 2 * (k + 2) * 2.0 ** -24 * size
                assert_within(got[a:b], want, off + UNIT[dtype] * (want.abs() + off) + TINY[dtype])
            assert bool((got[LIVE:] == 0).all())
        w = weights(g, k, n // 2 * 2, dtype, order, shift)
        got = ej.gated_matmul(x, w, r, gather=True)
        h, eh, *_ = gated64(x, r.rows, r.offsets, w, SLOTS, "silu")
        assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])


@pytest.mark.parametrize("shift", [0, 1, 3])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k,n", [(1030, 1031), (1027, 1025), (70, 133)])
def test_weight_gradients_of_unaligned_rows(gpu, k, n, dtype, shift):
    g, r = rng(n + shift), relation(n)
    x = at_offset(randn(g, SLOTS, k, dtype=dtype), shift)
    grad = at_offset(randn(g, SLOTS, n, dtype=dtype), (shift + 2) % 4)
    ends = [0] + torch.tensor(SIZES).cumsum(0).tolist()
    for order in ("kn", "nk"):
        w = weights(g, k, n, dtype, order, 0)
        for gather in (False, True):
            _, got = ej.grouped_matmul_vjp(x, w, r, grad, gather=gather, need_x=False)
            for e, (a, b) in enumerate(zip(ends, ends[1:])):
                xe = (x[r.rows[a:b].long()] if gather else x[a:b]).double()
                ge = grad[a:b].double()
                want = xe.T @ ge
                off = 2 * (b - a + 2) * 2.0 ** -24 * (xe.abs().T @ ge.abs())
                assert_within(got[e], want, off + UNIT[dtype] * (want.abs() + off) + TINY[dtype])


@pytest.mark.parametrize("shift", range(5))
@pytest.mark.parametrize("k,n", [(259, 1801), (262, 1795), (17, 1800), (1000, 1793)])
def test_8_bit_products_of_unaligned_rows(gpu, k, n, shift):
    g, r, e = rng(k + shift), relation(n), len(SIZES)
    q = at_offset(torch.randint(-128, 128, (SLOTS, k), generator=g, device="cuda").to(torch.int8),
                  shift)
    w = at_offset(torch.randint(-128, 128, (e, n, k), generator=g, device="cuda").to(torch.int8),
                  (shift + 3) % 4)
    one = torch.ones(SLOTS, device="cuda")
    got = ej.int8_matmul(q, one, w, torch.ones(e, n, device="cuda"), r, gather=True, out_dtype=F32)
    ends = [0] + torch.tensor(SIZES).cumsum(0).tolist()
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        # below 2^24: exact
        assert torch.equal(got[a:b].double(), q[r.rows[a:b].long()].double() @ w[i].double().T)
    q, w = at_offset(operands(g, SLOTS, k), shift), at_offset(operands(g, n, k, (e,)), shift + 1)
    qs, ws = scales(g, SLOTS, blocks(k)) * 1e-2, scales(g, e, blocks(n), blocks(k)) * 1e-4
    for dtype in (F32, BF16):
        got = ej.fp8_matmul(q, qs, w, ws, r, gather=True, out_dtype=dtype)
        want, size = fp8_64(q, qs, w, ws, r.rows, r.offsets, SLOTS)
        assert_product(got, want, size, k, dtype)
        assert bool((got[LIVE:] == 0).all())
