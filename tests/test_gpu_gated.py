"""Gated products against their definition in 64 bits.

Bounds are those of the arithmetic.  Each projection is a sum of k products in
fp32, off by 2 (k + 2) 2^-24 of the sum of their magnitudes; what follows
(activation, its slope, products) adds the relative errors that ``ROOM`` counts;
every rounding to the operands' type counts its unit roundoff once: one of the
result, and in gradients one of the projections' gradient, which the products of
the backward pass take in the operands' type, and one of theirs.
"""

import math

import pytest
import torch

import einjax_amd as ej
from test_gpu_experts import (BF16, F16, F32, LARGE, PRODUCTS, TINY, UNIT, assert_within,
                              product_case, randn, rng, row_groups, sum_bound)

pytestmark = pytest.mark.gpu

ACTS = ["silu", "gelu", "gelu_tanh"]


def act64(name, g):
    """Activation and slope in 64 bits."""
    if name == "silu":
        p = torch.sigmoid(g)
        return g * p, p * (1 + g * torch.sigmoid(-g))
    if name == "gelu":
        p = 0.5 * torch.special.erfc(-g / math.sqrt(2))
        return g * p, p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    c = math.sqrt(2 / math.pi)
    z = 2 * c * (g + 0.044715 * g ** 3)
    p = torch.sigmoid(z)
    return g * p, p + g * p * torch.sigmoid(-z) * 2 * c * (1 + 3 * 0.044715 * g * g)


def ROOM(g):
    """Relative error of an activation at g in fp32: the argument of the
    exponential, at most 1.6 |g| + 0.072 |g|^3 or g^2 / 2, is off by 4 units in
    its last place, which is its absolute error and the exponential's relative
    one; 24 units for the functions, the division and the products."""
    a = g.abs()
    return (24 + 8 * a + 2 * a * a + 0.3 * a ** 3) * 2.0 ** -24


def gated64(x, rows, offsets, w, slots, act):
    """(h, bound of its error in fp32, gate, up, their error bounds)."""
    n = w.shape[2] // 2
    gu = torch.zeros(slots, 2 * n, dtype=torch.double, device="cuda")
    err = torch.zeros_like(gu)
    ends = [0, slots] if offsets is None else offsets.tolist()
    for e in range(w.shape[0]):
        a, b = ends[e], ends[e + 1]
        xe = (x[rows[a:b].long()] if rows is not None else x[a:b]).double()
        gu[a:b] = xe @ w[e].double()
        err[a:b] = 2 * (x.shape[1] + 2) * 2.0 ** -24 * (xe.abs() @ w[e].double().abs())
    g, u, eg, eu = gu[:, :n], gu[:, n:], err[:, :n], err[:, n:]
    a, _ = act64(act, g)
    # slopes are at most 1.13
    ea = 1.13 * eg + ROOM(g) * a.abs() + 1e-37 * (1 + g.abs())
    eh = ea * u.abs() + a.abs() * eu + ea * eu + 2.0 ** -23 * (a * u).abs()
    return a * u, eh, g, u, eg, eu, ea


def projections_gradient(act, g, u, eg, eu, ea, dh, dtype):
    """dg | du and the bound of their error in the operands' type."""
    a, slope = act64(act, g)
    # second derivatives are at most 1.2; a slope is a sum of two terms of at
    # most 1 and 1.13, each with an activation's relative error
    es = 1.2 * eg + 2.2 * ROOM(g)
    dg, du = dh * u * slope, dh * a
    eg = dh.abs() * (u.abs() * es + slope.abs() * eu + es * eu) + 2.0 ** -22 * dg.abs()
    eu = dh.abs() * ea + 2.0 ** -23 * du.abs()
    d, e = torch.cat([dg, du], 1), torch.cat([eg, eu], 1)
    return d, e + UNIT[dtype] * (d.abs() + e) + TINY[dtype]


def gated_case(t, e, k, n_in, n, kind, dtype, order, gather):
    g, r, x, w = product_case(t, e, k, n_in, 2 * n, kind, dtype, order, gather)
    return g, r, x, w


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k,n_in,n,kind", PRODUCTS)
def test_gated_matmul(gpu, t, e, k, n_in, n, kind, dtype, order):
    for gather, act in ((False, "silu"), (True, "gelu"), (True, "gelu_tanh")):
        _, r, x, w = gated_case(t, e, k, n_in, n, kind, dtype, order, gather)
        got = ej.gated_matmul(x, w, r, activation=act, gather=gather)
        h, eh, *_ = gated64(x, r.rows if gather else None, r.offsets, w, t * k, act)
        assert got.dtype == dtype
        assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])
        assert bool((got[int(r.offsets[-1]):] == 0).all())
        if not gather:
            again = ej.gated_matmul(x, w, r.offsets.long(), activation=act)
            assert torch.equal(again, got)


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k,n_in,n,kind", PRODUCTS)
def test_gated_matmul_gradients(gpu, t, e, k, n_in, n, kind, dtype, order):
    for gather, act in ((False, "gelu_tanh"), (True, "silu"), (False, "gelu")):
        gen, r, x, w = gated_case(t, e, k, n_in, n, kind, dtype, order, gather)
        rows = r.rows if gather else None
        x.requires_grad_()
        w = w.detach().requires_grad_()
        y = ej.gated_matmul(x, w, r, activation=act, gather=gather)
        cot = randn(gen, t * k, n, dtype=dtype)
        gx, gw = torch.autograd.grad(y, (x, w), cot)
        assert gx.dtype == dtype and gw.dtype == dtype and gw.stride() == w.stride()
        x, w = x.detach(), w.detach()
        assert torch.equal(y.detach(), ej.gated_matmul(x, w, r, activation=act, gather=gather))
        again = ej.gated_matmul_vjp(x, w, r, cot, activation=act, gather=gather)
        assert torch.equal(gx, again[0]) and torch.equal(gw, again[1])
        _, _, g, u, eg, eu, ea = gated64(x, rows, r.offsets, w, t * k, act)
        d, ed = projections_gradient(act, g, u, eg, eu, ea, cot.double(), dtype)
        _, ends = row_groups(r.offsets, t * k)
        wx = torch.zeros(t * k, n_in, dtype=torch.double, device="cuda")
        ex = torch.zeros_like(wx)
        for i in range(e):
            a, b = ends[i], ends[i + 1]
            at = rows[a:b].long() if gather else torch.arange(a, b, device="cuda")
            xi, wi, di, ei = x[at].double(), w[i].double(), d[a:b], ed[a:b]
            wx[a:b] = di @ wi.T
            size = (di.abs() + ei) @ wi.abs().T
            ex[a:b] = ei @ wi.abs().T + 2 * (2 * n + 2) * 2.0 ** -24 * size
            want, size = xi.T @ di, xi.abs().T @ (di.abs() + ei)
            off = xi.abs().T @ ei + 2 * (b - a + 2) * 2.0 ** -24 * size
            assert_within(gw[i], want, off + UNIT[dtype] * (want.abs() + off) + TINY[dtype])
        if gather:
            total, room, size = (torch.zeros(t, n_in, dtype=torch.double, device="cuda")
                                 for _ in range(3))
            at = r.rows[:ends[-1]].long()
            total.index_add_(0, at, wx[:ends[-1]])
            room.index_add_(0, at, ex[:ends[-1]])
            size.index_add_(0, at, wx[:ends[-1]].abs() + ex[:ends[-1]])
            wx, ex = total, room + 2 * (k + 2) * 2.0 ** -24 * size
        assert_within(gx, wx, ex + UNIT[dtype] * (wx.abs() + ex) + TINY[dtype])


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes,dead,k,n", LARGE)
def test_gated_matmul_large_blocks(gpu, sizes, dead, k, n, dtype, order):
    g, e, live = rng(k + n), len(sizes), sum(sizes)
    offsets = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32,
                           device="cuda")
    x = randn(g, live + dead, k, dtype=dtype)
    w = randn(g, e, k, n, dtype=dtype, scale=k ** -0.5)
    if order == "nk":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    x[live:] = float("nan")
    got = ej.gated_matmul(x, w, offsets)
    leaf = x.detach().requires_grad_()
    assert torch.equal(got, ej.gated_matmul(leaf, w, offsets).detach())  # keeps both projections
    x[live:] = 0
    h, eh, *_ = gated64(x, None, offsets, w, live + dead, "silu")
    assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,k,n", [(0, 8, 8), (1, 64, 64), (1, 4096, 512), (4, 77, 131),
                                   (16, 2048, 2048), (17, 2048, 40), (130, 2500, 70),
                                   (130, 0, 16), (3, 16, 0), (512, 4096, 64), (999, 264, 1032)])
def test_gated_matmul_dense(gpu, m, k, n, dtype):
    g = rng(m + k + n)
    x = randn(g, m, k, dtype=dtype)
    for order in ("kn", "nk"):
        w = randn(g, k, 2 * n, dtype=dtype, scale=max(k, 1) ** -0.5)
        if order == "nk":
            w = w.t().contiguous().t()
        h, eh, gate, up, eg, eu, ea = gated64(x, None, None, w[None], m, "silu")
        for wt in (w, w[None]):
            got = ej.gated_matmul(x, wt)
            assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])
        leaves = x.detach().requires_grad_(), w.detach().requires_grad_()
        cot = randn(g, m, n, dtype=dtype)
        gx, gw = torch.autograd.grad(ej.gated_matmul(*leaves), leaves, cot)
        assert gw.shape == w.shape
        d, ed = projections_gradient("silu", gate, up, eg, eu, ea, cot.double(), dtype)
        w64 = w.double()
        for got, want, off, size, terms in (
                (gx, d @ w64.T, ed @ w64.abs().T, (d.abs() + ed) @ w64.abs().T, 2 * n),
                (gw, x.double().T @ d, x.double().abs().T @ ed,
                 x.double().abs().T @ (d.abs() + ed), m)):
            off = off + 2 * (terms + 2) * 2.0 ** -24 * size
            assert_within(got, want, off + UNIT[dtype] * (want.abs() + off) + TINY[dtype])
        again = ej.gated_matmul_vjp(x, w, None, cot)
        assert torch.equal(again[0], gx) and torch.equal(again[1], gw)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes,k,n,shift", [
    ([4, 0, 9, 1], 1539, 294, 0), ([130], 2500, 70, 0), ([60, 12], 2048, 36, 0),
    ([60, 12], 2048, 36, 1), ([100, 0, 300], 4096, 32, 0), ([100, 0, 300], 4096, 31, 0)])
def test_gated_matmul_split_contractions(gpu, sizes, k, n, shift, dtype):
    """Few tiles over a long contraction, whose parts are summed apart."""
    g, e, slots = rng(k + n + shift), len(sizes), sum(sizes) + 3
    offsets = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32,
                           device="cuda")
    x = randn(g, slots * k + 8, dtype=dtype)[shift:shift + slots * k].view(slots, k)
    for order in ("kn", "nk"):
        w = randn(g, e, k, 2 * n, dtype=dtype, scale=k ** -0.5)
        if order == "nk":
            w = w.transpose(1, 2).contiguous().transpose(1, 2)
        got = ej.gated_matmul(x, w, offsets)
        leaf = x.detach().requires_grad_()
        assert torch.equal(got, ej.gated_matmul(leaf, w, offsets).detach())
        h, eh, *_ = gated64(x, None, offsets, w, slots, "silu")
        assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])
        assert bool((got[sum(sizes):] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_matmul_views(gpu, dtype):
    """Row strides, bases off 16 bytes, weights of neither order, strided cotangents."""
    g, r, _, _ = product_case(150, 4, 2, 64, 64, "skew", dtype, "kn", False)
    slots = 300
    wide = randn(g, slots, 200, dtype=dtype)
    weights = randn(g, 4, 80, 90, dtype=dtype, scale=0.1)
    for x in (wide[:, :64], wide[:, 1:65], wide.t()[:64].t(), wide[:1, :64].expand(slots, 64)):
        for w in (weights[:, :64, :72], weights[:, 1:65, 3:69], weights[:1, :64].expand(4, 64, 90),
                  weights[:, :64, ::3], weights.transpose(1, 2)[:, 2:66, 5:75]):
            h, eh, *_ = gated64(x, None, r.offsets, w, slots, "silu")
            got = ej.gated_matmul(x, w, r)
            assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])
            cot = randn(g, slots, w.shape[2], dtype=dtype)[:, ::2]
            gx, gw = ej.gated_matmul_vjp(x, w, r, cot)
            hx, hw = ej.gated_matmul_vjp(x.contiguous(), w.contiguous(), r, cot.contiguous())
            # the same projections' gradient but for the order of the sums
            near = 8 * UNIT[dtype]
            assert_within(gx, hx.double(), near * hx.double().abs() + near)
            assert_within(gw, hw.double(), near * hw.double().abs() + near * 20)


@pytest.mark.parametrize("act", ACTS)
def test_gated_gradients_against_differences(gpu, act):
    g, r, x, w = gated_case(40, 5, 2, 24, 18, "skew", F32, "kn", True)
    cot = randn(g, 80, 18)
    gx, gw = ej.gated_matmul_vjp(x, w, r, cot, activation=act, gather=True)
    for leaf, grad, at in ((x, gx, 0), (w, gw, 1)):
        v = randn(g, *leaf.shape)
        v = v / v.norm()
        step = 2.0 ** -6

        def value(sign):
            moved = [x, w]
            moved[at] = leaf + sign * step * v
            return (ej.gated_matmul(*moved, r, activation=act, gather=True).double() * cot).sum()

        num = float(value(1) - value(-1)) / (2 * step)
        want = float((grad.double() * v).sum())
        # rounding: 1440 values of about 1e-6 each over 2^-5; the third
        # derivative's term, step^2 / 6 of about the gradient's size each way
        size = float(gx.norm() + gw.norm())
        assert abs(num - want) <= 1e-3 * size, (num, want, size)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("act", ACTS)
def test_gated_values_far_out(gpu, act, dtype):
    """Gates from none to the largest: finite results and gradients, exact
    limits, NaN where an input has one."""
    gate = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 0.5, -0.5, 5, -5, 12, -12, 40, -40, 90, -90,
                         300, -300, 3e4, -3e4], device="cuda")
    if dtype != F16:
        gate = torch.cat([gate, torch.tensor([1e10, -1e10, 1e20, -1e20, 3e38, -3e38],
                                             device="cuda")])
    gate = gate.to(dtype)
    n = len(gate)
    x = torch.ones(1, 1, dtype=dtype, device="cuda")
    w = torch.cat([gate, torch.full_like(gate, 0.5)])[None]
    leaf = w.detach().requires_grad_()
    h = ej.gated_matmul(x, leaf, activation=act)
    (gw,) = torch.autograd.grad(h, leaf, torch.ones_like(h))
    a, slope = act64(act, gate.double().clamp(-1e6, 1e6))
    a = torch.where(gate.double() > 1e6, gate.double(), a)
    big = gate.abs().double() > 1e6
    slope = torch.where(big, (gate.double() > 0).double(), slope)
    room = torch.where(big, 2.0 ** -22, ROOM(gate.double().clamp(-1e6, 1e6)).clamp(max=1.0))
    # far out the exponential is below 1e-37 and its relative error without bound
    slack = 1e-37 * (1 + gate.double().abs()) + TINY[dtype]
    assert_within(h[0], 0.5 * a, 0.5 * a.abs() * (room + UNIT[dtype]) + slack)
    assert_within(gw[0, :n], 0.5 * slope, 0.5 * slope.abs() * UNIT[dtype] + 1.1 * room.clamp(max=1e-4)
                  + TINY[dtype])
    assert_within(gw[0, n:], a, a.abs() * (room + 2 * UNIT[dtype]) + slack)
    for at in (0, n):
        bad = w.clone()
        bad[0, at] = float("nan")
        leaf = bad.requires_grad_()
        h = ej.gated_matmul(x, leaf, activation=act)
        (gw,) = torch.autograd.grad(h, leaf, torch.ones_like(h))
        assert bool(torch.isnan(h[0, 0])) and torch.isfinite(h[0, 1:]).all()
        assert bool(torch.isnan(gw[0, 0])), "the gate's gradient needs both"
        assert torch.isfinite(gw[0, 1:n]).all()


def test_gated_infinities_stay_in_their_rows(gpu):
    for dtype in (F32, BF16):
        for n_in, n in ((72, 40), (71, 37)):
            g = rng(1)
            offsets = torch.tensor([0, 5, 5, 40], dtype=torch.int32, device="cuda")
            x, w = randn(g, 50, n_in, dtype=dtype), randn(g, 3, n_in, 2 * n, dtype=dtype)
            x[3, n_in - 1] = float("nan")
            x[45:] = float("nan")             # slots of no group
            w[1] = float("nan")               # an expert without slots
            w[2, 0, n - 1] = float("nan")     # a gate
            w[2, 0, n] = float("nan")         # column 0 of the other projection
            y = ej.gated_matmul(x, w, offsets)
            bad = ~torch.isfinite(y)
            want = torch.zeros_like(bad)
            want[3] = True
            want[5:40, n - 1] = True
            want[5:40, 0] = True
            assert torch.equal(bad, want)
            assert bool((y[40:] == 0).all())
            cot = randn(g, 50, n, dtype=dtype)
            cot[40:] = float("nan")
            gx, gw = ej.gated_matmul_vjp(x, w, offsets, cot)
            assert bool((gx[40:] == 0).all()) and bool((gw[1] == 0).all())
            assert torch.isfinite(gx[:3]).all()


def test_gated_offsets_not_covering(gpu):
    g = rng(2)
    x, w = randn(g, 500, 64, dtype=BF16), randn(g, 2, 64, 128, dtype=BF16, scale=0.1)
    offsets = torch.tensor([100, 130, 300], dtype=torch.int32, device="cuda")
    y = ej.gated_matmul(x, w, offsets)
    assert bool((y[:100] == 0).all()) and bool((y[300:] == 0).all())
    gx, _ = ej.gated_matmul_vjp(x, w, offsets, y)
    assert bool((gx[:100] == 0).all()) and bool((gx[300:] == 0).all())
    for o in ([-5, 10, 1 << 30], [500, 500, 500], [9, 3, 2]):  # no access outside
        offsets = torch.tensor(o, dtype=torch.int32, device="cuda")
        assert ej.gated_matmul(x, w, offsets).shape == y.shape
        assert ej.gated_matmul_vjp(x, w, offsets, y)[0].shape == x.shape


def test_gated_matmul_past_32_bits(gpu):
    """Kept projections of more than 2^32 bytes and 2^31 elements."""
    g = rng(4)
    rows, k, n = 68_000, 16, 16_384
    x = randn(g, rows, k, dtype=BF16)
    w = randn(g, k, 2 * n, dtype=BF16, scale=0.25)
    leaves = x.detach().requires_grad_(), w.detach().requires_grad_()
    h = ej.gated_matmul(*leaves)
    cot = torch.zeros(rows, n, dtype=BF16, device="cuda")
    cot[-3:] = randn(g, 3, n, dtype=BF16)
    gx, gw = torch.autograd.grad(h, leaves, cot)
    want, eh, gate, up, eg, eu, ea = gated64(x[-3:], None, None, w[None], 3, "silu")
    assert_within(h[-3:].detach(), want, eh + UNIT[BF16] * (want.abs() + eh) + TINY[BF16])
    d, ed = projections_gradient("silu", gate, up, eg, eu, ea, cot[-3:].double(), BF16)
    w64 = w.double()
    want, off = d @ w64.T, ed @ w64.abs().T
    off = off + 2 * (2 * n + 2) * 2.0 ** -24 * ((d.abs() + ed) @ w64.abs().T)
    assert_within(gx[-3:], want, off + UNIT[BF16] * (want.abs() + off))
    assert bool((gx[:-3] == 0).all())
    want, off = x[-3:].double().T @ d, x[-3:].double().abs().T @ ed
    assert_within(gw, want, off + UNIT[BF16] * (want.abs() + off) + 1e-6)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gated_results_repeat(gpu, dtype):
    g, r, x, w = gated_case(900, 7, 3, 200, 164, "skew", dtype, "kn", True)
    cot = randn(g, 2700, 164, dtype=dtype)
    first = (ej.gated_matmul(x, w, r, gather=True),
             *ej.gated_matmul_vjp(x, w, r, cot, gather=True))
    for _ in range(3):
        again = (ej.gated_matmul(x, w, r, gather=True),
                 *ej.gated_matmul_vjp(x, w, r, cot, gather=True))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_gated_gradients_of_one_side(gpu):
    g, r, x, w = gated_case(100, 4, 2, 64, 48, "padded", BF16, "nk", True)
    cot = randn(g, 200, 48, dtype=BF16)
    gx, gw = ej.gated_matmul_vjp(x, w, r, cot, gather=True)
    lx, lw = x.detach().requires_grad_(), w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(ej.gated_matmul(lx, w, r, gather=True), lx, cot)[0], gx)
    assert torch.equal(torch.autograd.grad(ej.gated_matmul(x, lw, r, gather=True), lw, cot)[0], gw)
    assert ej.gated_matmul_vjp(x, w, r, cot, gather=True, need_x=False)[0] is None
    assert ej.gated_matmul_vjp(x, w, r, cot, gather=True, need_w=False)[1] is None
    # a broadcast cotangent, and accumulation over two uses
    y = ej.gated_matmul(lx, lw, r, gather=True)
    (y.sum() + y.sum()).backward()
    ones = torch.ones_like(y)
    wx, ww = ej.gated_matmul_vjp(x, w, r, 2 * ones, gather=True)
    assert torch.equal(lx.grad, wx) and torch.equal(lw.grad, ww)
    with pytest.raises(RuntimeError, match="first order"):
        (gx,) = torch.autograd.grad(ej.gated_matmul(lx, w, r, gather=True).sum(), lx,
                                    create_graph=True)
        gx.sum().backward()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, x)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ej.gated_matmul(dual, w, r, gather=True)


def test_gated_training_in_a_graph(gpu):
    """Forward and backward captured once, replayed on new data between eager
    calls."""
    g, r, x, w = gated_case(300, 4, 2, 128, 96, "skew", BF16, "kn", True)
    cot = randn(g, 600, 96, dtype=BF16)

    def step():
        return (ej.gated_matmul(x, w, r, gather=True),
                *ej.gated_matmul_vjp(x, w, r, cot, gather=True))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(4):
        x.copy_(randn(g, *x.shape, dtype=BF16))
        cot.copy_(randn(g, *cot.shape, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_gated_refusals_of_gpu_tensors(gpu):
    x = torch.zeros(6, 8, device="cuda")
    w = torch.zeros(2, 8, 10, device="cuda")
    r = ej.group_by_expert(torch.zeros(6, 1, dtype=torch.int32, device="cuda"), 2)
    with pytest.raises(ValueError, match="activation"):
        ej.gated_matmul(x, w, r, activation="relu6")
    with pytest.raises(ValueError, match="columns"):
        ej.gated_matmul(x, w[:, :, :9], r)
    with pytest.raises(ValueError, match="needs groups"):
        ej.gated_matmul(x, w)
    with pytest.raises(ValueError, match="needs groups"):
        ej.gated_matmul(x, w[:1], gather=True)
    with pytest.raises(ValueError, match="must be"):
        ej.gated_matmul(x, w[:, :7], r)
    with pytest.raises(ValueError, match="gather=True needs"):
        ej.gated_matmul(x, w, r.offsets, gather=True)
    with pytest.raises(ValueError, match="experts"):
        ej.gated_matmul(x, w[:1], r)
    with pytest.raises(ValueError, match="rows"):
        ej.gated_matmul(x[:5], w, r)
    with pytest.raises(TypeError):
        ej.gated_matmul(x, w.half(), r)
    with pytest.raises(TypeError):
        ej.gated_matmul(x.double(), w.double(), r)
    with pytest.raises(TypeError):
        ej.gated_matmul(x.cpu(), w, r)
    with pytest.raises(ValueError, match="grad_out"):
        ej.gated_matmul_vjp(x, w, r, torch.zeros(6, 10, device="cuda"))
