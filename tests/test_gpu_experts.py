"""Expert operators against their definitions in 64 bits.

Bounds are those of the arithmetic: a sum of n products formed in fp32 is off
by at most about n 2^-24 times the sum of the products' magnitudes (twice that
is allowed, for sums formed in another order and of products rounded before
they are added), and one rounding to the result's type by its unit roundoff.
"""

import pytest
import torch

import einjax_amd as ej

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
UNIT = {F32: 2.0 ** -24, BF16: 2.0 ** -8, F16: 2.0 ** -11}
TINY = {F32: 2.0 ** -149, BF16: 2.0 ** -133, F16: 2.0 ** -24}


def rng(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(g, *shape, dtype=F32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)


def assert_within(got, want, bound):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bad.any(), (f"{int(bad.sum())} of {bad.numel()} off, worst "
                           f"{float((err / bound.clamp(min=1e-300)).max()):.3g} times the bound")


def sum_bound(want, magnitudes, n, dtype):
    return UNIT[dtype] * want.abs() + 2 * (n + 2) * 2.0 ** -24 * magnitudes + TINY[dtype]


def make_picks(t, k, e, seed, kind="even"):
    """Distinct experts of each token: even, skewed, all on the first ones,
    with padded tokens, with single missing picks, or none at all."""
    g = rng(seed)
    score = torch.rand(t, e, generator=g, device="cuda")
    if kind == "skew":
        score = score * torch.exp(2 * torch.randn(e, generator=g, device="cuda"))
    if kind == "first":
        score = -torch.arange(e, device="cuda").float().expand(t, e)
    picks = torch.sort(score, dim=1, descending=True).indices[:, :k].contiguous()
    if kind == "padded" and t:
        picks[torch.rand(t, generator=g, device="cuda") < 0.3] = -1
    if kind == "holes" and t:
        picks[torch.rand(t, k, generator=g, device="cuda") < 0.3] = -1
    if kind == "none":
        picks.fill_(-1)
    return picks


def plain_grouping(picks, e):
    t, k = picks.shape
    flat = picks.reshape(-1).tolist()
    order = sorted((p for p in range(t * k) if 0 <= flat[p] < e), key=lambda p: flat[p])
    offsets, rows, slots = [0] * (e + 1), [0] * (t * k), [-1] * (t * k)
    for s, p in enumerate(order):
        rows[s], slots[p] = p // k, s
        offsets[flat[p] + 1] += 1
    for i in range(e):
        offsets[i + 1] += offsets[i]
    return offsets, rows, [slots[i * k:(i + 1) * k] for i in range(t)]


# ---- routing ------------------------------------------------------------------

ROUTES = [(0, 4, 2), (1, 1, 1), (1, 64, 4), (3, 7, 7), (17, 16, 16), (255, 33, 3), (256, 8, 2),
          (257, 8, 2), (300, 128, 8), (1000, 200, 5), (4097, 60, 6), (700, 257, 9),
          (90, 1024, 16), (500, 1000, 4)]


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k", ROUTES)
def test_route(gpu, t, e, k, dtype, renorm):
    g = rng(t + e)
    logits = randn(g, t, e, dtype=dtype, scale=2.0)
    if t > 4 and e > 8:
        logits[1] = 0.5                     # all equal: the lowest experts
        logits[2, ::2] = -float("inf")      # half excluded
        logits[3] = -float("inf")           # a padding token
        logits[4] = torch.finfo(dtype).min  # all of the lowest value
        logits[0, :3] = -0.0
        logits[0, 3:6] = 0.0
    r = ej.route_experts(logits, k, renormalize=renorm)
    l64 = logits.double()
    order = torch.sort(l64, dim=1, descending=True, stable=True)
    picks = order.indices[:, :k].clone()
    held = order.values[:, :k] > -float("inf")
    picks[~held] = -1
    assert torch.equal(r.experts.long(), picks)
    offsets, rows, slots = plain_grouping(picks, e)
    assert r.offsets.tolist() == offsets
    assert r.rows.tolist() == rows
    assert r.slots.tolist() == slots
    top = torch.where(held, order.values[:, :k], -float("inf"))
    want = torch.softmax(top, 1) if renorm else torch.softmax(l64, 1).gather(
        1, order.indices[:, :k])
    want = torch.where(held, want, torch.zeros_like(want))
    # exp within 2 ulp, of an argument rounded once; a sum of e terms; a division
    arg = 40.0 if t > 4 and e > 8 else 20.0
    assert_within(r.weights, want, (arg + e + 8) * 2.0 ** -24 * want + 1e-37)


def test_route_nan_and_infinity(gpu):
    logits = torch.zeros(4, 6, device="cuda")
    logits[1, 4] = float("nan")
    logits[2, 3] = float("inf")
    logits[3, 1] = 1.0
    r = ej.route_experts(logits, 2)
    assert r.experts.tolist() == [[0, 1], [4, 0], [3, 0], [1, 0]]
    w = r.weights.cpu()
    assert torch.isnan(w[1]).all() and torch.isnan(w[2]).all()
    assert torch.isfinite(w[0]).all() and torch.isfinite(w[3]).all()


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k", [r for r in ROUTES if r[0] > 0])
def test_route_gradient(gpu, t, e, k, dtype, renorm):
    g = rng(t * e)
    logits = randn(g, t, e, dtype=dtype, scale=1.5)
    if t > 4 and e > 8:
        logits[2, ::2] = -float("inf")
        logits[3] = -float("inf")
    leaf = logits.clone().requires_grad_()
    r = ej.route_experts(leaf, k, renormalize=renorm)
    cot = randn(g, t, k)
    (got,) = torch.autograd.grad(r.weights, leaf, cot)
    assert got.dtype == dtype
    l64 = logits.double()
    picks = r.experts.long().clamp(min=0)
    held = (r.experts >= 0)
    p = torch.exp(l64 - torch.clamp(l64.amax(1, keepdim=True), min=-1e30))
    if renorm:
        p = torch.zeros_like(p).scatter_add(1, picks, p.gather(1, picks) * held)
    p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    full = torch.zeros_like(p).scatter_add(1, picks, cot.double() * held)
    dot = (p * full).sum(1, keepdim=True)
    want = p * (full - dot)
    mag = p * (full.abs() + (p * full.abs()).sum(1, keepdim=True))
    assert_within(got, want, UNIT[dtype] * want.abs() + (60 + 2 * e) * 2.0 ** -24 * mag
                  + TINY[dtype])


def test_route_gradient_against_differences(gpu):
    g = rng(5)
    logits = randn(g, 12, 10)
    cot = randn(g, 12, 3)
    for renorm in (True, False):
        r = ej.route_experts(logits, 3, renormalize=renorm)
        grad = ej.route_experts_vjp(logits, r.experts, cot, renormalize=renorm)
        d = randn(g, 12, 10)
        h = 2.0 ** -7
        up = ej.route_experts(logits + h * d, 3, renormalize=renorm)
        down = ej.route_experts(logits - h * d, 3, renormalize=renorm)
        same = (up.experts == r.experts).all(1) & (down.experts == r.experts).all(1)
        assert int(same.sum()) >= 6
        num = ((up.weights - down.weights).double() * cot).sum(1) / (2 * h)
        want = (grad.double() * d).sum(1)
        # central differences: h^2 times third derivatives of a softmax along d
        # (at most |d|^3 |cot|), and rounding 2^-22 / h
        room = (h * h * d.norm(dim=1) ** 3 + 2.0 ** -22 / h * 4) * cot.norm(dim=1)
        assert (((num - want).abs() <= room) | ~same).all()


def test_route_takes_strided_logits(gpu):
    g = rng(9)
    wide = randn(g, 40, 50)
    for logits in (wide[:, 3:19], wide[::2, :20], wide.t()[:30]):
        a = ej.route_experts(logits, 4)
        b = ej.route_experts(logits.contiguous(), 4)
        assert torch.equal(a.experts, b.experts) and torch.equal(a.weights, b.weights)
        ga = ej.route_experts_vjp(logits, a.experts, a.weights)
        gb = ej.route_experts_vjp(logits.contiguous(), a.experts, a.weights)
        assert torch.equal(ga, gb)


@pytest.mark.parametrize("kind", ["even", "skew", "first", "padded", "holes", "none"])
@pytest.mark.parametrize("t,e,k", [(0, 3, 2), (1, 5, 1), (200, 9, 3), (256, 300, 16), (1500, 9, 3),
                                   (3000, 1024, 7)])
def test_group_by_expert(gpu, t, e, k, kind):
    picks = make_picks(t, k, e, 7, kind)
    if t > 3:
        picks[3, 0] = e + 5  # outside: no slot
    r = ej.group_by_expert(picks, e)
    offsets, rows, slots = plain_grouping(picks, e)
    assert r.offsets.tolist() == offsets
    assert r.rows.tolist() == rows
    assert r.slots.tolist() == slots
    assert bool((r.weights == 1).all())


# ---- grouped products ------------------------------------------------------------

def row_groups(offsets, slots):
    """Group of each slot, -1 for none."""
    ends = offsets.tolist()
    owner = torch.full((slots,), -1, dtype=torch.long)
    for e in range(len(ends) - 1):
        owner[ends[e]:ends[e + 1]] = e
    return owner.tolist(), ends


def product64(x, rows, offsets, w, slots):
    out = torch.zeros(slots, w.shape[2], dtype=torch.double, device="cuda")
    mag = torch.zeros_like(out)
    _, ends = row_groups(offsets, slots)
    for e in range(w.shape[0]):
        a, b = ends[e], ends[e + 1]
        if a == b:
            continue
        xe = x[rows[a:b].long()].double() if rows is not None else x[a:b].double()
        out[a:b] = xe @ w[e].double()
        mag[a:b] = xe.abs() @ w[e].double().abs()
    return out, mag


# tokens, experts, picks, k, n, kind of picks
PRODUCTS = [
    (1, 1, 1, 64, 64, "even"), (1, 4, 2, 128, 96, "even"), (2, 16, 2, 2048, 512, "even"),
    (5, 3, 2, 1, 1, "even"), (7, 2, 1, 8, 8, "even"), (40, 6, 3, 72, 200, "padded"),
    (33, 5, 2, 77, 131, "skew"), (129, 4, 1, 64, 264, "first"), (300, 70, 2, 96, 136, "skew"),
    (257, 8, 2, 520, 392, "holes"), (600, 3, 2, 320, 640, "skew"), (700, 9, 4, 129, 67, "even"),
    (64, 4, 2, 256, 128, "none"), (1500, 2, 2, 200, 1030, "skew"), (2048, 2, 1, 1024, 512, "even"),
]


def product_case(t, e, k, n_in, n_out, kind, dtype, order, gather, seed=3):
    g = rng(seed + t + n_in)
    r = ej.group_by_expert(make_picks(t, k, e, seed, kind), e)
    x = randn(g, t if gather else t * k, n_in, dtype=dtype)
    w = randn(g, e, n_in, n_out, dtype=dtype, scale=n_in ** -0.5)
    if order == "nk":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    return g, r, x, w


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k,n_in,n_out,kind", PRODUCTS)
def test_grouped_matmul(gpu, t, e, k, n_in, n_out, kind, dtype, order):
    for gather in (False, True):
        _, r, x, w = product_case(t, e, k, n_in, n_out, kind, dtype, order, gather)
        got = ej.grouped_matmul(x, w, r, gather=gather)
        want, mag = product64(x, r.rows if gather else None, r.offsets, w, t * k)
        assert got.dtype == dtype
        assert_within(got, want, sum_bound(want, mag, n_in, dtype))
        if not gather:
            again = ej.grouped_matmul(x, w, r.offsets.long(), out_dtype=F32)
            assert again.dtype == F32
            assert_within(again, want, sum_bound(want, mag, n_in, F32))


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k,n_in,n_out,kind", PRODUCTS)
def test_grouped_matmul_gradients(gpu, t, e, k, n_in, n_out, kind, dtype, order):
    for gather in (False, True):
        g, r, x, w = product_case(t, e, k, n_in, n_out, kind, dtype, order, gather)
        x.requires_grad_()
        w = w.detach().requires_grad_()
        y = ej.grouped_matmul(x, w, r, gather=gather)
        cot = randn(g, t * k, n_out, dtype=dtype)
        gx, gw = torch.autograd.grad(y, (x, w), cot)
        assert gx.dtype == dtype and gw.dtype == dtype and gw.stride() == w.stride()
        _, ends = row_groups(r.offsets, t * k)
        x, w = x.detach(), w.detach()
        wx = torch.zeros(t * k, n_in, dtype=torch.double, device="cuda")
        mx = torch.zeros_like(wx)
        for i in range(e):
            a, b = ends[i], ends[i + 1]
            at = r.rows[a:b].long() if gather else torch.arange(a, b, device="cuda")
            xi, gi, wi = x[at].double(), cot[a:b].double(), w[i].double()
            wx[a:b], mx[a:b] = gi @ wi.T, gi.abs() @ wi.abs().T
            assert_within(gw[i], xi.T @ gi,
                          sum_bound(xi.T @ gi, xi.abs().T @ gi.abs(), b - a, dtype))
        bound = sum_bound(wx, mx, n_out, dtype)
        if gather:
            # each slot's row is rounded to the operands' type, then summed
            total, room, size = (torch.zeros(t, n_in, dtype=torch.double, device="cuda")
                                 for _ in range(3))
            at = r.rows[:ends[-1]].long()
            total.index_add_(0, at, wx[:ends[-1]])
            room.index_add_(0, at, bound[:ends[-1]])
            size.index_add_(0, at, wx[:ends[-1]].abs() + bound[:ends[-1]])
            wx, bound = total, room + UNIT[dtype] * (total.abs() + room) + 2 * (k + 2) * \
                2.0 ** -24 * size + TINY[dtype]
        assert_within(gx, wx, bound)


# Groups of 256-row blocks that are cut in different ways: rows of each group,
# slots of no group behind them, k, n.
LARGE = [
    ([1000], 24, 64, 4096), ([1024, 0, 512], 0, 64, 4104), ([300, 0, 724], 0, 128, 6144),
    ([900, 1100, 1000, 1096], 5, 72, 4096), ([900, 1100, 1000, 1096], 0, 16, 6400),
    ([129, 128, 1, 1790], 3, 192, 4112),
]


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes,dead,k,n", LARGE)
def test_grouped_matmul_large_blocks(gpu, sizes, dead, k, n, dtype, order):
    g, e, live = rng(k + n), len(sizes), sum(sizes)
    offsets = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32,
                           device="cuda")
    x = randn(g, live + dead, k, dtype=dtype)
    w = randn(g, e, k, n, dtype=dtype, scale=k ** -0.5)
    if order == "nk":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    x[live:] = float("nan")
    got = ej.grouped_matmul(x, w, offsets)
    x[live:] = 0
    want, mag = product64(x, None, offsets, w, live + dead)
    assert_within(got, want, sum_bound(want, mag, k, dtype))
    if dtype == F16:
        return
    # the gradient to x with the same blocks, k and n exchanged, and in 8 bits
    wt = w.transpose(1, 2)
    cot = randn(g, live + dead, k, dtype=dtype)
    gx, _ = ej.grouped_matmul_vjp(randn(g, live + dead, n, dtype=dtype), wt, offsets, cot,
                                  need_w=False)
    cot[live:] = 0
    want, mag = product64(cot, None, offsets, w, live + dead)
    assert_within(gx, want, sum_bound(want, mag, k, dtype))
    q = torch.randint(-128, 128, (live + dead, k), generator=g, device="cuda").to(torch.int8)
    p = torch.randint(-128, 128, (e, n, k), generator=g, device="cuda").to(torch.int8)
    qs, ps = (torch.rand(s, generator=g, device="cuda") for s in (live + dead, (e, n)))
    got = ej.int8_matmul(q, qs, p, ps, offsets, out_dtype=F32)
    q[live:] = 0
    want, _ = product64(q, None, offsets, p.transpose(1, 2), live + dead)
    owner = torch.tensor([max(o, 0) for o in row_groups(offsets, live + dead)[0]], device="cuda")
    want = want * qs.double()[:, None] * ps[owner].double()
    assert_within(got, want, 5 * 2.0 ** -24 * want.abs() + TINY[F32])


@pytest.mark.parametrize("gather", [False, True])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes,m,n", [
    ([70, 0, 131, 64], 1024, 1024), ([40, 0, 200, 1, 65, 31, 90, 33, 64], 2048, 2048),
    ([3, 70, 64, 90, 1, 0, 128, 40, 10], 2048, 2312), ([129, 30, 0, 77], 2048, 4000),
    ([70, 0, 131, 64, 3, 9, 20, 1], 1023, 1029), ([5, 200, 0, 77, 1], 1031, 1800)])
def test_grouped_weight_gradient_large_blocks(gpu, sizes, m, n, dtype, gather):
    g, e, live = rng(m + n), len(sizes), sum(sizes)
    r = ej.group_by_expert(torch.repeat_interleave(torch.arange(e), torch.tensor(sizes))
                           [torch.randperm(live, generator=torch.Generator().manual_seed(n))]
                           .cuda()[:, None], e)
    x, w = randn(g, live, m, dtype=dtype), randn(g, e, m, n, dtype=dtype)
    cot = randn(g, live, n, dtype=dtype)
    _, gw = ej.grouped_matmul_vjp(x, w, r, cot, gather=gather, need_x=False)
    _, ends = row_groups(r.offsets, live)
    for i in range(e):
        a, b = ends[i], ends[i + 1]
        xi = (x[r.rows[a:b].long()] if gather else x[a:b]).double()
        gi = cot[a:b].double()
        assert_within(gw[i], xi.T @ gi, sum_bound(xi.T @ gi, xi.abs().T @ gi.abs(), b - a, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes,k,n,shift", [
    ([4, 0, 9, 1], 1539, 294, 0), ([16, 30, 2], 2047, 129, 0), ([130], 2500, 70, 0),
    ([60, 12], 2048, 72, 0), ([60, 12], 2048, 72, 1), ([100, 0, 300], 4096, 64, 0)])
def test_grouped_matmul_split_contractions(gpu, sizes, k, n, shift, dtype):
    """Few tiles over a long contraction, whose parts are summed apart: rows on
    and off 16 bytes, operands that start off 16 bytes (shift elements)."""
    g, e, slots = rng(k + n + shift), len(sizes), sum(sizes) + 3
    offsets = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32,
                           device="cuda")
    x = randn(g, slots * k + 8, dtype=dtype)[shift:shift + slots * k].view(slots, k)
    for order in ("kn", "nk"):
        w = randn(g, e, k, n, dtype=dtype, scale=k ** -0.5)
        if order == "nk":
            w = w.transpose(1, 2).contiguous().transpose(1, 2)
        got = ej.grouped_matmul(x, w, offsets)
        want, mag = product64(x, None, offsets, w, slots)
        assert_within(got, want, sum_bound(want, mag, k, dtype))
        assert bool((got[sum(sizes):] == 0).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes,m,n,shift", [
    ([3000, 0, 700], 75, 151, 0), ([9, 5000], 64, 40, 0), ([2500], 128, 128, 1),
    ([1200, 800, 1], 77, 64, 0)])
def test_grouped_weight_gradient_split_contractions(gpu, sizes, m, n, shift, dtype):
    g, e, slots = rng(m + n + shift), len(sizes), sum(sizes)
    offsets = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32,
                           device="cuda")
    x = randn(g, slots * m + 8, dtype=dtype)[shift:shift + slots * m].view(slots, m)
    cot, w = randn(g, slots, n, dtype=dtype), randn(g, e, m, n, dtype=dtype)
    for wt in (w, w.transpose(1, 2).contiguous().transpose(1, 2)):
        _, gw = ej.grouped_matmul_vjp(x, wt, offsets, cot, need_x=False)
        ends = offsets.tolist()
        for i in range(e):
            xi, gi = (v[ends[i]:ends[i + 1]].double() for v in (x, cot))
            assert_within(gw[i], xi.T @ gi,
                          sum_bound(xi.T @ gi, xi.abs().T @ gi.abs(), len(xi), dtype))


def test_grouped_gradients_against_differences(gpu):
    g, r, x, w = product_case(40, 5, 2, 24, 36, "skew", F32, "kn", True)
    cot = randn(g, 80, 36)
    gx, gw = ej.grouped_matmul_vjp(x, w, r, cot, gather=True)
    dx, dw = randn(g, *x.shape), randn(g, *w.shape)
    # the product is bilinear: central differences are exact up to rounding
    for direction, grad, move in ((dx, gx, lambda h: (x + h * dx, w)),
                                  (dw, gw, lambda h: (x, w + h * dw))):
        up, down = (ej.grouped_matmul(*move(h), r, gather=True).double() for h in (0.5, -0.5))
        num = ((up - down) * cot).sum()
        want = (grad.double() * direction).sum()
        size = (up.abs() * cot.abs()).sum() + (grad.abs() * direction.abs()).double().sum()
        assert abs(float(num - want)) <= 2 * 100 * 2.0 ** -24 * float(size)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_grouped_matmul_views(gpu, dtype):
    """Row strides, bases off 16 bytes and weights of neither order."""
    g, r, _, _ = product_case(150, 4, 2, 64, 64, "skew", dtype, "kn", False)
    slots = 300
    wide = randn(g, slots, 200, dtype=dtype)
    weights = randn(g, 4, 80, 90, dtype=dtype)
    for x in (wide[:, :64], wide[:, 1:65], wide[:, 8:72], wide.t()[:64].t(),
              wide[:1, :64].expand(slots, 64)):
        for w in (weights[:, :64, :72], weights[:, 1:65, 3:70], weights[:, :, :64].transpose(1, 2)
                  [:, :, :80], weights[:1, :64].expand(4, 64, 90), weights[:, :64, ::2],
                  weights.transpose(1, 2)[:, 2:66, 5:75]):
            got = ej.grouped_matmul(x, w, r)
            want, mag = product64(x, None, r.offsets, w, slots)
            assert_within(got, want, sum_bound(want, mag, 64, dtype))
            cot = randn(g, slots, 2 * w.shape[2], dtype=dtype)[:, ::2]
            gx, gw = ej.grouped_matmul_vjp(x, w, r, cot)
            hx, hw = ej.grouped_matmul_vjp(x.contiguous(), w.contiguous(), r, cot.contiguous())
            assert_within(gx, hx.double(), 4 * UNIT[dtype] * hx.double().abs() + 1e-3)
            assert_within(gw, hw.double(), 4 * UNIT[dtype] * hw.double().abs() + 1e-3)


def test_grouped_matmul_infinities_stay_in_their_rows(gpu):
    """A NaN or infinity reaches its own results only: not other rows, not
    other groups, not what pads a tile."""
    for dtype in (F32, BF16):
        for n_in, n_out in ((72, 40), (71, 37)):
            g = rng(1)
            offsets = torch.tensor([0, 5, 5, 40], dtype=torch.int32, device="cuda")
            x, w = randn(g, 50, n_in, dtype=dtype), randn(g, 3, n_in, n_out, dtype=dtype)
            x[3, n_in - 1] = float("inf")
            x[45:] = float("nan")         # slots of no group
            w[1] = float("nan")           # an expert without slots
            w[2, 0, n_out - 1] = float("nan")
            y = ej.grouped_matmul(x, w, offsets)
            bad = ~torch.isfinite(y)
            want = torch.zeros_like(bad)
            want[3] = True
            want[5:40, n_out - 1] = True
            assert torch.equal(bad, want)
            assert bool((y[40:] == 0).all())
            cot = randn(g, 50, n_out, dtype=dtype)
            cot[40:] = float("nan")
            gx, gw = ej.grouped_matmul_vjp(x, w, offsets, cot)
            assert bool((gx[40:] == 0).all()) and bool((gw[1] == 0).all())
            assert torch.isfinite(gx[:5]).all() and torch.isfinite(gw[2]).all()


def test_grouped_matmul_offsets_not_covering(gpu):
    """Slots before the first offset and past the last are zero."""
    g = rng(2)
    x, w = randn(g, 500, 64, dtype=BF16), randn(g, 2, 64, 128, dtype=BF16)
    offsets = torch.tensor([100, 130, 300], dtype=torch.int32, device="cuda")
    y = ej.grouped_matmul(x, w, offsets)
    assert bool((y[:100] == 0).all()) and bool((y[300:] == 0).all())
    want, mag = torch.zeros(500, 128, dtype=torch.double, device="cuda"), None
    want[100:130] = x[100:130].double() @ w[0].double()
    want[130:300] = x[130:300].double() @ w[1].double()
    mag = x.double().abs() @ w.double().abs().amax(0)
    assert_within(y, want, sum_bound(want, mag, 64, BF16))


def test_grouped_matmul_wild_offsets_stay_in_bounds(gpu):
    """Offsets outside the slots give undefined rows, no access outside."""
    g = rng(2)
    x, w = randn(g, 64, 64, dtype=BF16), randn(g, 3, 64, 64, dtype=BF16)
    for o in ([-5, 10, 7, 1 << 30], [0, 64, 64, 64], [64, 64, 64, 64], [9, 3, 2, 1]):
        offsets = torch.tensor(o, dtype=torch.int32, device="cuda")
        assert ej.grouped_matmul(x, w, offsets).shape == (64, 64)
        gx, gw = ej.grouped_matmul_vjp(x, w, offsets, x)
        assert gx.shape == x.shape and gw.shape == w.shape


def test_grouped_matmul_past_32_bits(gpu):
    """Operands and results of more than 2^31 elements."""
    g = rng(4)
    rows, n_in, n_out = 530_000, 4096, 64
    x = torch.empty(rows, n_in, dtype=BF16, device="cuda")   # 2.17e9 elements
    last = randn(g, 40, n_in, dtype=BF16)
    x[-40:] = last
    w = randn(g, 2, n_in, n_out, dtype=BF16, scale=n_in ** -0.5)
    offsets = torch.tensor([rows - 40, rows - 15, rows], dtype=torch.int32, device="cuda")
    y = ej.grouped_matmul(x, w, offsets)
    want = torch.cat([last[:25].double() @ w[0].double(), last[25:].double() @ w[1].double()])
    mag = torch.cat([last[:25].double().abs() @ w[0].double().abs(),
                     last[25:].double().abs() @ w[1].double().abs()])
    assert_within(y[-40:], want, sum_bound(want, mag, n_in, BF16))
    _, gw = ej.grouped_matmul_vjp(x, w, offsets, y, need_x=False)
    got = y[-40:].double()
    for i, (a, b) in enumerate(((0, 25), (25, 40))):
        wg = last[a:b].double().T @ got[a:b]
        assert_within(gw[i], wg, sum_bound(wg, last[a:b].double().abs().T @ got[a:b].abs(), 25,
                                           BF16))
    del x
    w = randn(g, 1, 8, 131_072, dtype=BF16)
    x = randn(g, 17_000, 8, dtype=BF16)
    y = ej.grouped_matmul(x, w, torch.tensor([0, 17_000], device="cuda"))  # 2.2e9 elements
    want = x[-3:].double() @ w[0].double()
    assert_within(y[-3:], want, sum_bound(want, x[-3:].double().abs() @ w[0].double().abs(), 8,
                                          BF16))


def test_grouped_matmul_on_another_stream(gpu):
    _, r, x, w = product_case(300, 4, 2, 256, 256, "skew", BF16, "kn", True)
    want = ej.grouped_matmul(x, w, r, gather=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ej.grouped_matmul(x, w, r, gather=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)


def test_expert_layer_in_a_graph(gpu):
    """Routing, products and the sum captured once and replayed on new data."""
    g = rng(8)
    x = randn(g, 64, 128, dtype=BF16)
    gate = randn(g, 128, 8, dtype=BF16)
    up, down = randn(g, 8, 128, 256, dtype=BF16), randn(g, 8, 256, 128, dtype=BF16)

    def layer():
        r = ej.route_experts(x @ gate, 2)
        h = ej.grouped_matmul(x, up, r, gather=True)
        return ej.combine_experts(ej.grouped_matmul(h, down, r), r)

    layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer()
    for i in range(4):
        x.copy_(randn(g, 64, 128, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_grouped_results_repeat(gpu, dtype):
    g, r, x, w = product_case(900, 7, 3, 200, 328, "skew", dtype, "kn", True)
    cot = randn(g, 2700, 328, dtype=dtype)
    first = (ej.grouped_matmul(x, w, r, gather=True),
             *ej.grouped_matmul_vjp(x, w, r, cot, gather=True))
    for _ in range(3):
        again = (ej.grouped_matmul(x, w, r, gather=True),
                 *ej.grouped_matmul_vjp(x, w, r, cot, gather=True))
        assert all(torch.equal(a, b) for a, b in zip(first, again))


# ---- back to tokens ---------------------------------------------------------------

@pytest.mark.parametrize("kind", ["even", "padded", "holes", "none"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k,n", [(1, 2, 1, 1), (1, 8, 4, 2048), (37, 5, 3, 77), (37, 5, 3, 72),
                                     (300, 16, 16, 40), (513, 6, 2, 4104)])
def test_combine(gpu, t, e, k, n, dtype, kind):
    g = rng(t + n)
    r = ej.group_by_expert(make_picks(t, k, e, 3, kind), e, torch.rand(t, k, generator=g,
                                                                       device="cuda"))
    y = randn(g, t * k, n, dtype=dtype)
    live = int(r.offsets[-1])
    y[live:] = float("nan")  # rows of no pair are not read
    yl, wl = y.clone().requires_grad_(), r.weights.clone().requires_grad_()
    out = ej.combine_experts(yl, r, wl)
    assert torch.equal(out, ej.combine_experts(y, r, wl.detach()))
    slots = r.slots.long()
    held = slots >= 0
    if live:
        at = y[slots.clamp(min=0, max=live - 1)].double() * held[..., None]
    else:
        at = torch.zeros(t, k, n, dtype=torch.double, device="cuda")
    w = r.weights.double()[..., None]
    want = (w * at).sum(1)
    assert_within(out, want, sum_bound(want, (w * at).abs().sum(1), k, dtype))
    cot = randn(g, t, n, dtype=dtype)
    gy, gw = torch.autograd.grad(out, (yl, wl), cot)
    wy = torch.zeros(t * k + 1, n, dtype=torch.double, device="cuda")
    wy[torch.where(held, slots, t * k).reshape(-1)] = \
        (w * cot.double()[:, None]).reshape(-1, n)
    wy = wy[:-1]
    wy[live:] = 0
    assert_within(gy, wy, (UNIT[dtype] + 2.0 ** -23) * wy.abs() + TINY[dtype])
    ww = (at * cot.double()[:, None]).sum(2)
    assert_within(gw, ww, 2 * (n + 2) * 2.0 ** -24 * (at * cot.double()[:, None]).abs().sum(2)
                  + 1e-37)


def test_combine_strided(gpu):
    g = rng(6)
    r = ej.group_by_expert(make_picks(50, 2, 4, 3, "holes"), 4)
    wide = randn(g, 100, 300, dtype=BF16)
    cots = randn(g, 50, 300, dtype=BF16)
    for sl in (slice(0, 64), slice(3, 67), slice(0, 128, 2)):
        y, c = wide[:, sl], cots[:, sl]
        assert torch.equal(ej.combine_experts(y, r), ej.combine_experts(y.contiguous(), r))
        a = ej.combine_experts_vjp(y, r, c)
        b = ej.combine_experts_vjp(y.contiguous(), r, c.contiguous())
        assert torch.equal(a[0], b[0])
        bound = 2 * 66 * 2.0 ** -24 * (y.double().abs().amax() * c.double().abs().sum(1))
        assert ((a[1] - b[1]).double().abs() <= bound[:, None]).all()


# ---- 8-bit integers ----------------------------------------------------------------

@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n", [(0, 5), (1, 1), (3, 64), (5, 77), (130, 2048), (9, 10000)])
def test_quantize_rows(gpu, m, n, dtype):
    g = rng(m + n)
    x = randn(g, m, n, dtype=dtype, scale=3.0)
    if m >= 3:
        x[1] = 0
    q, scale = ej.quantize_rows(x)
    assert q.dtype == torch.int8 and q.shape == x.shape and scale.shape == (m,)
    want = x.float().abs().amax(1) * torch.tensor(1 / 127, device="cuda") if m else scale
    assert torch.equal(scale, want)
    exact = torch.where(scale[:, None] > 0, x.double() / scale.double()[:, None], 0.0)
    # a tie may go either way where the quotient's own rounding decides it
    assert ((q.double() - exact).abs() <= 0.5 + 128 * 2.0 ** -24).all()
    assert int(q.abs().amax()) <= 127 if m else True
    if m:
        assert torch.equal(q.abs().amax(1) == 127, scale > 0)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [7, 9, 513, 1001, 2055, 4095])
def test_combine_rows_of_no_whole_pieces(gpu, n, dtype):
    test_combine(gpu, 33, 5, 3, n, dtype, "holes")


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n", [(2000, 77), (2000, 1001), (1100, 4095), (3, 4097), (2, 30001)])
def test_quantize_rows_of_no_whole_pieces(gpu, m, n, dtype):
    test_quantize_rows(gpu, m, n, dtype)


def test_quantize_rows_not_finite_and_tiny(gpu):
    x = torch.ones(5, 40, device="cuda")
    x[1, 7] = float("inf")
    x[2, 39] = float("nan")
    x[3] = 1e-45
    x[4] = 3e38
    q, scale = ej.quantize_rows(x)
    assert torch.isnan(scale[1:3]).all() and torch.isfinite(scale[[0, 3, 4]]).all()
    assert bool((q[1:3] == 0).all()) and bool((q[[0, 4]] == 127).all())
    w, ws = ej.quantize_rows(torch.randn(16, 40, device="cuda"))
    y = ej.int8_matmul(q, scale, w, ws)
    assert torch.isnan(y[1:3]).all() and torch.isfinite(y[[0, 3]]).all()
    # the last row's products reach infinity where bf16 ends, and only there
    want = (q[4].double() @ w.double().T) * scale[4].double() * ws.double()
    assert torch.equal(torch.isinf(y[4]), want.abs() >= 2.0 ** 128 - 2.0 ** 119)


def test_quantize_rows_views(gpu):
    g = rng(3)
    wide = randn(g, 4, 30, 200, dtype=BF16)
    for x in (wide, wide[:, :, 3:75], wide[:, ::2, :64], wide.transpose(1, 2)):
        q, s = ej.quantize_rows(x)
        p, t = ej.quantize_rows(x.contiguous())
        assert torch.equal(q, p) and torch.equal(s, t)


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k,n_in,n_out,kind", PRODUCTS)
def test_int8_matmul(gpu, t, e, k, n_in, n_out, kind, out_dtype):
    g = rng(t + n_out)
    r = ej.group_by_expert(make_picks(t, k, e, 3, kind), e)
    w = torch.randint(-128, 128, (e, n_out, n_in), generator=g, device="cuda").to(torch.int8)
    ws = torch.rand(e, n_out, generator=g, device="cuda") * 1e-4
    for gather in (False, True):
        m = t if gather else t * k
        q = torch.randint(-128, 128, (m, n_in), generator=g, device="cuda").to(torch.int8)
        qs = torch.rand(m, generator=g, device="cuda")
        got = ej.int8_matmul(q, qs, w, ws, r, gather=gather, out_dtype=out_dtype)
        assert got.dtype == out_dtype
        want = torch.zeros(t * k, n_out, dtype=torch.double, device="cuda")
        _, ends = row_groups(r.offsets, t * k)
        for i in range(e):
            a, b = ends[i], ends[i + 1]
            at = r.rows[a:b].long() if gather else torch.arange(a, b, device="cuda")
            want[a:b] = (q[at].double() @ w[i].double().T) * qs[at].double()[:, None] \
                * ws[i].double()
        # the sum is exact; its conversion and two products round
        assert_within(got, want, (UNIT[out_dtype] + 4 * 2.0 ** -24) * want.abs()
                      + TINY[out_dtype])


@pytest.mark.parametrize("m,n_in,n_out", [(0, 64, 32), (1, 4096, 256), (4, 100, 33), (200, 256, 300)])
def test_int8_matmul_dense(gpu, m, n_in, n_out):
    g = rng(m + 1)
    x, w = randn(g, m, n_in), randn(g, n_out, n_in)
    q, qs = ej.quantize_rows(x)
    p, ps = ej.quantize_rows(w)
    want = (q.double() @ p.double().T) * qs.double()[:, None] * ps.double()
    for pw, pss in ((p, ps), (p[None], ps[None])):
        got = ej.int8_matmul(q, qs, pw, pss, out_dtype=F32)
        assert_within(got, want, 5 * 2.0 ** -24 * want.abs() + 1e-37)
    # the largest sums that 32 bits hold
    k = 131_071
    a = torch.full((2, k), -128, dtype=torch.int8, device="cuda")
    one = torch.ones(2, device="cuda")
    got = ej.int8_matmul(a, one, a, one, out_dtype=F32)
    assert bool((got.double() == float(torch.tensor(128.0 * 128 * k, dtype=F32))).all())


def test_int8_weights_past_32_bits(gpu):
    g = rng(11)
    w = torch.empty(1100, 2048, 1024, dtype=torch.int8, device="cuda")  # 2.3e9 bytes
    w[-1] = torch.randint(-128, 128, (2048, 1024), generator=g, device="cuda").to(torch.int8)
    q = torch.randint(-128, 128, (5, 1024), generator=g, device="cuda").to(torch.int8)
    offsets = torch.zeros(1101, dtype=torch.int32, device="cuda")
    offsets[-1] = 5
    ws = torch.ones(1100, 2048, device="cuda")
    got = ej.int8_matmul(q, torch.ones(5, device="cuda"), w, ws, offsets, out_dtype=F32)
    assert torch.equal(got.double(), q.double() @ w[-1].double().T)


# ---- binding -----------------------------------------------------------------------

def test_lengths_of_zero(gpu):
    x, offsets = torch.ones(4, 0, device="cuda"), torch.tensor([0, 1, 4], device="cuda")
    y = ej.grouped_matmul(x, torch.ones(2, 0, 5, device="cuda"), offsets)
    assert y.shape == (4, 5) and bool((y == 0).all())
    gx, gw = ej.grouped_matmul_vjp(x, torch.ones(2, 0, 5, device="cuda"), offsets, y)
    assert gx.shape == (4, 0) and gw.shape == (2, 0, 5)
    x = torch.ones(4, 6, device="cuda")
    assert ej.grouped_matmul(x, torch.ones(2, 6, 0, device="cuda"), offsets).shape == (4, 0)
    gx, gw = ej.grouped_matmul_vjp(x, torch.ones(2, 6, 0, device="cuda"), offsets,
                                   torch.ones(4, 0, device="cuda"))
    assert bool((gx == 0).all()) and gw.shape == (2, 6, 0)
    none = ej.route_experts(torch.ones(0, 5, device="cuda"), 2)
    w = torch.ones(5, 6, 7, device="cuda")
    y = ej.grouped_matmul(torch.ones(0, 6, device="cuda"), w, none, gather=True)
    assert y.shape == (0, 7)
    gx, gw = ej.grouped_matmul_vjp(torch.ones(0, 6, device="cuda"), w, none, y, gather=True)
    assert gx.shape == (0, 6) and bool((gw == 0).all()) and gw.shape == w.shape
    assert ej.combine_experts(y, none).shape == (0, 7)
    q, s = ej.quantize_rows(torch.ones(3, 0, device="cuda"))
    assert q.shape == (3, 0) and s.tolist() == [0, 0, 0]
    assert bool((ej.int8_matmul(q, s, torch.ones(4, 0, device="cuda").to(torch.int8),
                                torch.ones(4, device="cuda")) == 0).all())


def test_gradients_are_first_order(gpu):
    x = torch.randn(6, 8, device="cuda", requires_grad=True)
    w = torch.randn(2, 8, 8, device="cuda", requires_grad=True)
    logits = torch.randn(6, 4, device="cuda", requires_grad=True)
    offsets = torch.tensor([0, 2, 6], device="cuda")
    r = ej.route_experts(logits, 1, renormalize=False)
    for out, leaf in ((ej.grouped_matmul(x, w, offsets), x), (ej.grouped_matmul(x, w, offsets), w),
                      (r.weights, logits), (ej.combine_experts(x, r), x)):
        plain = torch.autograd.grad(out.sum(), leaf, retain_graph=True)[0]
        (g,) = torch.autograd.grad(out.sum(), leaf, create_graph=True)
        assert torch.equal(g, plain)
        with pytest.raises(RuntimeError, match="first order"):
            g.sum().backward()


def test_gradients_of_one_side_and_accumulation(gpu):
    g = rng(12)
    offsets = torch.tensor([0, 10, 30], device="cuda")
    x, w = randn(g, 30, 24), randn(g, 2, 24, 16)
    both = ej.grouped_matmul_vjp(x, w, offsets, torch.ones(30, 16, device="cuda"))
    for side in (0, 1):
        leaf = (x, w)[side].clone().requires_grad_()
        args = [x, w]
        args[side] = leaf
        for _ in range(2):
            ej.grouped_matmul(*args, offsets).sum().backward()  # an expanded cotangent
        assert torch.equal(leaf.grad, 2 * both[side])
    assert ej.grouped_matmul_vjp(x, w, offsets, both[0][:, :16], need_x=False)[0] is None
    with torch.no_grad():
        assert not ej.grouped_matmul(x, leaf, offsets).requires_grad


def test_refusals_of_gpu_tensors(gpu):
    f = torch.zeros(4, 8, device="cuda")
    w = torch.zeros(2, 8, 8, device="cuda")
    offsets = torch.tensor([0, 2, 4], device="cuda")
    r = ej.group_by_expert(torch.zeros(4, 1, dtype=torch.long, device="cuda"), 2)
    value = [lambda: ej.route_experts(f[0], 1), lambda: ej.route_experts(f, 0),
             lambda: ej.route_experts(f, 9), lambda: ej.grouped_matmul(f, w[0], offsets),
             lambda: ej.grouped_matmul(f[:, :7], w, offsets),
             lambda: ej.grouped_matmul(f, w, offsets[:2]),
             lambda: ej.grouped_matmul(f, w, offsets, gather=True),
             lambda: ej.grouped_matmul(f[:3], w, r, gather=True),
             lambda: ej.grouped_matmul(f, w[:1], r),
             lambda: ej.grouped_matmul_vjp(f, w, offsets, f[:3]),
             lambda: ej.combine_experts(f[:3], r),
             lambda: ej.combine_experts(f, r, torch.zeros(4, 2, device="cuda")),
             lambda: ej.combine_experts(f, r, torch.zeros(4, 1, device="cuda").double()),
             lambda: ej.combine_experts_vjp(f, r, f[:, :4]),
             lambda: ej.group_by_expert(offsets, 2),
             lambda: ej.group_by_expert(offsets[None], 2, f),
             lambda: ej.quantize_rows(f[0, 0])]
    kind = [lambda: ej.route_experts(f.int(), 1), lambda: ej.grouped_matmul(f.double(), w, offsets),
            lambda: ej.grouped_matmul(f, w.bfloat16(), offsets),
            lambda: ej.grouped_matmul(f, w, offsets.float()),
            lambda: ej.grouped_matmul(f, w, offsets, out_dtype=torch.float16),
            lambda: ej.grouped_matmul(f, w, offsets.cpu()),
            lambda: ej.combine_experts(f.int(), r), lambda: ej.quantize_rows(f.int()),
            lambda: ej.int8_matmul(f, f[:, 0], f, f[:, 0])]
    for call in value:
        with pytest.raises(ValueError):
            call()
    for call in kind:
        with pytest.raises(TypeError):
            call()
    with pytest.raises(NotImplementedError):
        ej.route_experts(torch.zeros(2, 2000, device="cuda"), 2)
    with pytest.raises(NotImplementedError):
        ej.route_experts(torch.zeros(2, 100, device="cuda"), 17)


def test_a_refused_gradient_raises(gpu):
    """Refusals of a backward, which runs on autograd's thread without Python's lock."""
    e = 1 << 24
    x = torch.zeros(0, 1, device="cuda")
    w = torch.zeros(e, 1, 1, device="cuda", requires_grad=True)
    offsets = torch.zeros(e + 1, dtype=torch.int32, device="cuda")
    y = ej.grouped_matmul(x, w, offsets)
    with pytest.raises(NotImplementedError, match="too many"):
        y.sum().backward()
    with pytest.raises(NotImplementedError, match="too many"):
        ej.grouped_matmul_vjp(x, w.detach(), offsets, y.detach(), need_x=False)


@pytest.mark.parametrize("k", [0, 17])
def test_gathered_products_refuse_a_gradient_they_do_not_have(gpu, k):
    """More picks than the sum back to the tokens takes: said before the product."""
    g = rng(17)
    x, w = randn(g, 3, 8), randn(g, 2, 8, 5)
    slots = torch.arange(3 * k, dtype=torch.int32, device="cuda").reshape(3, k)
    r = ej.ExpertRouting(torch.ones(3, k, device="cuda"), torch.zeros_like(slots),
                         torch.tensor([0, 3 * k, 3 * k], dtype=torch.int32, device="cuda"),
                         (torch.arange(3 * k, device="cuda") // max(k, 1)).int(), slots)
    y = ej.grouped_matmul(x, w, r, gather=True)
    want, mag = product64(x, r.rows, r.offsets, w, 3 * k)
    assert_within(y, want, sum_bound(want, mag, 8, F32))
    with pytest.raises(NotImplementedError, match="slots of a token"):
        ej.grouped_matmul(x.clone().requires_grad_(), w, r, gather=True)
    with pytest.raises(NotImplementedError, match="slots of a token"):
        ej.grouped_matmul_vjp(x, w, r, y, gather=True)
    leaf = w.clone().requires_grad_()
    (gw,) = torch.autograd.grad(ej.grouped_matmul(x, leaf, r, gather=True), leaf, y)
    xi = x[r.rows.long()].double()
    assert_within(gw[0], xi.T @ y.double(),
                  sum_bound(xi.T @ y.double(), xi.abs().T @ y.double().abs(), 3 * k, F32))


@pytest.mark.parametrize("n", [1, 8])
def test_combine_of_more_tokens_than_a_launch_holds(gpu, n):
    """2^24 workgroups and more, of which a launch holds fewer."""
    g, t = rng(n), (1 << 24) + 777
    slots = torch.arange(t, device="cuda").flip(0).int()[:, None]
    slots[-3:] = -1
    offsets = torch.tensor([0, t], dtype=torch.int32, device="cuda")
    weights = randn(g, t, 1)
    y, cot = randn(g, t, n, dtype=BF16), randn(g, t, n, dtype=BF16)
    r = ej.ExpertRouting(weights, torch.zeros_like(slots), offsets, slots.flatten(), slots)
    at = y.flip(0)
    at[-3:] = 0
    # one product and one rounding: the same in torch
    assert torch.equal(ej.combine_experts(y, r), (weights * at.float()).to(BF16))
    gy, gw = ej.combine_experts_vjp(y, r, cot)
    want = (weights * cot.float()).to(BF16).flip(0)
    assert torch.equal(gy[3:], want[3:])
    ww = (at.double() * cot.double()).sum(1, keepdim=True)
    mag = (at.double() * cot.double()).abs().sum(1, keepdim=True)
    assert_within(gw, ww, 2 * (n + 2) * 2.0 ** -24 * mag + 1e-37)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,k,n", [(40, 3, 1), (40, 3, 2), (40, 3, 77), (900, 4, 1024),
                                   (901, 3, 2047), (300_000, 4, 2), (300_001, 4, 3)])
def test_combine_gradient_of_pairs_taken_out(gpu, t, k, n, dtype):
    """Pairs whose slot a caller set to -1, as beyond an expert's capacity: their
    rows of y get a gradient of zero, whatever the memory held before."""
    g = rng(t + n)
    r = ej.group_by_expert(make_picks(t, k, 6, 3, "holes"), 6,
                           torch.rand(t, k, generator=g, device="cuda"))
    r.slots[torch.rand(t, k, generator=g, device="cuda") < 0.2] = -1
    y, cot = randn(g, t * k, n, dtype=dtype), randn(g, t, n, dtype=dtype)
    held = r.slots >= 0
    at = y[r.slots.clamp(min=0).long()].double() * held[..., None]
    want = torch.zeros(t * k, n, dtype=torch.double, device="cuda")
    want[r.slots[held].long()] = (r.weights.double()[..., None] * cot.double()[:, None])[held]
    ww = (at * cot.double()[:, None]).sum(2)
    for before in (float("nan"), 0, -1):
        fill = torch.full((t * k, n), before, dtype=dtype, device="cuda")
        del fill  # the allocator hands out the same block again
        gy, gw = ej.combine_experts_vjp(y, r, cot)
        assert_within(gy, want, (UNIT[dtype] + 2.0 ** -23) * want.abs() + TINY[dtype])
        assert bool((gy[~torch.isin(torch.arange(t * k, device="cuda"), r.slots)] == 0).all())
        assert_within(gw, ww, 2 * (n + 2) * 2.0 ** -24 * (at * cot.double()[:, None]).abs().sum(2)
                      + 1e-37)
        del gy


def test_combine_gradient_below_the_first_offset(gpu):
    """Slots of no pair in front of the groups, and offsets short of the last pair."""
    g = rng(3)
    slots = torch.tensor([[7, 3], [4, -1], [6, 9]], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([3, 5, 8], dtype=torch.int32, device="cuda")
    w = torch.rand(3, 2, generator=g, device="cuda")
    r = ej.ExpertRouting(w, torch.zeros_like(slots), offsets, torch.zeros_like(slots).flatten(),
                         slots)
    y = randn(g, 6, 40)
    with pytest.raises(ValueError):
        ej.combine_experts_vjp(randn(g, 10, 40), r, randn(g, 3, 40))
    r.slots = torch.where(slots >= 4, slots - 4, -1)  # 3, -1; 0, -1; 2, 5
    cot = randn(g, 3, 40)
    gy, gw = ej.combine_experts_vjp(y, r, cot)
    want = torch.zeros(6, 40, device="cuda")
    for i, j in ((0, 0), (1, 0), (2, 0), (2, 1)):
        want[int(r.slots[i, j])] = w[i, j] * cot[i]
    assert torch.equal(gy, want)
    assert bool((gw[r.slots < 0] == 0).all())


def test_forward_mode_is_refused(gpu):
    """No operator drops the tangent of a dual tensor, with or without reverse mode."""
    import torch.autograd.forward_ad as forward

    g = rng(31)
    offsets = torch.tensor([0, 2, 6], device="cuda")
    r = ej.route_experts(randn(g, 6, 4), 1)
    q, s = ej.quantize_rows(randn(g, 6, 8))
    p, ps = ej.quantize_rows(randn(g, 4, 8))
    x, w, cot = randn(g, 6, 8), randn(g, 2, 8, 4), randn(g, 6, 4)
    calls = {
        "logits": (randn(g, 6, 4), lambda d: ej.route_experts(d, 2)),
        "x": (x, lambda d: ej.grouped_matmul(d, w, offsets)),
        "w": (w, lambda d: ej.grouped_matmul(x, d, offsets)),
        "w transposed": (w, lambda d: ej.grouped_matmul(cot, d.transpose(1, 2), offsets)),
        "y": (x, lambda d: ej.combine_experts(d, r)),
        "weights": (r.weights, lambda d: ej.combine_experts(x, r, d)),
        "rows": (x, lambda d: ej.quantize_rows(d)),
        "row scales": (s, lambda d: ej.int8_matmul(q, d, p, ps)),
        "column scales": (ps, lambda d: ej.int8_matmul(q, s, p, d)),
        "cotangent of weights": (r.weights, lambda d: ej.route_experts_vjp(cot, r.experts, d)),
        "cotangent of product": (cot, lambda d: ej.grouped_matmul_vjp(x, w, offsets, d)),
        "cotangent of sum": (x, lambda d: ej.combine_experts_vjp(x, r, d)),
    }
    for leaf in (False, True):
        for primal, call in calls.values():
            with forward.dual_level():
                primal = primal.detach().clone().requires_grad_(leaf)
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(forward.make_dual(primal, torch.ones_like(primal)))
    # a backward on a dual cotangent
    leaf = x.clone().requires_grad_()
    y = ej.grouped_matmul(leaf, w, offsets)
    with forward.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
        torch.autograd.grad(y, leaf, forward.make_dual(cot, cot))


@pytest.mark.parametrize("out_dtype", [None, F32])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("t,e,k,n_in,n_out", [(40, 6, 3, 72, 200), (33, 5, 2, 77, 131),
                                              (300, 9, 4, 520, 392), (1500, 4, 4, 256, 128)])
def test_gathered_gradients_are_rounded_once(gpu, t, e, k, n_in, n_out, dtype, out_dtype):
    """A token's slots are added in fp32 and their sum is rounded once; a float32
    cotangent is rounded to the operands' dtype, element by element, before."""
    g, r, x, w = product_case(t, e, k, n_in, n_out, "holes", dtype, "kn", True)
    x.requires_grad_()
    w.requires_grad_()
    y = ej.grouped_matmul(x, w, r, gather=True, out_dtype=out_dtype)
    assert y.dtype == (out_dtype or dtype)
    cot = randn(g, t * k, n_out, dtype=y.dtype)
    gx, gw = torch.autograd.grad(y, (x, w), cot)
    assert gx.dtype == dtype and gw.dtype == dtype
    off = UNIT[dtype] if out_dtype == F32 else 0.0   # of the cotangent, and below its normals:
    low = TINY[dtype] if out_dtype == F32 else 0.0
    x, w = x.detach().double(), w.detach().double()
    _, ends = row_groups(r.offsets, t * k)
    total, room, size = (torch.zeros(t, n_in, dtype=torch.double, device="cuda") for _ in range(3))
    for i in range(e):
        a, b = ends[i], ends[i + 1]
        at, gi = r.rows[a:b].long(), cot[a:b].double()
        s, mag = gi @ w[i].T, gi.abs() @ w[i].abs().T
        slack = (off + 2 * (n_out + 2) * 2.0 ** -24) * mag + low * w[i].abs().sum(1)
        total.index_add_(0, at, s)
        room.index_add_(0, at, slack)
        size.index_add_(0, at, s.abs() + slack)
        wg, mg = x[at].T @ gi, x[at].abs().T @ gi.abs()
        assert_within(gw[i], wg, sum_bound(wg, mg, b - a, dtype) + off * mg * (1 + UNIT[dtype])
                      + low * x[at].abs().sum(0)[:, None])
    room = room + 2 * (k + 2) * 2.0 ** -24 * size
    assert_within(gx, total, room + UNIT[dtype] * (total.abs() + room) + TINY[dtype])


def test_cotangents_beyond_float16(gpu):
    """The float32 cotangent of a float16 product is a float16 one to its gradients."""
    x, w = (torch.ones(2, 8, dtype=F16, device="cuda") for _ in range(2))
    w, offsets = w[None, :, :].transpose(1, 2).contiguous(), torch.tensor([0, 2], device="cuda")
    cot = torch.tensor([[65504.0, -65504.0], [65520.0, 1.0]], device="cuda")
    gx, gw = ej.grouped_matmul_vjp(x, w, offsets, cot)
    assert bool((gx[0] == 0).all()) and bool((gx[1] == float("inf")).all())
    assert bool((gw[0, :, 0] == float("inf")).all()) and bool((gw[0, :, 1] == -65504).all())


def test_8_bit_results_are_constants(gpu):
    x = torch.randn(4, 8, device="cuda", requires_grad=True)
    q, s = ej.quantize_rows(x)
    assert not q.requires_grad and not s.requires_grad
    scale = s.clone().requires_grad_()
    assert not ej.int8_matmul(q, scale, q, scale).requires_grad


@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("m,k,n", [(3, 64, 70), (3, 77, 70), (200, 256, 300), (200, 1000, 301),
                                   (700, 500, 900), (4096, 128, 4096)])
def test_int8_scales_far_apart(gpu, m, k, n, out_dtype):
    """Scales whose product leaves float32's range, under sums that bring it back.
    They are powers of two and the sums below 2^24, so the results are exact."""
    g = rng(m + k)
    q, w = (torch.randint(-128, 128, s, generator=g, device="cuda").to(torch.int8)
            for s in ((m, k), (n, k)))
    q[0] = 0
    qs, ws = (2.0 ** torch.randint(-140, 100, (s,), generator=g, device="cuda").double()
              for s in (m, n))
    qs[0], qs[1], ws[0], ws[1] = 2.0 ** 90, 2.0 ** -75, 2.0 ** 90, 2.0 ** -75
    qs, ws = qs.float().double(), ws.float().double()  # the power function's last bit
    want = (q.double() @ w.double().T) * qs[:, None] * ws
    got = ej.int8_matmul(q, qs.float(), w, ws.float(), out_dtype=out_dtype)
    assert torch.equal(got, want.float().to(out_dtype))


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("t,e,k", [(5, 1, 2), (300, 3, 8), (2000, 7, 16)])
def test_group_by_expert_of_fewer_experts_than_picks(gpu, t, e, k, index):
    """Some of the experts that the tokens picked, as one device of several holds them."""
    picks = make_picks(t, k, 32, t, "holes").to(index)
    r = ej.group_by_expert(picks, e)
    offsets, rows, slots = plain_grouping(picks, e)
    assert r.n_experts == e and r.offsets.tolist() == offsets
    assert r.rows.tolist() == rows and r.slots.tolist() == slots
    g = rng(e)
    x, w = randn(g, t, 24), randn(g, e, 24, 40)
    got = ej.grouped_matmul(x, w, r, gather=True)
    want, mag = product64(x, r.rows, r.offsets, w, t * k)
    assert_within(got, want, sum_bound(want, mag, 24, F32))
    with pytest.raises(ValueError):
        ej.group_by_expert(picks, 0)


# name -> (shapes of the inputs, call)
STREAM_CALLS = {
    "route": (((500, 20),), lambda l: ej.route_experts(l, 3)),
    "route small": (((9, 20),), lambda l: ej.route_experts(l, 3)),
    "route gradient": (((500, 20), (500, 3)),
                       lambda l, d: ej.route_experts_vjp(l, ej.route_experts(l, 3).experts, d)),
    "group": (((500, 20),), lambda l: ej.group_by_expert(l.argmax(1, keepdim=True), 20)),
    "product": (((300, 64), (3, 64, 96)), lambda x, w: ej.grouped_matmul(x, w, _thirds(x))),
    "product in parts": (((300, 4096), (3, 4096, 64)),
                         lambda x, w: ej.grouped_matmul(x, w, _thirds(x))),
    "product gradients": (((300, 64), (3, 64, 96), (300, 96)),
                          lambda x, w, d: ej.grouped_matmul_vjp(x, w, _thirds(x), d)),
    "product gradients in parts": (((9000, 64), (3, 64, 40), (9000, 40)),
                                   lambda x, w, d: ej.grouped_matmul_vjp(x, w, _thirds(x), d)),
    "gathered gradients": (((300, 20), (300, 64), (20, 64, 96), (600, 96)),
                           lambda l, x, w, d: ej.grouped_matmul_vjp(
                               x, w, ej.route_experts(l, 2), d, gather=True)),
    "sum": (((300, 20), (600, 70)), lambda l, y: ej.combine_experts(y, ej.route_experts(l, 2))),
    "sum gradients": (((300, 20), (600, 70), (300, 70)),
                      lambda l, y, d: ej.combine_experts_vjp(y, ej.route_experts(l, 2), d)),
    "8 bits": (((300, 128), (90, 128)),
               lambda x, w: ej.int8_matmul(*ej.quantize_rows(x), *ej.quantize_rows(w))),
    "layer": (((300, 20), (300, 64), (20, 64, 96), (300, 96)), lambda *v: _layer_gradients(*v)),
}


def _thirds(x):
    n = x.shape[0] // 3
    return torch.arange(4, device="cuda") * n


def _layer_gradients(logits, x, w, cot):
    leaves = [v.detach().requires_grad_() for v in (logits, x, w)]
    r = ej.route_experts(leaves[0], 2)
    out = ej.combine_experts(ej.grouped_matmul(leaves[1], leaves[2], r, gather=True), r)
    return [out.detach(), *torch.autograd.grad(out, leaves, cot)]


def _tensors(out):
    if isinstance(out, ej.ExpertRouting):
        return [out.weights, out.experts, out.offsets, out.rows, out.slots]
    return list(out) if isinstance(out, (tuple, list)) else [out]


@pytest.mark.parametrize("name", list(STREAM_CALLS))
def test_operators_run_on_the_current_stream(gpu, name):
    """On a side stream: the inputs are filled there behind work that takes a while,
    and the results are read there.  Work on any other stream would see zeros."""
    shapes, call = STREAM_CALLS[name]
    g = rng(len(name))
    values = [randn(g, *s) for s in shapes]
    want = [t.clone() for t in _tensors(call(*values))]
    inputs = [torch.zeros_like(v) for v in values]
    busy = randn(g, 4096, 4096)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(8):
            busy = busy @ busy * 0.01
        for i, v in zip(inputs, values):
            i.copy_(v)
        got = [t.clone() for t in _tensors(call(*inputs))]
        for i in inputs:
            i.zero_()
    torch.cuda.current_stream().wait_stream(side)
    assert len(got) == len(want)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,k,n_in,n_out,shift", [(60, 2, 2048, 72, 0), (60, 2, 2047, 72, 0),
                                                  (60, 2, 2048, 72, 1), (200, 1, 4096, 64, 0)])
def test_gathered_products_in_parts(gpu, t, k, n_in, n_out, shift, dtype):
    """Few tiles over a long contraction, summed in parts, of gathered rows."""
    g, e = rng(t + n_in), 3
    r = ej.group_by_expert(make_picks(t, k, e, 5, "holes"), e)
    x = randn(g, t * n_in + 8, dtype=dtype)[shift:shift + t * n_in].view(t, n_in)
    for order in ("kn", "nk"):
        w = randn(g, e, n_in, n_out, dtype=dtype, scale=n_in ** -0.5)
        if order == "nk":
            w = w.transpose(1, 2).contiguous().transpose(1, 2)
        got = ej.grouped_matmul(x, w, r, gather=True)
        want, mag = product64(x, r.rows, r.offsets, w, t * k)
        assert_within(got, want, sum_bound(want, mag, n_in, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,k,n_in,n_out,shift", [(3000, 2, 72, 152, 0), (3000, 2, 75, 151, 0),
                                                  (2500, 1, 128, 128, 1)])
def test_gathered_weight_gradients_in_parts(gpu, t, k, n_in, n_out, shift, dtype):
    g, e = rng(t + n_in), 3
    r = ej.group_by_expert(make_picks(t, k, e, 5, "holes"), e)
    x = randn(g, t * n_in + 8, dtype=dtype)[shift:shift + t * n_in].view(t, n_in)
    cot, w = randn(g, t * k, n_out, dtype=dtype), randn(g, e, n_in, n_out, dtype=dtype)
    ends = r.offsets.tolist()
    for wt in (w, w.transpose(1, 2).contiguous().transpose(1, 2)):
        _, gw = ej.grouped_matmul_vjp(x, wt, r, cot, gather=True, need_x=False)
        for i in range(e):
            a, b = ends[i], ends[i + 1]
            xi, gi = x[r.rows[a:b].long()].double(), cot[a:b].double()
            assert_within(gw[i], xi.T @ gi,
                          sum_bound(xi.T @ gi, xi.abs().T @ gi.abs(), b - a, dtype))


def test_int8_matmul_views(gpu):
    """Rows and weights with strides, off 16 bytes, expanded, and not in rows of k."""
    g, e = rng(40), 4
    r = ej.group_by_expert(make_picks(150, 2, e, 3, "skew"), e)
    wide = torch.randint(-128, 128, (300, 400), generator=g, device="cuda").to(torch.int8)
    base = torch.randint(-128, 128, (e, 90, 200), generator=g, device="cuda").to(torch.int8)
    scales = torch.rand(300, 2, generator=g, device="cuda")
    for q in (wide[:, :128], wide[:, 1:129], wide[:, 16:144], wide[:, ::2][:, :128],
              wide[:, :128].t().contiguous().t(), wide[:1, :128].expand(300, 128)):
        for w in (base[:, :, :128], base[:, 3:80, 1:129], base[:1, :, :128].expand(e, 90, 128),
                  base[:, :, ::2][:, :, :100], base.transpose(1, 2)[:, 5:133]):
            k = min(q.shape[1], w.shape[2])
            a, b = q[:, :k], w[:, :, :k]
            qs = scales[:, 0]
            ws = torch.rand(2, e, b.shape[1], generator=g, device="cuda").transpose(0, 1)[:, 0]
            got = ej.int8_matmul(a, qs, b, ws, r, out_dtype=F32)
            same = ej.int8_matmul(a.contiguous(), qs.contiguous(), b.contiguous(),
                                  ws.contiguous(), r, out_dtype=F32)
            want, _ = product64(a, None, r.offsets, b.transpose(1, 2), 300)
            owner = torch.tensor([max(o, 0) for o in row_groups(r.offsets, 300)[0]], device="cuda")
            want = want * qs.double()[:, None] * ws.double()[owner]
            assert_within(got, want, 5 * 2.0 ** -24 * want.abs() + TINY[F32])
            assert torch.equal(got, same)


@pytest.mark.parametrize("e,k", [(4, 2), (32, 4), (33, 4), (64, 8), (128, 8), (256, 3), (257, 3),
                                 (1024, 16)])
def test_route_of_every_small_batch(gpu, e, k):
    """One workgroup or all: the same picks, weights and groups on both sides of
    every number of tokens at which that changes."""
    g = rng(e)
    logits = randn(g, 260, e)
    whole = ej.route_experts(logits, k)
    for t in (1, 7, 8, 9, 12, 15, 16, 17, 31, 32, 33, 63, 64, 65, 124, 125, 127, 128, 129, 255,
              256, 257):
        r = ej.route_experts(logits[:t], k)
        assert torch.equal(r.experts, whole.experts[:t])
        assert torch.equal(r.weights, whole.weights[:t])
        offsets, rows, slots = plain_grouping(r.experts, e)
        assert r.offsets.tolist() == offsets
        assert r.rows.tolist() == rows and r.slots.tolist() == slots
        again = ej.group_by_expert(r.experts, e)
        assert all(torch.equal(getattr(again, f), getattr(r, f))
                   for f in ("offsets", "rows", "slots"))
