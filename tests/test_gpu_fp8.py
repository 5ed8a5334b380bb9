"""8-bit floating-point blocks and their products against their definition in
64 bits.

A product: each block's sum of at most 128 products of e4m3 values and the
addition of the blocks' shares are formed in fp32, off by 2 (k + 2) 2^-24 of the
sum of the magnitudes; the product of the two scales and its product with the
sum round twice more.  The result is rounded once.  Where it is rounded to 16
bits, the 8-bit matrix instructions form the sums: of 8 consecutive k they drop
what lies below 2^-13 of the largest product, in the 7 others.
"""

import pytest
import torch

import einjax_amd as ej
from test_gpu_experts import (BF16, F16, F32, PRODUCTS, TINY, UNIT, assert_within, make_picks,
                              randn, rng, row_groups)

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


def blocks(n):
    return (n + 127) // 128


def spread(scale, rows, m, n):
    """Scales [..., row blocks, column blocks] as the values' [..., m, n]."""
    return scale.repeat_interleave(rows, -2)[..., :m, :].repeat_interleave(128, -1)[..., :n]


def same(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


def plain_blocks(x, rows):
    """(q in float32, scale) of x [..., m, n]: the largest magnitude times
    fp32's 1 / 448, x / scale in fp32, rounded by the type's conversion; NaN and
    q = 0 where the largest is not finite."""
    m, n = x.shape[-2:]
    x = x.float()
    padded = torch.nn.functional.pad(x, (0, -n % 128, 0, -m % rows))
    tiles = padded.reshape(*x.shape[:-2], padded.shape[-2] // rows, rows, blocks(n), 128)
    most = tiles.abs().amax((-3, -1))
    scale = torch.where(torch.isfinite(most), most * (1.0 / 448.0), float("nan"))
    by = spread(scale, rows, m, n)
    q = torch.where(by > 0, x / by, torch.zeros_like(x)).clamp(-448, 448)
    return q.to(E4M3).float(), scale


QUANTIZED = [(1, 1), (1, 128), (1, 4096), (3, 7), (5, 129), (16, 127), (130, 256), (128, 128),
             (257, 1000), (1000, 384), (2049, 2048), (4, 131), (300, 8), (77, 2051)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n", QUANTIZED)
def test_quantize_blocks(gpu, m, n, dtype):
    g = rng(m * n)
    x = randn(g, m, n) * torch.exp(3 * randn(g, m, 1))
    x = x.to(dtype)
    if m > 2:
        x[1] = 0
        x[2, : n // 2] = 0
    for rows in (1, 128):
        q, scale = ej.quantize_blocks(x, block_rows=rows)
        want, by = plain_blocks(x, rows)
        assert q.dtype == E4M3 and q.shape == x.shape
        assert same(scale, by)
        assert torch.equal(q.float(), want)
        for b in range(blocks(n)):  # every block reaches the largest value
            part = q.float()[:, b * 128:(b + 1) * 128].abs()
            most = part.amax(1) if rows == 1 else part.amax()[None]
            live = (by[:, b] > 0) if rows == 1 else (by[:, b].amax() > 0)[None]
            if rows == 1:
                assert bool((most[live] == 448).all())
        # off by half a step: 2^-4 of the value, 2^-10 of the scale for the smallest
        err = (q.double() * spread(scale, rows, m, n).double() - x.double()).abs()
        step = torch.maximum(x.double().abs() * 2.0 ** -4, spread(scale, rows, m, n) * 2.0 ** -10)
        near = err <= step * (1 + 2.0 ** -18)
        assert bool((near | torch.isnan(spread(scale, rows, m, n))).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_quantize_blocks_of_every_value(gpu, dtype):
    """Every 16-bit value (or a spread of fp32's) against a block's largest of a
    power of two, where the quotients fall on the ties between e4m3 values, and
    of others."""
    if dtype == F32:
        v = randn(rng(1), 1 << 16) * torch.exp(8 * randn(rng(2), 1 << 16))
    else:
        v = torch.arange(1 << 16, dtype=torch.int32, device="cuda").to(torch.int16).view(dtype)
        v = v[torch.isfinite(v)]
    for most in (448.0, 1.75, 1.0, 1.171875, 1e-3, 240.0):
        top = torch.tensor(most, device="cuda").to(dtype)
        x = v[v.abs() <= top]
        x = x[: len(x) // 127 * 127].reshape(-1, 127)
        x = torch.cat([x, top.expand(len(x), 1)], 1)
        q, scale = ej.quantize_blocks(x)
        want, by = plain_blocks(x, 1)
        assert torch.equal(scale, by) and torch.equal(q.float(), want)


@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_blocks_not_finite_and_tiny(gpu, rows):
    x = randn(rng(3), 300, 400)
    x[5, 130] = float("nan")
    x[200, 399] = float("inf")
    x[201, 0] = -float("inf")
    q, scale = ej.quantize_blocks(x, block_rows=rows)
    clean = x.clone()
    clean[5, 130] = clean[200, 399] = clean[201, 0] = 0
    want, by = plain_blocks(clean, rows)
    bad = torch.zeros_like(by, dtype=torch.bool)
    for r, c in ((5, 1), (200, 3), (201, 0)):
        bad[r // rows, c] = True
    assert torch.equal(torch.isnan(scale), bad)
    assert torch.equal(scale[~bad], by[~bad])
    good = ~spread(bad.float(), rows, 300, 400).bool()
    assert torch.equal(q.float()[good], want[good])
    w, ws = ej.quantize_blocks(randn(rng(4), 64, 400), block_rows=128)
    y = ej.fp8_matmul(*ej.quantize_blocks(x), w, ws)
    lost = torch.zeros(300, dtype=torch.bool, device="cuda")
    lost[[5, 200, 201]] = True
    assert torch.equal(torch.isnan(y).all(1), lost) and torch.equal(torch.isnan(y).any(1), lost)
    for tiny in (1e-38, 1e-42, 1.4e-45, 3e38):
        x = randn(rng(5), 130, 256).clamp(-4, 4) / 4 * tiny
        q, scale = ej.quantize_blocks(x, block_rows=rows)
        want, by = plain_blocks(x, rows)
        assert torch.equal(scale, by) and torch.equal(q.float(), want)


def test_quantize_blocks_views(gpu):
    g = rng(6)
    wide = randn(g, 4, 150, 400, dtype=BF16)
    for x in (wide[:, :, :300], wide[:, 3:, 1:301], wide[::2, ::2], wide.transpose(1, 2),
              wide.transpose(0, 1), wide[0], wide[1, :, 7:], wide[0, 0], wide[:, :1],
              wide[:1].expand(3, 150, 400), wide[None], wide[:, :, :0], wide[:0]):
        for rows in (1, 128):
            if x.dim() < 2 and rows == 128:
                continue
            q, scale = ej.quantize_blocks(x, block_rows=rows)
            p, same = ej.quantize_blocks(x.contiguous(), block_rows=rows)
            assert q.shape == x.shape
            assert torch.equal(scale, same) and torch.equal(q.float(), p.float())
            if x.numel() and x.dim() > 1:
                want, by = plain_blocks(x, rows)
                assert torch.equal(scale, by) and torch.equal(q.float(), want)


def operands(g, m, k, lead=()):
    """e4m3 values over their whole range, the subnormal ones among them, and
    scales over six decades."""
    q = (randn(g, *lead, m, k) * torch.exp2(torch.randint(-9, 8, (*lead, m, k), generator=g,
                                                          device="cuda").float())).clamp(-448, 448)
    return q.to(E4M3)


def scales(g, *shape):
    return torch.exp(3 * randn(g, *shape)) * torch.where(
        torch.rand(*shape, generator=g, device="cuda") < 0.05, 0.0, 1.0)


def fp8_64(q, qs, w, ws, rows, offsets, slots):
    """The product, the sum of its magnitudes and that of the largest of every 8,
    in 64 bits."""
    n, k = w.shape[-2:]
    x = q.double() * spread(qs, 1, len(q), k).double()
    out = torch.zeros(slots, n, dtype=torch.double, device="cuda")
    mag, eights = torch.zeros_like(out), torch.zeros_like(out)
    ends = [0, slots] if offsets is None else offsets.tolist()
    for e in range(len(w)):
        a, b = ends[e], ends[e + 1]
        xe = x[rows[a:b].long()] if rows is not None else x[a:b]
        we = w[e].double() * spread(ws[e], 128, n, k).double()
        out[a:b], mag[a:b] = xe @ we.T, xe.abs() @ we.abs().T
        eights[a:b] = largest_of_8(xe) @ largest_of_8(we).T
    return out, (mag, eights)


def largest_of_8(v):
    m, k = v.shape
    v = torch.nn.functional.pad(v.abs(), (0, -k % 8))
    return v.reshape(m, v.shape[1] // 8, 8).amax(2)


def assert_product(got, want, sizes, k, dtype):
    """Within the bound, or infinite where the sum passes the type's range."""
    bound = fp8_bound(want, sizes, k, dtype)
    past = torch.isinf(got) & (got.sign() == want.sign()) & \
        (want.abs() + bound >= torch.finfo(dtype).max * (1 + UNIT[dtype] / 2))
    assert_within(torch.where(past, 0.0, got.double()), torch.where(past, 0.0, want), bound)


def fp8_bound(want, sizes, k, dtype):
    mag, eights = sizes
    err = 2 * (k + 4) * 2.0 ** -24 * mag + 1e-37
    if dtype != F32:
        err = err + 7 * 2.0 ** -13 * eights
    return err + UNIT[dtype] * (want.abs() + err) + TINY[dtype]


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,e,k,n_in,n_out,kind", PRODUCTS)
def test_fp8_matmul(gpu, t, e, k, n_in, n_out, kind, out_dtype):
    g = rng(t + n_out)
    r = ej.group_by_expert(make_picks(t, k, e, 3, kind), e)
    w, ws = operands(g, n_out, n_in, (e,)), scales(g, e, blocks(n_out), blocks(n_in)) * 1e-4
    for gather in (False, True):
        m = t if gather else t * k
        q, qs = operands(g, m, n_in), scales(g, m, blocks(n_in)) * 1e-2
        got = ej.fp8_matmul(q, qs, w, ws, r, gather=gather, out_dtype=out_dtype)
        assert got.dtype == out_dtype and got.shape == (t * k, n_out)
        want, mag = fp8_64(q, qs, w, ws, r.rows if gather else None, r.offsets, t * k)
        assert_product(got, want, mag, n_in, out_dtype)
        assert bool((got[int(r.offsets[-1]):] == 0).all())


# rows of each group, slots of no group behind them, k, n
LARGE_F8 = [([1000], 24, 128, 4096), ([1024, 0, 512], 0, 256, 4104), ([300, 0, 724], 3, 640, 6144),
            ([900, 1100, 1000, 1096], 5, 400, 4096), ([129, 128, 1, 1790], 3, 192, 4112),
            ([4096], 0, 1024, 2048), ([700, 3000, 60, 5], 7, 528, 2304)]


@pytest.mark.parametrize("sizes,dead,k,n", LARGE_F8)
def test_fp8_matmul_large_blocks(gpu, sizes, dead, k, n):
    g, e, live = rng(k + n), len(sizes), sum(sizes)
    offsets = torch.tensor([sum(sizes[:i]) for i in range(e + 1)], dtype=torch.int32,
                           device="cuda")
    slots = live + dead
    q, qs = operands(g, slots, k), scales(g, slots, blocks(k)) * 1e-2
    w, ws = operands(g, n, k, (e,)), scales(g, e, blocks(n), blocks(k)) * 1e-4
    qs[live:] = float("nan")
    got = ej.fp8_matmul(q, qs, w, ws, offsets, out_dtype=F32)
    want, mag = fp8_64(q, torch.nan_to_num(qs), w, ws, None, offsets, slots)
    assert_product(got, want, mag, k, F32)
    assert bool((got[live:] == 0).all())
    r = ej.group_by_expert(torch.repeat_interleave(torch.arange(e), torch.tensor(sizes))
                           [torch.randperm(live, generator=torch.Generator().manual_seed(n))]
                           .cuda()[:, None], e)
    got = ej.fp8_matmul(q[:live], qs[:live], w, ws, r, gather=True, out_dtype=BF16)
    want, mag = fp8_64(q[:live], qs[:live], w, ws, r.rows, r.offsets, live)
    assert_product(got, want, mag, k, BF16)


@pytest.mark.parametrize("m,n_in,n_out", [(0, 64, 32), (1, 4096, 256), (4, 100, 33), (3, 0, 9),
                                          (200, 256, 300), (17, 129, 129), (64, 8192, 40),
                                          (2, 128, 0), (2000, 1000, 1283)])
def test_fp8_matmul_dense(gpu, m, n_in, n_out):
    g = rng(m + 1)
    x, weight = randn(g, m, n_in), randn(g, n_out, n_in)
    q, qs = ej.quantize_blocks(x)
    w, ws = ej.quantize_blocks(weight, block_rows=128)
    want, mag = fp8_64(q, qs, w[None], ws[None], None, None, m)
    for pw, ps in ((w, ws), (w[None], ws[None])):
        got = ej.fp8_matmul(q, qs, pw, ps, out_dtype=F32)
        assert_product(got, want, mag, n_in, F32)
    # the 8 bits' own distance: 2^-4 of each factor, one more part for what
    # falls below the blocks' smallest step
    full = x.double() @ weight.double().T
    room = (2.0 ** -4 * (2 + 2.0 ** -4) * (x.double().abs() @ weight.double().abs().T)
            + n_in * 2.0 ** -10 / 448 * 20)
    assert bool(((want - full).abs() <= room * 1.01).all())


def test_fp8_matmul_views(gpu):
    """Row strides, starts off 16 bytes, strided scales."""
    g = rng(7)
    e, k, n = 3, 200, 90
    sizes = torch.tensor([0, 100, 100, 290], dtype=torch.int32, device="cuda")
    wide = operands(g, 300, 400)
    base = operands(g, 100, 260, (e,))
    qs = scales(g, 300, 6)
    ws = scales(g, e, 2, 4)
    for q in (wide[:, :k], wide[:, 1:k + 1], wide[:, 16:k + 16], wide.t()[:k].contiguous().t(),
              wide[:1, :k].expand(300, k)):
        for w in (base[:, :n, :k], base[:, 3:n + 3, 5:k + 5], base[:, 10:, :k],
                  base[:, :n, :k].transpose(1, 2).contiguous().transpose(1, 2)):
            for s, t in ((qs[:, :2], ws[:, :1, :2]), (qs[:, ::3], ws[:, 1:, 1::2])):
                got = ej.fp8_matmul(q, s, w, t, sizes, out_dtype=F32)
                want, mag = fp8_64(q, s, w, t, None, sizes, 300)
                assert_product(got, want, mag, k, F32)


def test_fp8_weights_past_32_bits(gpu):
    g = rng(8)
    w = torch.empty(1100, 2048, 1024, dtype=torch.uint8, device="cuda").view(E4M3)  # 2.3e9 bytes
    w[-1] = operands(g, 2048, 1024)
    ws = scales(g, 1100, 16, 8)
    q, qs = operands(g, 5, 1024), scales(g, 5, 8)
    offsets = torch.zeros(1101, dtype=torch.int32, device="cuda")
    offsets[-1] = 5
    got = ej.fp8_matmul(q, qs, w, ws, offsets, out_dtype=F32)
    want, mag = fp8_64(q, qs, w[-1:], ws[-1:], None, None, 5)
    assert_product(got, want, mag, 1024, F32)


def test_fp8_wild_offsets_stay_in_bounds(gpu):
    g = rng(9)
    q, qs = operands(g, 64, 128), scales(g, 64, 1)
    w, ws = operands(g, 64, 128, (3,)), scales(g, 3, 1, 1)
    for o in ([-5, 10, 7, 1 << 30], [0, 64, 64, 64], [64, 64, 64, 64], [9, 3, 2, 1]):
        offsets = torch.tensor(o, dtype=torch.int32, device="cuda")
        assert ej.fp8_matmul(q, qs, w, ws, offsets).shape == (64, 64)


def test_fp8_repeats_and_replays(gpu):
    """Captured once and replayed on new data between eager calls; the same bits
    every time."""
    g = rng(10)
    r = ej.group_by_expert(make_picks(300, 2, 5, 3, "skew"), 5)
    x = randn(g, 300, 520, dtype=BF16)
    w, ws = ej.quantize_blocks(randn(g, 5, 392, 520, dtype=BF16), block_rows=128)

    def call():
        return ej.fp8_matmul(*ej.quantize_blocks(x), w, ws, r, gather=True)

    first = call()
    assert all(torch.equal(first, call()) for _ in range(3))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for _ in range(4):
        x.copy_(randn(g, 300, 520, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call())


def test_fp8_results_are_constants(gpu):
    x = randn(rng(11), 4, 256).requires_grad_()
    q, scale = ej.quantize_blocks(x)
    assert not q.requires_grad and not scale.requires_grad
    w, ws = ej.quantize_blocks(x, block_rows=128)
    assert not ej.fp8_matmul(q, scale, w, ws).requires_grad
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x.detach(), x.detach())
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ej.quantize_blocks(dual)
        dual = torch.autograd.forward_ad.make_dual(scale, scale)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ej.fp8_matmul(q, dual, w, ws)


def test_fp8_refusals_of_gpu_tensors(gpu):
    f = torch.zeros(4, 256, device="cuda")
    q, s = ej.quantize_blocks(f)
    w, ws = ej.quantize_blocks(f, block_rows=128)
    many, ms = ej.quantize_blocks(f.expand(2, 4, 256), block_rows=128)
    offsets = torch.tensor([0, 2, 4], device="cuda")
    for call in (lambda: ej.quantize_blocks(f.double()), lambda: ej.quantize_blocks(f.int()),
                 lambda: ej.fp8_matmul(f, s, w, ws), lambda: ej.fp8_matmul(q, s, f, ws),
                 lambda: ej.fp8_matmul(q, s.half(), w, ws),
                 lambda: ej.fp8_matmul(q, s, w, ws.double()),
                 lambda: ej.fp8_matmul(q, s, w, ws, out_dtype=torch.float64),
                 lambda: ej.fp8_matmul(q, s, w, ws, out_dtype=E4M3),
                 lambda: ej.fp8_matmul(q.view(torch.int8), s, w, ws),
                 lambda: ej.fp8_matmul(q.cpu(), s, w, ws)):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: ej.quantize_blocks(f, block_rows=64),
                 lambda: ej.quantize_blocks(f[0], block_rows=128),
                 lambda: ej.quantize_blocks(f.sum()),
                 lambda: ej.fp8_matmul(q, s[:, :1], w, ws), lambda: ej.fp8_matmul(q, s, w, ws[0]),
                 lambda: ej.fp8_matmul(q, s[:3], w, ws), lambda: ej.fp8_matmul(q, s, many, ms),
                 lambda: ej.fp8_matmul(q, s, w, ws, gather=True),
                 lambda: ej.fp8_matmul(q, s, w[:, :128], ws[:, :1]),
                 lambda: ej.fp8_matmul(q, s, many, ms, offsets, gather=True),
                 lambda: ej.fp8_matmul(q, s, many, ms, offsets[:2]),
                 lambda: ej.fp8_matmul(q[0], s[0], w, ws)):
        with pytest.raises(ValueError):
            call()
