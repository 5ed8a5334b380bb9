"""Products at sizes that take the tiles between the smallest and the large ones,
and each operator's kernels that the sizes of its own tests leave out: a middling
number of rows a group, many groups, short rows, narrow tables.

The bounds are those of the operators' tests (``sum_bound``, ``gated64``,
``assert_product``, ``check_gradient``), which count the roundings.
"""

import pytest
import torch

import einjax_amd as ej
from test_gpu_experts import (BF16, F16, F32, TINY, UNIT, assert_within, product64, randn, rng,
                              sum_bound)
from test_gpu_fp8 import (LARGE_F8, QUANTIZED, assert_product, blocks, fp8_64, operands,
                          plain_blocks, scales)
from test_gpu_gated import gated64
from test_gpu_tokens import check_gradient, make_tokens
from test_gpu_unaligned_rows import at_offset

pytestmark = pytest.mark.gpu


def ends_of(sizes, first=0):
    """Offsets of groups that begin at slot `first`."""
    return torch.tensor([first + sum(sizes[:i]) for i in range(len(sizes) + 1)],
                        dtype=torch.int32, device="cuda")


# ---- 8-bit floats ---------------------------------------------------------------


@pytest.mark.parametrize("out_dtype", [BF16, F16])
@pytest.mark.parametrize("first", [0, 7])
@pytest.mark.parametrize("sizes,dead,k,n", LARGE_F8)
def test_fp8_large_blocks_of_rows_as_they_lie(gpu, sizes, dead, k, n, first, out_dtype):
    """The pipelined large blocks on rows that are not gathered, as a layer's
    second product takes them: slots of no group before and behind the groups,
    whose scales are NaN, and rows that lie apart."""
    g, e, live = rng(k + n + first), len(sizes), sum(sizes)
    offsets, slots = ends_of(sizes, first), first + live + dead
    q = operands(g, slots, k + 32)[:, 16:k + 16]
    qs = scales(g, slots, blocks(k)) * 1e-2
    w, ws = operands(g, n, k, (e,)), scales(g, e, blocks(n), blocks(k)) * 1e-4
    qs[:first] = qs[first + live:] = float("nan")
    got = ej.fp8_matmul(q, qs, w, ws, offsets, out_dtype=out_dtype)
    want, size = fp8_64(q, torch.nan_to_num(qs), w, ws, None, offsets, slots)
    assert_product(got, want, size, k, out_dtype)
    assert bool((got[:first] == 0).all()) and bool((got[first + live:] == 0).all())


@pytest.mark.parametrize("out_dtype", [BF16, F16])
@pytest.mark.parametrize("m,k,n", [(4096, 1024, 2048), (1000, 400, 8192), (2500, 128, 4100),
                                   (2049, 2160, 2050)])
def test_fp8_large_blocks_without_groups(gpu, m, k, n, out_dtype):
    g = rng(m + k)
    q, qs = operands(g, m, k), scales(g, m, blocks(k)) * 1e-2
    w, ws = operands(g, n, k), scales(g, blocks(n), blocks(k)) * 1e-4
    got = ej.fp8_matmul(q, qs, w, ws, out_dtype=out_dtype)
    want, size = fp8_64(q, qs, w[None], ws[None], None, None, m)
    assert_product(got, want, size, k, out_dtype)


# ---- a middling number of rows a group ------------------------------------------------

# rows of each group, slots of no group, k, n of a plain product
MIDDLE = [([70, 0, 61, 100, 3, 64, 129, 53], 4, 136, 3336), ([60] * 16, 0, 64, 2048),
          ([99, 1, 128, 172], 0, 200, 8000)]
# the same for gated ones, whose n is that of the results: 49 to 64 rows, and
# fewer with many columns of W [k][n]
MIDDLE_GATED = [([70, 0, 61, 100, 3, 64, 129, 53], 4, 136, 1640), ([16, 0, 33, 5, 20, 17, 1, 40],
                                                                   0, 72, 2728),
                ([16] * 16, 3, 264, 1024)]


def product_operands(sizes, dead, k, n, dtype, order):
    g, slots = rng(k + n), sum(sizes) + dead
    x = randn(g, slots, k, dtype=dtype)
    w = randn(g, len(sizes), k, n, dtype=dtype, scale=k ** -0.5)
    if order == "nk":
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    x[slots - dead:] = float("nan")
    return g, slots, x, w


def shuffled(sizes, dead, seed):
    """The relation of rows in a shuffled order, `dead` of them of no group."""
    g = torch.Generator().manual_seed(seed)
    picks = torch.repeat_interleave(torch.arange(len(sizes)), torch.tensor(sizes))
    picks = torch.cat([picks, torch.full((dead,), -1)])
    return ej.group_by_expert(picks[torch.randperm(len(picks), generator=g)].cuda()[:, None],
                              len(sizes))


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes,dead,k,n", MIDDLE)
def test_grouped_matmul_of_some_rows_a_group(gpu, sizes, dead, k, n, dtype, order):
    g, slots, x, w = product_operands(sizes, dead, k, n, dtype, order)
    offsets, live = ends_of(sizes), sum(sizes)
    got, wide = ej.grouped_matmul(x, w, offsets), ej.grouped_matmul(x, w, offsets, out_dtype=F32)
    x[live:] = 0
    want, mag = product64(x, None, offsets, w, slots)
    assert_within(got, want, sum_bound(want, mag, k, dtype))
    assert_within(wide, want, sum_bound(want, mag, k, F32))
    r = shuffled(sizes, dead, n)
    got = ej.grouped_matmul(x, w, r, gather=True)
    want, mag = product64(x, r.rows, r.offsets, w, slots)
    assert_within(got, want, sum_bound(want, mag, k, dtype))
    assert bool((got[live:] == 0).all())


@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("sizes,dead,k,n", MIDDLE_GATED)
def test_gated_matmul_of_some_rows_a_group(gpu, sizes, dead, k, n, dtype, order):
    g, slots, x, w = product_operands(sizes, dead, k, 2 * n, dtype, order)
    offsets, live = ends_of(sizes), sum(sizes)
    got = ej.gated_matmul(x, w, offsets)
    leaf = x.detach().requires_grad_()
    assert torch.equal(got, ej.gated_matmul(leaf, w, offsets).detach())  # keeps both projections
    x[live:] = 0
    h, eh, *_ = gated64(x, None, offsets, w, slots, "silu")
    assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])
    r = shuffled(sizes, dead, n)
    got = ej.gated_matmul(x, w, r, activation="gelu_tanh", gather=True)
    h, eh, *_ = gated64(x, r.rows, r.offsets, w, slots, "gelu_tanh")
    assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])
    assert bool((got[live:] == 0).all())


@pytest.mark.parametrize("shift", [0, 1, 3, 4])
@pytest.mark.parametrize("order", ["kn", "nk"])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("k,n", [(77, 1283), (260, 1090)])
def test_gated_matmul_of_some_unaligned_rows_a_group(gpu, k, n, dtype, order, shift):
    sizes, dead = [100, 0, 128, 64, 200, 1, 90, 217], 5
    g, slots, x, w = product_operands(sizes, dead, k, 2 * n, dtype, order)
    x = at_offset(x, shift)
    if order == "nk":
        w = at_offset(w.transpose(1, 2), (shift + 1) % 8).transpose(1, 2)
    else:
        w = at_offset(w, (shift + 1) % 8)
    offsets, live = ends_of(sizes), sum(sizes)
    got = ej.gated_matmul(x, w, offsets)
    x[live:] = 0
    h, eh, *_ = gated64(x, None, offsets, w, slots, "silu")
    assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])
    r = shuffled(sizes, dead, n)
    got = ej.gated_matmul(x, w, r, activation="gelu", gather=True)
    h, eh, *_ = gated64(x, r.rows, r.offsets, w, slots, "gelu")
    assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])
    assert bool((got[live:] == 0).all())


@pytest.mark.parametrize("out_dtype", [F32, BF16, F16])
@pytest.mark.parametrize("sizes,dead,k,n", [
    ([100] * 16, 0, 272, 1409), ([128, 90, 0, 200, 7, 64, 150, 99, 100, 33], 6, 400, 2050),
    ([300, 0, 250, 120, 7, 100], 3, 200, 1300), ([150] * 4, 0, 131, 1500)])
def test_fp8_matmul_of_some_rows_a_group(gpu, sizes, dead, k, n, out_dtype):
    g, live, e = rng(k + n), sum(sizes), len(sizes)
    slots = live + dead
    w, ws = operands(g, n, k, (e,)), scales(g, e, blocks(n), blocks(k)) * 1e-4
    q, qs = operands(g, slots, k), scales(g, slots, blocks(k)) * 1e-2
    qs[live:] = float("nan")
    got = ej.fp8_matmul(q, qs, w, ws, ends_of(sizes), out_dtype=out_dtype)
    want, size = fp8_64(q, torch.nan_to_num(qs), w, ws, None, ends_of(sizes), slots)
    assert_product(got, want, size, k, out_dtype)
    qs[live:] = 1.0
    r = shuffled(sizes, dead, n)
    got = ej.fp8_matmul(q, qs, w, ws, r, gather=True, out_dtype=out_dtype)
    want, size = fp8_64(q, qs, w, ws, r.rows, r.offsets, slots)
    assert_product(got, want, size, k, out_dtype)
    assert bool((got[live:] == 0).all())


@pytest.mark.parametrize("sizes,dead,k,n", [([70, 0, 61, 100, 3, 64, 129, 53], 4, 144, 3336),
                                            ([60] * 16, 0, 64, 2049)])
def test_int8_matmul_of_some_rows_a_group(gpu, sizes, dead, k, n):
    g, live, e = rng(k + n), sum(sizes), len(sizes)
    slots = live + dead
    q = torch.randint(-128, 128, (slots, k), generator=g, device="cuda").to(torch.int8)
    w = torch.randint(-128, 128, (e, n, k), generator=g, device="cuda").to(torch.int8)
    one, ones = torch.ones(slots, device="cuda"), torch.ones(e, n, device="cuda")
    r = shuffled(sizes, dead, n)
    for gather, groups in ((False, ends_of(sizes)), (True, r)):
        got = ej.int8_matmul(q, one, w, ones, groups, gather=gather, out_dtype=F32)
        x = q[r.rows.long()] if gather else q
        ends = ends_of(sizes).tolist()
        for i, (a, b) in enumerate(zip(ends, ends[1:])):
            # below 2^24: exact
            assert torch.equal(got[a:b].double(), x[a:b].double() @ w[i].double().T)
        assert bool((got[live:] == 0).all())


# ---- rows shorter than 16 bytes ---------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("k,n", [(3, 70), (70, 3), (2, 5), (3, 2), (7, 7), (130, 1)])
def test_products_of_short_rows(gpu, k, n, dtype):
    """k or n of less than 16 bytes in either order of W, with the gradients,
    of gathered rows and of rows as they lie."""
    sizes, dead = [40, 0, 131, 3, 66], 4
    live = sum(sizes)
    for order in ("kn", "nk"):
        g, slots, x, w = product_operands(sizes, dead, k, 2 * n, dtype, order)
        x[live:] = 0
        r = shuffled(sizes, dead, n)
        ends = r.offsets.tolist()
        grad = randn(g, slots, 2 * n, dtype=dtype)
        grad[live:] = float("nan")
        for gather in (False, True):
            rows = r.rows if gather else None
            got = ej.grouped_matmul(x, w, r, gather=gather)
            want, mag = product64(x, rows, r.offsets, w, slots)
            assert_within(got, want, sum_bound(want, mag, k, dtype))
            got = ej.gated_matmul(x, w, r, gather=gather)
            h, eh, *_ = gated64(x, rows, r.offsets, w, slots, "silu")
            assert_within(got, h, eh + UNIT[dtype] * (h.abs() + eh) + TINY[dtype])
            gx, gw = ej.grouped_matmul_vjp(x, w, r, grad, gather=gather)
            slot_x = torch.zeros(slots, k, dtype=torch.double, device="cuda")
            slot_mag = torch.zeros_like(slot_x)
            for i, (a, b) in enumerate(zip(ends, ends[1:])):
                xe = (x[r.rows[a:b].long()] if gather else x[a:b]).double()
                ge, we = grad[a:b].double(), w[i].double()
                assert_within(gw[i], xe.T @ ge,
                              sum_bound(xe.T @ ge, xe.abs().T @ ge.abs(), b - a, dtype))
                slot_x[a:b], slot_mag[a:b] = ge @ we.T, ge.abs() @ we.abs().T
            if gather:  # one slot a row
                want, mag = torch.zeros_like(slot_x), torch.zeros_like(slot_x)
                at = r.rows[:live].long()
                want[at], mag[at] = slot_x[:live], slot_mag[:live]
            else:
                want, mag = slot_x, slot_mag
            assert_within(gx, want, sum_bound(want, mag, 2 * n, dtype))


# rows of a table shorter than 16 bytes whose sums span chunks of the tokens
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,v,n,kind", [(3000, 3, 1, "zipf"), (3000, 5, 3, "padded"),
                                        (20000, 4, 2, "one"), (40000, 6000, 3, "zipf"),
                                        (16384, 300, 3, "runs")])
def test_table_gradients_of_narrow_rows(gpu, t, v, n, kind, dtype, index):
    g = rng(t + n)
    tokens, cot = make_tokens(t, v, kind, 1, index), randn(g, t, n, dtype=dtype)
    table = randn(g, v, n, dtype=dtype)
    got = ej.embed_tokens_vjp(tokens, table, cot, scale=1.5)
    check_gradient(got, tokens, v, cot, 1.5, dtype)


# ---- quantization of matrices ----------------------------------------------------------------


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("m,n", QUANTIZED)
def test_blocks_of_128_rows_reach_the_largest_value(gpu, m, n, dtype):
    """Every finite 128 x 128 block that is not zero has a value of 448: its
    largest over the scale is 448 within three roundings.  (Some of float16's
    pass its range: their blocks have scale NaN and values of 0.)"""
    g = rng(m * n)
    x = (randn(g, m, n) * torch.exp(3 * randn(g, m, 1))).to(dtype)
    x[m // 2:, : n // 2] = 0
    q, scale = ej.quantize_blocks(x, block_rows=128)
    padded = torch.nn.functional.pad(q.float().abs(), (0, -n % 128, 0, -m % 128))
    most = padded.reshape(padded.shape[0] // 128, 128, blocks(n), 128).amax((1, 3))
    plain = torch.nn.functional.pad(x.float().abs(), (0, -n % 128, 0, -m % 128))
    top = plain.reshape(most.shape[0], 128, blocks(n), 128).amax((1, 3))
    live = (top > 0) & torch.isfinite(top)
    assert torch.equal(scale > 0, live) and torch.equal(torch.isnan(scale), torch.isinf(top))
    assert torch.equal(most, torch.where(live, 448.0, 0.0))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("rows", [1, 128])
def test_quantize_blocks_of_matrices_that_lie_apart(gpu, rows, dtype):
    g = rng(12)
    wide = (randn(g, 5, 140, 400) * torch.exp(3 * randn(g, 5, 140, 1))).to(dtype)
    for x in (wide[:, :130], wide[:, 3:, 1:301], wide[::2, ::2, :7], wide[:, :1, 5:],
              wide[:1].expand(4, 140, 400)):
        q, scale = ej.quantize_blocks(x, block_rows=rows)
        want, by = plain_blocks(x, rows)
        assert torch.equal(scale, by) and torch.equal(q.float(), want)
