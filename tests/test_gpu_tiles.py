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
from test_gpu_fp8 import (LARGE_F8, assert_product, blocks, fp8_64, operands, scales)

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
