"""Rows of a table for tokens, and their gradient, against their definition in
64 bits.

A row is its value times the scale, in fp32 (whose rounding counts, as the
scale's own does), rounded once.  A gradient is a sum of c terms in fp32, off by
2 (c + 2) 2^-24 of the sum of their magnitudes, times the scale, rounded once.
"""

import pytest
import torch

import einjax_amd as ej
from test_gpu_experts import BF16, F16, F32, TINY, UNIT, assert_within, randn, rng

pytestmark = pytest.mark.gpu

# tokens, rows, n, kind of tokens
TABLES = [(0, 5, 8, "even"), (1, 1, 1, "even"), (1, 1000, 4096, "even"), (3, 7, 5, "padded"),
          (31, 10, 64, "one"), (32, 10, 64, "one"), (33, 10, 64, "one"), (64, 50, 72, "zipf"),
          (65, 1, 2051, "one"), (100, 33, 8, "runs"), (257, 5000, 264, "zipf"),
          (1000, 3, 131, "padded"), (1999, 5003, 771, "zipf"), (4096, 100, 2048, "runs"),
          (4100, 2, 4099, "padded"), (5000, 40, 16, "none"), (16384, 30000, 128, "zipf"),
          (16385, 300, 96, "zipf"), (20000, 70000, 40, "padded"), (70001, 9, 24, "padded"),
          (131072, 1000, 8, "one")]


def make_tokens(t, v, kind, seed, dtype=torch.int64):
    g = rng(seed + t)
    u = torch.rand(t, generator=g, device="cuda", dtype=torch.double)
    tokens = (u * v).long()
    if kind == "zipf":
        tokens = (torch.exp(u * torch.log(torch.tensor(v + 1.0))) - 1).long().clamp(0, v - 1)
    if kind == "one":
        tokens[:] = v - 1
    if kind == "runs":
        tokens = (torch.arange(t, device="cuda") // 37) % v
    if kind == "none":
        tokens[:] = -1
    if kind == "padded":
        bad = torch.tensor([-1, v, -(1 << 31), (1 << 31) - 1], device="cuda")
        if dtype == torch.int64:
            bad = torch.cat([bad, torch.tensor([1 << 32, (1 << 32) + 1, -(1 << 62), 1 << 62],
                                               device="cuda")])
        pick = torch.rand(t, generator=g, device="cuda") < 0.3
        tokens = torch.where(pick, bad[torch.arange(t, device="cuda") % len(bad)], tokens)
    return tokens.to(dtype)


def embed64(tokens, table, scale):
    held = (tokens >= 0) & (tokens < len(table))
    out = table[torch.where(held, tokens, 0).long()].double() * scale
    return out * held[:, None]


def gradient64(tokens, v, grad, scale):
    """(gradient, sum of the terms' magnitudes, terms of each row), summed on the
    CPU: many tokens of one row would wait for each other on the GPU."""
    tokens, grad = tokens.cpu(), grad.cpu()
    held = (tokens >= 0) & (tokens < v)
    at, g = tokens[held].long(), grad[held].double() * scale
    zero = torch.zeros(v, grad.shape[1], dtype=torch.double)
    count = torch.bincount(at, minlength=v)[:, None]
    return [t.cuda() for t in (zero.index_add(0, at, g), zero.index_add(0, at, g.abs()), count)]


def check_gradient(got, tokens, v, grad, scale, dtype):
    want, mag, count = gradient64(tokens, v, grad, scale)
    assert got.dtype == dtype and got.shape == want.shape
    err = (2 * (count + 2) + 2) * 2.0 ** -24 * mag
    assert_within(got, want, err + UNIT[dtype] * (want.abs() + err) + TINY[dtype] * (mag > 0))


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("t,v,n,kind", TABLES)
def test_embed_tokens(gpu, t, v, n, kind, dtype, index):
    g = rng(t + n)
    tokens = make_tokens(t, v, kind, 1, index)
    table, cot = randn(g, v, n, dtype=dtype), randn(g, t, n, dtype=dtype)
    for scale in (1.0, 45.254834):
        leaf = table.clone().requires_grad_()
        out = ej.embed_tokens(tokens, leaf, scale=scale)
        assert out.dtype == dtype and out.shape == (t, n)
        want = embed64(tokens, table, scale)
        assert_within(out.detach(), want, (UNIT[dtype] + 3 * 2.0 ** -24) * want.abs()
                      + TINY[dtype] * (want != 0))
        if scale == 1.0:
            assert torch.equal(out.detach().double(), want)
        (got,) = torch.autograd.grad(out, leaf, cot)
        check_gradient(got, tokens, v, cot, scale, dtype)
        assert torch.equal(got, ej.embed_tokens_vjp(tokens, table, cot, scale=scale))


def test_embed_tokens_shapes(gpu):
    g = rng(2)
    table = randn(g, 50, 24, dtype=BF16)
    for shape in ((), (3,), (2, 0), (2, 5), (4, 1, 3)):
        tokens = torch.randint(-1, 50, shape, generator=g, device="cuda")
        leaf = table.clone().requires_grad_()
        out = ej.embed_tokens(tokens, leaf)
        assert out.shape == (*shape, 24)
        want = embed64(tokens.reshape(-1), table, 1.0)
        assert torch.equal(out.detach().double().reshape(-1, 24), want)
        cot = randn(g, *shape, 24, dtype=BF16)
        (got,) = torch.autograd.grad(out, leaf, cot)
        check_gradient(got, tokens.reshape(-1), 50, cot.reshape(-1, 24), 1.0, BF16)


def test_embed_tokens_views(gpu):
    """Strided tokens, tables and cotangents, rows off 16 bytes, a cotangent of
    another type, broadcast ones."""
    g = rng(3)
    wide, tokens = randn(g, 60, 200, dtype=BF16), torch.randint(0, 40, (300, 2), generator=g,
                                                                device="cuda")
    for table in (wide[:40, :64], wide[:40, 1:66], wide[1:41, 8:72], wide[::2][:40, 3:],
                  wide.t()[:64].t(), wide[:1, :64].expand(40, 64)):
        n = table.shape[1]
        for tok in (tokens[:, 0], tokens.t()[1], tokens[::3]):
            flat = tok.reshape(-1)
            rows = embed64(flat, table, 1.0)
            assert torch.equal(ej.embed_tokens(tok, table).double().reshape(-1, n), rows)
            cots = randn(g, *tok.shape, 2 * n + 1, dtype=BF16)
            for cot in (cots[..., :n], cots[..., 1:n + 1], cots[..., ::2][..., :n],
                        cots[..., :n].float(), cots[..., :1].expand(*tok.shape, n)):
                got = ej.embed_tokens_vjp(tok, table, cot)
                check_gradient(got, flat, len(table), cot.reshape(-1, n).to(BF16), 1.0, BF16)


def test_embed_gradient_against_differences(gpu):
    g = rng(4)
    tokens, table = make_tokens(500, 60, "zipf", 5), randn(g, 60, 33)
    cot, v = randn(g, 500, 33), randn(g, 60, 33)
    got = ej.embed_tokens_vjp(tokens, table, cot, scale=3.0)
    # linear: differences are exact up to rounding
    up, down = (ej.embed_tokens(tokens, table + h * v, scale=3.0).double() for h in (0.5, -0.5))
    num, want = float(((up - down) * cot).sum()), float((got.double() * v).sum())
    size = float((up.abs() * cot.abs()).sum() + (got.abs() * v.abs()).double().sum())
    assert abs(num - want) <= 600 * 2.0 ** -24 * size


@pytest.mark.parametrize("t", [700, 20000])
def test_embed_infinities_stay_in_their_rows(gpu, t):
    g = rng(6)
    tokens = make_tokens(t, 90, "padded", 6)
    table, cot = randn(g, 90, 40, dtype=BF16), randn(g, t, 40, dtype=BF16)
    table[7, 3], table[8, 4] = float("nan"), float("inf")
    bad = torch.nonzero((tokens == 11) | (tokens < 0))[:, 0]
    cot[bad] = float("nan")
    out = ej.embed_tokens(tokens, table)
    assert torch.equal(~torch.isfinite(out), ~torch.isfinite(embed64(tokens, table, 1.0)))
    assert bool((out[(tokens < 0) | (tokens >= 90)] == 0).all())
    got = ej.embed_tokens_vjp(tokens, table, cot)
    want = torch.zeros(90, dtype=torch.bool, device="cuda")
    want[11] = True
    assert torch.equal(torch.isnan(got).any(1), want) and torch.isnan(got[11]).all()


def test_embed_past_32_bits(gpu):
    """A table of more than 2^31 elements, and results of as many."""
    v, n = 530_000, 4096
    table = torch.zeros(v, n, dtype=BF16, device="cuda")
    last = randn(rng(7), 3, n, dtype=BF16)
    table[-3:] = last
    tokens = torch.tensor([v - 1, 0, v - 3, v, v - 2, v - 1], device="cuda")
    out = ej.embed_tokens(tokens, table)
    assert torch.equal(out[[0, 2, 4, 5]], last[[2, 0, 1, 2]])
    assert bool((out[[1, 3]] == 0).all())
    got = ej.embed_tokens_vjp(tokens, table, out)
    check_gradient(got[-3:], tokens - (v - 3), 3, out, 1.0, BF16)
    assert bool((got[:-3] == 0).all())
    del table, got
    tokens = torch.zeros(v, dtype=torch.int32, device="cuda")
    tokens[-1] = 1
    small = last[:2].contiguous()
    out = ej.embed_tokens(tokens, small)
    assert torch.equal(out[-2:], small) and torch.equal(out[v // 2], small[0])
    out[:-2] = 0
    got = ej.embed_tokens_vjp(tokens, small, out)
    assert torch.equal(got, small)


@pytest.mark.parametrize("t", [3000, 40000])
def test_embed_repeats_replays_and_streams(gpu, t):
    g = rng(8)
    tokens, table = make_tokens(t, 500, "zipf", 9), randn(g, 500, 200, dtype=BF16)
    cot = randn(g, t, 200, dtype=BF16)

    def call():
        return ej.embed_tokens(tokens, table, scale=2.5), ej.embed_tokens_vjp(tokens, table, cot)

    first = call()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, call()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, got))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(4):
        tokens.copy_(make_tokens(t, 500, "padded", i))
        cot.copy_(randn(g, t, 200, dtype=BF16))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, call()))


def test_embed_gradient_order_and_accumulation(gpu):
    g = rng(9)
    tokens, table = make_tokens(200, 30, "zipf", 9), randn(g, 30, 16)
    leaf = table.clone().requires_grad_()
    out = ej.embed_tokens(tokens, leaf)
    (out.sum() + ej.embed_tokens(tokens[:50], leaf).sum()).backward()
    ones = torch.ones(200, 16, device="cuda")
    want = ej.embed_tokens_vjp(tokens, table, ones) + ej.embed_tokens_vjp(tokens[:50], table,
                                                                          ones[:50])
    assert torch.equal(leaf.grad, want)
    with pytest.raises(RuntimeError, match="first order"):
        (gt,) = torch.autograd.grad(ej.embed_tokens(tokens, leaf).sum(), leaf, create_graph=True)
        gt.sum().backward()
    with torch.no_grad():
        assert not ej.embed_tokens(tokens, leaf).requires_grad
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(table, table)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ej.embed_tokens(tokens, dual)


def test_embed_refusals_of_gpu_tensors(gpu):
    table, tokens = torch.zeros(5, 8, device="cuda"), torch.zeros(3, dtype=torch.int32,
                                                                  device="cuda")
    for call in (lambda: ej.embed_tokens(tokens.float(), table),
                 lambda: ej.embed_tokens(tokens.short(), table),
                 lambda: ej.embed_tokens(tokens, table.double()),
                 lambda: ej.embed_tokens(tokens, table.int()),
                 lambda: ej.embed_tokens(tokens.cpu(), table),
                 lambda: ej.embed_tokens([0, 1], table),
                 lambda: ej.embed_tokens_vjp(tokens, table, torch.zeros(3, 8))):
        with pytest.raises(TypeError):
            call()
    for call in (lambda: ej.embed_tokens(tokens, table[0]),
                 lambda: ej.embed_tokens(tokens, table[None]),
                 lambda: ej.embed_tokens_vjp(tokens, table, table),
                 lambda: ej.embed_tokens_vjp(tokens, table, table[:3, :7])):
        with pytest.raises(ValueError):
            call()
    # no rows: every token is padding
    assert bool((ej.embed_tokens(tokens, table[:0]) == 0).all())
    assert ej.embed_tokens_vjp(tokens, table[:0], table[:3]).shape == (0, 8)
    assert ej.embed_tokens(tokens, table[:, :0]).shape == (3, 0)
    assert ej.embed_tokens_vjp(tokens, table[:, :0], table[:3, :0]).shape == (5, 0)
