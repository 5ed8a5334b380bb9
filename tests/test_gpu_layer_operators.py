"""The operators of a gated expert layer used together: token rows, routing, the
gated product, the second product and the sum, forward and backward, in a graph,
and the same in 8-bit floating point."""

import runpy
import threading
from pathlib import Path

import pytest
import torch

import einjax_amd as ej
from test_gpu_experts import BF16, F16, F32, randn, rng
from test_gpu_fp8 import plain_blocks, spread
from test_gpu_tokens import make_tokens

pytestmark = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parent.parent / "examples" / "gated_layer.py"


def layer_case(t, v, dim, hidden, e, dtype):
    g = rng(t + dim)
    return dict(tokens=make_tokens(t, v, "padded", 3), table=randn(g, v, dim, dtype=dtype),
                router=randn(g, dim, e, dtype=F32, scale=dim ** -0.5),
                w_in=randn(g, e, dim, 2 * hidden, dtype=dtype, scale=dim ** -0.5),
                w_out=randn(g, e, hidden, dim, dtype=dtype, scale=hidden ** -0.5),
                cot=randn(g, t, dim, dtype=dtype))


def run_layer(c, leaves, k=2):
    table, w_in, w_out = leaves
    x = ej.embed_tokens(c["tokens"], table, scale=2.0)
    logits = x.detach().float() @ c["router"]
    logits = logits.masked_fill((c["tokens"] < 0)[:, None], -float("inf"))  # padding: no expert
    r = ej.route_experts(logits, k)
    h = ej.gated_matmul(x, w_in, r, gather=True)
    return r, ej.combine_experts(ej.grouped_matmul(h, w_out, r), r)


def layer64(c, leaves, routing):
    """The same over dense products in 64 bits, for the picks of `routing`."""
    table, w_in, w_out = leaves
    held = (c["tokens"] >= 0) & (c["tokens"] < len(table))
    x = table[torch.where(held, c["tokens"], 0)] * 2.0 * held[:, None]
    y = 0
    for e in range(len(w_in)):
        share = (routing.weights * (routing.experts == e)).sum(1, keepdim=True).double()
        gate, up = (x @ w_in[e]).chunk(2, 1)
        y = y + share * ((torch.nn.functional.silu(gate) * up) @ w_out[e])
    return y


@pytest.mark.parametrize("dtype,room", [(F32, 2e-6), (BF16, 2e-2), (F16, 3e-3)])
@pytest.mark.parametrize("t,v,dim,hidden,e", [(1, 9, 64, 64, 4), (37, 11, 72, 40, 3),
                                              (700, 300, 256, 384, 8), (1500, 90, 77, 131, 5),
                                              (2600, 700, 512, 256, 4)])
def test_layer_and_its_gradients(gpu, t, v, dim, hidden, e, dtype, room):
    c = layer_case(t, v, dim, hidden, e, dtype)
    leaves = [c[n].clone().requires_grad_() for n in ("table", "w_in", "w_out")]
    r, y = run_layer(c, leaves)
    grads = torch.autograd.grad(y, leaves, c["cot"])
    wide = [c[n].double().requires_grad_() for n in ("table", "w_in", "w_out")]
    want = layer64(c, wide, r)
    wants = torch.autograd.grad(want, wide, c["cot"].double())
    # six operators, each rounding its results once to the type: at most eight half
    # steps on the way to any gradient, of a norm each below the result's own twice
    for got, ref in zip((y.detach(), *grads), (want.detach(), *wants)):
        assert got.dtype == dtype
        off = float((got.double() - ref).norm()), float(ref.norm())
        assert off[0] <= room * off[1] + 1e-30, off


def test_layer_gradients_in_a_graph(gpu):
    """A training step's forward and backward by the ``*_vjp`` calls, captured
    once, replayed on new tokens between eager steps."""
    c = layer_case(600, 80, 128, 96, 4, BF16)

    def step():
        x = ej.embed_tokens(c["tokens"], c["table"], scale=2.0)
        r = ej.route_experts(x.float() @ c["router"], 2)
        h = ej.gated_matmul(x, c["w_in"], r, gather=True)
        y = ej.grouped_matmul(h, c["w_out"], r)
        gy, _ = ej.combine_experts_vjp(y, r, c["cot"], need_weights=False)
        gh, g_out = ej.grouped_matmul_vjp(h, c["w_out"], r, gy)
        gx, g_in = ej.gated_matmul_vjp(x, c["w_in"], r, gh, gather=True)
        return ej.combine_experts(y, r), g_out, g_in, ej.embed_tokens_vjp(
            c["tokens"], c["table"], gx, scale=2.0)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(4):
        c["tokens"].copy_(make_tokens(600, 80, "zipf", i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_two_layers_interleaved_on_two_streams(gpu):
    """Two calls at once, each with workspaces of its own."""
    cases = [layer_case(900, 50, 256, 128, 4, BF16), layer_case(400, 70, 128, 256, 8, BF16)]
    want = []
    for c in cases:
        leaves = [c[n].clone().requires_grad_() for n in ("table", "w_in", "w_out")]
        _, y = run_layer(c, leaves)
        want.append((y.detach(), *torch.autograd.grad(y, leaves, c["cot"])))
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        for i, (c, s) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(s):
                leaves = [c[n].clone().requires_grad_() for n in ("table", "w_in", "w_out")]
                _, y = run_layer(c, leaves)
                got[i] = (y.detach(), *torch.autograd.grad(y, leaves, c["cot"]))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("t", [1, 5, 300, 1200])
def test_layer_in_8_bits(gpu, t):
    """Both products in 8 bits, against the quantized values' own in 64 bits."""
    g, e, dim, hidden = rng(t), 4, 256, 192
    x = randn(g, t, dim, dtype=BF16)
    w_in, w_out = randn(g, e, 2 * hidden, dim, dtype=BF16), randn(g, e, dim, hidden, dtype=BF16)
    r = ej.route_experts(randn(g, t, e), 2)
    q, s = ej.quantize_blocks(x)
    both = ej.fp8_matmul(q, s, *ej.quantize_blocks(w_in, block_rows=128), r, gather=True)
    gate, up = both.float().chunk(2, 1)
    h = (torch.nn.functional.silu(gate) * up).to(BF16)
    y = ej.fp8_matmul(*ej.quantize_blocks(h), *ej.quantize_blocks(w_out, block_rows=128), r)
    out = ej.combine_experts(y, r)

    def values(v, rows):
        p, by = plain_blocks(v, rows)
        return p.double() * spread(by, rows, *v.shape[-2:]).double()

    xe, wi, wo = values(x, 1), values(w_in, 128), values(w_out, 128)
    ends = r.offsets.tolist()
    want = torch.zeros(t, dim, dtype=torch.double, device="cuda")
    he = values(h, 1)
    for i in range(e):
        a, b = ends[i], ends[i + 1]
        at = r.rows[a:b].long()
        first = xe[at] @ wi[i].T
        assert float((both[a:b].double() - first).norm()) <= 4e-3 * float(first.norm()) + 1e-30
        share = (r.weights * (r.experts == i)).sum(1)[at].double()
        want.index_add_(0, at, share[:, None] * (he[a:b] @ wo[i].T))
    # rounded to bf16 as a product and as a sum: 2^-8 of their norms each
    assert float((out.double() - want).norm()) <= 2 * 2.0 ** -8 * 1.5 * float(want.norm())


def test_gated_layer_example(gpu):
    module = runpy.run_path(str(EXAMPLE))
    losses, error, model = module["main"](steps=3, verbose=False)
    assert len(losses) == 3 and all(0 < v < 100 for v in losses)
    # each product rounds rows and weights by at most 2^-4 of a value
    assert error < 4 * 2.0 ** -4
    # its gradients, against differences along the gradients themselves
    tokens = torch.arange(300, device="cuda")
    wide = module["TokenModel"](300, 64, 32, 4, 2, torch.float32)
    with torch.no_grad():
        picks = ej.route_experts(ej.embed_tokens(tokens, wide.table, scale=wide.scale)
                                 @ wide.layer.router, 2)
    params = [wide.layer.gate_up, wide.layer.down]

    def value():
        x = ej.embed_tokens(tokens, wide.table, scale=wide.scale)
        h = ej.gated_matmul(x, params[0], picks, gather=True)
        return ej.combine_experts(ej.grouped_matmul(h, params[1], picks), picks).square().sum()

    grads = torch.autograd.grad(value(), params)
    size = sum(float(g.double().square().sum()) for g in grads)
    step = 1e-3 / size ** 0.5
    ends = []
    for sign in (1, -1):
        with torch.no_grad():
            for p, g in zip(params, grads):
                p.add_(g, alpha=sign * step)
            ends.append(float(value()))
            for p, g in zip(params, grads):
                p.sub_(g, alpha=sign * step)
    assert abs((ends[0] - ends[1]) / (2 * step) / size - 1) < 0.02


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_nothing_to_do(gpu, dtype):
    """No experts, no tokens, no rows, no columns: empty results, or zeros."""
    def new(*shape):
        return torch.zeros(*shape, dtype=dtype, device="cuda")

    none = ej.group_by_expert(torch.full((5, 2), -1, device="cuda"), 3)
    for offsets in (torch.zeros(1, dtype=torch.int32, device="cuda"), none):
        e = 0 if offsets is not none else 3
        x, w = torch.ones_like(new(10, 16)), torch.ones_like(new(e, 16, 24))
        h = ej.gated_matmul(x, w, offsets)
        assert h.shape == (10, 12) and not h.any()
        gx, gw = ej.gated_matmul_vjp(x, w, offsets, torch.ones_like(h))
        assert gx.shape == x.shape and gw.shape == w.shape and not gx.any() and not gw.any()
        (q, qs), (p, ps) = ej.quantize_blocks(x), ej.quantize_blocks(w, block_rows=128)
        got = ej.fp8_matmul(q, qs, p.transpose(1, 2).contiguous(), ps, offsets)
        assert got.shape == (10, 24) and not got.any()
    no_tokens = torch.zeros(0, dtype=torch.int64, device="cuda")
    table = torch.ones_like(new(4, 8))
    assert ej.embed_tokens(no_tokens, table).shape == (0, 8)
    grad = ej.embed_tokens_vjp(no_tokens, table, new(0, 8))
    assert grad.shape == (4, 8) and not grad.any()
    tokens = torch.arange(3, device="cuda")
    out = ej.embed_tokens(tokens, new(0, 8))
    assert out.shape == (3, 8) and not out.any()
    assert ej.embed_tokens_vjp(tokens, new(0, 8), new(3, 8)).shape == (0, 8)
    assert ej.embed_tokens_vjp(tokens, new(4, 0), new(3, 0)).shape == (4, 0)


def test_two_graphs_of_one_pool(gpu):
    """Graphs that share their memory, replayed in turn on new inputs: split
    contractions, the sorts of few and of many tokens, sums in parts."""
    g = rng(12)
    x, w = randn(g, 12, 2048, dtype=BF16), randn(g, 2048, 1024, dtype=BF16, scale=2048 ** -0.5)
    cot = randn(g, 12, 512, dtype=BF16)
    tokens = make_tokens(20000, 300, "zipf", 1)
    few = tokens[:700].clone()
    table, grad = randn(g, 300, 96, dtype=BF16), randn(g, 20000, 96, dtype=BF16)

    def first():
        return (ej.gated_matmul(x, w), *ej.gated_matmul_vjp(x, w, None, cot),
                ej.embed_tokens_vjp(few, table, grad[:700]))

    def second():
        (q, qs), (p, ps) = ej.quantize_blocks(x), ej.quantize_blocks(w.t(), block_rows=128)
        return (ej.fp8_matmul(q, qs, p, ps), ej.embed_tokens(tokens, table),
                ej.embed_tokens_vjp(tokens, table, grad))

    first(), second()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for step in (first, second):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=graphs[0].pool() if graphs else None):
            outs.append(step())
        graphs.append(graph)
    for i in range(4):
        x.copy_(randn(g, 12, 2048, dtype=BF16))
        tokens.copy_(make_tokens(20000, 300, "zipf", i + 2))
        few.copy_(tokens[:700])
        for graph, step, out in zip(graphs, (first, second), outs):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_calls_of_two_threads(gpu):
    """Two threads, a stream each: the same results as one call after the other."""
    cases = [layer_case(500, 40, 128, 64, 4, BF16), layer_case(90, 60, 77, 131, 5, F16)]

    def work(c):
        leaves = [c[n].clone().requires_grad_() for n in ("table", "w_in", "w_out")]
        _, y = run_layer(c, leaves)
        grads = torch.autograd.grad(y, leaves, c["cot"])
        q, qs = ej.quantize_blocks(y)
        w, ws = ej.quantize_blocks(c["w_in"].transpose(1, 2)[0], block_rows=128)
        return (y.detach(), *grads, ej.fp8_matmul(q, qs, w, ws))

    want = [work(c) for c in cases]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i].append(work(cases[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as error:  # shown by the assertion below
            errors.append(error)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, runs in zip(want, got):
        assert len(runs) == 5
        for b in runs:
            assert all(torch.equal(x, y) for x, y in zip(a, b))
