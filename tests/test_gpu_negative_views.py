"""Operands that torch keeps as the negatives of what lies in memory: the imaginary
part of a conjugate is such a view, and a column of one is taken as it lies."""

import pytest
import torch

import einjax_amd as ej
from test_gpu_experts import F32, randn, rng

pytestmark = pytest.mark.gpu


def negated(g, *shape):
    """Values of `shape` in a view of the negative bit; the last extent is 1, so
    that the stride of 2 along it does not count."""
    v = torch.complex(randn(g, *shape[:-1], 4), randn(g, *shape[:-1], 4))[..., :1].conj().imag
    assert v.is_neg() and v.shape == shape
    return v


def test_products_of_negated_columns(gpu):
    g = rng(1)
    offsets = torch.tensor([0, 3, 9], dtype=torch.int32, device="cuda")
    x, w = negated(g, 9, 1), randn(g, 2, 1, 6)
    plain = x.resolve_neg()
    grad = randn(g, 9, 6)
    for op, cot in ((ej.grouped_matmul, grad), (ej.gated_matmul, grad[:, :3])):
        assert torch.equal(op(x, w, offsets), op(plain, w, offsets))
        leaf = plain.clone().requires_grad_()
        weight = w.clone().requires_grad_()
        want = torch.autograd.grad(op(leaf, weight, offsets), (leaf, weight), cot)
        vjp = {ej.grouped_matmul: ej.grouped_matmul_vjp, ej.gated_matmul: ej.gated_matmul_vjp}[op]
        assert all(torch.equal(a, b) for a, b in zip(vjp(x, w, offsets, cot), want))
    # weights of one column, and their gradient's cotangent of one column
    x, w, cot = randn(g, 9, 5), negated(g, 2, 5, 1), negated(g, 9, 1)
    assert torch.equal(ej.grouped_matmul(x, w, offsets),
                       ej.grouped_matmul(x, w.resolve_neg(), offsets))
    for a, b in zip(ej.grouped_matmul_vjp(x, w, offsets, cot),
                    ej.grouped_matmul_vjp(x, w.resolve_neg(), offsets, cot.resolve_neg())):
        assert torch.equal(a, b)


def test_negated_cotangents_of_autograd(gpu):
    """A result that goes on as the imaginary part of a complex number: its
    cotangent is a view of the negative bit."""
    g = rng(2)
    tokens = torch.tensor([2, 0, 2, 4], device="cuda")
    table = randn(g, 5, 1)
    weight = torch.complex(randn(g, 4, 1), randn(g, 4, 1))

    def loss(rows):
        return (torch.complex(torch.zeros_like(rows), rows).conj() * weight).real.sum()

    leaf = table.clone().requires_grad_()
    (got,) = torch.autograd.grad(loss(ej.embed_tokens(tokens, leaf)), leaf)
    (want,) = torch.autograd.grad(loss(leaf[tokens]), leaf)
    assert torch.equal(got, want)
    x, w = randn(g, 4, 3), randn(g, 1, 3, 1)
    offsets = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    leaf = x.clone().requires_grad_()
    (got,) = torch.autograd.grad(loss(ej.grouped_matmul(leaf, w, offsets)), leaf)
    cot = weight.imag
    assert torch.equal(got, ej.grouped_matmul_vjp(x, w, offsets, cot.contiguous())[0])


def test_other_operators_of_negated_columns(gpu):
    g = rng(3)
    tokens = torch.tensor([2, 0, 2, -1], device="cuda")
    table, cot = negated(g, 5, 1), negated(g, 4, 1)
    assert torch.equal(ej.embed_tokens(tokens, table), ej.embed_tokens(tokens, table.resolve_neg()))
    assert torch.equal(ej.embed_tokens_vjp(tokens, table, cot),
                       ej.embed_tokens_vjp(tokens, table, cot.resolve_neg()))
    x = negated(g, 7, 1)
    for quantize in (ej.quantize_rows, ej.quantize_blocks):
        (q, s), (p, t) = quantize(x), quantize(x.resolve_neg())
        assert torch.equal(q.to(F32), p.to(F32)) and torch.equal(s, t)
    (q, s), (p, t) = (ej.quantize_blocks(v, block_rows=128) for v in (x, x.resolve_neg()))
    assert torch.equal(q.to(F32), p.to(F32)) and torch.equal(s, t)
    # one token of one expert: scales, logits and weights of one value
    one = negated(g, 1, 1)
    plain = one.resolve_neg()
    q = torch.ones(1, 16, device="cuda")
    w8 = torch.ones(4, 16, device="cuda")
    for cast, product, scales in ((torch.int8, ej.int8_matmul, torch.ones(4, device="cuda")),
                                  (torch.float8_e4m3fn, ej.fp8_matmul,
                                   torch.ones(1, 1, device="cuda"))):
        scale = (one[:, 0], plain[:, 0]) if cast == torch.int8 else (one, plain)
        got, want = (product(q.to(cast), s, w8.to(cast), scales) for s in scale)
        assert torch.equal(got, want)
    r = ej.route_experts(plain, 1)
    for renorm in (True, False):
        a = ej.route_experts(one, 1, renormalize=renorm)
        assert torch.equal(a.weights, ej.route_experts(plain, 1, renormalize=renorm).weights)
    y = randn(g, 1, 1)
    assert torch.equal(ej.combine_experts(one, r), ej.combine_experts(plain, r))
    assert torch.equal(ej.combine_experts(y, r, one), ej.combine_experts(y, r, plain))
    got = ej.combine_experts_vjp(y, r, one, weights=plain)
    want = ej.combine_experts_vjp(y, r, plain, weights=plain)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    two = torch.cat([plain, -plain], 1)
    assert torch.equal(ej.route_experts_vjp(two, r.experts, one),
                       ej.route_experts_vjp(two, r.experts, plain))
