"""Differentiable sparse einsum (reference: autodiff/__init__.py) and expert
operators.

Gradients flow through tile values only; coordinates and matched pair
indices are static structure.  The backward runs in libejhip.so
(ej_pair_einsum_vjp).
"""

from .custom_vjp import sparse_einsum, sparse_einsum_raw, sparse_einsum_raw_vjp
from .experts import (
    combine_experts,
    combine_experts_vjp,
    gated_matmul,
    gated_matmul_vjp,
    grouped_matmul,
    grouped_matmul_vjp,
    route_experts,
    route_experts_vjp,
)
from .tokens import embed_tokens, embed_tokens_vjp

__all__ = ["sparse_einsum", "sparse_einsum_raw", "sparse_einsum_raw_vjp", "route_experts",
           "route_experts_vjp", "grouped_matmul", "grouped_matmul_vjp", "gated_matmul",
           "gated_matmul_vjp", "combine_experts", "combine_experts_vjp", "embed_tokens",
           "embed_tokens_vjp"]
