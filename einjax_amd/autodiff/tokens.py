"""Rows of a table for tokens, and their gradient.

The lookup is a relation of tokens and rows; the gradient to the table is its
segment sum over the sorted tokens.  Arguments are checked, and the library
called, by the compiled binding (``csrc/experts_torch.cpp``); tensors are on the
GPU and work runs on torch's current stream of their device.  The reference has
no such operator.
"""

from __future__ import annotations

from .. import _lib

__all__ = ["embed_tokens", "embed_tokens_vjp"]


def embed_tokens(tokens, table, *, scale: float = 1.0):
    """out[..., :] = scale * table[tokens[...]].

    tokens int32 or int64 of any shape, table [rows, n] (float32, bfloat16 or
    float16); a token outside [0, rows), -1 for padding say, gets a row of zeros.
    The product with scale is in float32, rounded once to table's dtype.
    Differentiable in table (first order, reverse mode): the gradient is dense,
    zero in rows without tokens; a row's terms are summed in float32, in an order
    that the tokens alone set, times scale and rounded once.  The cotangent is
    rounded to table's dtype."""
    return _lib.experts().embed_tokens(tokens, table, scale)


def embed_tokens_vjp(tokens, table, grad_out, *, scale: float = 1.0):
    """Gradient of ``embed_tokens`` to table for the cotangent grad_out
    [..., n], which is rounded to table's dtype."""
    return _lib.experts().embed_tokens_vjp(tokens, table, grad_out, scale)
