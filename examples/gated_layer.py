"""A small token model on a gated expert layer: training, then answering with
weights and activations in 8-bit floating point.

    python3 examples/gated_layer.py

Tokens take their rows of a table, a layer of gated experts maps them, and the
same table gives a score for every token that may follow.  The model learns a
fixed random map of the tokens.
"""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import einjax_amd as ej  # noqa: E402


class GatedExpertLayer(torch.nn.Module):
    """y = sum over a token's k experts of weight * down_e(silu(gate_e(x)) * up_e(x))."""

    def __init__(self, dim, hidden, n_experts, k, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.k = k

        def param(*shape):
            return torch.nn.Parameter(
                torch.randn(*shape, device=device).mul_(shape[-2] ** -0.5).to(dtype))

        self.router = param(dim, n_experts)
        self.gate_up = param(n_experts, dim, 2 * hidden)  # the gate's columns first
        self.down = param(n_experts, hidden, dim)

    def forward(self, x):
        routing = ej.route_experts(x @ self.router, self.k)
        h = ej.gated_matmul(x, self.gate_up, routing, gather=True)
        return ej.combine_experts(ej.grouped_matmul(h, self.down, routing), routing)


class BlockQuantizedLayer:
    """The same with 8-bit weights (a scale for each block of 128 x 128) and 8-bit
    activations (a scale for every 128 values of a row), for answering."""

    def __init__(self, layer):
        self.k, self.router, self.dtype = layer.k, layer.router.detach(), layer.down.dtype
        # rows of [experts, n_out, n_in] are output channels
        self.gate_up = ej.quantize_blocks(layer.gate_up.detach().transpose(1, 2), block_rows=128)
        self.down = ej.quantize_blocks(layer.down.detach().transpose(1, 2), block_rows=128)

    def __call__(self, x):
        routing = ej.route_experts(x @ self.router, self.k)
        both = ej.fp8_matmul(*ej.quantize_blocks(x), *self.gate_up, routing, gather=True,
                             out_dtype=self.dtype)
        gate, up = both.chunk(2, 1)
        h = torch.nn.functional.silu(gate) * up
        y = ej.fp8_matmul(*ej.quantize_blocks(h), *self.down, routing, out_dtype=self.dtype)
        return ej.combine_experts(y, routing)


class TokenModel(torch.nn.Module):
    def __init__(self, tokens, dim, hidden, n_experts, k, dtype=torch.bfloat16):
        super().__init__()
        self.table = torch.nn.Parameter(
            (torch.randn(tokens, dim, device="cuda") * dim ** -0.5).to(dtype))
        self.scale = dim ** 0.5
        self.layer = GatedExpertLayer(dim, hidden, n_experts, k, dtype)

    def scores(self, tokens, layer=None):
        x = ej.embed_tokens(tokens, self.table, scale=self.scale)
        return ((x + (layer or self.layer)(x)) @ self.table.t()).float()


def main(tokens=512, dim=256, hidden=256, n_experts=8, k=2, batch=4096, steps=60, verbose=True):
    torch.manual_seed(0)
    model = TokenModel(tokens, dim, hidden, n_experts, k)
    follows = torch.randperm(tokens, device="cuda")
    opt = torch.optim.Adam(model.parameters(), lr=2e-3)
    losses = []
    for step in range(steps):
        seen = torch.randint(0, tokens, (batch,), device="cuda")
        loss = torch.nn.functional.cross_entropy(model.scores(seen), follows[seen])
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if verbose and (step % 10 == 0 or step == steps - 1):
            print(f"step {step:3d} loss {losses[-1]:.4f}", flush=True)

    answer = BlockQuantizedLayer(model.layer)
    with torch.no_grad():
        seen = torch.arange(64, device="cuda")
        full = model.scores(seen)
        single = torch.cat([model.scores(t[None], answer) for t in seen])
    error = float((single - full).norm() / full.norm())
    if verbose:
        print(f"64 tokens one by one in 8 bits: {error:.4f} off the bf16 model (relative)")
    return losses, error, model


if __name__ == "__main__":
    main()
