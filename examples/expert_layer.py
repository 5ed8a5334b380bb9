"""A mixture-of-experts layer on the expert operators: training, then answering
single tokens with 8-bit weights.

    python3 examples/expert_layer.py

Routing makes the relation of tokens and experts, two products grouped by
expert contract over it (the first takes the tokens' rows through the relation,
without a copy), and the weighted sum takes the results back to the tokens.
The layer is fitted to a fixed random teacher of the same shape.
"""

import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import einjax_amd as ej  # noqa: E402


class ExpertLayer(torch.nn.Module):
    """y = sum over a token's k experts of weight * down_e(silu(up_e(x)))."""

    def __init__(self, dim, hidden, n_experts, k, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.k = k

        def param(*shape):
            return torch.nn.Parameter(
                torch.randn(*shape, device=device).mul_(shape[-2] ** -0.5).to(dtype))

        self.gate = param(dim, n_experts)
        self.up = param(n_experts, dim, hidden)
        self.down = param(n_experts, hidden, dim)

    def forward(self, x):
        routing = ej.route_experts(x @ self.gate, self.k)
        h = ej.grouped_matmul(x, self.up, routing, gather=True)
        y = ej.grouped_matmul(torch.nn.functional.silu(h), self.down, routing)
        return ej.combine_experts(y, routing)


class QuantizedExpertLayer:
    """The same with 8-bit weights (a scale for each output channel) and 8-bit
    activations (a scale for each row), for answering."""

    def __init__(self, layer):
        self.k, self.gate, self.dtype = layer.k, layer.gate.detach(), layer.up.dtype
        # rows of [experts, n_out, n_in] are output channels
        self.up, self.up_scale = ej.quantize_rows(layer.up.detach().transpose(1, 2))
        self.down, self.down_scale = ej.quantize_rows(layer.down.detach().transpose(1, 2))

    def __call__(self, x):
        routing = ej.route_experts(x @ self.gate, self.k)
        h = ej.int8_matmul(*ej.quantize_rows(x), self.up, self.up_scale, routing, gather=True,
                           out_dtype=self.dtype)
        y = ej.int8_matmul(*ej.quantize_rows(torch.nn.functional.silu(h)), self.down,
                           self.down_scale, routing, out_dtype=self.dtype)
        return ej.combine_experts(y, routing)


def main(dim=256, hidden=512, n_experts=8, k=2, tokens=4096, steps=60, verbose=True):
    torch.manual_seed(0)
    teacher = ExpertLayer(dim, hidden, n_experts, k)
    layer = ExpertLayer(dim, hidden, n_experts, k)
    with torch.no_grad():
        layer.gate.copy_(teacher.gate)  # the same relation: the experts are what is learned
    opt = torch.optim.Adam([layer.up, layer.down], lr=2e-3)
    losses = []
    for step in range(steps):
        x = torch.randn(tokens, dim, device="cuda", dtype=torch.bfloat16)
        with torch.no_grad():
            want = teacher(x)
        loss = (layer(x).float() - want.float()).square().mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
        if verbose and (step % 10 == 0 or step == steps - 1):
            print(f"step {step:3d} loss {losses[-1]:.4f}", flush=True)

    answer = QuantizedExpertLayer(layer)
    x = torch.randn(64, dim, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        full = layer(x).float()
        single = torch.cat([answer(row[None]) for row in x]).float()
    error = float((single - full).norm() / full.norm())
    if verbose:
        print(f"64 tokens one by one in 8 bits: {error:.4f} off the bf16 layer (relative)")
    return losses, error


if __name__ == "__main__":
    main()
