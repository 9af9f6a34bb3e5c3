"""An expert layer as a model trains and serves it, on one GPU:

  training   route -> the tokens' rows sorted by expert -> gmm_swiglu -> gmm_scatter -> the router's weights,
             with a balancing loss from the experts' mass
  decode     route -> moe_few_tokens, two launches for the whole layer

and, beside a projection that all requests share, the low-rank adapter of each request.

    python examples/expert_layer.py
"""
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from grouped_gemm import ops  # noqa: E402


class ExpertLayer(torch.nn.Module):
    def __init__(self, hidden, ffn, experts, top_k, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        self.top_k = top_k
        make = lambda *shape: torch.nn.Parameter(  # noqa: E731
            (torch.randn(*shape, device=device) * shape[-2] ** -0.5).to(dtype))
        self.router = make(hidden, experts)
        self.w13 = make(experts, hidden, 2 * ffn)   # gate | up
        self.w2 = make(experts, ffn, hidden)

    def forward(self, x):
        """(tokens, hidden) -> the layer's output and a loss that is 1 where the tokens are spread evenly."""
        r = ops.route(x @ self.router, self.top_k, with_mass=True)
        h = ops.gmm_swiglu(x.index_select(0, r.row_index), self.w13, r.batch_sizes)
        y = ops.gmm_scatter(h, self.w2, r.batch_sizes, r.order)
        y = (y.view(x.shape[0], self.top_k, -1) * r.weights.unsqueeze(2)).sum(1).to(x.dtype)
        share = r.batch_sizes / (x.shape[0] * self.top_k)
        return y, r.batch_sizes.numel() * (share * r.mass / x.shape[0]).sum()

    @torch.no_grad()
    def decode(self, x):
        """The same for the few tokens of a decode step."""
        r = ops.route(x @ self.router, self.top_k)
        return ops.moe_few_tokens(x, self.w13, self.w2, r.experts, r.weights)


class AdaptedProjection(torch.nn.Module):
    """x @ weight^T, and for each row the low-rank adapter of its request (-1: none)."""

    def __init__(self, hidden_in, hidden_out, adapters, rank, dtype=torch.bfloat16, device="cuda"):
        super().__init__()
        make = lambda *shape: (torch.randn(*shape, device=device) * shape[-1] ** -0.5).to(dtype)  # noqa: E731
        self.weight = torch.nn.Parameter(make(1, hidden_out, hidden_in))
        self.a, self.b = make(adapters, rank, hidden_in), make(adapters, hidden_out, rank)
        self.scales = torch.full((adapters,), 0.5, device=device)

    @torch.no_grad()
    def forward(self, x, adapters):
        rows = torch.tensor([x.shape[0]])
        y = ops.gmm(x, self.weight, rows, trans_b=True)
        return ops.lora(x, self.a, self.b, adapters, base=y, scales=self.scales, c=y)


def main(hidden=512, ffn=1024, experts=16, top_k=2, tokens=2048, steps=20):
    torch.manual_seed(0)
    layer = ExpertLayer(hidden, ffn, experts, top_k)
    x = torch.randn(tokens, hidden, device="cuda").bfloat16()
    target = torch.randn(tokens, hidden, device="cuda").bfloat16()
    optimizer = torch.optim.AdamW(layer.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        y, balance = layer(x)
        loss = torch.nn.functional.mse_loss(y.float(), target.float())
        (loss + 0.01 * balance).backward()
        optimizer.step()
        optimizer.zero_grad()
        losses.append((loss.detach(), balance.detach()))
    losses = [(float(a), float(b)) for a, b in losses]
    print(f"training: loss {losses[0][0]:.3f} -> {losses[-1][0]:.3f}, balance {losses[0][1]:.3f} -> {losses[-1][1]:.3f}")

    few = x[:12]
    with torch.no_grad():
        one, _ = layer(few)
    other = layer.decode(few)
    print(f"decode: 12 tokens, largest difference from the training form {float((one.float() - other.float()).abs().max()):.4f} "
          f"of values up to {float(one.float().abs().max()):.2f}")

    projection = AdaptedProjection(hidden, 3 * hidden, adapters=8, rank=16)
    adapters = torch.tensor([3, 3, -1, 0, 7, 7, 7, 1, -1, 2, 5, 4], dtype=torch.int32, device="cuda")
    y = projection(few, adapters)
    print(f"adapters: {tuple(y.shape)}")
    return losses, one, other, y, projection, few, adapters


if __name__ == "__main__":
    main()
