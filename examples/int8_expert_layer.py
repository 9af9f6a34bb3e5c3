"""An expert layer whose router is kept balanced while it trains, and that is served in 8-bit integers, on one GPU:

  training   route -> gmm_swiglu -> gmm_scatter -> the router's weights, with balance_loss over the packed sequences
             of the batch
  serving    route -> quantize_rows, a row for each chosen expert -> gmm_int8 -> swiglu_quantize -> gmm_int8,
             the router's weights in the scales of the second product's rows

    python examples/int8_expert_layer.py
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
            (torch.randn(*shape, device=device) * shape[-1] ** -0.5).to(dtype))
        self.router = make(experts, hidden)
        self.w13 = make(experts, 2 * ffn, hidden)   # gate | up, stored (out, in)
        self.w2 = make(experts, hidden, ffn)

    def forward(self, x, offsets=None, mask=None):
        """(tokens, hidden) -> the layer's output and the losses of its router (see ops.balance_loss)."""
        logits = (x @ self.router.t()).float()
        r = ops.route(logits, self.top_k)
        h = ops.gmm_swiglu(x.index_select(0, r.row_index), self.w13, r.batch_sizes, trans_b=True)
        y = ops.gmm_scatter(h, self.w2, r.batch_sizes, r.order, trans_b=True)
        y = (y.view(x.shape[0], self.top_k, -1) * r.weights.unsqueeze(2)).sum(1).to(x.dtype)
        return y, ops.balance_loss(logits, r.experts, offsets, mask)


class Int8ExpertLayer:
    """The same for serving: weights in 8-bit integers, a scale for each of their rows."""

    def __init__(self, layer):
        self.top_k, self.router = layer.top_k, layer.router.detach()
        self.w13, self.w2 = ops.quantize_rows(layer.w13.detach()), ops.quantize_rows(layer.w2.detach())

    @torch.no_grad()
    def __call__(self, x):
        r = ops.route((x @ self.router.t()).float(), self.top_k)
        rows = ops.quantize_rows(x, r.row_index)
        gate_up = ops.gmm_int8(rows.values, rows.scales, self.w13.values, self.w13.scales, r.batch_sizes, dtype=x.dtype)
        h = ops.swiglu_quantize(gate_up)
        scales = h.scales * r.weights.view(-1).index_select(0, r.order)
        y = ops.gmm_int8(h.values, scales, self.w2.values, self.w2.scales, r.batch_sizes, dtype=x.dtype)
        return torch.zeros(x.shape, dtype=torch.float32, device=x.device).index_add_(0, r.row_index, y.float()).to(x.dtype)


def main(hidden=512, ffn=1024, experts=16, top_k=2, tokens=2048, steps=20):
    torch.manual_seed(0)
    layer = ExpertLayer(hidden, ffn, experts, top_k)
    x = torch.randn(tokens, hidden, device="cuda").bfloat16()
    target = torch.randn(tokens, hidden, device="cuda").bfloat16()
    # five sequences of different lengths, one behind the other; the last tokens of the batch are padding
    offsets = torch.tensor([0, 700, 720, 1500, 1501, tokens - 40], dtype=torch.int32, device="cuda")
    real = (torch.arange(tokens, device="cuda") < tokens - 40).unsqueeze(1)
    optimizer = torch.optim.AdamW(layer.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        y, router = layer(x, offsets)
        loss = ((y.float() - target.float()).square() * real).mean()
        (loss + 0.01 * router.balance + 0.001 * router.z).backward()
        optimizer.step()
        optimizer.zero_grad()
        losses.append((loss.detach(), router.balance.detach(), router.counts))
    losses = [(float(a), float(b), c) for a, b, c in losses]
    print(f"training: loss {losses[0][0]:.3f} -> {losses[-1][0]:.3f}, balance {losses[0][1]:.3f} -> {losses[-1][1]:.3f}")

    served = Int8ExpertLayer(layer)
    with torch.no_grad():
        one, _ = layer(x)
    other = served(x)
    off = float((one.float() - other.float()).norm() / one.float().norm())
    print(f"serving: {tokens} tokens in 8-bit integers, {100 * off:.2f} % from the training form; one token: {tuple(served(x[:1]).shape)}")
    return layer, losses, one, other, served


if __name__ == "__main__":
    main()
