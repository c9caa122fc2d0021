"""A mixture-of-experts layer whose experts are frozen 4-bit microscaled weights:
its router trained with the balance loss, then the layer served.

    python examples/mx_moe.py [--experts 64 --hidden 2048 --inner 1024 --top-k 6]

Training runs the prompts' tokens, in quantised activations, grouped by expert;
the gradient reaches the router through the choice's weights and the balance
loss.  Serving runs one token a step in 16 bits, from a captured graph.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "mlx-iqk_amd"))

from mlx_iqk_amd import mx, router  # noqa: E402


class MoE(torch.nn.Module):
    """``y = sum_i w_i down_i(silu(gate_i x) * up_i x)`` over a token's top-k experts."""

    def __init__(self, experts: int, hidden: int, inner: int, k: int, device="cuda"):
        super().__init__()
        self.k = k
        self.score = torch.nn.Linear(hidden, experts, bias=False, device=device)
        self.gate = mx.MxSwitchLinear(experts, inner, hidden, device=device)
        self.up = mx.MxSwitchLinear(experts, inner, hidden, device=device)
        self.down = mx.MxSwitchLinear(experts, hidden, inner, device=device)

    def load(self, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor) -> None:
        """Quantise 16-bit stacks ``[experts, out, in]`` into the layer."""
        for projection, w in ((self.gate, gate), (self.up, up), (self.down, down)):
            projection.load(mx.quantize(w))

    def forward(self, x: torch.Tensor, quantized: bool = False):
        """``x`` 16-bit ``[tokens, hidden]`` -> (y ``[tokens, hidden]``, logits, ids).

        ``quantized``: the experts' activations in 4 bits too.  The experts have no
        gradient in ``x``: one that wants it is refused.
        """
        logits = self.score(x.float())
        weights, ids = router.topk(logits, self.k)
        cast = mx.quantize if quantized else (lambda t: t)
        rows = cast(x[:, None, None])  # [tokens, 1, 1, hidden]: a row for all its pairs
        hidden = torch.nn.functional.silu(self.gate(rows, ids)) * self.up(rows, ids)
        y = self.down(cast(hidden), ids)[:, :, 0]  # [tokens, k, hidden]: a row a pair
        return (weights[..., None] * y).sum(1).to(x.dtype), logits, ids


def train_step(moe: MoE, optimizer, x: torch.Tensor, target: torch.Tensor, mask: torch.Tensor, alpha: float):
    """One step of the router over ``x`` ``[sequences, tokens, hidden]``; masked-out
    tokens count for nothing.  Returns (fit, balance loss, tokens of each expert)."""
    sequences, tokens, hidden = x.shape
    y, logits, ids = moe(x.view(-1, hidden), quantized=True)
    fit = ((y.view_as(x).float() - target) ** 2).mean(-1)[mask].mean()
    # a loss for each sequence
    balance, counts = router.balance_loss(logits.view(sequences, tokens, -1), ids.view(sequences, tokens, -1),
                                          mask=mask)
    optimizer.zero_grad()
    (fit + alpha * balance.mean()).backward()
    optimizer.step()
    return fit.detach(), balance.detach().mean(), counts


class Server:
    """One decode step of the layer, captured once and replayed."""

    def __init__(self, moe: MoE, tokens: int, dtype=torch.bfloat16):
        self.x = torch.zeros(tokens, moe.gate.in_features, dtype=dtype, device=moe.score.weight.device)
        with torch.no_grad():
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                moe(self.x)
            torch.cuda.current_stream().wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.y = moe(self.x)[0]

    def __call__(self, x: torch.Tensor) -> torch.Tensor:
        self.x.copy_(x)
        self.graph.replay()
        return self.y


def random_layer(experts: int, hidden: int, inner: int, k: int) -> MoE:
    moe = MoE(experts, hidden, inner, k)
    moe.load(*(0.02 * torch.randn(experts, out, n, device="cuda", dtype=torch.bfloat16)
               for out, n in ((inner, hidden), (inner, hidden), (hidden, inner))))
    return moe


def main(argv=None) -> list[float]:
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--experts", type=int, default=64)
    p.add_argument("--hidden", type=int, default=2048)
    p.add_argument("--inner", type=int, default=1024)
    p.add_argument("--top-k", type=int, default=6)
    p.add_argument("--sequences", type=int, default=4)
    p.add_argument("--tokens", type=int, default=500)
    p.add_argument("--steps", type=int, default=20)
    a = p.parse_args(argv)
    torch.manual_seed(0)
    moe = random_layer(a.experts, a.hidden, a.inner, a.top_k)
    with torch.no_grad():  # a router that favours a few experts
        moe.score.weight[: max(1, a.experts // 8)] += 0.02
    x = torch.randn(a.sequences, a.tokens, a.hidden, device="cuda", dtype=torch.bfloat16) + 0.25
    target = torch.zeros_like(x, dtype=torch.float32)
    length = torch.linspace(a.tokens // 2, a.tokens, a.sequences, device="cuda").long()
    mask = torch.arange(a.tokens, device="cuda") < length[:, None]
    optimizer = torch.optim.Adam(moe.score.parameters(), lr=1e-3)
    balances = []
    for step in range(a.steps):
        fit, balance, counts = train_step(moe, optimizer, x, target, mask, alpha=1.0)
        balances.append(float(balance))
        if step % 5 == 0 or step == a.steps - 1:
            print(f"step {step}: fit {float(fit):.4g}, balance {balances[-1]:.3f}, "
                  f"most tokens of one expert {int(counts.sum(0).max())}", flush=True)
    serve = Server(moe, 1)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for t in range(200):
        y = serve(x[0, t % a.tokens])
    end.record()
    end.synchronize()
    print(f"serving: {start.elapsed_time(end) / 200 * 1e3:.1f} us a token, |y| {float(y.float().abs().mean()):.3g}")
    return balances


if __name__ == "__main__":
    main()
