"""A mixture-of-experts layer whose experts are frozen 4-bit microscaled weights:
its router trained with the balance loss, then the layer served.

    python examples/mx_moe.py [--experts 64 --hidden 2048 --inner 1024 --top-k 6 --requests 8]

Training runs the prompts' tokens, in quantised activations, grouped by expert;
the gradient reaches the router through the choice's weights and the balance
loss.  Serving runs one token of each request a step in 16 bits, from a captured graph, beside
a projection that all tokens share, to which each request brings a low-rank adapter.
"""

from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "mlx-iqk_amd"))

from mlx_iqk_amd import adapters, mx, router  # noqa: E402


class MoE(torch.nn.Module):
    """``y = sum_i w_i down_i(silu(gate_i x) * up_i x)`` over a token's top-k experts, and with a
    ``shared`` projection (an ``MxLinear``) its output added."""

    def __init__(self, experts: int, hidden: int, inner: int, k: int, device="cuda"):
        super().__init__()
        self.k = k
        self.shared = None
        self.score = torch.nn.Linear(hidden, experts, bias=False, device=device)
        self.gate = mx.MxSwitchLinear(experts, inner, hidden, device=device)
        self.up = mx.MxSwitchLinear(experts, inner, hidden, device=device)
        self.down = mx.MxSwitchLinear(experts, hidden, inner, device=device)

    def load(self, gate: torch.Tensor, up: torch.Tensor, down: torch.Tensor) -> None:
        """Quantise 16-bit stacks ``[experts, out, in]`` into the layer."""
        for projection, w in ((self.gate, gate), (self.up, up), (self.down, down)):
            projection.load(mx.quantize(w))

    def forward(self, x: torch.Tensor, quantized: bool = False, bank=None, requests=None):
        """``x`` 16-bit ``[tokens, hidden]`` -> (y ``[tokens, hidden]``, logits, ids).

        ``quantized``: the experts' activations in 4 bits too.  The experts have no
        gradient in ``x``: one that wants it is refused.  ``bank``: adapters of the shared
        projection, of which ``requests`` ``[tokens]`` names each token's.
        """
        logits = self.score(x.float())
        weights, ids = router.topk(logits, self.k)
        cast = mx.quantize if quantized else (lambda t: t)
        rows = cast(x[:, None, None])  # [tokens, 1, 1, hidden]: a row for all its pairs
        hidden = torch.nn.functional.silu(self.gate(rows, ids)) * self.up(rows, ids)
        y = self.down(cast(hidden), ids)[:, :, 0]  # [tokens, k, hidden]: a row a pair
        if self.shared is None and (bank is not None or requests is not None):
            raise ValueError("adapters add to the shared projection, which this layer has not")
        shared = None if self.shared is None else self.shared(x, bank, requests)
        return router.combine(y, weights, add=shared), logits, ids


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
    """One decode step of the layer, captured once and replayed; with a ``bank``, each
    token's adapter may be another one in every step."""

    def __init__(self, moe: MoE, tokens: int, dtype=torch.bfloat16, bank=None):
        device = moe.score.weight.device
        self.x = torch.zeros(tokens, moe.gate.in_features, dtype=dtype, device=device)
        self.requests = None if bank is None else torch.full((tokens,), -1, dtype=torch.int32, device=device)
        with torch.no_grad():
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                moe(self.x, bank=bank, requests=self.requests)
            torch.cuda.current_stream().wait_stream(side)
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph):
                self.y = moe(self.x, bank=bank, requests=self.requests)[0]

    def __call__(self, x: torch.Tensor, requests: torch.Tensor | None = None) -> torch.Tensor:
        """``requests``: each token's adapter (-1: none), with a bank and only with one."""
        if (requests is None) != (self.requests is None):
            raise ValueError("requests name adapters of the bank, for which the server was made without" if requests is not None
                             else "the server was made with a bank: name each token's adapter, -1 for none")
        self.x.copy_(x)
        if requests is not None:
            self.requests.copy_(requests)
        self.graph.replay()
        return self.y


def random_layer(experts: int, hidden: int, inner: int, k: int) -> MoE:
    moe = MoE(experts, hidden, inner, k)
    moe.load(*(0.02 * torch.randn(experts, out, n, device="cuda", dtype=torch.bfloat16)
               for out, n in ((inner, hidden), (inner, hidden), (hidden, inner))))
    return moe


def random_bank(moe: MoE, adapters_held: int, rank: int, dtype=torch.bfloat16) -> adapters.LowRankAdapters:
    """Give the layer a shared projection, and it a bank of adapters."""
    hidden, device = moe.gate.in_features, moe.score.weight.device
    moe.shared = mx.MxLinear(hidden, hidden, device=device)
    moe.shared.load(mx.quantize(0.02 * torch.randn(hidden, hidden, device=device, dtype=torch.bfloat16)))
    bank = adapters.LowRankAdapters(adapters_held, hidden, hidden, rank, dtype=dtype, device=device)
    for i in range(adapters_held):
        bank.load(i, hidden ** -0.5 * torch.randn(rank, hidden, device=device),
                  0.02 * torch.randn(hidden, rank, device=device), 2.0)
    return bank


def main(argv=None) -> list[float]:
    p = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    p.add_argument("--experts", type=int, default=64)
    p.add_argument("--hidden", type=int, default=2048)
    p.add_argument("--inner", type=int, default=1024)
    p.add_argument("--top-k", type=int, default=6)
    p.add_argument("--sequences", type=int, default=4)
    p.add_argument("--tokens", type=int, default=500)
    p.add_argument("--steps", type=int, default=20)
    p.add_argument("--requests", type=int, default=8, help="requests served together, each with its adapter")
    a = p.parse_args(argv)
    if not 0 < a.requests <= min(a.sequences * a.tokens, adapters.MAX_ADAPTERS):
        p.error(f"--requests must be 1 .. {min(a.sequences * a.tokens, adapters.MAX_ADAPTERS)}, the prompts' tokens or the "
                f"adapters of a bank, got {a.requests}")
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
    bank = random_bank(moe, a.requests, 16)
    serve = Server(moe, a.requests, bank=bank)
    requests = torch.arange(a.requests, device="cuda")
    prompts = x.view(-1, a.hidden)
    start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    start.record()
    for t in range(200):
        at = t * a.requests % (prompts.shape[0] - a.requests + 1)
        y = serve(prompts[at:at + a.requests], requests)
    end.record()
    end.synchronize()
    print(f"serving {a.requests} requests: {start.elapsed_time(end) / 200 * 1e3:.1f} us a step, "
          f"|y| {float(y.float().abs().mean()):.3g}")
    return balances


if __name__ == "__main__":
    main()
