"""The example layer: its outputs against float64 through the experts' own values, its router's
gradient against the formula's, a served step from a graph, and a few steps of training."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

EXAMPLE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "mx_moe.py")


@pytest.fixture(scope="module")
def mx_moe():
    spec = importlib.util.spec_from_file_location("mx_moe", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _exact(moe, x, cast):
    """y and the router's logits in float64; ``cast`` rounds the experts' activations as the layer does."""
    logits = moe.score(x.float()).detach().double()
    top = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids, w = top.indices[:, :moe.k], torch.softmax(top.values[:, :moe.k], -1)
    gate, up, down = (m.dequantized(torch.float32).double() for m in (moe.gate, moe.up, moe.down))
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    parts = torch.zeros(*ids.shape, x.shape[1], dtype=torch.float64, device=x.device)
    for t in range(x.shape[0]):
        row = cast(x[t]).double()
        for i, e in enumerate(ids[t].tolist()):
            a, b = (gate[e] @ row).to(x.dtype), (up[e] @ row).to(x.dtype)
            h = torch.nn.functional.silu(a) * b
            parts[t, i] = down[e] @ cast(h).double()
            y[t] += w[t, i] * parts[t, i]
    return y, w, ids, parts


# Each output rounds to 8 (11) bits at the hidden values, twice or three times, and once at
# the end: relative errors of at most 2^-8 each, those of a hidden row independent, so that
# the norm of the difference is at most 4 2^-8 (2^-11) of the output's.  The quantised form
# may also see a hidden value that rounds the other way, by half a step of its block (1/4 at
# most), for one in 50 of them: sqrt(1/50) / 4 < 0.04 of the norm.
@pytest.mark.parametrize("tokens", (1, 40))
@pytest.mark.parametrize("dtype,quantized,bound", ((torch.float16, False, 2e-3), (torch.bfloat16, False, 1.6e-2),
                                                   (torch.bfloat16, True, 5e-2)))
def test_layer(mx_moe, tokens, dtype, quantized, bound):
    print(f"layer {tokens} {dtype} {quantized}", flush=True)
    torch.manual_seed(tokens)
    moe = mx_moe.random_layer(12, 160, 96, 3)
    x = torch.randn(tokens, 160, device="cuda", dtype=dtype)
    cast = (lambda t: mx_moe.mx.quantize(t).dequantize()) if quantized else (lambda t: t)
    want, w, ids, parts = _exact(moe, x, cast)
    y, logits, got_ids = moe(x, quantized=quantized)
    assert torch.equal(got_ids.long(), ids)
    assert float((y.double() - want).norm()) <= bound * float(want.norm())
    # d loss / d logits of loss = (y * dy).sum(): w_i (s_i - sum_j w_j s_j), s_i = dy . part_i
    dy = torch.randn_like(want)
    (dlogits,) = torch.autograd.grad(y, logits, dy.to(y.dtype))
    s = (dy.to(y.dtype).double()[:, None] * parts).sum(-1)
    exact = torch.zeros_like(dlogits, dtype=torch.float64).scatter(-1, ids, w * (s - (w * s).sum(-1, keepdim=True)))
    scale = float((w * (dy[:, None] * parts).norm(dim=-1)).norm())  # the sums' size without cancellation
    assert float((dlogits.double() - exact).norm()) <= 2 * bound * scale


def test_served_from_a_graph(mx_moe):
    torch.manual_seed(3)
    moe = mx_moe.random_layer(12, 160, 96, 3)
    serve = mx_moe.Server(moe, 2)
    for _ in range(4):
        x = torch.randn(2, 160, device="cuda", dtype=torch.bfloat16)
        with torch.no_grad():
            want = moe(x)[0]
        torch.cuda.synchronize()
        assert torch.equal(serve(x), want)


def test_training_balances_the_router(mx_moe):
    balances = mx_moe.main("--experts 16 --hidden 160 --inner 96 --top-k 2 --sequences 3 --tokens 70 --steps 30".split())
    assert balances[-1] < balances[0]


@pytest.mark.parametrize("quantized", (False, True))
def test_a_gradient_in_x_is_refused(mx_moe, quantized):
    """The layer's experts have no gradient in x, so a part of it (the router's) is not offered."""
    moe = mx_moe.random_layer(12, 160, 96, 3)
    x = torch.randn(5, 160, device="cuda", dtype=torch.bfloat16)
    want = moe(x, quantized=quantized)[0]
    with pytest.raises(RuntimeError, match="detach"):
        moe(x.clone().requires_grad_(), quantized=quantized)
    with torch.no_grad():
        assert torch.equal(moe(x.clone().requires_grad_(), quantized=quantized)[0], want)
