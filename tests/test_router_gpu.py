"""The router's choice of experts and its balance loss, with their gradients,
against plain 64-bit forms."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mxref
from mlx_iqk_amd import router
from mlx_iqk_amd.kernels import IqkKernelError

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = (F32, F16, BF16)
ULP = 2.0 ** -23
FLOOR = 2.0 ** -126  # f32's smallest normal: exponentials below it flush


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().to(torch.float64).numpy()


def _logits(rng, *shape, dtype, device) -> torch.Tensor:
    return torch.from_numpy(rng.standard_normal(shape) * 2).to(dtype).to(device)


def _rel(experts: int) -> float:
    """Relative error of a probability: exponentials to 4 ulp, a sum of experts /
    16 in a lane and 4 over lanes, a division."""
    return (experts / 16 + 16) * ULP


def _rounded(dtype) -> float:
    return 0.0 if dtype == F32 else mxref.HALF_ULP[dtype]


# experts at both sides of each register count, odd ones; k from one to all
SHAPES = ((1, 1, 1), (1, 8, 8), (5, 60, 4), (33, 64, 6), (17, 65, 64), (100, 128, 17), (7, 161, 8), (64, 256, 6),
          (3, 257, 33), (9, 512, 16), (2, 1023, 10), (4, 1024, 64), (1000, 160, 6))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("tokens,experts,k", SHAPES)
def test_topk(device, dtype, normalize, tokens, experts, k):
    print(f"topk {dtype} {normalize} {tokens} {experts} {k}", flush=True)
    rng = np.random.default_rng(experts + k)
    logits = _logits(rng, tokens, experts, dtype=dtype, device=device)
    weights, ids = router.topk(logits, k, normalize=normalize)
    want_w, want_ids = mxref.topk(_f64(logits), k, normalize)
    assert weights.dtype == F32 and ids.dtype == torch.int32
    np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
    assert (np.abs(_f64(weights) - want_w) <= (_rel(experts) + k * ULP) * want_w + FLOOR).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("normalize", (True, False))
@pytest.mark.parametrize("tokens,experts,k", SHAPES)
def test_topk_gradient(device, dtype, normalize, tokens, experts, k):
    print(f"topk gradient {dtype} {normalize} {tokens} {experts} {k}", flush=True)
    rng = np.random.default_rng(experts + k + 1)
    logits = _logits(rng, tokens, experts, dtype=dtype, device=device).requires_grad_()
    dw = rng.standard_normal((tokens, k)).astype(np.float32)
    weights, ids = router.topk(logits, k, normalize=normalize)
    (got,) = torch.autograd.grad(weights, logits, torch.from_numpy(dw).to(device))
    assert got.dtype == dtype and got.shape == logits.shape
    x = _f64(logits)
    want = mxref.topk_grad(x, k, normalize, dw.astype(np.float64))
    w, at = mxref.topk(x, k, normalize)
    # |w| (|dw| + sum |w dw|), each of them as exact as a probability
    q = np.zeros_like(x)
    np.put_along_axis(q, at, w, -1)
    size = np.zeros_like(x)
    np.put_along_axis(size, at, w * np.abs(dw), -1)
    p = q if normalize else mxref.softmax(x)
    size += p * (w * np.abs(dw)).sum(-1, keepdims=True)
    bound = 3 * (_rel(experts) + k * ULP) * size + _rounded(dtype) * np.abs(want) + mxref.TINY[dtype] + 64 * FLOOR
    assert (np.abs(_f64(got) - want) <= bound).all()


@pytest.mark.parametrize("normalize", (True, False))
def test_topk_gradient_against_differences(device, normalize):
    """Central differences of the plain 64-bit weights along random directions
    (logits far enough apart that no choice changes)."""
    print(f"topk differences {normalize}", flush=True)
    rng = np.random.default_rng(11)
    x = (rng.permuted(np.tile(np.arange(24.0), (6, 1)), axis=1) * 0.25).astype(np.float32)
    logits = torch.from_numpy(x).to(device).requires_grad_()
    dw = rng.standard_normal((6, 5))
    weights, _ = router.topk(logits, 5, normalize=normalize)
    (got,) = torch.autograd.grad(weights, logits, torch.from_numpy(dw).to(device, F32))
    step = 1e-5
    for _ in range(4):
        d = rng.standard_normal(x.shape)
        hi, lo = (mxref.topk(x + s * step * d, 5, normalize)[0] for s in (1, -1))
        slope = ((hi - lo) / (2 * step) * dw).sum()
        # differences: step^2 and 1e-16 / step; the gradient: 24 x 6 terms to 1e-6
        assert abs((_f64(got) * d).sum() - slope) <= 1e-6 * np.abs(_f64(got) * d).sum() + 1e-8 + 40 * 2e-6 * 1e-2


@pytest.mark.parametrize("dtype", DTYPES)
def test_topk_ties_masks_and_bad_values(device, dtype):
    print(f"topk ties {dtype}", flush=True)
    inf, nan = float("inf"), float("nan")
    rows = [[1.0] * 20, [0.0, -0.0] * 10, [-inf] * 20, [-inf] * 18 + [2.0, 3.0], [2.0, -inf, 2.0] + [-inf] * 17,
            list(range(20)), [5.0, 5.0, 7.0, 7.0] * 5, [-60000.0] * 10 + [60000.0] * 10, [60000.0] + [-60000.0] * 19]
    logits = torch.tensor(rows, dtype=torch.float64).to(dtype).to(device).requires_grad_()
    for normalize in (True, False):
        for k in (1, 3, 20):
            weights, ids = router.topk(logits, k, normalize=normalize)
            want_w, want_ids = mxref.topk(_f64(logits), k, normalize)
            np.testing.assert_array_equal(ids.cpu().numpy(), want_ids)
            assert (np.abs(_f64(weights) - want_w) <= (_rel(20) + k * ULP) * want_w + FLOOR).all()
            (grad,) = torch.autograd.grad(weights, logits, torch.ones_like(weights))
            assert bool(torch.isfinite(grad).all())
            assert not bool(grad[2].any())  # nothing to choose from
    bad = torch.tensor([[1.0, nan, 2.0, nan, inf], [1.0, inf, 2.0, 0.0, inf], [0.0, 1.0, 2.0, 3.0, 4.0]]).to(dtype)
    weights, ids = router.topk(bad.to(device), 3)
    assert ids.tolist() == [[1, 3, 4], [1, 4, 2], [4, 3, 2]]
    assert bool(torch.isnan(weights[:2]).all()) and bool(torch.isfinite(weights[2]).all())


def test_topk_shapes_and_strides(device):
    print("topk shapes", flush=True)
    base = torch.randn((6, 50, 80), device=device)
    for logits in (base[0, 0], base[:, 0], base[:, ::3, 1:61], base.transpose(0, 2)[:, :, 0][:, :50].T.contiguous().T,
                   base[:0], base.to(BF16)[..., 1:78]):
        weights, ids = router.topk(logits, 3)
        flat = logits.reshape(-1, logits.shape[-1])
        want_w, want_ids = mxref.topk(_f64(flat), 3, True)
        assert weights.shape == ids.shape == (*logits.shape[:-1], 3)
        np.testing.assert_array_equal(ids.cpu().numpy().reshape(-1, 3), want_ids.reshape(-1, 3))
    # gradients of strided logits and of a broadcast gradient
    x = torch.randn((40, 30), device=device).requires_grad_()
    weights, _ = router.topk(x.T, 4, normalize=False)
    weights.sum().backward()
    y = x.detach().T.contiguous().requires_grad_()
    router.topk(y, 4, normalize=False)[0].sum().backward()
    assert torch.equal(x.grad, y.grad.T)


# ------------------------------------------------------------- balance loss ---

BALANCE = ((1, 1, 1, 1), (1, 7, 60, 4), (1, 33, 64, 2), (2, 100, 65, 6), (3, 31, 128, 8), (1, 500, 161, 6),
           (5, 64, 256, 6), (2, 70, 512, 3), (2, 40, 1023, 10), (1, 3000, 16, 2), (300, 5, 8, 2))


def _balance_case(rng, groups, tokens, experts, k, dtype, device, masked):
    logits = _logits(rng, groups, tokens, experts, dtype=dtype, device=device)
    ids = np.stack([mxref.topk(x, k, True)[1] for x in _f64(logits)])
    mask = rng.random((groups, tokens)) < 0.7 if masked else np.ones((groups, tokens), bool)
    return logits, ids, mask


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("masked", (False, True))
@pytest.mark.parametrize("groups,tokens,experts,k", BALANCE)
def test_balance_loss_and_gradient(device, dtype, masked, groups, tokens, experts, k):
    print(f"balance {dtype} {masked} {groups} {tokens} {experts} {k}", flush=True)
    rng = np.random.default_rng(tokens + experts)
    logits, ids, mask = _balance_case(rng, groups, tokens, experts, k, dtype, device, masked)
    if masked and groups > 1:
        mask[1] = False  # a sequence that is all padding
    logits.requires_grad_()
    loss, counts = router.balance_loss(logits, torch.from_numpy(ids).to(device, torch.int32),
                                       mask=torch.from_numpy(mask).to(device) if masked else None)
    dloss = rng.standard_normal(groups).astype(np.float32)
    (got,) = torch.autograd.grad(loss, logits, torch.from_numpy(dloss).to(device))
    assert loss.shape == (groups,) and counts.shape == (groups, experts) and got.dtype == dtype
    # sums of positive terms: a lane's tokens, the wavefronts, the shares
    steps = tokens / 32 + 8 + min(256, tokens / 32 + 1) + experts / 64 + 8
    x = _f64(logits)
    for g in range(groups):
        want, want_counts = mxref.balance(x[g], ids[g], mask[g])
        np.testing.assert_array_equal(counts[g].cpu().numpy(), want_counts)
        assert abs(_f64(loss)[g] - want) <= (_rel(experts) + steps * ULP) * want
        grad = dloss[g] * mxref.balance_grad(x[g], ids[g], mask[g])
        n = max(int(mask[g].sum()), 1)
        p = mxref.softmax(x[g]) * mask[g][:, None]
        size = abs(dloss[g]) * experts / (k * n * n) * p * (want_counts + (p * want_counts).sum(-1, keepdims=True))
        bound = 3 * _rel(experts) * size + _rounded(dtype) * np.abs(grad) + mxref.TINY[dtype] + 64 * FLOOR
        assert (np.abs(_f64(got)[g] - grad) <= bound).all()


def test_balance_gradient_against_differences(device):
    print("balance differences", flush=True)
    rng = np.random.default_rng(12)
    logits, ids, mask = _balance_case(rng, 1, 40, 20, 3, F32, device, True)
    flat = logits[0].clone().requires_grad_()
    loss, _ = router.balance_loss(flat, torch.from_numpy(ids[0]).to(device), mask=torch.from_numpy(mask[0]).to(device))
    assert loss.shape == ()
    loss.backward()
    x, step = _f64(flat), 1e-5
    for _ in range(4):
        d = rng.standard_normal(x.shape)
        hi, lo = (mxref.balance(x + s * step * d, ids[0], mask[0])[0] for s in (1, -1))
        terms = np.abs(_f64(flat.grad) * d).sum()
        assert abs((_f64(flat.grad) * d).sum() - (hi - lo) / (2 * step)) <= 1e-5 * terms + 1e-8


def test_balance_even_and_uneven_loads(device):
    """1 where every expert gets its share, experts / k where k experts take all."""
    print("balance loads", flush=True)
    even = torch.zeros((64, 16), device=device)
    ids = (torch.arange(64, device=device)[:, None] * 2 + torch.arange(2, device=device)) % 16
    assert float(router.balance_loss(even, ids)[0]) == pytest.approx(1.0, rel=_rel(16) + 16 * ULP)
    worst = torch.full((64, 16), -float("inf"), device=device)
    worst[:, :2] = 3.0
    loss, counts = router.balance_loss(worst, torch.tensor([[0, 1]], device=device).expand(64, 2))
    assert float(loss) == pytest.approx(8.0, rel=_rel(16) + 16 * ULP)
    assert counts.tolist() == [64, 64] + [0] * 14


def test_balance_ids_outside_the_stack_and_empty_rows(device):
    print("balance outside", flush=True)
    rng = np.random.default_rng(13)
    logits = _logits(rng, 30, 12, dtype=F32, device=device)
    logits[4] = -float("inf")
    logits.requires_grad_()
    ids = rng.integers(0, 12, (30, 3))
    ids[3], ids[9, 1], ids[10, 0] = (-1, 12, 2 ** 31), -2 ** 40, 2 ** 32 + 1
    named = torch.from_numpy(ids).to(device)
    loss, counts = router.balance_loss(logits, named)
    (grad,) = torch.autograd.grad(loss, logits)
    want, want_counts = mxref.balance(_f64(logits), ids, np.ones(30, bool))
    np.testing.assert_array_equal(counts.cpu().numpy(), want_counts)
    assert float(loss.detach()) == pytest.approx(want, rel=1e-5)
    assert bool(torch.isfinite(grad).all()) and not bool(grad[4].any())
    none = torch.zeros((30,), dtype=torch.bool, device=device)
    loss, counts = router.balance_loss(logits, named, mask=none)
    (grad,) = torch.autograd.grad(loss, logits)
    assert float(loss.detach()) == 0.0 and not bool(counts.any()) and not bool(grad.any())
    empty = torch.zeros((3, 0, 12), device=device)
    loss, counts = router.balance_loss(empty, torch.zeros((3, 0, 2), dtype=torch.int32, device=device))
    assert loss.tolist() == [0.0] * 3 and not bool(counts.any())
    assert router.balance_loss(torch.zeros((0, 4, 12), device=device),
                               torch.zeros((0, 4, 2), dtype=torch.int32, device=device))[0].shape == (0,)


def test_masked_tokens_may_hold_anything(device):
    print("masked tokens", flush=True)
    rng = np.random.default_rng(14)
    logits, ids, mask = _balance_case(rng, 1, 90, 40, 4, F32, device, True)
    named, keep = torch.from_numpy(ids).to(device), torch.from_numpy(mask).to(device)
    clean = logits.clone().requires_grad_()
    want = router.balance_loss(clean, named, mask=keep)
    spoiled = torch.where(keep[..., None], logits, torch.tensor(float("nan"), device=device)).requires_grad_()
    got = router.balance_loss(spoiled, named, mask=keep)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    one = torch.ones(1, device=device)
    a, b = torch.autograd.grad(want[0], clean, one)[0], torch.autograd.grad(got[0], spoiled, one)[0]
    assert torch.equal(a, b)


def test_repeats_and_streams(device):
    """The same bits on every call and on another stream."""
    print("repeats", flush=True)
    rng = np.random.default_rng(15)
    logits = _logits(rng, 2, 5000, 64, dtype=BF16, device=device).requires_grad_()
    dw = torch.randn((2, 5000, 4), device=device)

    def step():
        weights, ids = router.topk(logits, 4)
        loss, counts = router.balance_loss(logits, ids)
        (grad,) = torch.autograd.grad((weights, loss), logits, (dw, torch.ones_like(loss)))
        return weights, ids, loss, counts, grad

    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for g, w in zip(got, want))


def test_graph_replays(device):
    """The forward passes from a captured graph, as a serving step holds them."""
    print("router graph", flush=True)
    logits = torch.randn((2, 5000, 64), device=device).to(BF16)

    def step():
        weights, ids = router.topk(logits, 4)
        return weights, ids, *router.balance_loss(logits, ids)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(4):
        logits.copy_(torch.randn(logits.shape, device=device))
        graph.replay()
        torch.cuda.synchronize()
        got = [h.clone() for h in held]
        assert all(torch.equal(g, w) for g, w in zip(got, step()))


def test_a_second_derivative_is_refused(device):
    print("second derivative", flush=True)
    logits = torch.randn((6, 12), device=device).requires_grad_()
    weights, ids = router.topk(logits, 3)
    loss, _ = router.balance_loss(logits, ids)
    for out in ((weights ** 2).sum(), loss ** 2):
        (grad,) = torch.autograd.grad(out, logits, create_graph=True, retain_graph=True)
        with pytest.raises(RuntimeError, match="second time"):
            grad.sum().backward()
        (again,) = torch.autograd.grad(out, logits, retain_graph=True)
        assert torch.equal(again, grad) and not again.requires_grad


def test_refusals(device):
    print("router refusals", flush=True)
    z = lambda *s, dtype=F32: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    for logits, k in ((torch.zeros(3, 8), 2), (z(3, 8), 0), (z(3, 8), 9), (z(3, 1025), 2), (z(3, 100), 65), (z(3, 0), 1),
                      (z(3, 8, dtype=torch.float64), 2), (z(3, 8, dtype=torch.int32), 2), (None, 1)):
        with pytest.raises(IqkKernelError):
            router.topk(logits, k)
    ids = z(3, 2, dtype=torch.int32)
    for logits, named, mask in ((z(8), ids, None), (z(4, 8), ids, None), (z(3, 8), z(3, 2), None),
                                (z(3, 8), ids.cpu(), None), (z(3, 8), z(3, 9, dtype=torch.int32), None),
                                (z(3, 8), ids, z(3)), (z(3, 8), ids, z(4, dtype=torch.bool)),
                                (z(3, 8), ids, torch.zeros(3, dtype=torch.bool)), (torch.zeros(3, 8), ids, None)):
        with pytest.raises(IqkKernelError):
            router.balance_loss(logits, named, mask=mask)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("experts", (20, 60, 64, 161, 256, 1000))
def test_kept_tokens_without_numbers_show(device, dtype, experts):
    """A kept token whose logits are NaN, or NaN and -inf, makes its group's loss and its own
    gradient NaN; the other tokens' gradients stay as they are."""
    print(f"balance NaN {dtype} {experts}", flush=True)
    rng = np.random.default_rng(experts)
    logits, ids, mask = _balance_case(rng, 4, 40, experts, 2, dtype, device, False)
    clean = logits.clone()
    inf, nan = float("inf"), float("nan")
    logits[0, 3] = nan
    logits[1, 5] = -inf
    logits[1, 5, experts // 2] = nan
    logits[2, 7, :-1] = nan
    logits[2, 7, -1] = -inf
    named, one = torch.from_numpy(ids).to(device), torch.ones(4, device=device)
    grads = []
    for x in (logits, clean):
        x.requires_grad_()
        loss, _ = router.balance_loss(x, named)
        grads.append(_f64(torch.autograd.grad(loss, x, one)[0]))
        np.testing.assert_array_equal(np.isnan(_f64(loss)),
                                      [np.isnan(mxref.balance(_f64(x)[g], ids[g], mask[g])[0]) for g in range(4)])
    assert not np.isnan(grads[1]).any()
    bad = np.zeros((4, 40), bool)
    bad[[0, 1, 2], [3, 5, 7]] = True
    assert np.isnan(grads[0][bad]).all()
    np.testing.assert_array_equal(grads[0][~bad], grads[1][~bad])
    # the choice's weights and gradient
    for normalize in (True, False):
        weights, _ = router.topk(logits, 2, normalize=normalize)
        (grad,) = torch.autograd.grad(weights, logits, torch.ones_like(weights))
        want_w, want_ids = mxref.topk(_f64(logits).reshape(160, experts), 2, normalize)
        np.testing.assert_array_equal(np.isnan(_f64(weights)).reshape(160, 2), np.isnan(want_w))
        hit = np.zeros((160, experts), bool)
        np.put_along_axis(hit, want_ids, True, -1)
        hit = hit.reshape(4, 40, experts) if normalize else np.ones((4, 40, experts), bool)
        got = np.isnan(_f64(grad))
        assert got[bad][hit[bad]].all() and not got[~bad].any()


def test_a_second_derivative_is_refused_under_constant_gradients(device):
    """The gradients depend on the logits also where what comes from above is a constant."""
    print("second derivative, constant gradients", flush=True)
    logits = torch.randn((6, 12), device=device).requires_grad_()
    dw = torch.randn((6, 3), device=device)
    weights, ids = router.topk(logits, 3)
    full, _ = router.topk(logits, 3, normalize=False)
    loss, _ = router.balance_loss(logits, ids)
    for out in (loss, (weights * dw).sum(), (full * dw).sum(), weights[0, 0] + 2 * loss):
        (plain,) = torch.autograd.grad(out, logits, retain_graph=True)
        assert not plain.requires_grad
        (grad,) = torch.autograd.grad(out, logits, create_graph=True)
        assert torch.equal(grad, plain)
        with pytest.raises(RuntimeError, match="second time"):
            grad.sum().backward(retain_graph=True)
        # beside a term that has a second derivative
        (both,) = torch.autograd.grad(out + (logits ** 2).sum(), logits, create_graph=True)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(both.sum(), logits, retain_graph=True)


def test_forward_mode_derivatives_are_refused(device):
    print("router forward mode", flush=True)
    fwd = torch.autograd.forward_ad
    logits, ids = torch.randn((6, 12), device=device), torch.zeros((6, 2), dtype=torch.int32, device=device)
    want = router.topk(logits, 2)
    for base in (logits, logits.clone().requires_grad_(), logits.T.contiguous().T):
        with fwd.dual_level():
            x = fwd.make_dual(base, torch.ones_like(base))
            for call in (lambda: router.topk(x, 2), lambda: router.topk(x, 2, normalize=False),
                         lambda: router.balance_loss(x, ids)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
            # what carries no tangent is computed as before
            assert all(torch.equal(a, b) for a, b in zip(router.topk(logits, 2), want))


@pytest.mark.parametrize("normalize", (True, False))
def test_topk_past_32_bits(device, normalize):
    """More than 2^28 tokens (2^32 threads) and 2^32 logits, with the gradient."""
    print(f"topk past 2^32 {normalize}", flush=True)
    rows, experts, k = 2 ** 28 + 37, 17, 2
    g = torch.Generator(device=device).manual_seed(7)
    logits = torch.empty((rows, experts), dtype=F16, device=device)
    for part in logits.split(2 ** 25):
        part.copy_(torch.randn(part.shape, dtype=F16, device=device, generator=g))
    assert logits.numel() > 2 ** 32
    at = np.r_[0, 1, 2 ** 27 - 1, 2 ** 27, 2 ** 28 - 16, 2 ** 28 - 1, 2 ** 28, rows - 1]
    index = torch.from_numpy(at).to(device)
    x = _f64(logits[index])
    weights, ids = router.topk(logits.requires_grad_(), k, normalize=normalize)
    want_w, want_ids = mxref.topk(x, k, normalize)
    np.testing.assert_array_equal(ids[index].cpu().numpy(), want_ids)
    assert (np.abs(_f64(weights[index]) - want_w) <= (_rel(experts) + k * ULP) * want_w + FLOOR).all()
    few, few_ids = router.topk(logits.detach()[-99:], k, normalize=normalize)
    assert torch.equal(weights.detach()[-99:], few) and torch.equal(ids[-99:], few_ids)
    dw = torch.arange(1, k + 1, device=device, dtype=F32).expand(rows, k)
    (grad,) = torch.autograd.grad(weights, logits, dw)
    want = mxref.topk_grad(x, k, normalize, np.broadcast_to(np.arange(1.0, k + 1), (len(at), k)))
    # |p| (|dw| + sum |w dw|) <= 2 k, each as exact as a probability, and the rounding
    bound = 3 * (_rel(experts) + k * ULP) * 2 * k + _rounded(F16) * np.abs(want) + mxref.TINY[F16]
    assert (np.abs(_f64(grad[index]) - want) <= bound).all()


def test_balance_past_32_bits(device):
    """A group of more than 2^32 logits, with its gradient."""
    print("balance past 2^32", flush=True)
    tokens, experts, k = 2 ** 22 + 5, 1024, 2
    g = torch.Generator(device=device).manual_seed(8)
    logits = torch.empty((tokens, experts), dtype=F16, device=device)
    for part in logits.split(2 ** 19):
        part.copy_(torch.randn(part.shape, dtype=F16, device=device, generator=g))
    assert logits.numel() > 2 ** 32
    ids = torch.randint(0, experts, (tokens, k), dtype=torch.int32, device=device, generator=g)
    mean = torch.zeros(experts, dtype=torch.float64, device=device)
    for part in logits.split(2 ** 19):
        mean += torch.softmax(part.double(), -1).sum(0) / tokens
    loss, counts = router.balance_loss(logits.requires_grad_(), ids)
    want_counts = torch.bincount(ids.reshape(-1), minlength=experts)
    assert torch.equal(counts.long(), want_counts)
    want = float(experts * (want_counts.double() / (k * tokens) * mean).sum())
    # a lane adds its share's tokens, then wavefronts, shares and experts
    steps = tokens / 512 / 32 + 8 + 512 + experts / 64 + 8
    assert abs(float(loss.detach()) - want) <= (_rel(experts) + steps * ULP) * want
    # times 2^22, so that fp16 holds it
    (grad,) = torch.autograd.grad(loss, logits, torch.tensor(2.0 ** 22, device=device))
    at = np.r_[0, 2 ** 21, 2 ** 22 - 1, tokens - 1]
    index = torch.from_numpy(at).to(device)
    p, c = mxref.softmax(_f64(logits[index])), want_counts.double().cpu().numpy()
    factor = 2.0 ** 22 * experts / (k * float(tokens) ** 2)
    exact = factor * p * (c - (c * p).sum(-1, keepdims=True))
    size = factor * p * (c + (c * p).sum(-1, keepdims=True))
    bound = 3 * _rel(experts) * size + _rounded(F16) * np.abs(exact) + mxref.TINY[F16]
    assert (np.abs(_f64(grad[index]) - exact) <= bound).all()


def test_balance_takes_65535_groups(device):
    """And says so for one more."""
    print("balance groups", flush=True)
    rng = np.random.default_rng(16)
    logits = _logits(rng, 1, 1, 65536, 1, 8, dtype=F32, device=device)[0]
    ids = torch.from_numpy(rng.integers(0, 8, (1, 65536, 1, 2))).to(device)
    with pytest.raises(IqkKernelError, match="65535"):
        router.balance_loss(logits, ids)
    with pytest.raises(RuntimeError, match="iqk_balance_work"):  # nor 2^31 tokens
        router.balance_loss(logits.view(-1)[:1].to(F16).expand(2 ** 31, 1), ids.view(-1)[:1].expand(2 ** 31, 1))
    logits = logits[:, 1:].clone().requires_grad_()
    loss, counts = router.balance_loss(logits, ids[:, 1:])
    (grad,) = torch.autograd.grad(loss, logits, torch.ones_like(loss))
    assert loss.shape == (1, 65535) and counts.shape == (1, 65535, 8)
    for g in (0, 32768, 65534):
        x, named, one = _f64(logits)[0, g], ids[0, 1 + g].cpu().numpy(), np.ones(1, bool)
        want, want_counts = mxref.balance(x, named, one)
        np.testing.assert_array_equal(counts[0, g].cpu().numpy(), want_counts)
        assert abs(_f64(loss)[0, g] - want) <= (_rel(8) + 8 * ULP) * want
        p = mxref.softmax(x)
        size = 8 / 2 * p * (want_counts + (p * want_counts).sum(-1, keepdims=True))
        assert (np.abs(_f64(grad)[0, g] - mxref.balance_grad(x, named, one)) <= 3 * _rel(8) * size + 64 * FLOOR).all()


def test_gradients_under_capture_are_refused(device):
    """The nodes themselves, without the autograd engine: nothing of a backward pass runs under
    the capture, and the graph of what was captured beside them replays."""
    print("gradients under capture", flush=True)
    logits = torch.randn((6, 12), device=device).requires_grad_()
    weights, ids = router.topk(logits, 3)
    loss, _ = router.balance_loss(logits, ids)
    dw, one, x = torch.ones_like(weights), torch.ones_like(loss), torch.zeros(8, device=device)
    with torch.no_grad():
        weights.grad_fn(dw, None)  # not captured: as ever
        loss.grad_fn(one, None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with torch.no_grad():
            for node, above in ((weights.grad_fn, dw), (loss.grad_fn, one)):
                with pytest.raises(RuntimeError, match="captured"):
                    node(above, None)
    for n in (1, 2):
        graph.replay()
        torch.cuda.synchronize()
        assert x.tolist() == [float(n)] * 8
