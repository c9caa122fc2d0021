"""Pairs sorted by expert, their rows dispatched and combined, with the gradients, against
plain 64-bit forms on the CPU."""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

import mxref
from mlx_iqk_amd import mx, router
from mlx_iqk_amd.kernels import IqkKernelError

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
DTYPES = (F32, F16, BF16)
I32, I64 = torch.int32, torch.int64
U = 2.0 ** -24  # half a step of f32, relative


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().to(torch.float64).numpy()


def _bits(t: torch.Tensor) -> torch.Tensor:
    return t.detach().cpu().contiguous().view({2: torch.int16, 4: torch.int32}[t.element_size()])


def _rounded(dtype) -> float:
    return 0.0 if dtype == F32 else mxref.HALF_ULP[dtype]


def _sorted(ids: np.ndarray, experts: int) -> dict:
    key = np.where((ids >= 0) & (ids < experts), ids, experts).reshape(-1)
    pairs = np.argsort(key, kind="stable")
    slots = np.empty(key.size, np.int64)
    slots[pairs] = np.arange(key.size)
    return {"offsets": np.searchsorted(key[pairs], np.arange(experts + 1)), "ids": key[pairs],
            "tokens": pairs // ids.shape[-1], "slots": slots.reshape(ids.shape)}


def _check_order(order, ids: np.ndarray, experts: int) -> dict:
    want = _sorted(ids, experts)
    assert order.num_experts == experts
    for name, value in want.items():
        got = getattr(order, name)
        assert got.dtype == I32 and tuple(got.shape) == value.shape
        np.testing.assert_array_equal(got.cpu().numpy(), value)
    return want


def _ids(rng, tokens: int, k: int, experts: int, spread: float = 0.0, out: float = 0.1) -> np.ndarray:
    """Ids uneven by ``spread``, a share ``out`` of them outside the experts."""
    weight = np.arange(1, experts + 1, dtype=np.float64) ** -spread
    ids = rng.permutation(experts)[rng.choice(experts, size=(tokens, k), p=weight / weight.sum())].astype(np.int64)
    left = rng.random((tokens, k)) < out
    ids[left] = rng.choice((-1, experts, experts + 7, -2 ** 31, 2 ** 31 - 1), size=int(left.sum()))
    return ids


# tokens, k, experts: one pair, odd counts, more pairs than one share and than one launch counts
SORTS = ((1, 1, 1), (1, 6, 256), (3, 5, 7), (8, 6, 256), (64, 1, 64), (65, 1, 3), (100, 8, 1024), (171, 3, 1023),
         (1024, 1, 2), (513, 2, 60), (256, 64, 300), (2731, 6, 256), (257, 64, 8), (4097, 4, 1024), (40000, 7, 512))


@pytest.mark.parametrize("dtype", (I32, I64))
@pytest.mark.parametrize("tokens,k,experts", SORTS)
def test_sort(device, dtype, tokens, k, experts):
    print(f"sort {dtype} {tokens} {k} {experts}", flush=True)
    rng = np.random.default_rng(tokens + k)
    for spread, out in ((0.0, 0.0), (1.1, 0.2)):
        ids = _ids(rng, tokens, k, experts, spread, out)
        if dtype == I64 and out:
            ids.reshape(-1)[0] = 2 ** 32  # whose low word is expert 0
            ids.reshape(-1)[-1] = -2 ** 32 + 1
        _check_order(router.sort(torch.from_numpy(ids).to(device, dtype), experts), ids, experts)


@pytest.mark.parametrize("tokens", (1, 70, 5000))
def test_sort_of_one_key(device, tokens):
    """All of one expert, the last one too, and nothing but left-out pairs."""
    print(f"sort one key {tokens}", flush=True)
    for e in (0, 8, 9, -1):
        ids = np.full((tokens, 4), e, np.int64)
        _check_order(router.sort(torch.from_numpy(ids).to(device), 9), ids, 9)


def test_sort_takes_what_ids_come_in(device):
    print("sort id types", flush=True)
    rng = np.random.default_rng(3)
    ids = rng.integers(0, 12, (5, 7, 3))
    whole = torch.from_numpy(ids).to(device)
    for given in (whole.to(torch.uint8), whole.to(torch.int16), whole.transpose(0, 1).contiguous().transpose(0, 1),
                  whole.to(I32).repeat_interleave(2, -1)[..., ::2]):
        _check_order(router.sort(given, 12), ids, 12)
    one = router.sort(whole[0, 0], 12)  # a single token without a leading axis
    _check_order(one, ids[0, 0], 12)
    shifted = torch.empty(106, dtype=I64, device=device)[1:].view(5, 7, 3).copy_(whole)
    _check_order(router.sort(shifted, 12), ids, 12)


def test_no_tokens(device):
    print("no tokens", flush=True)
    ids = torch.empty((0, 3), dtype=I32, device=device)
    x = torch.empty((0, 40), dtype=F16, device=device, requires_grad=True)
    rows, order = router.dispatch(x, ids, 5)
    assert rows.shape == (0, 40) and order.offsets.tolist() == [0] * 6 and order.slots.shape == (0, 3)
    weights = torch.empty((0, 3), device=device, requires_grad=True)
    out = router.combine(rows, weights, order)
    assert out.shape == (0, 40)
    dx, dw = torch.autograd.grad(out, (x, weights), torch.empty_like(out))
    assert dx.shape == x.shape and dw.shape == weights.shape
    assert router.combine(torch.empty((0, 3, 40), device=device), weights.detach()).shape == (0, 40)


# tokens, k, cols: rows of one value, of whole chunks, and of odd rests; more than one group of choices
ROWS = ((1, 1, 1), (1, 6, 4096), (3, 2, 7), (5, 9, 8), (33, 3, 9), (300, 4, 64), (17, 64, 40), (7, 17, 513), (40, 6, 1441),
        (9, 3, 2048), (2, 8, 8200), (700, 5, 100))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,cols", ROWS)
def test_dispatch(device, dtype, tokens, k, cols):
    print(f"dispatch {dtype} {tokens} {k} {cols}", flush=True)
    rng = np.random.default_rng(cols + k)
    experts = 13
    for out in (0.0, 0.25, 1.0):
        ids = _ids(rng, tokens, k, experts, 0.5, out)
        x = torch.from_numpy(rng.standard_normal((tokens, cols))).to(dtype).to(device).requires_grad_()
        rows, order = router.dispatch(x, torch.from_numpy(ids).to(device), experts)
        want = _check_order(order, ids, experts)
        left = want["ids"] == experts
        source = x.detach().cpu()[torch.from_numpy(want["tokens"])]
        source[torch.from_numpy(left)] = 0
        assert rows.dtype == dtype and torch.equal(_bits(rows), _bits(source))
        drows = torch.from_numpy(rng.standard_normal(rows.shape)).to(dtype).to(device)
        (dx,) = torch.autograd.grad(rows, x, drows)
        assert dx.dtype == dtype and dx.shape == x.shape
        parts = np.where(left[:, None], 0.0, _f64(drows))[want["slots"]]  # [tokens, k, cols]
        exact, size = parts.sum(1), np.abs(parts).sum(1)
        # k - 1 additions in f32, each off by half a step of at most `size`; one rounding
        error = k * U * size
        assert (np.abs(_f64(dx) - exact) <= error + _rounded(dtype) * (np.abs(exact) + error)).all()


def _combine_case(rng, tokens, k, cols, dtype, device, out):
    experts = 11
    ids = _ids(rng, tokens, k, experts, 0.5, out)
    tensor = lambda *s: torch.from_numpy(rng.standard_normal(s)).to(dtype).to(device)  # noqa: E731
    weights = torch.from_numpy(rng.standard_normal((tokens, k)).astype(np.float32)).to(device)
    return ids, experts, tensor(tokens * k, cols), weights, tensor(tokens, cols), tensor(tokens, cols)


def _check_combine(dtype, got, dy, dw, y, w, add, dout, slots, left):
    """Against float64; slots [tokens, k] places in y [pairs, cols], left the pairs not counted."""
    k, cols = w.shape[1], y.shape[1]
    parts = np.where(left[..., None], 0.0, y[slots])
    exact = (w[..., None] * parts).sum(1) + add
    # k fused additions and one more in f32, one rounding
    size = (np.abs(w[..., None] * parts)).sum(1) + np.abs(add)
    error = (k + 1) * U * size
    assert (np.abs(_f64(got) - exact) <= error + _rounded(dtype) * (np.abs(exact) + error) + mxref.TINY[dtype]).all()
    if dy is not None:
        want = np.zeros_like(y)
        want[slots] = np.where(left[..., None], 0.0, w[..., None] * dout[:, None])
        # a product in f32, one rounding
        assert (np.abs(_f64(dy).reshape(want.shape) - want) <= (_rounded(dtype) + 2 * U) * np.abs(want)
                + mxref.TINY[dtype]).all()
    if dw is not None:
        want, size = (parts * dout[:, None]).sum(-1), np.abs(parts * dout[:, None]).sum(-1)
        # a lane's fused additions (at most cols / 64 and a chunk), then 6 + 3 of sums
        assert (np.abs(_f64(dw) - want) <= (cols / 64 + 8 + 10) * U * size).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,cols", ROWS)
def test_combine(device, dtype, tokens, k, cols):
    print(f"combine {dtype} {tokens} {k} {cols}", flush=True)
    rng = np.random.default_rng(cols + k + 1)
    for out in (0.0, 0.25, 1.0):
        ids, experts, y, weights, add, dout = _combine_case(rng, tokens, k, cols, dtype, device, out)
        order = router.sort(torch.from_numpy(ids).to(device), experts)
        want = _sorted(ids, experts)
        left = want["slots"] >= want["offsets"][-1]
        for given in (None, add):
            leaves = [t.clone().requires_grad_() for t in (y, weights) + ((add,) if given is not None else ())]
            got = router.combine(leaves[0], leaves[1], order, add=leaves[2] if given is not None else None)
            assert got.dtype == dtype and got.shape == (tokens, cols)
            dy, dw, *dadd = torch.autograd.grad(got, leaves, dout)
            _check_combine(dtype, got, dy, dw, _f64(y), _f64(weights), _f64(add) if given is not None else np.zeros(1),
                           _f64(dout), want["slots"], left)
            assert not dadd or torch.equal(dadd[0], dout)
            # one gradient alone, and none
            alone = router.combine(y, leaves[1], order, add=given)
            assert torch.equal(torch.autograd.grad(alone, leaves[1], dout)[0], dw) and torch.equal(alone, got)
            alone = router.combine(leaves[0], weights, order, add=given)
            assert torch.equal(torch.autograd.grad(alone, leaves[0], dout)[0], dy)
            assert torch.equal(router.combine(y, weights, order, add=given), got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,cols", ROWS)
def test_combine_of_rows_in_the_tokens_order(device, dtype, tokens, k, cols):
    print(f"combine unsorted {dtype} {tokens} {k} {cols}", flush=True)
    rng = np.random.default_rng(cols + k + 2)
    _, _, y, weights, add, dout = _combine_case(rng, tokens, k, cols, dtype, device, 0.0)
    leaves = [t.clone().requires_grad_() for t in (y.view(tokens, k, cols), weights, add)]
    got = router.combine(*leaves[:2], add=leaves[2])
    dy, dw, dadd = torch.autograd.grad(got, leaves, dout)
    assert dy.shape == (tokens, k, cols) and torch.equal(dadd, dout)
    slots = np.arange(tokens * k).reshape(tokens, k)
    _check_combine(dtype, got, dy, dw, _f64(y), _f64(weights), _f64(add), _f64(dout), slots, np.zeros_like(slots, bool))


def test_leading_axes_and_16_bit_weights(device):
    print("leading axes", flush=True)
    rng = np.random.default_rng(9)
    x = torch.from_numpy(rng.standard_normal((2, 5, 3, 24))).to(BF16).to(device).requires_grad_()
    ids = torch.from_numpy(_ids(rng, 30, 4, 6)).to(device).view(2, 5, 3, 4)
    rows, order = router.dispatch(x, ids, 6)
    flat, flat_order = router.dispatch(x.detach().view(30, 24), ids.view(30, 4), 6)
    assert torch.equal(rows, flat) and torch.equal(order.slots.view(30, 4), flat_order.slots)
    assert order.slots.shape == (2, 5, 3, 4)
    for dtype in (F32, BF16, F16):
        w = torch.from_numpy(rng.random((2, 5, 3, 4))).to(dtype).to(device).requires_grad_()
        out = router.combine(rows, w, order)
        assert out.shape == x.shape and out.dtype == BF16
        same = router.combine(flat, w.detach().float().view(30, 4), flat_order)
        assert torch.equal(out.detach().view(30, 24), same)
        dx, dw = torch.autograd.grad(out, (x, w), torch.ones_like(out), retain_graph=True)
        assert dx.shape == x.shape and dw.shape == w.shape and dw.dtype == dtype
    # one token without a leading axis
    rows, order = router.dispatch(x.detach()[0, 0, 0], ids[0, 0, 0], 6)
    assert rows.shape == (4, 24) and router.combine(rows, w.detach()[0, 0, 0], order).shape == (24,)


@pytest.mark.parametrize("dtype", DTYPES)
def test_any_address_and_stride(device, dtype):
    """Operands that start at an odd element, transposed ones, expanded ones; their gradients too."""
    print(f"addresses {dtype}", flush=True)
    rng = np.random.default_rng(10)
    tokens, k, cols, experts = 21, 3, 72, 8
    ids, _, y, weights, add, dout = _combine_case(rng, tokens, k, cols, dtype, device, 0.2)
    named = torch.from_numpy(ids).to(device)

    def odd(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=device)[1:].view(t.shape).copy_(t)

    def turned(t):
        return t.transpose(0, 1).contiguous().transpose(0, 1)

    order = router.sort(named, experts)
    want = router.combine(y, weights, order, add=add)
    rows, _ = router.dispatch(add, named, experts)
    for change in (odd, turned):
        assert torch.equal(router.dispatch(change(add), change(named), experts)[0], rows)
        leaves = [change(t).requires_grad_() for t in (y, weights, add)]
        got = router.combine(*leaves[:2], order, add=leaves[2])
        assert torch.equal(got, want)
        base = [t.clone().requires_grad_() for t in (y, weights, add)]
        grads = torch.autograd.grad(router.combine(*base[:2], order, add=base[2]), base, dout)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(got, leaves, change(dout)), grads))
        x = change(add).requires_grad_()
        moved, _ = router.dispatch(x, named, experts)
        (dx,) = torch.autograd.grad(moved, x, change(y))
        x = add.clone().requires_grad_()
        assert torch.equal(dx, torch.autograd.grad(router.dispatch(x, named, experts)[0], x, y)[0])
    # one row for all tokens, and a gradient that is one number expanded
    x = add[:1].clone().requires_grad_()
    moved, _ = router.dispatch(x.expand(tokens, cols), named, experts)
    (dx,) = torch.autograd.grad(moved.float().sum(), x)
    kept = int(((ids >= 0) & (ids < experts)).sum(1).astype(float).sum())
    # whole numbers up to 3 a token, whose sum torch rounds once more
    assert dx.shape == (1, cols) and (np.abs(_f64(dx) - kept) <= (mxref.HALF_ULP[dtype] + 21 * U) * kept).all()


def test_what_is_left_out_counts_for_nothing(device):
    """Rows, weights and gradients of pairs left out may hold anything; a NaN row of a kept pair
    reaches its own token only."""
    print("left out", flush=True)
    rng = np.random.default_rng(11)
    nan, inf = float("nan"), float("inf")
    for cols in (40, 2048):
        ids, experts, y, weights, _, dout = _combine_case(rng, 50, 4, cols, F16, device, 0.4)
        ids[7] = -1  # a token without any
        order = router.sort(torch.from_numpy(ids).to(device), experts)
        kept = int(order.offsets[-1])
        left = torch.from_numpy(_sorted(ids, experts)["slots"] >= kept).to(device)
        assert 0 < kept < 190
        y[kept:] = 0
        clean = weights.masked_fill(left, 0.0)
        want = router.combine(y, clean, order)
        dirty_y, dirty_w = y.clone(), weights.masked_fill(left, nan)
        dirty_y[kept::2], dirty_y[kept + 1::2] = nan, inf
        leaves = [dirty_y.requires_grad_(), dirty_w.requires_grad_()]
        got = router.combine(*leaves, order)
        assert torch.equal(got, want) and not got[7].any()
        dy, dw = torch.autograd.grad(got, leaves, dout)
        assert not dy[kept:].any() and not dw[left].any() and bool(dy.isfinite().all()) and bool(dw.isfinite().all())
        # the dispatch's gradient skips them too
        x = torch.zeros((50, cols), dtype=F16, device=device, requires_grad=True)
        rows, _ = router.dispatch(x, torch.from_numpy(ids).to(device), experts)
        (dx,) = torch.autograd.grad(rows, x, dirty_y.detach())
        assert bool(dx.isfinite().all()) and not dx[7].any()
        # a kept row of NaN
        slot, token = kept // 2, int(order.tokens[kept // 2])
        y[slot] = nan
        bad = router.combine(y, clean, order).isnan()
        assert bad[token].all() and int(bad.any(-1).sum()) == 1


def test_gradients_by_differences(device):
    """Both calls are linear in each operand: a difference of any size is the derivative."""
    print("differences", flush=True)
    rng = np.random.default_rng(12)
    tokens, k, cols, experts = 12, 3, 20, 5
    ids = torch.from_numpy(_ids(rng, tokens, k, experts, 0.0, 0.2)).to(device)

    def tensor(*shape):  # small whole numbers: every sum below is exact in f32
        return torch.from_numpy(rng.integers(-4, 5, shape).astype(np.float32)).to(device)

    x, w, add, dout = tensor(tokens, cols), tensor(tokens, k), tensor(tokens, cols), tensor(tokens, cols)

    def loss(x, w, add):
        rows, order = router.dispatch(x, ids, experts)
        return (router.combine(rows * 2, w, order, add=add) * dout).sum()

    leaves = [t.clone().requires_grad_() for t in (x, w, add)]
    grads = torch.autograd.grad(loss(*leaves), leaves)
    for i, g in enumerate(grads):
        step = tensor(*g.shape)
        moved = [t + step if j == i else t for j, t in enumerate((x, w, add))]
        assert float(loss(*moved) - loss(x, w, add)) == float((g * step).sum())


def test_second_derivatives_and_tangents_are_refused(device):
    print("dispatch second derivative", flush=True)
    ids = torch.tensor([[0, 1], [2, 0]], device=device)
    x = torch.randn((2, 8), device=device).requires_grad_()
    w = torch.randn((2, 2), device=device).requires_grad_()
    rows, order = router.dispatch(x, ids, 3)
    out = router.combine(rows, w, order)
    assert rows.grad_fn is not None and not order.slots.requires_grad
    for value, leaf in (((rows ** 2).sum(), x), (out.sum(), w), (out.sum(), x), ((out ** 2).sum(), w)):
        (grad,) = torch.autograd.grad(value, leaf, create_graph=True, retain_graph=True)
        with pytest.raises(RuntimeError, match="second time"):
            grad.sum().backward(retain_graph=True)
        (again,) = torch.autograd.grad(value, leaf, retain_graph=True)
        assert torch.equal(again, grad) and not again.requires_grad
    # of what is linear in x alone, the gradient is a constant
    (grad,) = torch.autograd.grad(rows.sum(), x, create_graph=True)
    assert not grad.requires_grad
    fwd = torch.autograd.forward_ad
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t.detach(), torch.ones_like(t))  # noqa: E731
        for call in (lambda: router.dispatch(dual(x), ids, 3), lambda: router.combine(dual(rows), w, order),
                     lambda: router.combine(rows, dual(w), order), lambda: router.combine(rows, w, order, add=dual(x))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()


def test_replayed_from_a_graph_and_on_another_stream(device):
    print("dispatch graph", flush=True)
    rng = np.random.default_rng(13)
    cases = [(tokens, torch.from_numpy(_ids(rng, tokens, 6, 64)).to(device),
              torch.from_numpy(rng.standard_normal((tokens, 264))).to(BF16).to(device),
              torch.from_numpy(rng.random((tokens, 6)).astype(np.float32)).to(device)) for tokens in (3, 3000)]
    for tokens, ids, x, w in cases:
        def step():
            rows, order = router.dispatch(x, ids, 64)
            return rows, router.combine(rows, w, order, add=x), *(getattr(order, n) for n in order.__slots__)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            held = step()
        for turn in range(4):
            ids.copy_(torch.from_numpy(_ids(rng, tokens, 6, 64, turn / 2)))
            x.add_(1)
            w.mul_(0.5)
            graph.replay()
            torch.cuda.synchronize()
            got = [h.clone() for h in held]
            assert all(torch.equal(g, v) for g, v in zip(got, step()))
            torch.cuda.synchronize()
        del eager


def test_gradients_under_capture_are_refused(device):
    """The nodes themselves, without the autograd engine."""
    print("dispatch gradients under capture", flush=True)
    ids = torch.tensor([[0, 1], [2, 0]], device=device)
    x = torch.randn((2, 8), device=device).requires_grad_()
    rows, order = router.dispatch(x, ids, 3)
    out = router.combine(rows, torch.ones((2, 2), device=device), order)
    above, z = (torch.ones_like(rows), torch.ones_like(out)), torch.zeros(8, device=device)
    with torch.no_grad():
        rows.grad_fn(above[0])
        out.grad_fn(above[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        z += 1
        with torch.no_grad():
            for node, grad in ((rows.grad_fn, above[0]), (out.grad_fn, above[1])):
                with pytest.raises(RuntimeError, match="captured"):
                    node(grad)
    for n in (1, 2):
        graph.replay()
        torch.cuda.synchronize()
        assert z.tolist() == [float(n)] * 8


def test_refusals(device):
    print("dispatch refusals", flush=True)
    z = lambda *s, dtype=F32: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    ids = z(3, 2, dtype=I32)
    for named, experts in ((ids.cpu(), 4), (z(3, 2), 4), (z(3, 2, dtype=torch.bool), 4), (ids, 0), (ids, 1025),
                           (z(3, 0, dtype=I32), 4), (z(3, 65, dtype=I32), 4), (ids[0, 0], 4), (None, 4),
                           (ids[:1, :1].expand(2 ** 30, 2), 4)):
        with pytest.raises(IqkKernelError):
            router.sort(named, experts)
    for x in (z(2, 8), z(3, 0), torch.zeros(3, 8), z(3, 8, dtype=torch.float64), z(3, 8, dtype=I32), None, z(8),
              z(3, 1)[:, :1].expand(3, 2 ** 28)):
        with pytest.raises(IqkKernelError):
            router.dispatch(x, ids, 4)
    order = router.sort(ids, 4)
    w, y = z(3, 2), z(6, 8)
    other = router.Order(order.offsets, order.ids, order.tokens, order.slots.long())
    host = router.Order(*(getattr(order, n).cpu() for n in order.__slots__))
    for args, add in (((y.cpu(), w, order), None), ((y, w.cpu(), order), None), ((y, ids, order), None),
                      ((y, z(3, 3), order), None), ((z(5, 8), w, order), None), ((y, w), None), ((z(3, 3, 8), w), None),
                      ((z(3, 2, 0), w), None), ((y, w, other), None), ((y, w, host), None), ((y, w, ids), None),
                      ((y, w, order), z(3, 9)), ((y, w, order), z(3, 8, dtype=F16)), ((y, w, order), torch.zeros(3, 8)),
                      ((y, w, order), z(2, 8)), ((y.long(), w, order), None), ((None, w), None), ((z(3, 65, 8), z(3, 65)), None)):
        with pytest.raises(IqkKernelError):
            router.combine(*args, add=add)


def test_an_order_without_offsets_is_refused(device):
    print("order without offsets", flush=True)
    order = router.sort(torch.zeros((3, 2), dtype=I32, device=device), 4)
    bare = router.Order(order.offsets[:0], order.ids, order.tokens, order.slots)
    with pytest.raises(IqkKernelError, match="offset"):
        router.combine(torch.zeros((6, 8), device=device), torch.ones((3, 2), device=device), bare)


def test_an_order_with_foreign_slots_reads_and_writes_nothing_outside(device):
    """Slots are bounded where they are used: what lies outside is skipped, as if left out."""
    print("foreign slots", flush=True)
    order = router.sort(torch.tensor([[0, 1], [2, 0]], device=device), 3)
    y = torch.ones((4, 8), device=device, requires_grad=True)
    bad = router.Order(order.offsets, order.ids, order.tokens,
                       torch.tensor([[-1, 2 ** 30], [4, 1]], dtype=I32, device=device))
    w = torch.ones((2, 2), device=device, requires_grad=True)
    out = router.combine(y, w, bad)
    assert out.detach().tolist() == [[0.0] * 8, [1.0] * 8]
    _, dw = torch.autograd.grad(out, (y, w), torch.ones_like(out))
    assert dw.tolist() == [[0.0, 0.0], [0.0, 8.0]]


def test_rows_past_32_bits(device):
    """More than 2^32 bytes and 2^31 values of rows, and their gradients."""
    print("rows past 2^32", flush=True)
    tokens, k, cols, experts = 2 ** 17 + 11, 3, 8192, 5
    g = torch.Generator(device=device).manual_seed(5)
    x = torch.empty((tokens, cols), dtype=BF16, device=device)
    for part in x.split(2 ** 14):
        part.copy_(torch.randint(-8, 9, part.shape, dtype=torch.int8, device=device, generator=g))
    ids = torch.randint(-1, experts, (tokens, k), dtype=I32, device=device, generator=g)
    rows, order = router.dispatch(x, ids, experts)
    assert rows.numel() > 2 ** 31
    kept = int(order.offsets[-1])
    for at in range(0, tokens * k, 2 ** 15):  # what each slot holds
        part, source = rows[at:at + 2 ** 15], x[order.tokens[at:at + 2 ** 15].long()]
        source[max(0, kept - at):] = 0
        assert torch.equal(part, source)
    weights = torch.randint(-3, 4, (tokens, k), device=device, generator=g).float().requires_grad_()
    rows.requires_grad_()
    out = router.combine(rows, weights, order)  # whole numbers of at most 72: exact
    factor = (weights.detach() * ((ids >= 0) & (ids < experts))).sum(-1, keepdim=True)
    for at in range(0, tokens, 2 ** 14):
        assert torch.equal(out.detach()[at:at + 2 ** 14].float(), factor[at:at + 2 ** 14] * x[at:at + 2 ** 14].float())
    dy, dw = torch.autograd.grad(out, (rows, weights), x)
    square = torch.empty(tokens, device=device)
    for at in range(0, tokens, 2 ** 14):
        square[at:at + 2 ** 14] = (x[at:at + 2 ** 14].float() ** 2).sum(-1)  # at most 2^19: exact
    assert torch.equal(dw, square[:, None] * ((ids >= 0) & (ids < experts)))
    flat = torch.empty(tokens * k, device=device)
    flat[order.slots.long().reshape(-1)] = weights.detach().reshape(-1)
    flat[kept:] = 0
    for at in range(0, tokens * k, 2 ** 15):  # whole numbers of at most 24
        want = flat[at:at + 2 ** 15, None] * x[order.tokens[at:at + 2 ** 15].long()].float()
        assert torch.equal(dy[at:at + 2 ** 15].float(), want)


def test_many_tokens(device):
    """More than 2^23 workgroups' tokens: a launch for each part of them."""
    print("many tokens", flush=True)
    tokens, cols = 2 ** 25 + 2 ** 20 + 5, 1
    g = torch.Generator(device=device).manual_seed(6)
    ids = torch.randint(0, 3, (tokens, 1), dtype=I32, device=device, generator=g)
    x = torch.randint(-100, 101, (tokens, cols), dtype=torch.int8, device=device, generator=g).to(F16)
    rows, order = router.dispatch(x, ids, 3)
    stable = torch.sort(ids.view(-1), stable=True)
    assert torch.equal(order.ids, stable.values) and torch.equal(order.tokens.long(), stable.indices)
    assert torch.equal(rows, x[stable.indices])
    w = torch.full((tokens, 1), 2.0, device=device, requires_grad=True)
    y = rows.detach().requires_grad_()
    out = router.combine(y, w, order)
    assert torch.equal(out.detach(), 2 * x)
    dy, dw = torch.autograd.grad(out, (y, w), x)
    assert torch.equal(dw, x.float() ** 2) and torch.equal(dy, 2 * rows)
    # parts of long rows
    x = torch.randint(-100, 101, (5, 2 ** 20 + 3), dtype=torch.int8, device=device, generator=g).to(F32)
    rows, order = router.dispatch(x, ids[:5].expand(5, 1).contiguous(), 3)
    assert torch.equal(rows, x[order.tokens.long()])
    assert torch.equal(router.combine(rows, w.detach()[:5].contiguous(), order), 2 * x)


# A layer as a server runs it and as a trainer does: the router's choice, 4-bit experts over
# sorted rows, the weighted sum.
@pytest.mark.parametrize("tokens", (1, 9, 300))
def test_a_layer_of_experts(device, tokens):
    print(f"layer of experts {tokens}", flush=True)
    torch.manual_seed(tokens)
    experts, n, k = 10, 128, 3
    proj = mx.MxSwitchLinear(experts, n, n, device=device)
    proj.load(mx.quantize(0.1 * torch.randn((experts, n, n), dtype=BF16, device=device)))
    x = torch.randn((tokens, n), dtype=BF16, device=device)
    logits = torch.randn((tokens, experts), device=device).requires_grad_()
    weights, ids = router.topk(logits, k)
    rows, order = router.dispatch(x, ids, experts)
    y = proj(rows[:, None], order.ids, sorted_indices=True)[:, 0]
    out = router.combine(y, weights, order, add=x)
    direct = proj(x[:, None, None], ids, sorted_indices=True)[:, :, 0]
    # the same products, whose sums may be in another order where other slots are beside them
    w64, values = _f64(proj.dequantized(F32)), _f64(x)
    named = ids.cpu().numpy()
    size = np.stack([np.abs(w64[named[:, j]]) @ np.abs(values)[..., None] for j in range(k)], 1)[..., 0]
    back = y[order.slots.long()]
    assert (np.abs(_f64(back) - _f64(direct)) <= 2 * (mxref.HALF_ULP[BF16] + 2 * n * U) * size).all()
    same = router.combine(back.contiguous(), weights, add=x)
    assert torch.equal(same, out)
    dout = torch.randn_like(out)
    (got,) = torch.autograd.grad(out, logits, dout, retain_graph=True)
    (want,) = torch.autograd.grad(same, logits, dout)
    assert torch.equal(got, want) and bool(got.any())


def test_trained_experts(device):
    """Experts of a caller's own between the two calls: every gradient against the whole layer's in float64."""
    print("trained experts", flush=True)
    torch.manual_seed(4)
    tokens, experts, n, k = 40, 6, 24, 2
    x, w = torch.randn((tokens, n), device=device), 0.3 * torch.randn((experts, n, n), device=device)
    logits, dout = torch.randn((tokens, experts), device=device), torch.randn((tokens, n), device=device)
    leaves = [t.requires_grad_() for t in (x, w, logits)]
    weights, ids = router.topk(logits, k)
    rows, order = router.dispatch(x, ids, experts)
    first = order.offsets.tolist()
    y = torch.cat([rows[first[e]:first[e + 1]] @ w[e].T for e in range(experts)])
    grads = torch.autograd.grad(router.combine(y, weights, order, add=x), leaves, dout)
    x64, w64, l64 = (t.detach().cpu().double().requires_grad_() for t in leaves)
    named = ids.cpu().long()
    gate = torch.softmax(torch.gather(l64, -1, named), -1)
    out = x64 + sum(gate[:, j, None] * (w64[named[:, j]] @ x64[..., None])[..., 0] for j in range(k))
    for got, want in zip(grads, torch.autograd.grad(out, (x64, w64, l64), dout.cpu().double())):
        # f32 throughout: sums of at most 24 to 80 terms of the size of the largest results
        assert float((got.cpu().double() - want).abs().max()) <= 100 * U * 8 * float(want.abs().max())


def test_rows_that_no_pair_has_get_zero_gradients(device):
    """Orders whose slots are no permutation: made by a caller, assigned, or changed in place (pairs dropped)."""
    print("rows without a pair", flush=True)
    experts, tokens, k = 7, 300, 3
    rng = np.random.default_rng(21)
    ids = torch.from_numpy(rng.integers(0, experts, (tokens, k))).to(device)
    for cols, dtype in ((8, F32), (2048, F16)):
        y = torch.from_numpy(rng.standard_normal((tokens * k, cols))).to(dtype).to(device).requires_grad_()
        w = torch.from_numpy(rng.random((tokens, k)).astype(np.float32)).to(device).requires_grad_()
        dout = torch.from_numpy(rng.standard_normal((tokens, cols))).to(dtype).to(device)
        whole = router.sort(ids, experts)
        want_dy, want_dw = torch.autograd.grad(router.combine(y, w, whole), (y, w), dout)
        drop = torch.from_numpy(rng.random((tokens, k)) < 0.4).to(device)
        kept = torch.ones(tokens * k, dtype=torch.bool, device=device)
        kept[whole.slots[drop].long()] = False
        lists = whole.offsets, whole.ids, whole.tokens
        made = router.Order(*lists, whole.slots.masked_fill(drop, -1))
        assigned = router.sort(ids, experts)
        assigned.slots = made.slots
        changed = router.sort(ids, experts)
        changed.slots.masked_fill_(drop, tokens * k)
        _, moved = router.dispatch(torch.zeros((tokens, 4), device=device), ids, experts)
        moved.slots[drop] = -1
        for order in (made, assigned, changed, moved, copy.copy(changed), copy.deepcopy(changed)):
            for _ in range(2):
                torch.full_like(y, float("nan"))  # what memory that is taken up again holds
                dy, dw = torch.autograd.grad(router.combine(y, w, order), (y, w), dout)
                assert torch.equal(dy[kept], want_dy[kept]) and not dy[~kept].any() and not dy.isnan().any()
                assert torch.equal(dw, want_dw.masked_fill(drop, 0.0))
        for order in (whole, copy.copy(whole), copy.deepcopy(whole)):
            got = torch.autograd.grad(router.combine(y, w, order), (y, w), dout)
            assert torch.equal(got[0], want_dy) and torch.equal(got[1], want_dw)


def test_an_orders_foreign_slots_leave_zero_gradients(device):
    print("foreign slots' gradients", flush=True)
    order = router.sort(torch.tensor([[0, 1], [2, 0]], device=device), 3)
    y = torch.ones((4, 8), device=device, requires_grad=True)
    bad = router.Order(order.offsets, order.ids, order.tokens,
                       torch.tensor([[-1, 2 ** 30], [4, 1]], dtype=I32, device=device))
    torch.full((4, 8), float("nan"), device=device)
    (dy,) = torch.autograd.grad(router.combine(y, torch.ones((2, 2), device=device), bad), y, torch.ones((2, 8), device=device))
    assert dy.tolist() == [[0.0] * 8, [1.0] * 8, [0.0] * 8, [0.0] * 8]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens,k,cols,spread", ((1, 1, 8, 1), (3, 2, 7, 2), (40, 5, 64, 9), (300, 3, 1030, 200), (700, 6, 33, 4), (64, 64, 8, 1),
                                                  (500, 4, 4100, 1500)))
def test_a_row_of_several_pairs_gets_the_sum_of_their_gradients(device, dtype, tokens, k, cols, spread):
    """A caller's order in which pairs share rows (tokens alike, say), some rows without a pair, some pairs left out."""
    print(f"shared rows {dtype} {tokens} {k} {cols} {spread}", flush=True)
    rng = np.random.default_rng(tokens + cols)
    pairs = tokens * k
    slots = rng.integers(0, min(spread, pairs), (tokens, k))
    slots[rng.random((tokens, k)) < 0.1] = -1
    kept = max(1, min(spread, pairs) - 1)  # the last of these are left out
    order = router.Order(torch.tensor([0, kept], dtype=I32, device=device), *(torch.zeros(pairs, dtype=I32, device=device),) * 2,
                         torch.from_numpy(slots).to(device, I32))
    y = torch.from_numpy(rng.standard_normal((pairs, cols))).to(dtype).to(device).requires_grad_()
    w = torch.from_numpy(rng.standard_normal((tokens, k)).astype(np.float32)).to(device).requires_grad_()
    dout = torch.from_numpy(rng.standard_normal((tokens, cols))).to(dtype).to(device)
    out = router.combine(y, w, order)
    dy, dw = torch.autograd.grad(out, (y, w), dout)
    w64, d64, y64 = _f64(w), _f64(dout), _f64(y)
    live = (slots >= 0) & (slots < kept)
    want, size = np.zeros((pairs, cols)), np.zeros((pairs, cols))
    for t, j in zip(*np.nonzero(live)):
        want[slots[t, j]] += w64[t, j] * d64[t]
        size[slots[t, j]] += np.abs(w64[t, j] * d64[t])
    most = int(np.bincount(slots[live], minlength=1).max()) if live.any() else 1
    # so many fused additions in f32, half a step of the sum each; one rounding
    error = most * U * size
    assert (np.abs(_f64(dy) - want) <= error + _rounded(dtype) * (np.abs(want) + error) + mxref.TINY[dtype]).all()
    sums = np.where(live[..., None], w64[..., None] * y64[np.where(live, slots, 0)], 0.0)
    error = k * U * np.abs(sums).sum(1)
    assert (np.abs(_f64(out) - sums.sum(1)) <= error + _rounded(dtype) * (np.abs(sums.sum(1)) + error) + mxref.TINY[dtype]).all()
    dots = np.where(live[..., None], d64[:, None] * y64[np.where(live, slots, 0)], 0.0)
    assert (np.abs(_f64(dw) - dots.sum(-1)) <= cols * U * np.abs(dots).sum(-1) + 2.0 ** -140).all()
    again = torch.autograd.grad(router.combine(y, w, order), (y,), dout)[0]
    assert torch.equal(again, dy)
