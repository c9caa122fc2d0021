"""Low-rank adapters of many requests, against plain 64-bit forms on the CPU."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mxref
from mlx_iqk_amd import mx
from mlx_iqk_amd.adapters import LowRankAdapters
from mlx_iqk_amd.kernels import IqkKernelError
from mlx_iqk_amd.nn import IqkRuntimeError

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = (F16, BF16)
U = 2.0 ** -24


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().to(torch.float64).numpy()


def _bank(rng, adapters, out, n, rank, dtype, device, ranks=None):
    bank = LowRankAdapters(adapters, out, n, rank, dtype=dtype, device=device)
    for a in range(adapters):
        r = rank if ranks is None else ranks[a % len(ranks)]
        bank.load(a, torch.from_numpy(rng.standard_normal((r, n)) * n ** -0.5).to(dtype),
                  torch.from_numpy(rng.standard_normal((out, r)) * r ** -0.5).to(dtype), 2.0 - a / adapters)
    return bank


def _rows(rng, rows, n, dtype, device):
    return torch.from_numpy(rng.standard_normal((rows, n))).to(dtype).to(device)


def _check(got, bank, x, ids, y, dtype):
    """got against float64, row by row; ids one a row."""
    down, up, scales = (np.stack(parts) for parts in zip(*(
        (_f64(down), _f64(up), scale) for down, up, scale in map(bank.adapter, range(bank.num_adapters)))))
    x, y, got = _f64(x), _f64(y), _f64(got)
    n, rank = down.shape[2], down.shape[1]
    for a in sorted(set(ids.tolist())):
        rows = np.nonzero(ids == a)[0]
        if a == -1:
            np.testing.assert_array_equal(got[rows], y[rows])
            continue
        if not 0 <= a < len(down):
            assert np.isnan(got[rows]).all()
            continue
        t, t_size = x[rows] @ down[a].T * scales[a], np.abs(x[rows]) @ np.abs(down[a]).T * abs(scales[a])
        want, size = y[rows] + t @ up[a].T, np.abs(y[rows]) + np.abs(t) @ np.abs(up[a]).T
        # exact products, n and then rank + 1 of them summed in f32 in any order, at most a
        # step off each (matrix cores may truncate); the scale's product; one rounding
        error = ((2 * n + 2) * U * t_size) @ np.abs(up[a]).T + (2 * rank + 4) * U * size
        bound = error + mxref.HALF_ULP[dtype] * (np.abs(want) + error) + mxref.TINY[dtype]
        assert (np.abs(got[rows] - want) <= bound).all(), (a, np.max(np.abs(got[rows] - want) / bound))


# rows, adapters, rank, out, in: one row, few and many; ranks that are no multiple of 8, outputs of any count
SHAPES = ((1, 1, 1, 1, 8), (1, 8, 16, 1024, 512), (2, 3, 8, 100, 64), (5, 5, 20, 77, 264), (16, 4, 64, 512, 128),
          (33, 40, 16, 257, 96), (64, 2, 4, 1001, 72), (65, 7, 24, 130, 1000), (150, 9, 20, 333, 1440), (300, 3, 128, 64, 200),
          (257, 64, 16, 96, 256), (1000, 1, 256, 48, 136), (2100, 30, 32, 200, 104))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,adapters,rank,out,n", SHAPES)
def test_adapters(device, dtype, rows, adapters, rank, out, n):
    print(f"adapters {dtype} {rows} {adapters} {rank} {out} {n}", flush=True)
    rng = np.random.default_rng(rows + rank)
    bank = _bank(rng, adapters, out, n, rank, dtype, device)
    x, y = _rows(rng, rows, n, dtype, device), _rows(rng, rows, out, dtype, device)
    keep = x.clone(), y.clone()
    runs = np.sort(rng.integers(0, adapters, rows))
    for ids in (rng.integers(0, adapters, rows), runs, rng.integers(-1, adapters, rows), np.full(rows, adapters - 1),
                rng.choice((-1, -2, 0, adapters, 2 ** 31 - 1, -2 ** 31), rows)):
        named = torch.from_numpy(ids).to(device)
        got = bank(x, named, y)
        assert got.dtype == dtype and got.shape == y.shape
        _check(got, bank, x, ids, y, dtype)
        assert torch.equal(bank(x, named.to(torch.int32), y).view(torch.int16), got.view(torch.int16))
    assert torch.equal(x, keep[0]) and torch.equal(y, keep[1])


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows", (3, 200))
def test_adapters_of_several_ranks(device, dtype, rows):
    """Smaller ranks than the bank's, also after a larger one in the same place; adapters not loaded add nothing."""
    print(f"adapter ranks {dtype} {rows}", flush=True)
    rng = np.random.default_rng(rows)
    bank = _bank(rng, 6, 120, 80, 40, dtype, device)
    for a, r in ((1, 1), (2, 39), (4, 8)):
        bank.load(a, torch.from_numpy(rng.standard_normal((r, 80))).to(dtype),
                  torch.from_numpy(rng.standard_normal((120, r))).to(dtype), -0.5)
        down, up, scale = bank.adapter(a)
        assert not down[r:].any() and not up[:, r:].any() and scale == -0.5
    x, y = _rows(rng, rows, 80, dtype, device), _rows(rng, rows, 120, dtype, device)
    ids = rng.integers(0, 6, rows)
    _check(bank(x, torch.from_numpy(ids).to(device), y), bank, x, ids, y, dtype)
    empty = LowRankAdapters(2, 120, 80, 5, dtype=dtype, device=device)
    assert torch.equal(empty(x, torch.ones(rows, dtype=torch.int32, device=device), y), y)


@pytest.mark.parametrize("rows", (2, 90))
def test_ids_of_requests(device, rows):
    """An id for all rows of a request, of several leading axes; 64-bit ids past 32 bits are outside."""
    print(f"ids of requests {rows}", flush=True)
    rng = np.random.default_rng(rows)
    bank = _bank(rng, 3, 72, 64, 8, BF16, device)
    x, y = _rows(rng, 4 * rows, 64, BF16, device).view(2, 2, rows, 64), _rows(rng, 4 * rows, 72, BF16, device).view(2, 2, rows, 72)
    ids = np.array([[0, 2], [-1, 1]])
    named = torch.from_numpy(ids).to(device)
    want = bank(x, named[..., None].expand(2, 2, rows), y)
    _check(want.view(-1, 72), bank, x.view(-1, 64), np.repeat(ids.reshape(-1), rows), y.view(-1, 72), BF16)
    assert torch.equal(bank(x, named[..., None], y), want)
    assert torch.equal(bank(x, named[..., None].to(torch.int16), y), want)
    assert torch.equal(bank(x[0, 0], named[0, :1], y[0, 0]), bank(x[0, 0], named[0, 0].expand(rows), y[0, 0]))
    one = bank(x[0, 0, 0], named[0, 1], y[0, 0, 0])  # a row without a leading axis
    _check(one[None], bank, x[0, 0, :1], ids[0, 1:], y[0, 0, :1], BF16)
    wide = torch.tensor([2 ** 32, 2 ** 32 - 1, -2 ** 32 + 1, -1], device=device)[:, None]
    got = bank(x.view(4, rows, 64), wide, y.view(4, rows, 72))
    assert got[:3].isnan().all() and torch.equal(got[3], y[1, 1])


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows", (1, 7, 140))
def test_any_address_and_stride(device, dtype, rows):
    print(f"adapter addresses {dtype} {rows}", flush=True)
    rng = np.random.default_rng(rows)
    bank = _bank(rng, 4, 123, 88, 12, dtype, device)
    x, y = _rows(rng, rows, 88, dtype, device), _rows(rng, rows, 123, dtype, device)
    ids = torch.from_numpy(rng.integers(0, 4, rows)).to(device)
    want = bank(x, ids, y)
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=device)[1:].view(t.shape).copy_(t) for t in (x, ids, y)]
    assert torch.equal(bank(*odd), want)
    turned = [t.transpose(0, -1).contiguous().transpose(0, -1) for t in (x, ids.repeat(2, 1).T[:, 0], y)]
    assert torch.equal(bank(*turned), want)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows", (4, 130))
def test_bad_rows_stay_where_they_are(device, dtype, rows):
    """A row of x or y with NaN or infinities, and an adapter that holds them, reach their own rows only."""
    print(f"adapter bad rows {dtype} {rows}", flush=True)
    rng = np.random.default_rng(rows)
    bank = _bank(rng, 4, 90, 64, 20, dtype, device)
    x, y = _rows(rng, rows, 64, dtype, device), _rows(rng, rows, 90, dtype, device)
    ids = rng.integers(0, 4, rows)
    ids[:4] = (0, 1, 2, 0)
    named = torch.from_numpy(ids).to(device)
    want = bank(x, named, y)
    nan, inf = float("nan"), float("inf")
    bad_x, bad_y = x.clone(), y.clone()
    bad_x[1, 3], bad_x[3] = nan, inf
    bad_y[2, 5] = nan
    got = bank(bad_x, named, bad_y)
    assert got[1].isnan().all() and not got[3].isfinite().any() and bool(got[2, 5].isnan())
    got[2, 5] = want[2, 5]
    rest = [r for r in range(rows) if r not in (1, 3)]
    assert torch.equal(got[rest], want[rest])
    bank.down[3, 0, 0, 0] = nan
    bank.up[3, 1, 7, 2] = inf
    got = bank(x, named, y)
    others = torch.from_numpy(ids != 3).to(device)
    assert torch.equal(got[others], want[others]) and bool(got[~others].isnan().all())


@pytest.mark.parametrize("rows", (6, 100))
def test_large_and_small_values(device, rows):
    """A x far outside f16, and far below it, in f16 as in bf16: it stays f32."""
    print(f"adapter ranges {rows}", flush=True)
    rng = np.random.default_rng(rows)
    for dtype, big in ((F16, 2.0 ** 9), (BF16, 2.0 ** 40)):
        for factor, back in ((big, 1 / big ** 2), (1 / big, big)):
            bank = LowRankAdapters(2, 80, 64, 16, dtype=dtype, device=device)
            for a in range(2):
                bank.load(a, torch.from_numpy(rng.standard_normal((16, 64)) * factor),
                          torch.from_numpy(rng.standard_normal((80, 16))), back)
            x = _rows(rng, rows, 64, dtype, device) * factor
            y = torch.zeros((rows, 80), dtype=dtype, device=device)
            ids = rng.integers(0, 2, rows)
            _check(bank(x, torch.from_numpy(ids).to(device), y), bank, x, ids, y, dtype)


def test_no_rows(device):
    print("no rows", flush=True)
    bank = LowRankAdapters(2, 80, 64, 16, device=device)
    y = bank(torch.empty((0, 64), dtype=BF16, device=device), torch.empty(0, dtype=torch.int32, device=device),
             torch.empty((0, 80), dtype=BF16, device=device))
    assert y.shape == (0, 80)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows", (1, 24, 200))
def test_beside_a_4_bit_projection(device, dtype, rows):
    """``MxLinear``'s call with adapters is the two calls, bit for bit."""
    print(f"beside MxLinear {dtype} {rows}", flush=True)
    rng = np.random.default_rng(rows)
    n, out = 160, 200
    proj = mx.MxLinear(out, n, device=device)
    proj.load(mx.quantize(torch.from_numpy(0.05 * rng.standard_normal((out, n))).to(dtype).to(device)))
    bank = _bank(rng, 5, out, n, 16, dtype, device)
    x = _rows(rng, rows, n, dtype, device)
    ids = rng.integers(-1, 5, rows)
    named = torch.from_numpy(ids).to(device)
    plain = proj(x)
    got = proj(x, bank, named)
    assert torch.equal(got, bank(x, named, plain)) and torch.equal(proj(x), plain)
    _check(got, bank, x, ids, plain, dtype)
    assert torch.equal(proj(x, adapters=bank, adapter_ids=torch.full_like(named, -1)), plain)
    q = mx.quantize(x)
    with pytest.raises(IqkRuntimeError, match="16-bit activations"):
        proj(q, bank, named)
    both = bank(x, named, proj(q))
    _check(both, bank, x, ids, proj(q), dtype)
    for other in (LowRankAdapters(5, out, n + 32, 16, dtype=dtype, device=device),
                  LowRankAdapters(5, out + 1, n, 16, dtype=dtype, device=device), object()):
        with pytest.raises(IqkRuntimeError):
            proj(x, other, named)
    with pytest.raises(IqkKernelError):
        proj(x, bank)


@pytest.mark.parametrize("rows", (1, 40, 700))
def test_replayed_from_a_graph_and_on_another_stream(device, rows):
    print(f"adapters graph {rows}", flush=True)
    rng = np.random.default_rng(rows)
    bank = _bank(rng, 9, 264, 128, 16, BF16, device)
    x, y = _rows(rng, rows, 128, BF16, device), _rows(rng, rows, 264, BF16, device)
    ids = torch.from_numpy(rng.integers(-1, 9, rows)).to(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = bank(x, ids, y)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, bank(x, ids, y))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = bank(x, ids, y)
        twice = bank(x, ids, held)  # a second call in one graph
    for turn in range(4):
        ids.copy_(torch.from_numpy(rng.integers(-1, 9, rows)))
        x.add_(0.5)
        bank.load(turn, torch.from_numpy(rng.standard_normal((16, 128)) * 0.1), torch.from_numpy(rng.standard_normal((264, 16))))
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone(), twice.clone()
        want = bank(x, ids, y)
        assert torch.equal(got[0], want) and torch.equal(got[1], bank(x, ids, want))
        torch.cuda.synchronize()


def test_outputs_past_32_bits(device):
    """More than 2^31 outputs, and 2^32 bytes of x; whole numbers, so that every sum is exact."""
    print("adapters past 2^31", flush=True)
    rows, n, out = 2 ** 18 + 9, 8192, 8200
    g = torch.Generator(device=device).manual_seed(3)
    bank = LowRankAdapters(3, out, n, 8, dtype=BF16, device=device)
    for a in range(3):
        down, up = torch.zeros((8, n)), torch.zeros((out, 8))
        down[torch.arange(8), torch.arange(8) * (n // 8) + a] = 1.0  # picks eight columns
        up[torch.arange(out), torch.arange(out) % 8] = float(a + 1)
        bank.load(a, down, up, 1.0)
    x = torch.zeros((rows, n), dtype=BF16, device=device)
    ids = torch.randint(-1, 3, (rows,), dtype=torch.int32, device=device, generator=g)
    column = torch.arange(8, device=device) * (n // 8)
    picks = torch.randint(-8, 9, (rows, 8), device=device, generator=g)
    for a in range(3):
        x[:, column + a] = (picks + a).to(BF16)
    y = torch.ones((rows, out), dtype=BF16, device=device)
    assert y.numel() > 2 ** 31 and x.numel() * 2 > 2 ** 32
    got = bank(x, ids, y)
    for at in range(0, rows, 2 ** 14):
        a = ids[at:at + 2 ** 14]
        eight = torch.where(a[:, None] < 0, 0, (picks[at:at + 2 ** 14] + a[:, None]) * (a[:, None] + 1))
        want = 1 + eight[:, torch.arange(out, device=device) % 8]
        assert torch.equal(got[at:at + 2 ** 14].long(), want)


def test_state_dict(device):
    print("adapters state", flush=True)
    rng = np.random.default_rng(2)
    bank = _bank(rng, 3, 40, 32, 10, F16, device)
    other = LowRankAdapters(3, 40, 32, 10, dtype=F16, device=device)
    other.load_state_dict(bank.state_dict())
    x, y = _rows(rng, 5, 32, F16, device), _rows(rng, 5, 40, F16, device)
    ids = torch.tensor([0, 1, 2, -1, 1], device=device)
    assert torch.equal(other(x, ids, y), bank(x, ids, y))


def test_refusals(device):
    print("adapter refusals", flush=True)
    z = lambda *s, dtype=BF16: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    bank = LowRankAdapters(4, 48, 32, 8, device=device)
    ids, x, y = z(3, dtype=torch.int32), z(3, 32), z(3, 48)
    for args in ((x.cpu(), ids, y), (x, ids.cpu(), y), (x, ids, y.cpu()), (x.half(), ids, y), (x, ids, y.float()),
                 (x, ids.float(), y), (x, ids.bool(), y), (None, ids, y), (x, None, y), (x, ids, None), (z()[None][0], ids, y)):
        with pytest.raises(IqkKernelError):
            bank(*args)
    for args in ((z(3, 40), ids, y), (x, ids, z(3, 40)), (x, ids[:2], y), (x, ids, z(2, 48)), (x, ids[None], y),
                 (z(2, 3, 32), ids, z(2, 3, 48)), (z(2, 3, 32), ids[None], z(2, 3, 48)), (x, ids[0], y)):
        with pytest.raises(IqkRuntimeError):
            bank(*args)
    for args in ((x.clone().requires_grad_(), ids, y), (x, ids, y.clone().requires_grad_())):
        with pytest.raises(IqkRuntimeError, match="no gradient"):
            bank(*args)
        with torch.no_grad():
            assert torch.equal(bank(*args), y)
    fwd = torch.autograd.forward_ad
    with fwd.dual_level():
        for args in ((fwd.make_dual(x, torch.ones_like(x)), ids, y), (x, ids, fwd.make_dual(y, torch.ones_like(y)))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                bank(*args)
    with pytest.raises(IqkKernelError):
        LowRankAdapters(4, 48, 32, 8)(x, ids, y)  # a bank on the host
    with pytest.raises(IqkKernelError):
        LowRankAdapters(4, 48, 32, 8, device=device).half()(x.half(), ids, y.half())  # scales in 16 bits


# rows sorted by adapter: banks of many adapters with a row or two each, one for all, none; columns
# that do not divide among the parts; every count of ranks that has a form of its own, and its neighbours
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,adapters,rank,out,n", (
    (3000, 1024, 8, 40, 64), (1100, 1000, 16, 24, 72), (2500, 1, 17, 300, 4104), (1600, 2, 33, 1030, 1032), (1100, 5, 65, 264, 520),
    (1090, 3, 72, 1025, 2056), (1200, 4, 129, 90, 1160), (1050, 2, 200, 513, 4096), (5000, 13, 40, 256, 256), (1030, 64, 64, 2048, 512)))
def test_sorted_rows(device, dtype, rows, adapters, rank, out, n):
    print(f"sorted rows {dtype} {rows} {adapters} {rank} {out} {n}", flush=True)
    rng = np.random.default_rng(rows + rank)
    bank = _bank(rng, min(adapters, 8), out, n, rank, dtype, device) if adapters <= 8 else None
    if bank is None:  # a large bank, filled at once
        bank = LowRankAdapters(adapters, out, n, rank, dtype=dtype, device=device)
        g = torch.Generator(device=device).manual_seed(rows)
        bank.down.normal_(0, n ** -0.5, generator=g)
        bank.up.normal_(0, rank ** -0.5, generator=g)
        bank.scales.uniform_(0.5, 2.0, generator=g)
    x, y = _rows(rng, rows, n, dtype, device), _rows(rng, rows, out, dtype, device)
    kinds = (rng.integers(-1, adapters, rows), np.sort(rng.integers(0, adapters, rows)), np.full(rows, -1),
             np.where(rng.random(rows) < 0.02, rng.integers(0, adapters, rows), -1))
    for ids in kinds if adapters <= 64 else kinds[:1] + kinds[2:]:
        named = torch.from_numpy(ids).to(device)
        got = bank(x, named, y)
        _check(got, bank, x, ids, y, dtype)
        assert torch.equal(bank(x, named, y), got)  # again, bit for bit


def test_hooks_and_other_forwards_run_beside_a_projection(device):
    print("adapters' hooks", flush=True)
    rng = np.random.default_rng(8)
    proj = mx.MxLinear(64, 96, device=device)
    proj.load(mx.quantize(torch.from_numpy(0.05 * rng.standard_normal((64, 96))).to(BF16).to(device)))
    bank = _bank(rng, 3, 64, 96, 8, BF16, device)
    x, ids = _rows(rng, 5, 96, BF16, device), torch.tensor([0, 1, -1, 2, 1], device=device)
    plain = proj(x)
    want = bank(x, ids, plain)
    seen = []

    def before(module, args):
        seen.append([t.clone() for t in args])

    def after(module, args, out):
        seen.append(out)
        return out * 2

    handles = [bank.register_forward_pre_hook(before), bank.register_forward_hook(after)]
    assert torch.equal(proj(x, bank, ids), want * 2)
    assert len(seen) == 2 and all(torch.equal(a, b) for a, b in zip(seen[0], (x, ids, plain))) and torch.equal(seen[1], want)
    for handle in handles:
        handle.remove()
    assert torch.equal(proj(x, bank, ids), want) and len(seen) == 2
    calls = []
    handle = torch.nn.modules.module.register_module_forward_hook(lambda module, args, out: calls.append(module))
    try:
        assert torch.equal(proj(x, bank, ids), want)
    finally:
        handle.remove()
    assert any(m is bank for m in calls)

    class Doubled(LowRankAdapters):
        def forward(self, x, ids, y):
            return super().forward(x, ids, y) * 2

    other = Doubled(3, 64, 96, 8, device=device)
    other.load_state_dict(bank.state_dict())
    assert torch.equal(proj(x, other, ids), want * 2)
    bank.forward = lambda x, ids, y: y * 3
    assert torch.equal(proj(x, bank, ids), plain * 3)


@pytest.mark.parametrize("dtype", (torch.uint8, torch.int8, torch.int16, torch.uint16, torch.uint32, torch.uint64))
def test_ids_of_any_integer_type(device, dtype):
    """-1 where the type has it; its largest value lies outside the bank."""
    print(f"ids of {dtype}", flush=True)
    rng = np.random.default_rng(9)
    bank = _bank(rng, 3, 40, 32, 8, F16, device)
    x, y = _rows(rng, 4, 32, F16, device), _rows(rng, 4, 40, F16, device)
    info = torch.iinfo(dtype)
    ids = np.array([2, 0, info.max, -1 if info.min < 0 else info.max - 1], dtype=str(dtype).split(".")[1])
    got = bank(x, torch.from_numpy(ids).to(device), y)
    _check(got[:2], bank, x[:2], np.array([2, 0]), y[:2], F16)
    assert bool(got[2].isnan().all())
    assert torch.equal(got[3], y[3]) if info.min < 0 else bool(got[3].isnan().all())
