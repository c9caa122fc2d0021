"""Low-rank adapters of rows in tiles, sorted by adapter, against float64.  Each case asserts which of the two
forms it takes, rows alone or tiles, so that a change of the rule between them takes no tests from either."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mxref
from mlx_iqk_amd import _native, mx
from mlx_iqk_amd.adapters import LowRankAdapters

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
HALF = (F16, BF16)
U = 2.0 ** -24


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().to(torch.float64).numpy()


def _words(bank: LowRankAdapters, rows: int) -> int:
    """The workspace of a call: 0 where each row is computed alone."""
    return _native.load().iqk_adapters_work(bank.in_features, bank.out_features, bank.down.shape[2], bank.num_adapters, rows)


def _check(got, bank, x, ids, y, dtype):
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
        # rank by rank: n exact products summed in f32 in any order, at most a step (2 U) off each (matrix cores
        # may truncate), the scale's product, and a rounding where f16's pieces stand for it; rank + 1 sums; one rounding
        error = ((2 * n + 4) * U * t_size) @ np.abs(up[a]).T + (2 * rank + 4) * U * size
        bound = error + mxref.HALF_ULP[dtype] * (np.abs(want) + error) + mxref.TINY[dtype]
        assert (np.abs(got[rows] - want) <= bound).all(), (a, np.max(np.abs(got[rows] - want) / bound))


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("small", (-8, -16))
@pytest.mark.parametrize("rank", (8, 20, 33, 72, 200))
@pytest.mark.parametrize("rows", (5, 4300))
def test_ranks_far_apart(device, dtype, small, rank, rows):
    """Ranks 2^36 and 2^50 below a row's largest count at the outputs that do not take the largest ones, in rows and
    in tiles; rows without the large ones lie in the same tiles."""
    print(f"ranks far apart {dtype} {small} {rank} {rows}", flush=True)
    rng = np.random.default_rng(rank)
    n, out, half = 64, 72, 32

    def normal(*shape):
        return torch.from_numpy(rng.standard_normal(shape))

    bank = LowRankAdapters(3, out, n, rank, dtype=dtype, device=device)
    for a in range(3):
        down, up = torch.zeros((rank, n), dtype=torch.float64), torch.zeros((out, rank), dtype=torch.float64)
        down[0::2, :half] = normal(*down[0::2, :half].shape) * 2.0 ** 6
        down[1::2, half:] = normal(*down[1::2, half:].shape) * 2.0 ** small
        up[0::2, 1::2] = normal(*up[0::2, 1::2].shape) * 2.0 ** 13
        up[1::2, 0::2] = normal(*up[1::2, 0::2].shape) * 2.0 ** -13
        bank.load(a, down, up, 1.0 - a / 4)
    x = normal(rows, n)
    x[:, :half] *= 2.0 ** 10 * torch.from_numpy(rng.random((rows, 1)) < (0.7 if rows < 64 else 0.05))
    x[:, half:] *= 2.0 ** (small - 2)
    x, y = x.to(dtype).to(device), torch.zeros((rows, out), dtype=dtype, device=device)
    ids = rng.integers(0, 3, rows)
    assert (_words(bank, rows) > 0) == (rows > 64)
    got = bank(x, torch.from_numpy(ids).to(device), y)
    _check(got, bank, x, ids, y, dtype)
    assert bool(got[:, 0::2].any())


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rank", (2, 40, 200))
@pytest.mark.parametrize("rows", (3, 4300))
def test_an_infinity_beside_large_ranks(device, dtype, rank, rows):
    """A scaled sum past f32 is an infinity, and finite sums past f16 beside it stay finite."""
    print(f"infinity beside large ranks {dtype} {rank} {rows}", flush=True)
    bank = LowRankAdapters(1, 24, 16, rank, dtype=dtype, device=device)
    down, up = torch.zeros((rank, 16)), torch.zeros((24, rank))
    down[0, 0], down[1, 1] = 1.0, 2.0 ** -14
    up[0::3, 0], up[1::3, 0], up[2::3, 0] = 1.0, -1.0, 0.5
    up[:, 1] = torch.arange(24) % 2 * 2.0 - 1
    bank.load(0, down, up, 2.0 ** 126)
    x = torch.zeros((rows, 16), dtype=dtype, device=device)
    x[:, 0], x[:, 1] = 8.0, 2.0 ** -10  # 2^129 and 2^102 when scaled
    x[2::3, 0] = 0.0  # rows without the infinity
    y = torch.ones((rows, 24), dtype=dtype, device=device)
    assert (_words(bank, rows) > 0) == (rows > 64)
    got = _f64(bank(x, torch.zeros(rows, dtype=torch.int32, device=device), y))
    want = np.sign(_f64(up[:, 0])) * np.inf
    rest = np.sign(_f64(up[:, 1])) * (np.inf if dtype == F16 else 2.0 ** 102)
    for r in range(rows):
        np.testing.assert_array_equal(got[r], rest if r % 3 == 2 else want)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rank,at", ((2, 1), (40, 33), (72, 70), (128, 127), (200, 150), (256, 64)))
@pytest.mark.parametrize("rows", (3, 4300))
def test_an_infinity_behind_large_ranks(device, dtype, rank, at, rows):
    """Finite sums near f32's end in the ranks before an infinity do not become infinities of their own."""
    print(f"infinity behind large ranks {dtype} {rank} {at} {rows}", flush=True)
    bank = LowRankAdapters(1, 24, 16, rank, dtype=dtype, device=device)
    down, up = torch.zeros((rank, 16)), torch.zeros((24, rank))
    down[0, 0], down[at, 1] = 2.0 ** -6, 1.0
    up[:, 0] = 1.0
    up[:, at] = torch.arange(24) % 2 * 2.0 - 1
    bank.load(0, down, up, 2.0 ** 126)
    x = torch.zeros((rows, 16), dtype=dtype, device=device)
    x[:, 0], x[:, 1] = 2.0 ** -4, 8.0  # 2^116 and 2^129 when scaled
    assert (_words(bank, rows) > 0) == (rows > 64)
    got = _f64(bank(x, torch.zeros(rows, dtype=torch.int32, device=device), torch.ones((rows, 24), dtype=dtype, device=device)))
    np.testing.assert_array_equal(got, np.broadcast_to(np.sign(_f64(up[:, at])) * np.inf, got.shape))


def _normal(rng, *shape):
    return torch.from_numpy(rng.standard_normal(shape))


def _bank(rng, adapters, out, n, rank, dtype, device, ranks=None):
    bank = LowRankAdapters(adapters, out, n, rank, dtype=dtype, device=device)
    for a in range(adapters):
        r = rank if ranks is None else ranks[a % len(ranks)]
        bank.load(a, _normal(rng, r, n) * n ** -0.5, _normal(rng, out, r) * r ** -0.5, 2.0 - a / adapters)
    return bank


def _rows(rng, rows, n, dtype, device):
    return _normal(rng, rows, n).to(dtype).to(device)


# few rows alone, and as many as fill tiles; outputs of several turns of a workgroup, and a part of one
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,out,n,rank", ((4, 90, 64, 20), (1300, 90, 64, 20), (1300, 1300, 72, 40), (1100, 600, 136, 130)))
def test_bad_rows_stay_where_they_are(device, dtype, rows, out, n, rank):
    """NaN and infinities in a row of x or y, or in an adapter, reach their own rows only, whatever their tile holds."""
    print(f"bad rows in tiles {dtype} {rows} {out} {n} {rank}", flush=True)
    rng = np.random.default_rng(rows + rank)
    bank = _bank(rng, 4, out, n, rank, dtype, device)
    assert (_words(bank, rows) > 0) == (rows > 4)
    x, y = _rows(rng, rows, n, dtype, device), _rows(rng, rows, out, dtype, device)
    ids = rng.integers(0, 4, rows)
    ids[:4] = (0, 1, 2, 0)
    named = torch.from_numpy(ids).to(device)
    want = bank(x, named, y)
    nan, inf = float("nan"), float("inf")
    bad_x, bad_y = x.clone(), y.clone()
    at = range(0, rows, 4)  # one in four of every tile: 1 a row of NaN, 2 of infinities, 3 a y, 0 none
    for i in at:
        bad_x[i + 1, 3], bad_x[i + 2], bad_y[i + 3, 5] = nan, inf, -inf
    got = bank(bad_x, named, bad_y)
    assert got[1::4].isnan().all() and not got[2::4].isfinite().any() and bool((got[3::4, 5] == -inf).all())
    got[3::4, 5] = want[3::4, 5]
    good = torch.arange(rows, device=device) % 4
    good = (good == 0) | (good == 3)
    if rows == 4:
        assert torch.equal(got[good], want[good])
    else:  # bit for bit but where a chunk of their group went another way, which is as near
        _check(got[good], bank, x[good], ids[good.cpu().numpy()], y[good], dtype)
    bank.down[3, 0, 0, 0] = nan
    got = bank(x, named, y)
    others = torch.from_numpy(ids != 3).to(device)
    assert torch.equal(got[others], want[others]) and bool(got[~others].isnan().all())


@pytest.mark.parametrize("rows,rank", ((6, 16), (1200, 16), (1200, 70), (1100, 130)))
def test_large_and_small_values(device, rows, rank):
    """A x far outside f16, and far below it, in f16 as in bf16: it stays f32."""
    print(f"ranges in tiles {rows} {rank}", flush=True)
    rng = np.random.default_rng(rows + rank)
    for dtype, big in ((F16, 2.0 ** 9), (BF16, 2.0 ** 40)):
        for factor, back in ((big, 1 / big ** 2), (1 / big, big)):
            bank = LowRankAdapters(2, 80, 64, rank, dtype=dtype, device=device)
            for a in range(2):
                bank.load(a, _normal(rng, rank, 64) * factor, _normal(rng, 80, rank), back)
            assert (_words(bank, rows) > 0) == (rows > 6)
            x = (_normal(rng, rows, 64) * factor).to(dtype).to(device)
            y = torch.zeros((rows, 80), dtype=dtype, device=device)
            ids = rng.integers(0, 2, rows)
            _check(bank(x, torch.from_numpy(ids).to(device), y), bank, x, ids, y, dtype)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows", (3, 1500))
def test_adapters_of_several_ranks(device, dtype, rows):
    """Smaller ranks than the bank's, also after a larger one in the same place; adapters not loaded add nothing."""
    print(f"ranks in tiles {dtype} {rows}", flush=True)
    rng = np.random.default_rng(rows)
    bank = _bank(rng, 6, 120, 80, 40, dtype, device)
    for a, r in ((1, 1), (2, 39), (4, 8)):
        bank.load(a, _normal(rng, r, 80), _normal(rng, 120, r), -0.5)
    assert (_words(bank, rows) > 0) == (rows > 3)
    x, y = _rows(rng, rows, 80, dtype, device), _rows(rng, rows, 120, dtype, device)
    ids = rng.integers(-1, 7, rows)
    _check(bank(x, torch.from_numpy(ids).to(device), y), bank, x, ids, y, dtype)
    empty = LowRankAdapters(2, 120, 80, 5, dtype=dtype, device=device)
    assert torch.equal(empty(x, torch.ones(rows, dtype=torch.int32, device=device), y), y)


@pytest.mark.parametrize("id_type", (torch.int32, torch.int64))
@pytest.mark.parametrize("rows", (2, 90, 431))
def test_ids_of_requests(device, id_type, rows):
    """An id for all rows of a request: the sort reads it once for each of its rows."""
    print(f"requests in tiles {id_type} {rows}", flush=True)
    rng = np.random.default_rng(rows)
    bank = _bank(rng, 3, 72, 64, 8, BF16, device)
    requests = 6
    x, y = _rows(rng, requests * rows, 64, BF16, device), _rows(rng, requests * rows, 72, BF16, device)
    ids = np.array([0, 2, -1, 1, 5, 2])
    named = torch.from_numpy(ids).to(device).to(id_type)
    assert (_words(bank, requests * rows) > 0) == (rows > 200)
    whole = np.repeat(ids, rows)
    want = bank(x, torch.from_numpy(whole).to(device), y)
    _check(want, bank, x, whole, y, BF16)
    got = bank(x.view(requests, rows, 64), named[:, None], y.view(requests, rows, 72))
    assert torch.equal(got.view(torch.int16), want.view(requests, rows, 72).view(torch.int16))  # NaN and all
    got = bank(x.view(2, 3, rows, 64), named.view(2, 3)[..., None], y.view(2, 3, rows, 72))
    assert torch.equal(got.view(torch.int16), want.view(2, 3, rows, 72).view(torch.int16))
    if id_type == torch.int64:
        past = torch.tensor([2 ** 32, 2 ** 32 - 1, -2 ** 32 + 1, -1, 2 ** 40 + 1, 0], device=device)[:, None]
        got = bank(x.view(requests, rows, 64), past, y.view(requests, rows, 72))
        _check(got.view(-1, 72), bank, x, np.repeat([9, 9, 9, -1, 9, 0], rows), y, BF16)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,out", ((7, 123), (1400, 123), (1100, 1027)))
def test_any_address_and_stride(device, dtype, rows, out):
    print(f"addresses in tiles {dtype} {rows} {out}", flush=True)
    rng = np.random.default_rng(rows)
    bank = _bank(rng, 4, out, 88, 12, dtype, device)
    assert (_words(bank, rows) > 0) == (rows > 7)
    x, y = _rows(rng, rows, 88, dtype, device), _rows(rng, rows, out, dtype, device)
    ids = rng.integers(-1, 4, rows)
    named = torch.from_numpy(ids).to(device)
    want = bank(x, named, y)
    _check(want, bank, x, ids, y, dtype)
    for shift in (1, 3):
        odd = [torch.empty(t.numel() + shift, dtype=t.dtype, device=device)[shift:].view(t.shape).copy_(t) for t in (x, named, y)]
        assert torch.equal(bank(*odd), want)
    turned = [t.transpose(0, -1).contiguous().transpose(0, -1) for t in (x, named.repeat(2, 1).T[:, 0], y)]
    assert torch.equal(bank(*turned), want)


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("rows,out", ((24, 200), (1300, 200), (1100, 1300), (4500, 4096)))
def test_in_the_place_of_a_projections_output(device, dtype, rows, out):
    """``MxLinear`` adds in y's place, whose next columns are on their way meanwhile."""
    print(f"in place {dtype} {rows} {out}", flush=True)
    rng = np.random.default_rng(rows)
    n = 160
    proj = mx.MxLinear(out, n, device=device)
    proj.load(mx.quantize((0.05 * _normal(rng, out, n)).to(dtype).to(device)))
    for rank in (16, 70):
        bank = _bank(rng, 5, out, n, rank, dtype, device)
        assert (_words(bank, rows) > 0) == (rows > 24)
        x, ids = _rows(rng, rows, n, dtype, device), rng.integers(-1, 5, rows)
        named = torch.from_numpy(ids).to(device)
        plain = proj(x)
        got = proj(x, bank, named)
        assert torch.equal(got, bank(x, named, plain)) and torch.equal(proj(x), plain)
        if rows < 4000:
            _check(got, bank, x, ids, plain, dtype)


@pytest.mark.parametrize("dtype", HALF)
def test_replayed_from_a_graph(device, dtype):
    """Tiles in a graph: other ids, rows and adapters in every replay, two calls in one graph."""
    print(f"tiles in a graph {dtype}", flush=True)
    rng = np.random.default_rng(5)
    rows = 1700
    bank = _bank(rng, 9, 264, 128, 40, dtype, device)
    assert _words(bank, rows) > 0
    x, y = _rows(rng, rows, 128, dtype, device), _rows(rng, rows, 264, dtype, device)
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
        twice = bank(x, ids, held)
    for turn in range(4):
        named = rng.integers(-1, 9, rows) if turn != 2 else np.full(rows, 3)
        ids.copy_(torch.from_numpy(named))
        x.add_(0.5)
        bank.load(turn, _normal(rng, 40 - turn, 128) * 0.1, _normal(rng, 264, 40 - turn))
        graph.replay()
        torch.cuda.synchronize()
        got = held.clone(), twice.clone()
        want = bank(x, ids, y)
        assert torch.equal(got[0], want) and torch.equal(got[1], bank(x, ids, want))
        _check(want, bank, x, named, y, dtype)
        torch.cuda.synchronize()


def test_calls_on_two_streams_at_once(device):
    """Each call's workspace is its own."""
    print("tiles on two streams", flush=True)
    rng = np.random.default_rng(4)
    bank = _bank(rng, 7, 520, 512, 16, BF16, device)
    jobs = []
    for rows in (2500, 1700):
        assert _words(bank, rows) > 0
        jobs.append((_rows(rng, rows, 512, BF16, device), torch.from_numpy(rng.integers(-1, 7, rows)).to(device),
                     _rows(rng, rows, 520, BF16, device)))
    want = [bank(*job) for job in jobs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in jobs], [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(bank(*jobs[i]))
    torch.cuda.synchronize()
    for outs, expected in zip(got, want):
        assert all(torch.equal(out, expected) for out in outs)
