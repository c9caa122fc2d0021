"""Low-rank adapters of rows in tiles, sorted by adapter, against float64: values that the tiles' second
product has to keep.  Each case asserts which of the two forms it takes, rows alone or tiles."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mxref
from mlx_iqk_amd import _native
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
