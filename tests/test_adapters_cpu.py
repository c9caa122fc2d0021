"""Refusals of the sort, dispatch, combine and adapter calls that need no GPU: the modules' and the C ABI's."""

from __future__ import annotations

import ctypes
import importlib.util
from pathlib import Path

import pytest
import torch

import mlx_iqk_amd
from mlx_iqk_amd import _native, build, mx, router
from mlx_iqk_amd.adapters import MAX_ADAPTERS, MAX_RANK, LowRankAdapters
from mlx_iqk_amd.kernels import IqkKernelError
from mlx_iqk_amd.nn import IqkRuntimeError


@pytest.fixture(scope="module")
def lib():
    if not build.HIP_LIB.is_file():
        build.build_hip()
    return _native.load()


def test_banks_are_refused():
    for args in ((0, 8, 8, 4), (MAX_ADAPTERS + 1, 8, 8, 4), (2, 0, 8, 4), (2, 8, 0, 4), (2, 8, 12, 4), (2, 8, 8, 0),
                 (2, 8, 8, MAX_RANK + 1)):
        with pytest.raises(IqkRuntimeError):
            LowRankAdapters(*args)
    with pytest.raises(IqkRuntimeError):
        LowRankAdapters(2, 8, 8, 4, dtype=torch.float32)
    assert mlx_iqk_amd.LowRankAdapters is LowRankAdapters


def test_load_on_the_host():
    bank = LowRankAdapters(2, 6, 16, 5, dtype=torch.float16)
    assert bank.down.shape == (2, 2, 8, 8) and bank.up.shape == (2, 1, 6, 8)
    down, up = torch.randn(3, 16), torch.randn(6, 3)
    bank.load(1, torch.randn(5, 16), torch.randn(6, 5))
    bank.load(1, down, up, 0.25)
    got_down, got_up, scale = bank.adapter(1)
    assert torch.equal(got_down[:3], down.half()) and torch.equal(got_up[:, :3], up.half()) and scale == 0.25
    assert not got_down[3:].any() and not got_up[:, 3:].any() and bank.scales.tolist() == [0.0, 0.25]
    assert torch.equal(bank.down[1, 1, 2], down[2, 8:].half()) and torch.equal(bank.up[1, 0, 4, :3], up[4].half())
    assert not bank.down[0].any()
    bank.load(0, down, up.T.contiguous().T)
    assert torch.equal(bank.adapter(0)[1], got_up)
    with pytest.raises(IqkRuntimeError):
        bank.adapter(2)
    for index, a, b in ((2, down, up), (-1, down, up), (0, torch.randn(6, 16), torch.randn(6, 6)),
                        (0, down, torch.randn(6, 2)), (0, torch.randn(3, 8), up), (0, down, torch.randn(5, 3)),
                        (0, down[0], up)):
        with pytest.raises(IqkRuntimeError):
            bank.load(index, a, b)


def test_host_tensors_are_refused():
    ids = torch.zeros((3, 2), dtype=torch.int32)
    with pytest.raises(IqkKernelError, match="GPU"):
        router.sort(ids, 4)
    with pytest.raises(IqkKernelError, match="GPU"):
        router.dispatch(torch.zeros(3, 8), ids, 4)
    with pytest.raises(IqkKernelError, match="GPU"):
        router.combine(torch.zeros(3, 2, 8), torch.zeros(3, 2))
    bank = LowRankAdapters(2, 6, 16, 5)
    with pytest.raises(IqkKernelError, match="GPU"):
        bank(torch.zeros(3, 16, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int32),
             torch.zeros(3, 6, dtype=torch.bfloat16))


def test_sort_and_rows_refuse_bad_arguments(lib):
    p = ctypes.c_void_p(16)  # never dereferenced: every call below is refused first
    big = 1 << 31
    assert lib.iqk_sort_work(8, 6, 256) == 0
    assert lib.iqk_sort_work(1 << 20, 6, 256) > 0
    for tokens, k, experts in ((-1, 6, 8), (8, 0, 8), (8, 65, 8), (8, 6, 0), (8, 6, 1025), (big, 1, 8), (1 << 30, 2, 8),
                               (1 << 62, 4, 8)):
        assert lib.iqk_sort_work(tokens, k, experts) == -1
        assert lib.iqk_sort(p, 0, tokens, k, experts, p, p, p, p, p, None) == _native.ERR_GEOMETRY
    assert lib.iqk_sort(None, 0, 8, 6, 8, p, p, p, p, p, None) == _native.ERR_ARGUMENT
    assert lib.iqk_sort(p, 0, 8, 6, 8, p, None, p, p, p, None) == _native.ERR_ARGUMENT
    assert lib.iqk_sort(p, 0, 8, 6, 8, p, p, p, p, None, None) == _native.ERR_ARGUMENT
    assert lib.iqk_sort(p, 0, 1 << 20, 6, 8, None, p, p, p, p, None) == _native.ERR_ARGUMENT  # no workspace
    for dtype, tokens, k, cols in ((3, 8, 6, 64), (-1, 8, 6, 64), (0, -1, 6, 64), (0, 8, 0, 64), (0, 8, 65, 64),
                                   (0, 8, 6, 0), (0, 8, 6, 1 << 28), (0, 1 << 30, 2, 64), (0, big, 1, 64)):
        assert lib.iqk_dispatch(dtype, p, p, 0, tokens, k, 8, cols, p, p, p, p, p, p, None) == _native.ERR_GEOMETRY
        assert lib.iqk_combine(dtype, p, p, p, p, p, tokens, k, cols, p, None) == _native.ERR_GEOMETRY
        assert lib.iqk_combine_grad(dtype, p, p, p, p, p, tokens, k, cols, p, p, None) == _native.ERR_GEOMETRY
    for experts in (0, 1025):
        assert lib.iqk_dispatch(0, p, p, 0, 8, 6, experts, 64, p, p, p, p, p, p, None) == _native.ERR_GEOMETRY
    for tokens in (8, 1 << 18):  # sorting in its own launch, and before
        good = [0, p, p, 0, tokens, 6, 8, 64, p, p, p, p, p, p, None]
        for place in (1, 2, 9, 10, 11, 12, 13):
            assert lib.iqk_dispatch(*[None if i == place else v for i, v in enumerate(good)]) == _native.ERR_ARGUMENT
    assert lib.iqk_dispatch(*[None if i == 8 else v for i, v in enumerate(good)]) == _native.ERR_ARGUMENT  # no workspace
    assert lib.iqk_combine(0, None, p, p, p, p, 8, 6, 64, p, None) == _native.ERR_ARGUMENT
    assert lib.iqk_combine(0, p, p, p, p, p, 8, 6, 64, None, None) == _native.ERR_ARGUMENT
    assert lib.iqk_combine_grad(0, None, p, p, p, p, 8, 6, 64, p, p, None) == _native.ERR_ARGUMENT
    assert lib.iqk_combine_grad(0, p, None, p, p, p, 8, 6, 64, p, p, None) == _native.ERR_ARGUMENT  # dweights want y
    assert lib.iqk_combine_grad(0, p, p, p, p, None, 8, 6, 64, p, p, None) == _native.ERR_ARGUMENT
    # nothing to do: no launch
    assert lib.iqk_combine(0, None, None, None, None, None, 0, 6, 64, None, None) == _native.OK
    assert lib.iqk_combine_grad(0, p, p, p, p, p, 8, 6, 64, None, None, None) == _native.OK


def test_adapters_refuse_bad_arguments(lib):
    p, odd = ctypes.c_void_p(16), ctypes.c_void_p(24)  # never dereferenced: every call below is refused first
    f = lib.iqk_adapters
    assert lib.iqk_adapters_work(64, 48, 8, 4, 3) == 0 and lib.iqk_adapters_work(64, 48, 8, 4, 5000) > 0
    for n, out, rank, adapters, rows in ((0, 48, 8, 4, 3), (60, 48, 8, 4, 3), (64, 0, 8, 4, 3), (64, 48, 0, 4, 3),
                                         (64, 48, 12, 4, 3), (64, 48, 264, 4, 3), (64, 48, 8, 0, 3), (64, 48, 8, 1025, 3),
                                         (64, 48, 8, 4, -1), (64, 48, 8, 4, 1 << 31), (1 << 31, 48, 8, 4, 3),
                                         (64, 1 << 31, 8, 4, 3)):
        assert lib.iqk_adapters_work(n, out, rank, adapters, rows) == -1
        assert f(2, n, out, rank, adapters, p, rows, p, 0, 1, p, p, p, p, p, p, None) == _native.ERR_GEOMETRY
    for dtype in (0, 3, -1):
        assert f(dtype, 64, 48, 8, 4, p, 3, p, 0, 1, p, p, p, p, p, p, None) == _native.ERR_ARGUMENT
    good = [2, 64, 48, 8, 4, p, 3, p, 0, 1, p, p, p, p, p, p, None]
    for rows, places in ((3, (5, 7, 10, 11, 12, 14, 15)), (5000, (5, 7, 10, 11, 12, 13, 14, 15))):
        for place in places:
            assert f(*[None if i == place else rows if i == 6 else v for i, v in enumerate(good)]) == _native.ERR_ARGUMENT
        for place in (10, 11, 13):
            assert f(*[odd if i == place else rows if i == 6 else v for i, v in enumerate(good)]) == _native.ERR_ARGUMENT
    for per_id in (0, -1, 1 << 31):
        assert f(*[per_id if i == 9 else v for i, v in enumerate(good)]) == _native.ERR_ARGUMENT
    assert f(2, 64, 48, 8, 4, None, 0, None, 0, 1, None, None, None, None, None, None, None) == _native.OK


def test_no_rows_need_no_workspace(lib):
    """Also for sizes of which one row is too much for a workgroup of its own, and so is sorted."""
    p = ctypes.c_void_p(16)  # never dereferenced: no rows, no launch
    for n, out, rank, adapters in ((4096, 4096, 16, 64), (4096, 4096, 128, 64), (4096, 4096, 256, 1024), (1 << 20, 8, 8, 1)):
        assert lib.iqk_adapters_work(n, out, rank, adapters, 0) == 0
        assert lib.iqk_adapters(1, n, out, rank, adapters, p, 0, p, 0, 1, p, p, p, None, p, p, None) == _native.OK
        assert lib.iqk_adapters_work(n, out, rank, adapters, 1) >= 0
    assert lib.iqk_adapters_work(4096, 4096, 128, 64, 1) > 0


@pytest.mark.parametrize("requests", ("0", "-3", "41", "1025"))
def test_the_example_refuses_requests_that_its_prompts_do_not_hold(requests, capsys):
    spec = importlib.util.spec_from_file_location("mx_moe", Path(__file__).parents[1] / "examples" / "mx_moe.py")
    mx_moe = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mx_moe)
    tokens = "10" if requests != "1025" else "2000"
    with pytest.raises(SystemExit):
        mx_moe.main(["--sequences", "4", "--tokens", tokens, "--requests", requests])
    assert "--requests must be" in capsys.readouterr().err


def test_ids_without_adapters_are_refused():
    proj = mx.MxLinear(64, 32)
    with pytest.raises(IqkRuntimeError, match="adapter_ids"):
        proj(torch.zeros(3, 32, dtype=torch.bfloat16), adapter_ids=torch.zeros(3, dtype=torch.int32))
    with pytest.raises(IqkRuntimeError, match="adapter_ids"):
        proj(torch.zeros(3, 32, dtype=torch.bfloat16), None, torch.zeros(3, dtype=torch.int32))


def test_gradients_of_any_slots_refuse_bad_arguments(lib):
    p = ctypes.c_void_p(16)  # never dereferenced: every call below is refused first
    f = lib.iqk_combine_grad_rows
    for dtype, tokens, k, cols in ((3, 8, 6, 64), (0, -1, 6, 64), (0, 8, 0, 64), (0, 8, 65, 64), (0, 8, 6, 0), (0, 8, 6, 1 << 28),
                                   (0, 1 << 30, 2, 64)):
        assert f(dtype, p, p, p, p, tokens, k, cols, p, p, None) == _native.ERR_GEOMETRY
    good = [0, p, p, p, p, 8, 6, 64, p, p, None]
    for place in (1, 2, 4, 8, 9):
        assert f(*[None if i == place else v for i, v in enumerate(good)]) == _native.ERR_ARGUMENT
    assert f(0, None, None, None, None, 0, 6, 64, None, None, None) == _native.OK
