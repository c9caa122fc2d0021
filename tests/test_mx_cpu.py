"""The 4-bit and router entry points without a GPU: what the C ABI and the Python
surface refuse before anything is launched."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import mxref
from mlx_iqk_amd import _native, build, mx, router
from mlx_iqk_amd.kernels import IqkKernelError
from mlx_iqk_amd.nn import IqkRuntimeError

OK, GEOMETRY, ARGUMENT = _native.OK, _native.ERR_GEOMETRY, _native.ERR_ARGUMENT
P = 64  # an address that no refused call reads


@pytest.fixture(scope="module")
def lib():
    if not build.HIP_LIB.is_file():
        build.build_hip()
    return _native.load()


def test_cast_entry_points_refuse_bad_arguments(lib):
    q, d = lib.iqk_mx_quantize, lib.iqk_mx_dequantize
    for cols in (0, 31, 33, -32, 1 << 32):
        assert q(0, P, 4, cols, cols, P, P, 8, None) == GEOMETRY
        assert d(0, P, P, 4, cols, 8, P, None) == GEOMETRY
    assert q(3, P, 4, 64, 64, P, P, 2, None) == ARGUMENT
    assert q(-1, P, 4, 64, 64, P, P, 2, None) == ARGUMENT
    assert q(0, P, -1, 64, 64, P, P, 2, None) == ARGUMENT
    assert q(0, P, 1 << 42, 64, 64, P, P, 2, None) == ARGUMENT  # past what the counters hold
    assert q(0, P, 4, 64, 64, P, P, 1, None) == ARGUMENT        # rows of scales overlap
    assert q(0, P, 4, 64, 66, P, P, 2, None) == ARGUMENT        # rows off 16 bytes
    assert q(1, P, 4, 64, 68, P, P, 2, None) == ARGUMENT
    assert q(0, P + 4, 4, 64, 64, P, P, 2, None) == ARGUMENT
    assert q(0, None, 4, 64, 64, P, P, 2, None) == ARGUMENT
    assert q(0, P, 4, 64, 64, None, P, 2, None) == ARGUMENT
    assert d(0, P, None, 4, 64, 2, P, None) == ARGUMENT
    assert d(0, P, P, 4, 64, 2, P + 8, None) == ARGUMENT
    assert q(0, None, 0, 64, 64, None, None, 2, None) == OK
    assert d(0, None, None, 0, 64, 2, None, None) == OK


def test_weight_entry_points_refuse_bad_arguments(lib):
    pack, unpack = lib.iqk_mx_pack, lib.iqk_mx_unpack
    for n, out, experts in ((0, 16, 1), (48, 16, 1), (64, 0, 1), (64, 16, 0), (64, 1 << 24, 1), (64, 16, 1 << 20)):
        assert pack(n, out, experts, P, P, 1 << 20, P, P, P, None) == GEOMETRY
        assert unpack(0, n, out, experts, P, P, P, P, None) == GEOMETRY
    assert pack(64, 16, 1, P + 8, P, 2, P, P, P, None) == ARGUMENT
    assert pack(64, 16, 1, P, P, 1, P, P, P, None) == ARGUMENT
    assert pack(64, 16, 1, P, P, 2, P, None, P, None) == ARGUMENT
    assert unpack(5, 64, 16, 1, P, P, P, P, None) == ARGUMENT
    assert unpack(0, 64, 16, 1, P, P, P, None, None) == ARGUMENT


def test_product_entry_points_refuse_bad_arguments(lib):
    def pairs(act=0, n=64, out=16, experts=2, x=P, rows=4, xs=None, xss=0, tiles=P, ids=P, per=1, pairs=4, y=P):
        return lib.iqk_mx_pairs(act, n, out, experts, x, rows, xs, xss, tiles, P, P, ids, 0, per, pairs, y, None)

    def groups(act=0, n=64, out=16, experts=2, x=P, rows=4, xs=None, xss=0, tiles=P, offs=P, slots=4, y=P):
        return lib.iqk_mx_groups(act, n, out, experts, x, rows, xs, xss, tiles, P, P, offs, P, P, slots, y, None)

    for f in (pairs, groups):
        for bad in (dict(act=4), dict(act=-1), dict(experts=0), dict(experts=4097), dict(x=None), dict(x=P + 8),
                    dict(rows=0), dict(rows=1 << 31), dict(tiles=None), dict(tiles=P + 8), dict(y=None),
                    dict(act=2), dict(act=2, xs=P, xss=2), dict(act=3, xs=P, xss=6), dict(act=2, xs=P + 2, xss=4),
                    dict(act=2, n=160, xs=P, xss=4)):
            assert f(**bad) == ARGUMENT, bad
        for bad in (dict(n=0), dict(n=48), dict(n=1 << 24), dict(out=0), dict(out=1 << 24)):
            assert f(**bad) == GEOMETRY, bad
    assert pairs(ids=None) == ARGUMENT and groups(offs=None) == ARGUMENT  # of two experts
    assert pairs(per=0) == ARGUMENT and pairs(per=2, rows=1) == ARGUMENT  # four pairs name two rows
    assert pairs(pairs=-1) == ARGUMENT and groups(slots=1 << 31) == ARGUMENT
    assert pairs(pairs=0) == OK and groups(slots=0) == OK


def test_grouped_call_refuses_bad_arguments(lib):
    def prefill(act=0, n=64, out=16, experts=2, x=P, rows=4, ids=P, pairs=4, per_pair=1, per_row=1, work=P, y=P):
        return lib.iqk_mx_prefill(act, n, out, experts, x, rows, None, 0, P, P, P, ids, 0, pairs, per_pair, per_row,
                                  work, y, None)

    for bad in (dict(act=4), dict(experts=4097), dict(x=None), dict(y=None), dict(ids=None), dict(work=None),
                dict(per_pair=0), dict(per_row=0), dict(pairs=-1), dict(pairs=1 << 20, per_pair=1 << 20),
                dict(rows=3), dict(act=2)):
        assert prefill(**bad) == ARGUMENT, bad
    assert prefill(n=48) == GEOMETRY and prefill(pairs=0) == OK


def test_torch_binding_is_built_from_the_same_sources(lib):
    binding = _native.torch_binding()
    assert binding.source_hash() == lib.iqk_hip_source_hash().decode()
    for name, args in (("topk", 3), ("balance", 3), ("mx_quantize", 2), ("mx_dequantize", 4), ("mx_project", 14)):
        with pytest.raises(TypeError):
            getattr(binding, name)()
        with pytest.raises(TypeError):
            getattr(binding, name)(*[0] * args)  # not tensors


def test_a_missing_or_stale_torch_binding_is_refused(monkeypatch, tmp_path, lib):
    monkeypatch.setattr(_native, "_TORCH", None)
    monkeypatch.setattr(_native, "TORCH_EXT", tmp_path / "absent.so")
    with pytest.raises(_native.IqkNativeError, match="not built"):
        _native.torch_binding()


def test_router_entry_points_refuse_bad_arguments(lib):
    topk, grad = lib.iqk_router_topk, lib.iqk_router_topk_grad
    for rows, experts, k in ((4, 0, 1), (4, 1025, 1), (4, 8, 0), (4, 8, 9), (4, 100, 65), (-1, 8, 1), (1 << 31, 8, 1)):
        assert topk(0, P, rows, experts, k, 1, P, P, None) == GEOMETRY
        assert grad(0, P, P, P, P, rows, experts, k, 1, P, None) == GEOMETRY
    assert topk(3, P, 4, 8, 2, 1, P, P, None) == ARGUMENT
    assert topk(0, None, 4, 8, 2, 1, P, P, None) == ARGUMENT
    assert grad(0, None, P, P, P, 4, 8, 2, 0, P, None) == ARGUMENT  # the softmax over all needs the logits
    assert grad(0, P, P, P, None, 4, 8, 2, 1, P, None) == ARGUMENT
    assert topk(0, None, 0, 8, 2, 1, None, None, None) == OK
    bal, bgrad = lib.iqk_balance, lib.iqk_balance_grad
    for g, t, experts, k in ((-1, 4, 8, 2), (65536, 4, 8, 2), (1, -1, 8, 2), (1, 4, 1025, 2), (1, 4, 8, 9)):
        assert bal(0, P, P, None, g, t, experts, k, P, P, P, P, None) == GEOMETRY
        assert bgrad(0, P, None, P, P, P, g, t, experts, k, P, None) == GEOMETRY
    assert bal(0, P, None, None, 1, 4, 8, 2, P, P, P, P, None) == ARGUMENT
    assert bal(0, P, P, None, 1, 4, 8, 2, None, P, P, P, None) == ARGUMENT
    assert bgrad(0, P, None, P, None, P, 1, 4, 8, 2, P, None) == ARGUMENT
    assert bal(0, None, None, None, 0, 4, 8, 2, None, None, None, None, None) == OK
    assert lib.iqk_balance_work(0, 4, 8) == -1 and lib.iqk_balance_work(1, 4, 1025) == -1
    assert lib.iqk_balance_work(1, 0, 8) == 17 and lib.iqk_balance_work(2, 33, 8) == 2 * 2 * 17
    assert lib.iqk_hip_last_error() == 0


def test_nothing_falls_back_to_the_cpu():
    with pytest.raises(IqkKernelError):
        mx.quantize(torch.zeros(4, 32))
    q = mx.MxTensor(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8))
    assert q.shape == (4, 32) and q.dtype == torch.float16
    with pytest.raises(IqkKernelError):
        q.dequantize()
    line = mx.MxLinear(4, 32)
    with pytest.raises(IqkKernelError):
        line.load(q)
    with pytest.raises(IqkKernelError):
        line(torch.zeros(2, 32, dtype=torch.float16))
    with pytest.raises(IqkKernelError):
        line.dequantized()
    with pytest.raises(IqkKernelError):
        router.topk(torch.zeros(4, 8), 2)
    with pytest.raises(IqkKernelError):
        router.balance_loss(torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.int32))


def test_modules_refuse_shapes():
    for E, out, n in ((0, 16, 32), (4097, 16, 32), (2, 0, 32)):
        with pytest.raises(IqkRuntimeError):
            mx.MxSwitchLinear(E, out, n)
    for n in (0, 16, 100):
        with pytest.raises(IqkKernelError):
            mx.MxLinear(16, n)


def test_plain_quantisation_finds_the_nearest_code():
    """The oracle itself: no code is nearer than the one it takes, and a tie takes the even one."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((40, 64))
    codes, scales = mxref.quantize(x)
    got = mxref.values(codes, scales)
    unit = np.repeat(np.ldexp(1.0, scales.astype(int) - 127), 32, -1)
    best = np.abs(x[..., None] - mxref.VALUES * unit[..., None]).min(-1)
    np.testing.assert_array_equal(np.abs(x - got), best)
    top = np.abs(x.reshape(40, 2, 32)).max(-1) / np.ldexp(1.0, scales.astype(int) - 127)
    assert ((top >= 4) & (top < 8)).all()
    ties = np.array([[0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 4.0] * 4])
    np.testing.assert_array_equal(mxref.values(*mxref.quantize(ties))[0, :8], [0, 1, 1, 2, 2, 4, 4, 4])


def test_grids_that_cannot_be_launched_are_refused(lib):
    """2^32 threads are one too many: 256 or 512 a workgroup."""
    def pairs(n, rows, out=16):
        return lib.iqk_mx_pairs(0, n, out, 2, P, rows, None, 0, P, P, P, P, 0, 1, rows, P, None)

    assert pairs(64, 1 << 24) == ARGUMENT and pairs(64, 1 << 20, out=256) == ARGUMENT
    assert pairs(4096, 1 << 23) == ARGUMENT and pairs(4096, 1 << 19, out=256) == ARGUMENT
    assert lib.iqk_mx_groups(0, 64, 512, 2, P, 4, None, 0, P, P, P, P, P, P, 1 << 30, P, None) == ARGUMENT
    assert lib.iqk_mx_groups(0, 64, 512, 1, P, 4, None, 0, P, P, P, None, None, None, 1 << 30, P, None) == ARGUMENT
    assert lib.iqk_mx_pack(64, 272, (1 << 20) - 1, P, P, 2, P, P, P, None) == GEOMETRY
    assert lib.iqk_hip_last_error() == 0  # none reached a launch
    # a module groups its pairs before there are so many
    few = mx.MxSwitchLinear(4096, 1 << 18, 32, device="meta")._pair_limit
    assert few == 512 < mx.pair_limit(4096)


def test_a_torch_binding_of_another_source_or_torch_is_refused(monkeypatch, tmp_path, lib):
    assert _native.torch_binding().binding_hash() == build.torch_binding_hash()
    edited = tmp_path / "iqk_torch.cpp"
    edited.write_bytes(build.TORCH_SOURCE.read_bytes() + b"\n")
    for at, name, value in ((build, "TORCH_SOURCE", edited), (torch, "__version__", torch.__version__ + "x")):
        with monkeypatch.context() as m:
            m.setattr(_native, "_TORCH", None)
            m.setattr(at, name, value)
            with pytest.raises(_native.IqkNativeError, match="another"):
                _native.torch_binding()
    with monkeypatch.context() as m:  # a library of other sources than the binding's
        m.setattr(_native, "_TORCH", None)
        m.setattr(_native, "_import", lambda *_: type("Stale", (), {"source_hash": staticmethod(lambda: "0" * 16)}))
        with pytest.raises(_native.IqkNativeError, match="other sources"):
            _native.torch_binding()
    assert _native.torch_binding() is not None


def test_every_public_name_is_there():
    import mlx_iqk_amd
    for module in (mlx_iqk_amd, mx, router):
        for name in module.__all__:
            assert getattr(module, name) is not None, (module.__name__, name)
