"""4-bit microscaled quantisation and the projections with such weights, against
plain 64-bit forms."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import mxref
from mlx_iqk_amd import mx
from mlx_iqk_amd.kernels import IqkKernelError
from mlx_iqk_amd.nn import IqkRuntimeError

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
HALF = (F16, BF16)


def _f64(t: torch.Tensor) -> np.ndarray:
    return t.detach().cpu().to(torch.float64).numpy()


def _dev(a: np.ndarray, device, dtype=None) -> torch.Tensor:
    t = torch.from_numpy(np.array(a, order="C")).to(device)
    return t if dtype is None else t.to(dtype)


def _same_codes(q: mx.MxTensor, x: torch.Tensor) -> None:
    codes, scales = mxref.quantize(_f64(x))
    np.testing.assert_array_equal(q.scales.cpu().numpy(), scales)
    np.testing.assert_array_equal(q.codes.cpu().numpy(), codes)


# ------------------------------------------------------------ quantisation ---


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
@pytest.mark.parametrize("shape", ((32,), (1, 32), (3, 96), (2, 5, 160), (33, 1440), (0, 64), (257, 4096)))
def test_quantize(device, dtype, shape):
    print(f"quantize {dtype} {shape}", flush=True)
    rng = np.random.default_rng(len(shape) + shape[-1])
    x = _dev(rng.standard_normal(shape) * np.exp2(rng.integers(-9, 9, shape)), device, dtype)
    q = mx.quantize(x)
    assert q.shape == x.shape and q.dtype == dtype
    _same_codes(q, x)
    for out in (F32, F16, BF16):
        want = torch.from_numpy(mxref.values(q.codes.cpu().numpy(), q.scales.cpu().numpy())).to(out)
        assert torch.equal(q.dequantize(out).cpu(), want)


@pytest.mark.parametrize("dtype", (F32, F16, BF16))
def test_quantize_edges(device, dtype):
    """Ties, saturation, zeros of both signs, blocks of zeros, one value in a
    block, the smallest and largest magnitudes of the type, NaN and infinities."""
    print(f"quantize edges {dtype}", flush=True)
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.9, 6.0, -0.25, -5.0, 0.0, -0.0, 0.5, -7.5]
    rows = [ties * 2, [0.0] * 32, [-0.0] * 31 + [1.0], [0.0] * 31 + [-3.0]]
    info = torch.finfo(dtype)
    for v in (info.tiny, info.smallest_normal * 2 ** -4, info.max, 2.0 ** -14, 1.0):
        rows += [[v * s for s in (1, -1, 0.5, 0.25)] * 8]
    if dtype != F16:
        rows += [[2.0 ** -126 * s for s in (1, 0.5, 0.25, -0.125)] * 8, [2.0 ** -124 * s for s in (1, -0.3)] * 16,
                 [2.0 ** -63, 2.0 ** -64, 2.0 ** -65, -2.0 ** -66] * 8, [2.0 ** -61, 2.0 ** -62] * 16]
    for v in (float("nan"), float("inf"), float("-inf")):
        rows += [[1.0] * 31 + [v]]
    x = torch.tensor(rows, dtype=torch.float64).to(dtype).to(device)
    q = mx.quantize(x)
    _same_codes(q, x)
    bad = q.dequantize(F32)[-3:]
    assert bool(torch.isnan(bad).all())


def test_quantize_every_float16(device):
    """Every finite fp16 value, alone with a block maximum above it."""
    print("quantize every f16", flush=True)
    bits = np.arange(1 << 16, dtype=np.uint16).view(np.float16)
    bits = bits[np.isfinite(bits)]
    blocks = np.repeat(bits[: len(bits) // 31 * 31].reshape(-1, 31), 1, axis=0)
    top = np.abs(blocks).max(1, keepdims=True)
    x = _dev(np.concatenate([blocks, top], 1), device)
    _same_codes(mx.quantize(x), x)


def test_quantize_views(device):
    """Rows apart, columns apart, transposed, expanded, an odd start."""
    print("quantize views", flush=True)
    base = torch.randn((40, 400), device=device)
    for x in (base[:, :64], base[:, 8:72], base[:, 1:65], base[::2, :96], base.T[:64, :32], base[:1, :64].expand(5, 64),
              base[:, ::2][:, :64], base.view(8, 5, 400)[:, 1:3, :32], base.to(F16)[:, 4:68], base.to(F16)[3:5, 8:40]):
        q = mx.quantize(x)
        _same_codes(q, x)
        assert torch.equal(q.dequantize(), mx.quantize(x.contiguous()).dequantize())


def test_dequantize_every_code_and_scale(device):
    print("dequantize every code and scale", flush=True)
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(16, 16), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8), 16)[:, None]
    q = mx.MxTensor(_dev(codes, device), _dev(scales, device))
    want = mxref.values(codes, scales)
    for dtype in (F32, F16, BF16):
        got = q.dequantize(dtype).cpu()
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(torch.from_numpy(want).to(dtype)))
        assert torch.equal(torch.isnan(got), torch.from_numpy(np.isnan(want)))
    strided = mx.MxTensor(_dev(codes, device), _dev(np.repeat(scales, 3, 1), device)[:, 1:2])
    assert torch.equal(torch.nan_to_num(strided.dequantize(F32)), torch.nan_to_num(q.dequantize(F32)))


# ---------------------------------------------------------------- the layout ---


def _switch(rng, E, out, n, device, **scales):
    codes, s = mxref.random_codes(rng, (E, out, n), **scales)
    module = mx.MxSwitchLinear(E, out, n, device=device)
    module.load(mx.MxTensor(_dev(codes, device), _dev(s, device)))
    return module, mxref.values(codes, s)


@pytest.mark.parametrize("E,out,n", ((1, 1, 32), (3, 16, 128), (2, 33, 160), (5, 250, 1440), (1, 300, 4096)))
def test_load_and_dequantized(device, E, out, n):
    print(f"load {E} {out} {n}", flush=True)
    module, w = _switch(np.random.default_rng(n), E, out, n, device, lo=90, hi=160)
    for dtype in (F32, F16, BF16):
        assert torch.equal(module.dequantized(dtype).cpu(), torch.from_numpy(w).to(dtype))


def test_load_takes_scales_of_blocks_without_values(device):
    """Blocks of zeros may carry any scale, also the largest; a NaN block stays one."""
    print("load zeros and NaN", flush=True)
    rng = np.random.default_rng(3)
    codes, s = mxref.random_codes(rng, (1, 16, 256))
    codes[0, :, 16:32] = 0x88  # zeros of both signs
    codes[0, ::2, 16:32] = 0
    s[0, :, 1] = 254
    s[0, 3, 4] = 255
    module = mx.MxSwitchLinear(1, 16, 256, device=device)
    module.load(mx.MxTensor(_dev(codes, device), _dev(s, device)))
    want = mxref.values(codes, s)
    got = _f64(module.dequantized(F32))
    np.testing.assert_array_equal(got, want)
    x = torch.ones((4, 1, 256), dtype=F16, device=device)
    y = _f64(module(x, torch.zeros((4,), dtype=torch.int32, device=device)))
    assert np.isnan(y[..., 3]).all() and np.isfinite(np.delete(y, 3, -1)).all()


# ---------------------------------------------------------------- products ---


def _check(y: torch.Tensor, x: np.ndarray, w: np.ndarray, ids: np.ndarray, dtype) -> None:
    """y [pairs, out] against each pair's row x [pairs, n] through w[ids]."""
    got = _f64(y)
    assert y.dtype == dtype and got.shape == (len(ids), w.shape[1])
    for e in np.unique(ids):
        at = np.nonzero(ids == e)[0]
        want, bound = mxref.product_bound(x[at], w[e], dtype)
        off = np.abs(got[at] - want) - bound
        assert (off <= 0).all(), (e, np.abs(got[at] - want).max(), off.max())


def _operand(rng, rows, n, dtype, quantized, device):
    """Rows as the module takes them, and their values."""
    x = _dev(rng.standard_normal((rows, n)), device, dtype)
    if not quantized:
        return x, _f64(x)
    q = mx.quantize(x)
    return q, _f64(q.dequantize(F32))


def _shape(x, *shape):
    if isinstance(x, mx.MxTensor):
        return mx.MxTensor(x.codes.view(*shape, -1), x.scales.reshape(*shape, x.scales.shape[-1]), x.dtype)
    return x.view(*shape, -1)


@pytest.mark.parametrize("quantized", (False, True))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("E,out,n", ((4, 48, 128), (3, 17, 32), (6, 250, 1440), (2, 64, 4096), (2, 33, 2080),
                                     (2, 16, 9216)))
def test_few_pairs(device, quantized, dtype, E, out, n):
    print(f"pairs {quantized} {dtype} {E} {out} {n}", flush=True)
    rng = np.random.default_rng(out + n)
    module, w = _switch(rng, E, out, n, device)
    for tokens, k, per_pair, wide in ((1, 1, False, False), (1, 2, False, True), (4, 2, False, False),
                                      (5, 2, True, True)):
        ids = rng.integers(0, E, (tokens, k))
        x, xv = _operand(rng, tokens * k if per_pair else tokens, n, dtype, quantized, device)
        y = module(_shape(x, tokens, k, 1) if per_pair else _shape(x, tokens, 1, 1),
                   _dev(ids, device, torch.int64 if wide else torch.int32))
        assert y.shape == (tokens, k, 1, out)
        rows = xv if per_pair else np.repeat(xv, k, 0)
        _check(y.view(tokens * k, out), rows, w, ids.reshape(-1), dtype)


# pairs of each expert: none, one, the tile's quarters and both sides of them,
# a tile, one more, several; few outputs go to the tiles that split the reduction
# axis, thousands to the others
COUNTS = ([0, 1, 15, 16, 17, 0], [32, 33, 48, 49], [64, 65, 128, 129, 3], [300, 0, 0, 7, 81, 97, 113])


@pytest.mark.parametrize("quantized", (False, True))
@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("counts", COUNTS, ids=lambda c: "-".join(map(str, c)))
@pytest.mark.parametrize("out,n", ((48, 128), (257, 160), (300, 1440), (100, 3360), (4100, 160), (4352, 1440)))
def test_groups(device, quantized, dtype, counts, out, n):
    print(f"groups {quantized} {dtype} {counts} {out} {n}", flush=True)
    rng = np.random.default_rng(out + n + len(counts))
    module, w = _switch(rng, len(counts), out, n, device)
    ids = rng.permutation(np.repeat(np.arange(len(counts)), counts))
    x, xv = _operand(rng, len(ids), n, dtype, quantized, device)
    y = module(_shape(x, len(ids), 1), _dev(ids, device, torch.int32), sorted_indices=True)
    _check(y.view(len(ids), out), xv, w, ids, dtype)


@pytest.mark.parametrize("quantized", (False, True))
@pytest.mark.parametrize("E", (1, 63, 64, 65, 200, 4096))
def test_groups_of_many_experts(device, quantized, E):
    print(f"groups of {E} experts {quantized}", flush=True)
    rng = np.random.default_rng(E)
    module, w = _switch(rng, E, 32, 64, device)
    ids = rng.integers(0, E, (180, 3))
    ids[:90] = rng.integers(0, min(E, 5), (90, 3))
    x, xv = _operand(rng, 180, 64, F16, quantized, device)
    y = module(_shape(x, 180, 1, 1), _dev(ids, device, torch.int64))
    _check(y.view(540, 32), np.repeat(xv, 3, 0), w, ids.reshape(-1), F16)


@pytest.mark.parametrize("quantized", (False, True))
def test_broadcast_shapes(device, quantized):
    """Rows per pair, x that broadcasts over leading dimensions, extra leading ones."""
    print(f"broadcast {quantized}", flush=True)
    rng = np.random.default_rng(5)
    E, out, n = 7, 40, 96
    module, w = _switch(rng, E, out, n, device)
    for xshape, ishape in (((3, 1, 4), (3, 2)), ((1, 6, 1), (5, 6)), ((6, 1), (5, 6)), ((2, 1, 1, 1), (2, 30, 2)),
                           ((1,), ()), ((70, 1, 2), (70, 1)), ((9, 8, 1), (9, 8)), ((1, 1), (80,))):
        rows = int(np.prod(xshape))
        x, xv = _operand(rng, rows, n, BF16, quantized, device)
        ids = rng.integers(0, E, ishape)
        y = module(_shape(x, *xshape), _dev(np.asarray(ids), device))
        batch = np.broadcast_shapes(xshape[:-1], ishape)
        M = xshape[-1]
        assert y.shape == (*batch, M, out)
        full = np.broadcast_to(xv.reshape(*xshape, n), (*batch, M, n)).reshape(-1, n)
        _check(y.reshape(-1, out), full, w, np.repeat(np.broadcast_to(ids, batch).reshape(-1), M), BF16)


def test_nothing_to_do(device):
    print("nothing to do", flush=True)
    module = mx.MxSwitchLinear(3, 20, 64, device=device)
    x = torch.zeros((0, 1, 1, 64), dtype=F16, device=device)
    assert module(x, torch.zeros((0, 2), dtype=torch.int32, device=device)).shape == (0, 2, 1, 20)
    assert module(x, torch.zeros((0, 2), dtype=torch.int32, device=device), sorted_indices=True).shape == (0, 2, 1, 20)
    line = mx.MxLinear(20, 64, device=device)
    assert line(torch.zeros((0, 64), dtype=F16, device=device)).shape == (0, 20)
    # weights that were never loaded are zeros
    assert not bool(line(torch.ones((9, 64), dtype=F16, device=device)).any())


@pytest.mark.parametrize("quantized", (False, True))
@pytest.mark.parametrize("many", (False, True))
def test_ids_outside_the_stack_give_nan(device, quantized, many):
    print(f"bad ids {quantized} {many}", flush=True)
    rng = np.random.default_rng(8)
    E, out, n = 4, 30, 64
    module, w = _switch(rng, E, out, n, device)
    pairs = 200 if many else 12
    ids = rng.integers(0, E, (pairs,))
    bad = rng.permutation(pairs)[:6]
    for wide, values in ((False, (-1, E, 2 ** 31 - 1, -5, 99, -2 ** 31)),
                         (True, (-1, E, 2 ** 32, 2 ** 32 + 1, -2 ** 40, 2 ** 62))):
        named = ids.copy()
        named[bad] = values
        x, xv = _operand(rng, pairs, n, F16, quantized, device)
        y = module(_shape(x, pairs, 1), _dev(named, device, torch.int64 if wide else torch.int32)).view(pairs, out)
        assert bool(torch.isnan(y[torch.from_numpy(bad)]).all())
        good = np.setdiff1d(np.arange(pairs), bad)
        _check(y[torch.from_numpy(good)], xv[good], w, ids[good], F16)


@pytest.mark.parametrize("quantized", (False, True))
@pytest.mark.parametrize("E,out", ((1, 40), (8, 32), (8, 2100), (100, 300), (512, 33), (513, 33)))
@pytest.mark.parametrize("pairs", (255, 257, 768, 1023, 1024, 1025))
def test_pairs_that_the_products_group(device, quantized, E, out, pairs):
    """Both sides of where the workgroups sort the pairs themselves: pairs in rounds of
    256, an expert with most of them, ids outside the stack, rows of one pair or of three."""
    print(f"group {quantized} {E} {out} {pairs}", flush=True)
    rng = np.random.default_rng(E + out + pairs)
    n, k = 96, 3 if pairs % 3 == 0 else 1
    module, w = _switch(rng, E, out, n, device)
    ids = np.where(rng.random(pairs) < 0.3, rng.integers(0, E), rng.integers(0, E, pairs))
    bad = rng.permutation(pairs)[:5]
    for dtype, values in ((torch.int32, (-1, E, E + 7, 2 ** 31 - 1, -2 ** 31)),
                          (torch.int64, (-1, E, 2 ** 32, 2 ** 32 + E - 1, -2 ** 62))):
        named = ids.copy()
        named[bad] = values
        x, xv = _operand(rng, pairs // k, n, BF16, quantized, device)
        y = module(_shape(x, pairs // k, 1, 1), _dev(named.reshape(-1, k), device, dtype), sorted_indices=True)
        y = y.view(pairs, out)
        assert bool(torch.isnan(y[torch.from_numpy(bad)]).all())
        good = np.setdiff1d(np.arange(pairs), bad)
        _check(y[torch.from_numpy(good)], np.repeat(xv, k, 0)[good], w, ids[good], BF16)


@pytest.mark.parametrize("quantized", (False, True))
@pytest.mark.parametrize("n", (96, 128, 1440))
@pytest.mark.parametrize("pairs", (5, 100))
def test_bad_rows_stay_where_they_are(device, quantized, n, pairs):
    """A row with NaN or infinities reaches its own outputs only, also where
    the next row's values stand right behind its end."""
    print(f"bad rows {quantized} {n} {pairs}", flush=True)
    rng = np.random.default_rng(n)
    module, w = _switch(rng, 2, 33, n, device)
    x = torch.randn((pairs, n), device=device).to(F16)
    x[1, 0] = float("nan")
    x[3, -1] = float("inf")
    good = np.setdiff1d(np.arange(pairs), (1, 3))
    q = mx.quantize(x) if quantized else x
    xv = _f64(q.dequantize(F32) if quantized else x)
    ids = rng.integers(0, 2, pairs)
    y = module(_shape(q, pairs, 1), _dev(ids, device)).view(pairs, 33)
    _check(y[torch.from_numpy(good)], xv[good], w, ids[good], F16)
    assert bool(torch.isnan(y[1]).all())
    want = xv[3] @ w[ids[3]].T if not quantized else np.full(33, np.nan)
    got = _f64(y[3])
    np.testing.assert_array_equal(np.isfinite(got), np.isfinite(want))
    np.testing.assert_array_equal(got[~np.isfinite(want)], want[~np.isfinite(want)])


@pytest.mark.parametrize("dtype", HALF)
@pytest.mark.parametrize("pairs", (5, 100, 1500))
def test_rows_of_very_different_scales(device, dtype, pairs):
    """Rows from 2^-100 to 2^100, blocks 36 powers of two apart in a row, by every route."""
    print(f"scales apart {dtype} {pairs}", flush=True)
    rng = np.random.default_rng(21)
    E, out, n = 2, 48, 256
    codes, s = mxref.random_codes(rng, (E, out, n), lo=0, hi=36)
    s = (s + np.linspace(20, 200, out).astype(int)[None, :, None]).astype(np.uint8)
    module = mx.MxSwitchLinear(E, out, n, device=device)
    module.load(mx.MxTensor(_dev(codes, device), _dev(s, device)))
    w = mxref.values(codes, s)
    ids = rng.integers(0, E, pairs)
    x, xv = _operand(rng, pairs, n, dtype, False, device)
    got = _f64(module(_shape(x, pairs, 1), _dev(ids, device)).view(pairs, out))
    for p in range(pairs):
        want, bound = mxref.product_bound(xv[p:p + 1], w[ids[p]], dtype)
        # f32 holds the exact sum scaled to the row; the rounding to fp16 may overflow
        with np.errstate(over="ignore"):
            top = torch.finfo(dtype).max
            inside = np.abs(want[0]) + bound[0] < top
            beyond = np.abs(want[0]) - bound[0] > 2 * top
        assert (np.abs(got[p] - want[0]) <= bound[0])[inside].all()
        assert np.isinf(got[p])[beyond].all()


@pytest.mark.parametrize("quantized", (False, True))
@pytest.mark.parametrize("rows,out,n", ((1, 33, 96), (4, 64, 1440), (5, 300, 160), (5, 4000, 160), (17, 1100, 3168),
                                        (128, 256, 512), (200, 700, 1056), (300, 1500, 1056),
                                        (300, 2100, 1056)))
def test_linear(device, quantized, rows, out, n):
    print(f"linear {quantized} {rows} {out} {n}", flush=True)
    rng = np.random.default_rng(rows)
    codes, s = mxref.random_codes(rng, (out, n))
    line = mx.MxLinear(out, n, device=device)
    line.load(mx.MxTensor(_dev(codes, device), _dev(s, device)))
    for dtype in HALF:
        x, xv = _operand(rng, rows, n, dtype, quantized, device)
        _check(line(x), xv, mxref.values(codes, s)[None], np.zeros(rows, int), dtype)
    one, value = _operand(rng, 1, n, F16, quantized, device)
    one = mx.MxTensor(one.codes[0], one.scales[0], F16) if quantized else one[0]
    assert line(one).shape == (out,)
    assert torch.equal(line.dequantized(F32).cpu(), torch.from_numpy(mxref.values(codes, s)).to(F32))


@pytest.mark.parametrize("rows,out,n", ((4096, 4096, 64), (4100, 4097, 160), (8200, 2050, 416)))
def test_linear_of_many_quantised_rows(device, rows, out, n):
    """Enough 4-bit rows and outputs for the tiles of 256 x 256, the last ones not whole."""
    print(f"linear of many rows {rows} {out} {n}", flush=True)
    rng = np.random.default_rng(rows)
    codes, s = mxref.random_codes(rng, (out, n))
    line = mx.MxLinear(out, n, device=device)
    line.load(mx.MxTensor(_dev(codes, device), _dev(s, device)))
    x, xv = _operand(rng, rows, n, BF16, True, device)
    _check(line(x), xv, mxref.values(codes, s)[None], np.zeros(rows, int), BF16)


def test_scales_and_codes_of_other_layouts(device):
    """Activations whose scales are contiguous, strided, or a slice with NaN
    scales behind the row; codes at an odd address."""
    print("operand layouts", flush=True)
    rng = np.random.default_rng(2)
    for n in (96, 160, 1440):
        module, w = _switch(rng, 2, 32, n, device)
        for rows in (3, 90):
            q, xv = _operand(rng, rows, n, F16, True, device)
            ids = rng.integers(0, 2, rows)
            want = module(_shape(q, rows, 1), _dev(ids, device)).view(rows, 32)
            _check(want, xv, w, ids, F16)
            nb = n // 32
            wide = torch.full((rows, nb + 9), 255, dtype=torch.uint8, device=device)
            wide[:, 4:4 + nb] = q.scales
            room = torch.zeros(q.codes.numel() + 1, dtype=torch.uint8, device=device)
            odd = room[1:].view(q.codes.shape).copy_(q.codes)
            spaced = torch.full((rows, 2 * nb), 255, dtype=torch.uint8, device=device)
            spaced[:, ::2] = q.scales
            aligned = torch.full((rows, (nb + 3) // 4 * 4 + 8), 255, dtype=torch.uint8, device=device)
            aligned[:, :nb] = q.scales
            for codes, scales in ((q.codes, q.scales.contiguous()), (odd, wide[:, 4:4 + nb]),
                                  (q.codes, spaced[:, ::2]), (q.codes, aligned[:, :nb])):
                got = module(_shape(mx.MxTensor(codes, scales), rows, 1), _dev(ids, device)).view(rows, 32)
                assert torch.equal(got, want)


def test_the_same_call_repeats_and_streams_do_not_mix(device):
    print("repeats and streams", flush=True)
    rng = np.random.default_rng(4)
    module, w = _switch(rng, 8, 512, 1024, device)
    side = torch.cuda.Stream()
    x = torch.randn((300, 1, 1, 1024), device=device).to(BF16)
    ids = _dev(rng.integers(0, 8, (300, 2)), device)
    want = [module(x, ids), module(mx.quantize(x), ids), module(x[:9], ids[:9])]
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(side):
            side.wait_stream(torch.cuda.default_stream())
            a = [module(x, ids), module(mx.quantize(x), ids), module(x[:9], ids[:9])]
        b = [module(x, ids), module(mx.quantize(x), ids), module(x[:9], ids[:9])]
        torch.cuda.synchronize()
        for got in (a, b):
            assert all(torch.equal(g, v) for g, v in zip(got, want))


def test_graph_replays(device):
    print("graph", flush=True)
    rng = np.random.default_rng(6)
    module, _ = _switch(rng, 8, 256, 512, device)
    x = torch.randn((90, 1, 1, 512), device=device).to(F16)
    ids = _dev(rng.integers(0, 8, (90, 2)), device, torch.int32)

    def step():
        return module(x, ids), module(mx.quantize(x), ids), module(x[:4], ids[:4])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for seed in range(4):
        x.copy_(torch.randn(x.shape, generator=torch.Generator(device=device).manual_seed(seed), device=device))
        ids.copy_(_dev(rng.integers(0, 8, (90, 2)), device, torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [h.clone() for h in held]
        assert all(torch.equal(g, v) for g, v in zip(got, step()))


def test_state_dict_moves_the_weights(device):
    print("state dict", flush=True)
    module, w = _switch(np.random.default_rng(1), 2, 20, 64, device)
    other = mx.MxSwitchLinear(2, 20, 64, device=device)
    other.load_state_dict({k: v.cpu() for k, v in module.state_dict().items()})
    assert torch.equal(other.dequantized(F32), module.dequantized(F32))


# ---------------------------------------------------------------- refusals ---


def test_refusals(device):
    print("refusals", flush=True)
    zeros = lambda *s, dtype=F16: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    for bad in (zeros(3, 33), zeros(3, 32, dtype=torch.int32), zeros(3, 32, dtype=torch.float64), torch.zeros(3, 32)):
        with pytest.raises(IqkKernelError):
            mx.quantize(bad)
    u8 = lambda *s: zeros(*s, dtype=torch.uint8)  # noqa: E731
    for codes, scales in ((u8(2, 16), u8(2, 2)), (u8(2, 16), u8(3, 1)), (u8(2, 0), u8(2, 0)), (zeros(2, 16), u8(2, 1))):
        with pytest.raises(IqkKernelError):
            mx.MxTensor(codes, scales)
    with pytest.raises(IqkKernelError):
        mx.quantize(zeros(2, 32)).dequantize(torch.float64)
    module = mx.MxSwitchLinear(2, 20, 64, device=device)
    for shape in ((2, 20, 32), (1, 20, 64), (20, 64)):
        with pytest.raises(IqkRuntimeError):
            module.load(mx.quantize(zeros(*shape)))
    with pytest.raises(IqkRuntimeError):
        module.load(zeros(2, 20, 64))
    ids = zeros(3, 2, dtype=torch.int32)
    for x in (zeros(3, 1, 1, 32), zeros(64)):
        with pytest.raises(IqkRuntimeError):
            module(x, ids)
    for x in (zeros(3, 1, 1, 64, dtype=F32), torch.zeros((3, 1, 1, 64), dtype=F16), mx.quantize(zeros(3, 1, 1, 64, dtype=F32)),
              [1.0]):
        with pytest.raises((IqkKernelError, IqkRuntimeError, AttributeError, TypeError)):
            module(x, ids)
    with pytest.raises(IqkKernelError):
        module(zeros(3, 1, 1, 64), zeros(3, 2))
    with pytest.raises(RuntimeError):  # shapes that do not broadcast
        module(zeros(3, 1, 1, 64), zeros(4, 2, dtype=torch.int32))
    grad = zeros(3, 1, 1, 64).requires_grad_()
    with pytest.raises(IqkRuntimeError):
        module(grad, ids)
    with torch.no_grad():
        assert module(grad, ids).shape == (3, 2, 1, 20)


def test_weights_past_32_bits(device):
    """The last expert of a stack whose tiles take more than 4 GiB, by each route."""
    print("weights past 4 GiB", flush=True)
    E, out, n = 1030, 2048, 4096
    g = torch.Generator(device=device).manual_seed(4)
    codes = torch.randint(0, 256, (E, out, n // 2), dtype=torch.uint8, device=device, generator=g)
    scales = torch.randint(110, 126, (E, out, n // 32), dtype=torch.uint8, device=device, generator=g)
    module = mx.MxSwitchLinear(E, out, n, device=device)
    module.load(mx.MxTensor(codes, scales))
    assert module.tiles.numel() > 2 ** 32
    w = mxref.values(codes[-1:].cpu().numpy(), scales[-1:].cpu().numpy())
    del codes, scales
    rng = np.random.default_rng(3)
    for quantized in (False, True):
        for pairs in (3, 40, 2100):
            x, xv = _operand(rng, pairs, n, BF16, quantized, device)
            ids = torch.full((pairs,), E - 1, dtype=torch.int32, device=device)
            y = module(_shape(x, pairs, 1), ids, sorted_indices=pairs > 3).view(pairs, out)
            rows = np.r_[:2, pairs - 1]
            _check(y[torch.from_numpy(rows)], xv[rows], w, np.zeros(3, dtype=np.int64), BF16)


def test_rows_past_32_bits(device):
    """Activations and outputs of more than 4 GiB; quantised, codes of more than 2."""
    print("rows past 4 GiB", flush=True)
    rows, n, out = 1_060_000, 2080, 2096
    rng = np.random.default_rng(9)
    codes, s = mxref.random_codes(rng, (out, n))
    line = mx.MxLinear(out, n, device=device)
    line.load(mx.MxTensor(_dev(codes, device), _dev(s, device)))
    w = mxref.values(codes, s)[None]
    x = torch.randn((rows, n), dtype=BF16, device=device, generator=torch.Generator(device=device).manual_seed(5))
    at = np.r_[0, 1, 530_000, rows - 2, rows - 1]
    index = torch.from_numpy(at).to(device)
    y = line(x)
    assert x.numel() * 2 > 2 ** 32 and y.numel() * 2 > 2 ** 32
    _check(y[index], _f64(x[index]), w, np.zeros(5, dtype=np.int64), BF16)
    del y
    q = mx.quantize(x)
    part = mx.MxTensor(q.codes[index], q.scales[index], BF16)
    _same_codes(part, x[index])
    assert torch.equal(q.dequantize()[index], part.dequantize())
    y = line(q)
    _check(y[index], _f64(part.dequantize(F32)), w, np.zeros(5, dtype=np.int64), BF16)


def test_forward_mode_derivatives_are_refused(device):
    print("mx forward mode", flush=True)
    fwd = torch.autograd.forward_ad
    module, line = mx.MxSwitchLinear(2, 20, 64, device=device), mx.MxLinear(20, 64, device=device)
    ids = torch.zeros((3, 2), dtype=torch.int32, device=device)
    base = torch.randn((3, 1, 1, 64), device=device).to(F16)
    wide = torch.randn((3, 1, 1, 128), device=device).to(F16)[..., ::2]  # copied before the call
    with fwd.dual_level():
        for t in (base, wide):
            x = fwd.make_dual(t, torch.ones_like(t))
            for call in (lambda: mx.quantize(x), lambda: module(x, ids), lambda: module(x, ids, sorted_indices=True),
                         lambda: line(x)):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        assert line(base).shape == (3, 1, 1, 20) and line(wide).shape == (3, 1, 1, 20)


def test_quantising_what_wants_a_gradient_is_refused(device):
    """As a product of it is: codes carry no gradient."""
    print("quantise with gradient", flush=True)
    for dtype in (F32, F16, BF16):
        x = torch.randn((4, 256), device=device).to(dtype).requires_grad_()
        for t in (x, x[:, ::2], x[:, 8:72], x * 2, x[0], x[:0]):
            with pytest.raises(IqkRuntimeError, match="detach"):
                mx.quantize(t)
            want = mx.quantize(t.detach())
            with torch.no_grad():
                got = mx.quantize(t)
            assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)


@pytest.mark.parametrize("quantized", (False, True))
@pytest.mark.parametrize("pairs", (5, 100, 1500))
@pytest.mark.parametrize("exponent", (-112, 0, 118))
def test_small_and_large_bfloat16_rows(device, quantized, pairs, exponent):
    """Activations near both ends of f32, weights of ordinary size (scales of 2^-16 to 2^-6), by
    every route: as exact as between.  The sums stay inside f32."""
    print(f"range {quantized} {pairs} {exponent}", flush=True)
    rng = np.random.default_rng(pairs)
    E, out, n = 2, 48, 256
    module, w = _switch(rng, E, out, n, device, lo=111, hi=121)
    ids = rng.integers(0, E, pairs)
    x = _dev(np.ldexp(np.clip(rng.standard_normal((pairs, n)), -3.9, 3.9), exponent), device, BF16)
    q = mx.quantize(x) if quantized else x
    xv = _f64(q.dequantize(F32) if quantized else x)
    y = module(_shape(q, pairs, 1), _dev(ids, device)).view(pairs, out)
    _check(y, xv, w, ids, BF16)
    line = mx.MxLinear(out, n, device=device)
    one = module.dequantized(F32)[0]
    line.load(mx.quantize(one))
    _check(line(q), xv, _f64(line.dequantized(F32))[None], np.zeros(pairs, int), BF16)


def test_ordinary_rows_are_kept_as_they_are(device):
    """Rows with scales of 2^-13 .. 2^13 have no power of two taken out, others the least that
    brings them there, or their largest to 2^13; blocks without values have no say."""
    print("row exponents", flush=True)
    rows = ([127 - 13, 127 + 13], [120, 118], [127 - 14, 120], [127 - 40, 127 - 37], [127 + 14, 127], [127 + 30, 127 + 10],
            [10, 50], [127 + 60, 127 - 60], [0, 0], [254, 254], [254, 0], [120, 255], [255, 255])
    want = [0, 0, -1, -27, 1, 17, -90, 47, -114, 114, 114, 0, 0]
    codes = np.full((1, len(rows) + 2, 64), 0x3f, dtype=np.uint8)
    s = np.empty((1, len(rows) + 2, 4), dtype=np.uint8)
    s[0, :-2, :2] = rows
    s[0, -2:, :2] = [[130, 5], [5, 130]]
    codes[0, -2, 16:32] = codes[0, -1, :16] = 0x80
    codes[..., 32:] = 0x08
    s[..., 2:] = [3, 250]
    module = mx.MxSwitchLinear(1, len(rows) + 2, 128, device=device)
    module.load(mx.MxTensor(_dev(codes, device), _dev(s, device)))
    assert module.row_exps[0].tolist() == want + [0, 0] + [0]
    values = mxref.values(codes, s)
    values[0, 10, 32:64] = 0  # 2^254 below
    np.testing.assert_array_equal(_f64(module.dequantized(F32)), _f64(torch.from_numpy(values).to(F32)))


@pytest.mark.parametrize("pairs", (5, 100, 1500))
def test_blocks_far_below_their_rows_largest(device, pairs):
    """f16 rows take weights below 2^-36 of the row's largest scale as multiples of 2^-37 of
    it (one product at a time: sums of those are another matter); bf16 and quantised rows hold
    2^-140 of it, below which a block is zero."""
    print(f"blocks apart {pairs}", flush=True)
    rng = np.random.default_rng(31)
    out, n = 48, 160
    codes, s = mxref.random_codes(rng, (1, out, n))
    below = np.array([0, 36, 38, 100, 141])  # powers of two below the row's first block
    s[0] = 160 - below[None] - np.arange(out)[:, None] % 3
    module = mx.MxSwitchLinear(1, out, n, device=device)
    module.load(mx.MxTensor(_dev(codes, device), _dev(s, device)))
    w = mxref.values(codes, s)
    w[..., 128:] = 0
    np.testing.assert_array_equal(_f64(module.dequantized(F32)), w)
    ids = _dev(np.zeros(pairs, int), device)
    for quantized in (False, True):
        for first in (1, 2, 3, 4):  # only from this block on does the row have values
            x = rng.standard_normal((pairs, n))
            x[:, :32 * first] = 0
            t = _dev(x, device, BF16)
            q = mx.quantize(t) if quantized else t
            xv = _f64(q.dequantize(F32) if quantized else t)
            y = _f64(module(_shape(q, pairs, 1), ids).view(pairs, out))
            want, bound = mxref.product_bound(xv, w[0], BF16)
            assert (np.abs(y - want) <= bound).all(), (quantized, first)
    unit = np.ldexp(1.0, s[0, :, :1].astype(int) - 127 - 37)
    rounded = np.rint(w[0] / unit) * unit  # to the nearest, ties to even
    x = np.zeros((pairs, n))
    x[np.arange(pairs), rng.integers(32, n, pairs)] = rng.standard_normal(pairs)
    t = _dev(x, device, F16)
    y = _f64(module(_shape(t, pairs, 1), ids).view(pairs, out))
    want = _f64(t) @ rounded.T
    assert (np.abs(y - want) <= mxref.HALF_ULP[F16] * np.abs(want) + mxref.TINY[F16]).all()
