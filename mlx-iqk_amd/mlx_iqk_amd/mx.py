"""4-bit microscaled floats: quantisation, and projections whose weights are in them.

The format (the OCP microscaling MXFP4): 32 consecutive values along the last
axis share a scale ``2**(byte - 127)`` (byte 255: the block is NaN) and hold four
bits each, a sign and an index into 0, 0.5, 1, 1.5, 2, 3, 4, 6; 4.25 bits a
value.  A byte holds two codes, the even position's in its low half.

* :func:`quantize` / :func:`dequantize` convert tensors on the GPU;
* :class:`MxSwitchLinear` is the routed projection of
  :class:`~mlx_iqk_amd.nn.IqkSwitchLinear` over experts in this format: the same
  ``(x, indices, sorted_indices)`` call, shapes and treatment of ids out of range;
* :class:`MxLinear` is one such matrix.

Both projections take 16-bit activations, whose products with the weights are
exact and summed in f32, or an :class:`MxTensor`, quantised activations, which the
matrix cores multiply with the weights as they are, at four times the rate.

A row of weights whose scales do not lie within 2**-13 .. 2**13 is brought there by a power
of two before the products, which the sums get back.  What that costs: where the row's
scales are more than 2**26 apart, float16 activations meet weights under 2**-27 of the
largest scale in fewer bits, under 2**-36 as multiples of 2**-37 of it; and a block more than
2**140 below the row's largest is zero, in :meth:`~MxSwitchLinear.dequantized` too.  Sums of
such a row overflow where the scaled ones do, those of other rows where f32 does.

Outputs are rounded once.  The weights are frozen: no gradient flows through, and an
x that wants one, or has a forward-mode derivative, is refused.

Like every launch of this package, these run asynchronously on torch's current
stream, and raise where no GPU library is built; nothing falls back to the CPU.
"""

from __future__ import annotations

import math

import torch

from . import _native
from .kernels import ROUTE_MAX_EXPERTS, IqkKernelError, _require_cuda, _stream_ptr
from .nn import _KERNEL_IDS, IqkRuntimeError, _pairs_per_x_row

BLOCK = 32
"""Values that share a scale."""
_STEP = 128
_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_ACTS = {(torch.float16, False): 0, (torch.bfloat16, False): 1, (torch.float16, True): 2, (torch.bfloat16, True): 3}



def pair_limit(num_experts: int) -> int:
    """Token-expert pairs up to which each is computed on its own; beyond, experts are
    named so often that their weights are better read once for all their pairs.

    A token's experts distinct, else uniform, us alone and grouped, for 16-bit and for
    4-bit activations, whose pairs are a little cheaper: [2048 x 4096], 8 experts: 12 pairs
    9.3, 9.9 (8.4, 10.1), 16 pairs 10.2, 9.8 (8.7, 10.1); 16 experts: 16 pairs 12.3, 13.4
    (11.4, 13.4), 24 pairs 15.9, 15.5 (14.1, 15.5); 128 experts: 48 pairs 31.7, 36.4 (31.8,
    35.8), 72 pairs 45.0, 40.2 (44.6, 40.2); 256 experts: 72 pairs 47.1, 53.7 (45.1, 53.1),
    96 pairs 66.3, 65.3 (61.3, 65.9).  Of other sizes: [1000 x 1440], 60 experts: 42 pairs
    8.4, 9.4 (7.9, 9.9), 66 pairs 11.1, 10.7 (10.5, 11.7); [4096 x 2048], 256 experts: 120
    pairs 79, 85 (76, 84); [512 x 1024], 64 experts: 66 pairs 5.3, 7.1 (4.7, 8.0).
    """
    return min(num_experts + 6, 48 + num_experts // 6)


ROW_LIMIT = 16384
"""Outputs in all up to which the rows of an :class:`MxLinear` are computed on their
own (4096 columns, 16-bit activations and 4-bit ones: 2048 outputs, 8 rows 5.5 us
against 6.6 and 4.4 against 6.3, 16 rows 8.6 against 7.9 and 6.7 against 7.2; 8192 outputs, 2
rows 6.7 against 6.4 and 5.9 against 6.5, 4 rows 9.9 against 6.6 and 8.3 against 6.7)."""


def _refuse_gradient(x: torch.Tensor) -> None:
    if x.requires_grad and torch.is_grad_enabled():
        raise IqkRuntimeError("no gradient flows back to x through 4-bit codes or the projections: detach x, or call "
                              "under torch.no_grad()")


def _check_width(n: int) -> int:
    if n <= 0 or n % BLOCK:
        raise IqkKernelError(f"a row of {n} values is not whole blocks of {BLOCK}")
    return n


class MxTensor:
    """Codes ``u8 [..., n/2]`` and scales ``u8 [..., n/32]`` of a tensor ``[..., n]``.

    ``dtype`` is the type of the tensor that was quantised: what
    :meth:`dequantize` returns, and a projection of these values.
    """

    __slots__ = ("codes", "scales", "dtype")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.float16):
        for name, t in (("codes", codes), ("scales", scales)):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.dim() < 1:
                raise IqkKernelError(f"{name} must be a uint8 tensor of at least one dimension")
        if dtype not in _DTYPES:
            raise IqkKernelError(f"dtype must be one of {tuple(_DTYPES)}, got {dtype}")
        if codes.device != scales.device:
            raise IqkKernelError(f"codes are on {codes.device}, scales on {scales.device}")
        if codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != scales.shape[-1] * (BLOCK // 2) \
                or not scales.shape[-1]:
            raise IqkKernelError(f"codes {tuple(codes.shape)} and scales {tuple(scales.shape)} do not describe blocks "
                                 f"of {BLOCK} values (16 bytes and one scale each)")
        self.codes, self.scales, self.dtype = codes, scales, dtype

    @classmethod
    def _of(cls, codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> "MxTensor":
        """One of tensors known to belong together."""
        q = cls.__new__(cls)
        q.codes, q.scales, q.dtype = codes, scales, dtype
        return q

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], 2 * self.codes.shape[-1]))

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def dequantize(self, dtype: torch.dtype | None = None) -> torch.Tensor:
        """The values the codes stand for (:func:`dequantize`)."""
        return dequantize(self, dtype)

    def __repr__(self) -> str:
        return f"MxTensor({tuple(self.shape)}, {self.dtype}, {self.device})"


def _row_stride(t: torch.Tensor) -> int | None:
    """Elements from row to row of t taken as [rows, n], the last axis dense;
    None where rows are not evenly spaced."""
    if t.is_contiguous():
        return t.shape[-1]
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        return None
    stride = span = None
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if span is None:
            stride, span = step, size * step
        elif step == span:
            span = size * step
        else:
            return None
    return t.shape[-1] if stride is None else stride


def _aligned_codes(codes: torch.Tensor) -> torch.Tensor:
    """Codes, contiguous and at a 16-byte boundary."""
    codes = codes.contiguous()
    return codes if codes.data_ptr() % 16 == 0 else codes.clone()


def _product_scales(q: MxTensor) -> tuple[torch.Tensor, int]:
    """Scales as the products read an activation row's, four at a time: rows at
    multiples of four bytes with room for whole groups of four."""
    n = q.scales.shape[-1]
    if n % 4 == 0 and q.scales.is_contiguous() and q.scales.data_ptr() % 4 == 0:
        return q.scales, n
    rows, need = math.prod(q.scales.shape[:-1]), 4 * ((n + 3) // 4)
    stride = _row_stride(q.scales)
    if rows == 1 and stride is not None:
        stride = max(stride, need) // 4 * 4
    if stride is not None and stride % 4 == 0 and stride >= need and q.scales.data_ptr() % 4 == 0:
        left = q.scales.untyped_storage().nbytes() - q.scales.storage_offset()
        if (rows - 1) * stride + need <= left:
            return q.scales, stride
    room = torch.empty((rows, need), dtype=torch.uint8, device=q.scales.device)
    room[:, :n] = q.scales.reshape(rows, n)
    return room, need


def quantize(x: torch.Tensor) -> MxTensor:
    """``x`` (f32, f16 or bf16 ``[..., n]`` on a GPU, ``n`` a multiple of 32) in 4 bits.

    A block's scale is ``2**(floor(log2(largest magnitude)) - 2)``, at least
    2**-127; values round to nearest, ties to the even code, and saturate at 6
    scales.  A block that holds a NaN or an infinity becomes NaN.  Codes carry no
    gradient: an ``x`` that wants one is refused, as the projections refuse it.
    """
    if not isinstance(x, torch.Tensor):
        raise IqkKernelError("x must be a tensor of at least one dimension")
    binding, dtype = _native.torch_binding(), x.dtype
    if (got := binding.mx_quantize(x, 0)) is not None:
        return MxTensor._of(*got, dtype)
    # what the binding does not take as it is
    if x.dim() < 1:
        raise IqkKernelError("x must be a tensor of at least one dimension")
    if not x.is_cuda:
        raise IqkKernelError(f"x must live on a GPU, got {x.device}")
    if dtype not in _DTYPES:
        raise IqkKernelError(f"x must be one of {tuple(_DTYPES)}, got {dtype}")
    n = _check_width(x.shape[-1])
    _refuse_gradient(x)
    stride, at = n, x.data_ptr()
    if not x.is_contiguous() or at % 16:
        stride = _row_stride(x)
        if stride is None or stride < n or stride % (16 // x.element_size()) or at % 16:
            x, stride = x.contiguous(), n
            if x.data_ptr() % 16:
                x = x.clone()
    return MxTensor._of(*binding.mx_quantize(x, stride), dtype)


def dequantize(q: MxTensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values of ``q``, rounded once to ``dtype`` (its own by default; a
    value is exact in f32 and, but for the smallest scales, in bf16)."""
    dtype = q.dtype if dtype is None else dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise IqkKernelError(f"dtype must be one of {tuple(_DTYPES)}, got {dtype}")
    codes, scales, binding = q.codes, q.scales, _native.torch_binding()
    if (values := binding.mx_dequantize(codes, scales, 0, code)) is not None:
        return values
    if not codes.is_cuda:
        raise IqkKernelError(f"codes must live on a GPU, got {codes.device}")
    codes, stride = _aligned_codes(codes), _row_stride(scales)
    if stride is None or stride < scales.shape[-1]:
        scales, stride = scales.contiguous(), scales.shape[-1]
    return binding.mx_dequantize(codes, scales, stride, code)


class _MxStack(torch.nn.Module):
    """``num_experts`` matrices ``[out, in]`` in the products' layout, as buffers:

    * ``tiles`` u8 ``[E, out/16, in/128, 64, 16]``, the codes in the order that a
      wavefront loads them;
    * ``tile_scales`` u8 ``[E, in/128, out/64, 64, 4]``, the blocks' scales over their
      row's power of two;
    * ``row_exps`` i32 ``[E, out]``, that power: 0 for a row whose scales lie within
      2**-13 .. 2**13.

    ``out`` and ``in`` round up to whole tiles; 4.27 bits a weight.
    """

    def __init__(self, num_experts: int, out_features: int, in_features: int, device=None):
        super().__init__()
        self.num_experts, self.out_features = int(num_experts), int(out_features)
        self.in_features = _check_width(int(in_features))
        if not 0 < self.num_experts <= ROUTE_MAX_EXPERTS:
            raise IqkRuntimeError(f"a stack holds 1 .. {ROUTE_MAX_EXPERTS} experts (num_experts={num_experts})")
        if self.out_features <= 0:
            raise IqkRuntimeError(f"out_features must be positive, got {out_features}")
        rows, steps = (self.out_features + 15) // 16 * 16, (self.in_features + _STEP - 1) // _STEP
        E = self.num_experts
        self._pair_limit = min(pair_limit(E), 2 ** 27 // rows)  # 2**23 workgroups of 16 outputs can be launched
        self.register_buffer("tiles", torch.zeros((E, rows // 16, steps, 64, 16), dtype=torch.uint8, device=device))
        self.register_buffer("tile_scales", torch.zeros((E, steps, (rows + 63) // 64, 64, 4), dtype=torch.uint8,
                                                        device=device))
        self.register_buffer("row_exps", torch.zeros((E, rows), dtype=torch.int32, device=device))

    def _load(self, codes: torch.Tensor, scales: torch.Tensor) -> None:
        device = self.tiles.device
        if device.type != "cuda":
            raise IqkKernelError(f"the module must live on a GPU to load weights, got {device}")
        q = MxTensor(codes.to(device), scales.to(device))
        codes, scales, stride = _aligned_codes(q.codes), q.scales, _row_stride(q.scales)
        if stride is None or stride < self.in_features // BLOCK:
            scales, stride = scales.contiguous(), self.in_features // BLOCK
        rc = _native.load().iqk_mx_pack(self.in_features, self.out_features, self.num_experts, codes.data_ptr(),
                                        scales.data_ptr(), stride, self.tiles.data_ptr(), self.tile_scales.data_ptr(),
                                        self.row_exps.data_ptr(), _stream_ptr(device))
        _native.check(rc, f"iqk_mx_pack({self.num_experts}x{self.out_features}x{self.in_features})")

    def _dequantized(self, dtype: torch.dtype) -> torch.Tensor:
        if dtype not in _DTYPES:
            raise IqkKernelError(f"dtype must be one of {tuple(_DTYPES)}, got {dtype}")
        _require_cuda(self.tiles, "the module", torch.uint8)
        y = torch.empty((self.num_experts, self.out_features, self.in_features), dtype=dtype, device=self.tiles.device)
        rc = _native.load().iqk_mx_unpack(_DTYPES[dtype], self.in_features, self.out_features, self.num_experts,
                                          self.tiles.data_ptr(), self.tile_scales.data_ptr(), self.row_exps.data_ptr(),
                                          y.data_ptr(), _stream_ptr(y.device))
        _native.check(rc, f"iqk_mx_unpack({self.num_experts}x{self.out_features}x{self.in_features})")
        return y

    def _activations(self, x, tiles: torch.Tensor) -> tuple:
        """x's rows as the kernels take them: (act, rows, scales, scale stride)."""
        mx = isinstance(x, MxTensor)
        if not mx and not isinstance(x, torch.Tensor):
            raise IqkKernelError("x must be a tensor or an MxTensor")
        rows = x.codes if mx else x
        if not rows.is_cuda or rows.get_device() != tiles.get_device():
            raise IqkKernelError(f"x is on {x.device}, the module on {tiles.device}; both must be on one GPU")
        act = _ACTS.get((x.dtype, mx))
        if act is None:
            raise IqkKernelError(f"activations are float16 or bfloat16, or quantised from them; got {x.dtype}")
        width = 2 * rows.shape[-1] if mx else rows.shape[-1]
        if width != self.in_features:
            raise IqkRuntimeError(f"x has rows of {width} values, the weights take {self.in_features}")
        if mx:
            return (act, _aligned_codes(rows), *_product_scales(x))
        _refuse_gradient(rows)
        if not rows.is_contiguous() or rows.data_ptr() % 16:
            rows = rows.contiguous()
            rows = rows if rows.data_ptr() % 16 == 0 else rows.clone()
        return act, rows, None, 0

    def _project(self, x: tuple, ids, shape: tuple, pairs: int, M: int, per_row: int, grouped: bool) -> torch.Tensor:
        """Outputs ``shape`` of the activations ``x`` (:meth:`_activations`' first four)."""
        act, rows, scales, stride = x
        buffers = self._buffers  # without Module.__getattr__'s lookups
        return _native.torch_binding().mx_project(
            act, rows, scales, stride, buffers["tiles"], buffers["tile_scales"], buffers["row_exps"], ids, shape,
            self.in_features, pairs, M, per_row, grouped)

    def extra_repr(self) -> str:
        return f"{self.num_experts}, {self.out_features}, {self.in_features}"


class MxSwitchLinear(_MxStack):
    """One routed projection: ``num_experts`` 4-bit ``[out, in]`` matrices, called
    with ``(x, indices)`` as :class:`~mlx_iqk_amd.nn.IqkSwitchLinear` is: x
    ``[..., M, in]`` whose leading shape broadcasts with indices ``[..., top_k]``,
    outputs ``[..., top_k, M, out]`` in x's type.  An id outside the stack gives
    rows of NaN."""

    mode = "mx"

    def load(self, weights: MxTensor) -> None:
        """Take the codes and scales of ``weights`` ``[num_experts, out, in]``."""
        want = (self.num_experts, self.out_features, self.in_features)
        if not isinstance(weights, MxTensor) or tuple(weights.shape) != want:
            raise IqkRuntimeError(f"weights must be an MxTensor {want}, got "
                                  f"{tuple(weights.shape) if hasattr(weights, 'shape') else type(weights).__name__}")
        self._load(weights.codes, weights.scales)

    def dequantized(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """The weights' values ``[num_experts, out, in]``, rounded once to ``dtype``."""
        return self._dequantized(dtype)

    def forward(self, x, indices: torch.Tensor, sorted_indices: bool = False) -> torch.Tensor:
        """Project ``x`` through the experts named by ``indices``: few pairs
        each on its own (:func:`pair_limit`), else (or with ``sorted_indices``) grouped
        by expert on the device."""
        if len(x.shape) < 2:
            raise IqkRuntimeError(f"x must be [..., M, {self.in_features}], got {tuple(x.shape)}")
        tiles = self._buffers["tiles"]
        act, rows, scales, stride = self._activations(x, tiles)
        *xbatch, M, _ = rows.shape
        batch = indices.shape
        per_row = _pairs_per_x_row(xbatch, batch)
        if per_row is None:
            batch = torch.broadcast_shapes(xbatch, batch)
            per_row = _pairs_per_x_row(xbatch, batch)
        if per_row is None:  # x broadcasts over leading dimensions: a row of its own for each pair
            rows = rows.expand(*batch, M, rows.shape[-1]).contiguous()
            if scales is not None:
                n = self.in_features // BLOCK
                scales, stride = _product_scales(MxTensor(rows, x.scales.expand(*batch, M, n).contiguous()))
            per_row = 1
        ids = indices
        if ids.dtype not in _KERNEL_IDS or ids.shape != batch or not ids.is_contiguous() \
                or ids.get_device() != tiles.get_device():
            ids = self._ids(indices, batch)
        pairs = math.prod(batch)
        grouped = sorted_indices or M != 1 or pairs > self._pair_limit
        return self._project((act, rows, scales, stride), ids, (*batch, M, self.out_features), pairs, M, per_row,
                             grouped)

    def _ids(self, indices: torch.Tensor, batch) -> torch.Tensor:
        """Expert ids of the pairs in order, of a type the kernels read.  Other
        integers are clamped so that none wraps into the stack."""
        if indices.is_floating_point() or indices.is_complex() or indices.dtype == torch.bool:
            raise IqkKernelError(f"indices must be integers, got {indices.dtype}")
        ids = indices if indices.device == self.tiles.device else indices.to(self.tiles.device)
        if tuple(ids.shape) != tuple(batch):
            ids = ids.broadcast_to(batch)
        if ids.dtype not in _KERNEL_IDS:
            ids = torch.clamp(ids.to(torch.int64), -1, self.num_experts)
        return ids.reshape(-1).contiguous()


class MxLinear(_MxStack):
    """One 4-bit ``[out, in]`` matrix: x ``[..., in]`` to ``[..., out]`` in x's type."""

    mode = "mx"

    def __init__(self, out_features: int, in_features: int, device=None):
        super().__init__(1, out_features, in_features, device)

    def load(self, weights: MxTensor) -> None:
        """Take the codes and scales of ``weights`` ``[out, in]``."""
        want = (self.out_features, self.in_features)
        if not isinstance(weights, MxTensor) or tuple(weights.shape) != want:
            raise IqkRuntimeError(f"weights must be an MxTensor {want}, got "
                                  f"{tuple(weights.shape) if hasattr(weights, 'shape') else type(weights).__name__}")
        self._load(weights.codes, weights.scales)

    def dequantized(self, dtype: torch.dtype = torch.float16) -> torch.Tensor:
        """The weights' values ``[out, in]``, rounded once to ``dtype``."""
        return self._dequantized(dtype)[0]

    def forward(self, x) -> torch.Tensor:
        tiles = self._buffers["tiles"]
        x = self._activations(x, tiles)
        lead = x[1].shape[:-1]
        n = math.prod(lead)
        return self._project(x, None, (*lead, self.out_features), n, 1, 1, n > 1 and n * self.out_features > ROW_LIMIT)

    def extra_repr(self) -> str:
        return f"{self.out_features}, {self.in_features}"


__all__ = ["BLOCK", "ROW_LIMIT", "MxLinear", "MxSwitchLinear", "MxTensor", "dequantize", "pair_limit", "quantize"]
