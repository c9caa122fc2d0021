"""Low-rank adapters of many requests beside a projection that they share.

A server holds one set of weights and many small corrections to it: request by request
``W x + s B (A x)`` with ``A`` ``[rank, in]`` and ``B`` ``[out, rank]``.
:class:`LowRankAdapters` keeps a bank of them and adds each row's own to the projection's
output; :class:`~mlx_iqk_amd.mx.MxLinear` takes one in its call.

Products are exact and summed in f32, the sum with the projection's output is rounded
once.  A call repeats bit for bit; a row's last bits may differ between calls that hold other
rows beside it.  Adapters are for serving: no gradient flows through, and rows that want one, or have
a forward-mode derivative, are refused, as the projections refuse them.
"""

from __future__ import annotations

import torch

from . import _native
from .kernels import IqkKernelError
from .nn import _KERNEL_IDS, IqkRuntimeError, _pairs_per_x_row

MAX_ADAPTERS = 1024
MAX_RANK = 256
_HALF = (torch.float16, torch.bfloat16)


class LowRankAdapters(torch.nn.Module):
    """``num_adapters`` adapters of up to ``rank`` for a projection ``[out, in]``, as buffers in
    the kernels' layout, eight values of the reduction axis together (R: the rank rounded
    up to a multiple of 8):

    * ``down`` 16-bit ``[num_adapters, in/8, R, 8]`` and ``up`` ``[num_adapters, R/8, out, 8]``;
    * ``scales`` f32 ``[num_adapters]``.

    All zeros, which add nothing, until :meth:`load`; :meth:`adapter` gives one back.  Of the ranks up to R those
    past an adapter's own are zeros, with which an infinity in a row of ``x`` gives NaN.  An
    infinity in an adapter makes sums of its rows infinite or NaN.  ``scales`` stay f32: a bank that a model's ``half()`` or
    ``to(dtype)`` has cast is refused, so cast first and make the bank after.
    """

    def __init__(self, num_adapters: int, out_features: int, in_features: int, rank: int,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        super().__init__()
        self.num_adapters, self.out_features = int(num_adapters), int(out_features)
        self.in_features, self.rank = int(in_features), int(rank)
        if not 0 < self.num_adapters <= MAX_ADAPTERS:
            raise IqkRuntimeError(f"a bank holds 1 .. {MAX_ADAPTERS} adapters, got {num_adapters}")
        if not 0 < self.rank <= MAX_RANK:
            raise IqkRuntimeError(f"an adapter's rank is 1 .. {MAX_RANK}, got {rank}")
        if self.in_features <= 0 or self.in_features % 8:
            raise IqkRuntimeError(f"in_features must be a positive multiple of 8, got {in_features}")
        if self.out_features <= 0:
            raise IqkRuntimeError(f"out_features must be positive, got {out_features}")
        if dtype not in _HALF:
            raise IqkRuntimeError(f"adapters are float16 or bfloat16, got {dtype}")
        ranks = (self.rank + 7) // 8 * 8
        self.register_buffer("down", torch.zeros((self.num_adapters, self.in_features // 8, ranks, 8), dtype=dtype,
                                                 device=device))
        self.register_buffer("up", torch.zeros((self.num_adapters, ranks // 8, self.out_features, 8), dtype=dtype,
                                               device=device))
        self.register_buffer("scales", torch.zeros(self.num_adapters, dtype=torch.float32, device=device))

    def load(self, index: int, down: torch.Tensor, up: torch.Tensor, scale: float = 1.0) -> None:
        """Take adapter ``index``: ``down`` ``[r, in]`` and ``up`` ``[out, r]``, r up to the
        bank's rank, rounded to its type; ``scale`` is alpha / r, say.  Ranks past r become zeros."""
        if not 0 <= index < self.num_adapters:
            raise IqkRuntimeError(f"the bank holds adapters 0 .. {self.num_adapters - 1}, got {index}")
        if down.dim() != 2 or up.dim() != 2 or down.shape[0] != up.shape[1] or not 0 < down.shape[0] <= self.rank \
                or down.shape[1] != self.in_features or up.shape[0] != self.out_features:
            raise IqkRuntimeError(f"an adapter is [r, {self.in_features}] and [{self.out_features}, r] with r up to "
                                  f"{self.rank}, got {tuple(down.shape)} and {tuple(up.shape)}")
        r, a, b = down.shape[0], self.down[index], self.up[index]
        whole = r // 8 * 8
        with torch.no_grad():
            (a if r == a.shape[1] else a[:, :r]).copy_(down.reshape(r, -1, 8).transpose(0, 1))
            if whole:
                b[:whole // 8].copy_(up[:, :whole].reshape(-1, whole // 8, 8).transpose(0, 1))
            if r < a.shape[1]:
                a[:, r:].zero_()
                b[whole // 8:].zero_()
                if whole < r:
                    b[whole // 8, :, :r - whole].copy_(up[:, whole:])
            self.scales[index].fill_(float(scale))

    def adapter(self, index: int) -> tuple[torch.Tensor, torch.Tensor, float]:
        """Adapter ``index`` as :meth:`load` takes it, of rank R: ``(down, up, scale)``."""
        if not 0 <= index < self.num_adapters:
            raise IqkRuntimeError(f"the bank holds adapters 0 .. {self.num_adapters - 1}, got {index}")
        down, up = (blocks[index].transpose(0, 1).flatten(1) for blocks in (self.down, self.up))
        return down, up, float(self.scales[index])

    def forward(self, x: torch.Tensor, ids: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
        """``y + scales[a] up[a] (down[a] x)`` with each row's own ``a``, in y's type.

        ``x`` is ``[..., in]`` and ``y`` ``[..., out]``, both of the bank's type; ``ids`` (integers)
        has their leading shape, or 1 from some dimension on: one id for all rows below it (a
        request's).  A row with an id of -1 keeps its y, one with another id outside the bank
        becomes NaN.
        """
        return self._add(x, ids, y, None)

    def _called_as_it_is(self) -> bool:
        """Whether a call of the module is :meth:`_add` and nothing else, so that it can be made in y's place: no
        other ``forward``, no hooks."""
        return type(self).forward is LowRankAdapters.forward and "forward" not in self.__dict__ \
            and not (self._forward_hooks or self._forward_pre_hooks or torch.nn.modules.module._has_any_global_hook())

    def _add(self, x, ids, y, out) -> torch.Tensor:
        buffers, add = self._buffers, _native.torch_binding().adapters
        down, up, scales = buffers["down"], buffers["up"], buffers["scales"]
        if (got := add(x, ids, y, down, up, scales, out)) is not None:
            return got
        # what the kernels do not take as it is
        dtype = down.dtype
        if not down.is_cuda:
            raise IqkKernelError(f"the bank must live on a GPU, got {down.device}")
        if dtype not in _HALF or up.dtype != dtype or scales.dtype != torch.float32:
            raise IqkKernelError(f"the bank holds 16-bit down and up and float32 scales, got {dtype}, {up.dtype} and "
                                 f"{scales.dtype}")
        for name, t, n in (("x", x, self.in_features), ("y", y, self.out_features)):
            if not isinstance(t, torch.Tensor) or t.dim() < 1:
                raise IqkKernelError(f"{name} must be a tensor of at least one dimension")
            if t.device != down.device:
                raise IqkKernelError(f"{name} is on {t.device}, the bank on {down.device}")
            if t.dtype != dtype:
                raise IqkKernelError(f"{name} must be {dtype}, as the bank is, got {t.dtype}")
            if t.shape[-1] != n:
                raise IqkRuntimeError(f"{name} has rows of {t.shape[-1]} values, the bank takes {n}")
            if t.requires_grad and torch.is_grad_enabled():
                raise IqkRuntimeError(f"no gradient flows back to {name} through the adapters: detach it, or call under "
                                      "torch.no_grad()")
        lead = x.shape[:-1]
        if y.shape[:-1] != lead:
            raise IqkRuntimeError(f"x {tuple(x.shape)} and y {tuple(y.shape)} are not of the same rows")
        if not isinstance(ids, torch.Tensor) or ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
            raise IqkKernelError("ids must be an integer tensor")
        if ids.device != down.device:
            raise IqkKernelError(f"ids are on {ids.device}, the bank on {down.device}")
        if ids.dim() != len(lead) or _pairs_per_x_row(ids.shape, lead) is None:
            raise IqkRuntimeError(f"ids {tuple(ids.shape)} must have the rows' shape {tuple(lead)}, or 1 from some "
                                  "dimension on")
        if not x.numel():
            return y.clone() if out is None else out
        if ids.dtype not in _KERNEL_IDS:
            wraps = ids.dtype == torch.uint64  # 2**63 and more: not -1, but outside
            ids = torch.clamp(ids.to(torch.int64), -2, self.num_adapters)
            if wraps:
                ids = ids.masked_fill(ids < 0, self.num_adapters)
        return add(x.contiguous(), ids.contiguous(), y.contiguous(), down.contiguous(), up.contiguous(),
                   scales.contiguous(), out)

    def extra_repr(self) -> str:
        return f"{self.num_adapters}, {self.out_features}, {self.in_features}, rank={self.rank}"


__all__ = ["MAX_ADAPTERS", "MAX_RANK", "LowRankAdapters"]
