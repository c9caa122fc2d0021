"""The router of a layer of experts: which experts a token goes to, with what
weights, the loss that keeps the experts evenly loaded, and the tokens' rows on their
way to the experts and back; with gradients.

:func:`topk`'s ids are the ``indices`` of the switch modules
(:class:`~mlx_iqk_amd.nn.IqkSwitchLinear`, :class:`~mlx_iqk_amd.mx.MxSwitchLinear`),
its weights scale their outputs, which :func:`combine` sums.  Experts that want each
one's rows together (a caller's own products, ``gemv_union``) get them from
:func:`dispatch`, or their order from :func:`sort`, and :func:`combine` takes the rows
back in that order.  Logits and rows are f32, f16 or bf16 on a GPU, for up to
1024 experts; sums, probabilities, weights and losses are f32.  Gradients are
not differentiable again, and tensors with a forward-mode derivative are refused.
The calls can be captured in a graph; their gradients cannot, and raise under a capture.
"""

from __future__ import annotations

import math

import torch

from . import _native
from .kernels import IqkKernelError
from .mx import _DTYPES
from .nn import _KERNEL_IDS

MAX_EXPERTS = 1024
MAX_K = 64
MAX_GROUPS = 65535
"""Losses of one :func:`balance_loss` call."""
MAX_COLS = 2 ** 28
"""Rows that :func:`dispatch` and :func:`combine` move are shorter than this."""


def _check_logits(logits: torch.Tensor, dims: int) -> int:
    if not isinstance(logits, torch.Tensor) or logits.dim() < dims:
        raise IqkKernelError(f"logits must be a tensor of at least {dims} dimensions")
    if not logits.is_cuda:
        raise IqkKernelError(f"logits must live on a GPU, got {logits.device}")
    if logits.dtype not in _DTYPES:
        raise IqkKernelError(f"logits must be one of {tuple(_DTYPES)}, got {logits.dtype}")
    experts = int(logits.shape[-1])
    if not 0 < experts <= MAX_EXPERTS:
        raise IqkKernelError(f"a router takes 1 .. {MAX_EXPERTS} experts, got {experts}")
    return experts


def topk(logits: torch.Tensor, k: int, *, normalize: bool = True) -> tuple[torch.Tensor, torch.Tensor]:
    """The ``k`` experts of each token: ``(weights f32 [..., k], ids i32 [..., k])``.

    ``logits`` is ``[..., experts]``.  Ids are in falling order of their logits,
    ties to the lowest expert, NaN above all.  Weights are the softmax over the
    chosen (``normalize``), or over all experts.  Experts with -inf are
    masked: weight 0, chosen only where fewer than ``k`` others are left; a
    token with nothing else gets weights 0.  Differentiable in the logits.
    """
    experts = _check_logits(logits, 1)
    k = int(k)
    if not 0 < k <= min(MAX_K, experts):
        raise IqkKernelError(f"k must be 1 .. {min(MAX_K, experts)} of {experts} experts, got {k}")
    if not logits.is_contiguous():
        logits = logits.contiguous()
    return _native.torch_binding().topk(logits, k, normalize)


def balance_loss(logits: torch.Tensor, ids: torch.Tensor, *,
                 mask: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """How unevenly tokens fall on experts: ``(loss f32 [...], counts i32 [..., experts])``.

    ``logits`` is ``[..., tokens, experts]``, ``ids`` the chosen experts ``[..., tokens,
    k]``; each leading index (a sequence, say) has a loss of its own, up to
    :data:`MAX_GROUPS` of them.  With n
    tokens, ``f_e = counts_e / (k n)`` the share of the pairs that name expert e
    and ``P_e`` the mean of its softmax probability, ``loss = experts * sum_e f_e
    P_e``: 1 where either is even, up to ``experts / k`` where the same k experts
    take all.  Tokens whose ``mask`` (bool ``[..., tokens]``) is false are left out;
    with none left the loss is 0.  Ids outside the stack count for none.  A NaN in
    a token that is kept makes its loss and its own gradient NaN.
    Differentiable in the logits (through ``P``; counts are constants).
    """
    experts = _check_logits(logits, 2)
    if not isinstance(ids, torch.Tensor) or ids.is_floating_point() or ids.dtype == torch.bool:
        raise IqkKernelError("ids must be an integer tensor")
    if ids.device != logits.device or tuple(ids.shape[:-1]) != tuple(logits.shape[:-1]):
        raise IqkKernelError(f"ids {tuple(ids.shape)} on {ids.device} do not belong to logits {tuple(logits.shape)} "
                             f"on {logits.device}")
    k = int(ids.shape[-1])
    if not 0 < k <= min(MAX_K, experts):
        raise IqkKernelError(f"a token has 1 .. {min(MAX_K, experts)} of {experts} experts, got {k}")
    groups = math.prod(logits.shape[:-2])
    if groups > MAX_GROUPS:
        raise IqkKernelError(f"a call gives at most {MAX_GROUPS} losses, logits {tuple(logits.shape)} ask for {groups}")
    if mask is not None:
        if mask.dtype != torch.bool or mask.device != logits.device or tuple(mask.shape) != tuple(logits.shape[:-1]):
            raise IqkKernelError(f"mask must be bool {tuple(logits.shape[:-1])} on {logits.device}, got {mask.dtype} "
                                 f"{tuple(mask.shape)} on {mask.device}")
        mask = mask.contiguous()
    if ids.dtype != torch.int32:
        ids = torch.clamp(ids.to(torch.int64), -1, experts).to(torch.int32)
    return _native.torch_binding().balance(logits.contiguous(), ids.contiguous(), mask)


class _Slots:
    __slots__ = ("_permutation",)  # an order's slots, where they are known to be one


class Order(_Slots):
    """Token-expert pairs in the order of their experts (:func:`sort`): int32 tensors on
    the ids' device,

    * ``offsets`` ``[num_experts + 1]``: expert e's slots are ``offsets[e] .. offsets[e + 1]``,
      and those from ``offsets[num_experts]`` on belong to the pairs left out;
    * ``ids`` ``[pairs]``: each slot's expert, ``num_experts`` where left out;
    * ``tokens`` ``[pairs]``: each slot's token;
    * ``slots`` ``[..., k]``: each pair's slot, a permutation.

    Within an expert the pairs keep their order.  :func:`combine` also takes an order with other
    slots: one outside ``0 .. pairs - 1`` (-1, say) leaves its pair out, and one of several pairs
    counts for each of them.
    """

    __slots__ = ("offsets", "ids", "tokens", "slots")

    def __init__(self, offsets: torch.Tensor, ids: torch.Tensor, tokens: torch.Tensor, slots: torch.Tensor):
        self.offsets, self.ids, self.tokens, self.slots = offsets, ids, tokens, slots
        self._permutation = None

    def __reduce__(self):  # a copy's slots may have been changed before
        return Order, (self.offsets, self.ids, self.tokens, self.slots)

    @property
    def num_experts(self) -> int:
        return self.offsets.shape[0] - 1

    def __repr__(self) -> str:
        return f"Order({tuple(self.slots.shape)} pairs of {self.num_experts} experts, {self.slots.device})"


def _check_ids(ids: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, int]:
    """The pairs' ids as the kernels read them, and the experts' count."""
    if not isinstance(ids, torch.Tensor) or ids.is_floating_point() or ids.is_complex() or ids.dtype == torch.bool:
        raise IqkKernelError("ids must be an integer tensor")
    if ids.dim() < 1:
        raise IqkKernelError("ids must be [..., k]")
    if not ids.is_cuda:
        raise IqkKernelError(f"ids must live on a GPU, got {ids.device}")
    experts, k = int(num_experts), ids.shape[-1]
    if not 0 < experts <= MAX_EXPERTS:
        raise IqkKernelError(f"pairs are sorted by 1 .. {MAX_EXPERTS} experts, got {experts}")
    if not 0 < k <= MAX_K:
        raise IqkKernelError(f"a token has 1 .. {MAX_K} experts, got {k}")
    if ids.numel() >= 2 ** 31:
        raise IqkKernelError(f"fewer than 2**31 pairs are sorted, got {ids.numel()}")
    if ids.dtype not in _KERNEL_IDS:
        ids = torch.clamp(ids.to(torch.int64), -1, experts)
    return ids.contiguous(), experts


def sort(ids: torch.Tensor, num_experts: int) -> Order:
    """The pairs of ``ids`` ``[..., k]`` (a token's experts in its last axis) by expert.

    Pairs whose id is outside ``0 .. num_experts - 1`` are left out: padded tokens, or
    another rank's experts.  ``ids`` and ``tokens`` of the order are what
    ``gemv_sorted`` and ``gemv_union`` take.
    """
    sort_pairs = _native.torch_binding().sort
    if (lists := sort_pairs(ids, num_experts)) is None:  # ids that the kernels do not take as they are
        lists = sort_pairs(*_check_ids(ids, num_experts))
    order = Order(*lists)
    order._permutation = order.slots
    return order


def _check_rows(t: torch.Tensor, name: str, device: torch.device) -> None:
    if not isinstance(t, torch.Tensor) or t.dim() < 1:
        raise IqkKernelError(f"{name} must be a tensor of at least one dimension")
    if t.device != device:
        raise IqkKernelError(f"{name} is on {t.device}, expected {device}")
    if t.dtype not in _DTYPES:
        raise IqkKernelError(f"{name} must be one of {tuple(_DTYPES)}, got {t.dtype}")
    if not 0 < t.shape[-1] < MAX_COLS:
        raise IqkKernelError(f"{name} must have rows of 1 .. {MAX_COLS - 1} values, got {t.shape[-1]}")


def dispatch(x: torch.Tensor, ids: torch.Tensor, num_experts: int) -> tuple[torch.Tensor, Order]:
    """Each token's row for each of its experts, sorted by expert: ``(rows [pairs, n], order)``.

    ``x`` is ``[..., n]``, ``ids`` ``[..., k]`` with the same leading shape.  Slot ``s`` of
    ``rows`` holds the row of token ``order.tokens[s]``; the rows of pairs left out
    (:func:`sort`), behind all others, are zeros.  A switch module takes them as
    ``proj(rows[:, None], order.ids, sorted_indices=True)``.  Differentiable in ``x``: a token's gradient is the
    sum of its rows' (f32, rounded once), those left out not counted.
    """
    dispatch_rows = _native.torch_binding().dispatch
    if (got := dispatch_rows(x, ids, num_experts)) is None:  # what the kernels do not take as it is
        ids, experts = _check_ids(ids, num_experts)
        _check_rows(x, "x", ids.device)
        if x.shape[:-1] != ids.shape[:-1]:
            raise IqkKernelError(f"x {tuple(x.shape)} and ids {tuple(ids.shape)} are not of the same tokens")
        got = dispatch_rows(x.contiguous(), ids, experts)
    order = Order(*got[1:])
    order._permutation = order.slots
    return got[0], order


def combine(y: torch.Tensor, weights: torch.Tensor, order: Order | None = None, *,
            add: torch.Tensor | None = None) -> torch.Tensor:
    """Each token's expert outputs, weighted and summed: ``[..., n]`` in y's type.

    ``y`` is ``[pairs, n]`` in ``order``, or without one ``[..., k, n]``, a token's rows
    together as the switch modules return them (less their axis of one row).  ``weights`` is
    ``[..., k]``; ``add`` ``[..., n]``, y's type, is added (a shared
    expert's output, the residual).  Sums are f32, rounded once.  Pairs that the order leaves out count
    for nothing, whatever their rows hold; without an order every row counts.  Differentiable in
    ``y``, ``weights`` and ``add``; the gradients of pairs left out are 0, as are those of rows that no pair has.
    """
    combine_rows = _native.torch_binding().combine
    if order is None:
        out = combine_rows(y, weights, None, None, add, False)
    elif type(order) is Order:
        out = combine_rows(y, weights, order.slots, order.offsets, add, order._permutation is order.slots)
    else:
        raise IqkKernelError(f"order must be an Order, got {type(order).__name__}")
    if out is not None:
        return out
    # what the kernels do not take as it is
    if not isinstance(y, torch.Tensor) or not y.is_cuda:
        raise IqkKernelError(f"y must live on a GPU, got {getattr(y, 'device', type(y).__name__)}")
    _check_rows(y, "y", y.device)
    if not isinstance(weights, torch.Tensor) or weights.device != y.device or weights.dtype not in _DTYPES:
        raise IqkKernelError(f"weights must be one of {tuple(_DTYPES)} on {y.device}")
    if weights.dim() < 1 or not 0 < weights.shape[-1] <= MAX_K or weights.numel() >= 2 ** 31:
        raise IqkKernelError(f"weights must be [..., k] with k 1 .. {MAX_K} and fewer than 2**31 pairs, got "
                             f"{tuple(weights.shape)}")
    slots = offsets = None
    permutation = False
    if order is None:
        want = (*weights.shape, y.shape[-1])
    else:
        if order.slots.shape != weights.shape:
            raise IqkKernelError(f"order must be one of pairs {tuple(weights.shape)}, got {order!r}")
        slots, offsets, permutation = order.slots, order.offsets, order._permutation is order.slots
        for t in (slots, offsets):
            if t.device != y.device or t.dtype != torch.int32 or not t.is_contiguous():
                raise IqkKernelError(f"order must hold contiguous int32 tensors on {y.device}")
        if not offsets.numel():
            raise IqkKernelError("order must hold an offset behind its experts")
        want = (weights.numel(), y.shape[-1])
    if tuple(y.shape) != want:
        raise IqkKernelError(f"y must be {want} for weights {tuple(weights.shape)}, got {tuple(y.shape)}")
    if add is not None:
        _check_rows(add, "add", y.device)
        if add.dtype != y.dtype or tuple(add.shape) != (*weights.shape[:-1], y.shape[-1]):
            raise IqkKernelError(f"add must be {y.dtype} {(*weights.shape[:-1], y.shape[-1])}, got {add.dtype} "
                                 f"{tuple(add.shape)}")
        add = add.contiguous()
    return combine_rows(y.contiguous(), weights.float().contiguous(), slots, offsets, add, permutation)


__all__ = ["MAX_COLS", "MAX_EXPERTS", "MAX_GROUPS", "MAX_K", "Order", "balance_loss", "combine", "dispatch", "sort", "topk"]
