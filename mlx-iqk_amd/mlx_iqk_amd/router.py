"""The router of a layer of experts: which experts a token goes to, with what
weights, and the loss that keeps the experts evenly loaded; with gradients.

:func:`topk`'s ids are the ``indices`` of the switch modules
(:class:`~mlx_iqk_amd.nn.IqkSwitchLinear`, :class:`~mlx_iqk_amd.mx.MxSwitchLinear`),
its weights scale their outputs.  Logits are f32, f16 or bf16 on a GPU, for up to
1024 experts; sums, probabilities, weights and losses are f32.  Gradients are
not differentiable again, and logits with a forward-mode derivative are refused.
The calls can be captured in a graph; their gradients cannot, and raise under a capture.
"""

from __future__ import annotations

import math

import torch

from . import _native
from .kernels import IqkKernelError
from .mx import _DTYPES

MAX_EXPERTS = 1024
MAX_K = 64
MAX_GROUPS = 65535
"""Losses of one :func:`balance_loss` call."""


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


__all__ = ["MAX_EXPERTS", "MAX_GROUPS", "MAX_K", "balance_loss", "topk"]
