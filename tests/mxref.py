"""Plain 64-bit forms of the 4-bit microscaled format, the products with it, the
router's choice and its balance loss, on the CPU: what the kernels' tests compare
with.  Written from the definitions."""

from __future__ import annotations

import numpy as np
import torch

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)
VALUES = np.concatenate([GRID, -GRID])
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """f64 [..., n] -> codes u8 [..., n/2], scales u8 [..., n/32], by search of
    the grid (of two equally near values the even code)."""
    blocks = np.asarray(x, dtype=np.float64).reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = np.abs(blocks).max(-1)
    good = np.isfinite(top)
    with np.errstate(divide="ignore", invalid="ignore"):
        e = np.where(good & (top > 0), np.floor(np.log2(np.where(good & (top > 0), top, 1.0))), -1000)
    # log2 rounds: put the exponent right where it did
    e = np.where(good & (top > 0) & (np.ldexp(1.0, np.clip(e, -1000, 1000).astype(int)) > top), e - 1, e)
    e = np.where(good & (top > 0) & (np.ldexp(1.0, np.clip(e + 1, -1000, 1000).astype(int)) <= top), e + 1, e)
    byte = np.where(good, np.clip(e - 2, -127, 127) + 127, 255).astype(int)
    v = np.abs(np.where(good[..., None], blocks, 0.0)) / np.ldexp(1.0, np.where(good, byte - 127, 0))[..., None]
    dist = np.abs(v[..., None] - GRID)
    order = np.array([0, 2, 4, 6, 1, 3, 5, 7])  # even codes first, so they win ties
    mag = order[np.argmin(dist[..., order], axis=-1)]
    code = mag + 8 * np.signbit(blocks)
    code = np.where(good[..., None], code, 0).astype(np.uint8).reshape(x.shape)
    return (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), byte.astype(np.uint8)


def values(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """f64 values of codes and scales."""
    code = np.stack([codes & 15, codes >> 4], -1).reshape(*scales.shape, 32)
    s = np.where(scales == 255, np.nan, np.ldexp(1.0, scales.astype(int) - 127))
    return (VALUES[code] * s[..., None]).reshape(*codes.shape[:-1], 2 * codes.shape[-1])


def random_codes(rng, shape, lo=117, hi=131) -> tuple[np.ndarray, np.ndarray]:
    """Codes and scales of [..., n]: every code, scales 2^(lo - 127) .. 2^(hi - 127)."""
    *lead, n = shape
    return (rng.integers(0, 256, (*lead, n // 2), dtype=np.uint8),
            rng.integers(lo, hi + 1, (*lead, n // 32), dtype=np.uint8))


def product_bound(x: np.ndarray, w: np.ndarray, dtype) -> tuple[np.ndarray, np.ndarray]:
    """x [m, k] times w [n, k] in 64 bits, and how far a kernel may be off: f32
    sums of exact products, at most k/32 sequential ones and 16 within each, then
    one rounding to dtype."""
    want = x @ w.T
    span = np.abs(x) @ np.abs(w).T
    k = x.shape[-1]
    bound = HALF_ULP[dtype] * np.abs(want) + (k / 32 + 16) * 2.0 ** -23 * span + TINY[dtype]
    return want, bound


# ------------------------------------------------------------------ router ---


def softmax(x: np.ndarray) -> np.ndarray:
    top = x.max(-1, keepdims=True)
    with np.errstate(invalid="ignore"):
        e = np.exp(x - top)
        p = e / e.sum(-1, keepdims=True)
    return np.where(top == -np.inf, 0.0, p)


def topk(logits: np.ndarray, k: int, normalize: bool):
    """f64 [t, experts] -> weights, ids; NaN above all, ties to the lowest."""
    key = np.where(np.isnan(logits), np.inf, logits)
    rank = np.where(np.isnan(logits), 1, 0)
    ids = np.stack([np.lexsort((np.arange(logits.shape[1]), -key[t], -rank[t]))[:k] for t in range(len(logits))]) \
        if len(logits) else np.zeros((0, k), int)
    chosen = np.take_along_axis(logits, ids, -1)
    if normalize:
        return softmax(chosen), ids
    return np.take_along_axis(softmax(logits), ids, -1), ids


def topk_grad(logits, k, normalize, dweights):
    """The gradient by the softmax's Jacobian, written out."""
    w, ids = topk(logits, k, normalize)
    t, experts = logits.shape
    hot = np.zeros((t, k, experts))
    np.put_along_axis(hot, ids[..., None], 1.0, -1)
    q = (hot * w[..., None]).sum(1) if normalize else softmax(logits)
    jac = w[..., None] * (hot - q[:, None, :])
    return (jac * dweights[..., None]).sum(1)


def balance(logits, ids, mask):
    """f64 [tokens, experts], ids [tokens, k], mask [tokens] -> loss, counts."""
    experts, k = logits.shape[1], ids.shape[1]
    n = int(mask.sum())
    kept = ids[mask]
    counts = np.array([(kept == e).sum() for e in range(experts)])
    if n == 0:
        return 0.0, counts
    share = counts / (k * n)
    return float(experts * (share * softmax(logits[mask]).mean(0)).sum()), counts


def balance_grad(logits, ids, mask):
    """d loss / d logits, by the Jacobian of each kept token's softmax."""
    experts, k = logits.shape[1], ids.shape[1]
    n = int(mask.sum())
    out = np.zeros_like(logits)
    if n == 0:
        return out
    _, counts = balance(logits, ids, mask)
    p = softmax(logits[mask])
    jac = p[:, :, None] * (np.eye(experts)[None] - p[:, None, :])  # d p_e / d l_j
    out[mask] = experts / (k * n * n) * np.einsum("e,tej->tj", counts.astype(float), jac)
    return out
