"""Operators around the routed experts, as cases to measure: 4-bit microscaled
weights and activations (their quantisation, and products with them), the
router's choice of experts, and its balance loss.

* ``cast``: ``mx.quantize`` of a matrix and the values its codes stand for.
* ``experts``: ``mx.MxSwitchLinear`` called with ``(x, indices)``, the
  activations in 16 bits, or quantised first (``mx`` true).
* ``linear``: ``mx.MxLinear``, the same product with one matrix.
* ``topk``: ``router.topk`` and, where ``grad`` is true, its gradient.
* ``balance``: ``router.balance_loss`` and its gradient.

The geometry is the routed layer of this repository's benchmark (256 experts,
top-6, gate/up ``[2048 x 4096]``, down ``[4096 x 2048]``) and generic sizes
around it.  Weights are N(0, 0.02), activations N(0, 1) with a few louder
channels, router logits normal around a preference for some experts.

Where ``own`` is false the same operators are computed in their plain form:
elementary operations in 32 bits, rounded once.
"""

from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GATE, DOWN = (2048, 4096), (4096, 2048)  # out, in
CHUNK = 1 << 27  # weights made at a time


def listed() -> list[dict]:
    def experts(name, shape, tokens, **over):
        case = {"name": name, "kind": "experts", "experts": 256, "out": shape[0], "in": shape[1], "tokens": tokens,
                "top_k": 6, "zipf": 0.0, "per_pair": False, "dtype": "f16", "mx": False, "ids": "int32"}
        case.update(over)
        return case

    return [
        # the activations of a small decode batch, quantised before a projection
        {"name": "cast_rows_t8", "kind": "cast", "rows": 8, "cols": 4096, "dtype": "bf16"},
        # a projection of 64 experts quantised when a 16-bit checkpoint is loaded
        {"name": "cast_stack_e64", "kind": "cast", "rows": 64 * 2048, "cols": 4096, "dtype": "bf16"},
        # one token of one sequence through its experts: the smallest call, where latency counts
        experts("decode_gate_t1", GATE, 1),
        # eight sequences decoded together, the down projection with its row for each pair, ids from torch
        experts("decode_down_t8", DOWN, 8, per_pair=True, dtype="bf16", ids="int64"),
        # 24 sequences decoded together in 4-bit activations: one pair or two to an expert
        experts("batch_mx_gate_t24", GATE, 24, mx=True, dtype="bf16"),
        # a short prompt of odd length through a small model's experts of odd width
        experts("prefill_odd_t149", (1000, 1440), 149, experts=60, top_k=4),
        # the benchmark's prompt: 2048 tokens, some experts with thousands of rows and some with few
        experts("prefill_gate_t2048", GATE, 2048, zipf=1.1, dtype="bf16"),
        # a dense layer over a batch of prompts, weights and activations in 4 bits: bound by arithmetic
        {"name": "linear_mx_t8192", "kind": "linear", "tokens": 8192, "out": 8192, "in": 4096, "dtype": "bf16",
         "mx": True},
        # the router's choice for one token
        {"name": "topk_t1", "kind": "topk", "tokens": 1, "experts": 256, "top_k": 6, "dtype": "f32",
         "normalize": True, "grad": False},
        # the router's choice and its gradient in a training step over 65536 tokens
        {"name": "topk_train_t65536", "kind": "topk", "tokens": 65536, "experts": 256, "top_k": 6, "dtype": "bf16",
         "normalize": True, "grad": True},
        # the balance loss of one short sequence, an odd number of experts
        {"name": "balance_t500", "kind": "balance", "groups": 1, "tokens": 500, "experts": 60, "top_k": 4,
         "dtype": "f32", "mask": True},
        # the balance loss of each of 16 long sequences of a training step, padded ones among them
        {"name": "balance_g16_t4096", "kind": "balance", "groups": 16, "tokens": 4096, "experts": 256, "top_k": 6,
         "dtype": "f32", "mask": True},
    ]


def draw(rng) -> dict:
    def spread(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(("cast", "experts", "experts", "experts", "experts", "linear", "topk", "balance"))
    half = rng.choice(("f16", "bf16"))
    if kind == "cast":
        cols = 32 * spread(1, 256)
        return {"kind": kind, "rows": spread(1, min(131072, (1 << 29) // cols)), "cols": cols,
                "dtype": rng.choice(("f32", "f16", "bf16"))}
    if kind == "linear":
        return {"kind": kind, "tokens": spread(1, 8192), "out": spread(64, 8192), "in": 32 * spread(2, 128),
                "dtype": half, "mx": rng.random() < 0.6}
    if kind == "topk":
        experts = spread(8, 512)
        return {"kind": kind, "tokens": spread(1, 32768), "experts": experts, "top_k": rng.randint(1, min(12, experts)),
                "dtype": rng.choice(("f32", "f16", "bf16")), "normalize": rng.random() < 0.6, "grad": rng.random() < 0.7}
    if kind == "balance":
        experts = spread(8, 512)
        groups = rng.choice((1, 1, 2, 3, 8, 16))
        return {"kind": kind, "groups": groups, "tokens": spread(64, 32768 // groups), "experts": experts,
                "top_k": rng.randint(1, min(8, experts)), "dtype": rng.choice(("f32", "f16", "bf16")),
                "mask": rng.random() < 0.5}
    shape = rng.choice((GATE, DOWN, None))
    out, width = shape or (spread(256, 4096), 32 * rng.randint(16, 96))
    experts = rng.choice((8, 16, 32, 60, 128, 160, 256))
    top_k = rng.choice((1, 2, 4, 6, 8))
    tokens = spread(1, 12288 // top_k)
    return {"kind": kind, "experts": experts, "out": out, "in": width, "tokens": tokens, "top_k": top_k,
            "zipf": rng.choice((0.0, 1.1)), "per_pair": rng.random() < 0.4, "dtype": half,
            "mx": rng.random() < 0.4, "ids": rng.choice(("int32", "int64"))}


# ------------------------------------------------------------------ inputs ---


def _rng(seed: int, label: str) -> np.random.Generator:
    return np.random.default_rng([int(seed), *label.encode()])


def _generator(seed: int, label: str) -> torch.Generator:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(_rng(seed, label).integers(1 << 62)))
    return g


def _normal(shape, seed: int, label: str) -> torch.Tensor:
    return torch.randn(shape, generator=_generator(seed, label), device=DEVICE)


def _activations(rows: int, cols: int, dtype: str, seed: int) -> torch.Tensor:
    """Rows of N(0, 1) whose every 97th channel is twenty times as loud."""
    x = _normal((rows, cols), seed, "x")
    x[:, 5::97] *= 20.0
    return x.to(DTYPES[dtype])


def _round_blocks(x: torch.Tensor):
    """f32 ``[..., n]`` -> each value's magnitude on the 4-bit grid and each
    block's exponent: the largest magnitude of 32 values has the exponent
    e + 2, values are rounded to nearest, ties to even, in units of 2^e."""
    blocks = x.reshape(*x.shape[:-1], -1, 32)
    top = torch.frexp(blocks.abs().amax(-1, keepdim=True)).exponent - 1
    e = torch.clamp(top - 2, -127, 127)
    v = torch.ldexp(blocks.abs(), -e)
    step = torch.where(v < 2, 0.5, torch.where(v < 4, 1.0, 2.0))
    return torch.clamp(torch.round(v / step) * step, max=6.0), torch.signbit(blocks), e


def _plain_cast(x: torch.Tensor) -> torch.Tensor:
    """The values that 4-bit codes of x stand for, in f32."""
    mag, sign, e = _round_blocks(x.to(torch.float32))
    return torch.ldexp(torch.where(sign, -mag, mag), e).reshape(x.shape)


def _weight_codes(rows: int, cols: int, generator) -> tuple:
    """Codes (two a byte, the even column's in the low half) and block scales
    (2^(byte - 127)) of N(0, 0.02) rows."""
    w = torch.randn((rows, cols), generator=generator, device=DEVICE) * 0.02
    mag, sign, e = _round_blocks(w)
    code = torch.where(mag < 2, 2 * mag, torch.where(mag < 4, mag + 2, mag / 2 + 4)).to(torch.uint8)
    code = (code + 8 * sign.to(torch.uint8)).reshape(rows, cols)
    return code[:, 0::2] + 16 * code[:, 1::2], (e + 127).to(torch.uint8).reshape(rows, -1)


def _weights(case: dict, seed: int) -> tuple:
    """codes u8 [E, out, in/2] and scales u8 [E, out, in/32]."""
    E, out, n = case.get("experts", 1), case["out"], case["in"]
    codes = torch.empty((E * out, n // 2), dtype=torch.uint8, device=DEVICE)
    scales = torch.empty((E * out, n // 32), dtype=torch.uint8, device=DEVICE)
    g, rows = _generator(seed, "w"), max(1, CHUNK // n)
    for at in range(0, E * out, rows):
        codes[at:at + rows], scales[at:at + rows] = _weight_codes(min(rows, E * out - at), n, g)
    return codes.view(E, out, -1), scales.view(E, out, -1)


def _routing(case: dict, seed: int) -> np.ndarray:
    """``[tokens, top_k]`` expert ids, a token's ids distinct: uniform, or Zipf
    over a random order of the experts."""
    rng = _rng(seed, "routing")
    experts, tokens, k = case["experts"], case["tokens"], case["top_k"]
    order = rng.permutation(experts)
    weight = np.arange(1, experts + 1, dtype=np.float64) ** -case["zipf"]
    key = np.log(weight) + rng.gumbel(size=(tokens, experts))
    return order[np.argsort(-key, axis=1)[:, :k]].astype(np.int64)


def _logits(shape, dtype: str, seed: int) -> torch.Tensor:
    preference = 0.7 * _normal((shape[-1],), seed, "preference")
    return (1.5 * _normal(shape, seed, "logits") + preference).to(DTYPES[dtype])


def _highest(logits: torch.Tensor, k: int) -> torch.Tensor:
    return torch.sort(logits, dim=-1, descending=True, stable=True).indices[..., :k]


def _inputs(case: dict, seed: int) -> dict:
    """What both forms take, the weights as codes and scales."""
    kind = case["kind"]
    if kind == "cast":
        return {"x": _activations(case["rows"], case["cols"], case["dtype"], seed)}
    if kind in ("experts", "linear"):
        codes, scales = _weights(case, seed)
        state = {"codes": codes, "scales": scales, "mx": case["mx"]}
        if kind == "linear":
            state["x"] = _activations(case["tokens"], case["in"], case["dtype"], seed)
            return state
        ids = torch.from_numpy(_routing(case, seed)).to(DEVICE, getattr(torch, case["ids"]))
        T, k = ids.shape
        rows = T * k if case["per_pair"] else T
        x = _activations(rows, case["in"], case["dtype"], seed)
        state.update(x=x.view((T, k, 1, -1) if case["per_pair"] else (T, 1, 1, -1)), ids=ids)
        return state
    if kind == "topk":
        shape = (case["tokens"], case["experts"])
        state = {"logits": _logits(shape, case["dtype"], seed), "k": case["top_k"], "normalize": case["normalize"],
                 "grad": case["grad"]}
        if case["grad"]:
            state["dweights"] = _normal((case["tokens"], case["top_k"]), seed, "dweights")
        return state
    lead = (case["groups"],) if case["groups"] > 1 else ()
    shape = (*lead, case["tokens"], case["experts"])
    logits = _logits(shape, case["dtype"], seed)
    state = {"logits": logits, "ids": _highest(logits, case["top_k"]).to(torch.int32), "mask": None,
             "dloss": 0.01 * (1 + torch.rand(lead, generator=_generator(seed, "dloss"), device=DEVICE))}
    if case["mask"]:  # sequences of their own lengths, padded at the end
        length = torch.from_numpy(_rng(seed, "length").integers(case["tokens"] // 2, case["tokens"] + 1, (*lead, 1)))
        state["mask"] = torch.arange(case["tokens"], device=DEVICE) < length.to(DEVICE)
    return state


def prepare(case: dict, seed: int) -> dict:
    state = {"kind": case["kind"], **_inputs(case, seed)}
    if not own:
        return state
    if os.path.join(os.getcwd(), "mlx-iqk_amd") not in sys.path:
        sys.path.insert(1, os.path.join(os.getcwd(), "mlx-iqk_amd"))
    from mlx_iqk_amd import mx, router
    state.update(ops=mx if case["kind"] in ("cast", "experts", "linear") else router)
    if "codes" in state:  # the module that a program loads its weights into once
        codes, scales = state.pop("codes"), state.pop("scales")
        if case["kind"] == "experts":
            state["module"] = mx.MxSwitchLinear(case["experts"], case["out"], case["in"], device=DEVICE)
        else:
            state["module"] = mx.MxLinear(case["out"], case["in"], device=DEVICE)
            codes, scales = codes[0], scales[0]
        state["module"].load(mx.MxTensor(codes, scales))
    elif case["kind"] == "balance" or state.get("grad"):
        state["logits"].requires_grad_()
    return state


# --------------------------------------------------------------- the passes ---


def run(state: dict):
    return (_own if own else _plain)(state)


def _own(state: dict):
    kind, ops = state["kind"], state["ops"]
    if kind == "cast":
        return ops.quantize(state["x"]).dequantize()
    if kind in ("experts", "linear"):
        x = ops.quantize(state["x"]) if state["mx"] else state["x"]
        return state["module"](x, state["ids"]) if kind == "experts" else state["module"](x)
    if kind == "topk":
        weights, ids = ops.topk(state["logits"], state["k"], normalize=state["normalize"])
        if not state["grad"]:
            return {"weights": weights, "ids": ids}
        (dlogits,) = torch.autograd.grad(weights, state["logits"], state["dweights"])
        return {"weights": weights, "ids": ids, "dlogits": dlogits}
    loss, counts = ops.balance_loss(state["logits"], state["ids"], mask=state["mask"])
    (dlogits,) = torch.autograd.grad(loss, state["logits"], state["dloss"])
    return {"loss": loss, "counts": counts, "dlogits": dlogits}


def _grid(device, dtype) -> torch.Tensor:
    half = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=dtype, device=device)
    return torch.cat([half, -half])


def _values(codes: torch.Tensor, scales: torch.Tensor, dtype=torch.float32) -> torch.Tensor:
    """The values of codes [..., n/2] and scales [..., n/32]."""
    code = torch.stack([codes & 15, codes >> 4], dim=-1).reshape(*scales.shape, 32)
    value = _grid(codes.device, dtype)[code.to(torch.int32)]
    return torch.ldexp(value, scales[..., None].to(torch.int32) - 127).reshape(*codes.shape[:-1], -1)


def _softmax(logits: torch.Tensor) -> torch.Tensor:
    e = torch.exp(logits - logits.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain(state: dict):
    kind = state["kind"]
    if kind == "cast":
        return _plain_cast(state["x"]).to(state["x"].dtype)
    if kind in ("experts", "linear"):
        x = state["x"]
        dtype, x = x.dtype, _plain_cast(x) if state["mx"] else x.to(torch.float32)
        if kind == "linear":
            return (x @ _values(state["codes"][0], state["scales"][0]).T).to(dtype)
        return _plain_experts(x, state["ids"], state["codes"], state["scales"], torch.float32).to(dtype)
    if kind == "topk":
        logits = state["logits"].to(torch.float32)
        ids = _highest(logits, state["k"])
        p = _softmax(torch.gather(logits, -1, ids) if state["normalize"] else logits)
        weights = p if state["normalize"] else torch.gather(p, -1, ids)
        if not state["grad"]:
            return {"weights": weights, "ids": ids.to(torch.int32)}
        dw = state["dweights"]
        zeros = torch.zeros_like(logits)
        if state["normalize"]:
            dlogits = zeros.scatter(-1, ids, weights * (dw - (dw * weights).sum(-1, keepdim=True)))
        else:
            dlogits = p * (zeros.scatter(-1, ids, dw) - (dw * weights).sum(-1, keepdim=True))
        return {"weights": weights, "ids": ids.to(torch.int32), "dlogits": dlogits.to(state["logits"].dtype)}
    return _plain_balance(state, torch.float32)


def _plain_experts(x, ids, codes, scales, dtype):
    """Each pair's row through its expert's matrix: where few pairs are asked for, each
    with its own copy of the matrix, else expert by expert."""
    T, k = ids.shape
    flat = ids.reshape(-1).to(torch.int64)
    rows = x.expand(T, k, 1, x.shape[-1]).reshape(T * k, -1)
    if T * k <= 64:
        return (_values(codes[flat], scales[flat], dtype) @ rows[:, :, None]).reshape(T, k, 1, -1)
    order = torch.argsort(flat)
    counts = torch.bincount(flat, minlength=codes.shape[0]).tolist()
    groups = torch.split(rows[order], counts)
    parts = [g @ _values(codes[e], scales[e], dtype).T.contiguous() for e, g in enumerate(groups) if counts[e]]
    y = torch.empty((T * k, codes.shape[1]), dtype=dtype, device=x.device)
    y[order] = torch.cat(parts)
    return y.reshape(T, k, 1, -1)


def _plain_balance(state: dict, dtype):
    logits, ids = state["logits"].detach(), state["ids"].to(torch.int64)
    E, k = logits.shape[-1], ids.shape[-1]
    keep = torch.ones(logits.shape[:-1], dtype=dtype, device=logits.device)
    if state["mask"] is not None:
        keep = state["mask"].to(dtype)
    p = _softmax(logits.to(dtype)) * keep[..., None]
    n = keep.sum(-1, keepdim=True)
    pairs = keep[..., None].expand(ids.shape).reshape(*ids.shape[:-2], -1)
    counts = torch.zeros((*logits.shape[:-2], E), dtype=dtype, device=logits.device)
    counts = counts.scatter_add(-1, ids.reshape(*ids.shape[:-2], -1), pairs)
    factor = E / (k * n * n)
    loss = (factor * counts * p.sum(-2)).sum(-1)
    centred = counts[..., None, :] - (p * counts[..., None, :]).sum(-1, keepdim=True)
    dlogits = (state["dloss"].to(dtype)[..., None] * factor)[..., None] * p * centred
    whole = counts.to(torch.int32)
    return {"loss": loss, "counts": whole, "dlogits": dlogits.to(logits.dtype) if dtype == torch.float32 else dlogits}


# ---------------------------------------------------------- what it is held to ---


def work(case: dict) -> dict:
    """Bytes: each input read once, each output written once.  Of the weights,
    those of the experts that the routing names."""
    kind = case["kind"]
    size = DTYPES[case["dtype"]].itemsize
    if kind == "cast":
        n = case["rows"] * case["cols"]
        return {"bytes": 2 * size * n, "flops": 4 * n}
    if kind == "linear":
        T, out, n = case["tokens"], case["out"], case["in"]
        return {"bytes": out * n * 17 // 32 + size * T * (n + out), "flops": 2 * T * out * n}
    if kind == "experts":
        ids, out, n = _routing(case, 0), case["out"], case["in"]
        rows = ids.size if case["per_pair"] else case["tokens"]
        bytes_ = int(np.unique(ids).size) * out * n * 17 // 32 + size * (rows * n + ids.size * out)
        return {"bytes": bytes_ + ids.size * (8 if case["ids"] == "int64" else 4), "flops": 2 * ids.size * out * n}
    T, E, k = case.get("groups", 1) * case["tokens"], case["experts"], case["top_k"]
    if kind == "topk":
        grad = case["grad"]
        # with the normalised weights the gradient needs no logits again
        logits = E * size * (2 if grad else 1)
        return {"bytes": T * (logits + k * (12 if grad else 8)), "flops": T * E * (5 if grad else 3)}
    return {"bytes": T * (2 * E * size + 4 * k + int(case["mask"])), "flops": 12 * T * E}


# ----------------------------------------------------------------- in 64 bits ---


def _exact_cast(x: torch.Tensor) -> torch.Tensor:
    """float64 values of the 4-bit codes nearest to x in units of the block's
    2^(floor(log2 max) - 2), a tie to the even code, read off the midpoints
    between the grid's values."""
    blocks = x.to(torch.float64).reshape(*x.shape[:-1], -1, 32)
    unit = torch.exp2(torch.clamp(torch.floor(torch.log2(blocks.abs().amax(-1, keepdim=True))) - 2, -127, 127))
    v = blocks.abs() / unit
    grid = _grid(x.device, torch.float64)[:8]
    code = torch.bucketize(v, (grid[1:] + grid[:-1]) / 2)  # midpoints below v
    at_mid = (code < 7) & (v == ((grid[1:] + grid[:-1]) / 2)[code.clamp(max=6)])
    code = torch.where(at_mid & (code % 2 == 1), code + 1, code)
    return (torch.sign(blocks) * grid[code] * unit).reshape(x.shape)


def exact(case: dict, seed: int):
    kind = case["kind"]
    state = _inputs(case, seed)
    if kind == "cast":
        return _exact_cast(state["x"])
    if kind in ("experts", "linear"):
        x = _exact_cast(state["x"]) if case["mx"] else state["x"].to(torch.float64)
        if kind == "linear":
            return x @ _values(state["codes"][0], state["scales"][0], torch.float64).T.contiguous()
        T, k = state["ids"].shape
        flat, out = state["ids"].reshape(-1), case["out"]
        rows = x.expand(T, k, 1, case["in"]).reshape(T * k, -1)
        y = torch.empty((T * k, out), dtype=torch.float64, device=DEVICE)
        for e in torch.unique(flat).tolist():
            at = torch.nonzero(flat == e).reshape(-1)
            y[at] = rows[at] @ _values(state["codes"][e], state["scales"][e], torch.float64).T.contiguous()
        return y.view(T, k, 1, out)
    if kind == "topk":
        logits = state["logits"].to(torch.float64)
        ids = _highest(logits, case["top_k"])
        chosen = torch.gather(torch.log_softmax(logits, -1), -1, ids)
        weights = torch.exp(chosen)
        if case["normalize"]:
            weights = weights / weights.sum(-1, keepdim=True)
        got = {"weights": weights, "ids": None}
        if case["grad"]:
            dw = state["dweights"].to(torch.float64)
            # d w_i / d l_e = w_i (delta_ie - q_e), q the softmax that w is taken from
            q = torch.zeros_like(logits).scatter(-1, ids, weights) if case["normalize"] else torch.softmax(logits, -1)
            got["dlogits"] = torch.zeros_like(logits).scatter(-1, ids, weights * dw) \
                - q * (weights * dw).sum(-1, keepdim=True)
        return got
    logits = state["logits"].to(torch.float64)
    E, k = case["experts"], case["top_k"]
    keep = torch.ones(logits.shape[:-1], dtype=torch.float64, device=DEVICE)
    if state["mask"] is not None:
        keep = state["mask"].to(torch.float64)
    hits = torch.zeros_like(logits).scatter(-1, state["ids"].to(torch.int64), 1.0) * keep[..., None]
    share = hits.sum(-2) / (k * keep.sum(-1, keepdim=True))  # of the pairs, by expert
    p = torch.softmax(logits, -1)
    mean = (p * keep[..., None]).sum(-2) / keep.sum(-1, keepdim=True)
    loss = E * (share * mean).sum(-1)
    lean = (p * share[..., None, :]).sum(-1, keepdim=True)
    scale = (state["dloss"].to(torch.float64) * E / keep.sum(-1))[..., None, None]
    return {"loss": loss, "counts": None, "dlogits": scale * keep[..., None] * p * (share[..., None, :] - lean)}
