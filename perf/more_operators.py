"""Operators between the router, the experts and the layer's output, as cases to
measure: tokens sorted by expert, their outputs weighted and summed, and low-rank
adapters of many requests beside a shared projection.

* ``sort``: ``router.sort`` of the expert ids alone.
* ``dispatch``: ``router.dispatch``, the tokens' rows sorted by expert, and where
  ``grad`` is true its gradient.
* ``combine``: ``router.combine``, a token's expert outputs weighted and summed, from
  sorted rows or (``sorted`` false) as the switch modules return them, ``add`` with the
  shared projection's output added; where ``grad`` is true its gradients.
* ``adapters``: ``adapters.LowRankAdapters``, each row with the adapter its request names,
  added to the output of the projection they share.

The geometry is the routed layer of this repository's benchmark (256 experts,
top-6, rows of 4096) and generic sizes around it; the adapters' projections are
``[8192 x 4096]`` and around it.

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
LARGEST = 16384 * 6 * 4096  # values of the sorted rows in the largest listed case


def listed() -> list[dict]:
    def routed(name, kind, tokens, **over):
        case = {"name": name, "kind": kind, "tokens": tokens, "experts": 256, "top_k": 6, "cols": 4096, "dtype": "bf16",
                "zipf": 0.0, "padded": 0.0, "ids": "int32", "grad": False}
        if kind == "combine":
            case.update({"sorted": True, "add": False})
        case.update(over)
        return case

    def adapted(name, rows, **over):
        case = {"name": name, "kind": "adapters", "rows": rows, "adapters": 64, "rank": 16, "out": 8192, "in": 4096,
                "dtype": "bf16", "runs": 1, "bare": 0.0, "ids": "int32"}
        case.update(over)
        return case

    return [
        # the ids of a drafted block of 8 tokens sorted, for a verification that reads each expert once
        routed("sort_t8", "sort", 8),
        # a long prompt's ids from torch, sorted for a caller with products of its own
        routed("sort_t32768", "sort", 32768, zipf=1.1, ids="int64"),
        # one token of one sequence: the smallest call, where latency counts
        routed("dispatch_t1", "dispatch", 1, dtype="f16"),
        # a training step of a small model of odd width in f32, a fifth of its tokens padding
        routed("dispatch_odd_t1777", "dispatch", 1777, experts=60, top_k=4, cols=1441, dtype="f32", padded=0.2,
               ids="int64", grad=True),
        # a training step over 16384 tokens, some experts with thousands of rows and some with few
        routed("dispatch_train_t16384", "dispatch", 16384, zipf=1.1, grad=True),
        # one token's six expert outputs, as the switch modules return them
        routed("combine_t1", "combine", 1, dtype="f16", sorted=False),
        # the benchmark's prompt: 2048 tokens, the shared projection's output added
        routed("combine_add_t2048", "combine", 2048, zipf=1.1, add=True),
        # a training step over 16384 tokens: gradients of the rows and of the router's weights
        routed("combine_train_t16384", "combine", 16384, zipf=1.1, grad=True),
        # one request with its adapter: the smallest call
        adapted("adapters_t1", 1),
        # 32 requests decoded together, most with an adapter of their own, ids from torch
        adapted("adapters_t32", 32, ids="int64"),
        # a mixed batch of short prompts, odd sizes, a third of its rows without an adapter
        adapted("adapters_odd_t333", 333, adapters=9, rank=20, out=1001, **{"in": 1440}, dtype="f16", runs=24, bare=0.3),
        # a batch of prompts of 8192 rows in all, adapters of rank 64
        adapted("adapters_t8192", 8192, adapters=16, rank=64, runs=512),
    ]


def draw(rng) -> dict:
    def spread(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(("sort", "dispatch", "dispatch", "combine", "combine", "adapters", "adapters", "adapters"))
    if kind == "adapters":
        n = 8 * spread(16, 512)
        rows = spread(1, 8192)
        return {"kind": kind, "rows": rows, "adapters": spread(1, 128), "rank": rng.choice((4, 8, 16, 20, 32, 64)),
                "out": spread(128, 8192), "in": n, "dtype": rng.choice(("f16", "bf16")),
                "runs": 1 if rows < 64 else rng.choice((1, spread(2, 512))), "bare": rng.choice((0.0, 0.0, 0.3)),
                "ids": rng.choice(("int32", "int64"))}
    experts = spread(8, 512)
    top_k = rng.randint(1, min(12, experts))
    case = {"kind": kind, "experts": experts, "top_k": top_k, "cols": 0, "dtype": rng.choice(("f32", "f16", "bf16")),
            "zipf": rng.choice((0.0, 1.1)), "padded": rng.choice((0.0, 0.0, 0.2)), "ids": rng.choice(("int32", "int64")),
            "grad": False}
    if kind == "sort":
        return {**case, "tokens": spread(1, 32768 * 6 // top_k), "dtype": "f32"}
    case["cols"] = spread(64, 8192)
    case["tokens"] = spread(1, min(32768, LARGEST // (case["cols"] * top_k * (2 if case["dtype"] == "f32" else 1))))
    case["grad"] = rng.random() < 0.6
    if kind == "combine":
        case.update({"sorted": rng.random() < 0.6, "add": rng.random() < 0.4})
    return case


# ------------------------------------------------------------------ inputs ---


def _rng(seed: int, label: str) -> np.random.Generator:
    return np.random.default_rng([int(seed), *label.encode()])


def _normal(shape, seed: int, label: str, dtype: str, scale: float = 1.0) -> torch.Tensor:
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(_rng(seed, label).integers(1 << 62)))
    return (torch.randn(shape, generator=g, device=DEVICE) * scale).to(DTYPES[dtype])


def _routing(case: dict, seed: int) -> np.ndarray:
    """``[tokens, top_k]`` expert ids, a token's ids distinct: uniform, or Zipf over a
    random order of the experts; -1 for all of a padded token's."""
    rng = _rng(seed, "routing")
    experts, tokens, k = case["experts"], case["tokens"], case["top_k"]
    order = rng.permutation(experts)
    weight = np.arange(1, experts + 1, dtype=np.float64) ** -case["zipf"]
    key = np.log(weight) + rng.gumbel(size=(tokens, experts))
    top = np.argpartition(-key, k - 1, axis=1)[:, :k]
    top = np.take_along_axis(top, np.argsort(-np.take_along_axis(key, top, 1), axis=1), 1)
    ids = order[top].astype(np.int64)
    ids[rng.random(tokens) < case["padded"]] = -1
    return ids


def _requests(case: dict, seed: int) -> np.ndarray:
    """Each row's adapter: runs of ``runs`` rows on average (a request's), adapters
    named unequally often; -1 for the rows of a request without one."""
    rng = _rng(seed, "requests")
    rows, n = case["rows"], case["adapters"]
    change = rng.random(rows) < 1.0 / case["runs"]
    request = np.cumsum(change)
    weight = np.arange(1, n + 1, dtype=np.float64) ** -0.5
    adapter = rng.permutation(n)[rng.choice(n, size=rows + 1, p=weight / weight.sum())]
    adapter[rng.random(rows + 1) < case["bare"]] = -1
    return adapter[request].astype(np.int64)


def _weights(case: dict, seed: int) -> torch.Tensor:
    """The choice's softmax weights, f32 ``[tokens, top_k]``."""
    e = torch.exp(_normal((case["tokens"], case["top_k"]), seed, "weights", "f32"))
    return e / e.sum(-1, keepdim=True)


def _inputs(case: dict, seed: int) -> dict:
    kind, dtype = case["kind"], case["dtype"]
    id_type = getattr(torch, case["ids"])
    if kind == "adapters":
        N, r, out, n = case["adapters"], case["rank"], case["out"], case["in"]
        return {"ids": torch.from_numpy(_requests(case, seed)).to(DEVICE, id_type),
                "x": _normal((case["rows"], n), seed, "x", dtype), "y": _normal((case["rows"], out), seed, "y", dtype),
                "down": _normal((N, r, n), seed, "down", dtype, n ** -0.5),
                "up": _normal((N, out, r), seed, "up", dtype, 0.3 * r ** -0.5),
                "scales": [2.0 / (1 + i % 3) for i in range(N)]}
    T, k, n = case["tokens"], case["top_k"], case["cols"]
    state = {"ids": torch.from_numpy(_routing(case, seed)).to(DEVICE, id_type), "experts": case["experts"],
             "grad": case["grad"]}
    if kind == "dispatch":
        state["x"] = _normal((T, n), seed, "x", dtype)
        if case["grad"]:
            state["drows"] = _normal((T * k, n), seed, "drows", dtype)
    if kind == "combine":
        state["y"] = _normal((T * k, n) if case["sorted"] else (T, k, n), seed, "y", dtype)
        state["weights"] = _weights(case, seed)
        state["sorted"] = case["sorted"]
        state["add"] = _normal((T, n), seed, "add", dtype) if case["add"] else None
        if case["grad"]:
            state["dout"] = _normal((T, n), seed, "dout", dtype)
    return state


def prepare(case: dict, seed: int) -> dict:
    state = {"kind": case["kind"], **_inputs(case, seed)}
    if not own:
        if case["kind"] == "combine" and case["sorted"]:  # the order that the rows were sorted in
            state["order"] = _plain_sort(state["ids"], state["experts"])
        return state
    if os.path.join(os.getcwd(), "mlx-iqk_amd") not in sys.path:
        sys.path.insert(1, os.path.join(os.getcwd(), "mlx-iqk_amd"))
    from mlx_iqk_amd import adapters, router
    state["router"] = router
    if case["kind"] == "adapters":  # the bank that a server loads its adapters into
        bank = adapters.LowRankAdapters(case["adapters"], case["out"], case["in"], case["rank"],
                                        dtype=DTYPES[case["dtype"]], device=DEVICE)
        down, up = state.pop("down"), state.pop("up")
        for i, scale in enumerate(state.pop("scales")):
            bank.load(i, down[i], up[i], scale)
        state["bank"] = bank
    elif case["kind"] == "combine":
        state["order"] = router.sort(state["ids"], state["experts"]) if case["sorted"] else None
        if case["grad"]:
            state["y"].requires_grad_()
            state["weights"].requires_grad_()
            if case["add"]:
                state["add"].requires_grad_()
    elif case["grad"]:
        state["x"].requires_grad_()
    return state


# --------------------------------------------------------------- the passes ---


def run(state: dict):
    return (_own if own else _plain)(state)


def _own(state: dict):
    kind, router = state["kind"], state["router"]
    if kind == "adapters":
        return state["bank"](state["x"], state["ids"], state["y"])
    if kind == "sort":
        return _order(router.sort(state["ids"], state["experts"]))
    if kind == "dispatch":
        rows, order = router.dispatch(state["x"], state["ids"], state["experts"])
        got = {"rows": rows, **_order(order)}
        if state["grad"]:
            (got["dx"],) = torch.autograd.grad(rows, state["x"], state["drows"])
            got["rows"] = rows.detach()
        return got
    out = router.combine(state["y"], state["weights"], state["order"], add=state["add"])
    if not state["grad"]:
        return {"out": out}
    wanted = [state["y"], state["weights"]] + ([state["add"]] if state["add"] is not None else [])
    grads = torch.autograd.grad(out, wanted, state["dout"])
    return {"out": out.detach(), **dict(zip(("dy", "dweights", "dadd"), grads))}


def _order(order) -> dict:
    return {"offsets": order.offsets, "ids": order.ids, "tokens": order.tokens, "slots": order.slots}


def _plain_sort(ids: torch.Tensor, experts: int) -> dict:
    key = torch.where((ids >= 0) & (ids < experts), ids, torch.full_like(ids, experts)).reshape(-1)
    order = torch.sort(key, stable=True)
    slots = torch.empty_like(order.indices)
    slots[order.indices] = torch.arange(key.numel(), device=key.device)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=key.device)
    counts.scatter_add_(0, key.to(torch.int64), torch.ones_like(slots))
    offsets = torch.cumsum(counts, 0) - counts
    whole = torch.int32
    return {"offsets": offsets.to(whole), "ids": order.values.to(whole),
            "tokens": (order.indices // ids.shape[-1]).to(whole), "slots": slots.reshape(ids.shape).to(whole)}


def _kept(slots: torch.Tensor, offsets: torch.Tensor) -> torch.Tensor:
    return (slots < offsets[-1]).to(torch.float32)


def _plain(state: dict):
    kind = state["kind"]
    if kind == "adapters":
        return _plain_adapters(state)
    if kind == "sort":
        return _plain_sort(state["ids"], state["experts"])
    if kind == "dispatch":
        order, x = _plain_sort(state["ids"], state["experts"]), state["x"]
        kept = (order["ids"] < state["experts"]).to(x.dtype)
        got = {"rows": x[order["tokens"]] * kept[:, None], **order}
        if state["grad"]:
            parts = state["drows"][order["slots"].to(torch.int64)].to(torch.float32)
            got["dx"] = (parts * _kept(order["slots"], order["offsets"])[..., None]).sum(-2).to(x.dtype)
        return got
    y, weights, dtype = state["y"], state["weights"], state["y"].dtype
    if state["sorted"]:
        slots = state["order"]["slots"].to(torch.int64)
        weights = weights * _kept(slots, state["order"]["offsets"])
        parts = y[slots]
    else:
        parts = y
    parts = parts.to(torch.float32)
    out = (weights[..., None] * parts).sum(-2)
    if state["add"] is not None:
        out = out + state["add"].to(torch.float32)
    got = {"out": out.to(dtype)}
    if state["grad"]:
        dout = state["dout"].to(torch.float32)
        dy = (weights[..., None] * dout[:, None]).to(dtype)
        dweights = (parts * dout[:, None]).sum(-1)
        if state["sorted"]:
            dweights = dweights * _kept(slots, state["order"]["offsets"])
            flat = torch.empty_like(y)
            flat[slots] = dy
            dy = flat
        got.update({"dy": dy, "dweights": dweights})
        if state["add"] is not None:
            got["dadd"] = state["dout"].clone()
    return got


def _plain_adapters(state: dict):
    """Adapter by adapter over the rows that name it; few rows each with its own copy."""
    x, y, ids = state["x"].to(torch.float32), state["y"].to(torch.float32), state["ids"]
    down, up = state["down"], state["up"]
    if x.shape[0] <= 64:
        at = torch.clamp(ids, min=0)
        scales = torch.tensor(state["scales"], device=x.device)[at] * (ids >= 0)
        t = (down[at].to(torch.float32) @ x[:, :, None])[:, :, 0] * scales[:, None]
        return (y + (up[at].to(torch.float32) @ t[:, :, None])[:, :, 0]).to(state["y"].dtype)
    order = torch.argsort(ids)
    counts = torch.bincount(ids + 1, minlength=down.shape[0] + 1).tolist()
    for a, rows in enumerate(torch.split(order, counts), start=-1):
        if a >= 0 and rows.numel():
            t = (x[rows] @ down[a].to(torch.float32).T) * state["scales"][a]
            y[rows] += t @ up[a].to(torch.float32).T
    return y.to(state["y"].dtype)


# ---------------------------------------------------------- what it is held to ---


def work(case: dict) -> dict:
    """Bytes: each input read once, each output written once.  Of the adapters, those
    that the rows name."""
    kind, size = case["kind"], DTYPES[case["dtype"]].itemsize
    id_size = 8 if case["ids"] == "int64" else 4
    if kind == "adapters":
        ids = _requests(case, 0)
        T, r, out, n = case["rows"], case["rank"], case["out"], case["in"]
        bank = int(np.unique(ids[ids >= 0]).size) * r * (out + n)
        with_one = int((ids >= 0).sum())
        return {"bytes": size * (bank + with_one * n + 2 * T * out) + T * id_size, "flops": 2 * with_one * r * (out + n)}
    T, E, k, n = case["tokens"], case["experts"], case["top_k"], case["cols"]
    P = T * k
    lists = P * (id_size + 12) + 4 * (E + 1)
    if kind == "sort":
        return {"bytes": lists, "flops": P}
    if kind == "dispatch":
        both = 2 if case["grad"] else 1
        return {"bytes": lists + both * size * n * (T + P) + (4 * P if case["grad"] else 0),
                "flops": P * n if case["grad"] else 0}
    bytes_ = size * n * (P + T * (2 if case["add"] else 1)) + P * (8 if case["sorted"] else 4)
    flops = 2 * P * n
    if case["grad"]:
        bytes_ += size * n * (T + 2 * P + (T if case["add"] else 0)) + P * (12 if case["sorted"] else 8)
        flops += 3 * P * n
    return {"bytes": bytes_, "flops": flops}


# ----------------------------------------------------------------- in 64 bits ---


def _exact_slots(ids: np.ndarray, experts: int):
    """Each pair's slot and whether it is kept, by a stable sort on the host."""
    key = np.where((ids >= 0) & (ids < experts), ids, experts).reshape(-1)
    pairs = np.argsort(key, kind="stable")
    slots = np.empty(key.size, dtype=np.int64)
    slots[pairs] = np.arange(key.size)
    return torch.from_numpy(slots.reshape(ids.shape)).to(DEVICE), torch.from_numpy(key.reshape(ids.shape) < experts).to(DEVICE)


def exact(case: dict, seed: int):
    kind = case["kind"]
    state = _inputs(case, seed)
    if kind == "sort":  # whole numbers, which have to be equal
        return None
    f64 = torch.float64
    if kind == "adapters":
        out, x, ids = state["y"].to(f64), state["x"].to(f64), state["ids"].tolist()
        for a in sorted(set(ids) - {-1}):
            rows = torch.tensor([i for i, v in enumerate(ids) if v == a], device=DEVICE)
            whole = state["scales"][a] * (state["up"][a].to(f64) @ state["down"][a].to(f64))
            out.index_add_(0, rows, x.index_select(0, rows) @ whole.T.contiguous())
        return out
    T, k, n = case["tokens"], case["top_k"], case["cols"]
    if kind == "combine" and not case["sorted"]:
        slots = torch.arange(T * k, device=DEVICE).reshape(T, k)
        kept = torch.ones_like(slots, dtype=torch.bool)
    else:
        slots, kept = _exact_slots(_routing(case, seed), case["experts"])
    if kind == "dispatch":
        x = state["x"].to(f64)
        rows = torch.zeros((T * k, n), dtype=f64, device=DEVICE)
        for j in range(k):
            rows[slots[:, j]] = torch.where(kept[:, j, None], x, 0.0)
        got = {"rows": rows, "offsets": None, "ids": None, "tokens": None, "slots": None}
        if case["grad"]:
            got["dx"] = sum(torch.where(kept[:, j, None], state["drows"][slots[:, j]].to(f64), 0.0) for j in range(k))
        return got
    y, w = state["y"].reshape(T * k, n), state["weights"].to(f64)
    out = state["add"].to(f64) if case["add"] else torch.zeros((T, n), dtype=f64, device=DEVICE)
    dy, dw = torch.zeros((T * k, n), dtype=f64, device=DEVICE) if case["grad"] else None, torch.zeros_like(w)
    dout = state["dout"].to(f64) if case["grad"] else None
    for j in range(k):
        part = torch.where(kept[:, j, None], y[slots[:, j]].to(f64), 0.0)
        out = out + w[:, j, None] * part
        if case["grad"]:
            dw[:, j] = (part * dout).sum(-1)
            dy[slots[:, j]] = torch.where(kept[:, j, None], w[:, j, None] * dout, 0.0)
    got = {"out": out}
    if case["grad"]:
        got.update({"dy": dy.reshape(state["y"].shape), "dweights": dw})
        if case["add"]:
            got["dadd"] = dout
    return got
