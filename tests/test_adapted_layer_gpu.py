"""Sort, dispatch, combine and adapters as a program uses them together: a verified block of
drafted tokens, the example's layer with its shared projection, calls on two streams at once."""

from __future__ import annotations

import importlib.util
import os

import numpy as np
import pytest
import torch

import mxref
import wirepack
from mlx_iqk_amd import format as fmt
from mlx_iqk_amd import _native, mx, router
from mlx_iqk_amd.adapters import LowRankAdapters
from mlx_iqk_amd.nn import IqkSwitchLinear

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
U = 2.0 ** -24
EXAMPLE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "mx_moe.py")


@pytest.fixture(scope="module")
def mx_moe():
    spec = importlib.util.spec_from_file_location("mx_moe", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _bank(rng, adapters, out, n, rank, dtype, device):
    bank = LowRankAdapters(adapters, out, n, rank, dtype=dtype, device=device)
    for a in range(adapters):
        bank.load(a, torch.from_numpy(rng.standard_normal((rank, n)) * n ** -0.5),
                  torch.from_numpy(rng.standard_normal((out, rank)) * rank ** -0.5), 1.0)
    return bank


@pytest.mark.parametrize("tokens", (1, 8))
def test_a_verified_block(device, tokens):
    """Pairs sorted, decoded a run of one expert at a time, and combined: the module's own call, summed."""
    print(f"verified block {tokens}", flush=True)
    rng = np.random.default_rng(tokens)
    experts, out, n, k = 8, 256, 2048, 6
    module = IqkSwitchLinear("iq2_k", experts, out, n, device=device)
    wire = wirepack.random_wire("iq2_k", experts * out, n, seed=2, scales="serving")
    shapes = fmt.component_shapes("iq2_k", experts, out, n)
    module.load_streams({k: np.ascontiguousarray(v).reshape(shapes[k]) for k, v in fmt.pack("iq2_k", wire, n).items()})
    x = torch.from_numpy(rng.standard_normal((tokens, n))).to(F16).to(device)
    ids = torch.from_numpy(np.stack([rng.permutation(experts)[:k] for _ in range(tokens)])).to(device)
    weights = torch.from_numpy(rng.random((tokens, k)).astype(np.float32)).to(device)

    def step():
        order = router.sort(ids, experts)
        return router.combine(module.gemv_union(x, order.ids, order.tokens), weights, order)

    got = step()
    y = module.gemv(x[:, None, None], ids)[:, :, 0]  # the same products, bit for bit
    assert torch.equal(got, router.combine(y.contiguous(), weights))
    parts, w = y.double().cpu().numpy(), weights.double().cpu().numpy()[..., None]
    # k fused additions in f32, one rounding
    size = np.abs(w * parts).sum(1)
    bound = (k + 1) * U * size + mxref.HALF_ULP[F16] * (np.abs((w * parts).sum(1)) + k * U * size) + mxref.TINY[F16]
    assert (np.abs(got.double().cpu().numpy() - (w * parts).sum(1)) <= bound).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step()
    for _ in range(3):
        ids.copy_(torch.from_numpy(np.stack([rng.permutation(experts)[:k] for _ in range(tokens)])))
        graph.replay()
        torch.cuda.synchronize()
        replayed = held.clone()
        assert torch.equal(replayed, step())
        torch.cuda.synchronize()


@pytest.mark.parametrize("tokens", (1, 4, 70))
def test_the_examples_layer_with_a_shared_projection(mx_moe, tokens):
    """The shared projection's output, its adapters with it, is added to the experts' sum before the one rounding."""
    print(f"example with adapters {tokens}", flush=True)
    torch.manual_seed(tokens)
    moe = mx_moe.random_layer(12, 160, 96, 3)
    x = torch.randn(tokens, 160, device="cuda", dtype=BF16)
    with torch.no_grad():
        alone, logits, _ = moe(x)
        bank = mx_moe.random_bank(moe, 5, 8)
        requests = torch.arange(tokens, device="cuda") % 6 - 1  # one of them without
        y, same, _ = moe(x, bank=bank, requests=requests)
        shared = bank(x, requests, moe.shared(x))
    assert torch.equal(logits, same)
    # `alone` is rounded once, y once: the sum of both lies within those roundings
    want, bound = alone.double() + shared.double(), mxref.HALF_ULP[BF16] * alone.double().abs()
    assert bool(((y.double() - want).abs() <= bound + mxref.HALF_ULP[BF16] * (want.abs() + bound) + 2.0 ** -100).all())
    serve = mx_moe.Server(moe, tokens, bank=bank)
    for turn in range(4):
        x = torch.randn(tokens, 160, device="cuda", dtype=BF16)
        requests = (requests + 2 + turn) % 6 - 1
        with torch.no_grad():
            want = moe(x, bank=bank, requests=requests)[0]
        torch.cuda.synchronize()
        assert torch.equal(serve(x, requests), want)
        torch.cuda.synchronize()


def test_calls_on_two_streams_at_once(device):
    """Each call's workspace is its own: many calls on two streams give what one after the other gives."""
    print("two streams", flush=True)
    rng = np.random.default_rng(4)
    bank = _bank(rng, 7, 520, 512, 16, BF16, device)
    jobs = []
    for rows in (900, 700):
        x = torch.from_numpy(rng.standard_normal((rows, 512))).to(BF16).to(device)
        y = torch.from_numpy(rng.standard_normal((rows, 520))).to(BF16).to(device)
        ids = torch.from_numpy(rng.integers(-1, 7, (rows, 40))).to(device)
        weights = torch.from_numpy(rng.random((rows, 40)).astype(np.float32)).to(device)
        jobs.append((x, y, ids, weights))

    def call(x, y, ids, weights):
        rows, order = router.dispatch(x, ids, 7)
        return bank(x, ids[:, 0], y), router.combine(rows, weights, order), order.slots

    want = [call(*job) for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[], []]
    for _ in range(10):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(call(*jobs[i]))
    torch.cuda.synchronize()
    for outs, expected in zip(got, want):
        for out in outs:
            assert all(torch.equal(a, b) for a, b in zip(out, expected))


def test_a_projection_of_no_rows(device):
    print("no rows", flush=True)
    proj = mx.MxLinear(64, 32, device=device)
    bank = LowRankAdapters(2, 64, 32, 4, device=device)
    y = proj(torch.empty((0, 32), dtype=BF16, device=device), bank, torch.empty(0, dtype=torch.int64, device=device))
    assert y.shape == (0, 64) and y.dtype == BF16


@pytest.mark.parametrize("out", (1, 3, 7, 8, 9))
@pytest.mark.parametrize("rows", (2, 1500))
def test_narrow_outputs(device, out, rows):
    """Rows of fewer outputs than a load takes."""
    print(f"narrow {out} {rows}", flush=True)
    rng = np.random.default_rng(out)
    bank = _bank(rng, 3, out, 16, 8, F16, device)
    x = torch.from_numpy(rng.integers(-3, 4, (rows, 16))).to(F16).to(device)
    y = torch.from_numpy(rng.standard_normal((rows, out))).to(F16).to(device)
    ids = rng.integers(-1, 3, rows)
    got = bank(x, torch.from_numpy(ids).to(device), y).double().cpu().numpy()
    held = [bank.adapter(a) for a in range(3)]
    for a in range(-1, 3):
        at = np.nonzero(ids == a)[0]
        old = y.double().cpu().numpy()[at]
        if a < 0:
            np.testing.assert_array_equal(got[at], old)
            continue
        down, up = (t.double().cpu().numpy() for t in held[a][:2])
        t = x.double().cpu().numpy()[at] @ down.T
        size = np.abs(old) + np.abs(x.double().cpu().numpy()[at]) @ np.abs(down).T @ np.abs(up).T
        # sums of 16 and of 9 terms in f32, a step each; one rounding
        error = 60 * U * size
        want = old + t @ up.T
        assert (np.abs(got[at] - want) <= error + mxref.HALF_ULP[F16] * (np.abs(want) + error) + mxref.TINY[F16]).all()


def test_the_example_server_wants_requests_with_a_bank_only(mx_moe):
    """A step without requests would take those of the step before."""
    print("example server's requests", flush=True)
    torch.manual_seed(3)
    moe = mx_moe.random_layer(6, 64, 32, 2)
    x = torch.randn(2, 64, device="cuda", dtype=BF16)
    requests = torch.tensor([0, 1], device="cuda")
    bare = mx_moe.Server(moe, 2)
    with torch.no_grad():
        assert torch.equal(bare(x), moe(x)[0])
    with pytest.raises(ValueError, match="without"):
        bare(x, requests)
    bank = LowRankAdapters(2, 64, 64, 4, device="cuda")
    for given in ((bank, requests), (bank, None), (None, requests)):
        with pytest.raises(ValueError, match="shared"):
            moe(x, bank=given[0], requests=given[1])
    bank = mx_moe.random_bank(moe, 2, 4)
    serve = mx_moe.Server(moe, 2, bank=bank)
    with torch.no_grad():
        assert torch.equal(serve(x, requests), moe(x, bank=bank, requests=requests)[0])
    with pytest.raises(ValueError, match="-1 for none"):
        serve(x)


def test_the_example_serves_as_many_requests_as_its_prompts_hold(mx_moe):
    print("example of few prompts", flush=True)
    assert len(mx_moe.main(["--experts", "8", "--hidden", "256", "--inner", "128", "--top-k", "2", "--sequences", "2",
                            "--tokens", "6", "--steps", "2", "--requests", "12"])) == 2


def test_the_examples_layer_of_many_rows(mx_moe):
    """As many rows as go through the adapters' tiles, served from a graph as called."""
    print("example with tiles", flush=True)
    torch.manual_seed(9)
    tokens = 1100
    moe = mx_moe.random_layer(12, 160, 96, 3)
    x = torch.randn(tokens, 160, device="cuda", dtype=BF16)
    requests = torch.arange(tokens, device="cuda") % 6 - 1
    with torch.no_grad():
        alone = moe(x)[0]
        bank = mx_moe.random_bank(moe, 5, 8)
        assert _native.load().iqk_adapters_work(160, 160, 8, 5, tokens) > 0
        y = moe(x, bank=bank, requests=requests)[0]
        shared = bank(x, requests, moe.shared(x))
    # `alone` is rounded once, y once: the sum of both lies within those roundings
    want, bound = alone.double() + shared.double(), mxref.HALF_ULP[BF16] * alone.double().abs()
    assert bool(((y.double() - want).abs() <= bound + mxref.HALF_ULP[BF16] * (want.abs() + bound) + 2.0 ** -100).all())
    serve = mx_moe.Server(moe, tokens, bank=bank)
    for turn in range(3):
        x = torch.randn(tokens, 160, device="cuda", dtype=BF16)
        requests = (requests + 2 + turn) % 6 - 1
        with torch.no_grad():
            want = moe(x, bank=bank, requests=requests)[0]
        torch.cuda.synchronize()
        assert torch.equal(serve(x, requests), want)
        torch.cuda.synchronize()
