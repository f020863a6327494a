"""Layers of experts (comp_b200.experts) on the GPU against a restatement in 64 bits (oracle.mx). Whole numbers are exact.

Bounds. A routing weight is an f32 quotient of exponentials: exp is off by at most 2 units in the last place (2^-22), its argument
by half a unit of the difference (2^-24 of at most 104, where exp is 0), the sum of n by n * 2^-24, the quotient by 2^-24:
(2^-21 + 104 * 2^-24 + n * 2^-24) of the weight, and 2^-149 where it is next to 0. Products: see test_gpu_mx. A combined sum of n
rows is off by n * 2^-24 * mass before its own rounding."""

import os

import numpy as np
import pytest
import torch

from comp_b200 import experts, mx
from oracle import mx as ref
from tests.test_gpu_mx import DT, HALF, check, device_error, packed, planes

pytestmark = pytest.mark.gpu


def check_plan(plan, ids, n):
    offsets, pos, order = ref.sort(ids, n)
    assert np.array_equal(plan.offsets.cpu().numpy(), offsets)
    assert np.array_equal(plan.pos.cpu().numpy(), pos)
    assert np.array_equal(plan.order.cpu().numpy(), order)
    return offsets, pos, order


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("tokens,n,top", [(1, 1, 1), (1, 8, 2), (1, 128, 8), (3, 32, 32), (64, 33, 4), (128, 128, 8), (129, 64, 6),
                                          (1000, 257, 10), (5003, 40, 3), (257, 1024, 32), (4000, 512, 1)])
@pytest.mark.parametrize("normalize", [True, False])
def test_route(cuda, dtype, tokens, n, top, normalize):
    rng = np.random.default_rng(tokens + n)
    x = rng.standard_normal((tokens, n)) * 2
    x[:, rng.permutation(n)[: n // 4]] = -np.inf  # masked experts: where too few are left, ids are -1
    if tokens > 2:
        x[1] = -np.inf
        x[2, n // 2 :] = np.nan
    x = torch.from_numpy(x).to(DT[dtype])
    plan = experts.route(x.to(cuda), top, normalize=normalize)
    ids, weights = ref.route(x.float().numpy(), top, normalize)
    assert np.array_equal(plan.ids.cpu().numpy(), ids)
    check_plan(plan, ids, n)
    e = np.abs(plan.weights.double().cpu().numpy() - weights)
    assert (e <= (2.0**-21 + (104 + n) * 2.0**-24) * weights + 2.0**-149).all()
    assert device_error() == 0


def test_route_ties_and_infinities(cuda):
    x = torch.tensor([[1.0, 3.0, 3.0, 0.0, 3.0], [0.0, -0.0, 0.0, -0.0, 0.0], [float("inf"), 1.0, float("inf"), 5.0, -1.0],
                      [-3e38, -3.4e38, 3e38, float("-inf"), float("nan")], [1e-45, 0.0, -1e-45, 2e-45, -0.0]], device=cuda)
    plan = experts.route(x, 3)
    # (f32's smallest number is 1.4e-45: 1e-45 and 2e-45 are both rounded to it, so that the lower index comes first)
    assert plan.ids.tolist() == [[1, 2, 4], [0, 1, 2], [0, 2, 3], [2, 0, 1], [0, 3, 1]]
    ids, weights = ref.route(x.cpu().numpy(), 3)
    assert np.array_equal(plan.ids.cpu().numpy(), ids) and np.allclose(plan.weights.cpu().numpy(), weights, rtol=1e-6, atol=0)
    check_plan(plan, ids, 5)


def test_route_strides(cuda):
    x = torch.randn((200, 300), device=cuda)
    for v in (x[:, 7:90], x[::3, :64], x.T[:150, :100], x[:1].expand(9, 300)):
        a, b = experts.route(v, 4), experts.route(v.contiguous(), 4)
        for name in ("ids", "weights", "offsets", "pos", "order"):
            assert torch.equal(getattr(a, name), getattr(b, name))


@pytest.mark.parametrize("tokens,top,n", [(0, 1, 3), (1, 1, 1), (1, 8, 64), (7, 3, 5), (64, 8, 128), (1024, 4, 1000), (1025, 4, 17),
                                          (4097, 1, 2), (3000, 10, 160), (20000, 8, 1024), (131072, 1, 7),
                                          (128, 32, 600), (4096, 1, 33), (600, 32, 1000), (300000, 8, 64)])
def test_sort(cuda, tokens, top, n):
    rng = np.random.default_rng(tokens)
    ids = rng.integers(-1 if tokens % 2 else 0, n, (tokens, top))
    ids[: tokens // 3] = np.minimum(ids[: tokens // 3], n // 3)  # popular ones, and the same one twice
    check_plan(experts.sort(torch.from_numpy(ids.astype(np.int32)).to(cuda), n), ids, n)
    assert device_error() == 0


def test_sort_all_skipped_and_beyond(cuda):
    ids = torch.full((50, 4), -1, dtype=torch.int32, device=cuda)
    check_plan(experts.sort(ids, 9), ids.cpu().numpy(), 9)
    assert device_error() == 0
    ids[3, 1], ids[9, 2], ids[10, 0] = 9, 1 << 30, 2
    ids[11, 0] = -(1 << 31)
    check_plan(experts.sort(ids, 9), ids.cpu().numpy(), 9)
    assert device_error() == 5 and device_error() == 0


def expert_case(rng, tokens, top, n_experts, n, k, dtype, gather, skip=0, skew=False):
    ids = np.stack([rng.permutation(n_experts)[:top] for _ in range(tokens)]).reshape(tokens, top) if top <= n_experts else None
    if skew:
        ids[:, 0] = n_experts // 2
    if skip:
        ids.reshape(-1)[::skip] = -1
    rows = tokens if gather else tokens * top
    x = torch.from_numpy(rng.standard_normal((rows, k)) * np.exp(rng.standard_normal((rows, 1)))).to(DT[dtype])
    return ids, x, planes(rng, (n_experts, n, k))


@pytest.mark.parametrize("gather", [True, False])
@pytest.mark.parametrize("tokens,top,n_experts,n,k,skip", [
    (1, 1, 1, 1, 32, 0), (1, 8, 64, 256, 512, 0), (1, 2, 4, 300, 2080, 0), (3, 4, 8, 128, 4096, 0), (16, 2, 8, 700, 288, 3),
    (61, 6, 40, 512, 1440, 0), (64, 8, 160, 130, 256, 0), (200, 3, 4, 1000, 544, 5), (300, 2, 2, 260, 1024, 0),
    (1000, 2, 9, 513, 320, 7), (700, 4, 5, 3500, 96, 0), (5, 1, 1000, 64, 64, 0), (16, 8, 100, 200, 320, 0), (16, 1, 3, 4000, 96, 4),
    (2, 8, 9, 130, 5000 // 32 * 32, 0), (13, 9, 16, 20000, 64, 0), (17, 2, 6, 300, 288, 0)])
def test_linear(cuda, gather, tokens, top, n_experts, n, k, skip):
    rng = np.random.default_rng(tokens + n + k)
    dtype = ("f32", "f16", "bf16")[(tokens + n) % 3]
    ids, x, w = expert_case(rng, tokens, top, n_experts, n, k, dtype, gather, skip, skew=tokens > 100)
    plan = experts.sort(torch.from_numpy(ids.astype(np.int32)).to(cuda), n_experts)
    offsets, _, order = check_plan(plan, ids, n_experts)
    if not gather:
        x[offsets[-1] :] = float("nan")  # sorted rows that are nobody's
    vx = ref.values(*ref.quantize(x.float().numpy()))
    want, mass = ref.experts_linear(vx, ref.values(*w), offsets, order, top, gather)
    tw = packed(w, cuda)
    out = torch.full((tokens * top, n), 9.0, dtype=DT[dtype], device=cuda)
    for y, d in ((experts.linear(x.to(cuda), tw, plan, gather=gather, dtype=torch.float32), "f32"),
                 (experts.linear(x.to(cuda), tw, plan, gather=gather, out=out), dtype)):
        check(y[: offsets[-1]], want[: offsets[-1]], mass[: offsets[-1]], k, d)
    assert bool((out[offsets[-1] :] == 9).all())  # rows past the last stay as they were
    assert device_error() == 0


@pytest.mark.parametrize("counts", [[0, 40, 1, 0, 33, 64], [65, 0, 2, 100, 31, 0, 96, 1], [5] * 30 + [127, 128, 129, 0, 63],
                                    [0, 0, 300], [257, 1, 0, 3]])
@pytest.mark.parametrize("n,k", [(260, 352), (1500, 544)])
def test_popular_experts(cuda, counts, n, k):
    """Experts with far more rows than the average that the tiles are planned by, around the tiles' borders."""
    rng = np.random.default_rng(len(counts) + n)
    ids = rng.permutation(np.repeat(np.arange(len(counts)), counts))[:, None]
    tokens = len(ids)
    x = torch.from_numpy(rng.standard_normal((tokens, k)).astype(np.float32))
    w = (rng.integers(0, 256, (len(counts), n, k // 2), dtype=np.uint8),
         rng.integers(116, 122, (len(counts), n, k // 32), dtype=np.uint8))
    plan = experts.sort(torch.from_numpy(ids.astype(np.int32)).to(cuda), len(counts))
    offsets, _, order = check_plan(plan, ids, len(counts))
    want, mass = ref.experts_linear(ref.values(*ref.quantize(x.numpy())), ref.values(*w), offsets, order, 1)
    check(experts.linear(x.to(cuda), packed(w, cuda), plan), want, mass, k, "f32")
    assert device_error() == 0


@pytest.mark.parametrize("n", [100, 40000])
def test_same_expert_twice(cuda, n):
    """A token whose choices are all of one expert gets a row for each."""
    rng = np.random.default_rng(n)
    ids = np.array([[3, 3, 3], [0, 3, 0], [1, -1, 1]])
    x, w = torch.from_numpy(rng.standard_normal((3, 96)).astype(np.float32)), planes(rng, (4, n, 96))
    plan = experts.sort(torch.from_numpy(ids.astype(np.int32)).to(cuda), 4)
    offsets, _, order = check_plan(plan, ids, 4)
    want, mass = ref.experts_linear(ref.values(*ref.quantize(x.numpy())), ref.values(*w), offsets, order, 3)
    check(experts.linear(x.to(cuda), packed(w, cuda), plan)[: offsets[-1]], want[: offsets[-1]], mass[: offsets[-1]], 96, "f32")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("tokens,top,n", [(1, 1, 1), (1, 8, 4096), (33, 3, 113), (64, 8, 1000), (300, 10, 258), (7, 32, 20), (1, 5, 4)])
@pytest.mark.parametrize("weighted", [True, False])
def test_combine(cuda, dtype, tokens, top, n, weighted):
    rng = np.random.default_rng(tokens + n)
    ids = rng.integers(-1, 12, (tokens, top))
    if tokens > 3:
        ids[2] = -1  # a token whose choices all go nowhere
    plan = experts.sort(torch.from_numpy(ids.astype(np.int32)).to(cuda), 12)
    _, pos, _ = check_plan(plan, ids, 12)
    y = torch.from_numpy(rng.standard_normal((tokens * top, n))).to(DT[dtype])
    y[(pos >= 0).sum() :] = float("nan")  # rows that are nobody's are not read
    w = torch.from_numpy(rng.random((tokens, top)).astype(np.float32)) if weighted else None
    got = experts.combine(y.to(cuda), plan, w.to(cuda) if weighted else None)
    want, mass = ref.combine(y.double().numpy(), pos, None if w is None else w.numpy())
    assert got.dtype == DT[dtype] and got.shape == (tokens, n)
    e = np.abs(got.double().cpu().numpy() - want)
    assert (e <= top * 2.0**-24 * mass * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + 2.0**-25 * (dtype == "f16")).all()
    wide = torch.full((tokens, n + 3), 5.0, dtype=DT[dtype], device=cuda)
    padded = torch.cat([y, y[:, :1]], 1).to(cuda)
    experts.combine(padded[:, :n], plan, w.to(cuda) if weighted else None, out=wide[:, 1 : n + 1])
    assert torch.equal(wide[:, 1 : n + 1], got) and bool((wide[:, :1] == 5).all()) and bool((wide[:, n + 1 :] == 5).all())


def layer(x, logits, w_up, w_down, top):
    plan = experts.route(logits, top)
    gate, up = experts.linear(x, w_up, plan).chunk(2, dim=-1)
    y = experts.linear(torch.nn.functional.silu(gate) * up, w_down, plan, gather=False)
    return experts.combine(y, plan, plan.weights)


@pytest.mark.parametrize("tokens", [1, 5, 130])
def test_layer(cuda, tokens):
    """Routing, both products and the way back as a model calls them, step by step against 64 bits: each step's error is
    bounded above, so the chain is checked by giving every step the kernel's own input to it. Then captured and replayed."""
    rng = np.random.default_rng(tokens)
    hidden, inner, n, top = 320, 192, 16, 4
    up, down = planes(rng, (n, 2 * inner, hidden)), planes(rng, (n, hidden, inner))
    tu, td = packed(up, cuda), packed(down, cuda)
    x = torch.from_numpy(rng.standard_normal((tokens, hidden)).astype(np.float32)).to(cuda)
    logits = torch.from_numpy(rng.standard_normal((tokens, n)).astype(np.float32)).to(cuda)
    plan = experts.route(logits, top)
    ids, _ = ref.route(logits.cpu().numpy(), top)
    offsets, pos, order = check_plan(plan, ids, n)
    h = experts.linear(x, tu, plan)
    vx = ref.values(*ref.quantize(x.cpu().numpy()))
    check(h, *ref.experts_linear(vx, ref.values(*up), offsets, order, top), hidden, "f32")
    a = torch.nn.functional.silu(h[:, :inner]) * h[:, inner:]
    y = experts.linear(a, td, plan, gather=False)
    va = ref.values(*ref.quantize(a.cpu().numpy()))
    check(y, *ref.experts_linear(va, ref.values(*down), offsets, order, top, False), inner, "f32")
    out = experts.combine(y, plan, plan.weights)
    want, mass = ref.combine(y.double().cpu().numpy(), pos, plan.weights.cpu().numpy())
    assert (np.abs(out.double().cpu().numpy() - want) <= (top + 1) * 2.0**-24 * mass).all()
    assert torch.equal(layer(x, logits, tu, td, top), out)
    graph = torch.cuda.CUDAGraph()
    xs, ls = x.clone(), logits.clone()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = layer(xs, ls, tu, td, top)
    for i in range(3):
        xs.copy_(x.roll(i, 1))
        ls.copy_(logits.roll(i, 1))
        graph.replay()
        assert torch.equal(got, layer(x.roll(i, 1), logits.roll(i, 1), tu, td, top))
    assert device_error() == 0


def test_example(cuda):
    import runpy

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    main = runpy.run_path(os.path.join(root, "examples", "expert_layer.py"))["main"]
    assert main(["--hidden", "512", "--inner", "192", "--experts", "12", "--top", "3", "--prompt", "40", "--steps", "3"]) == 0


def test_no_tokens(cuda):
    w = packed(planes(np.random.default_rng(0), (3, 40, 64)), cuda)
    plan = experts.route(torch.empty((0, 3), device=cuda), 2)
    assert plan.offsets.tolist() == [0, 0, 0, 0] and plan.ids.shape == (0, 2)
    y = experts.linear(torch.empty((0, 64), device=cuda), w, plan)
    assert y.shape == (0, 40) and experts.combine(y, plan, plan.weights).shape == (0, 40)


def test_refusals(cuda):
    w = packed(planes(np.random.default_rng(0), (3, 40, 64)), cuda)
    logits = torch.zeros((4, 3), device=cuda)
    plan = experts.route(logits, 2)
    x, y = torch.ones((4, 64), device=cuda), torch.ones((8, 40), device=cuda)
    one = mx.quantize(x)
    small = torch.empty(128, dtype=torch.uint8, device=cuda)
    for call, kind in [(lambda: experts.route(logits, 4), ValueError), (lambda: experts.route(logits, 0), ValueError),
                       (lambda: experts.route(logits, 2.0), TypeError), (lambda: experts.route(logits[0], 1), ValueError),
                       (lambda: experts.route(logits.int(), 1), TypeError), (lambda: experts.route(logits.cpu(), 1), RuntimeError),
                       (lambda: experts.route(torch.zeros((2, 1025), device=cuda), 1), ValueError),
                       (lambda: experts.route(torch.zeros((2, 100), device=cuda), 33), ValueError),
                       (lambda: experts.sort(plan.ids.long(), 3), TypeError), (lambda: experts.sort(plan.ids, 0), ValueError),
                       (lambda: experts.sort(plan.ids, 1025), ValueError), (lambda: experts.sort(plan.ids[0], 3), ValueError),
                       (lambda: experts.sort(plan.ids.cpu(), 3), RuntimeError),
                       (lambda: experts.linear(x, one, plan), ValueError), (lambda: experts.linear(x, x, plan), TypeError),
                       (lambda: experts.linear(x, w, plan.ids), TypeError), (lambda: experts.linear(y, w, plan), ValueError),
                       (lambda: experts.linear(x, w, plan, gather=False), ValueError),
                       (lambda: experts.linear(x.cpu(), w, plan), RuntimeError),
                       (lambda: experts.linear(x, w, plan, dtype=torch.int8), TypeError),
                       (lambda: experts.linear(x, w, experts.route(torch.zeros((4, 4), device=cuda), 2)), ValueError),
                       (lambda: experts.linear(x, w, plan, out=y.T), ValueError),
                       (lambda: experts.linear(torch.ones((40, 64), device=cuda), w, experts.route(torch.zeros((40, 3), device=cuda), 2),
                                               workspace=small), ValueError),
                       (lambda: experts.combine(y[:7], plan), ValueError), (lambda: experts.combine(y.double(), plan), TypeError),
                       (lambda: experts.combine(y, plan, plan.weights.half()), TypeError),
                       (lambda: experts.combine(y, plan, plan.weights[:, :1]), ValueError),
                       (lambda: experts.combine(y, plan, out=y), ValueError), (lambda: experts.combine(y, None), TypeError)]:
        with pytest.raises(kind):
            call()
