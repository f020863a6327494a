"""Captured chains of MXFP4 calls equal the same calls made one by one, a refused question changes no product, and plans whose
choices all go nowhere."""

import copy

import pytest
import torch

from comp_b200 import experts, mx
from tests.test_gpu_mx import device_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m", [1, 4, 5, 70, 300])
def test_chain_replayed(cuda, m):
    """A product whose rows are the product before it and whose weights are quantized in the graph too; scratch of each call is
    its own at every replay."""
    gen = torch.Generator(device=cuda).manual_seed(m)
    w = mx.quantize(torch.randn((640, 1056), generator=gen, device=cuda))
    xs = [torch.randn((m, 1056), generator=gen, device=cuda) for _ in range(4)]
    vs = [torch.randn((33, 544), generator=gen, device=cuda) for _ in range(4)]

    def chain(x, v):
        y = mx.linear(x, w)
        v4 = mx.quantize(v)
        z = mx.linear(y[:, :544].contiguous(), v4)
        return y, z, mx.linear(z[:, :32].contiguous(), mx.quantize(y[:, :32]))

    want = [[t.clone() for t in chain(x, v)] for x, v in zip(xs, vs)]
    x, v = xs[0].clone(), vs[0].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = chain(x, v)
    for turn in range(3):
        for i in range(4):
            x.copy_(xs[i]), v.copy_(vs[i])
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(got, want[i])), (turn, i)
    assert device_error() == 0


def test_product_after_a_refused_question(cuda):
    gen = torch.Generator(device=cuda).manual_seed(2)
    w = mx.quantize(torch.randn((2, 300, 64), generator=gen, device=cuda))
    x = torch.randn((4, 64), generator=gen, device=cuda)
    other, plan = (experts.sort(torch.randint(0, 2, (4, 1), generator=gen, device=cuda, dtype=torch.int32), n) for n in (300, 2))
    with pytest.raises(ValueError, match="expected"):
        experts.workspace_size(other, w)
    assert torch.equal(experts.linear(x, w, plan), experts.linear(x, copy.deepcopy(w), plan))


@pytest.mark.parametrize("tokens,k", [(1, 64), (4, 4096), (40, 256), (700, 1024)])
@pytest.mark.parametrize("gather", [True, False])
def test_no_choice_goes_anywhere(cuda, tokens, k, gather):
    """All of a machine's experts are held elsewhere: products leave their rows as they were, and tokens get zeros."""
    w = mx.quantize(torch.randn((5, 300, k), device=cuda))
    plan = experts.sort(torch.full((tokens, 3), -1, dtype=torch.int32, device=cuda), 5)
    assert int(plan.offsets.abs().sum()) == 0 and bool((plan.order == -1).all())
    y = torch.full((tokens * 3, 300), 7.0, device=cuda)
    experts.linear(torch.randn((tokens if gather else tokens * 3, k), device=cuda), w, plan, gather=gather, out=y)
    assert bool((y == 7).all())
    out = experts.combine(torch.full_like(y, float("nan")), plan, torch.ones((tokens, 3), device=cuda))
    assert bool((out == 0).all()) and device_error() == 0
