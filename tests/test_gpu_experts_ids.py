"""The ids of a plan agree with its other parts, whatever becomes of the tensor that they were given in."""

import numpy as np
import pytest
import torch

from comp_b200 import experts
from oracle import mx as ref
from tests.test_gpu_mx import device_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,top,n", [(0, 2, 3), (1, 1, 1), (50, 4, 9), (700, 8, 257), (9000, 2, 5)])
def test_ids_outside_the_experts(cuda, tokens, top, n):
    """Negative ids, and ids beyond the experts, are -1, as their rows are."""
    rng = np.random.default_rng(tokens)
    ids = rng.integers(-3, n + 2, (tokens, top)).astype(np.int32)
    if tokens > 5:
        ids[1, 0], ids[2, 0] = -(1 << 31), (1 << 31) - 1
    plan = experts.sort(torch.from_numpy(ids).to(cuda), n)
    want = np.where((ids >= 0) & (ids < n), ids, -1)
    assert plan.ids.dtype == torch.int32 and plan.ids.shape == (tokens, top) and plan.weights is None
    assert np.array_equal(plan.ids.cpu().numpy(), want)
    assert np.array_equal(plan.pos.cpu().numpy(), ref.sort(want, n)[1])
    assert device_error() == (5 if (ids >= n).any() else 0)


@pytest.mark.parametrize("tokens", [30, 3000])
def test_ids_after_their_buffer_is_reused(cuda, tokens):
    """A step loop writes the next step's ids into the same tensor."""
    gen = torch.Generator(device=cuda).manual_seed(tokens)
    steps = [torch.randint(-1, 12, (tokens, 4), generator=gen, device=cuda, dtype=torch.int32) for _ in range(3)]
    buffer, plans = torch.empty_like(steps[0]), []
    for ids in steps:
        buffer.copy_(ids)
        plans.append(experts.sort(buffer, 12))
    for plan, ids in zip(plans, steps):
        assert torch.equal(plan.ids, ids)
    # captured: a replay's ids are those of its own step
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        plan = experts.sort(buffer, 12)
        inside = plan.ids
    for ids in steps:
        buffer.copy_(ids)
        graph.replay()
        buffer.zero_()
        assert torch.equal(plan.ids, ids) and torch.equal(inside, ids)
