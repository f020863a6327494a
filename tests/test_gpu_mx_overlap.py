"""Products of a few rows on many streams at once, and in the branches of one graph: their CTAs share SMs, whose tensor memory
they take and give back, and none waits for another call's. Results are those of the calls one by one."""

import pytest
import torch

from comp_b200 import experts, mx
from tests.test_gpu_mx import device_error

pytestmark = pytest.mark.gpu

# [N][K], rows: clusters of 8, 4 and 2 CTAs and single ones, from one stage a CTA to so many that scales take 512 columns
SIZES = [(1024, 4096, 1), (2048, 2048, 4), (2880, 2880, 2), (2000, 1024, 3), (4096, 1024, 1), (128, 256, 4), (9000, 27_136, 1),
         (20_000, 512, 2), (300, 61_440, 1), (5000, 9472, 3)]


def _calls(cuda):
    """Calls of a few rows, one of many, and a layer of experts for one token."""
    gen = torch.Generator(device=cuda).manual_seed(11)
    calls = []
    for n, k, m in SIZES:
        w = mx.quantize(torch.randn((n, k), generator=gen, device=cuda))
        x = torch.randn((m, k), generator=gen, device=cuda)
        calls.append(lambda w=w, x=x: mx.linear(x, w))
    w, a = (mx.quantize(torch.randn(s, generator=gen, device=cuda)) for s in ((4096, 1024), (300, 1024)))
    calls.append(lambda: mx.matmul(a, w))
    up = mx.quantize(torch.randn((16, 512, 2048), generator=gen, device=cuda))
    x, plan = torch.randn((1, 2048), generator=gen, device=cuda), experts.route(torch.randn((1, 16), generator=gen, device=cuda), 4)
    calls.append(lambda: experts.linear(x, up, plan))
    return calls


def test_streams(cuda):
    calls = _calls(cuda)
    want = [call() for call in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(8)]
    for turn in range(30):  # each time other calls beside one another
        got = []
        for i in range(len(calls) * 4):
            j = (i * (1 + turn % 5) + turn) % len(calls)
            with torch.cuda.stream(streams[i % 8]):
                got.append((j, calls[j]()))
        torch.cuda.synchronize()
        assert all(torch.equal(y, want[j]) for j, y in got)
    assert device_error() == 0


def test_branches_of_a_graph(cuda):
    calls = _calls(cuda)
    want = [call() for call in calls]
    torch.cuda.synchronize()
    graph, streams = torch.cuda.CUDAGraph(), [torch.cuda.Stream() for _ in calls]
    with torch.cuda.graph(graph):
        main, got = torch.cuda.current_stream(), []
        for call, s in zip(calls, streams):
            s.wait_stream(main)
            with torch.cuda.stream(s):
                got.append([call() for _ in range(3)])
        for s in streams:
            main.wait_stream(s)
    for _ in range(20):
        for row in got:
            for y in row:
                y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, w) for row, w in zip(got, want) for y in row)
    assert device_error() == 0
