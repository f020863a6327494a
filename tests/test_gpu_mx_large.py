"""MXFP4 and experts where offsets pass 32 bits, and calls that overlap on streams."""

import pytest
import torch

from comp_b200 import experts, mx
from tests.test_gpu_mx import device_error

pytestmark = pytest.mark.gpu


def _rows(n, k, dev):
    """A bf16 matrix too large to make at once with a generator's f32 numbers: rows that differ, cheaply."""
    base = torch.randn((4099, k), device=dev, generator=torch.Generator(device=dev).manual_seed(1)).bfloat16()
    x = torch.empty((n, k), dtype=torch.bfloat16, device=dev)
    for i in range(0, n, 4099):
        m = min(4099, n - i)
        x[i : i + m] = base[:m] * (1 + (i // 4099) % 7)
    return x


def test_image_past_32_bits(cuda):
    n, k = 1_050_001, 8192  # 8.6e9 values, an image of 4.57e9 bytes
    x = _rows(n, k, cuda)
    w = mx.quantize(x)
    assert w.nbytes > 1 << 32
    tail = x[-300:].contiguous()
    del x
    few = mx.quantize(tail)
    q = torch.randn((1, k), device=cuda)
    # the product's last columns are those of the last rows alone (the same order of sums: one tile's K is whole in both)
    y = mx.linear(q, w)
    assert y.shape == (1, n)
    z = mx.matmul(mx.quantize(q), few, dtype=torch.float32)
    assert torch.allclose(y[:, -300:], z, rtol=1e-5, atol=1e-5 * float(z.abs().max()))
    # and the image itself, read back from a view of its last tiles
    first = (n - 300) // 128
    end = mx.MXTensor(w.image[mx.image_bytes(first * 128, k) :], n - first * 128, k)
    assert torch.equal(mx.dequantize(end, torch.bfloat16)[-300:], mx.dequantize(few, torch.bfloat16))
    assert device_error() == 0


def test_results_past_32_bits(cuda):
    m, n, k = 70_003, 40_001, 64  # 2.8e9 results
    a, w = mx.quantize(_rows(m, k, cuda)), mx.quantize(torch.randn((n, k), device=cuda))
    y = mx.matmul(a, w)
    va, vw = mx.dequantize(a), mx.dequantize(w)
    for rows in (slice(0, 5), slice(35_000, 35_003), slice(m - 5, m)):
        want = (va[rows].double() @ vw.double().T).float()
        assert torch.allclose(y[rows].float(), want, rtol=2.0**-8, atol=1e-6 * float(want.abs().max()))
    assert device_error() == 0


@pytest.mark.parametrize("m,n,k", [(2, 10_000, 29_696), (4, 20_000, 27_904), (1, 130, 61_440), (3, 19_000, 16_384), (300, 500, 61_440)])
def test_long_sums(cuda, m, n, k):
    """Rows so long that one launch has no room for them, and just short enough; against 64 bits on the operands' own values
    (bound as in test_gpu_mx: K / 32 sums of blocks, each off by at most 2^-23 of the magnitudes so far)."""
    gen = torch.Generator(device=cuda).manual_seed(k)
    x, w = (torch.randn(s, generator=gen, device=cuda) for s in ((m, k), (n, k)))
    w = mx.quantize(w)
    y = mx.linear(x, w)
    va, vw = mx.dequantize(mx.quantize(x)).double(), mx.dequantize(w).double()
    want, mass = va @ vw.T, va.abs() @ vw.abs().T
    assert bool(((y.double() - want).abs() <= (k / 32 + 8) * 2.0**-23 * mass + 2.0**-24 * want.abs()).all())
    assert device_error() == 0


def test_combine_past_32_bits(cuda):
    tokens, top, n = 150_001, 2, 8192  # 2.46e9 values
    y = _rows(tokens * top, n, cuda)
    plan = experts.sort(torch.randint(0, 5, (tokens, top), dtype=torch.int32, device=cuda), 5)
    out = experts.combine(y, plan)
    for t in (0, 77_777, tokens - 1):
        want = (y[plan.pos[t].long()].double()).sum(0)
        assert torch.allclose(out[t].double(), want, rtol=2.0**-8, atol=1e-30)


def test_threads_on_the_default_stream(cuda):
    """Threads whose calls come between one another's launches: each has scratch of its own, of any size in turn."""
    import threading

    gen = torch.Generator(device=cuda).manual_seed(3)
    w = mx.quantize(torch.randn((700, 1024), generator=gen, device=cuda))
    xs = [[torch.randn((m, 1024), generator=gen, device=cuda) for m in (5 + i, 300, 20, 9000, 130)] for i in range(4)]
    want = [[mx.linear(x, w) for x in row] for row in xs]
    got = [[] for _ in xs]

    def work(i):
        for _ in range(30):
            got[i].append([mx.linear(x, w) for x in xs[i]])

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, rounds in enumerate(got):
        assert len(rounds) == 30 and all(torch.equal(a, b) for r in rounds for a, b in zip(r, want[i]))


@pytest.mark.parametrize("tokens", [1, 40, 700])
def test_layers_on_two_streams(cuda, tokens):
    """The same weights used by two streams at once, each call with memory of its own."""
    gen = torch.Generator(device=cuda).manual_seed(tokens)
    up, down = (mx.quantize(torch.randn(s, generator=gen, device=cuda)) for s in ((16, 512, 320), (16, 320, 512)))
    xs = [torch.randn((tokens, 320), generator=gen, device=cuda) for _ in range(2)]
    logits = [torch.randn((tokens, 16), generator=gen, device=cuda) for _ in range(2)]

    def layer(x, l):
        plan = experts.route(l, 4)
        return experts.combine(experts.linear(experts.linear(x, up, plan).tanh(), down, plan, gather=False), plan, plan.weights)

    want = [layer(x, l) for x, l in zip(xs, logits)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer(xs[i], logits[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])
    assert device_error() == 0
