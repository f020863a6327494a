"""MXFP4 operands and products (comp_b200.mx) on the GPU, through the C-ABI, against a restatement in 64 bits (oracle.mx).

Bounds. Codes, scales and the values that they stand for are exact (the steps are: an exponent, a product with a power of two,
one rounding). A product's sum over a block of 32 is a whole multiple of 1/4 of at most 32 * 36, exact in f32; K / 32 such sums and
up to 8 parts of K are added in f32, each step off by at most 2^-23 of the sum of magnitudes so far, whether it rounds or
cuts off: (K / 32 + 8) * 2^-23 * mass, mass = sum |a w|. A result in a type of p bits is off by half a step more, 2^-p
of its value (bf16 2^-8, f16 2^-11, f32 2^-24), and in f16 by half its smallest step, 2^-25."""

import ctypes

import numpy as np
import pytest
import torch

from comp_b200 import _lib, mx
from oracle import mx as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def device_error():
    code = ctypes.c_int()
    _lib.call("b2q_device_error", ctypes.byref(code), 1)
    return code.value


def bound(want, mass, k, dtype):
    return (k / 32 + 8) * 2.0**-23 * mass * (1 + 2.0**-8) + HALF[dtype] * np.abs(want) + (2.0**-25 if dtype == "f16" else 0)


def check(got, want, mass, k, dtype):
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    assert np.array_equal(np.isnan(got), np.isnan(want))
    worst = np.nan_to_num(np.abs(got - want) - bound(want, mass, k, dtype), nan=-1.0)
    assert worst.size == 0 or worst.max() <= 0, f"past the bound by {worst.max():.3e} at {np.unravel_index(worst.argmax(), worst.shape)}"


def planes(rng, shape, spread=0.0):
    """Planes of gaussian values whose blocks differ by powers of two around 2^spread."""
    x = rng.standard_normal(shape).astype(np.float32)
    if spread:
        x = x.reshape(*shape[:-1], -1, 32) * np.exp2(np.round(rng.standard_normal((*shape[:-1], shape[-1] // 32, 1)) * spread))
    return ref.quantize(x.reshape(shape).astype(np.float32))


def packed(p, dev):
    return mx.pack(*(torch.from_numpy(a).to(dev) for a in p))


def special_rows(k, dtype):
    """Rows where a block's scale or a rounding can go wrong."""
    rng = np.random.default_rng(7)
    i = np.arange(k)
    rows = [np.zeros(k), -np.zeros(k), np.full(k, 1e-42), (i % 97) * 0.0625, -(i % 64) * 0.125 * 2.0**-9,
            np.where(i % 32 == 31, 6.0, 0.25 * (i % 29)), np.where(i % 32 == 0, 7.99, 5.0), np.where(i % 32 == 5, 4.0, 2.5),
            rng.standard_normal(k) * 1e-38, np.where(i % 32 == 3, 3e38, 1.0), np.where(i % 64 == 40, np.inf, 1.0),
            np.where(i % 96 == 70, -np.inf, 2.0), np.where(i % 64 == 1, np.nan, 3.0), np.exp2(rng.integers(-120, 120, k))]
    x = torch.from_numpy(np.stack(rows)).to(DT[dtype])
    return x if dtype != "f16" else torch.cat([x, torch.full((1, k), 6.0e-8, dtype=DT[dtype])])


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 64), (129, 288), (128, 256), (37, 2080), (260, 512)])
def test_quantize(cuda, dtype, rows, k):
    rng = np.random.default_rng(rows + k)
    x = torch.from_numpy(rng.standard_normal((rows, k)) * np.exp2(rng.integers(-8, 8, (rows, 1)))).to(DT[dtype])
    p = ref.quantize(x.float().numpy())
    t = mx.quantize(x.to(cuda))
    assert t.shape == (rows, k) and t.nbytes == t.image.numel() == _lib.load().b2q_mx_bytes(1, rows, k)
    want = ref.image(*p).reshape(-1, 17408)
    got = t.image.cpu().numpy().reshape(-1, 17408)
    # rows past the last are not part of the tensor: compare the codes of those that are, and their scales
    stages = -(-k // 256)
    for tile in range(-(-rows // 128)):
        n = min(128, rows - tile * 128)
        a, b = (z[tile * stages : (tile + 1) * stages] for z in (got, want))
        assert np.array_equal(a[:, : n * 128], b[:, : n * 128])
        sa, sb = (z[:, 16384:].reshape(stages, 2, 32, 4, 4).transpose(0, 1, 3, 2, 4).reshape(stages, 2, 128, 4) for z in (a, b))
        assert np.array_equal(sa[:, :, :n], sb[:, :, :n])
    assert torch.equal(mx.dequantize(t, DT[dtype]).cpu(), torch.from_numpy(ref.values(*p)).to(DT[dtype]))
    assert torch.equal(packed(p, cuda).image.cpu(), torch.from_numpy(ref.image(*p)))


@pytest.mark.parametrize("dtype", DT)
def test_quantize_special_values(cuda, dtype):
    x = special_rows(192, dtype)
    p = ref.quantize(x.float().numpy())
    got = mx.dequantize(mx.quantize(x.to(cuda))).cpu().double().numpy()
    assert np.array_equal(got, ref.values(*p), equal_nan=True)


def test_every_code_and_scale(cuda):
    """All 16 codes at all 256 scales, read back in each type with one rounding."""
    codes = np.tile(np.arange(256, dtype=np.uint8)[None, :16] * 17, (256, 2))
    codes[:, 16:] = np.arange(16) | (15 - np.arange(16)) << 4
    scales = np.repeat(np.arange(256, dtype=np.uint8)[:, None], 2, 1)
    t = packed((codes, scales), cuda)
    want = torch.from_numpy(ref.values(codes, scales))
    for dtype in DT.values():
        assert torch.equal(mx.dequantize(t, dtype).cpu().nan_to_num(nan=1.25), want.to(dtype).nan_to_num(nan=1.25))


@pytest.mark.parametrize("dtype", DT)
def test_strides(cuda, dtype):
    """Columns of a wider tensor, every other row, a transposed view, and a base that is not aligned."""
    rng = np.random.default_rng(3)
    wide = torch.from_numpy(rng.standard_normal((40, 201))).to(DT[dtype]).to(cuda)
    for x in (wide[:, 8:136], wide[::2, 3:67], wide[:, :40].T[:, :32], wide[5:6, 1:129], wide[:1].expand(6, 201)[:, :96]):
        want = ref.values(*ref.quantize(x.float().cpu().numpy()))
        assert np.array_equal(mx.dequantize(mx.quantize(x)).double().cpu().numpy(), want)
        p = planes(rng, (70, x.shape[1]))
        w = ref.values(*p)
        check(mx.linear(x, packed(p, cuda), dtype=torch.float32), want @ w.T, np.abs(want) @ np.abs(w).T, x.shape[1], "f32")


SHAPES = [(1, 1, 32), (1, 128, 256), (1, 4096, 8192), (2, 130, 96), (5, 700, 4096), (16, 128, 2048), (31, 257, 288), (32, 128, 32),
          (33, 1000, 1440), (64, 128, 512), (65, 129, 544), (96, 2000, 4096), (127, 384, 4096), (128, 5003, 320), (129, 300, 2080),
          (200, 14336, 512), (255, 20000, 64), (256, 128, 256), (257, 4864, 1024), (300, 19000, 288), (700, 6000, 2304),
          (1500, 4096, 4096)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_matmul(cuda, m, n, k):
    rng = np.random.default_rng(m * 7 + n + k)
    a, w = planes(rng, (m, k)), planes(rng, (n, k))
    va, vw = (torch.from_numpy(ref.values(*p)).to(cuda) for p in (a, w))
    want, mass = (va @ vw.T).cpu().numpy(), (va.abs() @ vw.abs().T).cpu().numpy()
    ta, tw = packed(a, cuda), packed(w, cuda)
    for dtype in DT:
        check(mx.matmul(ta, tw, dtype=DT[dtype]), want, mass, k, dtype)
    assert device_error() == 0


@pytest.mark.parametrize("m,n,k", [(1, 300, 4096), (40, 200, 1024), (130, 260, 544), (400, 5000, 512)])
@pytest.mark.parametrize("spread", [3.0, 12.0])
def test_blocks_of_different_sizes(cuda, m, n, k, spread):
    """Scales far apart along K, so that sums are rounded."""
    rng = np.random.default_rng(m + k)
    a, w = planes(rng, (m, k), spread), planes(rng, (n, k), spread)
    va, vw = ref.values(*a), ref.values(*w)
    check(mx.matmul(packed(a, cuda), packed(w, cuda), dtype=torch.float32), va @ vw.T, np.abs(va) @ np.abs(vw).T, k, "f32")


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("m,n,k", [(1, 513, 96), (17, 384, 1056), (150, 128, 256), (260, 9000, 320), (1, 1, 32), (1, 1000, 4096),
                                   (2, 130, 8192), (8, 40000, 288), (9, 300, 2080), (16, 20000, 1056), (16, 128, 5120), (3, 2000, 14336),
                                   (1, 2000, 28672), (16, 9700, 7168)])
def test_linear(cuda, dtype, m, n, k):
    rng = np.random.default_rng(m + n)
    x = torch.from_numpy(rng.standard_normal((m, k))).to(DT[dtype])
    w = planes(rng, (n, k)) if n * k < 1 << 24 else (rng.integers(0, 256, (n, k // 2), dtype=np.uint8),
                                                     rng.integers(116, 122, (n, k // 32), dtype=np.uint8))
    vx, vw = (torch.from_numpy(ref.values(*p)).to(cuda) for p in (ref.quantize(x.float().numpy()), w))
    tw = packed(w, cuda)
    y = mx.linear(x.to(cuda), tw)
    assert y.dtype == DT[dtype] and device_error() == 0
    check(y, (vx @ vw.T).cpu().numpy(), (vx.abs() @ vw.abs().T).cpu().numpy(), k, dtype)
    # out: any row stride and alignment; what lies around it stays
    wide = torch.full((m, n + 5), 7.0, dtype=DT[dtype], device=cuda)
    assert mx.linear(x.to(cuda), tw, out=wide[:, 3 : n + 3]).data_ptr() == wide[:, 3:].data_ptr()
    assert torch.equal(wide[:, 3 : n + 3], y) and bool((wide[:, :3] == 7).all()) and bool((wide[:, n + 3 :] == 7).all())


@pytest.mark.parametrize("m", [1, 40, 300])
def test_not_finite(cuda, m):
    """A block that is not finite makes its row or its column NaN, and nothing else."""
    rng = np.random.default_rng(m)
    n, k = 200, 544
    x = rng.standard_normal((m, k)).astype(np.float32)
    x[m // 2, 40] = np.inf
    w = planes(rng, (n, k))
    w[1][77, 3] = 255
    vx, vw = ref.values(*ref.quantize(x)), ref.values(*w)
    with np.errstate(invalid="ignore"):
        check(mx.linear(torch.from_numpy(x).to(cuda), packed(w, cuda)), vx @ vw.T, np.abs(vx) @ np.abs(vw).T, k, "f32")


def test_no_rows(cuda):
    w = packed(planes(np.random.default_rng(0), (40, 64)), cuda)
    assert mx.linear(torch.empty((0, 64), device=cuda), w).shape == (0, 40)
    none = mx.quantize(torch.empty((0, 64), device=cuda))
    assert mx.dequantize(none).shape == (0, 64) and mx.matmul(none, w).shape == (0, 40)
    assert mx.matmul(w, none).shape == (40, 0) and mx.linear(torch.ones((3, 64), device=cuda), none).shape == (3, 0)


@pytest.mark.parametrize("dtype", DT)
def test_experts_in_one_tensor(cuda, dtype):
    """Operands of experts begin at whole tiles, whatever their rows."""
    rng = np.random.default_rng(6)
    for shape in ((1, 5, 32), (3, 1, 96), (4, 128, 64), (3, 200, 288), (1024, 2, 32)):
        x = torch.from_numpy(rng.standard_normal(shape)).to(DT[dtype])
        want = ref.values(*ref.quantize(x.float().numpy()))
        t = mx.quantize(x.to(cuda))
        assert t.shape == shape and t.nbytes == t.image.numel()
        assert np.array_equal(mx.dequantize(t).double().cpu().numpy(), want)
        assert torch.equal(mx.dequantize(packed(ref.quantize(x.float().numpy()), cuda)).double().cpu(), torch.from_numpy(want))
    t = mx.quantize(torch.randn((96, 3, 8), device=cuda).permute(1, 2, 0))  # any strides
    assert t.shape == (3, 8, 96)


def test_from_ggml(cuda):
    rng = np.random.default_rng(2)
    codes, scales = planes(rng, (3, 50, 96))
    blocks = np.concatenate([scales[..., None], codes.reshape(3, 50, 3, 16)], -1)
    t = mx.from_ggml(torch.from_numpy(blocks.reshape(-1)).to(cuda), 50, 96, experts=3)
    assert t.shape == (3, 50, 96)
    assert np.array_equal(mx.dequantize(t).double().cpu().numpy(), ref.values(codes, scales))
    one = mx.from_ggml(torch.from_numpy(blocks[1].reshape(-1)).to(cuda), 50, 96)
    assert torch.equal(mx.dequantize(one), mx.dequantize(t)[1])


def test_gguf(cuda, tmp_path):
    """A weight and a layer of experts through a GGUF file, against gguf-py's own reading of the blocks."""
    gguf = pytest.importorskip("gguf")
    from comp_b200 import gguf_io

    rng = np.random.default_rng(4)
    one, many = planes(rng, (40, 96), 5.0), planes(rng, (3, 20, 64), 5.0)
    kind = gguf.GGMLQuantizationType.MXFP4
    path = str(tmp_path / "w.gguf")
    w = gguf.GGUFWriter(path, "test")
    blocks = {}
    for name, (codes, scales) in (("one", one), ("many", many)):
        b = np.concatenate([scales[..., None], codes.reshape(*scales.shape, 16)], -1)
        blocks[name] = b.reshape(*scales.shape[:-1], -1)
        w.add_tensor(name, blocks[name], raw_dtype=kind)
    w.add_tensor("plain", np.zeros((4, 32), dtype=np.float32))
    w.write_header_to_file(), w.write_kv_data_to_file(), w.write_tensors_to_file(), w.close()
    for name, (codes, scales) in (("one", one), ("many", many)):
        t = gguf_io.load_mx(path, name, device=cuda)
        assert t.shape == (*scales.shape[:-1], scales.shape[-1] * 32)
        got = mx.dequantize(t).cpu().numpy()
        assert np.array_equal(got.astype(np.float64), ref.values(codes, scales))
        assert np.array_equal(got, gguf.dequantize(blocks[name], kind))
    with pytest.raises(ValueError):
        gguf_io.load_mx(path, "plain", device=cuda)
    with pytest.raises(KeyError):
        gguf_io.load_mx(path, "none", device=cuda)


@pytest.mark.parametrize("m", [1, 70, 300])
def test_streams_and_graphs(cuda, m):
    """Another stream, and a captured call that is replayed on new inputs while eager calls run on another stream."""
    rng = np.random.default_rng(m)
    n, k = 640, 1056
    w = packed(planes(rng, (n, k)), cuda)
    xs = [torch.from_numpy(rng.standard_normal((m, k)).astype(np.float32)).to(cuda) for _ in range(4)]
    want = [mx.linear(x, w) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    x = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = mx.linear(x, w)
        z = mx.linear(y[:, :544].contiguous(), mx.quantize(xs[1][:1, :544].expand(33, 544)))
    for i, a in enumerate(xs):
        x.copy_(a)
        with torch.cuda.stream(side):
            other = [mx.linear(b, w) for b in xs for _ in range(5)]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[i]) and bool(torch.isfinite(z).all())
        assert all(torch.equal(o, want[j // 5]) for j, o in enumerate(other))
    assert device_error() == 0


def test_same_result_every_time(cuda):
    rng = np.random.default_rng(5)
    a, w = packed(planes(rng, (3, 8192), 9.0), cuda), packed(planes(rng, (500, 8192), 9.0), cuda)
    first = mx.matmul(a, w, dtype=torch.float32)
    assert all(torch.equal(first, mx.matmul(a, w, dtype=torch.float32)) for _ in range(20))


def test_weights_quantized_right_before(cuda):
    """The product starts early beside the call's own quantizer; weights that the kernel before it writes are complete."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    for i in range(10):
        wv = torch.randn((4096, 1024), generator=gen, device=cuda)
        x = torch.randn((3, 1024), generator=gen, device=cuda)
        many = x.repeat(30, 1)
        calls = (lambda w: mx.linear(x, w), lambda w: mx.linear(many, w), lambda w: mx.matmul(mx.quantize(x), w))
        got = [call(mx.quantize(wv)) for call in calls]
        w = mx.quantize(wv)
        torch.cuda.synchronize()
        for call, y in zip(calls, got):
            assert torch.equal(call(w), y)


def test_refusals(cuda):
    w = packed(planes(np.random.default_rng(0), (40, 64)), cuda)
    we = packed(planes(np.random.default_rng(0), (2, 40, 64)), cuda)
    x = torch.ones((3, 64), device=cuda)
    for call, kind in [(lambda: mx.quantize(x.double()), TypeError), (lambda: mx.quantize(x.cpu()), RuntimeError),
                       (lambda: mx.quantize(x[:, :40]), ValueError), (lambda: mx.quantize(x[0]), ValueError),
                       (lambda: mx.quantize(x[:, :0]), ValueError), (lambda: mx.dequantize(x), TypeError),
                       (lambda: mx.dequantize(w, torch.int32), TypeError), (lambda: mx.linear(x[:, :32], w), ValueError),
                       (lambda: mx.linear(x, x), TypeError), (lambda: mx.linear(x, we), ValueError),
                       (lambda: mx.linear(x.cpu(), w), RuntimeError), (lambda: mx.linear(x.int(), w), TypeError),
                       (lambda: mx.linear(x, w, dtype=torch.float64), TypeError),
                       (lambda: mx.linear(x, w, out=torch.empty((3, 41), device=cuda)), ValueError),
                       (lambda: mx.linear(x, w, out=torch.empty((40, 3), device=cuda).T), ValueError),
                       (lambda: mx.linear(x, w, out=torch.empty((1, 40), device=cuda).expand(3, 40)), ValueError),
                       (lambda: mx.matmul(x, w), TypeError), (lambda: mx.matmul(w, we), ValueError),
                       (lambda: mx.matmul(mx.quantize(x[:, :32]), w), ValueError),
                       (lambda: mx.matmul(w, w, dtype=torch.int8), TypeError),
                       (lambda: mx.pack(torch.zeros((3, 16), device=cuda), torch.zeros((3, 1), device=cuda)), TypeError),
                       (lambda: mx.pack(torch.zeros((3, 16), dtype=torch.uint8, device=cuda),
                                        torch.zeros((3, 2), dtype=torch.uint8, device=cuda)), ValueError),
                       (lambda: mx.from_ggml(torch.zeros(33, dtype=torch.uint8, device=cuda), 1, 64), ValueError),
                       (lambda: mx.MXTensor(torch.zeros(100, dtype=torch.uint8, device=cuda), 1, 32), ValueError),
                       (lambda: mx.MXTensor(torch.zeros(17408 + 64, dtype=torch.uint8, device=cuda)[64:], 1, 32), ValueError),
                       (lambda: mx.MXTensor(torch.zeros(17408, dtype=torch.uint8), 1, 32), RuntimeError)]:
        with pytest.raises(kind):
            call()
