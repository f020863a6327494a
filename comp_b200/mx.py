"""MXFP4 operands and their products (an extension beyond the reference, whose formats are integer quants).

MXFP4 holds 4-bit floating-point values (a sign over 0, 0.5, 1, 1.5, 2, 3, 4, 6) in blocks of 32 along K that share a power of
two: 4.25 bits a value, for weights and activations alike, multiplied as they are by the tensor cores. An `MXTensor` is an
operand in the order that they read; `quantize` makes one from values, `pack` from planes of codes and scales, `from_ggml` from
ggml's block_mxfp4, and `dequantize` gives back the values that one stands for. `linear` is a layer's call: rows of f32, f16 or
bf16, quantized and multiplied. The kernels are this package's own, through the C-ABI (include/comp_b200.h, where the formulas
stand); like comp_b200.host the functions take CUDA tensors only, run on the current stream of their device, and raise
TypeError / ValueError / RuntimeError on what they do not take.

    w = mx.from_ggml(blocks, n, k)             # or mx.quantize(weights)
    y = mx.linear(x, w)                        # x [M][k] -> y [M][n] of x's type
"""

import struct
import threading

import torch

from . import _lib
from .kv import DTYPE_ID, _dtype_id, _on_device, _raw_stream

# A token's step is many calls of a few microseconds on the GPU: what a call costs on the host counts. So the functions
# look at the common case first (contiguous, aligned), make tensors from tensors, and enter the library once.
_current_device = torch._C._cuda_getDevice
_pack_linear = struct.Struct(_lib.MX_LINEAR_ARGS).pack

TILE_ROWS, STAGE, STAGE_BYTES = 128, 256, 17408  # an image: 128 rows by 256 values a run of bytes
MAX_EXPERTS = 1024
FUSED_ROWS = 4  # products of up to so many rows may quantize them in their own launch

# Scratch of a call that is launched on the default stream, where one call's kernels write it only once the call before has
# ended: each thread keeps up to 4 MB of it a device (another thread's launches may come between a call's two). Other streams,
# captured ones among them, get theirs call by call.
KEPT_BYTES = 4 << 20
_kept = threading.local()


def _scratch(index, need, like):
    """A tensor of `need` bytes at least, for use on the current stream of device `index`, which is like's."""
    if need > KEPT_BYTES or _raw_stream(index):
        return like.new_empty(need, dtype=torch.uint8)
    kept = _kept.__dict__.get(index)
    if kept is None or kept.numel() < need:
        kept = _kept.__dict__[index] = like.new_empty(min(KEPT_BYTES, 2 * need), dtype=torch.uint8)
    return kept


def image_bytes(rows, k, experts=1):
    """Bytes of the image of `experts` operands of [rows][k]."""
    return experts * -(-rows // TILE_ROWS) * -(-k // STAGE) * STAGE_BYTES


def _enter(index, entry, *args):
    """The library's entry on device `index` and its current stream (the last argument)."""
    if _current_device() == index:
        rc = entry(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = entry(*args, _raw_stream(index))
    if rc:
        raise (ValueError if rc in (-1, -2, -4) else _error(rc))(_lib.last_error())


def _error(code):
    return lambda text: _lib.B2QError(code, text)


def _check_k(name, k):
    if k < 32 or k % 32:
        raise ValueError(f"{name}: K={k} is not a positive multiple of the MXFP4 block (32)")


def _check_experts(name, experts):
    if not 1 <= experts <= MAX_EXPERTS:
        raise ValueError(f"{name}: {experts} experts (1..{MAX_EXPERTS})")


class MXTensor:
    """An MXFP4 operand [rows][k], or [experts][rows][k], as its image: uint8, 128-byte aligned, as quantize, pack and from_ggml
    make it (include/comp_b200.h)."""

    def __init__(self, image, rows, k, experts=None):
        _check_k("MXTensor", k)
        if rows < 0:
            raise ValueError(f"MXTensor: {rows} rows")
        if experts is not None:
            _check_experts("MXTensor", experts)
        if not isinstance(image, torch.Tensor) or image.device.type != "cuda":
            raise RuntimeError("comp_b200.MXTensor: the image must be a CUDA tensor (this backend has no CPU path)")
        if image.dtype != torch.uint8:
            raise TypeError(f"MXTensor: image dtype {image.dtype}, expected torch.uint8")
        need = image_bytes(rows, k, experts or 1)
        if image.dim() != 1 or image.numel() < need or not image.is_contiguous() or (need and image.data_ptr() % 128):
            raise ValueError(f"MXTensor: the image must be {need} contiguous bytes, 128-byte aligned, got {tuple(image.shape)}")
        self._set(image, rows, k, experts)

    def _set(self, image, rows, k, experts):
        self._image, self.rows, self.k, self.experts = image, rows, k, experts
        self._at, self._index = image.data_ptr(), image.get_device()
        self._sizes = {}  # workspaces of products with few rows

    def __reduce__(self):  # a copy's image lies elsewhere
        return MXTensor, (self._image, self.rows, self.k, self.experts)

    @property
    def image(self):
        return self._image

    @property
    def device(self):
        return self._image.device

    @property
    def shape(self):
        return (self.rows, self.k) if self.experts is None else (self.experts, self.rows, self.k)

    @property
    def nbytes(self):
        return image_bytes(self.rows, self.k, self.experts or 1)

    def __repr__(self):
        return f"MXTensor({list(self.shape)}, device={self.device})"


def _cuda(name, t):
    """The number of a CUDA tensor's device."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"comp_b200.{name}: tensors must be CUDA tensors (this backend has no CPU path)")
    return t.get_device()


def _same(name, index, t):
    """Raises unless t is a tensor on CUDA device `index`."""
    if not isinstance(t, torch.Tensor) or t.get_device() != index:
        _on_device(name, torch.device("cuda", index), t)


def _rows(t):
    """(t, its address, its row stride): unit column stride, a 16-byte aligned base and rows that do not overlap (a copy only
    when needed)."""
    at = t.data_ptr()
    if t.is_contiguous() and not at & 15:
        return t, at, t.shape[1]
    (m, k), (s0, s1) = t.shape, t.stride()
    if s1 != 1 or at & 15 or (m > 1 and (s0 * t.element_size() & 15 or s0 < k)):
        t = t.clone(memory_format=torch.contiguous_format)
        return t, t.data_ptr(), k
    return t, at, s0 if m > 1 else k


def _stride(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def quantize(x):
    """x [M][K], or [experts][M][K] (f32, f16 or bf16; any strides) -> MXTensor. Each block of 32 values along K takes the power
    of two that brings its largest magnitude to 4 .. 8; values are rounded to nearest even and cut off at 6. Blocks with an
    infinity or a NaN are NaN."""
    index = _cuda("quantize", x)
    did = DTYPE_ID.get(x.dtype)
    if did is None:
        _dtype_id("quantize: x", x)
    shape, experts = x.shape, None
    if len(shape) == 3:
        experts, m, k = shape
        _check_experts("quantize", experts)
        x = x.flatten(0, 1)
    elif len(shape) == 2:
        m, k = shape
    else:
        raise ValueError(f"quantize: x {tuple(shape)}, expected [M][K] or [experts][M][K]")
    _check_k("quantize", k)
    x, at, ldx = _rows(x)
    image = x.new_empty(image_bytes(m, k, experts or 1), dtype=torch.uint8)
    t = MXTensor.__new__(MXTensor)
    t._set(image, m, k, experts)
    _enter(index, _lib.load().b2q_mx_quantize, did, at, ldx, experts or 1, m, k, t._at)
    return t


def dequantize(t, dtype=torch.float32):
    """The values of an MXTensor, each rounded once to `dtype`: [rows][k], or [experts][rows][k]."""
    if not isinstance(t, MXTensor):
        raise TypeError(f"dequantize: expected an MXTensor, got {type(t).__name__}")
    did = _out_dtype("dequantize", dtype)
    y = t._image.new_empty(t.shape, dtype=dtype)
    _enter(t._index, _lib.load().b2q_mx_dequantize, t._at, t.experts or 1, t.rows, t.k, did, y.data_ptr(), t.k)
    return y


def pack(codes, scales):
    """Planes codes uint8 [N][K/2] (in a block of 16 bytes byte i = value i in the low nibble, value i + 16 in the high one) and
    scales uint8 [N][K/32], or with a leading axis of experts -> MXTensor."""
    index = _cuda("pack", codes)
    _same("pack", index, scales)
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise TypeError(f"pack: codes {codes.dtype} and scales {scales.dtype}, expected torch.uint8")
    if codes.dim() not in (2, 3) or codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != 16 * scales.shape[-1]:
        raise ValueError(f"pack: codes {tuple(codes.shape)} and scales {tuple(scales.shape)}, expected [..][N][K/2] and [..][N][K/32]")
    n, k = codes.shape[-2], codes.shape[-1] * 2
    _check_k("pack", k)
    experts = codes.shape[0] if codes.dim() == 3 else None
    if experts is not None:
        _check_experts("pack", experts)
    codes, scales = codes.contiguous(), scales.contiguous()
    if codes.data_ptr() % 16:
        codes = codes.clone()
    image = codes.new_empty(image_bytes(n, k, experts or 1))
    t = MXTensor.__new__(MXTensor)
    t._set(image, n, k, experts)
    _enter(index, _lib.load().b2q_mx_pack, codes.data_ptr(), scales.data_ptr(), experts or 1, n, k, t._at)
    return t


def from_ggml(blocks, n, k, experts=None):
    """ggml's block_mxfp4 (17 bytes: the scale, 16 bytes of codes) as a CUDA uint8 tensor, the bytes as stored in a GGUF file:
    n rows of k values, or `experts` times as many -> MXTensor."""
    _cuda("from_ggml", blocks)
    _check_k("from_ggml", k)
    count = (1 if experts is None else experts) * n * (k // 32)
    if blocks.dtype != torch.uint8:
        raise TypeError(f"from_ggml: blocks dtype {blocks.dtype}, expected torch.uint8")
    if n < 0 or (experts is not None and experts < 1) or blocks.numel() != count * 17:
        raise ValueError(f"from_ggml: {blocks.numel()} bytes do not hold {count} MXFP4 blocks of 17")
    b = blocks.reshape((n, k // 32, 17) if experts is None else (experts, n, k // 32, 17))
    return pack(b[..., 1:].flatten(-2), b[..., 0])


def _check_out(name, out, dtype, shape, index):
    """The address and row stride of a given output: unit column stride, rows that do not overlap."""
    _same(name, index, out)
    if out.dtype != dtype or out.shape != shape or (shape[1] > 1 and out.stride(1) != 1) or \
            (shape[0] > 1 and out.stride(0) < shape[1]):
        raise ValueError(f"{name}: out must be a {dtype} {shape} tensor with unit column stride on cuda:{index}")
    return out.data_ptr(), _stride(out)


def _out_dtype(name, dtype):
    did = DTYPE_ID.get(dtype)
    if did is None:
        raise TypeError(f"{name}: dtype {dtype}, expected float32, float16 or bfloat16")
    return did


def matmul(a, w, dtype=torch.bfloat16, out=None):
    """MXTensors a [M][K] and w [N][K] -> a w^T [M][N]: exact products, f32 sums, rounded once to `dtype`. out: the tensor for
    the result (any row stride; it shares no memory with the operands)."""
    for t, name in ((a, "a"), (w, "w")):
        if not isinstance(t, MXTensor):
            raise TypeError(f"matmul: {name} must be an MXTensor, got {type(t).__name__}")
        if t.experts is not None:
            raise ValueError(f"matmul: {name} {t.shape} has experts (comp_b200.experts.linear)")
    index = w._index
    if a.k != w.k or a._index != index:
        raise ValueError(f"matmul: a {a.shape} on {a.device} and w {w.shape} on {w.device}")
    did = _out_dtype("matmul", dtype)
    if out is None:
        out = a._image.new_empty((a.rows, w.rows), dtype=dtype)
        at, ldy = out.data_ptr(), w.rows
    else:
        at, ldy = _check_out("matmul", out, dtype, (a.rows, w.rows), index)
    _enter(index, _lib.load().b2q_mx_matmul, a._at, w._at, a.rows, w.rows, a.k, did, at, ldy)
    return out


def _few_size(w, key, name, *args):
    """The workspace of a product of w with few rows, which may be one launch that needs none."""
    size = w._sizes.get(key)
    if size is None:
        with torch.cuda.device(w.device):
            size = w._sizes[key] = getattr(_lib.load(), name)(*args)
    return size


def linear(x, w, dtype=None, out=None):
    """x [M][K] (f32, f16 or bf16; any strides), quantized to MXFP4, times w [N][K] -> [M][N] of `dtype` (default: x's).
    out: the tensor for the result (any row stride; it shares no memory with x)."""
    if not isinstance(w, MXTensor):
        raise TypeError(f"linear: w must be an MXTensor, got {type(w).__name__}")
    if w.experts is not None:
        raise ValueError(f"linear: w {w.shape} has experts (comp_b200.experts.linear)")
    index, k, n = w._index, w.k, w.rows
    _same("linear", index, x)
    given = x.dtype
    xid = DTYPE_ID.get(given)
    if xid is None:
        _dtype_id("linear: x", x)
    shape = x.shape
    if len(shape) != 2 or shape[1] != k:
        raise ValueError(f"linear: x {tuple(shape)}, expected [M][{k}]")
    m = shape[0]
    if dtype is None or dtype is given:
        dtype, did = given, xid
    else:
        did = _out_dtype("linear", dtype)
    x, x_at, ldx = _rows(x)
    if out is None:
        out = x.new_empty((m, n)) if did == xid else x.new_empty((m, n), dtype=dtype)
        at, ldy = out.data_ptr(), n
    else:
        at, ldy = _check_out("linear", out, dtype, (m, n), index)
    need = image_bytes(m, k) if m > FUSED_ROWS else _few_size(w, m, "b2q_mx_linear_workspace_size", m, n, k)
    workspace = _scratch(index, need, x) if need else None
    _enter(index, _lib.load().b2q_mx_linear,
           _pack_linear(x_at, w._at, at, workspace.data_ptr() if need else 0, ldx, m, n, k, ldy, need, xid, did))
    return out
