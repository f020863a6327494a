"""Quantized KV cache and the attention that reads it (an extension beyond the reference, which has no attention).

A `KVCache` holds paged keys and values as ggml blocks (q4_0: 4.5 bits a value, q8_0: 8.5 bits). `kv_write` quantizes
tokens into it, `kv_read` gives back the values that it stands for, and `attention` runs queries against it: single
tokens (decode), a few tokens a sequence (drafts) or prompt chunks, with capped scores, a bias by distance, sliding
windows, prefix and document masks. The kernels are this package's own, through the C-ABI (include/comp_b200.h, where
the layouts and formulas stand); like comp_b200.host the functions take CUDA tensors only, run on the current stream of
their device, and raise TypeError / ValueError / RuntimeError on what they do not take.

    cache = kv.KVCache("q4_0", pages=4096, page_size=64, heads=8, head_dim=128)
    kv.kv_write(cache, k, v, slots)                     # k, v [T][8][128]; slots int64 [T] = page * page_size + offset
    out = kv.attention(q, cache, table, lens)           # q [B][32][128]; table int32 [B][pages]; lens int32 [B]
"""

import ctypes
import numbers
import struct

import torch

from . import _lib
from .host import FMT_ID, _need_cuda

# A decode step's attention runs a few microseconds on the GPU, so that what these functions cost on the host is what a
# caller waits for: they check in few steps, take the stream's handle without making a Stream object, and pack the
# arguments in one call (measured on one sequence of 4097 tokens: 26 us a call before that, 18 since).
_raw_stream = torch._C._cuda_getCurrentRawStream

FORMATS = ("q4_0", "q8_0")
HEAD_DIMS = (64, 96, 128, 256)
BLOCK_BYTES = {"q4_0": 16, "q8_0": 32}
DTYPE_ID = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}


def _fmt(fmt):
    if fmt not in FORMATS:
        raise ValueError(f"unknown cache format {fmt!r}: expected one of {FORMATS}")
    return fmt


class KVCache:
    """Planes of a paged cache: quants uint8 [pages][heads][page_size][row bytes] and scales int16 (f16 bits)
    [pages][heads][page_size][head_dim / 32], for keys (kq, ks) and values (vq, vs)."""

    def __init__(self, fmt, pages, page_size, heads, head_dim, device="cuda"):
        _fmt(fmt)
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"KVCache: head_dim {head_dim} not in {HEAD_DIMS}")
        nb = head_dim // 32
        shape = (pages, heads, page_size)
        planes = [torch.zeros((*shape, n), dtype=dt, device=device) for _ in "kv"
                  for n, dt in ((nb * BLOCK_BYTES[fmt], torch.uint8), (nb, torch.int16))]
        self._set(fmt, *planes)

    @classmethod
    def from_planes(cls, fmt, kq, ks, vq, vs):
        """A cache on planes that the caller owns (contiguous, 16-byte aligned)."""
        self = cls.__new__(cls)
        self._set(_fmt(fmt), kq, ks, vq, vs)
        return self

    def _set(self, fmt, kq, ks, vq, vs):
        dev = _need_cuda("KVCache", kq, ks, vq, vs)
        if ks.dim() != 4:
            raise ValueError(f"KVCache: scales must be [pages][heads][page_size][head_dim/32], got {tuple(ks.shape)}")
        nb = ks.shape[3]
        for t, name, dtype, last in ((kq, "kq", torch.uint8, nb * BLOCK_BYTES[fmt]), (ks, "ks", torch.int16, nb),
                                     (vq, "vq", torch.uint8, nb * BLOCK_BYTES[fmt]), (vs, "vs", torch.int16, nb)):
            if t.dtype != dtype:
                raise TypeError(f"KVCache: {name}: dtype {t.dtype}, expected {dtype}")
            if tuple(t.shape) != (*ks.shape[:3], last):
                raise ValueError(f"KVCache: {name}: shape {tuple(t.shape)}, expected {(*ks.shape[:3], last)}")
            if not t.is_contiguous() or t.data_ptr() % 16:
                raise ValueError(f"KVCache: {name} must be contiguous and 16-byte aligned")
        pages, heads, page = ks.shape[:3]
        if nb * 32 not in HEAD_DIMS:
            raise ValueError(f"KVCache: head_dim {nb * 32} not in {HEAD_DIMS}")
        if page < 16 or page > 65536 or page & (page - 1):
            raise ValueError(f"KVCache: page_size {page} is not a power of two from 16 to 65536")
        if heads < 1 or heads > 4096:
            raise ValueError(f"KVCache: {heads} heads (1..4096)")
        self.fmt, self.kq, self.ks, self.vq, self.vs = fmt, kq, ks, vq, vs
        self.pages, self.heads, self.page_size, self.head_dim, self.device = pages, heads, page, nb * 32, dev
        self._desc = _lib.KVCacheDesc(kq.data_ptr(), ks.data_ptr(), vq.data_ptr(), vs.data_ptr(), pages, heads, page,
                                      nb * 32, FMT_ID[fmt])
        self._ref = ctypes.addressof(self._desc)
        self._sizes = {}  # attention workspaces by shape

    @property
    def nbytes(self):
        return sum(t.numel() * t.element_size() for t in (self.kq, self.ks, self.vq, self.vs))


def _dtype_id(name, t):
    did = DTYPE_ID.get(t.dtype)
    if did is None:
        raise TypeError(f"{name}: dtype {t.dtype}, expected float32, float16 or bfloat16")
    return did


def _on_device(name, dev, *tensors):
    """Raises unless all are tensors on dev."""
    for t in tensors:
        if not isinstance(t, torch.Tensor) or t.device != dev:
            _need_cuda(name, t)
            raise RuntimeError(f"comp_b200.{name}: tensors on different devices ({dev} and {t.device})")


def _call(dev, name, *args):
    """_lib.call with dev the current device."""
    if torch.cuda.current_device() == dev.index:
        return _lib.call(name, *args)
    with torch.cuda.device(dev):
        return _lib.call(name, *args)


def _slots(name, slots):
    if slots.dtype != torch.int64 or slots.dim() != 1:
        raise TypeError(f"{name}: slots must be a 1-D int64 tensor, got {slots.dtype} {tuple(slots.shape)}")
    return slots if slots.is_contiguous() else slots.contiguous()


def _heads_aligned(t):
    """t with a contiguous last axis, a 16-byte aligned base and strides of whole 16 bytes (a copy only when needed)."""
    a, b, c = t.stride()
    mult = 16 // t.element_size()
    if c != 1 or a % mult or b % mult or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def kv_write(cache, k, v, slots):
    """Quantizes k and v [T][heads][head_dim] (f32, f16 or bf16; any token and head strides) into the slots int64 [T] of
    the cache (page * page_size + offset; no slot twice). Negative slots are skipped (padding tokens). The blocks are ggml's, bit for
    bit, of the value widened to f32; a 16-bit caller needs no cast."""
    dev = cache.device
    _on_device("kv_write", dev, k, v, slots)
    slots = _slots("kv_write", slots)
    shape = (slots.shape[0], cache.heads, cache.head_dim)
    did = _dtype_id("kv_write: k", k)
    if v.dtype != k.dtype:
        raise TypeError(f"kv_write: k is {k.dtype}, v is {v.dtype}")
    if k.shape != shape or v.shape != shape:
        raise ValueError(f"kv_write: k {tuple(k.shape)} and v {tuple(v.shape)}, expected {shape}")
    k, v = _heads_aligned(k), _heads_aligned(v)
    ks, vs = k.stride(), v.stride()
    _call(dev, "b2q_kv_write", cache._ref, did, k.data_ptr(), ks[0], ks[1], v.data_ptr(), vs[0], vs[1],
          slots.data_ptr(), shape[0], _raw_stream(dev.index))


def kv_read(cache, slots, dtype=torch.float32):
    """-> (k, v) [T][heads][head_dim] of `dtype`: the values that the slots int64 [T] hold (f16 scale times quant, rounded
    once). Negative slots give zeros."""
    dev = cache.device
    _on_device("kv_read", dev, slots)
    did = DTYPE_ID.get(dtype)
    if did is None:
        raise TypeError(f"kv_read: dtype {dtype}, expected float32, float16 or bfloat16")
    slots = _slots("kv_read", slots)
    n = slots.shape[0]
    k = slots.new_empty((n, cache.heads, cache.head_dim), dtype=dtype)
    v = torch.empty_like(k)
    _call(dev, "b2q_kv_read", cache._ref, did, k.data_ptr(), v.data_ptr(), slots.data_ptr(), n,
          _raw_stream(dev.index))
    return k, v


def _index(t, name, shape, dev, dtype=torch.int32):
    """The address of an index tensor (0: None), and the tensor that holds it."""
    if t is None:
        return 0, None
    _on_device("attention", dev, t)
    if t.dtype != dtype:
        raise TypeError(f"attention: {name}: dtype {t.dtype}, expected {dtype}")
    if t.shape != shape:
        raise ValueError(f"attention: {name}: shape {tuple(t.shape)}, expected {shape}")
    if not t.is_contiguous():
        t = t.contiguous()
    return t.data_ptr(), t


_pack_args = struct.Struct("@9P8q3i2f").pack  # b2q_attention_args, field by field
assert struct.calcsize("@9P8q3i2f") <= ctypes.sizeof(_lib.AttentionArgs)


def attention_workspace_size(cache, T, batch, q_heads, dtype, max_q=1, return_lse=False):
    """Bytes of device workspace that attention needs for such a call (max_q as there: 1 without cu_q)."""
    if dtype not in DTYPE_ID:
        raise TypeError(f"attention_workspace_size: dtype {dtype}, expected float32, float16 or bfloat16")
    key = (T > 0 and batch > 0, q_heads, dtype, max_q if max_q and max_q < T else T, return_lse)
    size = cache._sizes.get(key)
    if size is None:
        one = 256  # any address: the plan looks at sizes and at whether lse and cu_q are given
        args = _lib.AttentionArgs(one, one, one if return_lse else None, one, one, one, None, None, None,
                                  cache.head_dim * q_heads, cache.head_dim, T, batch, 1, 1, max_q or 0, 0, q_heads,
                                  DTYPE_ID[dtype], 0, 1.0, 0.0)
        with torch.cuda.device(cache.device):
            size = _lib.load().b2q_attention_workspace_size(cache._ref, ctypes.addressof(args))
        if len(cache._sizes) >= 4096:  # every T of a long-lived server would stay
            cache._sizes.clear()
        cache._sizes[key] = size
    return size


def attention(q, cache, table, lens, scale=None, *, cu_q=None, max_q=None, max_len=None, softcap=0.0, window=0,
              slopes=None, prefix=None, starts=None, out=None, return_lse=False, workspace=None):
    """Attention of query tokens q [T][q_heads][head_dim] (f32, f16 or bf16) over the cache -> out of the same shape and
    type (and lse f32 [T][q_heads] when return_lse).

    table: int32 [B][P], the pages of each sequence; lens: int32 [B], its tokens in the cache, the query tokens' own
    among them. cu_q: int32 [B + 1], where each sequence's query tokens begin in q (default: one token each, T == B); the
    last one is at position lens - 1. q head h reads KV head h // (q_heads // heads). scale: default head_dim ** -0.5.

    softcap > 0: scores s -> softcap * tanh(s / softcap); slopes f32 [q_heads]: minus slopes[h] times the distance of
    query and key. A query at p sees the keys max(starts, p - window + 1) <= j < min(lens, max(p + 1, prefix)): window
    (0: none) slides, prefix int32 [B] keys are seen by the queries before them too (where their window and document reach
    back so far), starts int32 [T] is the first key of a query's document. A query that sees no key gives zeros (lse -inf).

    max_q / max_len: the most query tokens of a sequence and the longest length, where the caller knows them (default:
    T, or 1 without cu_q, and what the table can hold): max_q must not be less than what cu_q has (rows past it
    stay unwritten and set the device error word to 4), max_len only plans the work. workspace: a CUDA byte tensor of
    attention_workspace_size(...) bytes (allocated here when None). out: a contiguous tensor for the result that shares no
    memory with q. Rows outside cu_q's range (padding) stay unwritten."""
    dev = cache.device
    _on_device("attention", dev, q, table, lens)
    did = _dtype_id("attention: q", q)
    if q.dim() != 3 or q.shape[2] != cache.head_dim:
        raise ValueError(f"attention: q {tuple(q.shape)}, expected [T][q_heads][{cache.head_dim}]")
    T, heads, dim = q.shape
    if heads == 0 or heads % cache.heads:
        raise ValueError(f"attention: {heads} query heads over {cache.heads} KV heads")
    if table.dtype != torch.int32 or table.dim() != 2:
        raise TypeError(f"attention: table must be a 2-D int32 tensor, got {table.dtype} {tuple(table.shape)}")
    B, P = table.shape
    if B > 1 and (table.stride(1) != 1 or table.stride(0) < P) or P > 1 and table.stride(1) != 1:
        table = table.clone(memory_format=torch.contiguous_format)  # one row for all sequences, rows that overlap
    lens_at, lens = _index(lens, "lens", (B,), dev)
    if cu_q is None:
        if T != B:
            raise ValueError(f"attention: {T} query tokens for {B} sequences need cu_q")
        max_q = 1
    elif max_q is None:
        max_q = T
    cu_at, cu_q = _index(cu_q, "cu_q", (B + 1,), dev)
    prefix_at, prefix = _index(prefix, "prefix", (B,), dev)
    starts_at, starts = _index(starts, "starts", (T,), dev)
    slopes_at, slopes = _index(slopes, "slopes", (heads,), dev, torch.float32)
    q = _heads_aligned(q)
    if out is None:
        out = q.new_empty((T, heads, dim))
    elif out.dtype != q.dtype or out.shape != q.shape or out.device != dev or not out.is_contiguous():
        raise ValueError(f"attention: out must be a contiguous {q.dtype} {tuple(q.shape)} tensor on {dev}")
    lse = q.new_empty((T, heads), dtype=torch.float32) if return_lse else None
    if workspace is None:
        workspace = lens.new_empty(attention_workspace_size(cache, T, B, heads, q.dtype, max_q, return_lse) + 3 >> 2)
    else:
        _on_device("attention", dev, workspace)
        if not workspace.is_contiguous():
            raise ValueError("attention: workspace must be contiguous")
    q_st, q_sh, _ = q.stride()
    try:
        args = _pack_args(q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, table.data_ptr(), lens_at,
                          cu_at, prefix_at, starts_at, slopes_at, q_st, q_sh, T, B, table.stride(0) if B > 1 else P, P, max_q,
                          P * cache.page_size if max_len is None else max_len, heads, did, window,
                          dim**-0.5 if scale is None else scale, softcap)
    except (struct.error, OverflowError) as e:
        kinds = ((numbers.Integral, (max_q, window, 0 if max_len is None else max_len)),
                 (numbers.Real, (softcap, 1.0 if scale is None else scale)))
        if all(isinstance(x, kind) for kind, given in kinds for x in given):
            raise ValueError(f"attention: max_q, max_len, window, scale or softcap out of range: {e}") from None
        raise TypeError(f"attention: max_q, max_len and window are whole numbers, scale and softcap numbers: {e}") from None
    _call(dev, "b2q_attention", cache._ref, args, workspace.data_ptr(), workspace.numel() * workspace.element_size(),
          _raw_stream(dev.index))
    return (out, lse) if return_lse else out
