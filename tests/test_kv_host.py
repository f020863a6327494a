"""The quantized KV cache without a GPU: the C-ABI's refusals (checked before any launch), the binding's structures, the
oracle's layout against a second statement of it, and the oracle's quantizer against the existing one."""

import ctypes

import numpy as np
import pytest
import torch

from comp_b200 import _lib, kv
from oracle import kv as ref
from oracle import ref as gref


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def _desc(**kw):
    a = dict(kq=4096, ks=4096, vq=4096, vs=4096, pages=4, heads=2, page=16, dim=64, fmt=0) | kw
    return _lib.KVCacheDesc(*a.values())


def _args(**kw):
    a = dict(q=4096, out=4096, lse=None, table=4096, lens=4096, cu_q=None, prefix=None, starts=None, slopes=None, q_st=256,
             q_sh=64, T=2, batch=2, table_stride=3, table_pages=3, max_q=1, max_len=48, q_heads=4, dtype=0, window=0,
             scale=0.125, softcap=0.0) | kw
    return _lib.AttentionArgs(*a.values())


def test_structures_match_the_header():
    assert ctypes.sizeof(_lib.KVCacheDesc) == 56 and ctypes.sizeof(_lib.AttentionArgs) == 160
    a = _args(window=7, softcap=2.5, T=9, q_st=77)
    packed = kv._pack_args(4096, 4096, 0, 4096, 4096, 0, 0, 0, 0, 77, 64, 9, 2, 3, 3, 1, 48, 4, 0, 7, 0.125, 2.5)
    assert bytes(a)[: len(packed)] == packed


@pytest.mark.parametrize("bad,code", [(dict(fmt=1), -1), (dict(dim=80), -1), (dict(page=24), -1), (dict(page=8), -1),
                                      (dict(heads=0), -1), (dict(pages=-1), -1), (dict(kq=None), -1), (dict(vs=8), -2)])
def test_cache_refusals(lib, bad, code):
    d = _desc(**bad)
    assert lib.b2q_kv_write(ctypes.addressof(d), 0, 4096, 64, 64, 4096, 64, 64, 4096, 1, None) == code
    assert lib.b2q_kv_read(ctypes.addressof(d), 0, 4096, 4096, 4096, 1, None) == code
    a = _args()
    assert lib.b2q_attention(ctypes.addressof(d), ctypes.addressof(a), 4096, 1 << 30, None) == code
    assert lib.b2q_attention_workspace_size(ctypes.addressof(d), ctypes.addressof(a)) == 0
    assert "b2q_attention" in _lib.last_error()


def test_write_and_read_refusals(lib):
    d = ctypes.addressof(_desc_keep := _desc())
    w = lambda dtype=0, k=4096, st=64, sh=64, slots=4096, T=1: lib.b2q_kv_write(d, dtype, k, st, sh, 4096, 64, 64, slots, T, None)  # noqa: E731
    assert w(dtype=3) == -1 and w(k=None) == -1 and w(slots=None) == -1 and w(T=-1) == -1
    assert w(k=4100) == -2 and w(st=66) == -2 and w(dtype=1, sh=4) == -2 and w(slots=4100) == -2
    assert w(T=0) == 0 and w(T=1 << 40) == -4
    r = lambda dtype=0, k=4096, slots=4096, T=1: lib.b2q_kv_read(d, dtype, k, 4096, slots, T, None)  # noqa: E731
    assert r(dtype=-1) == -1 and r(slots=None) == -1 and r(k=4100) == -2 and r(T=0) == 0
    assert lib.b2q_kv_read(d, 0, None, None, 4096, 1, None) == 0
    assert lib.b2q_kv_write(None, 0, 4096, 64, 64, 4096, 64, 64, 4096, 1, None) == -1
    assert _desc_keep.dim == 64


@pytest.mark.parametrize("bad,code", [(dict(q_heads=3), -1), (dict(q_heads=0), -1), (dict(dtype=3), -1),
                                      (dict(scale=0.0), -1), (dict(scale=float("nan")), -1), (dict(softcap=-1.0), -1),
                                      (dict(window=-1), -1), (dict(T=3), -1), (dict(T=-1), -1), (dict(q=None), -1),
                                      (dict(out=None), -1), (dict(lens=None), -1), (dict(table=None), -1),
                                      (dict(table_stride=2), -1), (dict(q=4100), -2), (dict(q_st=65), -2),
                                      (dict(table_pages=1 << 40, table_stride=1 << 40), -4),
                                      (dict(T=1 << 31, batch=1 << 31), -4)])
def test_attention_refusals(lib, bad, code):
    d, a = _desc(), _args(**bad)
    assert lib.b2q_attention(ctypes.addressof(d), ctypes.addressof(a), 4096, 1 << 40, None) == code


def test_attention_workspace(lib):
    d, a = _desc(), _args()
    need = lib.b2q_attention_workspace_size(ctypes.addressof(d), ctypes.addressof(a))
    assert need > 0
    assert lib.b2q_attention(ctypes.addressof(d), ctypes.addressof(a), 4096, need - 1, None) == -1
    assert lib.b2q_attention(ctypes.addressof(d), ctypes.addressof(a), None, need, None) == -1
    assert lib.b2q_attention(ctypes.addressof(d), ctypes.addressof(a), 4100, need, None) == -1
    e = _args(T=0, batch=0)
    assert lib.b2q_attention(ctypes.addressof(d), ctypes.addressof(e), None, 0, None) == 0


def test_no_cpu_path():
    with pytest.raises(RuntimeError):
        kv.KVCache("q4_0", 2, 16, 2, 64, device="cpu")
    with pytest.raises(ValueError):
        kv.KVCache("tq2_0", 2, 16, 2, 64, device="cpu")
    assert torch.float16 in kv.DTYPE_ID


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("which", ["k", "v"])
def test_layout(fmt, dim, which):
    """The rows as [blocks][U][unit] stored as [U][blocks][unit], and back to the values."""
    x = np.random.default_rng(dim).standard_normal((7, dim)).astype(np.float32)
    rows, scales = ref.pack(fmt, x, which)
    q, s = ref.quantize(fmt, x)
    assert np.array_equal(scales, s)
    b = q.reshape(7, dim // 32, 32)
    raw = b[..., :16] | b[..., 16:] << 4 if fmt == "q4_0" else b
    u = ref.UNITS[which]
    assert np.array_equal(rows, raw.reshape(7, dim // 32, u, -1).transpose(0, 2, 1, 3).reshape(7, -1))
    v = ref.unpack(fmt, rows, scales, which)
    d = np.repeat(s.view(np.float16).astype(np.float64), 32, axis=-1)
    assert np.array_equal(v, (q.astype(np.float64) - (8 if fmt == "q4_0" else 128)) * d)


def test_q8_0_quants_are_the_activation_quantizers():
    x = np.random.default_rng(3).standard_normal((5, 128)).astype(np.float32)
    q, s = ref.quantize("q8_0", x)
    xq, xd = gref.quant_q8_0(x)
    assert np.array_equal(q.astype(np.int32) - 128, xq.astype(np.int32))
    assert np.array_equal(s.view(np.float16).astype(np.float32), xd)


def test_oracle_attention_masks():
    see = ref.visible([5, 3], np.array([0, 2, 3]), prefix=[0, 2], starts=[0, 4, 1], window=2)
    assert see == [(3, 2, 4), (4, 4, 5), (2, 1, 3)]
    k = [np.ones((3, 1, 32))]
    v = [np.arange(3.0)[:, None, None] * np.ones((3, 1, 32))]
    o, l, _, _ = ref.attention(np.zeros((1, 1, 32)), k, v, [3], np.array([0, 1]), 1.0)
    assert np.allclose(o, 1.0) and np.allclose(l, np.log(3))


def test_quantize_is_ggmls_loop():
    """ggml's q4_0 block as its steps are: the maximum begins at +0 and takes a value of larger magnitude only."""
    f = np.float32
    x = np.random.default_rng(4).standard_normal((9, 32)).astype(f)
    x[0], x[1] = 0.0, -0.0
    x[2, ::3], x[3] = -0.0, np.where(np.arange(32) % 2, f(-0.0), f(0.0))
    x[4, 7], x[4, 9], x[5, 7], x[5, 9] = 9.0, -9.0, -9.0, 9.0
    q, s = ref.quantize("q4_0", x)
    for row, quants, bits in zip(x, q, s[:, 0]):
        top, at = f(0), f(0)
        for v in row:
            if top < abs(v):
                top, at = abs(v), v
        d = at / f(-8)
        inv = f(1) / d if d else f(0)
        assert bits == np.float16(d).view(np.uint16)
        assert np.array_equal(quants, [min(15, int(v * inv + f(8.5))) for v in row])
