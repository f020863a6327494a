"""MXFP4 and layers of experts without a GPU: the C-ABI's refusals (checked before any launch) and the oracle against second
statements of its parts."""

import struct

import numpy as np
import pytest
import torch

from comp_b200 import _lib, experts, mx
from oracle import mx as ref


def pack(form, *values):
    return struct.pack(form, *(0 if v is None else v for v in values))


@pytest.fixture(scope="module")
def lib():
    return _lib.load()


def test_sizes(lib):
    assert lib.b2q_mx_bytes(1, 1, 32) == 17408 and lib.b2q_mx_bytes(3, 129, 288) == 3 * 2 * 2 * 17408
    assert lib.b2q_mx_bytes(1, 0, 32) == 0
    for bad in ((0, 1, 32), (1025, 1, 32), (1, -1, 32), (1, 1, 0), (1, 1, 33), (1, 1 << 31, 32)):
        assert lib.b2q_mx_bytes(*bad) == 0 and "b2q_mx_bytes" in _lib.last_error()
    for e, rows, k in ((1, 1, 32), (7, 300, 4096), (2, 128, 256)):
        assert lib.b2q_mx_bytes(e, rows, k) == mx.image_bytes(rows, k, e)
    assert lib.b2q_mx_linear_workspace_size(17, 300, 288) == 2 * 17408 and lib.b2q_mx_linear_workspace_size(1, 1, 20) == 0
    for t, top, e, k in ((17, 1, 1, 32), (64, 8, 128, 4096), (1000, 3, 9, 288), (50, 1, 1000, 64)):
        size = lib.b2q_experts_linear_workspace_size(t, top, e, 1, 64, k)
        # the most tiles that sorted rows can take
        counts = np.zeros(e, dtype=np.int64)
        n = t * top
        counts[: min(e, n)] = 1
        counts[0] += n - counts.sum()
        assert (-(-counts // 128)).sum() * -(-k // 256) * 17408 <= size


def test_plan_words(lib):
    for t, top, e in ((0, 1, 1), (1, 8, 64), (128, 8, 1024), (128, 9, 64), (1, 32, 1024), (129, 1, 5), (4097, 1, 5), (16384, 8, 256), (1 << 23, 8, 1024)):
        words = lib.b2q_experts_plan_words(t, top, e)
        plain = 2 * (e + 1) + 4 * t * top
        assert words == plain if t <= 128 and t * top <= 1024 else words > plain and (words - plain) % e == 0
    for bad in ((-1, 1, 1), (1, 0, 1), (1, 33, 64), (1, 1, 0), (1, 1, 1025), (1 << 26, 2, 4)):
        assert lib.b2q_experts_plan_words(*bad) == 0 and "b2q_experts_plan_words" in _lib.last_error()


def test_quantize_refusals(lib):
    q = lambda dtype=0, x=4096, ldx=64, rows=2, k=64, image=4096, e=1: lib.b2q_mx_quantize(dtype, x, ldx, e, rows, k, image, None)  # noqa: E731
    assert q(dtype=3) == -1 and q(x=None) == -1 and q(image=None) == -1 and q(rows=-1) == -1 and q(k=48) == -1 and q(ldx=32) == -1
    assert q(e=0) == -1 and q(e=1025) == -1 and q(e=2, rows=1, ldx=32) == -1
    assert q(x=4100) == -2 and q(ldx=66) == -2 and q(image=4096 + 64) == -2 and q(dtype=1, ldx=68) == -2
    assert q(rows=0, x=None, image=None) == 0
    d = lambda image=4096, rows=2, k=64, dtype=0, y=4096, ldy=64, e=1: lib.b2q_mx_dequantize(image, e, rows, k, dtype, y, ldy, None)  # noqa: E731
    assert d(image=None) == -1 and d(y=None) == -1 and d(dtype=-1) == -1 and d(k=0) == -1 and d(ldy=63) == -1
    assert d(y=4104) == -2 and d(ldy=65) == -2 and d(rows=0) == 0 and d(e=0) == -1
    p = lambda codes=4096, scales=4096, e=1, rows=2, k=64, image=4096: lib.b2q_mx_pack(codes, scales, e, rows, k, image, None)  # noqa: E731
    assert p(codes=None) == -1 and p(scales=None) == -1 and p(image=None) == -1 and p(e=0) == -1 and p(e=1025) == -1 and p(k=20) == -1
    assert p(codes=4100) == -2 and p(image=64) == -2 and p(rows=0) == 0


def test_product_refusals(lib):
    f = lambda a=4096, w=4096, m=2, n=3, k=64, dtype=0, y=4096, ldy=3: lib.b2q_mx_matmul(a, w, m, n, k, dtype, y, ldy, None)  # noqa: E731
    assert f(a=None) == -1 and f(w=None) == -1 and f(y=None) == -1 and f(m=-1) == -1 and f(n=-1) == -1 and f(k=16) == -1
    assert f(dtype=4) == -1 and f(ldy=2) == -1 and f(a=64) == -2 and f(w=64) == -2 and f(y=4098) == -2
    assert f(m=0) == 0 and f(n=0) == 0
    g = lambda x=4096, ldx=64, w=4096, y=4096, ws=4096, size=17408, m=20, dtype=2: lib.b2q_mx_linear(  # noqa: E731
        pack(_lib.MX_LINEAR_ARGS, x, w, y, ws, ldx, m, 3, 64, 3, size, 0, dtype), None)
    assert lib.b2q_mx_linear(None, None) == -1
    assert g(x=None) == -1 and g(w=None) == -1 and g(y=None) == -1 and g(ws=None) == -1 and g(size=17407) == -1 and g(dtype=9) == -1
    assert g(x=4100) == -2 and g(ldx=65) == -2 and g(ws=4096 + 16) == -1 and g(m=0, ws=None) == 0


def test_expert_refusals(lib):
    r = lambda dtype=0, x=4096, ld=8, t=2, e=8, top=2, ids=4096, w=4096, plan=4096: lib.b2q_experts_route(  # noqa: E731
        pack(_lib.EXPERTS_ROUTE_ARGS, x, ids, w, plan, ld, t, e, top, dtype, 1), None)
    assert r(dtype=5) == -1 and r(x=None) == -1 and r(ld=7) == -1 and r(t=-1) == -1 and r(e=0) == -1 and r(e=1025, ld=2000) == -1
    assert r(top=0) == -1 and r(top=9) == -1 and r(top=33, e=64, ld=64) == -1 and r(ids=None) == -1 and r(w=None) == -1
    assert r(plan=None) == -1 and r(plan=4098) == -2 and r(ids=4097) == -2 and r(x=4097) == -2 and r(t=1 << 26) == -4
    s = lambda ids=4096, t=2, top=2, e=8, plan=4096: lib.b2q_experts_sort(ids, t, top, e, plan, None)  # noqa: E731
    assert s(ids=None) == -1 and s(plan=None) == -1 and s(e=0) == -1 and s(top=33) == -1 and s(ids=4098) == -2
    f = lambda x=4096, ldx=64, w=4096, plan=4096, t=20, n=3, k=64, dtype=0, y=4096, ldy=3, ws=4096, size=1 << 20: (  # noqa: E731
        lib.b2q_experts_linear(pack(_lib.EXPERTS_LINEAR_ARGS, x, w, plan, y, ws, ldx, t, 2, 8, n, k, ldy, size, 0, dtype, 1), None))
    assert f(x=None) == -1 and f(w=None) == -1 and f(plan=None) == -1 and f(y=None) == -1 and f(ws=None) == -1 and f(k=40) == -1
    assert f(dtype=3) == -1 and f(ldy=2) == -1 and f(size=17408) == -1 and f(x=4104) == -2 and f(w=4096 + 64) == -2 and f(y=4098) == -2
    assert f(t=0, ws=None) == 0 and f(n=0) == 0
    c = lambda dtype=0, y=4096, ldy=4, plan=4096, w=4096, n=4, out=4096, ldo=4: lib.b2q_experts_combine(  # noqa: E731
        pack(_lib.EXPERTS_COMBINE_ARGS, y, plan, w, out, ldy, 2, 2, 8, n, ldo, dtype), None)
    assert all(f(None, None) == -1 for f in (lib.b2q_experts_route, lib.b2q_experts_linear, lib.b2q_experts_combine))
    assert c(dtype=3) == -1 and c(y=None) == -1 and c(out=None) == -1 and c(plan=None) == -1 and c(ldy=3) == -1 and c(ldo=3) == -1
    assert c(n=-1) == -1 and c(y=4098) == -2 and c(w=4098) == -2 and c(n=0) == 0


def test_python_refuses_cpu_tensors():
    x = torch.zeros((2, 64))
    for call in (lambda: mx.quantize(x), lambda: mx.pack(x.byte(), x.byte()), lambda: mx.from_ggml(x.byte(), 1, 32),
                 lambda: mx.MXTensor(torch.zeros(17408, dtype=torch.uint8), 1, 32), lambda: experts.route(x, 1),
                 lambda: experts.sort(x.int(), 3)):
        with pytest.raises(RuntimeError):
            call()


def test_oracle_rounding():
    """Every magnitude in a fine grid against the midpoints, ties to the even code."""
    a = np.arange(0, 8, 1 / 64)
    x = np.concatenate([a, -a, np.zeros((-2 * a.size) % 31)]).reshape(-1, 31).astype(np.float32)
    x = np.concatenate([x, np.full((x.shape[0], 1), 7.5, dtype=np.float32)], 1)  # the block's scale is 1
    codes, scales = ref.quantize(x)
    assert (scales == 127).all()
    mids = [(0.25, 0), (0.75, 2), (1.25, 2), (1.75, 4), (2.5, 4), (3.5, 6), (5.0, 6)]
    got = ref.values(codes, scales)
    for v, g in zip(x.ravel(), got.ravel()):
        level = sum(abs(v) > m or (abs(v) == m and tie == i + 1) for i, (m, tie) in enumerate(mids))
        assert abs(g) == ref.LEVELS[level] and (g == 0 or (g < 0) == (v < 0))


def test_oracle_scales():
    x = np.zeros((6, 32), dtype=np.float32)
    x[1, 3], x[2, 0], x[3, 9], x[4, 1], x[5, 2] = 1.0, -3.4e38, 1e-45, np.inf, 2.0**-125
    _, s = ref.quantize(x)
    assert s.ravel().tolist() == [0, 125, 252, 0, 255, 0]


def test_oracle_plan():
    rng = np.random.default_rng(0)
    ids = rng.integers(-1, 5, (30, 3))
    offsets, pos, order = ref.sort(ids, 5)
    flat = ids.ravel()
    rows = [i for e in range(5) for i in range(90) if flat[i] == e]
    assert order[: len(rows)].tolist() == rows and (order[len(rows) :] == -1).all() and offsets[-1] == len(rows)
    assert all(pos.ravel()[c] == i for i, c in enumerate(rows)) and ((pos.ravel() == -1) == (flat == -1)).all()
    assert [offsets[e + 1] - offsets[e] for e in range(5)] == [(flat == e).sum() for e in range(5)]


def test_image_layout():
    """The place of a code's byte and of a scale, by hand."""
    rng = np.random.default_rng(1)
    codes, scales = ref.quantize(rng.standard_normal((130, 544)).astype(np.float32))
    im = ref.image(codes, scales).reshape(2, 3, 17408)
    for r, b, i in ((0, 0, 0), (5, 9, 3), (129, 16, 15), (127, 7, 8), (33, 14, 1)):
        assert im[r // 128, b // 8, (r % 128) * 128 + 16 * ((b % 8) ^ (r % 8)) + i] == codes[r, 16 * b + i]
        at = 16384 + (b % 8 // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 + b % 4
        assert im[r // 128, b // 8, at] == scales[r, b]
    assert not im[1, :, 2 * 128 : 16384].any() and not im[:, 2, 16384 + 512 :].any()
