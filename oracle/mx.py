"""MXFP4 and layers of experts, restated in numpy and 64 bits: quantization by its definition, planes, products, routing, the
sort by expert and the way back: what the tests of comp_b200.mx and comp_b200.experts compare with."""

import numpy as np

LEVELS = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x):
    """f32 values [..., K] -> (codes uint8 [..., K/2], scales uint8 [..., K/32])."""
    x = np.asarray(x, dtype=np.float32)
    b = x.astype(np.float64).reshape(*x.shape[:-1], -1, 32)
    good = np.isfinite(b).all(-1)
    b = np.where(good[..., None], b, 0.0)
    amax = np.abs(b).max(-1)
    _, ex = np.frexp(amax)  # amax = m * 2^ex, 0.5 <= m < 1
    s = np.where(amax > 0, np.maximum(ex - 3 + 127, 0), 0)
    a = np.abs(b) * np.exp2(127.0 - s)[..., None]
    d = np.abs(a[..., None] - LEVELS)  # the nearest level; of two at the same distance the one with the even code
    best = d.min(-1, keepdims=True)
    even = np.where(np.arange(8) % 2 == 0, 0, 1)
    code = np.argmin(np.where(d == best, even, 2), axis=-1).astype(np.uint8)
    sign = np.signbit(x.reshape(b.shape)) & good[..., None]
    code |= sign.astype(np.uint8) << 3
    codes = (code[..., :16] | (code[..., 16:] << 4)).reshape(*x.shape[:-1], -1)
    return codes, np.where(good, s, 255).astype(np.uint8)


def values(codes, scales):
    """The values of planes, f64 [..., K]."""
    raw = codes.reshape(*scales.shape, 16)
    code = np.concatenate([raw & 15, raw >> 4], -1)
    v = np.where(code & 8, -1.0, 1.0) * LEVELS[code & 7]
    d = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v * d[..., None]).reshape(*scales.shape[:-1], -1)


def image(codes, scales):
    """Planes [rows][..] -> the operand image's bytes (rows and stages beyond the end are zeros)."""
    rows, nb = scales.shape
    tiles, stages = -(-rows // 128), -(-nb // 8)
    out = np.zeros((tiles, stages, 17408), dtype=np.uint8)
    for r in range(rows):
        for b in range(nb):
            run = out[r // 128, b // 8]
            i, j = r % 128, b % 8
            at = i * 128 + (j ^ (i % 8)) * 16
            run[at : at + 16] = codes[r, b * 16 : b * 16 + 16]
            run[16384 + j // 4 * 512 + i % 32 * 16 + i // 32 * 4 + j % 4] = scales[r, b]
    return out.reshape(-1)


def route(logits, top, normalize=True):
    """-> (ids, weights): the largest logits, the lowest index first among equals; -inf and NaN never."""
    x = np.asarray(logits, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    ids = np.argsort(-x, axis=1, kind="stable")[:, :top]
    v = np.take_along_axis(x, ids, 1)
    largest = v[:, :1]

    def e(y):
        with np.errstate(invalid="ignore"):
            return np.where(y == -np.inf, 0.0, np.where(y == largest, 1.0, np.exp(y - largest)))

    total = e(v).sum(1, keepdims=True) if normalize else e(x).sum(1, keepdims=True)
    some = v > -np.inf
    return np.where(some, ids, -1), np.where(some, e(v) / np.where(total > 0, total, 1.0), 0.0)


def sort(ids, experts):
    """-> (offsets, pos, order) of choices sorted by expert, stable; ids outside the experts go nowhere."""
    flat = np.asarray(ids).ravel()
    key = np.where((flat >= 0) & (flat < experts), flat, experts)
    order = np.argsort(key, kind="stable")
    offsets = np.searchsorted(key[order], np.arange(experts + 1))
    pos = np.empty(flat.size, dtype=np.int64)
    pos[order] = np.arange(flat.size)
    return (offsets, np.where(key < experts, pos, -1).reshape(np.shape(ids)),
            np.where(np.arange(flat.size) < offsets[-1], order, -1))


def experts_linear(x, w, offsets, order, top, gather=True):
    """x f64 rows (already rounded to MXFP4), w f64 [E][N][K] -> (y [choices][N], mass): mass = sum of |products|."""
    y = np.full((order.size, w.shape[1]), np.nan)
    mass = np.zeros_like(y)
    for e in range(w.shape[0]):
        rows = np.arange(offsets[e], offsets[e + 1])
        src = x[order[rows] // top if gather else rows]
        y[rows], mass[rows] = src @ w[e].T, np.abs(src) @ np.abs(w[e]).T
    return y, mass


def combine(y, pos, weights=None):
    """-> (out f64 [tokens][N], mass)."""
    w = np.ones(pos.shape) if weights is None else np.asarray(weights, dtype=np.float64)
    rows = np.where((pos >= 0)[..., None], y[np.maximum(pos, 0)], 0.0)
    return (w[..., None] * rows).sum(1), (np.abs(w)[..., None] * np.abs(rows)).sum(1)
