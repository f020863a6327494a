"""Plain restatement of the quantized KV cache and its attention (numpy, 64 bits), the oracle of comp_b200.kv.

The cache's layout is stated here element by element, apart from the kernels: element e of a head's row lies in block
b = e // 32 at i = e % 32; its ggml quant byte (q4_0: byte i % 16, low nibble for i < 16; q8_0: byte i, the quant plus
128) lies at byte ((byte // unit) * blocks + b) * unit + byte % unit of the row, unit = bytes of a block / U, with U = 4
for keys and 8 for values.
"""

import numpy as np

BLOCK_BYTES = {"q4_0": 16, "q8_0": 32}
UNITS = {"k": 4, "v": 8}


def _places(fmt, dim, which):
    """(byte within the row, shift) of each element."""
    e = np.arange(dim)
    nb = dim // 32
    b, i = e // 32, e % 32
    byte = i % 16 if fmt == "q4_0" else i
    unit = BLOCK_BYTES[fmt] // UNITS[which]
    return ((byte // unit) * nb + b) * unit + byte % unit, (4 * (i // 16) if fmt == "q4_0" else 0 * i)


def quantize(fmt, x):
    """ggml's blocks of f32 [..., dim]: (quants uint8 as stored, one per element, f16 scale bits uint16 [..., dim/32])."""
    f = np.float32
    b = np.asarray(x, f).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if fmt == "q4_0":
            first = np.abs(b).argmax(-1)[..., None]
            d = (np.take_along_axis(b, first, -1) + f(0)) / f(-8)  # the maximum begins at +0: zeros have the scale -0
        else:
            d = np.abs(b).max(-1, keepdims=True) / f(127)
        inv = np.divide(f(1), d, out=np.zeros_like(d), where=d != 0)
        y = b * inv
        if fmt == "q4_0":
            q = np.minimum(15, (y + f(8.5)).astype(np.int32))
        else:
            whole = np.trunc(y)
            q = (whole + np.where(np.abs(y - whole) >= f(0.5), np.sign(y), f(0))).astype(np.int32) + 128
    return q.astype(np.uint8).reshape(x.shape), d[..., 0].astype(np.float16).view(np.uint16)


def pack(fmt, x, which):
    """f32 [..., dim] -> (row bytes uint8 [..., row], scale bits uint16 [..., dim/32]) in the cache's layout."""
    q, s = quantize(fmt, x)
    place, shift = _places(fmt, x.shape[-1], which)
    row = np.zeros((*x.shape[:-1], x.shape[-1] // 32 * BLOCK_BYTES[fmt]), np.uint8)
    for e in range(x.shape[-1]):
        row[..., place[e]] |= q[..., e] << np.uint8(shift[e])
    return row, s


def unpack(fmt, rows, scales, which):
    """Row bytes and scale bits -> values in 64 bits."""
    dim = scales.shape[-1] * 32
    place, shift = _places(fmt, dim, which)
    q = rows[..., place].astype(np.int32)
    q = ((q >> shift) & 15) - 8 if fmt == "q4_0" else q - 128
    d = scales.view(np.float16).astype(np.float64)
    with np.errstate(invalid="ignore"):
        return q * np.repeat(d, 32, axis=-1)


def visible(lens, cu, prefix=None, starts=None, window=0):
    """Per query token (position, first visible key, end of the visible keys)."""
    out = []
    for b, n in enumerate(np.diff(cu)):
        for i in range(n):
            p = int(lens[b]) - int(n) + i
            hi = min(int(lens[b]), max(p + 1, int(prefix[b]) if prefix is not None else 0))
            lo = max(0, int(starts[cu[b] + i]) if starts is not None else 0)
            if window:
                lo = max(lo, p - window + 1)
            out.append((p, lo, max(lo, hi)))
    return out


def attention(q, keys, values, lens, cu, scale, softcap=0.0, slopes=None, prefix=None, starts=None, window=0,
              unread=None):
    """-> (out [T][q_heads][dim], lse [T][q_heads], reach [T][q_heads], mass [T][q_heads][dim]), all f64. keys / values:
    per sequence [len][heads][dim]; unread: per sequence bool [len], tokens that are masked for every query. reach is the
    largest scale * sum |q_i k_i| of a visible key and mass the attention of |v|: what a rounding of a score or a weight can
    move an output by is measured in them."""
    T, qh, dim = q.shape
    out, lse = np.zeros((T, qh, dim)), np.full((T, qh), -np.inf)
    reach, mass = np.zeros((T, qh)), np.zeros((T, qh, dim))
    see = visible(lens, cu, prefix, starts, window)
    for b in range(len(lens)):
        for t in range(int(cu[b]), int(cu[b + 1])):
            p, lo, hi = see[t]
            if lo >= hi:
                continue
            j = np.arange(lo, hi)
            if unread is not None:
                j = j[~unread[b][lo:hi]]
            if not len(j):
                continue
            k, v = keys[b][j], values[b][j]
            group = qh // k.shape[1]
            for h in range(qh):
                kh, vh, qt = k[:, h // group], v[:, h // group], q[t, h].astype(np.float64)
                s = scale * (kh @ qt)
                if softcap:
                    s = softcap * np.tanh(s / softcap)
                if slopes is not None:
                    s = s - float(slopes[h]) * np.abs(p - j)
                top = s.max()
                w = np.exp(s - top)
                total = w.sum()
                out[t, h], lse[t, h] = (w @ vh) / total, top + np.log(total)
                mass[t, h] = (w @ np.abs(vh)) / total
                reach[t, h] = scale * (np.abs(kh) @ np.abs(qt)).max()
    return out, lse, reach, mass
