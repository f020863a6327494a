"""comp_b200.kv where its inputs reach a limit: pages that cannot be read, tables shorter than their sequences, values past
f16's range, scales and caps at the ends of their ranges, long tails of small weights, rows on either side of the kernels'
boundary, calls on streams that overlap. Against the 64-bit restatement (oracle.kv), with the bounds of test_gpu_kv."""

import numpy as np
import pytest
import torch

from comp_b200 import kv
from oracle import kv as ref

from .test_gpu_kv import DT, U, _bounds, _cache, _device_error, _gather, _problem

pytestmark = pytest.mark.gpu


def _to(dev, *arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev) for a in arrays]


def _tensor_cores(dtype, rows, dim, with_lse):
    return dtype != "f32" and rows >= (64 if dtype == "f16" else 48) and not (dim == 256 and with_lse)


# ------------------------------------------------------------------------------------------------------- unread tokens


def _check_unread(seed, fmt, dtype, lens, queries, q_heads, heads, dim, page, dev, spoil, with_lse, softcap=0.0,
                  slopes=None, window=0, prefix=None):
    """Attention with table entries spoiled by spoil(table) -> the pages it cut the table to, or None. Its tokens are
    masked: the reference leaves them out, the other tokens' positions as they were."""
    planes, table, lens, cu, q = _problem(seed, fmt, dtype, lens, queries, q_heads, heads, dim, page)
    keys, values = _gather(fmt, planes, table, lens)
    pages = planes[0].shape[0]
    table = spoil(table.copy())
    unread = []
    for b, n in enumerate(lens):
        j = np.arange(n) // page
        ids = np.where(j < table.shape[1], table[b, np.minimum(j, table.shape[1] - 1)], -1)
        unread.append((ids < 0) | (ids >= pages))
    o, l, reach, mass = ref.attention(q.float().numpy(), keys, values, lens, cu, dim**-0.5, softcap, slopes, prefix, None,
                                      window, unread)
    _device_error()
    tt, tl, tc, tp = _to(dev, table, lens, cu, None if prefix is None else np.asarray(prefix, np.int32))
    ts = None if slopes is None else torch.tensor(slopes, dtype=torch.float32, device=dev)
    got = kv.attention(q.to(dev), _cache(fmt, planes, dev), tt, tl, cu_q=tc, max_q=max(queries), softcap=softcap,
                       window=window, slopes=ts, prefix=tp, return_lse=with_lse)
    see = ref.visible(lens, cu, prefix, None, window)
    met = any(unread[b][lo:hi].any() for b in range(len(lens)) for _, lo, hi in see[cu[b] : cu[b + 1]])
    assert _device_error() in ((3,) if met else (0, 3))  # a table too short is reported whatever is seen of it
    got, lse = got if with_lse else (got, None)
    tensor = _tensor_cores(dtype, max(queries) * (q_heads // heads), dim, with_lse)
    bound, e = _bounds(dtype, tensor, with_lse, dim, softcap, o, reach, mass)
    g = got.double().cpu().numpy()
    assert np.isfinite(g).all()
    assert (np.abs(g - o) <= bound).all(), float((np.abs(g - o) / bound).max())
    empty = np.isinf(l)
    assert (g[empty] == 0).all()
    if with_lse:
        x = lse.double().cpu().numpy()
        assert np.array_equal(np.isinf(x), empty) and (x[empty] < 0).all()
        d = np.abs(x[~empty] - l[~empty])
        assert (d <= (e[~empty] + 2.0**-21 * (1 + np.abs(l[~empty])))).all()
    return empty


SPOILS = {"middle": lambda t: _put(t, (0, 3), (1, 2)), "first": lambda t: _put(t, (0, 0), (0, 1), (1, 0)),
          "last": lambda t: _put(t, (0, 9), (1, 11)), "most": lambda t: _put(t, *((b, i) for b in (0, 1) for i in range(1, 9)))}


def _put(table, *places):
    for i, at in enumerate(places):
        table[at] = (-1, 2**31 - 1, 1000, -(2**31))[i % 4]
    return table


@pytest.mark.parametrize("where", SPOILS)
@pytest.mark.parametrize("fmt,dtype,queries,dim,with_lse", [
    ("q4_0", "f32", [1, 1], 64, True), ("q8_0", "bf16", [3, 2], 128, True), ("q4_0", "bf16", [70, 66], 128, False),
    ("q8_0", "f16", [70, 150], 64, True), ("q4_0", "f16", [100, 30], 96, True), ("q8_0", "bf16", [60, 60], 256, False)])
def test_pages_outside_the_cache_are_masked(cuda, where, fmt, dtype, queries, dim, with_lse):
    _check_unread(201, fmt, dtype, [155, 180], queries, 4, 2, dim, 16, cuda, SPOILS[where], with_lse)
    _check_unread(202, fmt, dtype, [155, 180], queries, 4, 2, dim, 16, cuda, SPOILS[where], with_lse, softcap=9.0,
                  slopes=2.0 ** -np.arange(1, 5), window=50, prefix=[40, 0])


@pytest.mark.parametrize("fmt,dtype", [("q4_0", "f16"), ("q8_0", "bf16"), ("q4_0", "f32")])
@pytest.mark.parametrize("with_lse", [True, False])
def test_rows_that_see_unread_pages_alone_are_empty(cuda, fmt, dtype, with_lse):
    """A whole chunk from the sequence's beginning: its first rows see the first page only, which is not the cache's; long
    enough for blocks of keys without any page, between two that have theirs."""
    empty = _check_unread(203, fmt, dtype, [500, 33], [500, 33], 4, 2, 64, 16, cuda, SPOILS["first"], with_lse)
    assert empty[:32].all() and not empty[32:500].any() and empty[500:516].all()
    _check_unread(204, fmt, dtype, [700, 33], [60, 33], 4, 2, 64, 16, cuda,
                  lambda t: _put(t, *((0, i) for i in range(7, 27))), with_lse)


@pytest.mark.parametrize("fmt,dtype,queries,with_lse", [
    ("q4_0", "f32", [1, 1], True), ("q8_0", "bf16", [5, 9], True), ("q4_0", "bf16", [70, 130], False),
    ("q8_0", "f16", [70, 130], True)])
@pytest.mark.parametrize("window", [0, 40, 90, 1000])
def test_a_table_shorter_than_its_sequence(cuda, fmt, dtype, queries, with_lse, window):
    """Tokens past the table are masked; the queries stay where they are, at the end of the whole sequence."""
    for keep in (4, 9):
        _check_unread(205, fmt, dtype, [150, 170], queries, 4, 2, 64, 16, cuda, lambda t: t[:, :keep].copy(), with_lse,
                      window=window)
        _check_unread(206, fmt, dtype, [150, 170], queries, 4, 2, 64, 16, cuda, lambda t: t[:, :keep].copy(), with_lse,
                      window=window, slopes=2.0 ** -np.arange(1, 5), prefix=[70, 10])


# ------------------------------------------------------------------------------------------- values past f16's range


def _large(planes, table, lens, page, fmt, which, rng, every):
    """Raises the scales of every `every`-th token of each sequence: one block past the largest whose values all fit f16,
    up to f16's largest; the token's other blocks as they were."""
    scales = planes[1 if which == "k" else 3]
    past = 8192.0 if fmt == "q4_0" else 512.0
    for b, n in enumerate(lens):
        for j in range(every // 2, n, every):
            h, blk = rng.integers(scales.shape[1]), rng.integers(scales.shape[3])
            d = np.float16(np.exp(rng.uniform(np.log(past), np.log(65504.0))))
            scales[table[b, j // page], h, j % page, blk] = d.view(np.uint16)


def _resolution(fmt, planes, table, lens, cu, keys, values, q, page, scale, softcap, tensor):
    """What an f16 weight's smallest step can move an output by, where a row's weights or its values' scales lie far apart.
    Streaming: products of weight and value scale are held to 2^-25, their largest (the largest weight times the largest
    scale, rounded up to a power of two) at 2^8 or more: 2^-32 of it for each whole quant. Tensor cores: weights to 2^-25,
    the largest at 2^7 or more, times 2^4 (q8_0: 2^8) for keys whose values need it: 2^-32 of it for each value."""
    out = np.zeros(q.shape)
    group = q.shape[1] // keys[0].shape[1]
    for b, n in enumerate(lens):
        at = table[b, np.arange(n) // page], np.arange(n) % page
        d = np.abs(planes[3][at[0], :, at[1]].view(np.float16).astype(np.float64))  # [len][heads][dim / 32]
        for t in range(cu[b], cu[b + 1]):
            hi = n - (cu[b + 1] - cu[b]) + t - cu[b] + 1
            for h in range(q.shape[1]):
                g = h // group
                s = scale * (keys[b][:hi, g] @ q[t, h])
                s = softcap * np.tanh(s / softcap) if softcap else s
                w = np.exp(s - s.max())
                top = 1 / w.sum()
                if tensor:
                    past = d[:hi, g].max() >= (8192.0 if fmt == "q4_0" else 512.0)
                    step = top * (1 if not past else 16 if fmt == "q4_0" else 256)
                    out[t, h] = 2.0**-32 * step * np.abs(values[b][:hi, g]).sum(0)
                else:
                    quants = np.abs(values[b][:hi, g]) / np.repeat(d[:hi, g], 32, axis=-1)
                    out[t, h] = 2.0**-32 * top * d[:, g].max() * quants.sum(0)
    return out


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
@pytest.mark.parametrize("dtype,queries,q_heads,heads,dim,with_lse", [
    ("f32", [1, 3], 4, 2, 64, True), ("bf16", [1, 1], 8, 2, 128, True), ("bf16", [80, 30], 4, 2, 128, False),
    ("bf16", [80, 30], 4, 2, 64, True), ("bf16", [130, 30], 6, 2, 96, True), ("bf16", [50, 50], 4, 2, 256, False)])
@pytest.mark.parametrize("softcap", [0.0, 10.0])
def test_values_past_the_range_of_f16(cuda, fmt, which, dtype, queries, q_heads, heads, dim, with_lse, softcap):
    """Finite values of up to 128 * 65504 are attended to like any others. Scores are scaled so that the large keys
    do not decide alone. A token that holds a value past 65504 keeps its values to 2^-17 (q4_0: 2^-21) at least."""
    rng = np.random.default_rng(301)
    planes, table, lens, cu, q = _problem(302, fmt, dtype, [170, 90], queries, q_heads, heads, dim, 16)
    scale = dim**-0.5
    for w in which:
        _large(planes, table, lens, 16, fmt, w, rng, 11)
    if "k" in which:
        scale *= 2.0 / 65504.0 / (2.0 if fmt == "q4_0" else 32.0)
    keys, values = _gather(fmt, planes, table, lens)
    assert max(np.abs(x).max() for x in (keys if "k" in which else values)) > 65504
    o, l, reach, mass = ref.attention(q.float().numpy(), keys, values, lens, cu, scale, softcap)
    tt, tl, tc = _to(cuda, table, lens, cu)
    one = list(queries) == [1] * len(lens)
    _device_error()
    got = kv.attention(q.to(cuda), _cache(fmt, planes, cuda), tt, tl, scale=scale, cu_q=None if one else tc,
                       max_q=max(queries), softcap=softcap, return_lse=with_lse)
    assert _device_error() == 0
    got, lse = got if with_lse else (got, None)
    tensor = _tensor_cores(dtype, max(queries) * (q_heads // heads), dim, with_lse)
    bound, e = _bounds(dtype, tensor, with_lse, dim, softcap, o, reach, mass)
    if "v" in which:
        bound = bound + _resolution(fmt, planes, table, lens, cu, keys, values, q.double().numpy(), 16, scale, softcap, tensor)
        if tensor:
            bound = bound + (2.0**-21 if fmt == "q4_0" else 2.0**-17)
    g = got.double().cpu().numpy()
    assert np.isfinite(g).all()
    assert (np.abs(g - o) <= bound).all(), float((np.abs(g - o) / bound).max())
    if with_lse:
        d = np.abs(lse.double().cpu().numpy() - l)
        assert (d <= e + 2.0**-21 * (1 + np.abs(l))).all()


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("with_lse", [True, False])
def test_one_large_key_alone(cuda, fmt, sign, with_lse):
    """Rows that see a single key, whose values lie past f16's range: its value, whatever the score's sign."""
    planes, table, lens, cu, _ = _problem(303, fmt, "bf16", [60], [60], 2, 1, 64, 16)
    planes[1][...] = np.float16(65504.0).view(np.uint16)
    planes[3][...] = np.float16(60000.0).view(np.uint16)
    keys, values = _gather(fmt, planes, table, lens)
    q = torch.from_numpy(np.sign(keys[0]).repeat(2, 1).astype(np.float32) * sign).to(torch.bfloat16)
    tt, tl, tc = _to(cuda, table, lens, cu)
    got = kv.attention(q.to(cuda), _cache(fmt, planes, cuda), tt, tl, cu_q=tc, max_q=60, window=1, scale=1e-6,
                       return_lse=with_lse)
    got, lse = got if with_lse else (got, None)
    want = values[0].repeat(2, 1)
    assert (np.abs(got.double().cpu().numpy() - want) <= 2.0**-8 * np.abs(want)).all()
    if with_lse:
        s = 1e-6 * (keys[0].repeat(2, 1) * q.double().numpy()).sum(-1)
        assert (np.abs(lse.double().cpu().numpy() - s) <= 2.0**-15 * np.abs(s)).all()


# ------------------------------------------------------------------------------------------------ scales, caps, tails


@pytest.mark.parametrize("dtype,n", [("f32", 1), ("bf16", 1), ("f16", 3), ("f32", 20), ("f16", 64), ("bf16", 64)])
@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("scale", [1e-44, 1e-38, 1e-30, 1e-12, 1.0, 1e12, 1e30])
@pytest.mark.parametrize("softcap", [0.0, 1e-20, 20.0, 1e20])
def test_rows_of_zeros_at_every_scale(cuda, dtype, n, fmt, scale, softcap):
    """Equal scores whatever the scale and the cap: the mean of the values, with keys that are masked beside them."""
    planes, table, lens, cu, q = _problem(401, fmt, dtype, [77, 130], [n, n], 4, 2, 64, 16)
    keys, values = _gather(fmt, planes, table, lens)
    o, l, reach, mass = ref.attention(q.float().numpy() * 0, keys, values, lens, cu, 1.0, window=70)
    tt, tl, tc = _to(cuda, table, lens, cu)
    got, lse = kv.attention(q.to(cuda) * 0, _cache(fmt, planes, cuda), tt, tl, cu_q=tc, max_q=n, scale=scale,
                            softcap=softcap, window=70, return_lse=True)
    bound, _ = _bounds(dtype, _tensor_cores(dtype, 2 * n, 64, True), True, 64, 0.0, o, reach, mass)
    assert (np.abs(got.double().cpu().numpy() - o) <= bound).all()
    assert (np.abs(lse.double().cpu().numpy() - l) <= 2.0**-19 * (1 + np.abs(l))).all()


@pytest.mark.parametrize("dtype,n", [("f32", 1), ("bf16", 1), ("f32", 20), ("bf16", 64)])
def test_tiny_queries_and_scales(cuda, dtype, n):
    """Scores far below 1 in products that pass f32's range on the way."""
    planes, table, lens, cu, q = _problem(402, "q4_0", dtype, [77, 130], [n, n], 4, 2, 64, 16)
    keys, values = _gather("q4_0", planes, table, lens)
    q = q * torch.tensor(1e-33, dtype=DT[dtype])
    o, l, reach, mass = ref.attention(q.float().numpy(), keys, values, lens, cu, 1e-20, window=70)
    tt, tl, tc = _to(cuda, table, lens, cu)
    got = kv.attention(q.to(cuda), _cache("q4_0", planes, cuda), tt, tl, cu_q=tc, max_q=n, scale=1e-20, window=70)
    bound, _ = _bounds(dtype, _tensor_cores(dtype, 2 * n, 64, False), False, 64, 0.0, o, reach, mass)
    assert (np.abs(got.double().cpu().numpy() - o) <= bound).all()


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dtype,queries", [("f32", 1), ("bf16", 1), ("f16", 16), ("bf16", 16)])
@pytest.mark.parametrize("nats", [8.0, 12.0, 17.0, 19.0])
def test_a_long_tail_of_small_weights(cuda, fmt, dtype, queries, nats):
    """One key of weight 1 and value 0 before many equal small weights, whose values are the answer; enough sequences that
    a thread block takes each of them whole. A weight is at least 2^7 for the row's largest and rounded at 2^-25 at worst:
    2^-32 of the largest for each key, beside its own 2^-11."""
    n, batch, page = 1088, 160, 64
    planes, table, lens, cu, q = _problem(403, fmt, dtype, [n] * batch, [queries] * batch, 4, 1, 64, page)
    off = 8 if fmt == "q4_0" else 128
    # keys of zeros but for the first one's first value, 7; values of 1 but for the first key's, 0
    kx, vx = np.zeros((n, 64)), np.ones((n, 64))
    kx[0, 0], vx[0] = 7.0, 0.0
    for x, (rows, scales), which in ((kx, planes[:2], "k"), (vx, planes[2:], "v")):
        place, shift = ref._places(fmt, 64, which)
        r = np.zeros((n, rows.shape[-1]), np.uint8)
        for e in range(64):
            r[:, place[e]] |= (x[:, e] + off).astype(np.uint8) << np.uint8(shift[e])
        rows[table, 0] = r.reshape(n // page, page, -1)
        scales[...] = np.float16(1.0).view(np.uint16)
    q = torch.zeros_like(q)
    q[:, :, 0] = 1.0
    keys, values = _gather(fmt, planes, table[:1], [n])
    assert np.array_equal(keys[0][:, 0], kx) and np.array_equal(values[0][:, 0], vx)
    scale = nats / 7.0
    # every sequence is the same one
    o, _, reach, mass = ref.attention(q[:queries].float().numpy(), keys, values, [n], cu[:2], scale)
    tt, tl, tc = _to(cuda, table, lens, cu)
    got = kv.attention(q.to(cuda), _cache(fmt, planes, cuda), tt, tl, cu_q=tc, max_q=queries, scale=scale)
    bound, _ = _bounds(dtype, _tensor_cores(dtype, 4 * queries, 64, False), False, 64, 0.0, o, reach, mass)
    bound = bound + n * 2.0**-32
    d = np.abs(got.double().cpu().numpy().reshape(batch, *o.shape) - o)
    assert (d <= bound).all(), float((d / bound).max())


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dim,heads,group", [(64, 2, 4), (96, 2, 3), (128, 2, 4), (256, 2, 2)])
@pytest.mark.parametrize("queries", [[1] * 24, [4] * 12, [200, 90]])
@pytest.mark.parametrize("with_lse", [True, False])
def test_f16_results_are_as_good_as_their_rounding(cuda, fmt, dim, heads, group, queries, with_lse):
    """Of what an f16 call rounds, the output and the values (tensor cores) or the weights (streaming) have 11 bits, all else
    20 or more: two roundings of a size, independent, so sqrt(2) of the output's own in the 2-norm."""
    lens = [300 + 37 * i for i in range(len(queries))]
    planes, table, lens, cu, q = _problem(406, fmt, "f16", lens, queries, heads * group, heads, dim, 32)
    keys, values = _gather(fmt, planes, table, lens)
    o, _, _, _ = ref.attention(q.float().numpy(), keys, values, lens, cu, dim**-0.5)
    tt, tl, tc = _to(cuda, table, lens, cu)
    got = kv.attention(q.to(cuda), _cache(fmt, planes, cuda), tt, tl, cu_q=tc, max_q=max(queries), return_lse=with_lse)
    g = (got[0] if with_lse else got).double().cpu().numpy()
    own = np.linalg.norm(o.astype(np.float16).astype(np.float64) - o)
    assert np.linalg.norm(g - o) <= 1.5 * own, np.linalg.norm(g - o) / own


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("with_lse", [True, False])
def test_f16_weights_of_values_that_cancel(cuda, fmt, dim, with_lse):
    """Rows that see two keys of opposite values, whole numbers: the difference of nearly equal weights, which carry 20 bits."""
    planes, table, lens, cu, q = _problem(407, fmt, "f16", [300], [200], 4, 2, dim, 32)
    rows, scales = planes[2:]
    one = np.random.default_rng(408).integers(-7, 8, dim)
    place, shift = ref._places(fmt, dim, "v")
    for sign in (1, -1):
        r = np.zeros(rows.shape[-1], np.uint8)
        for e in range(dim):
            r[place[e]] |= np.uint8(sign * one[e] + (8 if fmt == "q4_0" else 128)) << np.uint8(shift[e])
        rows[:, :, (0 if sign > 0 else 1) :: 2] = r
    scales[...] = np.float16(1.0).view(np.uint16)
    keys, values = _gather(fmt, planes, table, lens)
    scale = 0.02 * dim**-0.5
    o, _, reach, mass = ref.attention(q.float().numpy(), keys, values, lens, cu, scale, window=2)
    tt, tl, tc = _to(cuda, table, lens, cu)
    got = kv.attention(q.to(cuda), _cache(fmt, planes, cuda), tt, tl, cu_q=tc, max_q=200, scale=scale, window=2,
                       return_lse=with_lse)
    g = (got[0] if with_lse else got).double().cpu().numpy()
    if dim == 256 and with_lse:  # the streaming kernel: weights of 11 bits
        bound = U["f16"] * np.abs(o) + 2 * (2.0**-11 + 2.0**-15 * reach + 2.0**-20)[..., None] * mass
    else:
        bound = U["f16"] * np.abs(o) + 2 * (2.0**-20 + 2.0**-15 * reach + 2.0**-20)[..., None] * mass
    assert (np.abs(g - o) <= bound).all(), float((np.abs(g - o)[mass > 0] / bound[mass > 0]).max())


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dim", [64, 96, 128])
def test_f16_results_do_not_depend_on_lse(cuda, fmt, dim):
    planes, table, lens, cu, q = _problem(409, fmt, "f16", [300, 150], [200, 60], 8, 2, dim, 32)
    tt, tl, tc = _to(cuda, table, lens, cu)
    cache, q = _cache(fmt, planes, cuda), q.to(cuda)
    out, _ = kv.attention(q, cache, tt, tl, cu_q=tc, max_q=200, return_lse=True)
    assert torch.equal(kv.attention(q, cache, tt, tl, cu_q=tc, max_q=200), out)


@pytest.mark.parametrize("cap", [0.3, 1.0, 50.0])
@pytest.mark.parametrize("dtype,n", [("f32", 1), ("bf16", 50)])
def test_the_cap_against_tanh(cuda, cap, dtype, n):
    """lse of a row that sees one key is its capped score: scores from 1e-4 to 30 times the cap, both signs. The cap's own
    steps cost 2^-21 of its result at most (tanh within 2^-22, two roundings), the score 2^-19 of it (16-bit calls: 2^-15),
    which tanh, of slope at most 1, passes on; 2^x costs 2^-20, and lse is a product and a sum of logarithms, 2^-21 of 1 + |lse|."""
    rng = np.random.default_rng(404)
    batch = 400
    planes, table, lens, cu, q = _problem(405, "q8_0", dtype, [n] * batch, [n] * batch, 1, 1, 64, 64)
    keys, values = _gather("q8_0", planes, table, lens)
    k = np.concatenate([x[:, 0] for x in keys])
    x = np.exp(rng.uniform(np.log(1e-4), np.log(30.0), len(k))) * rng.choice([-1.0, 1.0], len(k)) * cap
    q = torch.from_numpy((k * (x / (k * k).sum(-1))[:, None]).astype(np.float32)[:, None]).to(DT[dtype])
    s = (q.double().numpy()[:, 0] * k).sum(-1)
    reach = np.abs(q.double().numpy()[:, 0] * k).sum(-1)
    want = cap * np.tanh(s / cap)
    tt, tl, tc = _to(cuda, table, lens, cu)
    _, lse = kv.attention(q.to(cuda), _cache("q8_0", planes, cuda), tt, tl, cu_q=tc, max_q=n, scale=1.0, softcap=cap,
                          window=1, return_lse=True)
    d = np.abs(lse.double().cpu().numpy()[:, 0] - want)
    slope = 1 - np.tanh(np.maximum(np.abs(s) - 2.0**-10 * reach, 0) / cap) ** 2
    bound = (2.0**-19 if dtype == "f32" else 2.0**-15) * reach * slope
    bound = bound + 2.0**-21 * np.abs(want) + 2.0**-20 + 2.0**-21 * (1 + np.abs(want))
    assert (d <= bound).all(), float((d / bound).max())


# ------------------------------------------------------------------------------------ the kernels' boundary, streams


@pytest.mark.parametrize("rows", [47, 48, 49, 63, 64, 65])
@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("with_lse", [True, False])
def test_rows_around_the_kernels_boundary(cuda, rows, fmt, dim, with_lse):
    """One query head a KV head, so that the rows are the query tokens; and the same rows with a group of heads."""
    for dtype in ("f16", "bf16"):
        shapes = [(rows, 1)] + [(rows // g, g) for g in (3, 7) if rows % g == 0]
        for n, group in shapes:
            planes, table, lens, cu, q = _problem(501, fmt, dtype, [200, 61], [n, n // 2], 2 * group, 2, dim, 32)
            keys, values = _gather(fmt, planes, table, lens)
            o, l, reach, mass = ref.attention(q.float().numpy(), keys, values, lens, cu, dim**-0.5)
            tt, tl, tc = _to(cuda, table, lens, cu)
            got = kv.attention(q.to(cuda), _cache(fmt, planes, cuda), tt, tl, cu_q=tc, max_q=n, return_lse=with_lse)
            got, lse = got if with_lse else (got, None)
            bound, e = _bounds(dtype, _tensor_cores(dtype, rows, dim, with_lse), with_lse, dim, 0.0, o, reach, mass)
            assert (np.abs(got.double().cpu().numpy() - o) <= bound).all()
            if with_lse:
                assert (np.abs(lse.double().cpu().numpy() - l) <= e + 2.0**-21 * (1 + np.abs(l))).all()


@pytest.mark.parametrize("dtype,queries", [("bf16", [30, 12]), ("f16", [100, 7]), ("f32", [9, 11])])
def test_without_max_q(cuda, dtype, queries):
    """T bounds the queries of a sequence: on the tensor cores with 42 * 4 and 107 * 4 rows."""
    planes, table, lens, cu, q = _problem(502, "q4_0", dtype, [177, 130], queries, 8, 2, 128, 16)
    keys, values = _gather("q4_0", planes, table, lens)
    o, l, reach, mass = ref.attention(q.float().numpy(), keys, values, lens, cu, 128**-0.5)
    tt, tl, tc = _to(cuda, table, lens, cu)
    for with_lse in (False, True):
        got = kv.attention(q.to(cuda), _cache("q4_0", planes, cuda), tt, tl, cu_q=tc, return_lse=with_lse)
        g = (got[0] if with_lse else got).double().cpu().numpy()
        bound, _ = _bounds(dtype, dtype != "f32", with_lse, 128, 0.0, o, reach, mass)
        assert (np.abs(g - o) <= bound).all()


def test_calls_on_streams_that_overlap(cuda):
    """Calls of both kernels on three streams at once, each with a workspace: the same bits as one after the other."""
    jobs = []
    for seed, dtype, lens, queries in ((601, "bf16", [3000, 900], [1, 1]), (602, "f16", [4000, 150], [300, 100]),
                                       (603, "f32", [2500, 1200], [4, 3])):
        planes, table, ln, cu, q = _problem(seed, "q4_0", dtype, lens, queries, 8, 2, 128, 64)
        tt, tl, tc = _to(cuda, table, ln, cu)
        cache, q = _cache("q4_0", planes, cuda), q.to(cuda)
        a = dict(cu_q=tc, max_q=max(queries))
        ws = torch.empty(kv.attention_workspace_size(cache, q.shape[0], 2, 8, q.dtype, max(queries)), dtype=torch.uint8,
                         device=cuda)
        jobs.append((q, cache, tt, tl, a, ws, kv.attention(q, cache, tt, tl, **a), torch.cuda.Stream()))
    torch.cuda.synchronize()
    outs = [[] for _ in jobs]
    for _ in range(20):
        for (q, cache, tt, tl, a, ws, want, stream), got in zip(jobs, outs):
            with torch.cuda.stream(stream):
                got.append(kv.attention(q, cache, tt, tl, workspace=ws, **a))
    torch.cuda.synchronize()
    for job, got in zip(jobs, outs):
        for x in got:
            assert torch.equal(x, job[6])
    assert _device_error() == 0


# ----------------------------------------------------------------------------------------------------------- refusals


def test_more_queries_than_max_q_are_reported(cuda):
    _device_error()
    for dtype, n, most in ((torch.float32, 40, 2), (torch.bfloat16, 300, 48)):
        cache = kv.KVCache("q4_0", 30, 16, 1, 64, device=cuda)
        q = torch.randn(n, 1, 64, device=cuda, dtype=dtype)
        table = torch.arange(30, dtype=torch.int32, device=cuda)[None]
        lens, cu = torch.tensor([400], dtype=torch.int32, device=cuda), torch.tensor([0, n], dtype=torch.int32, device=cuda)
        kv.attention(q, cache, table, lens, cu_q=cu, max_q=n)
        assert _device_error() == 0
        kv.attention(q, cache, table, lens, cu_q=cu, max_q=most)
        assert _device_error() == 4


def test_numbers_out_of_range_are_value_errors(cuda):
    c = kv.KVCache("q4_0", 4, 16, 2, 64, device=cuda)
    q = torch.zeros(2, 4, 64, device=cuda)
    table, lens = torch.zeros(2, 3, dtype=torch.int32, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    for bad in (dict(scale=1e39), dict(scale=float("inf")), dict(scale=1e-60), dict(softcap=1e39), dict(window=2**31),
                dict(window=-(2**40)), dict(max_len=2**63), dict(max_len=-1)):
        with pytest.raises(ValueError):
            kv.attention(q, c, table, lens, **bad)
    with pytest.raises(TypeError):
        kv.attention_workspace_size(c, 2, 2, 4, torch.int8)


# -------------------------------------------------------------------------------------------------------------- write


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_blocks_of_zeros_have_ggmls_scale(cuda, dtype):
    """ggml's maximum begins at +0 and takes larger magnitudes only: a block of zeros of either sign has the scale
    +0 / -8 = -0 in q4_0, and +0 in q8_0."""
    x = torch.zeros(4, 1, 64, dtype=DT[dtype])
    x[1], x[2, :, ::2], x[3, :, 1:] = -0.0, -0.0, -0.0
    slots = torch.arange(4, device=cuda)
    for fmt, bits in (("q4_0", 0x8000), ("q8_0", 0)):
        cache = kv.KVCache(fmt, 1, 16, 1, 64, device=cuda)
        kv.kv_write(cache, x.to(cuda), x.to(cuda), slots)
        for scales in (cache.ks, cache.vs):
            assert (scales.cpu().numpy().view(np.uint16)[0, 0, :4] == bits).all()
        for got in kv.kv_read(cache, slots):
            assert (got == 0).all()
