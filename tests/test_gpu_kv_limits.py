"""comp_b200.kv where its inputs reach a limit: pages that cannot be read, tables shorter than their sequences, values past
f16's range, scales and caps at the ends of their ranges, long tails of small weights, rows on either side of the kernels'
boundary, calls on streams that overlap. Against the 64-bit restatement (oracle.kv), with the bounds of test_gpu_kv."""

import numpy as np
import pytest
import torch

from comp_b200 import kv
from oracle import kv as ref

from .test_gpu_kv import _bounds, _cache, _device_error, _gather, _problem

pytestmark = pytest.mark.gpu


def _to(dev, *arrays):
    return [None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(dev) for a in arrays]


def _tensor_cores(dtype, rows, dim, with_lse):
    return dtype != "f32" and rows >= 48 and not (dim == 256 and with_lse)


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
