"""The quantized KV cache and its attention (comp_b200.kv) on the GPU, through the C-ABI, against a plain restatement in 64
bits (oracle.kv): bytes of a write and values of a read exactly, attention within bounds that follow from the roundings.

Bounds of attention. The result is rounded to the queries' type (u = 2^-8 bf16, 2^-11 f16, 2^-23 f32, as half an ulp's
share of a value at most, doubled for the sums before it). A weight carries a relative error of at most W (f16 weights:
2^-11 for its rounding and as much for its value's rounding in the tensor-core kernels; f32 calls: two f16 parts, 2^-20)
plus that of its score, at most S * reach (keys rounded to f16: 2^-11; whole quants whose sums are cut off at 2^-16 of
their largest term; f32 calls: 2^-19), plus 2^-20 for 2^x and, with a cap, 2^-20 * cap for the cap's own steps. A relative
error e of every weight moves an output by at most 2 e * mass (numerator and denominator), and lse by at most e.
"""

import numpy as np
import pytest
import torch

from comp_b200 import _lib, kv
from oracle import kv as ref

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
U = {"f32": 2.0**-22, "f16": 2.0**-11, "bf16": 2.0**-8}


def _device_error():
    import ctypes

    code = ctypes.c_int()
    _lib.call("b2q_device_error", ctypes.byref(code), 1)
    return code.value


def _planes(fmt, pages, heads, page, dim, rng, keys=None, values=None):
    """Random planes (numpy) with finite scales."""
    shape = (pages, heads, page, dim)
    out = []
    for which, x in (("k", keys), ("v", values)):
        x = rng.standard_normal(shape).astype(np.float32) if x is None else x
        out += list(ref.pack(fmt, x, which))
    return out


def _cache(fmt, planes, dev):
    kq, ks, vq, vs = (torch.from_numpy(p.view(np.int16) if p.dtype == np.uint16 else p).to(dev) for p in planes)
    return kv.KVCache.from_planes(fmt, kq, ks, vq, vs)


def _gather(fmt, planes, table, lens):
    """Per sequence (keys, values) [len][heads][dim] in 64 bits."""
    keys, values = [], []
    for b, n in enumerate(lens):
        for which, (rows, scales), into in (("k", planes[:2], keys), ("v", planes[2:], values)):
            page = rows.shape[2]
            ids = table[b, : -(-int(n) // page)]
            x = ref.unpack(fmt, rows[ids], scales[ids], which)  # [pages][heads][page][dim]
            into.append(x.transpose(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[: int(n)])
    return keys, values


def _bounds(dtype, tensor_cores, with_lse, dim, softcap, o, reach, mass):
    if dtype == "f32":
        w, s = 2.0**-20, 2.0**-19
    elif tensor_cores:
        w, s = 2.0**-10, (2.0**-15 if with_lse and dim != 256 else 2.0**-11)
    else:
        w, s = 2.0**-11, 2.0**-15
    e = s * reach + 2.0**-20 * (1 + softcap)
    return U[dtype] * np.abs(o) + 2 * (w + e)[..., None] * mass + 1e-30, e


def _problem(seed, fmt, dtype, lens, queries, q_heads, heads, dim, page, spare=3):
    rng = np.random.default_rng(seed)
    lens = np.asarray(lens)
    need = -(-lens // page)
    pages = int(need.sum()) + spare
    planes = _planes(fmt, pages, heads, page, dim, rng)
    perm = rng.permutation(pages)
    table = np.full((len(lens), max(1, int(need.max()))), -1, np.int32)  # entries past a sequence's end are nobody's
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at : at + n]
        at += n
    cu = np.concatenate([[0], np.cumsum(queries)]).astype(np.int32)
    q = torch.from_numpy(rng.standard_normal((int(cu[-1]), q_heads, dim)).astype(np.float32) * 1.5).to(DT[dtype])
    return planes, table, lens.astype(np.int32), cu, q


def _check(seed, fmt, dtype, lens, queries, q_heads, heads, dim, page, dev, softcap=0.0, slopes=None, prefix=None,
           starts=None, window=0, scale=None, max_q="exact", with_lse=True, poison=None):
    planes, table, lens, cu, q = _problem(seed, fmt, dtype, lens, queries, q_heads, heads, dim, page)
    keys, values = _gather(fmt, planes, table, lens)
    scale = dim**-0.5 if scale is None else scale
    o, l, reach, mass = ref.attention(q.float().numpy(), keys, values, lens, cu, scale, softcap, slopes, prefix, starts,
                                      window)
    if poison is not None:
        poison(planes, table)
    cache = _cache(fmt, planes, dev)
    t = lambda a, ty=np.int32: None if a is None else torch.from_numpy(np.ascontiguousarray(a, ty)).to(dev)  # noqa: E731
    most = int(max(queries))
    _device_error()
    got = kv.attention(q.to(dev), cache, t(table), t(lens), scale=scale,
                       cu_q=None if list(queries) == [1] * len(lens) else t(cu),
                       max_q=most if max_q == "exact" else max_q, max_len=int(lens.max()), softcap=softcap,
                       window=window, slopes=t(slopes, np.float32), prefix=t(prefix), starts=t(starts),
                       return_lse=with_lse)
    got, lse = got if with_lse else (got, None)
    assert got.dtype == DT[dtype] and got.shape == q.shape
    assert _device_error() == 0
    rows = (q.shape[0] if max_q is None else most) * (q_heads // heads)
    tc = dtype != "f32" and rows >= 64 and not (dim == 256 and with_lse)
    bound, e = _bounds(dtype, tc, with_lse, dim, softcap, o, reach, mass)
    g = got.double().cpu().numpy()
    assert np.isfinite(g).all()
    assert (np.abs(g - o) <= bound).all(), float((np.abs(g - o) / bound).max())
    empty = np.isinf(l)
    assert (g[empty] == 0).all()
    if with_lse:
        x = lse.double().cpu().numpy()
        assert np.array_equal(np.isinf(x), empty) and (x[empty] < 0).all()
        d = np.abs(x - l)[~empty]
        assert (d <= (e + 2.0**-21 * (1 + np.abs(np.where(empty, 0, l))))[~empty]).all()
    return g


# --------------------------------------------------------------------------------------------------------- write, read


def _values(rng, shape):
    """Normal values with what quantizers trip over: zeros, a zero block, equal magnitudes of both signs, outliers."""
    x = rng.standard_normal(shape).astype(np.float32)
    x[rng.random(shape) < 0.05] = 0.0
    x[rng.random(shape) < 0.01] *= 1000.0
    flat = x.reshape(-1, 32)
    flat[0] = 0.0
    flat[1] = -0.0
    flat[2, 5], flat[2, 9] = 3.5, -3.5
    flat[3, 5], flat[3, 9] = -3.5, 3.5
    flat[2, :5] = flat[3, :5] = 1.0
    flat[4] = np.linspace(-8, 7.5, 32)  # quants on and beside their halves
    return x


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dim,heads,page", [(64, 1, 16), (96, 5, 32), (128, 8, 64), (256, 3, 256)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_write_and_read_are_exact(cuda, fmt, dim, heads, page, dtype):
    rng = np.random.default_rng(dim + heads)
    tokens, pages = 2 * page + 7, 5
    before = _planes(fmt, pages, heads, page, dim, rng)
    cache = _cache(fmt, before, cuda)
    # k and v as views of one fused product
    qkv = torch.from_numpy(_values(rng, (tokens, 2 * heads + 1, dim))).to(DT[dtype]).to(cuda)
    k, v = qkv[:, 1 : heads + 1], qkv[:, heads + 1 :]
    slots = rng.permutation(pages * page)[:tokens]
    slots[3::5] = -1 - np.arange(len(slots[3::5]))
    ts = torch.from_numpy(slots).to(cuda)
    kv.kv_write(cache, k, v, ts)
    keep = slots >= 0
    for which, x, rows, scales, (r0, s0) in (("k", k, cache.kq, cache.ks, before[:2]), ("v", v, cache.vq, cache.vs, before[2:])):
        want_r, want_s = ref.pack(fmt, x.float().cpu().numpy(), which)
        r, s = r0.copy(), s0.copy()
        r[slots[keep] // page, :, slots[keep] % page] = want_r[keep]
        s[slots[keep] // page, :, slots[keep] % page] = want_s[keep]
        assert np.array_equal(rows.cpu().numpy(), r)
        assert np.array_equal(scales.cpu().numpy().view(np.uint16), s)
    for out in ("f32", "f16", "bf16"):
        gk, gv = kv.kv_read(cache, ts, dtype=DT[out])
        for which, g, rows, scales in (("k", gk, cache.kq, cache.ks), ("v", gv, cache.vq, cache.vs)):
            x = ref.unpack(fmt, rows.cpu().numpy(), scales.cpu().numpy().view(np.uint16), which)
            want = np.where(keep[:, None, None], x[slots // page * keep, :, slots % page * keep], 0.0)
            want = torch.from_numpy(want.astype(np.float32)).to(DT[out])  # f16 times a small integer is exact in f32
            assert torch.equal(g.cpu(), want)


def test_write_strides_and_order_do_not_matter(cuda):
    rng = np.random.default_rng(5)
    x = torch.from_numpy(rng.standard_normal((9, 4, 128)).astype(np.float32)).to(cuda)
    slots = torch.tensor([5, 17, 2, 63, 0, 31, 16, 40, 8], device=cuda)
    caches = [kv.KVCache("q4_0", 4, 16, 4, 128, device=cuda) for _ in range(4)]
    kv.kv_write(caches[0], x, x, slots)
    kv.kv_write(caches[1], x.transpose(0, 1).contiguous().transpose(0, 1), x, slots)  # heads outermost
    odd = torch.zeros(9 * 4 * 128 + 1, device=cuda)[1:].view(9, 4, 128).copy_(x)  # 4-byte aligned
    kv.kv_write(caches[2], odd, x.flip(2).flip(2), torch.stack([slots, slots], 1)[:, 0])
    perm = torch.randperm(9, device=cuda)
    kv.kv_write(caches[3], x[perm], x[perm], slots[perm])
    for c in caches[1:]:
        assert torch.equal(c.kq, caches[0].kq) and torch.equal(c.vs, caches[0].vs)
    assert caches[0].nbytes == 4 * 16 * 4 * 2 * (64 + 8)


def test_nothing_to_do(cuda):
    c = kv.KVCache("q8_0", 2, 16, 2, 64, device=cuda)
    e = torch.empty((0, 2, 64), device=cuda)
    none = torch.empty(0, dtype=torch.int64, device=cuda)
    kv.kv_write(c, e, e, none)
    k, v = kv.kv_read(c, none)
    assert k.shape == (0, 2, 64) and not c.kq.any()
    t = torch.empty((0, 3), dtype=torch.int32, device=cuda)
    assert kv.attention(e, c, t, torch.empty(0, dtype=torch.int32, device=cuda)).shape == (0, 2, 64)
    # sequences without tokens, a table without pages
    q = torch.randn(3, 2, 64, device=cuda)
    lens = torch.zeros(3, dtype=torch.int32, device=cuda)
    for pages in (0, 2):
        out, lse = kv.attention(q, c, torch.zeros((3, pages), dtype=torch.int32, device=cuda), lens, return_lse=True)
        assert not out.any() and torch.isinf(lse).all() and (lse < 0).all()


# ----------------------------------------------------------------------------------------------------------- attention


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dim,heads,group", [(64, 3, 1), (96, 2, 5), (128, 2, 4), (128, 1, 16), (256, 2, 3), (256, 1, 9)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_single_tokens(cuda, fmt, dim, heads, group, dtype):
    for page, lens in ((16, [1, 2, 15, 16, 17, 0, 33]), (64, [63, 64, 65, 1, 500, 129]), (256, [255, 256, 700])):
        _check(page, fmt, dtype, lens, [1] * len(lens), heads * group, heads, dim, page, cuda)


@pytest.mark.parametrize("fmt,dtype", [("q4_0", "bf16"), ("q8_0", "f16"), ("q4_0", "f32")])
@pytest.mark.parametrize("opts", [dict(softcap=20.0), dict(window=7), dict(window=100), dict(slopes=True), dict(scale=0.3),
                                  dict(starts=True), dict(softcap=5.0, window=33, slopes=True, starts=True)])
def test_single_tokens_options(cuda, fmt, dtype, opts):
    lens = [1, 40, 64, 129, 300, 301]
    o = dict(opts)
    if o.pop("slopes", False):
        o["slopes"] = 2.0 ** -np.arange(1, 9)
    if o.pop("starts", False):
        o["starts"] = [0, 39, 64, 100, 0, 999]  # one key, none (at its length), some, all, none
    _check(11, fmt, dtype, lens, [1] * 6, 8, 2, 128, 16, cuda, **o)


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,q_heads,heads", [(64, 4, 4), (128, 8, 2), (96, 12, 2), (256, 4, 2)])
def test_a_few_tokens(cuda, fmt, dtype, dim, q_heads, heads):
    _check(21, fmt, dtype, [5, 70, 1, 200, 64], [5, 3, 1, 0, 2], q_heads, heads, dim, 32, cuda)
    _check(22, fmt, dtype, [130, 66], [2, 5], q_heads, heads, dim, 64, cuda, softcap=10.0, prefix=[100, 3], window=90)


@pytest.mark.parametrize("fmt", ["q4_0", "q8_0"])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim,q_heads,heads", [(64, 2, 2), (96, 6, 2), (128, 8, 2), (256, 4, 2)])
@pytest.mark.parametrize("with_lse", [True, False])
def test_prompt_chunks(cuda, fmt, dtype, dim, q_heads, heads, with_lse):
    _check(31, fmt, dtype, [130, 64, 300, 1, 90], [65, 64, 33, 1, 0], q_heads, heads, dim, 16, cuda, with_lse=with_lse)


@pytest.mark.parametrize("fmt,dtype,with_lse", [("q4_0", "bf16", False), ("q8_0", "f16", True)])
@pytest.mark.parametrize("opts", [dict(softcap=8.0), dict(window=50), dict(slopes=True), dict(prefix=[90, 10, 150]),
                                  dict(docs=40), dict(softcap=30.0, window=70, slopes=True, prefix=[50, 60, 70], docs=64)])
def test_prompt_chunks_options(cuda, fmt, dtype, with_lse, opts):
    lens, queries = [200, 96, 150], [100, 96, 40]
    o = dict(opts)
    if o.pop("slopes", False):
        o["slopes"] = 2.0 ** -np.arange(1, 9)
    docs = o.pop("docs", 0)
    if docs:
        pos = np.concatenate([np.arange(n - m, n) for n, m in zip(lens, queries)])
        o["starts"] = pos // docs * docs
        o["starts"][7::50] = 1000  # rows that see nothing
    _check(41, fmt, dtype, lens, queries, 8, 2, 128, 64, cuda, with_lse=with_lse, **o)


def test_many_rows_and_long_keys_are_split_and_joined(cuda):
    # more tiles than the GPU has places, tiles that cross shares, and one long sequence over the whole GPU
    _check(51, "q4_0", "bf16", [3000, 40, 1, 2500], [70, 3, 1, 130], 16, 2, 64, 64, cuda)
    _check(52, "q8_0", "f16", [9000], [1], 4, 1, 64, 128, cuda)
    _check(53, "q4_0", "f32", [4097, 5], [1, 1], 8, 8, 64, 16, cuda)
    _check(54, "q4_0", "f16", [33] * 70, [1] * 70, 24, 12, 64, 32, cuda)


def test_default_bounds_and_fused_queries(cuda):
    """Without max_q and max_len, with queries cut out of a fused product, out and workspace of the caller's."""
    planes, table, lens, cu, q = _problem(61, "q4_0", "f16", [77, 130], [2, 9], 8, 2, 128, 16)
    cache = _cache("q4_0", planes, cuda)
    t = [torch.from_numpy(x).to(cuda) for x in (table, lens, cu)]
    want = kv.attention(q.to(cuda), cache, t[0], t[1], cu_q=t[2], max_q=9, max_len=130)
    wide = torch.zeros((11, 12, 128), dtype=torch.float16, device=cuda)
    wide[:, :8] = q.to(cuda)
    again = kv.attention(wide[:, :8], cache, t[0], t[1], cu_q=t[2], max_q=9)
    assert torch.equal(want, again)
    out = torch.full((11, 8, 128), 7.0, dtype=torch.float16, device=cuda)
    size = kv.attention_workspace_size(cache, 11, 2, 8, torch.float16, max_q=9)
    ws = torch.full((size,), 255, dtype=torch.uint8, device=cuda)  # whatever it held
    got = kv.attention(wide[:, :8], cache, t[0], t[1], cu_q=t[2], max_q=9, out=out, workspace=ws)
    assert got is out and torch.equal(out, want)
    # max_q left out: T bounds it
    keys, values = _gather("q4_0", planes, table, lens)
    o, _, reach, mass = ref.attention(q.float().numpy(), keys, values, lens, cu, 128**-0.5)
    bound, _ = _bounds("f16", True, False, 128, 0.0, o, reach, mass)
    free = kv.attention(q.to(cuda), cache, t[0], t[1], cu_q=t[2]).double().cpu().numpy()
    assert (np.abs(free - o) <= bound).all()


@pytest.mark.parametrize("queries,fmt,dtype", [([1, 1], "q4_0", "bf16"), ([3, 2], "q8_0", "f32"), ([70, 66], "q4_0", "f16"),
                                               ([70, 66], "q8_0", "bf16")])
def test_what_is_masked_does_not_enter(cuda, queries, fmt, dtype):
    """NaN and infinite scales in places that no query sees: past a sequence's end, before its window, in pages of nobody;
    and keys that some queries of a tile see and others must not."""
    lens, window, page = [150, 201], 40, 16
    bits = {"nan": 0x7E00, "inf": 0x7C00, "low": 0xFBFF}  # NaN, infinity, the type's lowest value

    for name, b in bits.items():
        def poison(planes, table):
            used = np.zeros(planes[0].shape[:1] + planes[0].shape[2:3], bool)
            for s, n in enumerate(lens):
                lo = max(0, n - max(queries) - window + 1)
                j = np.arange(lo, n)
                used[table[s, j // page], j % page] = True
            for scales in (planes[1], planes[3]):
                scales[np.broadcast_to(~used[:, None, :, None], scales.shape)] = b

        _check(71, fmt, dtype, lens, queries, 8, 2, 128, page, cuda, window=window, poison=poison)

    # a poisoned key that only the last query of the first sequence sees: its rows alone are not finite
    planes, table, ln, cu, q = _problem(72, fmt, dtype, lens, queries, 8, 2, 128, page)
    cu_t = None if queries == [1, 1] else torch.from_numpy(cu).to(cuda)
    args = [torch.from_numpy(x).to(cuda) for x in (table, ln)]
    clean = kv.attention(q.to(cuda), _cache(fmt, planes, cuda), *args, cu_q=cu_t, max_q=max(queries))
    for scales in (planes[1], planes[3]):
        scales[table[0, 149 // page], :, 149 % page] = 0x7E00
    got = kv.attention(q.to(cuda), _cache(fmt, planes, cuda), *args, cu_q=cu_t, max_q=max(queries))
    hit = int(cu[1]) - 1
    rest = [t for t in range(q.shape[0]) if t != hit]
    assert torch.isnan(got[hit]).all()
    assert torch.isfinite(got[rest]).all()
    assert torch.allclose(got[rest].float(), clean[rest].float(), atol=2e-3, rtol=2e-2)


def test_large_and_small_scales(cuda):
    """Values whose scales span f16, from its subnormals to 8000: no weight may overflow or vanish."""
    rng = np.random.default_rng(81)
    for dtype, queries in (("f32", 1), ("f32", 2), ("bf16", 1)):
        planes, table, lens, cu, q = _problem(82, "q4_0", dtype, [300], [queries], 4, 1, 64, 16)
        exps = rng.integers(-22, 13, planes[3].shape)
        planes[3][...] = np.ldexp(1.0, exps).astype(np.float16).view(np.uint16)
        keys, values = _gather("q4_0", planes, table, lens)
        o, l, reach, mass = ref.attention(q.float().numpy(), keys, values, lens, cu, 0.125)
        t = [torch.from_numpy(x).to(cuda) for x in (table, lens)]
        got = kv.attention(q.to(cuda), _cache("q4_0", planes, cuda), *t, scale=0.125,
                           cu_q=None if queries == 1 else torch.from_numpy(cu).to(cuda), max_q=queries)
        bound, _ = _bounds(dtype, False, False, 64, 0.0, o, reach, mass)
        assert (np.abs(got.double().cpu().numpy() - o) <= bound).all()


def test_scores_far_apart_and_large(cuda):
    """Scores of thousands (a softmax of one key), and a row of equal scores."""
    for dtype, queries in (("f32", [1]), ("bf16", [1]), ("f16", [80])):
        planes, table, lens, cu, q = _problem(91, "q4_0", dtype, [200], queries, 2, 1, 64, 16)
        keys, values = _gather("q4_0", planes, table, lens)
        t = [torch.from_numpy(x).to(cuda) for x in (table, lens)]
        cu_t = None if queries == [1] else torch.from_numpy(cu).to(cuda)
        for q_, scale in ((q, 300.0), (q * 0, 1.0)):
            o, _, reach, mass = ref.attention(q_.float().numpy(), keys, values, lens, cu, scale)
            got = kv.attention(q_.to(cuda), _cache("q4_0", planes, cuda), *t, scale=scale, cu_q=cu_t, max_q=queries[0])
            g = got.double().cpu().numpy()
            assert np.isfinite(g).all()
            if scale == 1.0:
                bound, _ = _bounds(dtype, queries != [1], False, 64, 0.0, o, reach, mass)
                assert (np.abs(g - o) <= bound).all()


def test_shared_pages_and_long_offsets(cuda):
    """Sequences that share pages; pages whose bytes lie past 2^32."""
    heads, dim, page, pages = 8, 256, 256, 8300  # 512 KB of quants a page and plane
    cache = kv.KVCache("q8_0", pages, page, heads, dim, device=cuda)
    assert cache.kq.numel() > 2**32
    x = torch.randn(400, heads, dim, device=cuda, dtype=torch.bfloat16)
    table = torch.tensor([[8299, 8250], [8299, 0]], dtype=torch.int32, device=cuda)
    t = torch.arange(400, device=cuda)
    slots = table[0].long()[t // page] * page + t % page
    kv.kv_write(cache, x, -x, slots)
    k, v = kv.kv_read(cache, slots, dtype=torch.bfloat16)
    assert torch.equal(k, -v) and (k - x).abs().max() < 0.05 * x.abs().max()
    lens = torch.tensor([400, 200], dtype=torch.int32, device=cuda)
    q = torch.randn(2, 16, dim, device=cuda, dtype=torch.bfloat16)
    got = kv.attention(q, cache, table, lens)
    kf, vf = k.double(), v.double()
    for b, n in enumerate((400, 200)):
        s = torch.einsum("hd,jhd->hj", q[b].double(), kf[:n].repeat_interleave(2, 1)) / 16
        want = torch.einsum("hj,jhd->hd", torch.softmax(s, -1), vf[:n].repeat_interleave(2, 1))
        assert (got[b].double() - want).abs().max() <= 2.0**-7 * vf.abs().max()
    big = kv.attention(q[:1].expand(130, 16, dim).contiguous(), cache, table[:1], lens[:1],
                       cu_q=torch.tensor([0, 130], dtype=torch.int32, device=cuda), max_q=130)
    assert (big[-1].double() - got[0].double()).abs().max() <= 2.0**-7 * vf.abs().max()


def test_results_repeat_bit_for_bit_and_in_graphs(cuda):
    for queries in ([1] * 5, [70, 1, 2, 0, 130]):
        planes, table, lens, cu, q = _problem(101, "q4_0", "bf16", [900, 33, 1, 64, 1500], queries, 16, 4, 128, 64)
        cache = _cache("q4_0", planes, cuda)
        t = [torch.from_numpy(x).to(cuda) for x in (table, lens)]
        kw = dict(cu_q=None if queries == [1] * 5 else torch.from_numpy(cu).to(cuda), max_q=max(queries), max_len=1500)
        qd = q.to(cuda)
        first = kv.attention(qd, cache, *t, **kw)
        for _ in range(3):
            assert torch.equal(kv.attention(qd, cache, *t, **kw), first)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = kv.attention(qd, cache, *t, **kw)
        side.synchronize()
        assert torch.equal(other, first)
        graph, buf = torch.cuda.CUDAGraph(), torch.empty_like(first)
        with torch.cuda.graph(graph):
            kv.attention(qd, cache, *t, out=buf, **kw)
        qd.neg_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(buf, kv.attention(qd, cache, *t, **kw)) and not torch.equal(buf, first)


def test_written_then_read_in_order(cuda):
    """A step's own keys are in the cache when its attention reads it, with nothing in between."""
    cache = kv.KVCache("q4_0", 8, 16, 2, 128, device=cuda)
    table = torch.arange(8, dtype=torch.int32, device=cuda)[None]
    k = torch.randn(100, 2, 128, device=cuda)
    q = torch.randn(1, 4, 128, device=cuda)
    steps = []
    for j in range(100):
        kv.kv_write(cache, k[j : j + 1], k[j : j + 1], torch.tensor([j], device=cuda))
        steps.append(kv.attention(q, cache, table, torch.tensor([j + 1], dtype=torch.int32, device=cuda)))
    kr, vr = kv.kv_read(cache, torch.arange(100, device=cuda))
    for j in (0, 1, 15, 16, 63, 64, 99):
        s = torch.einsum("hd,jhd->hj", q[0].double(), kr[: j + 1].double().repeat_interleave(2, 1)) / 128**0.5
        want = torch.einsum("hj,jhd->hd", torch.softmax(s, -1), vr[: j + 1].double().repeat_interleave(2, 1))
        assert (steps[j][0].double() - want).abs().max() < 1e-5


# ------------------------------------------------------------------------------------------------------------ refusals


def test_out_of_range_slots_and_pages_are_reported(cuda):
    _device_error()
    cache = kv.KVCache("q4_0", 2, 16, 1, 64, device=cuda)
    x = torch.randn(2, 1, 64, device=cuda)
    kv.kv_write(cache, x, x, torch.tensor([32, 5], device=cuda))  # 32 slots: the first is past the end
    assert _device_error() == 2 and cache.ks[0, 0, 5].any() and not cache.ks[1].any()
    k, _ = kv.kv_read(cache, torch.tensor([5, 10**9], device=cuda))
    assert _device_error() == 2 and k[0].any() and not k[1].any()
    q = torch.randn(1, 1, 64, device=cuda)
    # the second page is not the cache's: its tokens are masked, and the call says so; the same past the table's end
    lens = torch.tensor([20], dtype=torch.int32, device=cuda)
    want = kv.attention(q, cache, torch.tensor([[0, 1]], dtype=torch.int32, device=cuda),
                        torch.tensor([16], dtype=torch.int32, device=cuda))
    assert _device_error() == 0
    for table in ([[0, 7]], [[0, -1]], [[0]]):
        got = kv.attention(q, cache, torch.tensor(table, dtype=torch.int32, device=cuda), lens)
        assert _device_error() == 3
        assert torch.equal(got, want)
    many = torch.randn(70, 1, 64, device=cuda, dtype=torch.float16)
    got = kv.attention(many, cache, torch.tensor([[0, 7]], dtype=torch.int32, device=cuda), lens,
                       cu_q=torch.tensor([0, 70], dtype=torch.int32, device=cuda), max_q=70)
    assert _device_error() == 3 and torch.isfinite(got).all()


def test_refusals(cuda):
    c = kv.KVCache("q4_0", 4, 16, 2, 64, device=cuda)
    z = lambda *s, dtype=torch.float32: torch.zeros(*s, dtype=dtype, device=cuda)  # noqa: E731
    slots = z(3, dtype=torch.int64)
    for bad in ((z(3, 2, 96), z(3, 2, 96)), (z(3, 3, 64), z(3, 3, 64)), (z(4, 2, 64), z(4, 2, 64))):
        with pytest.raises(ValueError):
            kv.kv_write(c, *bad, slots)
    with pytest.raises(TypeError):
        kv.kv_write(c, z(3, 2, 64), z(3, 2, 64, dtype=torch.float16), slots)
    with pytest.raises(TypeError):
        kv.kv_write(c, z(3, 2, 64, dtype=torch.float64), z(3, 2, 64, dtype=torch.float64), slots)
    with pytest.raises(TypeError):
        kv.kv_write(c, z(3, 2, 64), z(3, 2, 64), slots.int())
    with pytest.raises(RuntimeError):
        kv.kv_write(c, z(3, 2, 64).cpu(), z(3, 2, 64), slots)
    with pytest.raises(RuntimeError):
        kv.kv_read(c, slots.cpu())
    with pytest.raises(TypeError):
        kv.kv_read(c, slots, dtype=torch.int8)
    q, table, lens = z(2, 4, 64), z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32)
    i32 = lambda n: z(n, dtype=torch.int32)  # noqa: E731
    kv.attention(q, c, table, lens)
    for kw, err in ((dict(q=z(2, 3, 64)), ValueError), (dict(q=z(2, 4, 128)), ValueError),
                    (dict(q=z(2, 4, 64, dtype=torch.float64)), TypeError), (dict(q=z(3, 4, 64)), ValueError),
                    (dict(table=z(2, 3, dtype=torch.int64)), TypeError), (dict(lens=z(3, dtype=torch.int32)), ValueError),
                    (dict(lens=z(2, dtype=torch.int64)), TypeError), (dict(cu_q=i32(2)), ValueError),
                    (dict(prefix=i32(3)), ValueError), (dict(starts=i32(3)), ValueError),
                    (dict(slopes=z(3)), ValueError), (dict(slopes=i32(4)), TypeError), (dict(softcap=-1.0), ValueError),
                    (dict(softcap=float("nan")), ValueError), (dict(window=-1), ValueError), (dict(scale=0.0), ValueError),
                    (dict(scale=-1.0), ValueError), (dict(out=z(2, 4, 64, dtype=torch.float16)), ValueError),
                    (dict(workspace=z(4, dtype=torch.uint8)), ValueError), (dict(q=q.cpu()), RuntimeError),
                    (dict(prefix=i32(2).cpu()), RuntimeError), (dict(q=None), RuntimeError),
                    (dict(workspace=torch.zeros(64 << 20, dtype=torch.uint8)), RuntimeError),
                    (dict(workspace=z(128 << 20, dtype=torch.uint8)[::2]), ValueError),
                    (dict(softcap=float("inf")), ValueError), (dict(softcap=1e-30), ValueError),
                    (dict(window=4.5), TypeError), (dict(scale="1"), TypeError), (dict(max_len=2.0), TypeError)):
        a = dict(q=q, table=table, lens=lens)
        a.update({k: v for k, v in kw.items() if k in a})
        rest = {k: v for k, v in kw.items() if k not in a}
        with pytest.raises(err):
            kv.attention(a["q"], c, a["table"], a["lens"], **rest)
    for bad in (dict(fmt="q4_k"), dict(head_dim=80), dict(page_size=24), dict(page_size=8), dict(heads=0)):
        a = dict(fmt="q4_0", pages=2, page_size=16, heads=2, head_dim=64) | bad
        with pytest.raises(ValueError):
            kv.KVCache(**a, device=cuda)
    with pytest.raises(ValueError):
        kv.KVCache.from_planes("q8_0", c.kq, c.ks, c.vq, c.vs)
    with pytest.raises(TypeError):
        kv.KVCache.from_planes("q4_0", c.kq, c.ks.float(), c.vq, c.vs)


@pytest.mark.parametrize("queries", [1, 70])
def test_tables_with_other_strides(cuda, queries):
    """One table row for every sequence, rows that overlap, columns of a wider table, one column: as their copies."""
    planes, _, _, _, q = _problem(91, "q4_0", "f16", [200, 150, 37], [queries] * 3, 8, 2, 64, 16)
    cache = _cache("q4_0", planes, cuda)
    q = q.to(cuda)
    lens = torch.tensor([180, 150, 72], dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, queries, 2 * queries, 3 * queries], dtype=torch.int32, device=cuda)
    row = torch.randperm(24, device=cuda).int()
    for table in (row[:12].expand(3, 12), row.as_strided((3, 12), (4, 1)), torch.stack([row, row + 1, row], 1)[:12].t(),
                  row[:3].view(1, 3).t(), row[:3].view(3, 1)):
        want = kv.attention(q, cache, table.clone(memory_format=torch.contiguous_format), lens, cu_q=cu, max_q=queries)
        _device_error()
        assert torch.equal(kv.attention(q, cache, table, lens, cu_q=cu, max_q=queries), want)
    for table in (row.view(1, 24), row.view(24, 1)[:12].t(), row.as_strided((1, 12), (0, 1)), row.as_strided((1, 12), (1, 2))):
        want = kv.attention(q[:queries], cache, table.clone(memory_format=torch.contiguous_format), lens[:1], cu_q=cu[:2])
        assert torch.equal(kv.attention(q[:queries], cache, table, lens[:1], cu_q=cu[:2]), want)
    _device_error()


@pytest.mark.parametrize("dtype,queries", [("f32", 9), ("bf16", 9), ("f16", 90)])
def test_a_window_of_all_keys_is_none(cuda, dtype, queries):
    """The largest window, with queries before the first key (more of them than keys) that see a prefix."""
    planes, table, lens, cu, q = _problem(92, "q8_0", dtype, [5, 40], [queries] * 2, 4, 2, 64, 16)
    cache = _cache("q8_0", planes, cuda)
    t = [torch.from_numpy(x).to(cuda) for x in (table, lens, cu)]
    prefix = torch.tensor([3, 3], dtype=torch.int32, device=cuda)
    a = dict(cu_q=t[2], max_q=queries, prefix=prefix)
    want = kv.attention(q.to(cuda), cache, t[0], t[1], **a)
    assert (want[0] != 0).any()
    for window in (2**31 - 1, 64):
        assert torch.equal(kv.attention(q.to(cuda), cache, t[0], t[1], window=window, **a), want)


def test_the_example_runs(cuda, capsys):
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decode_attention.py")
    spec = importlib.util.spec_from_file_location("decode_attention", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    assert m.main(["--hidden", "512", "--heads", "4", "--kv-heads", "2", "--prompt", "70", "--steps", "3"]) == 0
    assert "ok" in capsys.readouterr().out
