"""The quantized KV cache and the attention that reads it, as cases to be measured and checked.

Three operators of comp_b200.kv: kv_write (keys and values into a paged cache of ggml blocks), kv_read (the values that
the cache stands for) and attention (queries against the cache: single tokens, a few tokens, prompt chunks). With `own`
false, run() computes them from elementary torch operations in 32 bits.

Cache planes, for keys and for values alike: quants uint8 [pages][heads][page][row bytes] and scales f16 (int16 bits)
[pages][heads][page][dim / 32]. A row holds the quant bytes of ggml's blocks (q4_0: 16 bytes a block, byte i = value i
in the low nibble and value i + 16 in the high one; q8_0: 32 bytes, the quant plus 128), seen as [blocks][U][unit] and
stored as [U][blocks][unit], with U = 4 for keys and 8 for values. A slot is page * page_size + offset.
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK_BYTES = {"q4_0": 16, "q8_0": 32}
K_UNITS, V_UNITS = 4, 8


def _write(name, fmt, dtype, tokens, heads, dim, page, scattered=False, skip=0, fused=False):
    return {"name": name, "op": "write", "fmt": fmt, "dtype": dtype, "tokens": tokens, "heads": heads, "dim": dim,
            "page": page, "scattered": scattered, "skip": skip, "fused": fused}


def _read(name, fmt, dtype, tokens, heads, dim, page, scattered=False, skip=0):
    return {"name": name, "op": "read", "fmt": fmt, "dtype": dtype, "tokens": tokens, "heads": heads, "dim": dim,
            "page": page, "scattered": scattered, "skip": skip}


def _attn(name, fmt, dtype, batch, lens, queries, q_heads, heads, dim, page, softcap=0.0, window=0, slopes=False,
          prefix=0, doc=0, lse=False, fused=False):
    return {"name": name, "op": "attention", "fmt": fmt, "dtype": dtype, "batch": batch, "len_min": lens[0],
            "len_max": lens[1], "q_min": queries[0], "q_max": queries[1], "q_heads": q_heads, "heads": heads,
            "dim": dim, "page": page, "softcap": softcap, "window": window, "slopes": slopes, "prefix": prefix,
            "doc": doc, "lse": lse, "fused": fused}


def listed():
    return [
        # the new token of each of 64 running sequences, cut out of the fused qkv product (8 KV heads of 128)
        _write("write_step", "q4_0", "bf16", 64, 8, 128, 64, scattered=True, fused=True),
        # a long prompt's keys and values
        _write("write_prompt", "q4_0", "bf16", 16384, 8, 128, 64),
        # f32 activations, an odd batch of chunks with padding slots, 8-bit cache in small pages
        _write("write_ragged", "q8_0", "f32", 5003, 5, 96, 16, skip=7, fused=True),
        # a stored conversation read back for a kernel that takes 16-bit keys and values
        _read("read_prefix", "q4_0", "bf16", 131072, 8, 128, 64),
        # a few scattered tokens of a small model, widened to f32
        _read("read_scattered", "q8_0", "f32", 1237, 2, 64, 16, scattered=True, skip=11),
        # one user, a middling context: latency (32 query heads on 8 KV heads of 128)
        _attn("decode_one", "q4_0", "bf16", 1, (4097, 4097), (1, 1), 32, 8, 128, 64, fused=True),
        # a served batch of unequal contexts
        _attn("decode_batch", "q4_0", "bf16", 64, (100, 8192), (1, 1), 32, 8, 128, 64),
        # long contexts, 64 query heads on 8 KV heads
        _attn("decode_long", "q4_0", "f16", 8, (90001, 131072), (1, 1), 64, 8, 128, 256, lse=True),
        # capped scores and a sliding window over an 8-bit cache with wide heads
        _attn("decode_capped", "q8_0", "bf16", 24, (1, 20000), (1, 1), 16, 8, 256, 16, softcap=50.0, window=4096),
        # drafts of up to 5 tokens checked at once, f32, distance bias, a KV head for each query head
        _attn("verify_draft", "q4_0", "f32", 16, (7, 6001), (1, 5), 12, 12, 64, 32, slopes=True, lse=True),
        # a 2048-token chunk of a 32K prompt
        _attn("chunk_prompt", "q4_0", "bf16", 1, (32768, 32768), (2048, 2048), 32, 8, 128, 64),
        # packed documents after a prefix that is seen both ways; chunks of unequal lengths
        _attn("chunk_documents", "q8_0", "f16", 6, (300, 6000), (1, 1501), 24, 4, 96, 128, softcap=30.0, prefix=200,
              doc=700, lse=True, fused=True),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    fmt = rng.choice(["q4_0", "q4_0", "q8_0"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    dim = rng.choice([64, 96, 128, 128, 256])
    page = rng.choice([16, 32, 64, 128, 256])
    heads = rng.choice([1, 2, 3, 4, 5, 8, 8, 12])
    op = rng.choice(["write", "read", "attention", "attention"])
    if op in ("write", "read"):
        tokens = log(1, min(131072, 131072 * 1024 // (heads * dim)) // (4 if op == "write" else 1))
        c = _write("", fmt, dtype, tokens, heads, dim, page, scattered=rng.random() < 0.4,
                   skip=rng.choice([0, 0, 5, 9]), fused=rng.random() < 0.5)
        if op == "read":
            c["op"] = "read"
            del c["fused"]
    else:
        group = rng.choice([1, 2, 3, 4, 4, 6, 8, 8, 16])
        kind = rng.choice(["decode", "decode", "draft", "chunk"])
        batch = log(1, 96) if kind == "decode" else log(1, 24)
        # at most 400 000 tokens of 1024 key values in the cache, and a quarter of the long chunk's products
        longest = max(64, min(131072, 400_000 * 1024 // (batch * heads * dim)))
        if kind == "chunk":
            batch = log(1, 6)
            len_max = log(64, 12000)
            most = int(6e10 / (batch * len_max * group * heads * dim))
            q_max = log(17, max(18, min(len_max, most, 2048)))
        else:
            len_max = log(16, longest)
            q_max = 1 if kind == "decode" else rng.randint(2, 8)
        len_min = log(1, len_max)
        q_min = rng.randint(1, q_max)
        c = _attn("", fmt, dtype, batch, (len_min, len_max), (q_min, q_max), heads * group, heads, dim, page,
                  softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), window=rng.choice([0, 0, 0, log(1, 4096)]),
                  slopes=rng.random() < 0.25, prefix=rng.choice([0, 0, 0, log(1, 2048)]),
                  doc=rng.choice([0, 0, 0, log(16, 2048)]), lse=rng.random() < 0.5, fused=rng.random() < 0.5)
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------


def _spread(lo, hi, n, step):
    """n whole numbers between lo and hi, both among them when n > 1, in no order."""
    f = [(i * step) % 1.0 for i in range(n)]
    if n > 1:
        f[0], f[-1] = 1.0, 0.0
    else:
        f[0] = 1.0
    return np.array([lo + int(round((hi - lo) * x)) for x in f], dtype=np.int64)


def _geometry(c):
    """Lengths, query counts, prefixes and document starts of an attention case (they follow from the case alone)."""
    lens = _spread(c["len_min"], c["len_max"], c["batch"], 0.61803398875)
    queries = np.minimum(_spread(c["q_min"], c["q_max"], c["batch"], 0.41421356237), lens)
    cu = np.zeros(c["batch"] + 1, dtype=np.int64)
    cu[1:] = np.cumsum(queries)
    seq = np.repeat(np.arange(c["batch"]), queries)
    pos = lens[seq] - queries[seq] + (np.arange(cu[-1]) - cu[seq])
    prefix = np.minimum(lens, c["prefix"]) if c["prefix"] else None
    starts = pos // c["doc"] * c["doc"] if c["doc"] else None
    if starts is not None:  # every 101st query is a padding token of no document: its row sees nothing
        starts[100::101] = lens[seq][100::101]
    return lens, queries, cu, seq, pos, prefix, starts


def _visible(c, lens, seq, pos, prefix, starts):
    """[lo, hi) of the keys that each query token sees."""
    lo = np.zeros_like(pos) if starts is None else starts.copy()
    if c["window"]:
        lo = np.maximum(lo, pos - c["window"] + 1)
    hi = pos + 1
    if prefix is not None:
        hi = np.maximum(hi, prefix[seq])
    hi = np.minimum(hi, lens[seq])
    return lo, np.maximum(hi, lo)


def _slots(c, gen, device):
    """Slots of a write or read: a shuffled run of pages filled in order, or tokens anywhere; every skip-th is -1."""
    pages = -(-c["tokens"] // c["page"]) * 5 // 4 + 1
    if c["scattered"]:
        s = torch.randperm(pages * c["page"], generator=gen, device=device)[: c["tokens"]]
    else:
        t = torch.arange(c["tokens"], device=device)
        s = torch.randperm(pages, generator=gen, device=device)[t // c["page"]] * c["page"] + t % c["page"]
    if c["skip"]:
        s[c["skip"] - 1 :: c["skip"]] = -1
    return pages, s


def _gaussian(shape, dtype, gen, device, keys=False):
    x = torch.randn(shape, generator=gen, device=device, dtype=torch.float32)
    if keys:  # keys have a few channels that are much larger than the others
        x[..., 3::37] *= 4.0
    return x.to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    c, dtype = case, DTYPES[case["dtype"]]
    s = {"case": c, "dtype": dtype}
    if c["op"] == "attention":
        lens, queries, cu, seq, pos, prefix, starts = _geometry(c)
        need = -(-lens // c["page"])
        pages = int(need.sum()) + 3
        perm = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
        first = np.concatenate([[0], np.cumsum(need)[:-1]])
        at = np.minimum(first[:, None] + np.arange(int(need.max()))[None, :], pages - 1)
        s["table"] = perm[torch.from_numpy(at).to(dev)].contiguous()
        s["lens"] = torch.from_numpy(lens.astype(np.int32)).to(dev)
        s["cu_q"] = None if int(queries.max()) == 1 else torch.from_numpy(cu.astype(np.int32)).to(dev)
        s["max_q"], s["max_len"] = int(queries.max()), int(lens.max())
        s["prefix"] = None if prefix is None else torch.from_numpy(prefix.astype(np.int32)).to(dev)
        s["starts"] = None if starts is None else torch.from_numpy(starts.astype(np.int32)).to(dev)
        s["slopes"] = None
        if c["slopes"]:
            h = torch.arange(1, c["q_heads"] + 1, device=dev, dtype=torch.float32)
            s["slopes"] = torch.exp2(-8.0 * h / c["q_heads"])
        t = int(cu[-1])
        if c["fused"]:
            s["q"] = _gaussian((t, c["q_heads"] + 2 * c["heads"], c["dim"]), dtype, gen, dev)[:, : c["q_heads"]]
        else:
            s["q"] = _gaussian((t, c["q_heads"], c["dim"]), dtype, gen, dev)
        s["scale"] = 1.0 / math.sqrt(c["dim"])
    else:
        pages, s["slots"] = _slots(c, gen, dev)
    shape = (pages, c["heads"], c["page"], c["dim"])
    if c["op"] == "write":
        wide = (c["tokens"], 3 * c["heads"], c["dim"])
        if c["fused"]:
            qkv = _gaussian(wide, dtype, gen, dev, keys=True)
            s["k"], s["v"] = qkv[:, c["heads"] : 2 * c["heads"]], qkv[:, 2 * c["heads"] :]
        else:
            s["k"] = _gaussian((c["tokens"], c["heads"], c["dim"]), dtype, gen, dev, keys=True)
            s["v"] = _gaussian((c["tokens"], c["heads"], c["dim"]), dtype, gen, dev)
        nb = c["dim"] // 32
        planes = []
        for _ in "kv":  # a cache that has been in use: whatever it held
            planes.append(torch.randint(0, 256, (*shape[:3], nb * BLOCK_BYTES[c["fmt"]]), generator=gen, device=dev,
                                        dtype=torch.uint8))
            planes.append(torch.ones((*shape[:3], nb), device=dev, dtype=torch.float16).view(torch.int16))
    else:
        planes = [*_pack(c["fmt"], _gaussian(shape, torch.float32, gen, dev, keys=True), K_UNITS),
                  *_pack(c["fmt"], _gaussian(shape, torch.float32, gen, dev), V_UNITS)]
    s["planes"] = planes
    if own:
        from comp_b200 import kv

        s["cache"] = kv.KVCache.from_planes(c["fmt"], *planes)
    return s


# ---------------------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------------------


def _pack(fmt, x, units):
    """f32 [..., dim] -> (quant bytes [..., row], f16 bits [..., dim / 32]) in the cache's layout. The 32-bit steps are
    ggml's (one division for the scale, one for its reciprocal, one product), so that the quants are ggml's."""
    b = x.unflatten(-1, (-1, 32))
    mag = b.abs()
    amax = mag.amax(-1, keepdim=True)
    if fmt == "q4_0":
        i = torch.arange(32, device=x.device)
        first = torch.where(mag == amax, i, 32).amin(-1, keepdim=True).clamp_max(31)
        d = torch.gather(b, -1, first) * -0.125
        inv = torch.where(d != 0, torch.ones_like(d) / d, torch.zeros_like(d))
        q = (b * inv + 8.5).trunc().clamp(0, 15).to(torch.uint8)
        raw = q[..., :16] | (q[..., 16:] << 4)
    else:
        d = amax / torch.full_like(amax, 127.0)
        inv = torch.where(d != 0, torch.ones_like(d) / d, torch.zeros_like(d))
        y = b * inv
        whole = y.trunc()
        q = whole + torch.where((y - whole).abs() >= 0.5, y.sign(), torch.zeros_like(y))
        raw = (q + 128.0).to(torch.uint8)
    row = raw.unflatten(-1, (units, -1)).transpose(-3, -2).flatten(-3)
    return row.contiguous(), d.squeeze(-1).to(torch.float16).contiguous().view(torch.int16)


def _unpack(fmt, quants, scales, units):
    """The values, f32 [..., dim], of planes in the cache's layout."""
    nb = scales.shape[-1]
    raw = quants.unflatten(-1, (units, nb, -1)).transpose(-3, -2).flatten(-2)
    if fmt == "q4_0":
        q = torch.cat([raw & 15, raw >> 4], -1).to(torch.float32) - 8.0
    else:
        q = raw.to(torch.float32) - 128.0
    return (q * scales.view(torch.float16).to(torch.float32).unsqueeze(-1)).flatten(-2)


def _plain_write(s):
    c, slots = s["case"], s["slots"]
    ok = slots >= 0
    # a skipped token writes what its place holds already: its own copy of the first kept token's slot
    at = torch.where(ok, slots, slots.amax())
    src = torch.where(ok, torch.arange(slots.numel(), device=slots.device), slots.argmax())
    page, off = at // c["page"], at % c["page"]
    for x, quants, scales, units in ((s["k"], *s["planes"][:2], K_UNITS), (s["v"], *s["planes"][2:], V_UNITS)):
        raw, d = _pack(c["fmt"], x.to(torch.float32)[src], units)
        quants[page, :, off] = raw
        scales[page, :, off] = d
    return _plain_read(s)


def _plain_read(s):
    c, slots = s["case"], s["slots"]
    ok = (slots >= 0)[:, None, None]
    at = slots.clamp_min(0)
    page, off = at // c["page"], at % c["page"]
    out = []
    for quants, scales, units in ((*s["planes"][:2], K_UNITS), (*s["planes"][2:], V_UNITS)):
        x = _unpack(c["fmt"], quants[page, :, off], scales[page, :, off], units)
        out.append(torch.where(ok, x, 0.0).to(s["dtype"]))
    return {"k": out[0], "v": out[1]}


def _plain_attention(s):
    c, table, lens, q = s["case"], s["table"], s["lens"].long(), s["q"].to(torch.float32)
    dev, t, group = q.device, q.shape[0], c["q_heads"] // c["heads"]
    batch, span = table.shape[0], table.shape[1] * c["page"]
    j = torch.arange(span, device=dev)
    there = (j < lens[:, None])[:, None, :, None]

    def rows(quants, scales, units):  # [batch][heads][span][dim]; nothing where the sequence has no token
        x = _unpack(c["fmt"], quants[table], scales[table], units)
        return torch.where(there, x.transpose(1, 2).flatten(2, 3), 0.0)

    # the queries of each sequence, padded to the most that one has: [batch][heads][max_q * group][dim]
    cu = s["cu_q"].long() if s["cu_q"] is not None else torch.arange(batch + 1, device=dev)
    i = torch.arange(s["max_q"], device=dev)
    n = cu[1:] - cu[:-1]
    token = (cu[:-1, None] + i).clamp_max(t - 1)
    qp = q[token].unflatten(2, (c["heads"], group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    x = torch.matmul(qp, rows(*s["planes"][:2], K_UNITS).transpose(-1, -2)) * s["scale"]
    x = x.unflatten(2, (-1, group))  # [batch][heads][max_q][group][span]
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    pos = (lens - n)[:, None] + i
    if s["slopes"] is not None:
        far = (pos[:, :, None] - j).abs().to(torch.float32)
        x = x - s["slopes"].view(1, c["heads"], 1, group, 1) * far[:, None, :, None, :]
    hi = pos + 1 if s["prefix"] is None else torch.maximum(pos + 1, s["prefix"].long()[:, None])
    lo = torch.zeros_like(pos) if s["starts"] is None else s["starts"].long()[token]
    if c["window"]:
        lo = torch.maximum(lo, pos - c["window"] + 1)
    seen = ((j >= lo[..., None]) & (j < torch.minimum(hi, lens[:, None])[..., None]))[:, None, :, None, :]
    x = torch.where(seen, x, -math.inf)
    top = x.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    w = torch.exp(x - top)
    total = w.sum(-1, keepdim=True)
    some = total > 0
    o = torch.matmul(w.flatten(2, 3), rows(*s["planes"][2:], V_UNITS)).unflatten(2, (-1, group))
    o = torch.where(some, o / total, 0.0).permute(0, 2, 1, 3, 4).flatten(2, 3)  # [batch][max_q][q_heads][dim]
    seq = torch.searchsorted(cu, torch.arange(t, device=dev), right=True) - 1
    at = torch.arange(t, device=dev) - cu[seq]
    out = {"out": o[seq, at].to(s["dtype"])}
    if c["lse"]:
        l = (torch.log(total) + top).squeeze(-1).permute(0, 2, 1, 3).flatten(2)
        out["lse"] = l[seq, at]
    return out


def run(state):
    c = state["case"]
    if not own:
        return {"write": _plain_write, "read": _plain_read, "attention": _plain_attention}[c["op"]](state)
    from comp_b200 import kv

    if c["op"] == "attention":
        got = kv.attention(state["q"], state["cache"], state["table"], state["lens"], scale=state["scale"],
                           cu_q=state["cu_q"], max_q=state["max_q"], max_len=state["max_len"], softcap=c["softcap"],
                           window=c["window"], slopes=state["slopes"], prefix=state["prefix"], starts=state["starts"],
                           return_lse=c["lse"])
        return {"out": got[0], "lse": got[1]} if c["lse"] else {"out": got}
    if c["op"] == "write":  # the cache's updated state comes back as the values that it stands for
        kv.kv_write(state["cache"], state["k"], state["v"], state["slots"])
    k, v = kv.kv_read(state["cache"], state["slots"], dtype=state["dtype"])
    return {"k": k, "v": v}


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without, and its outputs in 64 bits
# ---------------------------------------------------------------------------------------------------------------


def work(case):
    c = case
    size = DTYPES[c["dtype"]].itemsize
    token = 2 * c["heads"] * (c["dim"] // 32) * (BLOCK_BYTES[c["fmt"]] + 2)  # bytes of a token in both planes
    values = 2 * c["heads"] * c["dim"]
    if c["op"] != "attention":
        kept = c["tokens"] - (c["tokens"] // c["skip"] if c["skip"] else 0)
        out = c["tokens"] * (values * size + 8)  # the slots and the values that come back
        if c["op"] == "read":
            return {"bytes": out + kept * token, "flops": kept * values}
        return {"bytes": out + kept * (values * size + 2 * token), "flops": 4 * kept * values}
    lens, queries, cu, seq, pos, prefix, starts = _geometry(c)
    lo, hi = _visible(c, lens, seq, pos, prefix, starts)
    pairs = int((hi - lo).sum())
    read = 0
    for b in range(c["batch"]):
        m = (seq == b) & (hi > lo)
        read += int(hi[m].max() - lo[m].min()) if m.any() else 0
    io = int(cu[-1]) * c["q_heads"] * (2 * c["dim"] * size + (4 if c["lse"] else 0))
    return {"bytes": read * token + io, "flops": 4 * pairs * c["q_heads"] * c["dim"]}


def _exact_values(fmt, quants, scales, units):
    """Values of plane rows in 64 bits, each element looked up at the byte where the layout puts it."""
    nb = scales.shape[-1]
    e = np.arange(nb * 32)
    block, i = e // 32, e % 32
    byte = i % 16 if fmt == "q4_0" else i
    unit = BLOCK_BYTES[fmt] // units
    where = ((byte // unit) * nb + block) * unit + byte % unit
    dev = quants.device
    raw = quants[..., torch.from_numpy(where).to(dev)].to(torch.int16)
    if fmt == "q4_0":
        raw = (raw >> torch.from_numpy(4 * (i // 16)).to(dev, torch.int16)).bitwise_and(15) - 8
    else:
        raw = raw - 128
    d = scales.view(torch.float16).to(torch.float64)[..., torch.from_numpy(block).to(dev)]
    return raw.to(torch.float64) * d


def _exact_quantized(fmt, x):
    """What ggml's blocks of x stand for. Their quants are defined by steps in 32 bits (ties hang on them), so those
    steps are taken in 32 bits; the values are 64-bit products."""
    f = np.float32
    b = x.reshape(*x.shape[:-1], -1, 32).astype(f)
    if fmt == "q4_0":
        first = np.abs(b).argmax(-1)
        d = np.take_along_axis(b, first[..., None], -1) / f(-8)
    else:
        d = np.abs(b).max(-1, keepdims=True) / f(127)
    inv = np.divide(f(1), d, out=np.zeros_like(d), where=d != 0)
    y = b * inv
    if fmt == "q4_0":
        q = np.minimum(15, (y + f(8.5)).astype(np.int32)) - 8
    else:
        whole = np.trunc(y)
        q = whole + np.where(np.abs(y - whole) >= f(0.5), np.sign(y), f(0))
    return (q.astype(np.float64) * d.astype(np.float16).astype(np.float64)).reshape(x.shape)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "write":
        keep = (s["slots"] >= 0).cpu().numpy()[:, None, None]
        return {n: np.where(keep, _exact_quantized(c["fmt"], s[n].to(torch.float32).cpu().numpy()), 0.0) for n in "kv"}
    if c["op"] == "read":
        slots = s["slots"]
        out = {}
        for n, (quants, scales), units in (("k", s["planes"][:2], K_UNITS), ("v", s["planes"][2:], V_UNITS)):
            flat_q, flat_s = (p.transpose(1, 2).reshape(-1, c["heads"], p.shape[-1]) for p in (quants, scales))
            x = _exact_values(c["fmt"], flat_q[slots.clamp_min(0)], flat_s[slots.clamp_min(0)], units)
            x[slots < 0] = 0.0
            out[n] = x
        return out
    lens, queries, cu, seq, pos, prefix, starts = _geometry(c)
    lo, hi = _visible(c, lens, seq, pos, prefix, starts)
    group, q = c["q_heads"] // c["heads"], s["q"]
    dev = q.device
    out = torch.zeros(q.shape, dtype=torch.float64, device=dev)
    lse = torch.full(q.shape[:2], -math.inf, dtype=torch.float64, device=dev)
    step = 256  # query tokens at a time
    for b in range(c["batch"]):
        pages = s["table"][b, : -(-int(lens[b]) // c["page"])].long()
        j = torch.arange(int(lens[b]), device=dev)
        for h in range(c["heads"]):
            k, v = (_exact_values(c["fmt"], quants[pages, h], scales[pages, h], units).flatten(0, 1)[: int(lens[b])]
                    for quants, scales, units in ((*s["planes"][:2], K_UNITS), (*s["planes"][2:], V_UNITS)))
            for t0 in range(int(cu[b]), int(cu[b + 1]), step):
                t1 = min(t0 + step, int(cu[b + 1]))
                ts, heads = slice(t0, t1), slice(h * group, (h + 1) * group)
                x = torch.einsum("tgd,jd->tgj", q[ts, heads].to(torch.float64), k) * s["scale"]
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                p = torch.from_numpy(pos[ts]).to(dev)
                if s["slopes"] is not None:
                    m = s["slopes"][heads].to(torch.float64)
                    x = x - m[None, :, None] * (p[:, None] - j).abs().to(torch.float64)[:, None, :]
                a, z = (torch.from_numpy(u[ts]).to(dev)[:, None, None] for u in (lo, hi))
                x = x.masked_fill((j < a) | (j >= z), -math.inf)
                l = torch.logsumexp(x, -1)
                lse[ts, heads] = l
                w = torch.exp(x - torch.where(l > -math.inf, l, 0.0)[..., None])
                out[ts, heads] = torch.einsum("tgj,jd->tgd", w, v)
    got = {"out": out}
    if c["lse"]:
        got["lse"] = lse
    return got
