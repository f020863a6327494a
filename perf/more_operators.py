"""A layer of experts on 4-bit microscaled floats (MXFP4), operator by operator, as cases to be measured and checked.

Five operators: quantize (f32 / f16 / bf16 rows to MXFP4 and the values that these stand for), linear (rows quantized and
multiplied with MXFP4 weights), route (the k largest logits of each token, their softmax weights, and the tokens sorted by
expert), experts (each expert's rows quantized and multiplied with that expert's weights, in sorted order) and combine
(rows brought back to their tokens, weighted and added). With `own` false, run() computes them from elementary torch
operations in 32 bits.

MXFP4: 32 values along K share a scale 2^(s - 127), s one byte: s = max(0, floor(log2 of the largest magnitude) + 125), 255
(NaN) where a value is not finite. A value divided by the scale is rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to
the one whose code is even) and cut off at 6; its code is 3 bits of magnitude and a sign. Planes: codes uint8 [rows][K / 2], byte i
of a block = value i in the low nibble and value i + 16 in the high one; scales uint8 [rows][K / 32].
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _quantize(name, dtype, rows, k, strided=False):
    return {"name": name, "op": "quantize", "dtype": dtype, "rows": rows, "k": k, "strided": strided}


def _linear(name, dtype, out, rows, n, k, strided=False):
    return {"name": name, "op": "linear", "dtype": dtype, "out": out, "rows": rows, "n": n, "k": k, "strided": strided}


def _route(name, dtype, tokens, experts, top, normalize=True, masked=0):
    return {"name": name, "op": "route", "dtype": dtype, "tokens": tokens, "experts": experts, "top": top,
            "normalize": normalize, "masked": masked}


def _experts(name, dtype, out, tokens, experts, top, n, k, gather=True):
    return {"name": name, "op": "experts", "dtype": dtype, "out": out, "tokens": tokens, "experts": experts, "top": top,
            "n": n, "k": k, "gather": gather}


def _combine(name, dtype, tokens, experts, top, n, skip=0):
    return {"name": name, "op": "combine", "dtype": dtype, "tokens": tokens, "experts": experts, "top": top, "n": n,
            "skip": skip}


def listed():
    return [
        # the hidden states of 64 running sequences
        _quantize("quantize_step", "bf16", 64, 4096),
        # a long prompt's hidden states
        _quantize("quantize_prompt", "bf16", 16384, 8192),
        # one user's next token through a square projection: latency
        _linear("linear_one", "bf16", "bf16", 1, 8192, 8192),
        # an odd batch and an odd layer, f32 in and out, rows cut out of a wider product
        _linear("linear_odd", "f32", "f32", 37, 5003, 2080, strided=True),
        # a prompt chunk through an up projection
        _linear("linear_prompt", "bf16", "bf16", 4096, 14336, 4096),
        # routing one step of 64 sequences
        _route("route_step", "f32", 64, 128, 8),
        # routing a prompt, some experts masked out, weights of the softmax over all experts
        _route("route_prompt", "bf16", 16384, 256, 8, normalize=False, masked=9),
        # one token and its 8 experts
        _experts("experts_one", "bf16", "bf16", 1, 64, 8, 2048, 4096),
        # the second product of a served batch: rows in sorted order, odd sizes
        _experts("experts_down", "f16", "f32", 61, 40, 6, 4096, 1440, gather=False),
        # a prompt chunk through 32 experts
        _experts("experts_prompt", "bf16", "bf16", 4096, 32, 4, 4096, 4096),
        # one step's rows back to their tokens
        _combine("combine_step", "f32", 64, 128, 8, 4096, skip=5),
        # a prompt's rows back to their tokens
        _combine("combine_prompt", "bf16", 8192, 64, 8, 4096),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    out = rng.choice(["bf16", "f16", "f32"])
    op = rng.choice(["quantize", "linear", "linear", "route", "experts", "experts", "combine"])
    k = 32 * log(2, 256)
    if op == "quantize":
        size = 2 if dtype == "f32" else 1
        c = _quantize("", dtype, log(1, min(60000, 16384 * 8192 // (k * size))), k, strided=rng.random() < 0.4)
    elif op == "linear":
        n = log(64, 16384)
        c = _linear("", dtype, out, log(1, min(8192, max(1, int(1.2e11 / (n * k))))), n, k, strided=rng.random() < 0.4)
    elif op == "route":
        experts = log(4, 512)
        c = _route("", dtype, log(1, 16384 * 256 // max(256, experts)), experts, rng.randint(1, min(10, experts)),
                   normalize=rng.random() < 0.6, masked=rng.choice([0, 0, rng.randint(1, experts // 2)]))
    elif op == "experts":
        experts = log(2, 160)
        n = log(64, 5000)
        k = 32 * log(2, max(2, min(256, 5 * 10**8 // (experts * n * 32))))
        top = rng.randint(1, min(8, experts))
        c = _experts("", dtype, out, log(1, min(4096, max(1, int(1.2e11 / (n * k * top))))), experts, top, n, k,
                     gather=rng.random() < 0.6)
    else:
        experts, n = log(2, 256), log(64, 8192)
        top = rng.randint(1, min(10, experts))
        c = _combine("", dtype, log(1, min(16384, 10**8 // (n * top))), experts, top, n, skip=rng.choice([0, 0, 3, 7]))
    del c["name"]
    return c


# ---------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------


def _choices(c):
    """Experts of each token, int64 [tokens][top], all different within a token: popular experts and rare ones (how many
    experts have tokens follows from the case alone)."""
    rng = np.random.default_rng(c["tokens"] * 1000 + c["experts"] * 10 + c["top"])
    pull = rng.standard_normal((c["tokens"], c["experts"])) + 0.7 * rng.standard_normal(c["experts"])
    return np.argpartition(-pull, c["top"] - 1, axis=1)[:, : c["top"]]


def _activations(rows, k, dtype, gen, dev, strided=False):
    """Hidden states: a few channels much larger than the others, tokens of different size."""
    x = torch.randn((rows, k), generator=gen, device=dev, dtype=torch.float32)
    x[:, 5::67] *= 12.0
    x *= torch.exp(0.5 * torch.randn((rows, 1), generator=gen, device=dev))
    x = x.to(dtype)
    if strided:  # the middle columns of a product that made more than these
        wide = torch.zeros((rows, k + 96), dtype=dtype, device=dev)
        wide[:, 32 : 32 + k] = x
        x = wide[:, 32 : 32 + k]
    return x


def _weights(lead, n, k, gen, dev):
    codes, scales = [], []
    for _ in range(lead):
        w = torch.randn((n, k), generator=gen, device=dev, dtype=torch.float32) * k**-0.5
        q, s = _to_mx(w)
        codes.append(q)
        scales.append(s)
    return torch.stack(codes), torch.stack(scales)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    c, dtype = case, DTYPES[case["dtype"]]
    s = {"case": c, "dtype": dtype}
    if c["op"] in ("experts", "combine"):
        # the seed says which experts are the popular ones and which tokens take them
        label = torch.randperm(c["experts"], generator=gen, device=dev)
        token = torch.randperm(c["tokens"], generator=gen, device=dev)
        ids = label[torch.from_numpy(_choices(c)).to(dev)][token].to(torch.int32)
        if c["op"] == "combine" and c["skip"]:  # choices that another machine holds
            ids.view(-1)[c["skip"] - 1 :: c["skip"]] = -1
        s["ids"] = ids.contiguous()
    if c["op"] == "quantize":
        s["x"] = _activations(c["rows"], c["k"], dtype, gen, dev, c["strided"])
    elif c["op"] == "linear":
        s["x"] = _activations(c["rows"], c["k"], dtype, gen, dev, c["strided"])
        codes, scales = _weights(1, c["n"], c["k"], gen, dev)
        s["codes"], s["scales"] = codes[0], scales[0]
    elif c["op"] == "route":
        x = torch.randn((c["tokens"], c["experts"]), generator=gen, device=dev) * 2.0
        x = x + torch.randn((c["experts"],), generator=gen, device=dev)
        if c["masked"]:  # experts that are not to be had
            x[:, torch.randperm(c["experts"], generator=gen, device=dev)[: c["masked"]]] = -math.inf
        s["logits"] = x.to(dtype)
    elif c["op"] == "experts":
        rows = c["tokens"] if c["gather"] else c["tokens"] * c["top"]
        s["x"] = _activations(rows, c["k"], dtype, gen, dev)
        s["codes"], s["scales"] = _weights(c["experts"], c["n"], c["k"], gen, dev)
    else:
        s["y"] = torch.randn((c["tokens"] * c["top"], c["n"]), generator=gen, device=dev).to(dtype)
        w = torch.rand((c["tokens"], c["top"]), generator=gen, device=dev) + 0.05
        s["weights"] = w / w.sum(-1, keepdim=True)
    if own:
        from comp_b200 import experts, mx

        if "codes" in s:
            s["w"] = mx.pack(s["codes"], s["scales"])
        if "ids" in s:
            s["plan"] = experts.sort(s["ids"], c["experts"])
    return s


# ---------------------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------------------


def _power(s):
    """2^(s - 127) as f32, NaN for 255, from s (int32)."""
    bits = torch.where(s > 0, s << 23, 1 << 22)
    return torch.where(s < 255, bits.view(torch.float32), math.nan)


def _to_mx(x):
    """f32 [rows][k] -> (codes uint8 [rows][k / 2], scales uint8 [rows][k / 32])."""
    b = x.unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    s = ((amax.view(torch.int32) >> 23) - 2).clamp_min(0)
    up = ((254 - s) << 23).view(torch.float32)
    a = torch.where(bad[..., None], 0.0, b.abs() * up[..., None])
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp_max(6.0)
    # magnitudes to codes: 0, .5, 1, 1.5, 2 are twice themselves, then 3, 4, 6 follow
    code = torch.where(a <= 2, a * 2, torch.where(a < 4, a + 2, a * 0.5 + 4)).to(torch.uint8)
    code = code | (torch.signbit(b).to(torch.uint8) << 3)
    s = torch.where(bad, 255, s)
    return (code[..., :16] | (code[..., 16:] << 4)).flatten(-2), s.to(torch.uint8)


def _from_mx(codes, scales):
    """The values, f32 [..., k]."""
    raw = codes.unflatten(-1, (-1, 16))
    code = torch.cat([raw & 15, raw >> 4], -1).to(torch.int64)
    table = torch.tensor([*MAGNITUDES, *(-m for m in MAGNITUDES)], device=codes.device)
    return (table[code] * _power(scales.to(torch.int32))[..., None]).flatten(-2)


def _rounded(x):
    return _from_mx(*_to_mx(x.to(torch.float32)))


def _sorted(ids, experts):
    """(offsets [experts + 1], pos [tokens][top], order [tokens * top]) of choices sorted by expert; -1: no place, no row."""
    flat = ids.flatten().to(torch.int64)
    key = torch.where(flat >= 0, flat, experts)
    order = torch.sort(key, stable=True).indices
    counts = (key[:, None] == torch.arange(experts, device=ids.device)).sum(0) if key.numel() * experts < 1 << 26 else \
        torch.bincount(key, minlength=experts + 1)[:experts]
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=ids.device)
    pos = torch.where(flat >= 0, place, -1).view(ids.shape)
    order = torch.where(torch.arange(order.numel(), device=ids.device) < offsets[-1], order, -1)
    return offsets.to(torch.int32), pos.to(torch.int32), order.to(torch.int32)


def _plain_route(s):
    c = s["case"]
    x = s["logits"].to(torch.float32) + 0.0
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = torch.sort(x, dim=-1, descending=True, stable=True)
    vals, ids = top.values[:, : c["top"]], top.indices[:, : c["top"]]
    some = vals > -math.inf
    ids = torch.where(some, ids, -1).to(torch.int32)

    def e(v):  # the largest is exp(0), infinities too
        return torch.where(v == vals[:, :1], 1.0, torch.exp(v - vals[:, :1]))

    total = torch.where(some, e(vals), 0.0).sum(-1, keepdim=True) if c["normalize"] else \
        torch.where(x > -math.inf, e(x), 0.0).sum(-1, keepdim=True)
    offsets, pos, order = _sorted(ids, c["experts"])
    return {"ids": ids, "weights": torch.where(some, e(vals) / total, 0.0), "offsets": offsets, "pos": pos, "order": order}


def _plain_experts(s):
    c = s["case"]
    offsets, _, order = _sorted(s["ids"], c["experts"])
    x = _rounded(s["x"])
    y = torch.empty((order.numel(), c["n"]), dtype=DTYPES[c["out"]], device=x.device)
    at = offsets.tolist()
    for e in range(c["experts"]):
        if at[e + 1] > at[e]:
            rows = slice(at[e], at[e + 1])
            xe = x[order[rows].long() // c["top"]] if c["gather"] else x[rows]
            y[rows] = torch.matmul(xe, _from_mx(s["codes"][e], s["scales"][e]).T).to(y.dtype)
    return y


def _plain_combine(s):
    c = s["case"]
    _, pos, _ = _sorted(s["ids"], c["experts"])
    out = torch.zeros((c["tokens"], c["n"]), dtype=torch.float32, device=pos.device)
    for j in range(c["top"]):
        p = pos[:, j].long()
        row = s["y"][p.clamp_min(0)].to(torch.float32) * s["weights"][:, j, None]
        out += torch.where((p >= 0)[:, None], row, 0.0)
    return out.to(s["dtype"])


def run(state):
    c, s = state["case"], state
    if not own:
        if c["op"] == "quantize":
            return _rounded(s["x"]).to(s["dtype"])
        if c["op"] == "linear":
            return torch.matmul(_rounded(s["x"]), _from_mx(s["codes"], s["scales"]).T).to(DTYPES[c["out"]])
        return {"route": _plain_route, "experts": _plain_experts, "combine": _plain_combine}[c["op"]](s)
    from comp_b200 import experts, mx

    if c["op"] == "quantize":  # what is held in 4 bits comes back as the values that it stands for
        return mx.dequantize(mx.quantize(s["x"]), s["dtype"])
    if c["op"] == "linear":
        return mx.linear(s["x"], s["w"], dtype=DTYPES[c["out"]])
    if c["op"] == "route":
        p = experts.route(s["logits"], c["top"], normalize=c["normalize"])
        return {"ids": p.ids, "weights": p.weights, "offsets": p.offsets, "pos": p.pos, "order": p.order}
    if c["op"] == "experts":
        return experts.linear(s["x"], s["w"], s["plan"], gather=c["gather"], dtype=DTYPES[c["out"]])
    return experts.combine(s["y"], s["plan"], s["weights"])


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without, and its outputs in 64 bits
# ---------------------------------------------------------------------------------------------------------------


def work(case):
    c = case
    size = DTYPES[c["dtype"]].itemsize
    if c["op"] == "quantize":  # the values in, the blocks written and read, the values that come back
        return {"bytes": c["rows"] * c["k"] * 2 * size + c["rows"] * c["k"] // 32 * 17 * 2, "flops": 4 * c["rows"] * c["k"]}
    if c["op"] == "linear":
        weights = c["n"] * c["k"] // 32 * 17
        return {"bytes": weights + c["rows"] * (c["k"] * size + c["n"] * DTYPES[c["out"]].itemsize),
                "flops": 2 * c["rows"] * c["n"] * c["k"]}
    pairs = c["tokens"] * c["top"]
    if c["op"] == "route":
        return {"bytes": c["tokens"] * c["experts"] * size + pairs * 16 + (c["experts"] + 1) * 4,
                "flops": 4 * c["tokens"] * c["experts"]}
    if c["op"] == "experts":
        used = len(np.unique(_choices(c)))
        rows = c["tokens"] if c["gather"] else pairs
        return {"bytes": used * c["n"] * c["k"] // 32 * 17 + rows * c["k"] * size + pairs * 4 +
                pairs * c["n"] * DTYPES[c["out"]].itemsize, "flops": 2 * pairs * c["n"] * c["k"]}
    kept = pairs - (pairs // c["skip"] if c["skip"] else 0)
    return {"bytes": kept * c["n"] * size + pairs * 8 + c["tokens"] * c["n"] * size, "flops": 2 * kept * c["n"]}


def _exact_mx(x):
    """What the MXFP4 blocks of x stand for, by its definition, in 64 bits: each value to the nearest magnitude, found
    between the midpoints; a midpoint itself goes to the magnitude whose code is even."""
    b = x.to(torch.float64).unflatten(-1, (-1, 32))
    amax = b.abs().amax(-1, keepdim=True)
    _, ex = torch.frexp(amax)  # amax = m 2^ex with m in [0.5, 1)
    ex = torch.where(amax > 0, ex - 3, -127).clamp_min(-127).to(torch.float64)
    a = b.abs() / torch.exp2(ex)
    val = torch.zeros_like(a)
    for i in range(1, 8):
        mid = (MAGNITUDES[i] + MAGNITUDES[i - 1]) / 2
        val = torch.where(a >= mid if i % 2 == 0 else a > mid, MAGNITUDES[i], val)
    val = val * torch.exp2(ex) * torch.sign(b)
    return torch.where(torch.isfinite(b).all(-1, keepdim=True), val, math.nan).flatten(-2)


def _exact_weights(codes, scales):
    """Values of planes in 64 bits, each looked up at the nibble where the layout puts it."""
    i = torch.arange(codes.shape[-1] * 2, device=codes.device)
    byte = codes[..., i // 32 * 16 + i % 16].to(torch.int32)
    code = torch.where(i % 32 < 16, byte & 15, byte >> 4)
    m, e = (code & 1).to(torch.float64), (code >> 1) & 3  # one bit of mantissa, two of exponent
    mag = torch.where(e > 0, (1 + m / 2) * torch.exp2(e.to(torch.float64) - 1), m / 2)
    return torch.where(code >= 8, -mag, mag) * torch.exp2(scales[..., i // 32].to(torch.float64) - 127)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quantize":
        return torch.cat([_exact_mx(x) for x in s["x"].split(2048)]).cpu()
    if c["op"] == "linear":
        w = _exact_weights(s["codes"], s["scales"])
        return torch.cat([_exact_mx(x) @ w.T for x in s["x"].split(1024)]).cpu()
    if c["op"] == "route":
        x = s["logits"].to(torch.float64).cpu().numpy()
        x = np.where(np.isnan(x), -np.inf, x)
        ids = np.argsort(-x, axis=1, kind="stable")[:, : c["top"]]
        vals = np.take_along_axis(x, ids, 1)
        d = np.exp(vals - vals[:, :1])
        total = d.sum(1, keepdims=True) if c["normalize"] else np.exp(x - vals[:, :1]).sum(1, keepdims=True)
        ids = np.where(vals > -np.inf, ids, -1)
        key = np.where(ids.ravel() >= 0, ids.ravel(), c["experts"])
        order = np.argsort(key, kind="stable")
        pos = np.empty(key.size, dtype=np.int64)
        pos[order] = np.arange(key.size)
        offsets = np.searchsorted(key[order], np.arange(c["experts"] + 1))
        return {"ids": ids, "weights": d / total, "offsets": offsets,
                "pos": np.where(ids.ravel() >= 0, pos, -1).reshape(ids.shape),
                "order": np.where(np.arange(key.size) < offsets[-1], order, -1)}
    flat = s["ids"].cpu().numpy().ravel()
    key = np.where(flat >= 0, flat, c["experts"])
    order = np.argsort(key, kind="stable")
    dev = s["ids"].device
    if c["op"] == "experts":
        y = torch.empty((flat.size, c["n"]), dtype=torch.float64, device=dev)
        for e in np.unique(flat):
            rows = np.flatnonzero(key[order] == e)
            src = order[rows] // c["top"] if c["gather"] else rows
            w = _exact_weights(s["codes"][e], s["scales"][e])
            y[torch.from_numpy(rows).to(dev)] = _exact_mx(s["x"][torch.from_numpy(src).to(dev)]) @ w.T
        return y.cpu()
    pos = np.empty(flat.size, dtype=np.int64)
    pos[order] = np.arange(flat.size)
    pos = pos.reshape(s["ids"].shape)
    out = torch.zeros((c["tokens"], c["n"]), dtype=torch.float64, device=dev)
    for j in range(c["top"]):
        p = torch.from_numpy(pos[:, j]).to(dev)
        t = torch.nonzero(s["ids"][:, j] >= 0).flatten()
        out[t] += s["y"][p[t]].to(torch.float64) * s["weights"][t, j, None].to(torch.float64)
    return out.cpu()
