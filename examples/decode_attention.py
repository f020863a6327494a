"""An attention block of a decoding model on Q4_0 weights and a quantized KV cache.

A prompt is taken in as one chunk, then tokens one by one. For each: the fused qkv product and the output product are
Q4_0 GEMVs (comp_b200.host), the new keys and values are quantized into the cache, and the queries attend to it
(comp_b200.kv). After each step the last token's attention is checked against plain 64-bit torch operations on the values
that the cache stands for.

    python examples/decode_attention.py [--hidden 4096] [--heads 32] [--kv-heads 8] [--prompt 500] [--steps 20]
                                        [--cache q4_0|q8_0]
"""

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from comp_b200 import host, kv  # noqa: E402


def random_q4_0(n, k, rng, dev):
    """Q4_0 planes of an n x k layer of random blocks whose products keep the size of what they are given."""
    wq = rng.integers(0, 256, (n, k // 2), dtype=np.uint8)
    d = np.abs(rng.normal(0, 0.2 / np.sqrt(k), (n, k // 32))).astype(np.float16)
    return torch.from_numpy(wq).to(dev), torch.from_numpy(d.view(np.int16)).to(dev)


class Block:
    def __init__(self, hidden, heads, kv_heads, dim, cache, tokens, dev, seed=0):
        rng = np.random.default_rng(seed)
        self.hidden, self.heads, self.kv_heads, self.dim, self.dev = hidden, heads, kv_heads, dim, dev
        self.n_qkv = (heads + 2 * kv_heads) * dim
        self.qkv = random_q4_0(self.n_qkv, hidden, rng, dev)
        self.out = random_q4_0(hidden, heads * dim, rng, dev)
        page = 64
        pages = -(-tokens // page)
        self.cache = kv.KVCache(cache, pages, page, kv_heads, dim, device=dev)
        # any order of pages will do: a server hands them out as they become free
        self.table = torch.from_numpy(rng.permutation(pages).astype(np.int32)).to(dev)[None]
        self.page, self.length = page, 0

    def slots(self, n):
        t = torch.arange(self.length, self.length + n, device=self.dev)
        return self.table[0].long()[t // self.page] * self.page + t % self.page

    def step(self, x):
        """x f32 [n][hidden], the next n tokens -> f32 [n][hidden]."""
        n = x.shape[0]
        qkv = host.quant_gemv("q4_0", *self.qkv, x, self.n_qkv, self.hidden).view(n, -1, self.dim)
        q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], dim=1)
        kv.kv_write(self.cache, k, v, self.slots(n))
        self.length += n
        lens = torch.tensor([self.length], dtype=torch.int32, device=self.dev)
        cu = None if n == 1 else torch.tensor([0, n], dtype=torch.int32, device=self.dev)
        o = kv.attention(q, self.cache, self.table, lens, cu_q=cu, max_q=n)
        return host.quant_gemv("q4_0", *self.out, o.view(n, -1), self.hidden, self.heads * self.dim), q, o

    def check(self, q, o):
        """The largest error of the last token's attention, relative to its size."""
        t = torch.arange(self.length, device=self.dev)
        slots = self.table[0].long()[t // self.page] * self.page + t % self.page
        k, v = (x.double().repeat_interleave(self.heads // self.kv_heads, 1) for x in kv.kv_read(self.cache, slots))
        w = torch.softmax(torch.einsum("hd,jhd->hj", q[-1].double(), k) * self.dim**-0.5, -1)
        want = torch.einsum("hj,jhd->hd", w, v)
        return float((o[-1].double() - want).abs().max() / want.abs().max())


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--heads", type=int, default=32)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--head-dim", type=int, default=128)
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--cache", choices=kv.FORMATS, default="q4_0")
    a = ap.parse_args(argv)
    if not torch.cuda.is_available():
        print("needs a CUDA GPU", file=sys.stderr)
        return 2
    dev = torch.device("cuda", torch.cuda.current_device())
    block = Block(a.hidden, a.heads, a.kv_heads, a.head_dim, a.cache, a.prompt + a.steps, dev)
    gen = torch.Generator(device=dev).manual_seed(1)
    y, q, o = block.step(torch.randn(a.prompt, a.hidden, device=dev, generator=gen))
    worst = block.check(q, o)
    for _ in range(a.steps):
        x = torch.nn.functional.normalize(y[-1:], dim=-1) * a.hidden**0.5
        y, q, o = block.step(x)
        worst = max(worst, block.check(q, o))
    ok = worst < 1e-5 and bool(torch.isfinite(y).all())
    print(f"{'ok  ' if ok else 'FAIL'} {a.prompt} prompt tokens and {a.steps} steps over a {a.cache} cache of "
          f"{block.cache.nbytes / 1e6:.1f} MB: attention within {worst:.1e} of 64-bit arithmetic")
    return 0 if ok else 1


if __name__ == "__main__":
    sys.exit(main())
