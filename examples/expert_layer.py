"""The feed-forward part of a decoding model: a router and experts on MXFP4 weights.

A prompt's tokens are taken in at once, then tokens one by one. For each: the router's logits choose experts
(comp_b200.experts), their gate and up products run on the tokens sorted by expert, and the down products come back weighted
and added. The last token's output is checked against 64-bit torch operations on the values that the weights stand for,
with the layer's own rounding of activations (comp_b200.mx).

    python examples/expert_layer.py [--hidden 2048] [--inner 768] [--experts 64] [--top 8] [--prompt 300] [--steps 10]
"""

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from comp_b200 import experts, mx  # noqa: E402


class Layer:
    def __init__(self, hidden, inner, count, top, dev, seed=0):
        gen = torch.Generator(device=dev).manual_seed(seed)

        def weights(*shape):
            return torch.randn(shape, generator=gen, device=dev) * shape[-1] ** -0.5

        self.inner, self.top = inner, top
        self.router = weights(count, hidden)
        self.up = mx.quantize(weights(count, 2 * inner, hidden))  # gate and up, one under the other
        self.down = mx.quantize(weights(count, hidden, inner))

    def __call__(self, x):
        """x f32 [n][hidden] -> the same shape."""
        plan = experts.route(x @ self.router.T, self.top)
        gate, up = experts.linear(x, self.up, plan).chunk(2, dim=-1)
        rows = experts.linear(torch.nn.functional.silu(gate) * up, self.down, plan, gather=False)
        return experts.combine(rows, plan, plan.weights)

    def check(self, x, y):
        """The error of one token's output, relative to its size."""
        plan = experts.route(x @ self.router.T, self.top)
        want = torch.zeros_like(y, dtype=torch.float64)
        for e, w in zip(plan.ids[0].tolist(), plan.weights[0].double()):
            h = mx.dequantize(mx.quantize(x)).double() @ self.values(self.up, e).T
            a = (torch.nn.functional.silu(h[:, : self.inner].float()) * h[:, self.inner :].float()).contiguous()
            want += w * (mx.dequantize(mx.quantize(a)).double() @ self.values(self.down, e).T)
        return float((y.double() - want).abs().max() / want.abs().max())

    @staticmethod
    def values(w, e):
        size = mx.image_bytes(w.rows, w.k)
        return mx.dequantize(mx.MXTensor(w.image[e * size : (e + 1) * size], w.rows, w.k)).double()


def main(argv=None):
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--hidden", type=int, default=2048)
    ap.add_argument("--inner", type=int, default=768)
    ap.add_argument("--experts", type=int, default=64)
    ap.add_argument("--top", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=300)
    ap.add_argument("--steps", type=int, default=10)
    a = ap.parse_args(argv)
    if not torch.cuda.is_available():
        print("needs a CUDA GPU", file=sys.stderr)
        return 2
    dev = torch.device("cuda", torch.cuda.current_device())
    layer = Layer(a.hidden, a.inner, a.experts, a.top, dev)
    x = torch.randn(a.prompt, a.hidden, device=dev, generator=torch.Generator(device=dev).manual_seed(1))
    y = layer(x)
    worst = layer.check(x[-1:], y[-1:])
    for _ in range(a.steps):
        x = torch.nn.functional.normalize(y[-1:], dim=-1) * a.hidden**0.5
        y = layer(x)
        worst = max(worst, layer.check(x, y))
    # an activation next to the border of two 4-bit values may fall to either side: one step of one of `inner` values
    ok = worst < 0.02 and bool(torch.isfinite(y).all())
    print(f"{'ok  ' if ok else 'FAIL'} {a.prompt} prompt tokens and {a.steps} steps through {a.experts} experts, "
          f"{(layer.up.nbytes + layer.down.nbytes) / 1e6:.1f} MB of weights: within {worst:.1e} of 64-bit arithmetic")
    return 0 if ok else 1


if __name__ == "__main__":
    sys.exit(main())
