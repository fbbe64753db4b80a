"""The feed-forward half of transformer layers with 4-bit weights:

    h = norm(x);  for each layer:  y = W2 relu(W1 h + b1)
                                   x, h = norm_residual(y, x)

norm_residual is the layer's norm after the block, its gate, the residual sum and
the next layer's norm in one pass.  Runs a prompt through the layers, then tokens one
by one from a captured graph, and says how far the results are from the same
layers in fp32 with the weights as the 4-bit codes give them.

    python examples/feed_forward.py [--rows 512] [--width 1024] [--hidden 4096] [--layers 2]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from acfun_amd import capi  # noqa: E402

BF16, F32, RMSNORM = 1, 0, 0
EPS = 1e-5


class Held:
    """An operand in MXFP4: weights [K, N] become one of N rows."""

    def __init__(self, lib, w, stream):
        K, N = w.shape
        self.c = torch.empty(lib.acfun_mxfp4_code_bytes(N, K), dtype=torch.uint8, device="cuda")
        self.s = torch.empty(lib.acfun_mxfp4_scale_bytes(N, K), dtype=torch.uint8, device="cuda")
        _ok(lib.acfun_dev_quantize_mxfp4(w.data_ptr(), F32, N, K, 1, self.c.data_ptr(),
                                         self.s.data_ptr(), stream))
        self.shape = (K, N)

    def values(self, lib, stream):
        K, N = self.shape
        w = torch.empty((N, K), device="cuda")
        _ok(lib.acfun_dev_dequantize_mxfp4(self.c.data_ptr(), self.s.data_ptr(), N, K, w.data_ptr(), F32,
                                           stream))
        return w


def _ok(rc):
    if rc != 0:
        raise RuntimeError(capi.last_error())


class FeedForward:
    def __init__(self, width, hidden, layers, seed=0):
        self.lib, self.stream = capi.lib(), torch.cuda.Stream()
        self.width, self.hidden = width, hidden
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
        with torch.cuda.stream(self.stream):
            s = self.stream.cuda_stream
            g.manual_seed(seed)
            self.first = 1 + 0.1 * normal(width)
            self.layers = []
            for _ in range(layers):
                up, down = normal(width, hidden) * width ** -0.5, normal(hidden, width) * hidden ** -0.5
                self.layers.append(dict(
                    up=Held(self.lib, up, s), down=Held(self.lib, down, s), bias=0.1 * normal(hidden),
                    post=1 + 0.1 * normal(width), pre=1 + 0.1 * normal(width),
                    gate=normal(1, width).bfloat16()))
            self.stream.synchronize()

    def buffers(self, rows):
        """Everything a pass over `rows` rows writes; kept by the caller for a graph."""
        new = lambda cols: torch.empty((rows, cols), dtype=torch.bfloat16, device="cuda")  # noqa: E731
        return dict(h=new(self.width), x=new(self.width), y=new(self.width), z=new(self.hidden))

    def run(self, x, b):
        """x [rows, width] (bf16) through the layers; the last norm's result in b["h"]."""
        L, s, rows, W, H = self.lib, self.stream.cuda_stream, x.shape[0], self.width, self.hidden
        _ok(L.acfun_dev_norm(x.data_ptr(), BF16, rows, W, RMSNORM, self.first.data_ptr(), None, EPS,
                             b["h"].data_ptr(), s))
        for p in self.layers:
            up, down = p["up"], p["down"]
            _ok(L.acfun_dev_fc_mxfp4(b["h"].data_ptr(), BF16, rows, W, up.c.data_ptr(), up.s.data_ptr(),
                                     p["bias"].data_ptr(), H, b["z"].data_ptr(), 1, s))
            _ok(L.acfun_dev_fc_mxfp4(b["z"].data_ptr(), BF16, rows, H, down.c.data_ptr(), down.s.data_ptr(),
                                     None, W, b["y"].data_ptr(), 0, s))
            _ok(L.acfun_dev_norm_residual(b["y"].data_ptr(), x.data_ptr(), BF16, rows, W, RMSNORM,
                                          p["post"].data_ptr(), None, p["gate"].data_ptr(), rows, 1.0,
                                          p["pre"].data_ptr(), None, EPS, b["x"].data_ptr(),
                                          b["h"].data_ptr(), s))
            x = b["x"]
        return b["h"]

    def plain(self, x):
        """The same in fp32, from the weights' 4-bit values and activations as they are."""
        s, x = self.stream.cuda_stream, x.float()
        norm = lambda v, w: v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS) * w  # noqa: E731
        with torch.cuda.stream(self.stream):
            h = norm(x, self.first)
            for p in self.layers:
                up, down = p["up"].values(self.lib, s), p["down"].values(self.lib, s)
                y = (h @ up.t() + p["bias"]).relu() @ down.t()
                x = x + p["gate"].float() * norm(y, p["post"])
                h = norm(x, p["pre"])
        return h


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--rows", type=int, default=512)
    ap.add_argument("--width", type=int, default=1024)
    ap.add_argument("--hidden", type=int, default=4096)
    ap.add_argument("--layers", type=int, default=2)
    a = ap.parse_args()
    m = FeedForward(a.width, a.hidden, a.layers)
    with torch.cuda.stream(m.stream):
        x = torch.randn((a.rows, a.width), device="cuda").bfloat16()
        b, token = m.buffers(a.rows), m.buffers(1)
        h, want = m.run(x, b).float(), m.plain(x)
        one = x[:1].clone()
        m.run(one, token)
        m.stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=m.stream):
            m.run(one, token)
        graph.replay()
        m.stream.synchronize()
        off = ((h - want).norm() / want.norm()).item()
        print(f"prompt of {a.rows}: {off:.3f} from fp32 activations (4-bit ones are about 0.1 off each layer)")
        print(f"one token from the graph: {(token['h'].float() - h[:1]).abs().max().item():.3g} from the "
              "prompt's first row")
        for name, f in (("prompt", lambda: m.run(x, b)), ("token", graph.replay)):
            for _ in range(20):
                f()
            m.stream.synchronize()
            t = time.perf_counter()
            for _ in range(200):
                f()
            m.stream.synchronize()
            print(f"{name}: {(time.perf_counter() - t) / 200 * 1e6:.1f} us")


if __name__ == "__main__":
    main()
