"""Feed-forward layers of a token model with 8-bit weights, and the draw of its next token:

    h = norm(x);  for each layer:  z = silu(Wg h) * (Wu h);  y = Wd z
                                   x, h = norm_residual(y, x)
    token = a draw from the logits Wv h at a temperature, with top-k, top-p and min-p

Every product is of 8-bit integers with a scale for each token and for each channel.  Runs a batch
of prompts' last tokens, then single tokens from a captured graph, each fed back through an
embedding, and says how far the logits are from the same layers in fp32 with the weights as
the 8-bit codes give them.

    python examples/next_token.py [--rows 64] [--width 1024] [--hidden 4096] [--layers 2] [--vocab 32000]
"""
import argparse
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from acfun_amd import capi  # noqa: E402

BF16, F32, RMSNORM, SILU = 1, 0, 0, 2
EPS = 1e-5


def _ok(rc):
    if rc != 0:
        raise RuntimeError(capi.last_error())


class Held:
    """An operand in Q8: weights [K, N] become one of N rows."""

    def __init__(self, lib, w, stream):
        K, N = w.shape
        self.c = torch.empty(lib.acfun_q8_code_bytes(N, K), dtype=torch.int8, device="cuda")
        self.s = torch.empty(lib.acfun_q8_scale_bytes(N) // 4, dtype=torch.float32, device="cuda")
        _ok(lib.acfun_dev_quantize_q8(w.data_ptr(), F32, N, K, 1, self.c.data_ptr(), self.s.data_ptr(), stream))
        self.shape, self.ptr = (K, N), (self.c.data_ptr(), self.s.data_ptr())

    def values(self, lib, stream):
        K, N = self.shape
        w = torch.empty((N, K), device="cuda")
        _ok(lib.acfun_dev_dequantize_q8(*self.ptr, N, K, w.data_ptr(), F32, stream))
        return w


class Model:
    def __init__(self, width, hidden, layers, vocab, seed=0):
        self.lib, self.stream = capi.lib(), torch.cuda.Stream()
        self.width, self.hidden, self.vocab = width, hidden, vocab
        g = torch.Generator(device="cuda").manual_seed(seed)
        normal = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
        with torch.cuda.stream(self.stream):
            g.manual_seed(seed)
            hold = lambda k, n: Held(self.lib, normal(k, n) * k ** -0.5, self.stream.cuda_stream)  # noqa: E731
            self.embed, self.first = normal(vocab, width).bfloat16(), 1 + 0.1 * normal(width)
            self.layers = [dict(gate=hold(width, hidden), up=hold(width, hidden), down=hold(hidden, width),
                                pre=1 + 0.1 * normal(width)) for _ in range(layers)]
            self.head = hold(width, vocab)
            self.stream.synchronize()

    def buffers(self, rows):
        """Everything a step of `rows` tokens reads and writes; kept by the caller for a graph."""
        new = lambda *shape, t=torch.bfloat16: torch.zeros(shape, dtype=t, device="cuda")  # noqa: E731
        f, i = torch.float32, torch.int32
        return dict(x=new(rows, self.width), r=new(rows, self.width), h=new(rows, self.width), y=new(rows, self.width),
                    z=new(rows, self.hidden), logits=new(rows, self.vocab, t=f), token=new(rows, t=i), prob=new(rows, t=f),
                    u=new(rows, t=f), temp=new(rows, t=f) + 0.8, k=new(rows, t=i) + 50, p=new(rows, t=f) + 0.95,
                    m=new(rows, t=f) + 0.02)

    def step(self, b):
        """The next tokens of b["x"]'s rows, in b["token"]."""
        L, s, rows, W, H = self.lib, self.stream.cuda_stream, b["x"].shape[0], self.width, self.hidden
        p = {n: t.data_ptr() for n, t in b.items()}
        _ok(L.acfun_dev_norm(p["x"], BF16, rows, W, RMSNORM, self.first.data_ptr(), None, EPS, p["h"], s))
        x = p["x"]
        for v in self.layers:
            _ok(L.acfun_dev_fc_gated_q8(p["h"], BF16, rows, W, *v["gate"].ptr, None, *v["up"].ptr, None, H, p["z"], SILU, s))
            _ok(L.acfun_dev_fc_q8(p["z"], BF16, rows, H, *v["down"].ptr, None, W, p["y"], 0, s))
            _ok(L.acfun_dev_norm_residual(p["y"], x, BF16, rows, W, RMSNORM, None, None, None, 1, 1.0, v["pre"].data_ptr(),
                                          None, EPS, p["r"], p["h"], s))
            x = p["r"]
        # (logits in fp32, of bf16 rows: quantized once, multiplied as an operand)
        K, N = self.head.shape
        if "hc" not in b:
            b["hc"] = torch.empty(L.acfun_q8_code_bytes(rows, K), dtype=torch.int8, device="cuda")
            b["hs"] = torch.empty(L.acfun_q8_scale_bytes(rows) // 4, dtype=torch.float32, device="cuda")
        hc, hs = b["hc"].data_ptr(), b["hs"].data_ptr()
        _ok(L.acfun_dev_quantize_q8(p["h"], BF16, rows, K, 0, hc, hs, s))
        _ok(L.acfun_dev_gemm_q8(rows, N, K, hc, hs, *self.head.ptr, p["logits"], F32, None, 0, s))
        _ok(L.acfun_dev_sample(p["logits"], F32, rows, N, N, p["temp"], p["k"], p["p"], p["m"], p["u"], p["token"],
                               p["prob"], s))

    def plain(self, x):
        """The logits in fp32, from the weights' 8-bit values and activations as they are."""
        s, x = self.stream.cuda_stream, x.float()
        norm = lambda v: v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS)  # noqa: E731
        with torch.cuda.stream(self.stream):
            h = norm(x) * self.first
            for v in self.layers:
                g, u, d = (v[n].values(self.lib, s) for n in ("gate", "up", "down"))
                x = x + norm(torch.nn.functional.silu(h @ g.t()) * (h @ u.t()) @ d.t())
                h = norm(x) * v["pre"]
            return h @ self.head.values(self.lib, s).t()


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("rows", 64), ("width", 1024), ("hidden", 4096), ("layers", 2), ("vocab", 32000)):
        ap.add_argument("--" + name, type=int, default=value)
    a = ap.parse_args()
    m = Model(a.width, a.hidden, a.layers, a.vocab)
    with torch.cuda.stream(m.stream):
        b, one = m.buffers(a.rows), m.buffers(1)
        b["x"].copy_(m.embed[torch.randint(a.vocab, (a.rows,), device="cuda")])
        b["u"].uniform_()
        m.step(b)
        want = m.plain(b["x"])
        off = ((b["logits"] - want).norm() / want.norm()).item()
        print(f"{a.rows} rows: logits {off:.3f} from fp32 activations (8-bit ones are about 0.01 off each product)")
        m.step(one)
        m.stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=m.stream):
            m.step(one)
        tokens = []
        for _ in range(8):
            one["u"].uniform_()
            graph.replay()
            one["x"].copy_(m.embed[one["token"].long()])
            tokens.append(one["token"].item())
        print("tokens from the graph:", *tokens)
        for name, f in (("batch", lambda: m.step(b)), ("token", graph.replay)):
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
