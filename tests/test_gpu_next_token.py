"""examples/next_token.py: norms, gated and plain 8-bit layers, the residual pass, logits and the draw
together, as a batch and as single tokens from a graph."""
import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from oracle import layers

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(ROOT, "examples"))
pytestmark = pytest.mark.gpu


def _weights(held):
    """An operand's codes [N, K] and scales."""
    K, N = held.shape
    c = held.c.cpu().numpy().reshape(-(-N // 16), -(-K // 64), 4, 16, 16).transpose(0, 3, 1, 2, 4)
    return c.reshape(c.shape[0] * 16, -1)[:N, :K], held.s.cpu().numpy()[:N]


def _product(x, w):
    """Rows of x quantized, times w: exact sums of codes, then the scales."""
    c, s = layers.q8_encode(x)
    return (c.astype(np.float64) @ w[0].astype(np.float64).T) * s.astype(np.float64)[:, None] * w[1].astype(np.float64)


@pytest.mark.parametrize("rows,width,hidden,vocab", [(1, 256, 1024, 5000), (5, 100, 333, 777), (70, 512, 776, 33000)])
def test_step(gpu, rows, width, hidden, vocab):
    """One layer and the draw against the oracle's formulas in 64 bits, each step from the values
    that the step before it stored, so that each step's own roundings bound it."""
    from next_token import EPS, Model
    m = Model(width, hidden, 1, vocab, seed=rows)
    with torch.cuda.stream(m.stream):
        b = m.buffers(rows)
        b["x"].copy_(torch.randn((rows, width), device="cuda"))
        b["u"].uniform_()
        m.step(b)
        p = m.layers[0]
        first = torch.empty_like(b["h"])
        assert m.lib.acfun_dev_norm(b["x"].data_ptr(), 1, rows, width, 0, m.first.data_ptr(), None, EPS, first.data_ptr(),
                                    m.stream.cuda_stream) == 0
        m.stream.synchronize()
    v = {k: t.double().cpu().numpy() for k, t in dict(b, f=first, first=m.first, pre=p["pre"]).items()}
    v |= {k: _weights(o) for k, o in dict(gate=p["gate"], up=p["up"], down=p["down"], head=m.head).items()}

    def near(got, want, size, half=2.0 ** -8):
        """The store's half step, and the fp32 steps between the sums and it."""
        tol = half * np.abs(want) + 40 * 2.0 ** -23 * size + 1e-30
        assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    h = layers.norm(v["x"], 0, v["first"], None, EPS)
    near(v["f"], h, np.abs(h))
    g, u = _product(v["f"], v["gate"]), _product(v["f"], v["up"])
    near(v["z"], layers.act(g, 2) * u, (np.abs(g) + np.abs(layers.act(g, 2)) + 1) * np.abs(u))
    y = _product(v["z"], v["down"])
    near(v["y"], y, np.abs(y))
    xo, h = layers.norm_residual(v["y"], v["x"], 0, None, None, None, 1, 1.0, v["pre"], None, EPS)
    near(v["r"], xo, np.abs(xo) + np.abs(v["x"]) + np.abs(xo - v["x"]))
    big = (np.abs(xo) + 2 * np.abs(v["x"])).max(1, keepdims=True) / np.sqrt((xo ** 2).mean(1, keepdims=True))
    near(v["h"], h, np.abs(h) + big * np.abs(v["pre"]))
    logits = _product(v["h"], v["head"])
    near(v["logits"], logits, np.abs(logits), 2.0 ** -24)
    for r in range(rows):
        token, prob = layers.sample(v["logits"][r], v["temp"][r], int(v["k"][r]), v["p"][r], v["m"][r], v["u"][r])
        assert v["token"][r] == token and abs(v["prob"][r] - prob) <= 2.0 ** -22 * prob


def test_command(gpu):
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "next_token.py"), "--rows", "20", "--width", "256",
                          "--hidden", "640", "--vocab", "3000"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stderr
    assert "tokens from the graph" in out.stdout
