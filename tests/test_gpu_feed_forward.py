"""examples/feed_forward.py: norms, 4-bit layers and the residual pass together, a prompt
and single tokens from a graph."""
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


@pytest.mark.parametrize("rows,width,hidden", [(1, 256, 1024), (5, 100, 333), (70, 512, 777)])
def test_layer(gpu, rows, width, hidden):
    """One layer against the oracle's formulas in 64 bits, each step from the bf16 values
    that the step before it stored, so that each step's own roundings bound it."""
    from feed_forward import EPS, FeedForward
    m = FeedForward(width, hidden, 1, seed=rows)
    with torch.cuda.stream(m.stream):
        x = torch.randn((rows, width), device="cuda").bfloat16()
        b = m.buffers(rows)
        m.run(x, b)
        p = m.layers[0]
        up, down = (p[n].values(m.lib, m.stream.cuda_stream) for n in ("up", "down"))
        first = torch.empty_like(b["h"])
        assert m.lib.acfun_dev_norm(x.data_ptr(), 1, rows, width, 0, m.first.data_ptr(), None, EPS,
                                    first.data_ptr(), m.stream.cuda_stream) == 0
        m.stream.synchronize()
    v = {k: t.double().cpu().numpy() for k, t in dict(xi=x, f=first, up=up, down=down, w=m.first, z=b["z"], y=b["y"],
                                                      xo=b["x"], h=b["h"]).items()}
    q = {k: p[k].double().cpu().numpy() for k in ("bias", "post", "pre", "gate")}

    def near(got, want, size):
        """The store's half step of bf16, and a fp32 sum's error: K / 32 + 4 steps of 2^-23."""
        tol = 2.0 ** -8 * np.abs(want) + (max(width, hidden) / 32 + 40) * 2.0 ** -23 * size * (1 + 2.0 ** -8) + 1e-30
        assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)

    def quantized(a):
        return layers.mx_decode(*layers.mx_encode(a), a.shape[1])
    h = layers.norm(v["xi"], 0, v["w"], None, EPS)
    near(v["f"], h, np.abs(h))
    a = quantized(v["f"])
    near(v["z"], np.maximum(a @ v["up"].T + q["bias"], 0), np.abs(a) @ np.abs(v["up"]).T + np.abs(q["bias"]))
    a = quantized(v["z"])
    near(v["y"], a @ v["down"].T, np.abs(a) @ np.abs(v["down"]).T)
    xo, h = layers.norm_residual(v["y"], v["xi"], 0, q["post"], None, q["gate"], rows, 1.0, q["pre"], None, EPS)
    near(v["xo"], xo, np.abs(xo) + np.abs(v["xi"]) + np.abs(xo - v["xi"]))
    big = (np.abs(xo) + 2 * np.abs(v["xi"])).max(1, keepdims=True) / np.sqrt((xo ** 2).mean(1, keepdims=True))
    near(v["h"], h, np.abs(h) + big * np.abs(q["pre"]))


def test_command(gpu):
    out = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "feed_forward.py"), "--rows", "48",
                          "--width", "256", "--hidden", "640"], capture_output=True, text=True, timeout=100)
    assert out.returncode == 0, out.stderr
    assert "token" in out.stdout
