"""Rows of up to 2^24 columns, the most that a call takes: many small weights, none of which is lost,
on the GPU against sums in extended precision."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from block_helpers import TYPES, values
from oracle import layers
from test_gpu_sample import _check, _logits, _sample

pytestmark = pytest.mark.gpu


def _off(cols):
    """How far a row's shares may be off: half a step of 2^-48 for each weight, of a sum that is 1 at
    least, and twice the exponential's 2^-39.8 (of the sum and of a part)."""
    return cols * 2.0 ** -49 + 2.0 ** -38.8


def _share(x, keep, T=1.0):
    """The kept weights' sums up to and with each token, as parts of all, extended precision."""
    w = np.where(keep, np.exp((x.astype(np.longdouble) - x.max()) / np.longdouble(T)), np.longdouble(0))
    c = np.cumsum(w)
    return w / c[-1], c / c[-1]


def _near(tok, prob, u, w, c, cols):
    """The token of u, or of a number that is _off() from it at most."""
    for r in range(len(u)):
        i = int(tok[r])
        assert c[i] + _off(cols) >= u[r] and c[i] - w[i] - _off(cols) <= u[r], (r, i, u[r], c[i], w[i])
        assert abs(prob[r] - w[i]) <= w[i] * (2.0 ** -24 + _off(cols)) + 2.0 ** -150, (r, prob[r], w[i])


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols,gap", [(1 << 24, 27.5), (1 << 24, 27.0), ((1 << 24) - 5, 20.0), ((1 << 22) + 3, 30.0),
                                      ((1 << 19) + 1, 31.0), (1 << 24, 0.0)])
def test_flat_tail(gpu, t, cols, gap):
    """One token `gap` above all others, last in order of index: each of the others has a small part
    of the sum, all of them up to an even one."""
    x = np.zeros((1, cols), np.float32)
    x[0, -1] = gap
    w, c = _share(x[0], np.ones(cols, bool))
    tail = float(c[-2])
    u = np.float32(np.array([1e-3, 0.1, 0.5, 0.9, 0.999]) * tail)
    u = np.concatenate([u, np.float32([0.25, 0.5, 1 - 2.0 ** -24])])
    for v in u:
        tok, prob = _sample(gpu, x, t, np.array([v]))
        _near(tok, prob, [float(v)], w, c, cols)
    k = cols // 3                                            # the first k in order: the last and k - 1 others
    w, c = _share(x[0], (np.arange(cols) < k - (gap > 0)) | ((np.arange(cols) == cols - 1) & (gap > 0)))
    for v in u[:4]:
        tok, prob = _sample(gpu, x, t, np.array([v]), k=np.array([k]))
        _near(tok, prob, [float(v)], w, c, cols)


@pytest.mark.parametrize("cols", [(1 << 19) + 1, (1 << 20) + 3])
def test_filters(gpu, rng, cols):
    rows = 4
    x, u = _logits(rng, rows, cols, "f32"), rng.random(rows)
    x[1, rng.integers(0, cols, cols)] = -np.inf
    x[2, rng.integers(0, cols, cols)] = np.nan
    T, k = np.array([0.5, 1.0, 1.5, 1e-3]), np.array([0, 50, 3000, cols // 2])
    p, m = np.array([0.9, 0.999, 1.0, 0.5]), np.array([0.0, 0.01, 0.0, 0.2])
    _check(gpu, x, "f32", u)
    _check(gpu, x, "f32", u, T=T, p=p)
    _check(gpu, x, "f32", u, k=k)
    _check(gpu, x, "f32", u, T, k, p, m, ld=cols + 3)
    _check(gpu, x, "f32", np.zeros(rows), k=k)
    _check(gpu, x, "f32", u, T=np.zeros(rows))


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_one_workgroup(gpu, rng, t):
    """More rows than are split, and a captured call: a workgroup to a row gives the same tokens."""
    cols, rows = (1 << 19) + 8, 260
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.Generator(device="cuda").manual_seed(5)
        x = (torch.randn((rows, cols), generator=g, device="cuda") * 2.5).to(TYPES[t][1])
        x[::2, 1:] -= 25.0                                   # (a tail of small weights under the first)
        x[::2, 0] = 12.0
        u = torch.rand(rows, generator=g, device="cuda")
        u[::4] *= 1e-4
        p = torch.full((rows,), 0.9999, device="cuda")
        k = torch.full((rows,), 400000, dtype=torch.int32, device="cuda")

        def call(first, n, top_k, top_p):
            tok, prob = torch.full((n,), -7, dtype=torch.int32, device="cuda"), torch.zeros(n, device="cuda")
            rc = gpu.acfun_dev_sample(x[first:].data_ptr(), TYPES[t][0], n, cols, cols, None,
                                      k[first:].data_ptr() if top_k else None, p[first:].data_ptr() if top_p else None, None,
                                      u[first:].data_ptr(), tok.data_ptr(), prob.data_ptr(), s.cuda_stream)
            assert rc == 0, capi.last_error()
            return tok, prob
        for top_k, top_p in ((False, False), (True, False), (False, True), (True, True)):
            tok, prob = call(0, rows, top_k, top_p)
            for r in (0, 1, 4, 131, rows - 2):
                one = call(r, 2 if r < rows - 2 else 1, top_k, top_p)       # split
                s.synchronize()
                assert one[0][0] == tok[r] and one[1][0] == prob[r], (r, top_k, top_p)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            held = call(0, 3, True, True)
        want = call(0, 3, True, True)
        for i in range(3):
            held[0].fill_(-7)
            graph.replay()
            s.synchronize()
            assert torch.equal(held[0], want[0]) and torch.equal(held[1], want[1]), i
        for r in (0, 1, 2, 4):
            got = call(r, 1, False, False)
            s.synchronize()
            w, c = _share(values(x[r]), np.ones(cols, bool))
            _near(got[0].cpu().numpy(), values(got[1]), [float(u[r])], w, c, cols)
            tok, _ = layers.sample(values(x[r]), u=float(u[r]))
            assert abs(c[tok] - c[int(got[0][0])]) <= 2 * _off(cols) + w[tok]
