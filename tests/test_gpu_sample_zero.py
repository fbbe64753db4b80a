"""u = 0 (and what is taken to it) draws the first kept token in order of index,
however small its weight: among the first top_k, of which fewer may weigh anything at all, on the
GPU against the numpy oracle in 64 bits."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from block_helpers import TYPES, values
from oracle import layers
from test_gpu_sample import _check

pytestmark = pytest.mark.gpu

ZEROS = [0.0, -1.0, np.nan, -np.inf]


def _rows(rng, rows, cols, live, t):
    """Logits of which `live` are within 8 of the largest and the others 40 to 300 below it, one of
    these first, some ruled out."""
    x = -40 - 260 * rng.random((rows, cols))
    for r in range(rows):
        at = 1 + rng.permutation(cols - 1)
        x[r, at[live:live + cols // 4]] = (-np.inf, np.nan)[r % 2]
        x[r, at[:live]] = -8 * rng.random(live)
        x[r, at[0]] = 0
    return values(torch.as_tensor(x).to(TYPES[t][1]))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("x,k,token", [([-60, 0, -50], 2, 1), ([0, 1, 2, 60, 100], 2, 3), ([-60, -50, 0, -70], 3, 0),
                                       ([-60, -60, 0, -60], 2, 0), ([-60, -50, -60, 0], 2, 1)])
def test_few_tokens(gpu, t, x, k, token):
    x = np.tile(np.array(x, np.float64), (4, 1))
    tok = _check(gpu, x, t, np.array(ZEROS), k=np.full(4, k))
    assert (tok == token).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols,live", [(9, 2), (300, 5), (3000, 1), (3000, 40), (20000, 7), (40000, 1), (40000, 300)])
def test_top_k_past_what_weighs(gpu, rng, cols, live, t):
    """One past the tokens that weigh something, some, most of the row; with min_p below and among
    the small weights, and with a nucleus, which ends before them."""
    x, u = _rows(rng, 4, cols, live, t), np.array(ZEROS)
    full = lambda v: np.full(4, v)  # noqa: E731
    for k in sorted({live, live + 1, live + 2, (live + cols) // 2, cols - cols // 4 - 1, cols - 1}):
        _check(gpu, x, t, u, k=full(k))
        _check(gpu, x, t, u, k=full(k), m=full(1e-30), ld=cols + 5)
        _check(gpu, x, t, u, k=full(k), p=full(0.99))
        _check(gpu, x, t, u, k=full(k), T=full(0.3))
        _check(gpu, x, t, u, k=full(k), T=full(20.0))
    _check(gpu, x, t, u, m=full(1e-30))
    _check(gpu, x, t, u)


@pytest.mark.parametrize("cols", [3000, 40000])
def test_captured(gpu, rng, cols):
    """The same from a replayed graph, which has no parts of a row."""
    x, u, k = _rows(rng, 4, cols, 9, "f32"), np.array(ZEROS), [10, 15, cols // 2, cols - 1]
    want = [layers.sample(x[r], k=k[r], u=0.0)[0] for r in range(4)]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        dx, du = torch.as_tensor(x, dtype=torch.float32).cuda(), torch.as_tensor(u, dtype=torch.float32).cuda()
        dk, tok = torch.tensor(k, dtype=torch.int32).cuda(), torch.zeros(4, dtype=torch.int32, device="cuda")

        def call():
            assert gpu.acfun_dev_sample(dx.data_ptr(), 0, 4, cols, cols, None, dk.data_ptr(), None, None, du.data_ptr(),
                                        tok.data_ptr(), None, s.cuda_stream) == 0, capi.last_error()
        call()
        s.synchronize()
        assert list(tok.cpu().numpy()) == want
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
        for i in range(3):
            tok.fill_(-7)
            g.replay()
            s.synchronize()
            assert list(tok.cpu().numpy()) == want, i
