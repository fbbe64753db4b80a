"""Layers that take two launches, but one on a stream that is being captured into a graph."""
import numpy as np
import pytest

import mx_plans

# rows, columns, K.  The last ones are the ends of what LDS holds: 16 rows of 35 pieces
# of 512 k, 8 rows of 71.
LAYERS = [(16, 4096, 4096), (8, 512, 28672), (16, 1024, 4096), (33, 200, 8000), (200, 1333, 5001), (512, 1500, 6000),
          (512, 2048, 2048), (9, 40, 17920), (17, 130, 17001), (8, 70, 36352), (5, 33, 36000)]


def test_plans(tmp_path):
    """Each of them is two launches, one when captured; past 512 rows or LDS two alone."""
    exe = mx_plans.build(tmp_path)
    for elem in (2, 4):
        for layer, got in zip(LAYERS, mx_plans.ask(exe, [mx_plans.fc(*v, elem) for v in LAYERS])):
            assert got.startswith("two/rows"), (layer, got)
        past = [(513, 2048, 2048), (16, 64, 17921), (8, 64, 36353), (600, 2000, 2000)]
        assert mx_plans.ask(exe, [mx_plans.fc(*v, elem) for v in past]) == ["two"] * 4


def test_every_layer_in_bounds(tmp_path):
    """What the header promises: one launch for N <= 512, Cin <= 17920 (36352 for N <= 8),
    Cout <= 4,000,000."""
    exe = mx_plans.build(tmp_path)
    sizes = [(M, N, K) for M in (1, 2, 3, 8, 9, 100, 512) for N in (1, 500, 9000, 300_000, 4_000_000)
             for K in (1, 1000, 9001, 17920, 36352) if K <= 17920 or M <= 8]
    for elem in (2, 4):
        for size, got in zip(sizes, mx_plans.ask(exe, [mx_plans.fc(*v, elem) for v in sizes])):
            assert "rows" in got, (size, got)


@pytest.mark.gpu
@pytest.mark.parametrize("i", range(len(LAYERS)))
def test_captured(gpu, rng, i):
    """Replays, with other inputs from one to the next and eager calls (two launches) between
    them: each against the oracle in 64 bits, and the same bits from the same input."""
    import torch

    from acfun_amd import capi
    from block_helpers import TYPES, Buf, values
    from oracle import layers
    from test_gpu_mxfp4 import _check_product, _operand
    M, N, K = LAYERS[i]
    t = list(TYPES)[i % 3]
    code, dt = TYPES[t]
    act = i % 2
    b = _operand(rng, N, K, 2)
    bv = layers.mx_decode(*b, K)
    bias = rng.standard_normal(N).astype(np.float32)
    xs = [values(torch.as_tensor(rng.standard_normal((M, K)) * np.exp(rng.standard_normal(K)) / 8).to(dt))
          for _ in range(2)]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        d = [torch.as_tensor(v).cuda() for v in layers.mx_tiles(*b)]
        tb = torch.as_tensor(bias).cuda()
        bx, out, eager = Buf((M, K), dt, xs[0], shift=i % 3), Buf((M, N), dt, shift=i % 2), Buf((M, N), dt)
        s.synchronize()

        def call(y):
            return gpu.acfun_dev_fc_mxfp4(bx.ptr, code, M, K, d[0].data_ptr(), d[1].data_ptr(), tb.data_ptr(), N,
                                          y.ptr, act, s.cuda_stream)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            rc = call(out)
        assert rc == 0, capi.last_error()
        seen = {}
        for n in range(4):
            x = xs[n % 2]
            bx.t.copy_(torch.as_tensor(x).to(dt))
            out.t.zero_()
            g.replay()
            s.synchronize()
            got = values(out.t)
            assert np.array_equal(seen.setdefault(n % 2, got), got)
            assert call(eager) == 0, capi.last_error()
            s.synchronize()
            assert out.intact() and eager.intact() and bx.intact()
            if n < 2:
                xq = layers.mx_decode(*layers.mx_encode(x), K)
                _check_product(got, xq, bv, bias, act, t)
                _check_product(values(eager.t), xq, bv, bias, act, t)
