"""MXFP4 quantizer and products on the GPU against the numpy oracle in 64 bits
(oracle/layers.py): the quantizer byte for byte, the products within the rounding
of their 32-bit sums."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from block_helpers import TYPES, Buf, half_step, smallest, values
from oracle import layers

pytestmark = pytest.mark.gpu


def _quantize(gpu, x, t, trans=False, shift=0):
    """(codes, scales) as numpy bytes of x [rows, K] (trans: given as [K, rows])."""
    code, dt = TYPES[t]
    rows, K = x.shape[::-1] if trans else x.shape
    nc, ns = gpu.acfun_mxfp4_code_bytes(rows, K), gpu.acfun_mxfp4_scale_bytes(rows, K)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx = Buf(x.shape, dt, x, shift)
        c, sc = Buf((nc,), torch.uint8), Buf((ns,), torch.uint8)
        rc = gpu.acfun_dev_quantize_mxfp4(bx.ptr, code, rows, K, int(trans), c.ptr, sc.ptr,
                                          s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    assert c.intact() and sc.intact() and bx.intact()
    return c, sc


def _check_bytes(c, sc, x):
    code, byte = layers.mx_encode(x)
    wc, ws = layers.mx_tiles(code, byte)
    gc, gs = c.t.cpu().numpy(), sc.t.cpu().numpy()
    assert np.array_equal(gs, ws)
    if (byte == 255).any():                                  # their codes are unspecified
        keep, _ = layers.mx_tiles(np.where(np.repeat(byte == 255, 32, 1), 0, 15).astype(np.uint8), byte)
        pad, _ = layers.mx_tiles(np.full_like(code, 15), byte)
        keep |= ~pad
        gc, wc = gc & keep, wc & keep
    assert np.array_equal(gc, wc)


ROWS_K = [(1, 1), (1, 32), (2, 31), (3, 33), (15, 127), (16, 128), (17, 129), (33, 500), (5, 512),
          (64, 513), (100, 1000), (1, 4096), (130, 2048), (31, 4100)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("rows,K", ROWS_K)
def test_quantize_bytes(gpu, rng, rows, K, trans, t):
    x = rng.standard_normal((rows, K)) * np.exp(rng.standard_normal((rows, 1)) * 3)
    x[:, rng.integers(0, K)] *= 30
    x = values(torch.as_tensor(x).to(TYPES[t][1]))           # the type's values
    c, sc = _quantize(gpu, x.T.copy() if trans else x, t, trans, shift=rows % 3)
    _check_bytes(c, sc, x)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("t", TYPES)
def test_quantize_edges(gpu, t, trans):
    """Every tie and its neighbours at every scale the type has, zeros of both signs,
    subnormals, the largest values, NaN and infinities."""
    dt = TYPES[t][1]
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, 7.9, 0, 0.5, 1, 1.5, 2, 3])
    v = torch.tensor(np.concatenate([ties, -ties])).to(dt).double().numpy()
    lo, hi = {"f32": (-149, 125), "bf16": (-133, 125), "f16": (-24, 13)}[t]
    rows = []
    for e in range(lo, hi + 1):
        a = torch.tensor(np.ldexp(v, e)).to(dt)
        rows.append(a.double().numpy())
        bits = a.view(torch.int32 if t == "f32" else torch.int16)
        for d in (-1, 1):                                    # the neighbours in the type
            n = torch.where(a == 0, bits, bits + d).view(dt).double().numpy()
            n[7] = rows[-1][7]
            rows.append(np.where(np.isfinite(n), n, 0))
    big = float(torch.finfo(dt).max)
    for special in (np.nan, np.inf, -np.inf, big, -big, float(torch.finfo(dt).tiny)):
        r = v.copy() if t != "f16" else v / 4
        r[11] = special
        rows.append(r)
    rows += [np.zeros(32), -np.zeros(32)]
    x = np.array(rows)
    x = np.concatenate([x, x[::-1], x], 1)                   # neighbours of a bad block are not touched
    x = values(torch.as_tensor(x).to(dt))
    c, sc = _quantize(gpu, x.T.copy() if trans else x, t, trans)
    _check_bytes(c, sc, x)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,K", ROWS_K)
def test_dequantize(gpu, rng, rows, K, t):
    code = rng.integers(0, 16, (rows, -(-K // 32) * 32)).astype(np.uint8)
    byte = rng.integers(0, 255, (rows, code.shape[1] // 32)).astype(np.uint8)
    byte[0, 0] = 255
    wc, ws = layers.mx_tiles(code, byte)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c, sc = torch.as_tensor(wc).cuda(), torch.as_tensor(ws).cuda()
        out = Buf((rows, K), TYPES[t][1], shift=K % 3)
        rc = gpu.acfun_dev_dequantize_mxfp4(c.data_ptr(), sc.data_ptr(), rows, K, out.ptr, TYPES[t][0],
                                            s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    want = torch.as_tensor(layers.mx_decode(code, byte, K)).to(TYPES[t][1]).double().numpy()
    got = values(out.t)
    assert out.intact()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(np.nan_to_num(got, posinf=1e300), np.nan_to_num(want, posinf=1e300))


def _operand(rng, rows, K, spread=6):
    code = rng.integers(0, 16, (rows, -(-K // 32) * 32)).astype(np.uint8)
    code[:, K:] = 0
    byte = rng.integers(127 - spread, 128 + spread, (rows, code.shape[1] // 32)).astype(np.uint8)
    return code, byte


def _check_product(got, a, b, bias, act, t):
    """One rounding for each block of 32 products and its addition (the matrix unit
    may truncate: a whole step of 2^-23 of the sum of magnitudes), the bias, the
    store."""
    K = a.shape[1]
    with np.errstate(invalid="ignore"):
        want = a @ b.T
        size = np.abs(a) @ np.abs(b).T
        if bias is not None:
            want, size = want + bias, size + np.abs(bias)
        if act:
            want = np.where(want > 0, want, 0.0 * np.nan_to_num(want))
    tol = (-(-K // 32) + 4) * 2.0 ** -23 * size + 2.0 ** -126 * (K + 1)
    tol = tol + half_step(t) * (np.abs(want) + tol) + smallest(t)
    bad = np.isnan(size)
    assert not np.isnan(got[~bad]).any()
    assert (np.abs(got - want)[~bad] <= tol[~bad]).all(), np.max((np.abs(got - want) / tol)[~bad])
    return bad


def _gemm(gpu, a, b, bias, act, t, M, N, K, stream=None):
    s = stream or torch.cuda.Stream()
    with torch.cuda.stream(s):
        d = [torch.as_tensor(v).cuda() for v in (*layers.mx_tiles(*a), *layers.mx_tiles(*b))]
        tb = None if bias is None else torch.as_tensor(bias, dtype=torch.float32).cuda()
        out = Buf((M, N), TYPES[t][1], shift=N % 2)
        rc = gpu.acfun_dev_gemm_mxfp4(M, N, K, *(v.data_ptr() for v in d), out.ptr, TYPES[t][0],
                                      None if tb is None else tb.data_ptr(), act, s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    assert out.intact()
    return values(out.t)


SHAPES = [(1, 1, 1), (1, 16, 128), (3, 5, 33), (16, 16, 512), (17, 33, 129), (1, 4096, 4096), (2, 777, 513),
          (13, 2048, 1000), (16, 100, 8192), (33, 515, 640), (64, 100, 2048), (40, 1000, 513), (128, 256, 1024),
          (128, 2048, 4096), (257, 130, 2000), (300, 511, 96), (512, 512, 512), (513, 769, 1153),
          (1000, 2500, 300), (2048, 2048, 256), (1025, 4097, 640)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm(gpu, rng, M, N, K, t):
    a, b = _operand(rng, M, K), _operand(rng, N, K)
    bias = rng.standard_normal(N).astype(np.float32) if (M + N) % 2 else None
    act = int(K % 3 == 0)
    if t == "f16":                                           # sums within half precision's range
        a = (a[0], np.minimum(a[1], 124) - 12)
    got = _gemm(gpu, a, b, bias, act, t, M, N, K)
    _check_product(got, layers.mx_decode(*a, K), layers.mx_decode(*b, K), bias, act, t)


@pytest.mark.parametrize("M,N,K", [(512, 2048, 4096), (512, 1111, 700), (1000, 600, 2048), (500, 2000, 4000)])
def test_gemm_middle(gpu, rng, M, N, K):
    a, b = _operand(rng, M, K), _operand(rng, N, K)
    bias = rng.standard_normal(N).astype(np.float32)
    got = _gemm(gpu, a, b, bias, 1, "bf16", M, N, K)
    _check_product(got, layers.mx_decode(*a, K), layers.mx_decode(*b, K), bias, 1, "bf16")


@pytest.mark.parametrize("t,M,N,K", [("f32", 3600, 4100, 200), ("bf16", 3585, 4097, 1), ("f16", 4096, 4096, 513),
                                     ("bf16", 20000, 1000, 700)])
def test_gemm_large(gpu, rng, M, N, K, t):
    """The largest tiles, whole and cut at both edges."""
    a, b = _operand(rng, M, K, 3), _operand(rng, N, K, 3)
    bias = rng.standard_normal(N).astype(np.float32)
    got = _gemm(gpu, a, b, bias, 0, t, M, N, K)
    _check_product(got, layers.mx_decode(*a, K), layers.mx_decode(*b, K), bias, 0, t)


@pytest.mark.parametrize("M,N,K", [(1, 48, 512), (20, 100, 1000), (300, 600, 640)])
def test_gemm_bad_blocks(gpu, rng, M, N, K):
    """A NaN block makes its row (or column) of C NaN and nothing else."""
    a, b = _operand(rng, M, K), _operand(rng, N, K)
    a[1][M // 2, -1] = 255
    b[1][N // 3, 0] = 255
    got = _gemm(gpu, a, b, None, 0, "f32", M, N, K)
    bad = _check_product(got, layers.mx_decode(*a, K), layers.mx_decode(*b, K), None, 0, "f32")
    want = np.zeros((M, N), bool)
    want[M // 2], want[:, N // 3] = True, True
    assert np.array_equal(bad, want) and np.array_equal(np.isnan(got), want)


@pytest.mark.parametrize("M,N,K", [(3, 40, 100), (1000, 2500, 300)])
def test_gemm_relu_nan(gpu, rng, M, N, K):
    """ReLU keeps NaN, as the product without it gives it."""
    a, b = _operand(rng, M, K), _operand(rng, N, K)
    a[1][M // 2, 0] = 255
    got = _gemm(gpu, a, b, None, 1, "f32", M, N, K)
    want = np.zeros((M, N), bool)
    want[M // 2] = True
    assert np.array_equal(np.isnan(got), want) and (got[~want] >= 0).all()


@pytest.mark.parametrize("M,N", [(1, 7), (40, 300), (300, 300)])
def test_gemm_no_k(gpu, rng, M, N):
    """K = 0: the bias alone; no operand is read."""
    bias = rng.standard_normal(N).astype(np.float32)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        tb, out = torch.as_tensor(bias).cuda(), Buf((M, N), torch.float32)
        assert gpu.acfun_dev_gemm_mxfp4(M, N, 0, None, None, None, None, out.ptr, 0, tb.data_ptr(), 1,
                                        s.cuda_stream) == 0, capi.last_error()
        s.synchronize()
        assert out.intact()
        assert np.array_equal(values(out.t), np.tile(np.maximum(bias, 0).astype(np.float64), (M, 1)))
        assert gpu.acfun_dev_fc_mxfp4(None, 0, M, 0, None, None, None, N, out.ptr, 0, s.cuda_stream) == 0
        s.synchronize()
        assert (values(out.t) == 0).all()


FC = [(1, 64, 32), (1, 4096, 4096), (2, 130, 1), (7, 100, 1000), (16, 2053, 777), (17, 300, 4096), (33, 64, 130),
      (100, 999, 513), (333, 2053, 1000), (600, 700, 2048), (1, 10, 8192), (5, 3000, 31)]


# rows quantized in the product's launch (tiles of 16, 32 and 64 columns, K that is
# whole pieces of 512, that ends between lanes and inside one) and in one before it
FC_MORE = [(1, 8192, 512), (128, 2048, 512), (33, 2053, 1000), (16, 64, 1024), (4, 40, 20000), (130, 2100, 510),
           (17, 3000, 520), (20, 300, 16), (64, 4100, 1536), (5, 8200, 2047), (16, 200, 8192), (300, 900, 3000),
           (1, 30, 40000), (2, 30, 33000), (3, 50, 20000), (8, 40, 17000), (16, 40, 17408), (7, 600, 1500)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", FC + FC_MORE)
def test_fc(gpu, rng, M, N, K, t):
    code, dt = TYPES[t]
    x = values(torch.as_tensor(rng.standard_normal((M, K)) * np.exp(rng.standard_normal(K))).to(dt))
    b = _operand(rng, N, K, 2)
    bias = rng.standard_normal(N).astype(np.float32) if M % 2 else None
    act = int(N % 2)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx = Buf((M, K), dt, x, shift=M % 3)
        d = [torch.as_tensor(v).cuda() for v in layers.mx_tiles(*b)]
        tb = None if bias is None else torch.as_tensor(bias).cuda()
        out = Buf((M, N), dt, shift=M % 2)
        rc = gpu.acfun_dev_fc_mxfp4(bx.ptr, code, M, K, d[0].data_ptr(), d[1].data_ptr(),
                                    None if tb is None else tb.data_ptr(), N, out.ptr, act,
                                    s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    assert out.intact() and bx.intact()
    _check_product(values(out.t), layers.mx_decode(*layers.mx_encode(x), K), layers.mx_decode(*b, K), bias,
                   act, t)


@pytest.mark.parametrize("M", [1, 40])
def test_fc_bad_rows(gpu, rng, M):
    """NaN and infinity in an activation make its row NaN and leave the others."""
    N, K = 50, 300
    x = rng.standard_normal((M, K)).astype(np.float32)
    x[0, 299] = np.inf
    if M > 1:
        x[M - 1, 0] = np.nan
    b = _operand(rng, N, K)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx, out = Buf((M, K), torch.float32, x), Buf((M, N), torch.float32)
        d = [torch.as_tensor(v).cuda() for v in layers.mx_tiles(*b)]
        assert gpu.acfun_dev_fc_mxfp4(bx.ptr, 0, M, K, d[0].data_ptr(), d[1].data_ptr(), None, N, out.ptr, 0,
                                      s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    nan = np.isnan(values(out.t))
    assert nan[0].all() and nan[M - 1].all() and not nan[1:M - 1].any()


def test_host_calls(gpu, rng):
    """acfun_quantize_weights_mxfp4 and acfun_fc_mxfp4 on host memory."""
    M, K, N = 9, 200, 77
    w = rng.standard_normal((K, N)).astype(np.float32)
    x, bias = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal(N).astype(np.float32)
    c = np.zeros(gpu.acfun_mxfp4_code_bytes(N, K), np.uint8)
    s = np.zeros(gpu.acfun_mxfp4_scale_bytes(N, K), np.uint8)
    gpu.acfun_quantize_weights_mxfp4(w.ctypes.data, K, N, c.ctypes.data, s.ctypes.data)
    code, byte = layers.mx_encode(w.T)
    wc, ws = layers.mx_tiles(code, byte)
    assert np.array_equal(c, wc) and np.array_equal(s, ws)
    y = np.zeros((M, N), np.float32)
    gpu.acfun_fc_mxfp4(x.ctypes.data, M, K, c.ctypes.data, s.ctypes.data, bias.ctypes.data, N,
                       y.ctypes.data, 1)
    _check_product(y, layers.mx_decode(*layers.mx_encode(x), K), layers.mx_decode(code, byte, K), bias, 1, "f32")


@pytest.mark.parametrize("M,N,K", [(1, 512, 1024), (4, 100, 300), (64, 512, 2048), (300, 300, 1000)])
def test_repeats_and_graph(gpu, rng, M, N, K):
    """The same operands give the same bits, call after call and from a replayed graph
    with other work between the replays."""
    b = _operand(rng, N, K)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.as_tensor(rng.standard_normal((M, K)), dtype=torch.bfloat16).cuda()
        d = [torch.as_tensor(v).cuda() for v in layers.mx_tiles(*b)]
        out = torch.zeros((M, N), dtype=torch.float32, device="cuda").bfloat16()

        def call():
            assert gpu.acfun_dev_fc_mxfp4(x.data_ptr(), 1, M, K, d[0].data_ptr(), d[1].data_ptr(), None, N,
                                          out.data_ptr(), 0, s.cuda_stream) == 0, capi.last_error()
        call()
        s.synchronize()
        first = out.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
        for i in range(4):
            out.zero_()
            g.replay()
            s.synchronize()
            assert torch.equal(out, first), i
            out.zero_()
            call()
            s.synchronize()
            assert torch.equal(out, first), i


def test_graph_of_many_rows(gpu, rng):
    """A layer that needs temporaries is refused while its stream is captured, with the
    capture left whole; quantizing into the caller's buffers and multiplying is captured
    and gives the layer's bits."""
    M, N, K = 600, 2000, 2000
    b = _operand(rng, N, K)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.as_tensor(rng.standard_normal((M, K)), dtype=torch.bfloat16).cuda()
        d = [torch.as_tensor(v).cuda() for v in layers.mx_tiles(*b)]
        c = torch.empty(gpu.acfun_mxfp4_code_bytes(M, K), dtype=torch.uint8, device="cuda")
        sc = torch.empty(gpu.acfun_mxfp4_scale_bytes(M, K), dtype=torch.uint8, device="cuda")
        want, out = (torch.zeros((M, N), dtype=torch.bfloat16, device="cuda") for _ in range(2))

        def fc(y):
            return gpu.acfun_dev_fc_mxfp4(x.data_ptr(), 1, M, K, d[0].data_ptr(), d[1].data_ptr(), None, N,
                                          y.data_ptr(), 0, s.cuda_stream)

        def parts():
            assert gpu.acfun_dev_quantize_mxfp4(x.data_ptr(), 1, M, K, 0, c.data_ptr(), sc.data_ptr(),
                                                s.cuda_stream) == 0, capi.last_error()
            assert gpu.acfun_dev_gemm_mxfp4(M, N, K, c.data_ptr(), sc.data_ptr(), d[0].data_ptr(),
                                            d[1].data_ptr(), out.data_ptr(), 1, None, 0,
                                            s.cuda_stream) == 0, capi.last_error()
        assert fc(want) == 0, capi.last_error()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            refused = fc(out), capi.last_error()
            parts()
        assert refused[0] == -1 and "temporaries" in refused[1]
        for i in range(3):
            out.zero_()
            g.replay()
            s.synchronize()
            assert torch.equal(out, want), i
            assert fc(out) == 0                              # other work between the replays
            s.synchronize()
