"""Q8 quantizer and products on the GPU against the numpy oracle in 64 bits
(oracle/layers.py): the quantizer byte for byte, the products within the roundings of
what follows their exact sums."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from block_helpers import TYPES, Buf, half_step, smallest, values
from oracle import layers

pytestmark = pytest.mark.gpu


def _quantize(gpu, x, t, trans=False, shift=0):
    """(codes, scales), guarded, of x [rows, K] (trans: given as [K, rows])."""
    code, dt = TYPES[t]
    rows, K = x.shape[::-1] if trans else x.shape
    nc, ns = gpu.acfun_q8_code_bytes(rows, K), gpu.acfun_q8_scale_bytes(rows)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx = Buf(x.shape, dt, x, shift)
        c, sc = Buf((nc,), torch.int8), Buf((ns // 4,), torch.float32)
        rc = gpu.acfun_dev_quantize_q8(bx.ptr, code, rows, K, int(trans), c.ptr, sc.ptr, s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    assert c.intact() and sc.intact() and bx.intact()
    return c, sc


def _check_codes(c, sc, x):
    wc, ws = layers.q8_tiles(*layers.q8_encode(x))
    assert np.array_equal(sc.t.cpu().numpy(), ws, equal_nan=True)
    assert np.array_equal(c.t.cpu().numpy(), wc)


ROWS_K = [(1, 1), (1, 63), (2, 64), (3, 65), (15, 127), (16, 128), (17, 129), (33, 500), (5, 512), (64, 513),
          (65, 100), (100, 1000), (1, 4096), (130, 2048), (31, 4100), (7, 9001), (2, 20000), (300, 4096), (1, 40000),
          (16, 8200)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("rows,K", ROWS_K)
def test_quantize_bytes(gpu, rng, rows, K, trans, t):
    x = rng.standard_normal((rows, K)) * np.exp(rng.standard_normal((rows, 1)) * 3)
    x[:, rng.integers(0, K)] *= 10
    x = values(torch.as_tensor(x).to(TYPES[t][1]))           # the type's values
    c, sc = _quantize(gpu, x.T.copy() if trans else x, t, trans, shift=rows % 3)
    _check_codes(c, sc, x)


@pytest.mark.parametrize("trans", [False, True])
@pytest.mark.parametrize("t", TYPES)
def test_quantize_edges(gpu, t, trans):
    """Halves of the scale's multiples and their neighbours at every size of row that the
    type has, rows whose scale is at the end of the normal numbers, zeros of both signs,
    subnormals, the largest values, NaN and infinities."""
    dt = TYPES[t][1]
    v = np.concatenate([np.arange(-64, 64) + 0.5, [0, -0.0, 63.5, 127, 1, 0.5, 0.49999, 3.0]])
    lo, hi = {"f32": (-149, 120), "bf16": (-133, 120), "f16": (-24, 8)}[t]
    rows = []
    for e in range(lo, hi + 1):
        for top in (127, 127 * 1.3, 254 / 3):
            r = torch.tensor(np.ldexp(v * (top / 127), e)).to(dt)
            bits = r.view(torch.int32 if t == "f32" else torch.int16)
            for d in (-1, 0, 1):                             # the neighbours in the type
                n = torch.where(r == 0, bits, bits + d).view(dt).double().numpy()
                rows.append(np.where(np.isfinite(n), n, 0))
    big, tiny = float(torch.finfo(dt).max), float(torch.finfo(dt).tiny)
    for special in (np.nan, np.inf, -np.inf, big, -big, big / 2, tiny, 127 * 2.0 ** -126, 127.5 * 2.0 ** -126,
                    126.9 * 2.0 ** -126, 2.0 ** -149):
        for scale in (0, 1, tiny):
            r = v * scale
            r[11] = special
            rows.append(r)
    rows += [np.zeros(len(v)), -np.zeros(len(v))]
    x = values(torch.as_tensor(np.array(rows)).to(dt))
    c, sc = _quantize(gpu, x.T.copy() if trans else x, t, trans)
    _check_codes(c, sc, x)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("rows,K", ROWS_K)
def test_dequantize(gpu, rng, rows, K, t):
    code = rng.integers(-127, 128, (rows, K)).astype(np.int8)
    scale = np.exp(rng.standard_normal(rows) * 2).astype(np.float32)
    big = float(torch.finfo(TYPES[t][1]).max)
    scale[-1] = np.float32(big / 127)                        # 127 of it may pass the largest
    scale[0] = np.nan if rows > 1 else scale[0]
    wc, ws = layers.q8_tiles(code, scale)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        c, sc = torch.as_tensor(wc).cuda(), torch.as_tensor(ws).cuda()
        out = Buf((rows, K), TYPES[t][1], shift=K % 3)
        rc = gpu.acfun_dev_dequantize_q8(c.data_ptr(), sc.data_ptr(), rows, K, out.ptr, TYPES[t][0], s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    want = np.clip(layers.q8_decode(code, scale), -big, big)
    want = torch.as_tensor(want.astype(np.float32)).to(TYPES[t][1]).double().numpy()     # (q scale in fp32, then stored)
    got = values(out.t)
    assert out.intact()
    assert np.array_equal(got, want, equal_nan=True)


# ------------------------------------------------------------------ products
def _operand(rng, rows, K, spread=1.0):
    code = rng.integers(-127, 128, (rows, K)).astype(np.int8)
    return code, (np.exp(rng.standard_normal(rows) * spread) / 127 / np.sqrt(K)).astype(np.float32)


def _linear(a, b, bias):
    """(value, error) of a projection in fp32 from its exact sum: the sum to fp32, two
    scales, the bias, each off by at most half a step of 2^-23."""
    sums = (a[0].astype(np.float64) @ b[0].astype(np.float64).T)
    with np.errstate(invalid="ignore"):
        v = sums * a[1].astype(np.float64)[:, None] * b[1].astype(np.float64)
    off = 3.01 * 2.0 ** -24 * np.abs(v) + 2.0 ** -148
    if bias is not None:
        v = v + bias
        off = off + 2.0 ** -24 * (np.abs(v) + off)
    return v, off


def _activated(v, off, kind, t):
    """An activation of v.  Its slope is at most 1.13.  exp(z) of the hardware is off by
    a step (2^-23) and by what the argument's roundings, at most 4 half steps of z, give;
    with fp32 results those of silu are added back.  erfc has the argument's, z^2 of the
    result for each step of z = v / sqrt 2.  Sums and quotients: 12 half steps.  A denominator past
    the range gives 0 for what is below |v| 2^-127."""
    y = layers.act(v, kind)
    with np.errstate(invalid="ignore"):
        z = {0: 0, 1: 0, 2: np.abs(v) * (t != "f32"), 3: 3 * v * v, 4: 8 * np.abs(v + 0.044715 * v ** 3)}[kind]
        own = 2.0 ** -24 * (12 + z) * np.abs(y) + np.abs(v) * 2.0 ** -125 if kind > 1 else 0
        return y, 1.13 * off + np.minimum(own, np.abs(y) + np.abs(v) * 2.0 ** -24)


def _check(got, want, off, t):
    off = off + half_step(t) * (np.abs(want) + off) + smallest(t)
    big = {"f32": 3.4e38, "bf16": 3.38e38, "f16": 65504}[t]
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(got), bad)
    near = ~bad & (np.abs(want) < big)
    with np.errstate(invalid="ignore"):
        assert (np.abs(got - want)[near] <= off[near]).all(), np.nanmax((np.abs(got - want) / off)[near])
        assert (np.abs(got)[~bad & ~near] >= 0.99 * big).all()


def _expect(a, bs, biases, kind, t):
    y, off = _activated(*_linear(a, bs[0], biases[0]), kind, t)
    if len(bs) == 2:
        u, du = _linear(a, bs[1], biases[1])
        off = off * np.abs(u) + np.abs(y) * du + off * du
        y = y * u
        off = off + 2.0 ** -24 * np.abs(y)
    return y, off


def _weights(bs):
    return [[torch.as_tensor(v).cuda() for v in layers.q8_tiles(*b)] for b in bs]


def _ptr(t):
    return None if t is None else t.data_ptr()


def _bias(rng, N, on):
    return rng.standard_normal(N).astype(np.float32) if on else None


def _call_gemm(gpu, a, bs, biases, kind, t, M, N, K, shift=0):
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        da = [torch.as_tensor(v).cuda() for v in layers.q8_tiles(*a)]
        db = _weights(bs)
        tb = [None if b is None else torch.as_tensor(b).cuda() for b in biases]
        out = Buf((M, N), TYPES[t][1], shift=shift)
        if len(bs) == 1:
            rc = gpu.acfun_dev_gemm_q8(M, N, K, _ptr(da[0]), _ptr(da[1]), _ptr(db[0][0]), _ptr(db[0][1]), out.ptr,
                                       TYPES[t][0], _ptr(tb[0]), kind, s.cuda_stream)
        else:
            rc = gpu.acfun_dev_gemm_gated_q8(M, N, K, _ptr(da[0]), _ptr(da[1]), _ptr(db[0][0]), _ptr(db[0][1]),
                                             _ptr(db[1][0]), _ptr(db[1][1]), out.ptr, TYPES[t][0], _ptr(tb[0]),
                                             _ptr(tb[1]), kind, s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    assert out.intact()
    return values(out.t)


def _call_fc(gpu, x, bs, biases, kind, t, M, N, K, shift=0):
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx, db = Buf((M, K), TYPES[t][1], x, shift=M % 3), _weights(bs)
        tb = [None if b is None else torch.as_tensor(b).cuda() for b in biases]
        out = Buf((M, N), TYPES[t][1], shift=shift)
        if len(bs) == 1:
            rc = gpu.acfun_dev_fc_q8(bx.ptr, TYPES[t][0], M, K, _ptr(db[0][0]), _ptr(db[0][1]), _ptr(tb[0]), N, out.ptr,
                                     kind, s.cuda_stream)
        else:
            rc = gpu.acfun_dev_fc_gated_q8(bx.ptr, TYPES[t][0], M, K, _ptr(db[0][0]), _ptr(db[0][1]), _ptr(tb[0]),
                                           _ptr(db[1][0]), _ptr(db[1][1]), _ptr(tb[1]), N, out.ptr, kind, s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    assert out.intact() and bx.intact()
    return values(out.t)


SHAPES = [(1, 1, 1), (1, 16, 64), (3, 5, 33), (16, 16, 512), (17, 33, 129), (1, 4096, 4096), (2, 777, 513),
          (13, 2048, 1000), (16, 100, 8192), (33, 515, 640), (64, 100, 2048), (40, 1000, 513), (128, 256, 1024),
          (128, 2048, 4096), (257, 130, 2000), (300, 511, 96), (512, 512, 512), (513, 769, 1153), (1000, 2500, 300),
          (2048, 2048, 256), (1025, 4097, 640)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gemm(gpu, rng, M, N, K, t):
    a, b, bias, kind = _operand(rng, M, K), _operand(rng, N, K), _bias(rng, N, (M + N) % 2), (M + K) % 5
    got = _call_gemm(gpu, a, [b], [bias], kind, t, M, N, K, shift=N % 2)
    _check(got, *_expect(a, [b], [bias], kind, t), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_gated(gpu, rng, M, N, K, t):
    a, bs = _operand(rng, M, K), [_operand(rng, N, K) for _ in range(2)]
    biases, kind = [_bias(rng, N, (M + N) % 2), _bias(rng, N, (M + N) % 3)], (M + K) % 5
    got = _call_gemm(gpu, a, bs, biases, kind, t, M, N, K, shift=N % 2)
    _check(got, *_expect(a, bs, biases, kind, t), t)


FC = [(1, 64, 32), (1, 4096, 4096), (2, 130, 1), (7, 100, 1000), (16, 2053, 777), (17, 300, 4096), (33, 64, 130),
      (100, 999, 513), (333, 2053, 1000), (600, 700, 2048), (1, 10, 8192), (5, 3000, 31), (1, 30, 40000), (2, 30, 33000),
      (3, 50, 20000), (8, 40, 17000), (16, 40, 9000), (16, 40, 12000), (7, 600, 1500), (1, 20, 131072)]


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("M,N,K", FC)
def test_fc(gpu, rng, M, N, K, t, gated):
    x = values(torch.as_tensor(rng.standard_normal((M, K)) * np.exp(rng.standard_normal(K))).to(TYPES[t][1]))
    n, kind = 1 + gated, (M + N + K) % 5
    bs, biases = [_operand(rng, N, K) for _ in range(n)], [_bias(rng, N, (M + g) % 2) for g in range(n)]
    got = _call_fc(gpu, x, bs, biases, kind, t, M, N, K, shift=M % 2)
    _check(got, *_expect(layers.q8_encode(x), bs, biases, kind, t), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("kind", range(5))
@pytest.mark.parametrize("gated", [False, True])
def test_activations(gpu, rng, gated, kind, t):
    """Over the whole range of the argument: far tails, zero, where a result overflows."""
    M, N, K = 5, 400, 64
    a, bs = _operand(rng, M, K), [_operand(rng, N, K) for _ in range(1 + gated)]
    bs[0][1][:] = 0                                          # the bias alone
    bias = np.concatenate([np.linspace(-30, 30, 300), [0, -0.0, 1e-30, -1e-30, 1e30, -1e30], np.linspace(-120, 120, 94)])
    biases = [bias.astype(np.float32)] + [None] * gated
    if t == "f16":
        biases[0] = np.clip(biases[0], -6e4, 6e4)
    if kind == 4:
        biases[0] = np.clip(biases[0], -1e10, 1e10)          # v^3 in fp32's range
    got = _call_gemm(gpu, a, bs, biases, kind, t, M, N, K)
    _check(got, *_expect(a, bs, biases, kind, t), t)


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 48, 512), (20, 100, 1000), (300, 600, 640), (1100, 1100, 640)])
def test_nan_rows(gpu, rng, M, N, K, gated):
    """A row with a NaN, a channel with one: NaN there, through every activation, and
    nowhere else; zero rows are zero."""
    for kind in (1, 2):
        a, bs = _operand(rng, M, K), [_operand(rng, N, K) for _ in range(1 + gated)]
        a[0][M // 2], a[1][M // 2] = 0, np.nan
        bs[-1][0][N // 3], bs[-1][1][N // 3] = 0, np.nan
        got = _call_gemm(gpu, a, bs, [None, None][:1 + gated], kind, "f32", M, N, K)
        want = np.zeros((M, N), bool)
        want[M // 2], want[:, N // 3] = True, True
        assert np.array_equal(np.isnan(got), want)


def test_fc_bad_rows(gpu, rng):
    for M in (1, 16, 40):
        N, K = 50, 300
        x = rng.standard_normal((M, K)).astype(np.float32)
        x[0, 299] = np.inf
        x[M - 1, 0] = np.nan
        if M > 2:
            x[1] = 0
        b = _operand(rng, N, K)
        got = _call_fc(gpu, x, [b], [None], 0, "f32", M, N, K)
        assert np.isnan(got[0]).all() and np.isnan(got[M - 1]).all() and not np.isnan(got[1:M - 1]).any()
        if M > 2:
            assert (got[1] == 0).all()


@pytest.mark.parametrize("K", [131072, 131009])
def test_longest_sums(gpu, K):
    """Every product 127^2: sums next to the end of 32 bits, exactly."""
    for M, N in ((2, 20), (300, 40)):
        a = (np.full((M, K), 127, np.int8), np.ones(M, np.float32))
        b = (np.full((N, K), -127, np.int8), np.ones(N, np.float32))
        got = _call_gemm(gpu, a, [b], [None], 0, "f32", M, N, K)
        assert (got == float(np.float32(-127.0 * 127 * K))).all()


@pytest.mark.parametrize("M,N", [(1, 7), (40, 300), (300, 300)])
def test_no_k(gpu, rng, M, N):
    """K = 0: the biases alone; no operand is read."""
    g, u = (rng.standard_normal(N).astype(np.float32) for _ in range(2))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        tg, tu, out = torch.as_tensor(g).cuda(), torch.as_tensor(u).cuda(), Buf((M, N), torch.float32)
        assert gpu.acfun_dev_gemm_q8(M, N, 0, None, None, None, None, out.ptr, 0, _ptr(tg), 1, s.cuda_stream) == 0
        s.synchronize()
        assert np.array_equal(values(out.t), np.tile(np.maximum(g, 0).astype(np.float64), (M, 1)))
        assert gpu.acfun_dev_gemm_gated_q8(M, N, 0, None, None, None, None, None, None, out.ptr, 0, _ptr(tg), _ptr(tu),
                                           0, s.cuda_stream) == 0
        s.synchronize()
        assert np.array_equal(values(out.t), np.tile((g * u).astype(np.float64), (M, 1)))
        assert gpu.acfun_dev_fc_q8(None, 0, M, 0, None, None, None, N, out.ptr, 0, s.cuda_stream) == 0
        s.synchronize()
        assert out.intact() and (values(out.t) == 0).all()


@pytest.mark.parametrize("M,N,K", [(1, 4100, 4096), (16, 500, 1000), (40, 300, 777), (200, 2053, 1000),
                                   (700, 1300, 512)])
def test_rows_alone(gpu, rng, M, N, K):
    """A row's result is the same bits in every batch, whatever kernel runs it."""
    x = torch.as_tensor(rng.standard_normal((M, K))).bfloat16()
    bs = [_operand(rng, N, K) for _ in range(2)]
    whole = _call_fc(gpu, x, bs, [None, None], 2, "bf16", M, N, K)
    for r in {0, M // 2, M - 1}:
        one = _call_fc(gpu, x[r:r + 1], bs, [None, None], 2, "bf16", 1, N, K)
        assert np.array_equal(one[0], whole[r])
    a = layers.q8_encode(values(x))
    assert np.array_equal(_call_gemm(gpu, a, bs, [None, None], 2, "bf16", M, N, K), whole)


def test_host_calls(gpu, rng):
    """The calls on host memory: weights, the layer, the gated layer."""
    M, K, N = 9, 200, 77
    w = [rng.standard_normal((K, N)).astype(np.float32) for _ in range(2)]
    x, bias = rng.standard_normal((M, K)).astype(np.float32), rng.standard_normal(N).astype(np.float32)
    held = []
    for v in w:
        c = np.zeros(gpu.acfun_q8_code_bytes(N, K), np.int8)
        s = np.zeros(gpu.acfun_q8_scale_bytes(N) // 4, np.float32)
        gpu.acfun_quantize_weights_q8(v.ctypes.data, K, N, c.ctypes.data, s.ctypes.data)
        wc, ws = layers.q8_tiles(*layers.q8_encode(v.T))
        assert np.array_equal(c, wc) and np.array_equal(s, ws)
        held.append((c, s))
    a, bs = layers.q8_encode(x), [layers.q8_encode(v.T) for v in w]
    y = np.zeros((M, N), np.float32)
    gpu.acfun_fc_q8(x.ctypes.data, M, K, held[0][0].ctypes.data, held[0][1].ctypes.data, bias.ctypes.data, N,
                    y.ctypes.data, 1)
    _check(y, *_expect(a, bs[:1], [bias], 1, "f32"), "f32")
    gpu.acfun_fc_gated_q8(x.ctypes.data, M, K, held[0][0].ctypes.data, held[0][1].ctypes.data, None,
                          held[1][0].ctypes.data, held[1][1].ctypes.data, bias.ctypes.data, N, y.ctypes.data, 2)
    _check(y, *_expect(a, bs, [None, bias], 2, "f32"), "f32")


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 512, 1024), (4, 100, 300), (64, 512, 2048), (300, 300, 1000), (512, 96, 8192)])
def test_repeats_and_graph(gpu, rng, M, N, K, gated):
    """The same operands give the same bits, call after call and from a replayed graph
    with other work between the replays."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.as_tensor(rng.standard_normal((M, K)), dtype=torch.bfloat16).cuda()
        d = _weights([_operand(rng, N, K) for _ in range(2)])
        out = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda")

        def call():
            if gated:
                rc = gpu.acfun_dev_fc_gated_q8(x.data_ptr(), 1, M, K, _ptr(d[0][0]), _ptr(d[0][1]), None, _ptr(d[1][0]),
                                               _ptr(d[1][1]), None, N, out.data_ptr(), 2, s.cuda_stream)
            else:
                rc = gpu.acfun_dev_fc_q8(x.data_ptr(), 1, M, K, _ptr(d[0][0]), _ptr(d[0][1]), None, N, out.data_ptr(), 0,
                                         s.cuda_stream)
            assert rc == 0, capi.last_error()
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
    M, N, K = 600, 1000, 2000
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.as_tensor(rng.standard_normal((M, K)), dtype=torch.bfloat16).cuda()
        (d,) = _weights([_operand(rng, N, K)])
        c = torch.empty(gpu.acfun_q8_code_bytes(M, K), dtype=torch.int8, device="cuda")
        sc = torch.empty(gpu.acfun_q8_scale_bytes(M) // 4, dtype=torch.float32, device="cuda")
        want, out = (torch.zeros((M, N), dtype=torch.bfloat16, device="cuda") for _ in range(2))

        def fc(y):
            return gpu.acfun_dev_fc_q8(x.data_ptr(), 1, M, K, _ptr(d[0]), _ptr(d[1]), None, N, y.data_ptr(), 0,
                                       s.cuda_stream)

        def parts():
            assert gpu.acfun_dev_quantize_q8(x.data_ptr(), 1, M, K, 0, _ptr(c), _ptr(sc), s.cuda_stream) == 0
            assert gpu.acfun_dev_gemm_q8(M, N, K, _ptr(c), _ptr(sc), _ptr(d[0]), _ptr(d[1]), out.data_ptr(), 1, None, 0,
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
