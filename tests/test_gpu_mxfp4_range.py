"""MXFP4 products and layers with scales at both ends of their range, large against small
ones, results that underflow and overflow; the host-memory calls' empty and missing
operands."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from block_helpers import TYPES, Buf, values
from oracle import layers
from test_gpu_mxfp4 import _check_product, _gemm

pytestmark = pytest.mark.gpu

# one size of each kernel: tiles of 16, 32, 64, 128 and 256
SIZES = [(33, 515, 700), (65, 2053, 2100), (300, 2053, 2048), (1000, 2500, 300), (3001, 3001, 2085)]
# scale bytes of A and of B, first and past the last: 127 is 1
SCALES = {"least x largest": ((0, 6), (247, 255)), "largest x least": ((247, 255), (0, 6)),
          "wide": ((27, 228), (125, 130)), "wide both": ((77, 178), (77, 178)),
          "results underflow": ((0, 30), (97, 127)), "least": ((0, 3), (0, 3)), "large": ((180, 195), (165, 171))}


def _operand(rng, rows, K, scales):
    code = rng.integers(0, 16, (rows, -(-K // 32) * 32)).astype(np.uint8)
    code[:, K:] = 0
    return code, rng.integers(*scales, (rows, code.shape[1] // 32)).astype(np.uint8)


@pytest.mark.parametrize("which", SCALES)
@pytest.mark.parametrize("i", range(len(SIZES)), ids=lambda i: "-".join(str(v) for v in SIZES[i]))
def test_scales(gpu, rng, i, which):
    M, N, K = SIZES[i]
    t = ("f32", "bf16")[(i + list(SCALES).index(which)) % 2]
    a, b = _operand(rng, M, K, SCALES[which][0]), _operand(rng, N, K, SCALES[which][1])
    got = _gemm(gpu, a, b, None, 0, t, M, N, K)
    _check_product(got, layers.mx_decode(*a, K), layers.mx_decode(*b, K), None, 0, t)


@pytest.mark.parametrize("i", range(len(SIZES)), ids=lambda i: "-".join(str(v) for v in SIZES[i]))
def test_overflow(gpu, rng, i):
    """Sums of products past fp32's range, all of one sign: an infinity of that sign, in the
    rows that have them alone."""
    M, N, K = SIZES[i]
    a, b = _operand(rng, M, K, (126, 129)), _operand(rng, N, K, (126, 129))
    a[0][:, 0], b[0][:, 0] = 7, 7                            # 6 in every row's first k
    a[0][M // 2], b[0][:] = np.where(a[0][M // 2] == 0, 0, (a[0][M // 2] & 7) | 8), b[0] & 7
    a[1][M // 2] = 254                                       # -6 2^127 and more of them
    got = _gemm(gpu, a, b, None, 0, "f32", M, N, K)
    assert (got[M // 2] == -np.inf).all()
    rest = np.arange(M) != M // 2
    _check_product(got[rest], layers.mx_decode(*a, K)[rest], layers.mx_decode(*b, K), None, 0, "f32")


@pytest.mark.parametrize("scale", [2.0 ** -140, 2.0 ** -127, 2.0 ** -100, 2.0 ** 100])
@pytest.mark.parametrize("M,N,K", [(1, 64, 200), (5, 300, 1000), (100, 999, 513), (33, 3000, 4096), (333, 2053, 1000)])
def test_layer(gpu, rng, M, N, K, scale):
    """Activations of the least and largest sizes, fp32's subnormals among them, against weights
    of the other end."""
    x = (rng.standard_normal((M, K)) * np.exp(rng.standard_normal(K)) * scale).astype(np.float32)
    mid = int(127 - np.clip(np.log2(scale), -126, 126))
    b = _operand(rng, N, K, (max(mid - 2, 0), min(mid + 2, 255)))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx, out = Buf((M, K), torch.float32, x), Buf((M, N), torch.float32)
        d = [torch.as_tensor(v).cuda() for v in layers.mx_tiles(*b)]
        assert gpu.acfun_dev_fc_mxfp4(bx.ptr, 0, M, K, d[0].data_ptr(), d[1].data_ptr(), None, N, out.ptr, 0,
                                      s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    assert out.intact()
    _check_product(values(out.t), layers.mx_decode(*layers.mx_encode(x), K), layers.mx_decode(*b, K), None, 0, "f32")


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("act", [0, 1])
def test_host_calls(gpu, rng, bias, act):
    """acfun_fc_mxfp4 on host memory without k and without a bias, and on operands of which
    some are in device memory."""
    M, K, N = 7, 130, 45
    bv = rng.standard_normal(N).astype(np.float32) if bias else None
    pb = bv.ctypes.data if bias else None
    y = np.full((M, N), 9, np.float32)
    gpu.acfun_fc_mxfp4(None, M, 0, None, None, pb, N, y.ctypes.data, act)
    want = np.tile(bv if bias else np.zeros(N, np.float32), (M, 1))
    assert np.array_equal(y, np.maximum(want, 0) if act else want)
    w, x = rng.standard_normal((K, N)).astype(np.float32), rng.standard_normal((M, K)).astype(np.float32)
    code, byte = layers.mx_encode(w.T)
    c, s = layers.mx_tiles(code, byte)
    want = layers.mx_decode(*layers.mx_encode(x), K), layers.mx_decode(code, byte, K)
    gpu.acfun_fc_mxfp4(x.ctypes.data, M, K, c.ctypes.data, s.ctypes.data, pb, N, y.ctypes.data, act)
    _check_product(y, *want, bv, act, "f32")
    first = y.copy()
    y[:] = 9
    dc, dx = torch.as_tensor(c).cuda(), torch.as_tensor(x).cuda()
    torch.cuda.synchronize()
    gpu.acfun_fc_mxfp4(dx.data_ptr(), M, K, dc.data_ptr(), s.ctypes.data, pb, N, y.ctypes.data, act)
    assert np.array_equal(y, first)
    for m, n in ((0, N), (M, 0), (-1, N), (M, -1)):          # nothing to do
        y[:] = 9
        gpu.acfun_fc_mxfp4(x.ctypes.data, m, K, c.ctypes.data, s.ctypes.data, pb, n, y.ctypes.data, act)
        assert (y == 9).all()


def test_host_refusals(gpu):
    """A missing operand: an error, the output as it was."""
    x, c, y = np.zeros((2, 64), np.float32), np.zeros(4096, np.uint8), np.full((2, 16), 9, np.float32)
    for missing in range(4):
        p = [x.ctypes.data, c.ctypes.data, c.ctypes.data, y.ctypes.data]
        p[missing] = None
        assert gpu.acfun_dev_norm(None, 9, 1, 1, 0, None, None, 0.0, None, None) == -1      # another error before
        assert "type" in capi.last_error()
        gpu.acfun_fc_mxfp4(p[0], 2, 64, p[1], p[2], None, 16, p[3], 0)
        assert "NULL" in capi.last_error() and (y == 9).all()
