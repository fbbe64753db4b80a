"""What the transformer-layer entry points refuse, before the device is touched
(CPU): an error, nothing written; empty outputs are no error."""
import numpy as np
import pytest

from acfun_amd import capi
from oracle import layers

P = 1 << 20           # stands for a device address: never read, the call is refused first


def _refused(rc, word):
    assert rc == -1 and word in capi.last_error(), (rc, capi.last_error())


def test_quantize():
    L = capi.lib()
    for f in (lambda x=P, t=0, r=4, k=64, c=P, s=P: L.acfun_dev_quantize_mxfp4(x, t, r, k, 0, c, s, None),
              lambda x=P, t=0, r=4, k=64, c=P, s=P: L.acfun_dev_dequantize_mxfp4(c, s, r, k, x, t, None)):
        _refused(f(t=3), "type")
        _refused(f(t=-1), "type")
        _refused(f(r=-1), "negative")
        _refused(f(k=-5), "negative")
        _refused(f(x=None), "NULL")
        _refused(f(c=None), "NULL")
        _refused(f(s=None), "NULL")
        _refused(f(c=P + 8), "aligned")
        _refused(f(s=P + 4), "aligned")
        _refused(f(x=P + 2), "aligned")
        _refused(f(t=2, x=P + 1), "aligned")
        assert f(r=0, x=None, c=None) == 0 and f(k=0, x=None, s=None) == 0


def test_products():
    L = capi.lib()

    def gemm(M=4, N=4, K=64, a=P, sa=P, b=P, sb=P, c=P, t=0, bias=None, act=0):
        return L.acfun_dev_gemm_mxfp4(M, N, K, a, sa, b, sb, c, t, bias, act, None)

    def fc(M=4, N=4, K=64, a=P, b=P, sb=P, c=P, t=0, bias=None, act=0):
        return L.acfun_dev_fc_mxfp4(a, t, M, K, b, sb, bias, N, c, act, None)
    for f in (gemm, fc):
        _refused(f(t=7), "type")
        _refused(f(act=2), "act")
        for size in "MNK":
            _refused(f(**{size: -1}), "negative")
        for p in ("a", "b", "sb", "c"):
            _refused(f(**{p: None}), "NULL")
        for p in ("b", "sb"):
            _refused(f(**{p: P + 8}), "aligned")
        _refused(f(c=P + 2), "aligned")
        _refused(f(bias=P + 2), "aligned")
        assert f(M=0, a=None, c=None) == 0 and f(N=0, b=None, c=None) == 0
    _refused(gemm(sa=None), "NULL")
    _refused(gemm(a=P + 1), "aligned")
    _refused(fc(a=P + 2), "aligned")


def test_norms():
    L = capi.lib()

    def norm(x=P, t=0, r=4, c=64, kind=0, w=None, b=None, eps=1e-5, h=P):
        return L.acfun_dev_norm(x, t, r, c, kind, w, b, eps, h, None)

    def res(x=P, t=0, r=4, c=64, kind=0, w=None, b=None, eps=1e-5, h=P, y=P, xo=2 * P, g=None, gg=1):
        return L.acfun_dev_norm_residual(y, x, t, r, c, kind, w, b, g, gg, 1.0, w, b, eps, xo, h, None)
    for f in (norm, res):
        _refused(f(t=3), "type")
        _refused(f(r=-1), "negative")
        _refused(f(c=-1), "negative")
        _refused(f(c=32769), "32768")
        _refused(f(kind=2), "kind")
        _refused(f(eps=-1.0), "eps")
        _refused(f(eps=float("nan")), "eps")
        _refused(f(x=None), "NULL")
        _refused(f(x=P + 2), "aligned")
        _refused(f(t=1, h=P + 1), "aligned")
        _refused(f(w=P + 2), "aligned")
        _refused(f(b=P + 1), "aligned")
        assert f(r=0, x=None) == 0 and f(c=0, x=None) == 0
    _refused(norm(h=None), "NULL")
    _refused(res(y=None), "NULL")
    _refused(res(xo=None), "NULL")
    _refused(res(xo=P), "same buffer")
    _refused(res(g=P, gg=0), "gate_group")
    _refused(res(g=P + 2), "aligned")


def test_without_a_gpu():
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    L = capi.lib()
    assert L.acfun_dev_norm(P, 0, 4, 4, 0, None, None, 1e-5, P, None) == -1
    assert "device" in capi.last_error()
    out = np.full(16, 7, np.uint8)
    w = np.ones((2, 2), np.float32)
    L.acfun_quantize_weights_mxfp4(w.ctypes.data, 2, 2, out.ctypes.data, out.ctypes.data)
    assert (out == 7).all()


@pytest.mark.parametrize("rows,K", [(1, 1), (16, 128), (17, 129), (5, 513), (4096, 8192), (0, 5), (5, 0), (-1, 4)])
def test_sizes(rows, K):
    """The arrays' sizes are those of the documented layout, past 32 bits too."""
    L = capi.lib()
    want = (0, 0)
    if rows > 0 and K > 0:
        want = tuple(v.size for v in layers.mx_tiles(np.zeros((rows, -(-K // 32) * 32), np.uint8),
                                                     np.zeros((rows, -(-K // 32)), np.uint8)))
    assert (L.acfun_mxfp4_code_bytes(rows, K), L.acfun_mxfp4_scale_bytes(rows, K)) == want
    assert L.acfun_mxfp4_code_bytes(2 ** 31 - 1, 128) == 2 ** 27 * 1024


def test_oracle_codes():
    """The oracle's quantizer against a search over all levels."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((4, 64)) * np.array([[1e-3], [1], [7], [1e30]])
    x[1, :16] = np.repeat([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], 2)
    x[1, 31] = 7.5
    code, byte = layers.mx_encode(x)
    v = layers.mx_decode(code, byte)
    for r in range(4):
        for b in range(2):
            blk = x[r, 32 * b:32 * b + 32]
            e = int(np.floor(np.log2(np.abs(blk).max()))) - 2
            assert byte[r, b] == e + 127
            grid = layers.LEVELS * 2.0 ** e
            for i in range(32):
                d = np.abs(grid - abs(blk[i]))
                near = np.flatnonzero(d == d.min())
                k = near[0] if len(near) == 1 else [n for n in near if n % 2 == 0][0]
                assert v[r, 32 * b + i] == np.sign(blk[i]) * grid[k]


def test_overlaps():
    """A result that overlaps an input, by its first or last bytes."""
    L = capi.lib()
    n = 4 * 64 * 4                                           # bytes of a 4 x 64 fp32 tensor
    far = [P + (i << 16) for i in range(8)]
    nc = L.acfun_mxfp4_code_bytes(4, 64)
    word = "overlaps"

    def quant(x=far[0], c=far[1], s=far[2]):
        return L.acfun_dev_quantize_mxfp4(x, 0, 4, 64, 0, c, s, None)

    def dequant(x=far[0], c=far[1], s=far[2]):
        return L.acfun_dev_dequantize_mxfp4(c, s, 4, 64, x, 0, None)
    for f in (quant, dequant):
        _refused(f(x=far[1]), word)
        _refused(f(x=far[1] + nc - 16), word)
        _refused(f(x=far[2] - n + 16), word)
    _refused(quant(s=far[1] + nc - 16), word)

    def gemm(c, bias=None):
        return L.acfun_dev_gemm_mxfp4(4, 64, 64, far[0], far[1], far[2], far[3], c, 0, bias, 0, None)
    for i in range(4):
        _refused(gemm(far[i] + 4), word)
        _refused(gemm(far[i] - n + 4), word)
    _refused(gemm(far[5], far[5] + n - 4), word)

    def fc(c, bias=None):
        return L.acfun_dev_fc_mxfp4(far[0], 0, 4, 64, far[1], far[2], bias, 64, c, 0, None)
    for i in range(3):
        _refused(fc(far[i]), word)
        _refused(fc(far[i] - n + 4), word)
    _refused(fc(far[5], far[5]), word)

    def norm(h, w=far[1], b=far[2]):
        return L.acfun_dev_norm(far[0], 0, 4, 64, 1, w, b, 1e-5, h, None)
    _refused(norm(far[0] + 4), word)
    _refused(norm(far[0] - n + 4), word)
    _refused(norm(far[1]), word)
    _refused(norm(far[2] - n + 4), word)

    def res(xo=far[2], h=far[3], gate=far[4], group=4):
        return L.acfun_dev_norm_residual(far[0], far[1], 0, 4, 64, 0, far[5], None, gate, group, 1.0, far[6],
                                         None, 1e-5, xo, h, None)
    for i in range(2):
        _refused(res(xo=far[i] + 4), word)
        _refused(res(h=far[i] - n + 4), word)
    _refused(res(h=far[2] + n - 4), word)
    _refused(res(xo=far[4]), word)
    _refused(res(h=far[4] - n + 4), word)
    _refused(res(xo=far[4] + n - 4, group=1), word)
    _refused(res(xo=far[5]), word)
    _refused(res(h=far[6] + 4), word)
