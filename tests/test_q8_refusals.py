"""What the entry points of Q8 operands and of sampling refuse, before the device is
touched (CPU): an error, nothing written; empty outputs are no error."""
import numpy as np

from acfun_amd import capi
from oracle import layers

P = 1 << 20           # stands for device addresses, apart: never read, the call is refused first
Q = [P << i for i in range(12)]


def _refused(rc, word):
    assert rc == -1 and word in capi.last_error(), (rc, capi.last_error())


def test_sizes():
    L = capi.lib()
    for rows, K in ((1, 1), (16, 64), (17, 65), (300, 1000), (2 ** 31 - 1, 1), (1, 2 ** 31 - 1), (2 ** 20, 2 ** 20)):
        assert L.acfun_q8_code_bytes(rows, K) == -(-rows // 16) * -(-K // 64) * 1024
        assert L.acfun_q8_scale_bytes(rows) == -(-rows // 16) * 64
    c, s = layers.q8_tiles(np.zeros((17, 65), np.int8), np.zeros(17, np.float32))
    assert c.nbytes == L.acfun_q8_code_bytes(17, 65) and s.nbytes == L.acfun_q8_scale_bytes(17)
    assert L.acfun_q8_code_bytes(0, 5) == L.acfun_q8_code_bytes(5, 0) == L.acfun_q8_scale_bytes(-1) == 0


def test_quantize():
    L = capi.lib()
    for f in (lambda x=Q[0], t=0, r=4, k=64, c=Q[1], s=Q[2]: L.acfun_dev_quantize_q8(x, t, r, k, 0, c, s, None),
              lambda x=Q[0], t=0, r=4, k=64, c=Q[1], s=Q[2]: L.acfun_dev_quantize_q8(x, t, r, k, 1, c, s, None),
              lambda x=Q[0], t=0, r=4, k=64, c=Q[1], s=Q[2]: L.acfun_dev_dequantize_q8(c, s, r, k, x, t, None)):
        _refused(f(t=3), "type")
        _refused(f(t=-1), "type")
        _refused(f(r=-1), "negative")
        _refused(f(k=-5), "negative")
        _refused(f(k=131073), "131072")
        for p in "xcs":
            _refused(f(**{p: None}), "NULL")
        _refused(f(c=Q[1] + 8), "aligned")
        _refused(f(s=Q[2] + 4), "aligned")
        _refused(f(x=Q[0] + 2), "aligned")
        _refused(f(t=2, x=Q[0] + 1), "aligned")
        _refused(f(x=Q[1] + 1000), "overlaps")
        _refused(f(x=Q[2] + 60), "overlaps")
        assert f(r=0, x=None, c=None) == 0 and f(k=0, x=None, s=None) == 0
    _refused(L.acfun_dev_quantize_q8(Q[0], 0, 4, 64, 0, Q[1], Q[1] + 512, None), "overlaps")


def test_products():
    L = capi.lib()

    def gemm(M=4, N=4, K=64, a=Q[0], sa=Q[1], b=Q[2], sb=Q[3], c=Q[6], t=0, bias=None, act=0):
        return L.acfun_dev_gemm_q8(M, N, K, a, sa, b, sb, c, t, bias, act, None)

    def fc(M=4, N=4, K=64, a=Q[0], b=Q[2], sb=Q[3], c=Q[6], t=0, bias=None, act=0):
        return L.acfun_dev_fc_q8(a, t, M, K, b, sb, bias, N, c, act, None)

    def gated(M=4, N=4, K=64, a=Q[0], sa=Q[1], b=Q[2], sb=Q[3], b2=Q[4], sb2=Q[5], c=Q[6], t=0, bias=None, bias2=None,
              act=2):
        return L.acfun_dev_gemm_gated_q8(M, N, K, a, sa, b, sb, b2, sb2, c, t, bias, bias2, act, None)

    def fc_gated(M=4, N=4, K=64, a=Q[0], b=Q[2], sb=Q[3], b2=Q[4], sb2=Q[5], c=Q[6], t=0, bias=None, bias2=None, act=2):
        return L.acfun_dev_fc_gated_q8(a, t, M, K, b, sb, bias, b2, sb2, bias2, N, c, act, None)
    for f in (gemm, fc, gated, fc_gated):
        two = f in (gated, fc_gated)
        operands = ["b", "sb"] + ["b2", "sb2"] * two + (["a", "sa"] if f in (gemm, gated) else [])
        _refused(f(t=7), "type")
        _refused(f(act=5), "act")
        _refused(f(act=-1), "act")
        for size in "MNK":
            _refused(f(**{size: -1}), "negative")
        _refused(f(K=131073), "131072")
        for p in operands + ["a", "c"]:
            _refused(f(**{p: None}), "NULL")
        for p in operands:
            _refused(f(**{p: Q[8] + 8}), "aligned")
            _refused(f(**{p: Q[6]}), "overlaps")
        _refused(f(c=Q[6] + 2), "aligned")
        _refused(f(a=Q[6] + 16), "overlaps")
        for p in ["bias"] + ["bias2"] * two:
            _refused(f(**{p: Q[7] + 2}), "aligned")
            _refused(f(**{p: Q[6] + 8}), "overlaps")
        assert f(M=0, a=None, c=None) == 0 and f(N=0, b=None, c=None) == 0
        _refused(f(M=2 ** 31 - 1, N=2 ** 31 - 1, a=None, c=None), "NULL")
        _refused(f(M=2 ** 31 - 1, N=2 ** 31 - 1, K=0), "too large")
    _refused(fc(a=Q[0] + 2), "aligned")


def test_sample():
    L = capi.lib()

    def f(x=Q[0], t=0, rows=4, cols=100, ld=100, T=Q[1], k=Q[2], p=Q[3], m=Q[4], u=Q[5], tok=Q[6], prob=Q[7]):
        return L.acfun_dev_sample(x, t, rows, cols, ld, T, k, p, m, u, tok, prob, None)
    _refused(f(t=3), "type")
    _refused(f(rows=-1), "negative")
    _refused(f(cols=-1), "negative")
    _refused(f(ld=99), "ld")
    _refused(f(cols=2 ** 24 + 1, ld=2 ** 25), "2^24")
    _refused(f(rows=2 ** 31 - 1), "too large")
    for a in ("x", "u", "tok"):
        _refused(f(**{a: None}), "NULL")
    for a in ("x", "T", "k", "p", "m", "u", "tok", "prob"):
        _refused(f(**{a: Q[8] + 2}), "aligned")
    for out in ("tok", "prob"):
        for a in ("T", "k", "p", "m", "u"):
            _refused(f(**{out: Q[9], a: Q[9] + 12}), "overlaps")
        _refused(f(**{out: Q[0] + 4 * 399}), "overlaps")
    _refused(f(tok=Q[7] + 4), "overlaps")
    assert f(rows=0, x=None, u=None, tok=None) == 0


def test_host_calls_with_missing_pointers():
    """Nothing is written and the error says why."""
    L = capi.lib()
    y, x = np.full(16, 7, np.float32), np.ones(64, np.float32)
    tok = np.full(4, 7, np.int32)
    L.acfun_fc_q8(x.ctypes.data, 4, 16, None, None, None, 4, y.ctypes.data, 0)
    assert "NULL" in capi.last_error()
    L.acfun_fc_gated_q8(x.ctypes.data, 4, 16, x.ctypes.data, x.ctypes.data, None, None, x.ctypes.data, None, 4,
                        y.ctypes.data, 2)
    assert "NULL" in capi.last_error()
    L.acfun_quantize_weights_q8(x.ctypes.data, 4, 16, None, x.ctypes.data)
    assert "NULL" in capi.last_error()
    L.acfun_sample(x.ctypes.data, 4, 16, None, None, None, None, None, tok.ctypes.data, None)
    assert "NULL" in capi.last_error()
    assert (y == 7).all() and (tok == 7).all()
