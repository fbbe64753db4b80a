"""Norms of more rows than the launch has workgroups for, so that each takes rows in turn
(k_norm_row keeps weights and gates from row to row and loads the next row while it works on
one): every row against the numpy oracle in 64 bits, with a last turn that not every
workgroup has."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from block_helpers import TYPES, Buf, values
from oracle import layers
from test_gpu_norm import EPS, U, _dev, _norm_tol, _param, _ptr, _rows, _stored

pytestmark = pytest.mark.gpu

# 16-byte chunks of a row, rows, and of the launch that they stand for: threads to a row,
# rows to a workgroup
SIZES = [(37, 10003, 64, 4), (100, 9999, 64, 4), (200, 2501, 256, 1), (400, 2503, 256, 1), (700, 1301, 512, 1),
         (1500, 701, 1024, 1), (2100, 601, 1024, 1), (4099, 299, 1024, 1)]


def _groups(rows, threads, per):
    """(workgroups, the rows of the last turn) as k_norm_row is launched: four waves to a SIMD."""
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    groups, most = -(-rows // per), cus * (1024 // max(threads, 256))
    grid = -(-groups // -(-groups // most))
    return grid, rows % (grid * per)


def _size(chunks, odd, t):
    n = 16 // torch.empty((), dtype=TYPES[t][1]).element_size()
    return chunks * n - (odd and n // 2 + 1)


CASES = [(c, odd, t) for c in SIZES for odd in (0, 1) for t in TYPES if _size(c[0], odd, t) <= 32768]


@pytest.mark.parametrize("size,odd,t", CASES)
def test_norm(gpu, rng, size, odd, t):
    chunks, rows, threads, per = size
    cols, layer = _size(chunks, odd, t), (chunks + odd) % 2
    grid, last = _groups(rows, threads, per)
    assert grid * per < rows and last != 0
    code, dt = TYPES[t]
    x = _rows(rng, rows, cols, t, off=2.0 if layer else 0.0)
    w, b = _param(rng, cols, True, 1), _param(rng, cols, layer, 0)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx, h = Buf(x.shape, dt, x, shift=odd), Buf(x.shape, dt)
        dw, db = _dev(w), _dev(b)
        for out in (h, bx):                                   # and in place
            assert gpu.acfun_dev_norm(bx.ptr, code, rows, cols, layer, _ptr(dw), _ptr(db), EPS, out.ptr,
                                      s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    got = values(h.t)
    want = layers.norm(x, layer, w, b, EPS)
    tol = _stored(_norm_tol(x, 0.0, layer, w, b), want, t)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    assert h.intact() and bx.intact() and np.array_equal(values(bx.t), got)


@pytest.mark.parametrize("size,odd,t", CASES)
def test_norm_residual(gpu, rng, size, odd, t):
    chunks, rows, threads, per = size
    n = CASES.index((size, odd, t))
    cols, layer = _size(chunks, odd, t), (n + 1) % 2
    grid, last = _groups(rows, threads, per)
    assert grid * per < rows and last != 0
    # gates: for each row; changing at every row's turn or within one; changing once; one for all
    group = [1, 3, rows // 2 + 7, rows, grid * per - 1][n % 5]
    code, dt = TYPES[t]
    x, y = _rows(rng, rows, cols, t), _rows(rng, rows, cols, t)
    pw, pb = _param(rng, cols, n % 7, 1), _param(rng, cols, layer, 0)
    w, b = _param(rng, cols, True, 1), _param(rng, cols, n % 3 == 0, 0)
    g = values(torch.as_tensor(rng.standard_normal((-(-rows // group), cols))).to(dt))
    scale = float(np.float32(0.7))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx, by, bg = Buf(x.shape, dt, x, shift=odd), Buf(x.shape, dt, y), Buf(g.shape, dt, g)
        xo, h = Buf(x.shape, dt), Buf(x.shape, dt, shift=odd)
        p = [_dev(v) for v in (pw, pb, w, b)]

        def call(out, hh):
            assert gpu.acfun_dev_norm_residual(by.ptr, bx.ptr, code, rows, cols, layer, _ptr(p[0]), _ptr(p[1]), bg.ptr,
                                               group, scale, _ptr(p[2]), _ptr(p[3]), EPS, out.ptr, hh.ptr,
                                               s.cuda_stream) == 0, capi.last_error()
            s.synchronize()
            assert all(v.intact() for v in (bx, by, bg, xo, h))
        call(xo, h)
        got_x, got_h = values(xo.t), values(h.t)
        if n % 2:                                             # in place of both, either way round
            call(by, bx)
            assert np.array_equal(values(by.t), got_x) and np.array_equal(values(bx.t), got_h)
        else:
            call(bx, by)
            assert np.array_equal(values(bx.t), got_x) and np.array_equal(values(by.t), got_h)
    want_x, want_h = layers.norm_residual(y, x, layer, pw, pb, g, group, scale, w, b, EPS)
    tol = _norm_tol(y, 0.0, layer, pw, pb) * np.abs(g[np.arange(rows) // group])
    tol = tol + U * (np.abs(want_x - scale * x) + np.abs(scale * x) + np.abs(want_x) + 2 * tol)
    tx = _stored(tol, want_x, t)
    assert (np.abs(got_x - want_x) <= tx).all(), np.max(np.abs(got_x - want_x) / tx)
    th = _stored(_norm_tol(want_x, tol, layer, w, b), want_h, t)
    assert (np.abs(got_h - want_h) <= th).all(), np.max(np.abs(got_h - want_h) / th)
