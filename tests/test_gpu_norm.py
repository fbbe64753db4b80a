"""Norms before and after a block on the GPU against the numpy oracle in 64 bits."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from block_helpers import TYPES, Buf, half_step, smallest, values
from oracle import layers

pytestmark = pytest.mark.gpu
EPS = 1e-5
U = 2.0 ** -24
SIZES = [(1, 1), (1, 4096), (2, 3), (3, 63), (5, 64), (2, 65), (8, 255), (4, 1000), (3, 2047), (300, 512),
         (2, 8192), (1, 8200), (2, 16384), (1, 20001), (1, 32768), (64, 1024), (7, 4104)]


def _stat_err(cols):
    """Relative error of a sum of `cols` values in 32 bits: a thread adds at most 128
    of them in a row, and at most 16 partial sums follow in a tree or in a row."""
    return (min(cols, 128) + 22 + 4) * U


def _norm_tol(v, dv, layer, w, b):
    """How far norm(v + dv') may be off, |dv'| <= dv: the statistics' errors, the
    error of v itself, and five roundings of the formula."""
    cols = v.shape[1]
    e = _stat_err(cols)
    dv = np.broadcast_to(dv, v.shape)
    mean = v.mean(1, keepdims=True) if layer else 0.0
    dmean = (e * np.abs(v).mean(1, keepdims=True) + dv.mean(1, keepdims=True)) if layer else 0.0
    c = v - mean
    dc = dv + dmean + U * np.abs(c)
    var = (c * c).mean(1, keepdims=True) + EPS
    dvar = (2 * np.abs(c) * dc + dc * dc).mean(1, keepdims=True) + (e + 4 * U) * var
    rs = 1 / np.sqrt(var)
    # 1/sqrt(var - dvar) - 1/sqrt(var), where dvar may be a good part of var
    drs = np.where(dvar < var, 1 / np.sqrt(np.maximum(var - dvar, 1e-300)) - rs, 1 / np.sqrt(EPS)) + 2 * U * rs
    n = np.abs(c) * rs
    aw = np.abs(w) if w is not None else 1.0
    ab = np.abs(b) if b is not None else 0.0
    return aw * (dc * (rs + drs) + np.abs(c) * drs) + 5 * U * (n * aw + ab)


def _stored(tol, want, t):
    return tol + half_step(t) * (np.abs(want) + tol) + smallest(t)


def _rows(rng, rows, cols, t, off=0.0):
    x = rng.standard_normal((rows, cols)) * np.exp(0.3 * rng.standard_normal(cols)) + off
    x[:, rng.integers(0, cols)] *= 20
    return values(torch.as_tensor(x).to(TYPES[t][1]))


def _param(rng, cols, on, base):
    return (base + 0.1 * rng.standard_normal(cols)).astype(np.float32) if on else None


def _dev(a):
    return None if a is None else torch.as_tensor(a).cuda()


def _ptr(t):
    return None if t is None else t.data_ptr()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("layer", [0, 1])
@pytest.mark.parametrize("rows,cols", SIZES)
def test_norm(gpu, rng, rows, cols, layer, t):
    code, dt = TYPES[t]
    x = _rows(rng, rows, cols, t, off=3.0 if layer else 0.0)
    w, b = _param(rng, cols, cols % 5 != 0, 1), _param(rng, cols, layer and cols % 3, 0)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx, h = Buf(x.shape, dt, x, shift=rows % 2), Buf(x.shape, dt, shift=cols % 2)
        dw, db = _dev(w), _dev(b)
        rc = gpu.acfun_dev_norm(bx.ptr, code, rows, cols, layer, _ptr(dw), _ptr(db), EPS, h.ptr,
                                s.cuda_stream)
        assert rc == 0, capi.last_error()
        s.synchronize()
        got = values(h.t)
        assert h.intact() and bx.intact()
        assert gpu.acfun_dev_norm(bx.ptr, code, rows, cols, layer, _ptr(dw), _ptr(db), EPS, bx.ptr,
                                  s.cuda_stream) == 0         # in place
        s.synchronize()
    want = layers.norm(x, layer, w, b, EPS)
    tol = _stored(_norm_tol(x, 0.0, layer, w, b), want, t)
    assert (np.abs(got - want) <= tol).all(), np.max(np.abs(got - want) / tol)
    assert bx.intact() and (np.abs(values(bx.t) - want) <= tol).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("gate", ["none", "row", "all", "group"])
@pytest.mark.parametrize("rows,cols,layer", [(r, c, (r + c) % 2) for r, c in SIZES])
def test_norm_residual(gpu, rng, rows, cols, layer, gate, t):
    code, dt = TYPES[t]
    x, y = _rows(rng, rows, cols, t), _rows(rng, rows, cols, t)
    pw, pb = _param(rng, cols, True, 1), _param(rng, cols, layer, 0)
    w, b = _param(rng, cols, gate != "row", 1), _param(rng, cols, layer, 0)
    group = {"none": 0, "row": 1, "all": rows, "group": 3}[gate]
    g = None if gate == "none" else values(torch.as_tensor(rng.standard_normal((-(-rows // group), cols))).to(dt))
    scale = np.float32(1.0 if gate == "all" else 0.7)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx, by = Buf(x.shape, dt, x, shift=1), Buf(x.shape, dt, y, shift=rows % 2)
        bg = None if g is None else Buf(g.shape, dt, g)
        xo, h = Buf(x.shape, dt), Buf(x.shape, dt, shift=rows % 2)
        p = [_dev(v) for v in (pw, pb, w, b)]

        def call(out, hh):
            rc = gpu.acfun_dev_norm_residual(by.ptr, bx.ptr, code, rows, cols, layer, _ptr(p[0]), _ptr(p[1]),
                                             bg.ptr if bg else None, group, scale, _ptr(p[2]), _ptr(p[3]), EPS,
                                             out, hh, s.cuda_stream)
            assert rc == 0, capi.last_error()
            s.synchronize()
        call(xo.ptr, h.ptr)
        got_x, got_h = values(xo.t), values(h.t)
        assert all(v.intact() for v in (bx, by, xo, h))
        xo.t.zero_()
        call(xo.ptr, None)                                    # no norm after
        assert np.array_equal(values(xo.t), got_x)
        call(bx.ptr, by.ptr)                                  # in place of both
        assert np.array_equal(values(bx.t), got_x) and np.array_equal(values(by.t), got_h)
        assert bx.intact() and by.intact()
    want_x, want_h = layers.norm_residual(y, x, layer, pw, pb, g, max(group, 1), float(scale), w, b, EPS)
    gg = 1.0 if g is None else np.abs(g[np.arange(rows) // group])
    tol = _norm_tol(y, 0.0, layer, pw, pb) * gg
    tol = tol + U * (np.abs(want_x - float(scale) * x) + np.abs(float(scale) * x) + np.abs(want_x) + 2 * tol)
    tx = _stored(tol, want_x, t)
    assert (np.abs(got_x - want_x) <= tx).all(), np.max(np.abs(got_x - want_x) / tx)
    th = _stored(_norm_tol(want_x, tol, layer, w, b), want_h, t)
    assert (np.abs(got_h - want_h) <= th).all(), np.max(np.abs(got_h - want_h) / th)


@pytest.mark.parametrize("cols", [1, 100, 4096])
def test_norm_odd_rows(gpu, rng, cols):
    """Rows of zeros, of one value, with NaN or an infinity: each row goes by itself."""
    x = rng.standard_normal((6, cols)).astype(np.float32)
    x[1], x[2] = 0, 5
    x[3, cols // 2], x[4, 0] = np.nan, np.inf
    for layer in (0, 1):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            bx, h = Buf(x.shape, torch.float32, x), Buf(x.shape, torch.float32)
            assert gpu.acfun_dev_norm(bx.ptr, 0, 6, cols, layer, None, None, EPS, h.ptr, s.cuda_stream) == 0
        s.synchronize()
        got = values(h.t)
        assert (got[1] == 0).all() and np.isnan(got[3]).all() and np.isnan(got[4, 0])
        if layer:
            assert (got[2] == 0).all()
        ok = [0, 2, 5]
        want = layers.norm(x[ok], layer, None, None, EPS)
        assert (np.abs(got[ok] - want) <= _stored(_norm_tol(x[ok].astype(np.float64), 0.0, layer, None, None), want,
                                                  "f32")).all()
