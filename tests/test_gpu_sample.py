"""Tokens drawn from logits on the GPU against the numpy oracle in 64 bits
(oracle/layers.py): the same tokens, and their probabilities within fp32's rounding."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from block_helpers import TYPES, Buf, values
from oracle import layers

pytestmark = pytest.mark.gpu


def _sample(gpu, x, t, u, T=None, k=None, p=None, m=None, ld=None, shift=0):
    """(tokens, probabilities) of rows of logits x [rows, cols] (numpy, the type's values)."""
    rows, cols = x.shape
    ld = ld or cols
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        wide = np.full((rows, ld), 1e4)                      # what lies between rows would win
        wide[:, :cols] = x
        bx = Buf((rows, ld), TYPES[t][1], wide, shift)
        dev = lambda v, dt: None if v is None else torch.as_tensor(np.asarray(v)).to(dt).cuda()  # noqa: E731
        f = torch.float32
        par = [dev(T, f), dev(k, torch.int32), dev(p, f), dev(m, f), dev(u, f)]
        tok, prob = Buf((rows,), torch.int32), Buf((rows,), f)
        rc = gpu.acfun_dev_sample(bx.ptr, TYPES[t][0], rows, cols, ld, *(None if v is None else v.data_ptr() for v in par),
                                  tok.ptr, prob.ptr, s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    assert tok.intact() and prob.intact() and bx.intact()
    return tok.t.cpu().numpy(), values(prob.t)


def _check(gpu, x, t, u, T=None, k=None, p=None, m=None, **kw):
    tok, prob = _sample(gpu, x, t, u, T, k, p, m, **kw)
    f32 = lambda v: None if v is None else np.asarray(v, np.float32).astype(np.float64)  # noqa: E731
    T, p, m, u = f32(T), f32(p), f32(m), f32(u)
    for r in range(len(x)):
        want, w = layers.sample(x[r], 1.0 if T is None else T[r], 0 if k is None else k[r], 1.0 if p is None else p[r],
                                0.0 if m is None else m[r], u[r])
        assert tok[r] == want, (r, tok[r], want)
        # the store's half step, and half a step of 2^-f for each of a row's weights
        f = min(48, 62 - int(x.shape[1] - 1).bit_length())
        assert abs(prob[r] - w) <= w * (2.0 ** -24 + 1.01 * x.shape[1] * 2.0 ** -f) + 2.0 ** -150, (r, prob[r], w)
    return tok


def _logits(rng, rows, cols, t, spread=2.5):
    x = rng.standard_normal((rows, cols)) * spread
    x[:, rng.integers(0, cols, 3)] += 4
    return values(torch.as_tensor(x).to(TYPES[t][1]))


COLS = [1, 2, 3, 63, 64, 65, 1000, 1023, 1024, 1025, 4096, 4099, 8193, 16384, 32003, 65537, 131072, 262147]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", COLS)
def test_filters(gpu, rng, cols, t):
    """Each filter alone and all together, settings of its own for each row."""
    rows = 24 if cols < 20000 else 12
    x, u = _logits(rng, rows, cols, t), rng.random(rows)
    pick = lambda v: rng.choice(np.array(v), rows)  # noqa: E731
    T, k = pick([0.0, 0.3, 0.7, 1.0, 1.5]), pick([0, -3, 1, 2, 20, 1000, cols - 1, cols, cols + 5])
    p, m = pick([0.0, 0.1, 0.5, 0.9, 0.99, 0.999999, 1.0, 2.0]), pick([0.0, -1.0, 0.01, 0.2, 1.0, 3.0])
    _check(gpu, x, t, u)
    _check(gpu, x, t, u, T=T, ld=cols + 3)
    _check(gpu, x, t, u, k=k, shift=1)
    _check(gpu, x, t, u, T=np.abs(T) + 0.1, p=p)
    _check(gpu, x, t, u, m=m)
    _check(gpu, x, t, u, T, k, p, m, ld=(cols + 63) // 64 * 64, shift=3)


@pytest.mark.parametrize("cols", [1, 7, 64, 1000, 5000, 40000, 131072])
def test_equal_logits(gpu, cols):
    """Ties go by index, borders are where real numbers have them: k of n equal tokens
    are the first k, and a nucleus of p = j / n is the first j of them."""
    u = np.array([0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0])
    x = np.full((len(u), cols), -3.0)
    at = np.minimum(u * cols, cols - 1).astype(int)
    tok, prob = _sample(gpu, x, "f32", u)
    if cols & (cols - 1) == 0:
        assert np.array_equal(tok, at)
    assert np.abs(tok - at).max() <= 1 and np.allclose(prob, 1 / cols, rtol=2.0 ** -23)
    n = 2 ** int(np.log2(cols))
    for k, p in ((n, None), (None, n / cols if cols == n else None), (n, 0.5), (n, 1.0)):
        if k is None and p is None:
            continue
        kept = n if p is None or p == 1 else max(1, n // 2) if k else n
        tok, prob = _sample(gpu, x, "f32", u, k=None if k is None else np.full(len(u), k),
                            p=None if p is None else np.full(len(u), p))
        assert np.array_equal(tok, np.minimum(u * kept, kept - 1).astype(int))
        assert (prob == np.float32(1 / kept)).all()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("cols", [50, 3000, 70000])
def test_many_ties(gpu, rng, cols, t):
    """A few values, many tokens with each: borders fall inside a value."""
    rows = 16
    x = rng.choice(np.array([-2.0, -1.0, 0.0, 0.5, 1.0]), (rows, cols))
    x[:, ::7] = np.where(x[:, ::7] == 0, -0.0, x[:, ::7])    # zeros of both signs are equal
    u = rng.random(rows)
    for k in (1, 2, 10, cols // 2, cols - 1):
        _check(gpu, x, t, u, k=np.full(rows, k))
        _check(gpu, x, t, u, k=np.full(rows, k), p=rng.random(rows), m=rng.random(rows) * 0.3)
    _check(gpu, x, t, u, p=rng.random(rows))


def test_what_is_never_drawn(gpu, rng):
    """Masked places: -infinity, NaN, the type's lowest value; rows of nothing else; rows
    with infinities."""
    for t in TYPES:
        low = float(torch.finfo(TYPES[t][1]).min)
        for cols in (5, 700, 33000):
            x = _logits(rng, 14, cols, t)
            x[0] = -np.inf
            x[1] = np.nan
            x[2, ::2], x[2, 1::2] = -np.inf, np.nan
            x[3] = low
            x[4, :-1] = -np.inf
            x[5, :-1] = low
            x[6, 1:] = np.nan
            x[7, rng.integers(0, cols, cols // 2)] = -np.inf
            x[8, rng.integers(0, cols, cols // 2)] = np.nan
            x[9, rng.integers(0, cols, cols // 2)] = low
            x[10, 2:4] = np.inf
            x[11, :] = np.inf
            x[12, 0] = np.inf
            x[13, 0], x[13, 1:] = -low, low
            for T in (0.0, 0.01, 1.0, 1e4):
                for k, p, m in ((None, None, None), (3, None, None), (0, 0.9, 0.01), (3, 0.5, 0.5)):
                    full = lambda v: None if v is None else np.full(14, v)  # noqa: E731
                    tok = _check(gpu, x, t, rng.random(14), np.full(14, T), full(k), full(p), full(m))
                    assert (tok[:3] == -1).all() and tok[4] == cols - 1 and tok[6] == 0


def test_settings_at_their_ends(gpu, rng):
    """Temperatures from the smallest to infinity, NaN in every setting, u outside [0, 1)."""
    nan, inf = np.nan, np.inf
    x = _logits(rng, 12, 3000, "f32")
    u = np.array([0.0, 1.0, 5.0, -1.0, nan, inf, -inf, 1 - 2.0 ** -24, 0.5, 0.3, 0.2, 0.1])
    for T in (1e-45, 1e-30, 1e-3, 1e30, inf, nan, -inf, -1.0):
        _check(gpu, x, "f32", u, T=np.full(12, T))
        _check(gpu, x, "f32", u, T=np.full(12, T), k=np.full(12, 100), p=np.full(12, 0.7), m=np.full(12, 0.1))
    for p in (nan, inf, -inf, -1.0, 1e-45, 1 - 2.0 ** -24):
        _check(gpu, x, "f32", u, p=np.full(12, p))
    for m in (nan, inf, -inf, 1e-45, 1.0):
        _check(gpu, x, "f32", u, m=np.full(12, m))
    for k in (-2 ** 31, 2 ** 31 - 1):
        _check(gpu, x, "f32", u, k=np.full(12, k))


@pytest.mark.parametrize("T", [float("inf"), 1e38, 3.0, 1e-40])
@pytest.mark.parametrize("cols", [5, 5000, 40000])
def test_masked_at_any_temperature(gpu, rng, cols, T):
    """Most tokens ruled out, the first among them, or not a number; finite ones over all of
    fp32's range."""
    x = _logits(rng, 8, cols, "f32")
    x[::2] *= 1e38
    with np.errstate(over="ignore"):
        x = x.astype(np.float32).astype(np.float64)
    for r in range(8):
        x[r, rng.integers(0, cols, 3 * cols)] = [-np.inf, np.nan][r % 2]
        x[r, cols // 2 + r % 2] = 2.0
    x[:, 0] = -np.inf
    u, full = rng.random(8), lambda v: np.full(8, v)  # noqa: E731
    _check(gpu, x, "f32", u, T=full(T))
    _check(gpu, x, "f32", u, T=full(T), k=full(2))
    _check(gpu, x, "f32", u, T=full(T), k=full(cols - 1), p=full(0.9))
    _check(gpu, x, "f32", u, T=full(T), p=full(0.5), m=full(0.1))
    _check(gpu, x, "f32", full(0.0), T=full(T), p=full(0.5), m=full(0.1))


@pytest.mark.parametrize("rows", [1, 2, 17, 300, 1100])
def test_rows_alone(gpu, rng, rows):
    """A row's token is the same in every batch."""
    cols = 9000
    x, u = _logits(rng, rows, cols, "bf16"), rng.random(rows)
    k, p = rng.integers(0, 300, rows), rng.random(rows)
    tok, prob = _sample(gpu, x, "bf16", u, k=k, p=p)
    for r in {0, rows // 2, rows - 1}:
        one = _sample(gpu, x[r:r + 1], "bf16", u[r:r + 1], k=k[r:r + 1], p=p[r:r + 1])
        assert one[0][0] == tok[r] and one[1][0] == prob[r]


def test_no_columns(gpu):
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        u, tok, prob = torch.zeros(70, device="cuda"), Buf((70,), torch.int32), Buf((70,), torch.float32)
        assert gpu.acfun_dev_sample(None, 0, 70, 0, 0, None, None, None, None, u.data_ptr(), tok.ptr, prob.ptr,
                                    s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    assert tok.intact() and prob.intact() and (tok.t == -1).all() and (prob.t == 0).all()


def test_frequencies(gpu, rng):
    """Evenly spread u give each token its share of the kept weight, to 2 in n."""
    n, cols = 4096, 40
    x = np.tile(_logits(rng, 1, cols, "f32"), (n, 1))
    tok, prob = _sample(gpu, x, "f32", (np.arange(n) + 0.5) / n, k=np.full(n, 10))
    w = np.exp(x[0] - x[0].max())
    w[np.argsort(-x[0], kind="stable")[10:]] = 0
    w /= w.sum()
    assert np.abs(np.bincount(tok, minlength=cols) / n - w).max() <= 2 / n
    assert np.allclose(prob, w[tok], rtol=2.0 ** -22)


def test_host_call(gpu, rng):
    rows, cols = 7, 900
    x, u = rng.standard_normal((rows, cols)).astype(np.float32), rng.random(rows).astype(np.float32)
    p, tok, prob = np.full(rows, 0.8, np.float32), np.zeros(rows, np.int32), np.zeros(rows, np.float32)
    gpu.acfun_sample(x.ctypes.data, rows, cols, None, None, p.ctypes.data, None, u.ctypes.data, tok.ctypes.data,
                     prob.ctypes.data)
    want = [layers.sample(x[r], p=float(p[r]), u=float(u[r])) for r in range(rows)]
    assert list(tok) == [a for a, _ in want] and np.allclose(prob, [b for _, b in want], rtol=2.0 ** -23)
    gpu.acfun_sample(x.ctypes.data, rows, cols, None, None, p.ctypes.data, None, u.ctypes.data, tok.ctypes.data, None)
    assert list(tok) == [a for a, _ in want]


@pytest.mark.parametrize("rows,cols", [(1, 131072), (3, 50000), (64, 32003), (300, 2000)])
def test_repeats_and_graph(gpu, rng, rows, cols):
    """The same tokens call after call and from a replayed graph, whose logits and numbers
    change between the replays."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x, u = torch.randn((rows, cols), device="cuda") * 2.5, torch.rand(rows, device="cuda")
        p, k = torch.full((rows,), 0.9, device="cuda"), torch.full((rows,), 500, dtype=torch.int32, device="cuda")
        tok, prob = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")

        def call():
            assert gpu.acfun_dev_sample(x.data_ptr(), 0, rows, cols, cols, None, k.data_ptr(), p.data_ptr(), None,
                                        u.data_ptr(), tok.data_ptr(), prob.data_ptr(), s.cuda_stream) == 0, capi.last_error()
        call()
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
        for i in range(4):
            x.copy_(torch.randn((rows, cols), device="cuda") * 2.5)
            u.copy_(torch.rand(rows, device="cuda"))
            call()
            s.synchronize()
            want = tok.clone(), prob.clone()
            tok.fill_(-7)
            prob.fill_(-7)
            g.replay()
            s.synchronize()
            assert torch.equal(tok, want[0]) and torch.equal(prob, want[1]), i
