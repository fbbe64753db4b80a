"""The transformer-layer operators in numpy, 64 bits: MXFP4 and Q8 operands (values,
codes, the library's byte layout), the norms around a block, activations and the draw
of a token.  Written from the definitions in include/acfun/acfun.h."""
import numpy as np

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def _up(n, m):
    return -(-n // m) * m


def mx_encode(x):
    """x [rows, K] -> (codes [rows, K32], scale bytes [rows, K32/32]), uint8, one
    code per byte; K32 = K rounded up to 32, zeros beyond K.  The codes of a block
    with scale byte 255 are unspecified (0 here)."""
    x = np.asarray(x, np.float64)
    R, K = x.shape
    v = np.zeros((R, _up(K, 32)))
    v[:, :K] = x
    v = v.reshape(R, -1, 32)
    bad = ~np.isfinite(v).all(2)
    a = np.abs(np.where(bad[..., None], 0, v))
    top = a.max(2)
    _, ex = np.frexp(top)                                    # top = m 2^ex, 1/2 <= m < 1
    e = np.where(top > 0, np.maximum(ex - 3, -127), -127)
    t = np.ldexp(a, -e[..., None])
    lo = np.clip(np.searchsorted(LEVELS, t, "right") - 1, 0, 7)      # the level at or below
    hi = np.minimum(lo + 1, 7)
    up, down = LEVELS[hi] - t, t - LEVELS[lo]
    code = np.where((up < down) | ((up == down) & (lo % 2 == 1)), hi, lo)
    code = code | (np.signbit(np.where(bad[..., None], 0, v)).astype(int) << 3)
    return code.reshape(R, -1).astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def mx_decode(code, byte, K=None):
    """The values (float64) of codes and scale bytes; NaN where the byte is 255."""
    v = LEVELS[code & 7] * np.where(code & 8, -1.0, 1.0)
    v = v.reshape(code.shape[0], -1, 32)
    v = np.where(byte[..., None] == 255, np.nan, np.ldexp(v, byte[..., None].astype(int) - 127))
    return v.reshape(code.shape)[:, :K]


def mx_tiles(code, byte):
    """(codes, scales) as the library lays them out, flat uint8 arrays."""
    R, K = code.shape
    c = np.zeros((_up(R, 16), _up(K, 128)), np.uint8)
    s = np.zeros((_up(R, 16), _up(K, 512) // 32), np.uint8)
    c[:R, :K], s[:R, :K // 32] = code, byte
    kt, st = c.shape[1] // 128, s.shape[1] // 16
    packed = c[:, 0::2] | (c[:, 1::2] << 4)
    out_c = np.empty((c.shape[0] // 16, kt, 4, 16, 16), np.uint8)
    out_s = np.empty((c.shape[0] // 16, st, 4, 16, 4), np.uint8)
    for j in range(4):
        for t in range(kt):
            out_c[:, t, j] = packed[:, 64 * t + 16 * j:64 * t + 16 * j + 16].reshape(-1, 16, 16)
        for t in range(st):
            for u in range(4):
                out_s[:, t, j, :, u] = s[:, 16 * t + 4 * u + j].reshape(-1, 16)
    return out_c.reshape(-1), out_s.reshape(-1)


def norm(v, layer, w=None, b=None, eps=1e-5):
    v = np.asarray(v, np.float64)
    if layer:
        v = v - v.mean(1, keepdims=True)
    v = v / np.sqrt((v * v).mean(1, keepdims=True) + eps)
    v = v if w is None else v * np.asarray(w, np.float64)
    return v if b is None else v + np.asarray(b, np.float64)


def norm_residual(y, x, layer, post_w, post_b, gate, group, scale, pre_w, pre_b, eps=1e-5):
    n = norm(y, layer, post_w, post_b, eps)
    if gate is not None:
        n = n * np.asarray(gate, np.float64)[np.arange(len(n)) // group]
    s = scale * np.asarray(x, np.float64) + n
    return s, norm(s, layer, pre_w, pre_b, eps)


def q8_encode(x):
    """x [rows, K] (fp32 values) -> (codes int8 [rows, K], scales float32 [rows])."""
    x = np.asarray(x, np.float64)
    top = np.abs(x).max(1) if x.shape[1] else np.zeros(len(x))
    bad = ~np.isfinite(x).all(1)
    s = (np.where(bad, 0, top) / 127).astype(np.float32)
    s[s < np.float32(2.0 ** -126)] = 0
    live = s > 0
    q = np.rint(np.where(bad[:, None], 0, x) / np.where(live, s, 1).astype(np.float64)[:, None])
    q[~live] = 0
    s[bad] = np.nan
    return q.astype(np.int8), s


def q8_decode(code, scale):
    with np.errstate(invalid="ignore"):
        return code.astype(np.float64) * scale.astype(np.float64)[:, None]


def q8_tiles(code, scale):
    """(codes, scales) as the library lays them out, flat arrays."""
    R, K = code.shape
    c = np.zeros((_up(R, 16), _up(K, 64)), np.int8)
    s = np.zeros(_up(R, 16), np.float32)
    c[:R, :K], s[:R] = code, scale
    kt = c.shape[1] // 64
    out = np.empty((c.shape[0] // 16, kt, 4, 16, 16), np.int8)
    for t in range(kt):
        for j in range(4):
            out[:, t, j] = c[:, 64 * t + 16 * j:64 * t + 16 * j + 16].reshape(-1, 16, 16)
    return out.reshape(-1), s


def act(v, kind):
    """Activations 0 to 4 of include/acfun/acfun.h; 1 + tanh z as 2 / (1 + exp(-2 z))."""
    with np.errstate(over="ignore"):
        if kind == 1:
            return np.where(v < 0, 0, v)
        if kind == 2:
            return v / (1 + np.exp(-v))
        if kind == 3:
            from scipy.special import erfc                   # (what uses no GELU needs no scipy)
            return 0.5 * v * erfc(-v / np.sqrt(2))
        if kind == 4:
            return v / (1 + np.exp(-2 * np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))
    return v


def sample(x, T=1.0, k=0, p=1.0, m=0.0, u=0.0):
    """One row of logits (float64) -> (token, its probability)."""
    x = np.asarray(x, np.float64)
    order = np.lexsort((np.arange(len(x)), np.where(np.isnan(x), np.inf, -x)))
    order = order[:int((x > -np.inf).sum())]
    if not len(order):
        return -1, 0.0
    if not T > 0:
        return int(order[0]), 1.0
    with np.errstate(invalid="ignore", divide="ignore"):
        d = (x[order] - x[order[0]]) / T
    w = np.where(x[order] == x[order[0]], 1.0, np.exp(np.where(np.isnan(d), -np.inf, d)))
    if k > 0:
        order, w = order[:k], w[:k]
    if p < 1:
        n = 1 + int((np.cumsum(w) < p * w.sum()).sum())
        order, w = order[:max(n, 1)], w[:max(n, 1)]
    if m > 0:
        keep = w >= min(m, 1.0)
        order, w = order[keep], w[keep]
    back = np.argsort(order)
    order, w = order[back], w[back]
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    c = np.cumsum(w)
    at = int((c <= u * c[-1]).sum())
    return int(order[at]), float(w[at] / c[-1])
