"""Timed workloads of the library's operators on 8-bit integers and of sampling: the
quantizer with a scale for each row, the products and layers on its operands, the
gated projections of a feed-forward block, and the draw of a token from logits.

listed() holds the fixed workloads, draw(rng) makes others of the same ranges,
prepare()/run() build and run one, work() gives the bytes and operations it
cannot do without, exact() its result from the definition in 64 bits.  With
`own` false run() computes the operators in elementary torch operations, with
`own` true through the C ABI's device-pointer entry points.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_CODES = {"f32": 0, "bf16": 1, "f16": 2}    # the C ABI's element types
_ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}    # and its activations


def listed():
    return [
        # A prompt's activations on their way into an 8-bit product, and read back.
        dict(name="quant_rows", kind="quant", rows=4096, K=4096, trans=False, type="bf16"),
        # A layer's fp32 weights [K][rows] made into 8-bit ones at load.
        dict(name="quant_weights", kind="quant", rows=8192, K=4096, trans=True, type="f32"),
        # A square layer on one token: the smallest product, where latency counts.
        dict(name="fc_token", kind="fc", M=1, N=4096, K=4096, type="bf16", bias=False, act="none"),
        # A fully connected layer of odd sizes with bias and ReLU, fp32 in and out.
        dict(name="fc_ragged", kind="fc", M=333, N=2053, K=1000, type="f32", bias=True, act="relu"),
        # A wide layer on a whole batch of prompts.
        dict(name="fc_large", kind="fc", M=8192, N=8192, K=8192, type="bf16", bias=False, act="none"),
        # One token of each of 128 sequences: quantized once, read by several layers.
        dict(name="gemm_batch", kind="gemm", M=128, N=8192, K=4096, type="bf16", bias=False, act="none"),
        # The gated half of a feed-forward block on one token.
        dict(name="gated_token", kind="gated", M=1, N=8192, K=4096, type="bf16", bias=False, act="silu"),
        # The same on a short batch with odd sizes and biases.
        dict(name="gated_ragged", kind="gated", M=77, N=2053, K=1000, type="f16", bias=True, act="gelu"),
        # The same on a prompt.
        dict(name="gated_prompt", kind="gated", M=4096, N=8192, K=4096, type="bf16", bias=False, act="silu"),
        # The next token of one sequence: every filter on.
        dict(name="sample_token", kind="sample", rows=1, cols=131072, pad=0, type="f32", mode="every"),
        # One token of each of 64 sequences with settings of their own, and logits whose
        # rows are padded to whole lines.
        dict(name="sample_batch", kind="sample", rows=64, cols=32003, pad=61, type="bf16", mode="mixed"),
        # A large batch drawn at a temperature with a nucleus.
        dict(name="sample_large", kind="sample", rows=512, cols=131072, pad=0, type="f32", mode="nucleus"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Two widths in three are a multiple of 64, as layers have them."""
    n = _log(rng, lo, hi)
    return max(64, (n + 32) // 64 * 64) if rng.random() < 2 / 3 else n


def draw(rng):
    kind = rng.choice(["quant", "fc", "fc", "gemm", "gated", "gated", "sample", "sample"])
    t = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "quant":
        return dict(kind=kind, rows=_log(rng, 1, 8192), K=_width(rng, 32, 4096), trans=rng.random() < 0.4, type=t)
    if kind == "sample":
        return dict(kind=kind, rows=_log(rng, 1, 512), cols=_width(rng, 64, 131072),
                    pad=rng.choice([0, 0, rng.randint(1, 64)]), type=t,
                    mode=rng.choice(["mixed", "mixed", "every", "nucleus", "topk", "temperature"]))
    g = kind == "gated"
    return dict(kind=kind, M=_log(rng, 1, 4096 if g else 8192), N=_width(rng, 16, 8192),
                K=_width(rng, 32, 4096 if g else 8192), type=t, bias=rng.random() < 0.5,
                act=rng.choice(["silu", "gelu", "gelu_tanh", "relu"] if g else ["none", "none", "relu", "gelu"]))


# ------------------------------------------------------------------ inputs
_stream = None


def _queue():
    """The caller's stream: one for the whole program."""
    global _stream
    if _stream is None:
        _stream = torch.cuda.Stream()
    return _stream


def _normal(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _uniform(g, shape):
    return torch.rand(shape, generator=g, device="cuda")


def _activations(g, rows, cols, t):
    """A norm's results: a few channels are many times the others."""
    ch = torch.exp(0.3 * _normal(g, (cols,)))
    ch = torch.where(_uniform(g, (cols,)) < 0.01, 10 * ch, ch)
    return (_normal(g, (rows, cols)) * ch).to(_TYPES[t])


def _pick(g, n, values, type):
    at = torch.randint(len(values), (n,), generator=g, device="cuda")
    return torch.tensor(values, dtype=type, device="cuda")[at]


def _settings(g, rows, mode):
    """What each sequence asks for; a filter that none asks for is absent."""
    f, i = torch.float32, torch.int32
    d = dict(temp=_pick(g, rows, [0.6, 0.8, 1.0, 1.3], f), k=None, p=None, m=None)
    if mode == "mixed":      # some greedy, some without one filter or another
        d = dict(temp=_pick(g, rows, [0.0, 0.6, 0.8, 1.0, 1.0, 1.3], f), k=_pick(g, rows, [0, 0, 20, 50, 1000], i),
                 p=_pick(g, rows, [1.0, 0.9, 0.95, 0.99], f), m=_pick(g, rows, [0.0, 0.0, 0.02, 0.1], f))
    elif mode == "every":
        d |= dict(k=_pick(g, rows, [50, 200], i), p=_pick(g, rows, [0.9, 0.95], f), m=_pick(g, rows, [0.01, 0.05], f))
    elif mode == "nucleus":
        d |= dict(p=_pick(g, rows, [0.9, 0.95, 0.99], f))
    elif mode == "topk":
        d |= dict(k=_pick(g, rows, [5, 40, 1000], i))
    return d


def _logits(g, rows, cols, ld, t):
    """A model's: most tokens near one another, a few candidates above them, and, for one
    sequence in four, half of the tokens ruled out."""
    x = _normal(g, (rows, ld), 2.5)
    x = torch.where(_uniform(g, (rows, ld)) < 20 / cols, x.abs() + 6 * _uniform(g, (rows, 1)), x)
    out = (_uniform(g, (rows, 1)) < 0.25) & (_uniform(g, (rows, ld)) < 0.5)
    return x.masked_fill(out, -math.inf).to(_TYPES[t])


def _inputs(case, seed):
    g, k, t = torch.Generator(device="cuda").manual_seed(seed), case["kind"], case["type"]
    if k == "quant":
        if case["trans"]:
            return dict(x=_normal(g, (case["K"], case["rows"]), 1 / math.sqrt(case["K"])).to(_TYPES[t]))
        return dict(x=_activations(g, case["rows"], case["K"], t))
    if k == "sample":
        R, C = case["rows"], case["cols"]
        d = dict(x=_logits(g, R, C, C + case["pad"], t), **_settings(g, R, case["mode"]))
        d["u"] = _uniform(g, (R,))
        return d
    M, N, K = case["M"], case["N"], case["K"]
    d = dict(x=_activations(g, M, K, t), w=_normal(g, (N, K), 1 / math.sqrt(K)))
    d["bias"] = _normal(g, (N,), 0.1) if case["bias"] else None
    if k == "gated":
        d["w2"] = _normal(g, (N, K), 1 / math.sqrt(K))
        d["bias2"] = _normal(g, (N,), 0.1) if case["bias"] else None
    return d


# ------------------------------------------------------------------ plain forms
def _up(n, m):
    return -(-n // m) * m


def _encode(x):
    """Row-major x [rows, K] as (codes, scales); the quotients in 64 bits, for those next
    to a half, and so the scale, whose last bit moves them."""
    s = (x.abs().amax(1).double() / 127).float()
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    q = torch.round(x.double() / torch.where(s > 0, s, 1.0).double().unsqueeze(1))
    return torch.where(s.unsqueeze(1) > 0, q, 0.0).to(torch.int8), s


def _decode(codes, s):
    return codes.float() * s.unsqueeze(1)


def _tiled(codes, s):
    """The library's layout: codes in tiles of 16 rows x 64 k, where the 16 bytes of the
    tile's j-th 16 k and row r are number 16 j + r; scales of rows padded to 16."""
    R, K = codes.shape
    c = torch.nn.functional.pad(codes, (0, _up(K, 64) - K, 0, _up(R, 16) - R))
    c = c.view(c.shape[0] // 16, 16, -1, 4, 16)
    return c.permute(0, 2, 3, 1, 4).contiguous(), torch.nn.functional.pad(s, (0, _up(R, 16) - R))


def _untiled(c, s, R, K):
    """Row-major codes [R, K] and their scales from the library's layout."""
    return c.permute(0, 3, 1, 2, 4).reshape(c.shape[0] * 16, -1)[:R, :K], s[:R]


def _act(v, act):
    if act == "relu":
        return v.relu()
    if act == "silu":
        return v / (1 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _product(a, b, bias):
    y = _decode(*a) @ _decode(*b).t()
    return y + bias if bias is not None else y


def _sample(t, cols):
    """Every row's tokens in order, with the filters as ranges of that order."""
    x = t["x"][:, :cols].double()
    v, order = torch.sort(torch.where(x.isnan(), -math.inf, x), dim=1, descending=True, stable=True)
    rank, T = torch.arange(cols, device=x.device), t["temp"].double().unsqueeze(1)
    w = torch.exp((v - v[:, :1]) / torch.where(T > 0, T, 1.0))
    w = torch.where((T > 0) | (rank == 0), torch.where(v == -math.inf, 0.0, w), 0.0)
    if t["k"] is not None:
        k = t["k"].unsqueeze(1)
        w = torch.where((k <= 0) | (rank < k), w, 0.0)
    if t["p"] is not None:
        c = torch.cumsum(w, 1)
        w = torch.where((c - w < t["p"].double().unsqueeze(1) * c[:, -1:]) | (rank == 0), w, 0.0)
    if t["m"] is not None:
        w = torch.where(w >= t["m"].double().unsqueeze(1), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)             # in the tokens' order
    c = torch.cumsum(w, 1)
    token = (c <= t["u"].double().unsqueeze(1) * c[:, -1:]).sum(1, keepdim=True).clamp(max=cols - 1)
    prob = w.gather(1, token) / c[:, -1:]
    return token.squeeze(1).int(), prob.squeeze(1).float()


def _plain(case, t):
    k, kept = case["kind"], _TYPES[case["type"]]
    if k == "quant":
        x = t["x"].t() if case["trans"] else t["x"]
        c, s = _tiled(*_encode(x))
        return _decode(*_untiled(c, s, case["rows"], case["K"])).to(kept)
    if k == "sample":
        return _sample(t, case["cols"])
    M, N, K = case["M"], case["N"], case["K"]
    a = _untiled(t["xc"], t["xs"], M, K) if k == "gemm" else _encode(t["x"])
    y = _act(_product(a, _untiled(t["wc"], t["ws"], N, K), t["bias"]), case["act"])
    if k == "gated":
        y = y * _product(a, _untiled(t["w2c"], t["w2s"], N, K), t["bias2"])
    return y.to(kept)


# ------------------------------------------------------------------ prepare, run
def prepare(case, seed):
    """The operands, the weights in the form a program keeps them, and the result's buffers."""
    t, k, kept = _inputs(case, seed), case["kind"], _TYPES[case["type"]]
    empty = lambda *shape, type=kept: torch.empty(shape, dtype=type, device="cuda")  # noqa: E731
    if k == "quant":
        R, K = case["rows"], case["K"]
        t["c"] = empty(_up(R, 16) // 16, _up(K, 64) // 64, 4, 16, 16, type=torch.int8)
        t["s"] = empty(_up(R, 16), type=torch.float32)
        t["out"] = empty(R, K)
    elif k == "sample":
        t["token"], t["prob"] = empty(case["rows"], type=torch.int32), empty(case["rows"], type=torch.float32)
    else:
        t["wc"], t["ws"] = _tiled(*_encode(t.pop("w")))
        if k == "gemm":
            t["xc"], t["xs"] = _tiled(*_encode(t.pop("x")))
        if k == "gated":
            t["w2c"], t["w2s"] = _tiled(*_encode(t.pop("w2")))
        t["out"] = empty(case["M"], case["N"])
    _queue().wait_stream(torch.cuda.current_stream())
    return dict(case=case, t=t, p={n: v.data_ptr() for n, v in t.items() if v is not None})


def _call(case, p, s):
    from acfun_amd import capi
    L, k, y = capi.lib(), case["kind"], _CODES[case["type"]]
    if k == "quant":
        R, K = case["rows"], case["K"]
        rc = L.acfun_dev_quantize_q8(p["x"], y, R, K, int(case["trans"]), p["c"], p["s"], s)
        rc = rc or L.acfun_dev_dequantize_q8(p["c"], p["s"], R, K, p["out"], y, s)
    elif k == "fc":
        rc = L.acfun_dev_fc_q8(p["x"], y, case["M"], case["K"], p["wc"], p["ws"], p.get("bias"), case["N"],
                               p["out"], _ACTS[case["act"]], s)
    elif k == "gemm":
        rc = L.acfun_dev_gemm_q8(case["M"], case["N"], case["K"], p["xc"], p["xs"], p["wc"], p["ws"], p["out"], y,
                                 p.get("bias"), _ACTS[case["act"]], s)
    elif k == "gated":
        rc = L.acfun_dev_fc_gated_q8(p["x"], y, case["M"], case["K"], p["wc"], p["ws"], p.get("bias"), p["w2c"],
                                     p["w2s"], p.get("bias2"), case["N"], p["out"], _ACTS[case["act"]], s)
    else:
        rc = L.acfun_dev_sample(p["x"], y, case["rows"], case["cols"], case["cols"] + case["pad"], p["temp"],
                                p.get("k"), p.get("p"), p.get("m"), p["u"], p["token"], p["prob"], s)
    if rc != 0:
        raise RuntimeError(capi.last_error())


def run(state):
    case, t = state["case"], state["t"]
    if not own:
        return _plain(case, t)
    _call(case, state["p"], _queue().cuda_stream)
    return (t["token"], t["prob"]) if case["kind"] == "sample" else t["out"]


# ------------------------------------------------------------------ work
def _held(rows, K):
    """Bytes of an operand in 8 bits with its scales."""
    return rows * (K + 4)


def work(case):
    k, b = case["kind"], 4 if case["type"] == "f32" else 2
    if k == "quant":
        R, K = case["rows"], case["K"]
        return {"bytes": 2 * R * K * b + _held(R, K), "flops": 4 * R * K}
    if k == "sample":
        R, C = case["rows"], case["cols"]
        return {"bytes": R * C * b + 28 * R, "flops": 10 * R * C}
    M, N, K = case["M"], case["N"], case["K"]
    n = 2 if k == "gated" else 1
    a = _held(M, K) if k == "gemm" else M * K * b
    return {"bytes": a + n * _held(N, K) + M * N * b + (4 * n * N if case["bias"] else 0), "flops": 2 * n * M * N * K}


# ------------------------------------------------------------------ in 64 bits
def _values64(x):
    """x [rows, K] as the values of its 8-bit codes: whole multiples of its row's scale,
    the nearest one, the even one of two."""
    x = x.double()
    s = (torch.linalg.vector_norm(x, math.inf, dim=1, keepdim=True) / 127).float().double()   # as it is kept
    q = x / s.clamp(min=1e-300)
    low = torch.floor(q)
    over = q - low
    low = low + ((over > 0.5) | ((over == 0.5) & (low % 2 != 0))).double()
    return low * s * (s >= 2.0 ** -126)


def _act64(v, act):
    if act == "silu":
        return v * torch.sigmoid(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":     # (1 + tanh z) / 2 is 1 / (1 + exp(-2 z))
        return v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return v.clamp(min=0) if act == "relu" else v


def _draw64(x, T, k, p, m, u):
    """One row: (token, its probability), dropping candidates one filter after another."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(x.size), -x))
    order = order[x[order] > -np.inf]
    if not order.size:
        return -1, 0.0
    if not T > 0:
        return int(order[0]), 1.0
    w = np.exp((x[order] - x[order[0]]) / T)
    if k > 0:
        order, w = order[:k], w[:k]
    if p < 1:
        n = 1 + int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left"))
        order, w = order[:n], w[:n]
    order, w = order[w >= min(m, 1.0)], w[w >= min(m, 1.0)]
    back = np.argsort(order)
    order, w = order[back], w[back]
    at = min(int(np.searchsorted(np.cumsum(w), u * w.sum(), side="right")), order.size - 1)
    return int(order[at]), float(w[at] / w.sum())


def exact(case, seed):
    k, t = case["kind"], _inputs(case, seed)
    if k == "quant":
        return _values64(t["x"].t() if case["trans"] else t["x"])
    if k == "sample":
        R, off = case["rows"], {"k": 0, "p": 1.0, "m": 0.0}
        x = t["x"][:, :case["cols"]].cpu().double().numpy()
        row = [t[n].cpu().double().numpy() if t[n] is not None else np.full(R, off[n]) for n in ("temp", "k", "p", "m", "u")]
        got = [_draw64(x[r], row[0][r], int(row[1][r]), row[2][r], row[3][r], row[4][r]) for r in range(R)]
        return (torch.tensor([a for a, _ in got], dtype=torch.int32), torch.tensor([b for _, b in got], dtype=torch.float64))
    a = _values64(t["x"])
    y = torch.matmul(a, _values64(t["w"]).t())
    y = _act64(y + t["bias"].double() if case["bias"] else y, case["act"])
    if k == "gated":
        z = torch.matmul(a, _values64(t["w2"]).t())
        y = y * (z + t["bias2"].double() if case["bias"] else z)
    return y
