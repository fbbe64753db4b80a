"""Timed workloads of the library's operators for transformer layers: the
microscaled 4-bit (MXFP4) quantizer and products, and the norms before and after
a block with its gate and residual scale.

listed() holds the fixed workloads, draw(rng) makes others of the same ranges,
prepare()/run() build and run one, work() gives the bytes and operations it
cannot do without, exact() its result from the definition in 64 bits.  With
`own` false run() computes the operators in elementary torch operations, with
`own` true through the C ABI's device-pointer entry points.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_CODES = {"f32": 0, "bf16": 1, "f16": 2}    # the C ABI's element types
_EPS = 1e-5


def listed():
    return [
        # A prompt's activations on their way into a 4-bit product, and read back.
        dict(name="quant_rows", kind="quant", rows=4096, K=4096, trans=False, type="bf16"),
        # A short batch whose width is no multiple of a block.
        dict(name="quant_ragged", kind="quant", rows=77, K=1000, trans=False, type="f32"),
        # A layer's fp32 weights [K][rows] made into 4-bit ones at load.
        dict(name="quant_weights", kind="quant", rows=8192, K=4096, trans=True, type="f32"),
        # A square layer on one token: the smallest product, where latency counts.
        dict(name="fc_token", kind="fc", M=1, N=4096, K=4096, type="bf16", bias=False, act=0),
        # A fully connected layer of odd sizes with bias and ReLU, fp32 in and out.
        dict(name="fc_ragged", kind="fc", M=333, N=2053, K=1000, type="f32", bias=True, act=1),
        # A wide layer on a whole batch of prompts.
        dict(name="fc_large", kind="fc", M=8192, N=8192, K=8192, type="bf16", bias=False, act=0),
        # One token of each of 128 sequences: quantized once, read by several layers.
        dict(name="gemm_batch", kind="gemm", M=128, N=8192, K=4096, type="bf16", bias=False, act=0),
        # A square product with an fp32 result.
        dict(name="gemm_square", kind="gemm", M=4096, N=4096, K=4096, type="f32", bias=True, act=0),
        # The norm before a block, for one token.
        dict(name="norm_token", kind="norm", rows=1, cols=4096, type="bf16", layer=False),
        # The same for a prompt, with mean and bias, in half precision.
        dict(name="norm_rows", kind="norm", rows=4096, cols=4096, type="f16", layer=True),
        # Between two blocks, one token of each of eight sequences, a gate for each.
        dict(name="residual_token", kind="residual", rows=8, cols=8192, type="bf16", layer=False,
             gate=1, scale=1.0),
        # Between two blocks of a batch of prompts, one gate vector for all rows.
        dict(name="residual_large", kind="residual", rows=8192, cols=8192, type="bf16",
             layer=False, gate=8192, scale=0.5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """Two widths in three are a multiple of 64, as layers have them."""
    n = _log(rng, lo, hi)
    return max(64, (n + 32) // 64 * 64) if rng.random() < 2 / 3 else n


def draw(rng):
    kind = rng.choice(["quant", "fc", "fc", "gemm", "norm", "residual"])
    t = rng.choice(["f32", "bf16", "bf16", "f16"])
    if kind == "quant":
        return dict(kind=kind, rows=_log(rng, 1, 8192), K=_width(rng, 32, 4096),
                    trans=rng.random() < 0.4, type=t)
    if kind in ("fc", "gemm"):
        return dict(kind=kind, M=_log(rng, 1, 8192), N=_width(rng, 16, 8192),
                    K=_width(rng, 32, 8192), type=t, bias=rng.random() < 0.5,
                    act=rng.randint(0, 1))
    c = dict(kind=kind, rows=_log(rng, 1, 8192), cols=_width(rng, 64, 8192), type=t,
             layer=rng.random() < 0.4)
    if t == "f32":
        c["rows"] = (c["rows"] + 1) // 2
    if kind == "residual":
        c["gate"] = rng.choice([0, 1, c["rows"], _log(rng, 1, c["rows"])])   # rows to a gate; 0: no gate
        c["scale"] = rng.choice([1.0, 0.5, round(rng.uniform(0.1, 2.0), 3)])
    return c


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


def _activations(g, rows, cols, t):
    """A residual stream's values: a few channels are many times the others."""
    ch = torch.exp(0.3 * _normal(g, (cols,)))
    ch = torch.where(torch.rand((cols,), generator=g, device="cuda") < 0.01, 20 * ch, ch)
    return (_normal(g, (rows, cols)) * ch).to(_TYPES[t])


def _inputs(case, seed):
    g, k, t = torch.Generator(device="cuda").manual_seed(seed), case["kind"], case["type"]
    if k == "quant":
        if case["trans"]:
            return dict(x=_normal(g, (case["K"], case["rows"]), 1 / math.sqrt(case["K"])).to(_TYPES[t]))
        return dict(x=_activations(g, case["rows"], case["K"], t))
    if k in ("fc", "gemm"):
        M, N, K = case["M"], case["N"], case["K"]
        d = dict(x=_activations(g, M, K, t), w=_normal(g, (N, K), 1 / math.sqrt(K)))
        d["bias"] = _normal(g, (N,), 0.1) if case["bias"] else None
        return d
    R, C = case["rows"], case["cols"]
    d = dict(x=_activations(g, R, C, t), w=1 + _normal(g, (C,), 0.1),
             b=_normal(g, (C,), 0.1) if case["layer"] else None)
    if k == "residual":
        d["y"] = _normal(g, (R, C)).to(_TYPES[t])
        d["post_w"] = 1 + _normal(g, (C,), 0.1)
        d["post_b"] = _normal(g, (C,), 0.1) if case["layer"] else None
        d["gate"] = (_normal(g, (-(-R // case["gate"]), C), 0.5).to(_TYPES[t])
                     if case["gate"] else None)
    return d


# ------------------------------------------------------------------ plain forms
def _pad(x, rows, cols):
    return torch.nn.functional.pad(x, (0, cols - x.shape[1], 0, rows - x.shape[0]))


def _up(n, m):
    return -(-n // m) * m


def _encode(x):
    """Row-major x [rows, K] as (codes [rows, K32], scale bytes [rows, K32 / 32])."""
    x = _pad(x.float(), x.shape[0], _up(x.shape[1], 32))
    v = x.view(x.shape[0], -1, 32)
    top = v.abs().amax(2)
    e = ((top.view(torch.int32) >> 23) - 2).clamp(min=0)
    a = v.abs() * ((254 - e) << 23).view(torch.float32).unsqueeze(2)    # times 2^(127 - e)
    c = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte()
         + (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5).byte())
    return (c | ((v < 0).byte() << 3)).view(x.shape), e.byte()


def _decode(codes, e):
    """The values (fp32) of row-major codes and scale bytes."""
    table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, 0, -.5, -1, -1.5, -2, -3, -4, -6],
                         device=codes.device)
    v = table[codes.int()].view(codes.shape[0], -1, 32)
    scale = torch.where(e > 0, e.int() << 23, 1 << 22).view(torch.float32)    # 2^(e - 127)
    return (v * scale.unsqueeze(2)).view(codes.shape)


def _tiled(codes, e):
    """The library's layout: codes in tiles of 16 rows x 128 k, where the 16 bytes of
    block j and row r of a tile are number 16 j + r, and scale bytes in tiles of 16 rows
    x 512 k, byte 4 (16 j + r) + s of a tile for block j of its s-th 128 k."""
    R, K = codes.shape
    c = _pad(codes, _up(R, 16), _up(K, 128))
    c = (c[:, 0::2] | (c[:, 1::2] << 4)).view(c.shape[0] // 16, 16, -1, 4, 16)
    s = _pad(e, _up(R, 16), _up(K, 512) // 32).view(c.shape[0], 16, -1, 4, 4)
    return c.permute(0, 2, 3, 1, 4).contiguous(), s.permute(0, 2, 4, 1, 3).contiguous()


def _untiled(c, s, R, K):
    """Row-major codes [R, K32] and scale bytes from the library's layout."""
    K = _up(K, 32)
    c = c.permute(0, 3, 1, 2, 4).reshape(c.shape[0] * 16, -1)
    c = torch.stack((c & 15, c >> 4), 2).view(c.shape[0], -1)
    s = s.permute(0, 3, 1, 4, 2).reshape(s.shape[0] * 16, -1)
    return c[:R, :K], s[:R, :K // 32]


def _norm(v, w, b, layer):
    if layer:
        v = v - v.mean(1, keepdim=True)
    v = v / torch.sqrt((v * v).mean(1, keepdim=True) + _EPS) * w
    return v + b if b is not None else v


def _plain(case, t):
    k, kept = case["kind"], _TYPES[case["type"]]
    if k == "quant":
        x = t["x"].t() if case["trans"] else t["x"]
        c, s = _tiled(*_encode(x))
        return _decode(*_untiled(c, s, case["rows"], case["K"]))[:, :case["K"]].to(kept)
    if k in ("fc", "gemm"):
        M, N, K = case["M"], case["N"], case["K"]
        a = _encode(t["x"]) if k == "fc" else _untiled(t["xc"], t["xs"], M, K)
        y = _decode(*a) @ _decode(*_untiled(t["wc"], t["ws"], N, K)).t()
        y = y + t["bias"] if t["bias"] is not None else y
        return (y.relu() if case["act"] else y).to(kept)
    if k == "norm":
        return _norm(t["x"].float(), t["w"], t["b"], case["layer"]).to(kept)
    y = _norm(t["y"].float(), t["post_w"], t["post_b"], case["layer"])
    if t["gate"] is not None:
        y = y * t["gate"].float().repeat_interleave(case["gate"], 0)[:case["rows"]]
    x = t["x"].float() * case["scale"] + y
    return x.to(kept), _norm(x, t["w"], t["b"], case["layer"]).to(kept)


# ------------------------------------------------------------------ prepare, run
def prepare(case, seed):
    """The operands, the weights in the form a program keeps them, and the result's buffers."""
    t, k, kept = _inputs(case, seed), case["kind"], _TYPES[case["type"]]
    empty = lambda *shape, type=kept: torch.empty(shape, dtype=type, device="cuda")  # noqa: E731
    if k == "quant":
        R, K = case["rows"], case["K"]
        t["c"] = empty(_up(R, 16) // 16, _up(K, 128) // 128, 4, 16, 16, type=torch.uint8)
        t["s"] = empty(_up(R, 16) // 16, _up(K, 512) // 512, 4, 16, 4, type=torch.uint8)
        t["out"] = empty(R, K)
    elif k in ("fc", "gemm"):
        t["wc"], t["ws"] = _tiled(*_encode(t.pop("w")))
        if k == "gemm":
            t["xc"], t["xs"] = _tiled(*_encode(t.pop("x")))
        t["out"] = empty(case["M"], case["N"])
    else:
        t["out"] = empty(case["rows"], case["cols"])
        if k == "residual":
            t["x_out"] = empty(case["rows"], case["cols"])
    _queue().wait_stream(torch.cuda.current_stream())
    return dict(case=case, t=t, p={n: v.data_ptr() for n, v in t.items() if v is not None})


def _call(case, p, s):
    from acfun_amd import capi
    L, k, y = capi.lib(), case["kind"], _CODES[case["type"]]
    if k == "quant":
        R, K = case["rows"], case["K"]
        rc = L.acfun_dev_quantize_mxfp4(p["x"], y, R, K, int(case["trans"]), p["c"], p["s"], s)
        rc = rc or L.acfun_dev_dequantize_mxfp4(p["c"], p["s"], R, K, p["out"], y, s)
    elif k == "fc":
        rc = L.acfun_dev_fc_mxfp4(p["x"], y, case["M"], case["K"], p["wc"], p["ws"], p.get("bias"),
                                  case["N"], p["out"], case["act"], s)
    elif k == "gemm":
        rc = L.acfun_dev_gemm_mxfp4(case["M"], case["N"], case["K"], p["xc"], p["xs"], p["wc"],
                                    p["ws"], p["out"], y, p.get("bias"), case["act"], s)
    elif k == "norm":
        rc = L.acfun_dev_norm(p["x"], y, case["rows"], case["cols"], int(case["layer"]), p["w"],
                              p.get("b"), _EPS, p["out"], s)
    else:
        rc = L.acfun_dev_norm_residual(p["y"], p["x"], y, case["rows"], case["cols"],
                                       int(case["layer"]), p["post_w"], p.get("post_b"),
                                       p.get("gate"), case["gate"], case["scale"], p["w"],
                                       p.get("b"), _EPS, p["x_out"], p["out"], s)
    if rc != 0:
        raise RuntimeError(capi.last_error())


def run(state):
    case, t = state["case"], state["t"]
    if not own:
        return _plain(case, t)
    _call(case, state["p"], _queue().cuda_stream)
    return (t["x_out"], t["out"]) if case["kind"] == "residual" else t["out"]


# ------------------------------------------------------------------ work
def _held(rows, K):
    """Bytes of an operand in 4 bits with its scales."""
    return rows * (K / 2 + -(-K // 32))


def work(case):
    k, b = case["kind"], 4 if case["type"] == "f32" else 2
    if k == "quant":
        R, K = case["rows"], case["K"]
        return {"bytes": 2 * R * K * b + _held(R, K), "flops": 4 * R * K}
    if k in ("fc", "gemm"):
        M, N, K = case["M"], case["N"], case["K"]
        a = M * K * b if k == "fc" else _held(M, K)
        return {"bytes": a + _held(N, K) + M * N * b + (4 * N if case["bias"] else 0),
                "flops": 2 * M * N * K}
    R, C = case["rows"], case["cols"]
    params = 8 * C if case["layer"] else 4 * C
    if k == "norm":
        return {"bytes": 2 * R * C * b + params, "flops": 5 * R * C}
    gates = -(-R // case["gate"]) if case["gate"] else 0
    return {"bytes": (4 * R + gates) * C * b + 2 * params, "flops": 12 * R * C}


# ------------------------------------------------------------------ in 64 bits
def _mx64(x):
    """x [rows, K] (float64) as its MXFP4 values: the nearest multiple of the step of
    the value's binade, halves to the even one."""
    R, K = x.shape
    v = _pad(x, R, _up(K, 32)).view(R, -1, 32)
    top = v.abs().amax(2, keepdim=True)
    e = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(min=-127)   # top = m 2^(e+3), m < 1
    scale = ((e.long() + 1023) << 52).view(torch.float64)    # 2^e
    a = v.abs() / scale
    step = 0.5 * (1 + (a >= 2).double() + 2 * (a >= 4).double())
    q = (torch.round(a / step) * step).clamp(max=6.0)
    return (q * scale * torch.sign(v)).view(R, -1)[:, :K]


def _norm64(v, w, b, layer):
    mu = v.mean(1, keepdim=True) if layer else torch.zeros_like(v[:, :1])
    r = ((v - mu).square().mean(1, keepdim=True) + _EPS).rsqrt()
    return (v - mu) * r * w.double() + (b.double() if b is not None else 0.0)


def exact(case, seed):
    k, t = case["kind"], _inputs(case, seed)
    if k == "quant":
        return _mx64((t["x"].t() if case["trans"] else t["x"]).double().contiguous())
    if k in ("fc", "gemm"):
        y = torch.matmul(_mx64(t["x"].double()), _mx64(t["w"].double()).t())
        if case["bias"]:
            y += t["bias"].double()
        return y.clamp(min=0) if case["act"] else y
    if k == "norm":
        return _norm64(t["x"].double(), t["w"], t["b"], case["layer"])
    y = _norm64(t["y"].double(), t["post_w"], t["post_b"], case["layer"])
    if case["gate"]:
        y *= t["gate"].double()[torch.arange(case["rows"], device="cuda") // case["gate"]]
    x = case["scale"] * t["x"].double() + y
    return x, _norm64(x, t["w"], t["b"], case["layer"])
