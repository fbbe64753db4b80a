"""Every kernel and tile of the MXFP4 products and layers in each result type, with and
without bias and ReLU, cut at both edges, K whole and ragged.  The sizes are chosen by the
kernel that runs them, which test_kinds asks of the library's own choice (256 CUs)."""
import numpy as np
import pytest

import mx_plans

# M, N, K, kind.  256 x 256 tiles: one row or column past a tile, K that ends in each of the
# four chunks of a group.  64 x 64: two and four units of a wave to a load of scales.
PRODUCTS = [(3001, 3001, 2085, "MANY256"), (4097, 2560, 2400, "MANY256"), (3500, 3333, 2500, "MANY256"),
            (3001, 3001, 2200, "MANY256"), (400, 4096, 2085, "MANY128"), (513, 4099, 1500, "MANY128"),
            (300, 2053, 2048, "FEW64"), (300, 2053, 2500, "FEW64"), (200, 2053, 4100, "FEW64"),
            (500, 1000, 3500, "FEW64"), (65, 2053, 2100, "FEW32"), (33, 515, 4700, "FEW16")]
# rows quantized by every workgroup for 64 columns with K past 4096, and layers in two
# launches, by the product's kind
LAYERS = [(33, 3000, 4096, "rows64", ""), (100, 1500, 4500, "rows64", ""), (40, 4100, 5000, "rows64", ""),
          (300, 2053, 2500, "two/rows64", "FEW64"), (513, 1000, 3001, "two", "FEW64"),
          (400, 4096, 2085, "two/rows64", "MANY128"), (3001, 3001, 2085, "two", "MANY256")]
NAMES = ["f32", "bf16", "f16"]


def test_kinds(tmp_path):
    exe = mx_plans.build(tmp_path)
    assert mx_plans.ask(exe, [mx_plans.gemm(*p[:3]) for p in PRODUCTS]) == [p[3] for p in PRODUCTS]
    for elem in (2, 4):
        assert mx_plans.ask(exe, [mx_plans.fc(*p[:3], elem) for p in LAYERS]) == [p[3] for p in LAYERS]
    two = [p for p in LAYERS if p[4]]
    assert mx_plans.ask(exe, [mx_plans.gemm(*p[:3]) for p in two]) == [p[4] for p in two]


def _scales(byte, t):
    """A's scale bytes; for fp16 so far below 1 that the sums stay in its range."""
    return byte if t != "f16" else np.minimum(byte, 124) - 12


@pytest.mark.gpu
@pytest.mark.parametrize("t", NAMES)
@pytest.mark.parametrize("i", range(len(PRODUCTS)), ids=lambda i: "-".join(str(v) for v in PRODUCTS[i]))
def test_product(gpu, rng, i, t):
    from oracle import layers
    from test_gpu_mxfp4 import _check_product, _gemm, _operand
    M, N, K, _ = PRODUCTS[i]
    n = i + NAMES.index(t)
    a, b = _operand(rng, M, K, 3), _operand(rng, N, K, 3)
    a = (a[0], _scales(a[1], t))
    bias = rng.standard_normal(N).astype(np.float32) if n % 3 != 1 else None
    act = int(n % 3 == 0)
    got = _gemm(gpu, a, b, bias, act, t, M, N, K)
    _check_product(got, layers.mx_decode(*a, K), layers.mx_decode(*b, K), bias, act, t)


@pytest.mark.gpu
@pytest.mark.parametrize("i", [0, 4, 7, 10], ids=lambda i: PRODUCTS[i][3])
def test_bad_blocks(gpu, rng, i):
    """A NaN block of A and one of B: their row and column of C, and nothing else."""
    from oracle import layers
    from test_gpu_mxfp4 import _check_product, _gemm, _operand
    M, N, K, _ = PRODUCTS[i]
    a, b = _operand(rng, M, K, 3), _operand(rng, N, K, 3)
    a[1][M - 1, -1] = 255
    b[1][N // 3, 0] = 255
    bias = rng.standard_normal(N).astype(np.float32)
    got = _gemm(gpu, a, b, bias, 1, "f32", M, N, K)
    want = np.zeros((M, N), bool)
    want[M - 1], want[:, N // 3] = True, True
    assert np.array_equal(np.isnan(got), want)
    _check_product(got, layers.mx_decode(*a, K), layers.mx_decode(*b, K), bias, 1, "f32")


@pytest.mark.gpu
@pytest.mark.parametrize("t", NAMES)
@pytest.mark.parametrize("i", range(len(LAYERS)), ids=lambda i: "-".join(str(v) for v in LAYERS[i][:4]).replace("/", "."))
def test_layer(gpu, rng, i, t):
    import torch

    from acfun_amd import capi
    from block_helpers import TYPES, Buf, values
    from oracle import layers
    from test_gpu_mxfp4 import _check_product, _operand
    M, N, K = LAYERS[i][:3]
    n = i + NAMES.index(t)
    code, dt = TYPES[t]
    x = values(torch.as_tensor(rng.standard_normal((M, K)) * np.exp(0.5 * rng.standard_normal(K))).to(dt))
    b = _operand(rng, N, K, 2)
    bias = rng.standard_normal(N).astype(np.float32) if n % 2 else None
    act = int(n % 3 == 0)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        bx, out = Buf((M, K), dt, x, shift=n % 3), Buf((M, N), dt, shift=n % 2)
        d = [torch.as_tensor(v).cuda() for v in layers.mx_tiles(*b)]
        tb = None if bias is None else torch.as_tensor(bias).cuda()
        rc = gpu.acfun_dev_fc_mxfp4(bx.ptr, code, M, K, d[0].data_ptr(), d[1].data_ptr(),
                                    None if tb is None else tb.data_ptr(), N, out.ptr, act, s.cuda_stream)
    assert rc == 0, capi.last_error()
    s.synchronize()
    assert out.intact() and bx.intact()
    _check_product(values(out.t), layers.mx_decode(*layers.mx_encode(x), K), layers.mx_decode(*b, K), bias, act, t)
