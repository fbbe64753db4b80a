"""Q8 and sampling calls on tensors and operands past 2^31 elements and 2^32 bytes: what their last
rows give, against the numpy oracle in 64 bits."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from block_helpers import values
from oracle import layers
from test_gpu_q8 import _check, _expect

pytestmark = pytest.mark.gpu
BF16 = 1


def _rows(codes, scales, first, rows, K):
    """Row-major codes and scales of rows first .. first + rows (first % 16 == 0)."""
    t, n, kt = first // 16, -(-rows // 16), -(-K // 64)
    c = codes[t * kt * 1024:(t + n) * kt * 1024].cpu().numpy().reshape(n, kt, 4, 16, 16).transpose(0, 3, 1, 2, 4)
    return c.reshape(n * 16, -1)[:rows, :K], scales[first:first + rows].cpu().numpy()


def _operand(g, lib, rows, K):
    """K is whole 64s."""
    c = torch.randint(-127, 128, (lib.acfun_q8_code_bytes(rows, K),), dtype=torch.int8, device="cuda", generator=g)
    s = torch.rand(lib.acfun_q8_scale_bytes(rows) // 4, device="cuda", generator=g) / (64 * K ** 0.5)
    return c, s


def _ptrs(*operands):
    return [t.data_ptr() for o in operands for t in o]


@pytest.mark.parametrize("M", [3, 200])
def test_weights(gpu, M):
    """Products and layers whose weights' codes pass 4 GiB."""
    N, K, last = 1_100_005, 4096, 37
    assert gpu.acfun_q8_code_bytes(N, K) > 1 << 32
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.Generator(device="cuda").manual_seed(M)
        a, b = _operand(g, gpu, M, K), _operand(g, gpu, N, K)
        x = torch.randn((M, K), device="cuda", generator=g).bfloat16()
        out, lay, gate = (torch.zeros((M, N), dtype=torch.bfloat16, device="cuda") for _ in range(3))
        assert gpu.acfun_dev_gemm_q8(M, N, K, *_ptrs(a, b), out.data_ptr(), BF16, None, 0, s.cuda_stream) == 0, capi.last_error()
        assert gpu.acfun_dev_fc_q8(x.data_ptr(), BF16, M, K, *_ptrs(b), None, N, lay.data_ptr(), 2,
                                   s.cuda_stream) == 0, capi.last_error()
        assert gpu.acfun_dev_gemm_gated_q8(M, N, K, *_ptrs(a, b, b), gate.data_ptr(), BF16, None, None, 2,
                                           s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    first = N // 16 * 16 - 32
    tail = tuple(v[-last:] for v in _rows(*b, first, N - first, K))
    held, rows = _rows(*a, 0, M, K), layers.q8_encode(values(x))
    _check(values(out[:, -last:]), *_expect(held, [tail], [None], 0, "bf16"), "bf16")
    _check(values(lay[:, -last:]), *_expect(rows, [tail], [None], 2, "bf16"), "bf16")
    _check(values(gate[:, -last:]), *_expect(held, [tail, tail], [None, None], 2, "bf16"), "bf16")


@pytest.mark.parametrize("K", [64, 0])
def test_results(gpu, K):
    """More than 2^31 results, of a layer whose rows are quantized first and, without k, of the small
    tiles."""
    M, N = 70_003, 32_771
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.Generator(device="cuda").manual_seed(9)
        x, bias = torch.randn((M, max(K, 1)), device="cuda", generator=g).bfloat16(), torch.randn(N, device="cuda", generator=g)
        b = _operand(g, gpu, N, 64)
        out = torch.zeros((M, N), dtype=torch.bfloat16, device="cuda")
        assert out.numel() > 1 << 31
        assert gpu.acfun_dev_fc_q8(x.data_ptr(), BF16, M, K, *_ptrs(b), bias.data_ptr(), N, out.data_ptr(), 0,
                                   s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    w, bv = _rows(*b, 0, N, 64), bias.cpu().numpy()
    for r in (0, M // 2, M - 1):
        row = layers.q8_encode(values(x[r:r + 1])) if K else (np.zeros((1, 64), np.int8), np.ones(1, np.float32))
        _check(values(out[r:r + 1]), *_expect(row, [w], [bv], 0, "bf16"), "bf16")


@pytest.mark.parametrize("trans", [0, 1])
def test_quantize(gpu, trans):
    """A tensor of more than 2^31 elements to 8 bits and back."""
    rows, K = (270_011, 8192) if not trans else (270_016, 8192)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.zeros((K, rows) if trans else (rows, K), dtype=torch.bfloat16, device="cuda")
        assert x.numel() > 1 << 31
        end = torch.randn((K, 21) if trans else (21, K), device="cuda").bfloat16()
        if trans:
            x[:, -21:] = end
        else:
            x[-21:] = end
        c = torch.empty(gpu.acfun_q8_code_bytes(rows, K), dtype=torch.int8, device="cuda")
        sc = torch.empty(gpu.acfun_q8_scale_bytes(rows) // 4, dtype=torch.float32, device="cuda")
        assert gpu.acfun_dev_quantize_q8(x.data_ptr(), BF16, rows, K, trans, c.data_ptr(), sc.data_ptr(),
                                         s.cuda_stream) == 0, capi.last_error()
        back = torch.empty((rows, K), dtype=torch.bfloat16, device="cuda")
        assert gpu.acfun_dev_dequantize_q8(c.data_ptr(), sc.data_ptr(), rows, K, back.data_ptr(), BF16,
                                           s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    e = values(end)
    code, scale = layers.q8_encode(e.T if trans else e)
    want = torch.as_tensor(layers.q8_decode(code, scale).astype(np.float32)).bfloat16().double().numpy()
    assert np.array_equal(values(back[-21:]), want)
    assert not back[:1000].any() and not back[rows // 2:rows // 2 + 1000].any()


def _drawn(x, tok, prob, u, p):
    for r in range(len(x)):
        want, w = layers.sample(values(x[r]), p=float(p), u=float(u[r]))
        assert int(tok[r]) == want and abs(float(prob[r]) - w) <= 2.0 ** -22 * w, r


def test_sample_rows(gpu):
    """More than 2^31 logits."""
    rows, cols, last = 70_003, 32_768, 9
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.Generator(device="cuda").manual_seed(2)
        x = torch.zeros((rows, cols), dtype=torch.bfloat16, device="cuda")
        assert x.numel() > 1 << 31
        x[:, 77] = 20.0
        x[-last:] = (torch.randn((last, cols), device="cuda", generator=g) * 2.5).bfloat16()
        u, p = torch.rand(rows, device="cuda", generator=g), torch.full((rows,), 0.9, device="cuda")
        tok, prob = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
        assert gpu.acfun_dev_sample(x.data_ptr(), BF16, rows, cols, cols, None, None, p.data_ptr(), None, u.data_ptr(),
                                    tok.data_ptr(), prob.data_ptr(), s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    _drawn(x[-last:], tok[-last:], prob[-last:], u[-last:], p[0])
    assert (tok[:-last] == 77).all() and (prob[:-last] == 1).all()


def test_sample_stride(gpu):
    """Rows further apart than 2^30 elements, drawn from in parts."""
    rows, cols, ld = 3, 40_000, (1 << 30) + 21
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.Generator(device="cuda").manual_seed(3)
        whole = torch.zeros(2 * ld + cols, dtype=torch.bfloat16, device="cuda")
        x = torch.as_strided(whole, (rows, cols), (ld, 1))
        for r in range(rows):
            x[r] = (torch.randn(cols, device="cuda", generator=g) * 2.5).bfloat16()
        u, p = torch.rand(rows, device="cuda", generator=g), torch.full((rows,), 0.9, device="cuda")
        tok, prob = torch.zeros(rows, dtype=torch.int32, device="cuda"), torch.zeros(rows, device="cuda")
        assert gpu.acfun_dev_sample(whole.data_ptr(), BF16, rows, cols, ld, None, None, p.data_ptr(), None, u.data_ptr(),
                                    tok.data_ptr(), prob.data_ptr(), s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    _drawn(x, tok, prob, u, p[0])
