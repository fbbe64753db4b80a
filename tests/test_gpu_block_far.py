"""Transformer-layer calls on tensors and operands past 2^31 elements and 2^32 bytes: what
their last rows give, against the numpy oracle in 64 bits."""
import numpy as np
import pytest
import torch

from acfun_amd import capi
from oracle import layers
from test_gpu_mxfp4 import _check_product
from test_gpu_norm import EPS, _norm_tol, _stored

pytestmark = pytest.mark.gpu
BF16 = 1


def _rows(lib, codes, scales, first, rows, K):
    """Row-major codes and scale bytes of rows first .. first + rows (first % 16 == 0)."""
    t, n = first // 16, -(-rows // 16)
    kt, st = -(-K // 128), -(-K // 512)
    c = codes[t * kt * 1024:(t + n) * kt * 1024].cpu().numpy().reshape(n, kt, 4, 16, 16).transpose(0, 3, 1, 2, 4)
    c = c.reshape(n * 16, -1)
    c = np.stack((c & 15, c >> 4), 2).reshape(n * 16, -1)[:rows, :-(-K // 32) * 32]
    s = scales[t * st * 256:(t + n) * st * 256].cpu().numpy().reshape(n, st, 4, 16, 4).transpose(0, 3, 1, 4, 2)
    return c, s.reshape(n * 16, -1)[:rows, :-(-K // 32)]


def _operand(g, lib, rows, K):
    c = torch.randint(0, 256, (lib.acfun_mxfp4_code_bytes(rows, K),), dtype=torch.uint8, device="cuda", generator=g)
    s = torch.randint(125, 129, (lib.acfun_mxfp4_scale_bytes(rows, K),), dtype=torch.uint8, device="cuda",
                      generator=g)
    return c, s


@pytest.mark.parametrize("M", [3, 200])
def test_weights(gpu, M):
    """Products and layers whose weights' codes pass 4 GiB."""
    N, K, last = 1_100_005, 8192, 37
    assert gpu.acfun_mxfp4_code_bytes(N, K) > 1 << 32
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        g = torch.Generator(device="cuda").manual_seed(M)
        a, b = _operand(g, gpu, M, K), _operand(g, gpu, N, K)
        x = torch.randn((M, K), device="cuda", generator=g).bfloat16()
        out, lay = (torch.zeros((M, N), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        assert gpu.acfun_dev_gemm_mxfp4(M, N, K, *(t.data_ptr() for t in (*a, *b)), out.data_ptr(), BF16, None, 0,
                                        s.cuda_stream) == 0, capi.last_error()
        assert gpu.acfun_dev_fc_mxfp4(x.data_ptr(), BF16, M, K, b[0].data_ptr(), b[1].data_ptr(), None, N,
                                      lay.data_ptr(), 0, s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    first = N // 16 * 16 - 32
    tail = layers.mx_decode(*_rows(gpu, *b, first, N - first, K), K)[-last:]
    _check_product(out[:, -last:].double().cpu().numpy(), layers.mx_decode(*_rows(gpu, *a, 0, M, K), K), tail, None,
                   0, "bf16")
    xq = layers.mx_decode(*layers.mx_encode(x.double().cpu().numpy()), K)
    _check_product(lay[:, -last:].double().cpu().numpy(), xq, tail, None, 0, "bf16")


@pytest.mark.parametrize("trans", [0, 1])
def test_quantize(gpu, trans):
    """A tensor of more than 2^31 elements to 4 bits and back."""
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
        c = torch.empty(gpu.acfun_mxfp4_code_bytes(rows, K), dtype=torch.uint8, device="cuda")
        sc = torch.empty(gpu.acfun_mxfp4_scale_bytes(rows, K), dtype=torch.uint8, device="cuda")
        assert gpu.acfun_dev_quantize_mxfp4(x.data_ptr(), BF16, rows, K, trans, c.data_ptr(), sc.data_ptr(),
                                            s.cuda_stream) == 0, capi.last_error()
        back = torch.empty((rows, K), dtype=torch.bfloat16, device="cuda")
        assert gpu.acfun_dev_dequantize_mxfp4(c.data_ptr(), sc.data_ptr(), rows, K, back.data_ptr(), BF16,
                                              s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    e = end.double().cpu().numpy()
    want = layers.mx_decode(*layers.mx_encode(e.T if trans else e), K)
    assert np.array_equal(back[-21:].double().cpu().numpy(), want)
    assert not back[:1000].any() and not back[rows // 2:rows // 2 + 1000].any()


def test_norms(gpu):
    rows, cols, last = 70_003, 32768, 5
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        x = torch.ones((rows, cols), dtype=torch.bfloat16, device="cuda")
        assert x.numel() > 1 << 31
        x[-last:] = torch.randn((last, cols), device="cuda").bfloat16()
        h, xo = torch.empty_like(x), torch.empty_like(x)
        assert gpu.acfun_dev_norm(x.data_ptr(), BF16, rows, cols, 0, None, None, EPS, h.data_ptr(),
                                  s.cuda_stream) == 0, capi.last_error()
        first = h[-last:].double().cpu().numpy()
        assert gpu.acfun_dev_norm_residual(h.data_ptr(), x.data_ptr(), BF16, rows, cols, 0, None, None, x.data_ptr(),
                                           1, 1.0, None, None, EPS, xo.data_ptr(), h.data_ptr(),
                                           s.cuda_stream) == 0, capi.last_error()
    s.synchronize()
    v = x[-last:].double().cpu().numpy()
    want = layers.norm(v, 0, None, None, EPS)
    assert (np.abs(first - want) <= _stored(_norm_tol(v, 0.0, 0, None, None), want, "bf16")).all()
    want, _ = layers.norm_residual(first, v, 0, None, None, v, 1, 1.0, None, None, EPS)
    tol = _norm_tol(first, 0.0, 0, None, None) * np.abs(v)
    tol = tol + 2.0 ** -24 * (np.abs(want - v) + np.abs(v) + np.abs(want) + 2 * tol)
    assert (np.abs(xo[-last:].double().cpu().numpy() - want) <= _stored(tol, want, "bf16")).all()
    assert (h[:2].float() - 1).abs().max() < 0.01
