"""The largest tiles of the Q8 products cut at both edges, in the types whose whole results are too
much for the oracle: the first and last rows of the results, and the last columns of all rows."""
import numpy as np
import pytest

import q8_plans
from test_gpu_q8 import _bias, _call_gemm, _check, _expect, _operand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    return q8_plans.build(tmp_path_factory.mktemp("q8_plan"))


def _some(operand, rows):
    return operand[0][rows], operand[1][rows]


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("gated,M,N,K", [(0, 5000, 3100, 2048), (0, 7000, 2304, 2100), (0, 5103, 3090, 1985),
                                         (1, 3000, 4100, 2048), (1, 4096, 2048, 2048), (1, 3500, 2200, 1978)])
def test_edges(gpu, exe, rng, gated, M, N, K, t):
    assert q8_plans.ask(exe, [q8_plans.gemm(M, N, K, gated)])[0] == "MANY256"
    a, bs = _operand(rng, M, K), [_operand(rng, N, K) for _ in range(1 + gated)]
    biases, act = [_bias(rng, N, g != 1) for g in range(1 + gated)], (N + K) % 5
    got = _call_gemm(gpu, a, bs, biases, act, t, M, N, K, shift=N % 2)
    rows = np.r_[0:2, 255:258, M - 150:M]
    _check(got[rows], *_expect(_some(a, rows), bs, biases, act, t), t)
    cols = np.r_[0:2, N - 45:N]
    few = [None if b is None else b[cols] for b in biases]
    _check(got[:, cols], *_expect(a, [_some(b, cols) for b in bs], few, act, t), t)
