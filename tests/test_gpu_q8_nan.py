"""NaN in an operand of the Q8 products: NaN in that row or column of the results, whatever the
activation and the type, and nowhere else."""
import numpy as np
import pytest

import q8_plans
from test_gpu_q8 import _bias, _call_gemm, _operand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    return q8_plans.build(tmp_path_factory.mktemp("q8_plan"))


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", range(5))
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("M,N,K,few", [(3, 50, 300, True), (300, 600, 640, True), (1100, 1100, 640, False)])
def test_nan(gpu, exe, rng, M, N, K, few, gated, kind, t):
    assert q8_plans.ask(exe, [q8_plans.gemm(M, N, K, gated)])[0].startswith("FEW" if few else "MANY")
    a, bs = _operand(rng, M, K), [_operand(rng, N, K) for _ in range(1 + gated)]
    biases = [_bias(rng, N, kind % 2)] + [None] * gated
    want = np.zeros((M, N), bool)
    a[0][M // 2], a[1][M // 2], want[M // 2] = 0, np.nan, True
    for g, b in enumerate(bs):                               # a channel of each projection
        n = N // 3 + 5 * g
        b[0][n], b[1][n], want[:, n] = 0, np.nan, True
    if biases[0] is not None:
        biases[0][1], want[:, 1] = np.nan, True
    got = _call_gemm(gpu, a, bs, biases, kind, t, M, N, K)
    assert np.array_equal(np.isnan(got), want)
