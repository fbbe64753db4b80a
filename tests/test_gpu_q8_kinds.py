"""Every tile of the Q8 products by the sizes that take it (the plan is asked on the host):
whole and cut at both edges, K of one chunk of 64 to several turns of the loop, ending in each
stage, each result type, with and without a gate."""
import pytest

import q8_plans
from test_gpu_q8 import _bias, _call_gemm, _check, _expect, _operand

pytestmark = pytest.mark.gpu

SIZES = {
    (0, "FEW16"): [(3, 100, 2048), (16, 4096, 2048), (60, 900, 200), (3, 2100, 200), (1, 33, 700)],
    (0, "FEW32"): [(17, 600, 64), (60, 2100, 500), (130, 300, 100), (130, 1300, 300), (32, 2048, 256)],
    (0, "FEW64"): [(200, 4100, 2048), (300, 2100, 2048), (500, 1300, 2048), (1000, 600, 2048)],
    (0, "MANY128"): [(500, 4100, 64), (500, 4100, 200), (700, 4100, 64 * 5), (700, 4100, 64 * 6 - 1), (1000, 4099, 64 * 7),
                     (512, 4096, 1024), (700, 2100, 700)],
    (0, "MANY256"): [(5000, 3100, 2048), (7000, 2304, 2100), (4096, 4096, 4096)],
    (1, "FEW16"): [(3, 100, 700), (16, 4096, 512), (3, 2100, 2048), (1, 33, 700)],
    (1, "FEW32"): [(17, 600, 64), (17, 100, 200), (40, 300, 300)],
    (1, "FEW64"): [(200, 1300, 700), (300, 1300, 200), (500, 600, 2048), (700, 600, 200)],
    (1, "MANY128"): [(500, 4100, 64), (500, 4100, 200), (700, 4100, 64 * 5), (700, 4100, 64 * 6 - 1), (700, 4099, 64 * 7),
                     (300, 4100, 700)],
    (1, "MANY256"): [(3000, 2100, 2048), (3000, 4100, 2048), (4096, 2048, 2048), (3500, 2200, 2048 - 70)],
}


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    return q8_plans.build(tmp_path_factory.mktemp("q8_plan"))


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("gated,kind,M,N,K", [(g, k, *s) for (g, k), v in SIZES.items() for s in v])
def test_tile(gpu, exe, rng, gated, kind, M, N, K, t):
    assert q8_plans.ask(exe, [q8_plans.gemm(M, N, K, gated)])[0] == kind
    if M * N * K > 2e10 and t != "bf16" and (M, N, K) != (4096, 4096, 4096):
        pytest.skip("the largest in one type")
    a, bs = _operand(rng, M, K), [_operand(rng, N, K) for _ in range(1 + gated)]
    biases, act = [_bias(rng, N, (M + g) % 2) for g in range(1 + gated)], (N + K) % 5
    got = _call_gemm(gpu, a, bs, biases, act, t, M, N, K, shift=(M + N) % 2)
    _check(got, *_expect(a, bs, biases, act, t), t)
