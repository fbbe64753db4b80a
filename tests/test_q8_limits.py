"""The plans of Q8 and sampling calls at the ends of their sizes: no launch of 2^32 threads or
more, indices within 32 bits (the program is built with the undefined-behaviour sanitizer)."""
import numpy as np
import pytest

import q8_plans
from acfun_amd import capi

BIG = 2 ** 31 - 1


@pytest.fixture(scope="module")
def exe(tmp_path_factory):
    return q8_plans.build(tmp_path_factory.mktemp("q8_plan"))


def test_products(exe):
    for gated in (0, 1):
        sizes = [(1, 1, 0), (1, BIG, 64), (BIG, 1, 64), (BIG, BIG, 64), (1 << 20, 1 << 20, 131072), (1, BIG, 131072),
                 (1 << 14, 1 << 18, 0), (1 << 16, 1 << 17, 64), (300, 300, 0)]
        got = q8_plans.ask(exe, [q8_plans.gemm(*s, gated) for s in sizes])
        for (M, N, K), kind in zip(sizes, got):
            edge = {"FEW16": 16, "FEW32": 32, "FEW64": 64, "MANY128": 128, "MANY256": 256}.get(kind)
            if kind == "none":
                assert M * N >= BIG
                continue
            threads = {"FEW16": 512, "FEW32": 256, "FEW64": 512, "MANY128": 256, "MANY256": 256}[kind]
            cols = edge // (1 + (gated and kind != "FEW16"))
            assert (-(-M // edge) * -(-N // cols) + 7) // 8 * 8 * threads < 2 ** 32
            assert K > 0 or kind.startswith("FEW")


def test_layers(exe):
    """What the header says of captured streams: one launch up to 512 rows of up to 8192, and a
    row of up to 131072."""
    ask = lambda M, K, g: q8_plans.ask(exe, [f"fc {M} 4096 {K} {g}"])[0]  # noqa: E731
    for g in (0, 1):
        for M in (1, 2, 5, 16, 17, 100, 512):
            assert ask(M, 8192, g).endswith("/rows") and ask(M, 64, g).endswith("/rows")
        assert ask(1, 131072, g).endswith("/rows")
        assert ask(513, 64, g) == "two" and ask(16, 20000, g) == "two"
        assert ask(1, 4096, g) == "one/rows" and ask(16, 4096, g) == "two/rows"


def test_quantizer(exe):
    lines = [f"quant {r} {k} {t}" for t in (0, 1) for r, k in ((1, 1), (BIG, 1), (1 << 19, 131072), (16, 131072), (1 << 23, 4096))]
    for line, got in zip(lines, q8_plans.ask(exe, lines)):
        rows = int(line.split()[1])
        assert got == ("not" if rows == BIG else "fits"), line


def test_sampling(exe):
    rng = np.random.default_rng(3)
    lines = [f"sample {r} {c} 256" for r in (1, 2, 7, 32, 200, 5000) for c in (0, 1, 1000, 1025, 24575, 24576, 32003, 131072, 1 << 24)]
    lines += [f"sample {int(2 ** rng.uniform(0, 12))} {int(2 ** rng.uniform(0, 24))} 256" for _ in range(300)]
    got = q8_plans.ask(exe, lines)
    assert any(int(g.split()[0]) > 1 for g in got) and any(g.startswith("1 ") for g in got)


def test_refused_before_the_device(exe):
    L = capi.lib()
    P = [1 << (20 + i) for i in range(8)]
    assert L.acfun_dev_gemm_q8(BIG, BIG, 0, None, None, None, None, P[0], 0, None, 0, None) == -1
    assert "too large" in capi.last_error()
    assert L.acfun_dev_quantize_q8(P[0] << 30, 0, BIG, 1, 0, P[1] << 34, P[2] << 36, None) == -1
    assert "too large" in capi.last_error()
