"""Nuclei of equal tokens on the GPU: of n = 2^b tokens a top_p of j / n, which fp32 has, keeps the first
j, exactly."""
import numpy as np
import pytest

from test_gpu_sample import _sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols", [2, 64, 1024, 4096, 32768, 131072, 1 << 20])
def test_nucleus(gpu, cols, t):
    u = np.array([0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 1.0])
    x = np.full((len(u), cols), -3.0)
    for j in sorted({1, cols // 4, cols // 2, cols - cols // 4, cols - 1} - {0}):
        tok, prob = _sample(gpu, x, t, u, p=np.full(len(u), j / cols))
        assert np.array_equal(tok, np.minimum(u * j, j - 1).astype(int)), j
        assert (prob == np.float32(1 / j)).all(), j
        one, prob = _sample(gpu, x[:1], t, u[2:3], p=np.full(1, j / cols))
        assert one[0] == j // 2 and prob[0] == np.float32(1 / j), j


@pytest.mark.parametrize("cols", [64, 4096, 131072])
def test_nucleus_among_the_first(gpu, cols):
    """The same of the first k = 2^b tokens of a row in which others are less, or ruled out."""
    u, k = np.array([0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24]), cols // 4
    for rest in (-4.0, -np.inf):
        x = np.full((len(u), cols), rest)
        at = np.arange(k) * 3 + 1
        x[:, at] = 2.0
        for j in (1, k // 2, k - 1):
            tok, prob = _sample(gpu, x, "f32", u, k=np.full(len(u), k), p=np.full(len(u), j / k))
            assert np.array_equal(tok, at[np.minimum(u * j, j - 1).astype(int)]), j
            assert (prob == np.float32(1 / j)).all(), j
