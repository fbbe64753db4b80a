"""Nuclei whose border the tokens' numbers alone name wrongly or not at all, on the GPU against
the numpy oracle in 64 bits."""
import numpy as np
import pytest
import torch

from block_helpers import TYPES, values
from test_gpu_sample import _check, _sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [700, 3000, 20001])
@pytest.mark.parametrize("m", [0.0, 0.3, 0.7])
def test_border_between_far_values(gpu, rng, cols, m):
    """Equal tokens off their bin's middle, then nothing for many bins: a nucleus that ends some
    tokens before the last of them, or after it, with min_p below and above them."""
    n = min(cols // 4, 900)
    offs = np.repeat(np.linspace(-0.5, -0.53, 16).astype(np.float32), 6)
    x = np.full((len(offs), cols), -2.5, np.float32)
    x[:, 5] = 0
    for r, v in enumerate(offs):
        x[r, rng.permutation(np.arange(6, cols))[:n]] = v
    w = np.exp(x.astype(np.float64))
    border = np.tile([-6.5, -2.5, -0.5, 0.5, 2.5, 6.5], 16)
    wa, wb = np.exp(offs.astype(np.float64)), np.exp(-2.5)
    need = 1 + n * wa + border * np.where(border < 0, wa, wb)
    p = need / w.sum(1)
    _check(gpu, x.astype(np.float64), "f32", rng.random(len(offs)), p=p, m=np.full(len(offs), m))
    # T and x in step: the same weights and bins
    _check(gpu, x.astype(np.float64) * 4, "f32", rng.random(len(offs)), T=np.full(len(offs), 4.0), p=p)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("cols", [700, 3000, 20001])
def test_border_in_a_full_bin(gpu, rng, cols, t):
    """More tokens in the border's bin, of one value and of several, than a list holds."""
    x = np.full((24, cols), -1.0)
    x[:, 3] = 0
    x[12:] += rng.integers(0, 3, (12, cols)) * 2.0 ** -7
    x[6:12, ::2] = -9.0
    _check(gpu, x, t, rng.random(24), p=rng.random(24), m=np.where(np.arange(24) % 3, 0, 0.36))


@pytest.mark.parametrize("cols", [700, 3000, 20001])
def test_flat_and_steep_rows(gpu, rng, cols):
    """Temperatures from where every token is in the first bin to where one has a weight."""
    T = np.repeat(10.0 ** np.arange(-4, 7), 4)
    x = rng.standard_normal((len(T), cols)).astype(np.float32).astype(np.float64)
    p = np.tile([1e-6, 0.3, 0.9, 1 - 2.0 ** -24], 11)
    _check(gpu, x, "f32", rng.random(len(T)), T=T, p=p)
    _check(gpu, x, "f32", rng.random(len(T)), T=T, p=p, k=rng.integers(1, cols, len(T)), m=p * 0.01)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("cols", [700, 3000, 20001, 40000])
def test_masked_places(gpu, rng, cols, t):
    """NaN and infinities among the logits, at temperatures up to infinity: none of a nucleus's mass."""
    rows = 60
    x = values(torch.as_tensor(rng.standard_normal((rows, cols)) * 2).to(TYPES[t][1]))
    for r in range(rows):
        x[r, rng.integers(0, cols, cols // (2 + r % 5))] = (np.nan, -np.inf)[r % 2]
    T = np.tile(np.array([0.5, 1.0, 30.0, 1e30, np.inf]), rows // 5)
    p = rng.random(rows)
    _check(gpu, x, t, rng.random(rows), T=T, p=p)
    _check(gpu, x, t, rng.random(rows), T=T, p=p, k=np.full(rows, cols // 2), m=np.full(rows, 0.1))


@pytest.mark.parametrize("cols", [4, 700, 40000])
def test_largest_value_beside_infinity(gpu, cols):
    """Finite logits have no weight beside an infinite one, the largest fp32 neither."""
    x = np.full((5, cols), float(torch.finfo(torch.float32).max))
    x[:, cols // 2] = np.inf
    off = np.ones(5)
    for T in (0.5, 1.0, np.inf):
        for p in (off, 0.5 * off):
            tok, prob = _sample(gpu, x, "f32", np.linspace(0, 0.99, 5), T=T * off, p=p)
            assert (tok == cols // 2).all() and (prob == 1).all()
