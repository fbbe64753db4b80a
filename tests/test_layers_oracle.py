"""The numpy oracle of the transformer layers (CPU): what needs no GELU works without scipy."""
import os
import subprocess
import sys

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PROGRAM = """
import sys
sys.modules["scipy"] = None
import numpy as np
from oracle import layers
x = np.linspace(-3, 3, 64).reshape(2, 32)
layers.mx_decode(*layers.mx_encode(x))
layers.norm(x, 1)
layers.q8_encode(x)
layers.act(x, 2)
layers.sample(x[0], k=3)
"""


def test_without_scipy():
    r = subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0, r.stderr
