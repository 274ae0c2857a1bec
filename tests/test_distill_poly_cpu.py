"""The polynomial of distill.cu's exp2_pair by itself: its error as the source states it, over [-1/2, 1/2]."""
import os
import re

import numpy as np

SRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sdmchat_b200", "csrc", "distill.cu")


def test_error_of_the_exponential():
    with open(SRC) as f:
        text = f.read()
    body = re.search(r"kExp2\[6\] = \{([^}]*)\}", text).group(1)
    coef = [float(np.float32(v.strip().rstrip("f"))) for v in body.split(",")]
    stated = [float(v) for v in re.search(r"relative error \((\S+) with its coefficients in float32, (\S+) evaluated", text).groups()]
    f = np.linspace(-0.5, 0.5, 1000001).astype(np.float32).astype(np.float64)
    exact = np.exp2(f)
    error = np.abs(np.polyval(coef[::-1], f) / exact - 1).max()
    assert 0.9 * stated[0] < error < 1.0 * stated[0]
    p = np.full_like(f, coef[5])
    for c in coef[4::-1]:  # a fused multiply-add rounds once
        p = (p * f + c).astype(np.float32).astype(np.float64)
    error = np.abs(p / exact - 1).max()
    assert 0.9 * stated[1] < error < 1.0 * stated[1]
