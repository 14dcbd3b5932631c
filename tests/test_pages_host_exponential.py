"""The polynomial that stands for some exponentials of the prompt attention, its coefficients read from the
source: in f32, each step rounded as a fused multiply-add rounds, against 2^x in 64 bits."""

import os
import re

import numpy as np

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "aero_b200", "csrc", "pages_prompt.cu")


def test_polynomial_is_as_exact_as_the_hardware():
    """Relative error at most 2^-22, what ex2.approx states, over all that a softmax asks for."""
    body = open(SOURCE).read().split("void ex2_poly(", 1)[1].split("\n}\n", 1)[0]
    steps = re.findall(r"pair\((\d\.\d+)f, \1f\)", body)
    c = [np.float32(x) for x in steps if float(x) < 0.7]  # highest power first
    assert len(c) >= 4 and abs(float(c[-1]) - np.log(2)) < 1e-4 and all(a < b for a, b in zip(c, c[1:]))
    x = np.concatenate([np.linspace(-126, 15, 400001), -np.logspace(-8, 0, 2001)]).astype(np.float32)
    n = np.rint(x.astype(np.float64))
    f = (x - n.astype(np.float32)).astype(np.float64)
    t = np.full_like(f, float(c[0]))
    for k in [*c[1:], np.float32(1)]:
        t = (t * f + float(k)).astype(np.float32).astype(np.float64)  # (one rounding of a product and a sum)
    got, want = t * 2.0**n, 2.0 ** x.astype(np.float64)
    assert np.abs(got / want - 1).max() <= 2.0**-22
