"""How exact the weights of drawn tokens are: random numbers next to the border between two tokens.

Two logits m > x: weights 1 and w = e^(x - m), as multiples of 2^-48 of the first (vocabularies of up to 2^14). The second is
drawn where u (1 + w) >= 1. The library's w is off by half of 2^-48 and by 2^-50 (its series 2^-52.6, the table's entry
2^-52, the arithmetic's roundings the rest), and u S, a product in 64 bits just below 2^48, by 2^-5 of a multiple. So where
u (1 + w) lies u (2^-49 + 2^-50) + 2^-53 or more from 1 the token is that of the exact weights. Each row lies a little further away, 2 % of 2^-48 and x's rounding:
u is chosen, w follows from it, and x - m from w, m the next f32 above and x the rest. What the f32s then
say exactly is worked out in 60 digits.
"""

import decimal
import math

import numpy as np
import pytest

from aero_b200 import native_cuda as nc

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

D = decimal.Decimal
UNIT = D(2)**-48


@pytest.fixture(autouse=True)
def _gpu(cuda_lib):
    nc.require_gpu()


def off(u):
    """How far u (1 + w) may be off, in multiples of 2^-48."""
    return u * (0.5 + 0.25) + 2.0**-5


def row(halvings, side):
    """(m, x, u, the token) with w about 2^-halvings and u (1 + w) on one side of 1."""
    u = np.float32(1 / (1 + 2.0**-halvings))
    w = (1 + side * D(off(float(u)) + 0.02) * UNIT) / D(float(u)) - 1
    d = -w.ln()
    m = np.float32(float(d))
    if D(float(m)) < d:
        m = np.nextafter(m, np.float32(np.inf))
    x = np.float32(float(D(float(m)) - d))
    while (D(float(x)) - (D(float(m)) - d)) * side < 0:  # (rounded away from the border)
        x = np.nextafter(x, np.float32(side * np.inf))
    exact = (D(float(u)) * (1 + (D(float(x)) - D(float(m))).exp()) - 1) / UNIT
    assert off(float(u)) <= abs(exact) < off(float(u)) + 1, exact
    return float(m), float(x), float(u), int(exact > 0)


@pytest.mark.parametrize("parts", [16, 32, 64, 37])
@pytest.mark.parametrize("side", [1, -1])
def test_random_numbers_next_to_a_border(parts, side):
    """Weights at the middles of a halving's parts, where a series about their ends is off most."""
    from aero_b200.logits import sample
    with decimal.localcontext() as c:
        c.prec = 60
        rows = [row((k + 0.5) / parts, side) for k in range(parts)]
    m, x, u, want = (list(v) for v in zip(*rows))
    assert all(a > b for a, b in zip(m, x)) and all(w == (side > 0) for w in want)
    logits = torch.tensor([m, x], device="cuda").T.contiguous()
    got = sample(logits, torch.tensor(u, device="cuda")).tolist()
    assert got == want, [k for k in range(parts) if got[k] != want[k]]
    # the other way round, with what is never drawn beside them
    wide = torch.full((parts, 5000), -math.inf, device="cuda")
    wide[:, 4000] = logits[:, 0]
    wide[:, 77] = logits[:, 1]
    got = sample(wide, torch.tensor(u, device="cuda")).tolist()
    assert got == [77 if w else 4000 for w in want]
