"""By-band scaling against its formula, evaluated apart from the code in 60 decimal digits:

    theta_i = base^(-2 i / d), turns r = L0 theta_i / (2 pi), g = clamp((r - slow) / (fast - slow), 0, 1),
    theta'_i = theta_i (g + (1 - g) / factor)

Tolerance: the exponent and the power err by a few 2^-53 each, the exponent's times ln(base) (at most 13), the ramp and the
sum by a few 2^-53 more, all relative: 64 x 2^-53 is enough for any order of the operations."""
import math
from decimal import Decimal, getcontext

import pytest

from lockstep_b200 import rotary as R

getcontext().prec = 60
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494")

CASES = [  # rotary_dim, base, factor, original, fast, slow
    (128, 10000.0, 32.0, 8192, 32.0, 1.0),
    (64, 500000.0, 8.0, 4096, 4.0, 1.0),
    (32, 10000.0, 4.0, 128, 32.0, 1.0),                # no pair is fast enough to be kept
    (256, 10000.0, 16.0, 1 << 20, 64.0, 0.5),
    (2, 10000.0, 2.0, 100, 32.0, 1.0),
]
# some values as they stand, so that the formula here cannot drift along with the code
PINNED = {(128, 25): 0.027384196342643614, (128, 26): 0.022911846811876101, (128, 30): 0.0072453621326395894,
          (128, 40): 0.00040743665431525205, (128, 49): 3.0553438774079709e-05, (128, 63): 3.6086937021545569e-06,
          (64, 15): 0.00050835348913790533, (64, 16): 0.00017677669529663688, (32, 0): 0.71867337215554683,
          (32, 3): 0.05574051687839747, (32, 5): 0.014256611975921029}


def by_formula(d, base, factor, original, fast, slow):
    out = []
    for i in range(d // 2):
        t = (-(Decimal(2 * i) / d) * Decimal(base).ln()).exp()
        g = (original * t / (2 * PI) - Decimal(slow)) / (Decimal(fast) - Decimal(slow))
        g = min(Decimal(1), max(Decimal(0), g))
        out.append(float(t * (g + (1 - g) / Decimal(factor))))
    return out


@pytest.mark.parametrize("d,base,factor,original,fast,slow", CASES)
def test_ramp(d, base, factor, original, fast, slow):
    scaling = {"kind": "bands", "factor": factor, "original": original, "fast": fast, "slow": slow}
    got, m = R.frequencies(d, base, scaling)
    want = by_formula(d, base, factor, original, fast, slow)
    tol = 64 * 2.0 ** -53
    for i, (a, b) in enumerate(zip(got, want)):
        assert math.isclose(a, b, rel_tol=tol), i
        assert (d, i) not in PINNED or math.isclose(a, PINNED[d, i], rel_tol=tol)
    assert math.isclose(m, 0.1 * math.log(factor) + 1.0)
    plan = R.make_plan(max(d, 8), d, base=base, scaling=scaling, device="cpu")
    for f, b in zip(plan.freq.tolist(), want):
        assert abs((f % (1 << 64)) - b / (2 * math.pi) * 2.0 ** 64) <= tol * 2.0 ** 64 * b / (2 * math.pi) + 1
