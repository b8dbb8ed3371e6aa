"""The rotary table against frequencies in 50 digits: every entry within
2^-63 turns per position, so that an angle is exact to 32 bits at any position
below 2^30 (2^-33 turns)."""

from __future__ import annotations

import math
from decimal import Decimal, getcontext

import pytest

from cybel_b200.paged_attention import RopeTable

getcontext().prec = 50
TWO_PI = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494")


def _exact(rot, theta, scaling, factor=1.0, original=0, low=1.0, high=4.0):
    theta, factor, low, high = (Decimal(x) for x in (theta, factor, low, high))
    out = []
    for p in range(rot // 2):
        f = (theta.ln() * (-2 * p) / rot).exp()
        if scaling == "linear":
            f /= factor
        elif scaling == "llama3":
            t = min(Decimal(1), max(Decimal(0), (original * f / TWO_PI - low) / (high - low)))
            f = (1 - t) * f / factor + t * f
        elif scaling == "yarn":
            def at(beta):
                return rot * (original / (beta * TWO_PI)).ln() / (2 * theta.ln())

            a, b = max(0, math.floor(at(high))), min(rot - 1, math.ceil(at(low)))
            b = b if b > a else a + Decimal("0.001")
            t = min(Decimal(1), max(Decimal(0), (p - a) / Decimal(b - a)))
            f = f / factor * t + f * (1 - t)
        out.append(f / TWO_PI)
    return out


@pytest.mark.parametrize("rot", [2, 34, 64, 128, 256])
@pytest.mark.parametrize("theta", [10000.0, 500000.0, 1.5])
@pytest.mark.parametrize("scaling,kw", [("none", {}), ("linear", dict(factor=3.0)),
                                        ("llama3", dict(factor=8.0, original_context=8192)),
                                        ("yarn", dict(factor=32.0, original_context=4096))])
def test_every_entry(rot, theta, scaling, kw):
    t = RopeTable(rot, theta, scaling=scaling, device="cpu", **kw)
    want = _exact(rot, theta, scaling, kw.get("factor", 1.0), kw.get("original_context", 0),
                  high=32.0 if scaling == "yarn" else 4.0)
    for p, w in enumerate(want):
        off = abs(Decimal(int(t.turns_host[p])) / 2 ** 64 - w)
        assert off <= Decimal(2) ** -63, (p, float(off))
