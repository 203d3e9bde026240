"""The polynomials of csrc/gelu.cuh against their fit, and GELU with them, restated in fp32, against 64 bits."""
import os
import re

import numpy as np
import pytest
from scipy.special import erfc, log_ndtr

import gelu_fit as fit

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "varda.cpp_b200", "csrc")


def coefficients(kind):
    with open(os.path.join(CSRC, "gelu.cuh")) as f:
        body = re.search(r"kF%s\[\] = \{([^}]*)\}" % kind[1:], f.read()).group(1)
    return np.array([np.float32(v.strip().rstrip("f")) for v in body.split(",")])


def gelu(x, c):
    """(fp32 operations: a product and a sum in 64 bits rounded once are the fused operation's within its rounding)"""
    n, p = np.maximum(-np.abs(x), np.float32(-fit.CLAMP)), np.full_like(x, c[-1])
    fma = lambda a, b, d: (a.astype(np.float64) * b + d).astype(np.float32)  # noqa: E731
    for a in c[-2::-1]:
        p = fma(n, p, a)
    e = np.where(p < -126, 0.0, np.exp2(p.astype(np.float64))).astype(np.float32)  # (ex2 flushes results below the normal ones)
    return fma(n, e, np.maximum(x, 0))


@pytest.mark.parametrize("kind", fit.KINDS)
def test_coefficients_are_the_fit(kind):
    c, (_, best) = coefficients(kind), fit.fit(kind)
    degree, f, s = fit.KINDS[kind]
    z = np.linspace(0, 5.6, 20001)
    v = np.polynomial.polynomial.polyval(-z, c.astype(np.float64))
    w, own = fit.weight(z, f, s), 2.0 ** -24 * np.polynomial.polynomial.polyval(z, np.abs(c.astype(np.float64)))
    assert len(c) == degree + 1
    assert (w * np.abs(v - fit.log2_phi(z)) <= 1.1 * best + w * own).all()  # (own: the coefficients' rounding)
    far = np.linspace(5.6, fit.CLAMP, 2001)
    v = np.polynomial.polynomial.polyval(-far, c.astype(np.float64))
    lo, hi = fit.tail_bounds(far)
    assert (np.diff(v) < 0).all() and v[-1] < -126 and (v >= lo - 0.1).all() and (v[far < 13.8] <= hi[far < 13.8] + 0.1).all()


@pytest.mark.parametrize("kind,worst,rms", [("fast", 2e-7, 1.2e-7), ("fine", 5e-9, 2.0e-8)])
def test_gelu_restated(kind, worst, rms):
    c = coefficients(kind)
    x = np.concatenate([np.linspace(-40, 40, 200001), np.linspace(-15, -5, 20001), np.logspace(-30, 1, 2001), -np.logspace(-30, 1, 2001)])
    x = x.astype(np.float32)
    y, d = gelu(x, c).astype(np.float64), x.astype(np.float64)
    exact, t = 0.5 * d * erfc(-d / np.sqrt(2)), np.abs(d) * np.exp(log_ndtr(-np.abs(d)))
    P = -fit.log2_phi(np.abs(d))
    assert (np.abs(y - exact) <= 2.0 ** -24 * np.abs(exact) + t * (1 + np.log(2) * (1 + P)) * 2.0 ** -22 + worst).all()
    far = d < -5.6
    assert (np.abs(y[far]) <= 16 * np.abs(exact[far]) + 2.0 ** -126).all() and (y[d < -fit.CLAMP] == 0).all()
    n = np.random.default_rng(0).normal(size=10 ** 6).astype(np.float32)
    e = gelu(n, c) - 0.5 * n.astype(np.float64) * erfc(-n.astype(np.float64) / np.sqrt(2))
    assert np.sqrt(np.mean(e * e)) <= rms
