"""The fit of the polynomials in csrc/gelu.cuh: P(z) near log2 Phi(-z), Phi the normal distribution function, so that
GELU(x) = max(x, 0) - z 2^P(z), z = |x|. Prints their coefficients, of (-z)^i (needs numpy and scipy).

P minimises the largest w(z) |P(z) - log2 Phi(-z)| on [0, 5.6] by linear programming, w = ln 2 max(z Phi(-z), the weight
that keeps small results' relative error small): the error of z 2^P. From 5.6 to 14 it only has to fall as the logarithm
does, within -0.05 (z - 5)^2 - 0.5 and 0.06 (z - 5.5)^2 + 0.3 of it, and to be below -130 from 13.9 on, where 2^P is 0."""
import numpy as np
from scipy.optimize import linprog
from scipy.special import log_ndtr

LN2 = np.log(2.0)
CLAMP = 14.0
#: degree, and the weight near 0 as f exp(-(z / s)^2)
KINDS = {"fast": (6, 0.1, 1.0), "fine": (10, 0.2, 1.5)}


def log2_phi(z):
    return log_ndtr(-z) / LN2


def weight(z, f, s):
    return LN2 * np.maximum(z * np.exp(log_ndtr(-z)), f * np.exp(-(z / s) ** 2))


def tail_bounds(z):
    t = log2_phi(z)
    return t - 0.05 * (z - 5.0) ** 2 - 0.5, np.where(z < CLAMP - 0.1, t + 0.06 * (z - 5.5) ** 2 + 0.3, -130.0)


def fit(kind):
    """(coefficients of (-z)^i, the largest weighted error)."""
    degree, f, s = KINDS[kind]
    z, far = np.linspace(0, 5.6, 1200), np.linspace(5.6, CLAMP, 169)
    v, vf = (np.vander(-a, degree + 1, increasing=True) for a in (z, far))
    scale = np.maximum(np.abs(v).max(0), np.abs(vf).max(0))
    w, t, (lo, hi), k = weight(z, f, s), log2_phi(z), tail_bounds(far), 1e7
    top = np.hstack([v / scale * w[:, None] * k, -np.ones((len(z), 1))])
    low = np.hstack([-v / scale * w[:, None] * k, -np.ones((len(z), 1))])
    up, down = (np.hstack([c * vf / scale, np.zeros((len(far), 1))]) for c in (1, -1))
    r = linprog(np.r_[np.zeros(degree + 1), 1.0], A_ub=np.vstack([top, low, up, down]),
                b_ub=np.concatenate([t * w * k, -t * w * k, hi, -lo]), bounds=[(None, None)] * (degree + 1) + [(0, None)],
                method="highs")
    assert r.status == 0, r.message
    return r.x[:-1] / scale, r.x[-1] / k


if __name__ == "__main__":
    for name in KINDS:
        c, e = fit(name)
        print(name, f"{e:.3e}", ", ".join(f"{np.float32(a):.9g}f" for a in c))
