"""Gradient norm, clipping and the clipped Adam update in float64 on the CPU, with bounds on a float32
evaluation (u = 2^-24, half a float32 step).

The factor c = min(1, max_norm / (norm + 1e-6)) from a norm rounded to float32: the norm, max_norm, the
sum and the quotient round once each, so c is within 4u and c g, rounded to the gradient's type, within
4u + (eps of the type) / 2 of it, or half the type's smallest step.
"""
import math

import torch

U = 2.0 ** -24


def norm(grads):
    return math.sqrt(sum(float(g.double().pow(2).sum()) for g in grads))


def factor(n, max_norm):
    return min(1.0, max_norm / (n + 1e-6))


def scaled(g, c):
    """(c g in float64, bound)"""
    fi = torch.finfo(g.dtype)
    r = g.double() * c
    own = 4 * U if g.dtype == torch.float32 else 5 * U
    return r, r.abs() * (own + fi.eps / 2) * 1.01 + fi.smallest_normal * fi.eps / 2


def adam(p, g, m, v, c, t, lr, b1, b2, eps):
    """(p, m, v) after step t on c g, and their bounds. g' = c g: 5u. m: w1 (g' - m) rounds in w1, the
    difference and the product, then the sum; v: 10u from g'^2 and four roundings, then the sum; the step:
    half of v's bound through the root, and six roundings more."""
    p, g, m, v = (x.double() for x in (p, g, m, v))
    g = g * c
    m2 = m + (1 - b1) * (g - m)
    v2 = b2 * v + (1 - b2) * g * g
    den = v2.sqrt() / math.sqrt(1 - b2 ** t) + eps
    step = lr / (1 - b1 ** t) * m2 / den
    tiny = 2.0 ** -148
    dm = U * ((1 - b1) * 9 * (g.abs() + m.abs()) + 2 * m2.abs()) + tiny
    dv = 16 * U * v2 + tiny
    dp = (lr / (1 - b1 ** t)) / den * dm + 18 * U * step.abs() + U * (p.abs() + step.abs()) + tiny
    return (p - step, m2, v2), (dp, dm, dv)
