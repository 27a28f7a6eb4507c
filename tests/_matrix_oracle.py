"""The matrix operators in 64 bits on the CPU, as their formulas are written."""
from __future__ import annotations

import math

import torch

COEFFICIENTS = (3.4445, -4.7750, 2.0315)


def momentum(grad, buf, mu, nesterov, scale=1.0):
    """(new momentum, update)."""
    r = grad.double().cpu() / scale
    m = buf.double().cpu()
    m = m + (r - m) * (1.0 - mu)
    return m, (r + (m - r) * mu if nesterov else m)


def orthogonal(u, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = u.double().cpu()
    if x.numel() == 0:
        return x
    x = x / x.square().sum((-2, -1), keepdim=True).sqrt().clamp(min=eps)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    for _ in range(steps):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.transpose(-2, -1) if tall else x


def ratio(rows, cols, how):
    return 0.2 * math.sqrt(max(rows, cols)) if how == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))


def step(param, grad, buf, *, lr, weight_decay=0.1, mu=0.95, nesterov=True, scale=1.0, how=None, row_blocks=1, steps=5):
    """(new parameter, new momentum)."""
    m, u = momentum(grad, buf, mu, nesterov, scale)
    rows, cols = param.shape[-2] // row_blocks, param.shape[-1]
    o = orthogonal(u.reshape(-1, rows, cols), steps).reshape(param.shape)
    return param.double().cpu() * (1.0 - lr * weight_decay) - lr * ratio(rows, cols, how) * o, m


def relative(x, y):
    """Norm of the difference over the norm of ``y`` (of the difference alone where y is 0)."""
    x, y = x.detach().double().cpu(), y.double().cpu()
    n = y.norm().item()
    return (x - y).norm().item() / (n or 1.0)


def half_bound(low, high, steps=5, coefficients=COEFFICIENTS, alike=True):
    """How far products of 11 bits can move the values that singular values of X0 in [``low``, ``high``] are sent to.

    Each rounding is off by at most u = 2^-11 of what it rounds (X's first half, d; A = X X^T, e; B = b A + c A A, f), and moves
    ``x -> a x + b x^3 + c x^5`` by ``x ((b x^2 + 2 c x^4)(2 d + e) + (b x^2 + c x^4)(f + d))``.  A step multiplies what was off before
    by at most the polynomial's largest slope between the value and the one it was moved to: taken over the interval that the bound
    itself spans, so that nothing of second order is left out.  ``alike``: every value is rounded by itself (matrices of one entry in a
    row and column, rank one with entries of one size).  Otherwise (singular values close to each other, entries of any size) the
    roundings of X in the two products need not be the same, and what they put beside a direction is multiplied by f(x) / x.
    u is taken 2^-6 larger, which covers fp32 sums of 4000 terms (l / 32 additions of 2^-24) and X's second half (2^-22).
    """
    a, b, c = coefficients
    u, error = 2.0**-11 * (1 + 2.0**-6), 0.0
    for _ in range(steps):
        x = torch.linspace(max(low - error, 0.0), high + error, 513, dtype=torch.float64)
        in_a, in_b = b * x**2 + 2 * c * x**4, b * x**2 + c * x**4
        moved = (2 * in_a + in_b).abs() + in_a.abs() + in_b.abs() if alike else 3 * in_a.abs() + 2 * in_b.abs()
        slope = (a + 3 * b * x**2 + 5 * c * x**4).abs()
        if not alike:
            slope = torch.maximum(slope, (a + in_b).abs())
        error = slope.max().item() * error + (u * x * moved).max().item()
        exact = torch.linspace(low, high, 513, dtype=torch.float64)
        exact = a * exact + b * exact**3 + c * exact**5
        low, high = exact.min().item(), exact.max().item()
    return error
