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
