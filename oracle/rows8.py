"""The 8-bit row operators in 64 bits, for the tests. TEST INFRASTRUCTURE ONLY, like oracle.py.

Every function takes arrays of the values that the operator reads (already rounded to the types it reads them in) and
computes in float64 from the definition; ``quantize`` is the exception: its scale is a defined fp32 number."""
from __future__ import annotations

import numpy as np

F64 = np.float64
TINY = np.float32(2.0 ** -126)


def bf16(x):
    """The nearest bf16 values (ties to even) of a float32 array, as float32."""
    b = np.ascontiguousarray(x, dtype=np.float32).view(np.uint32)
    r = ((b.astype(np.uint64) + 0x7FFF + ((b >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(x), np.float32(np.nan), r)


def scale_of(amax):
    """fp32: max(amax / 127, 2^-126), NaN where amax is not finite."""
    amax = np.asarray(amax, dtype=np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        return np.where(np.isfinite(amax), np.maximum(amax / np.float32(127), TINY), np.float32(np.nan)).astype(np.float32)


def quantize(x):
    """(q float64, scale fp32) of rows x (rows, features). q is the quotient by the scale before its rounding to fp32."""
    x = np.asarray(x, dtype=np.float32)
    a = np.abs(x).max(-1)
    s = scale_of(a)
    with np.errstate(invalid="ignore"):
        q = np.rint(127.0 * x.astype(F64) / np.maximum(a.astype(F64), 127.0 * 2.0 ** -126)[:, None])
    return np.where(np.isnan(q), 0.0, q), s


def rmsnorm(x, residual, gamma, eps):
    """(h, rstd, y) of rows."""
    h = np.asarray(x, dtype=F64) + (0.0 if residual is None else np.asarray(residual, dtype=F64))
    rstd = 1.0 / np.sqrt((h * h).mean(-1) + eps)
    return h, rstd, h * rstd[:, None] * (1.0 if gamma is None else np.asarray(gamma, dtype=F64))


def act(v, name):
    if name == "gelu":
        return 0.5 * v * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (v + 0.044715 * v ** 3)))
    if name == "silu":
        return v / (1.0 + np.exp(-v))
    if name == "relu":
        return np.where(v < 0, 0.0, v)
    return v


def linear(xq, xs, wq, ws, bias, name):
    """act(s_x s_w x_q W_q^T + b) from the integers and the scales."""
    acc = np.asarray(xq, dtype=F64) @ np.asarray(wq, dtype=F64).T
    v = acc * np.asarray(xs, dtype=F64)[:, None] * np.asarray(ws, dtype=F64)
    return act(v if bias is None else v + np.asarray(bias, dtype=F64), name)


def linear_backward(grad, x, w):
    """(grad_x, grad_w, grad_b) of y = x W^T + b."""
    g, x, w = (np.asarray(t, dtype=F64) for t in (grad, x, w))
    return g @ w, g.T @ x, g.sum(0)


def rmsnorm_backward(grad, h, rstd, gamma, grad_residual):
    """(grad_h, grad_gamma): n = h rstd, rstd (g - n mean(g n)) + grad_residual with g = grad gamma, sum grad n."""
    grad, h = np.asarray(grad, dtype=F64), np.asarray(h, dtype=F64)
    r = np.asarray(rstd, dtype=F64)[:, None]
    n = h * r
    g = grad * (1.0 if gamma is None else np.asarray(gamma, dtype=F64))
    gh = r * (g - n * (g * n).mean(-1, keepdims=True))
    return gh + (0.0 if grad_residual is None else np.asarray(grad_residual, dtype=F64)), (grad * n).sum(0)
