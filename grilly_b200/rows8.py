"""Rows in 8 bits: int8 values with one fp32 scale per row, and the operators of ``Compute().fnn`` on them.

A layer's input is written once in 8 bits (by :meth:`~Rows8Ops.quantize_rows`, or by the norm before the layer,
:meth:`~Rows8Ops.rmsnorm_residual_q8`), multiplied with weights in 8 bits (:meth:`~Rows8Ops.linear_q8`) and, in
training, kept instead of the 16- or 32-bit activation for the backward pass (:meth:`~Rows8Ops.linear_backward_q8`,
:meth:`~Rows8Ops.rmsnorm_backward_q8`). The reference has no 8-bit type; these stand beside its ``linear``, RMSNorm and
backward methods (backend/fnn.py:1394-1573, snn-rmsnorm.glsl:34-75).
"""
from __future__ import annotations

import math
from collections import namedtuple

import numpy as np

from . import _lib as L
from .device import DeviceTensor

_ACT = {None: L.ACT_NONE, "none": L.ACT_NONE, "gelu": L.ACT_GELU, "silu": L.ACT_SILU, "relu": L.ACT_RELU}
_FLOAT = ("f32", "bf16")

NormQ8 = namedtuple("NormQ8", "y8 h h8 rstd")
NormQ8.__doc__ = """What ``rmsnorm_residual_q8`` gives: the norm's output in 8-bit rows, the sum it was taken of, and, with
``keep``, that sum in 8-bit rows and 1 / root-mean-square of every row (else None) for ``rmsnorm_backward_q8``."""


def _check_shape(shape):
    if len(shape) < 1 or shape[-1] < 1 or min(shape) < 0:
        raise ValueError(f"8-bit rows need a shape (..., features) with at least one feature, not {shape}")


class Rows8:
    """A tensor of ``shape`` (..., features) in 8-bit rows on the device: element (r, c) stands for ``q[r, c] * scale[r]``.

    ``q`` is an 'i8' :class:`DeviceTensor` (rows, ld) with ld a multiple of 16 of at least ``features`` (what lies between
    is never used), ``scale`` an 'f32' one with one entry per row. A row whose scale is NaN stands for NaN."""

    __slots__ = ("q", "scale", "shape", "dev", "rows", "features", "ld")

    def __init__(self, q: DeviceTensor, scale: DeviceTensor, shape):
        shape = tuple(map(int, shape))
        _check_shape(shape)
        rows = math.prod(shape[:-1])
        features = shape[-1]
        if q.dtype != "i8" or len(q.shape) != 2 or scale.dtype != "f32":
            raise ValueError("q must be an 'i8' tensor (rows, ld), scale an 'f32' tensor")
        held, ld = q.shape
        if held != rows or (scale.shape != (rows,) and scale.size != rows):
            raise ValueError(f"q has {held} rows and scale {scale.size} entries, shape {shape} needs {rows}")
        if ld % 16 or ld < features:
            raise ValueError(f"q's row length {ld} must be a multiple of 16 and at least {features}")
        if q.dev is not scale.dev:
            raise ValueError("q and scale belong to different contexts")
        self.q = q
        self.scale = scale
        self.shape = shape
        self.dev = q.dev
        self.rows = rows
        self.features = features
        self.ld = ld

    @classmethod
    def empty(cls, dev, shape) -> "Rows8":
        """Uninitialised 8-bit rows in the pool of ``dev``, to be written by an operator."""
        shape = tuple(map(int, shape))
        _check_shape(shape)
        rows = math.prod(shape[:-1])
        return cls(dev.empty((rows, (shape[-1] + 15) // 16 * 16), "i8"), dev.empty((rows,)), shape)

    @property
    def nbytes(self) -> int:
        return self.q.nbytes + self.scale.nbytes

    def numpy(self) -> np.ndarray:
        """The values as a float32 array."""
        q = self.q.numpy()[:, : self.features].astype(np.float32)
        return (q * self.scale.numpy()[:, None]).reshape(self.shape)

    def free(self) -> None:
        self.q.free()
        self.scale.free()


def _ptr(t):
    return None if t is None else t.ptr


class Rows8Ops:
    """The 8-bit row methods of :class:`~grilly_b200.compute.FNN`.

    Floating operands are NumPy arrays (copied to the device in every call, nothing is cached) or 'f32' / 'bf16'
    DeviceTensors of this backend's context; with a NumPy operand the floating results are NumPy arrays. ``out`` takes
    the result's tensors, so that a call allocates nothing; a call that is captured into a CUDA graph needs it."""

    # ---- operands (checked in every call: kept short) -----------------------------------------
    def _float_in(self, x, name, host_dtype="f32"):
        """-> (DeviceTensor, came from the host)."""
        if isinstance(x, DeviceTensor):
            if x.dtype not in _FLOAT:
                raise ValueError(f"{name} must be f32 or bf16, not {x.dtype}")
            if x.dev is not self.dev:
                raise ValueError(f"{name} belongs to another context")
            return x, False
        return self.dev.upload(np.asarray(x, dtype=np.float32), host_dtype), True

    def _f32_vector(self, v, n, name):
        """A small fp32 vector of n entries (bias, gamma, rstd) on the device, or None."""
        if v is None:
            return None
        if isinstance(v, DeviceTensor):
            if v.dtype != "f32":
                raise ValueError(f"{name} must be f32, not {v.dtype}")
            if v.dev is not self.dev:
                raise ValueError(f"{name} belongs to another context")
            if v.shape != (n,) and v.size != n:
                raise ValueError(f"{name} has {v.size} entries, expected {n}")
            return v
        v = np.asarray(v, dtype=np.float32)
        if v.size != n:
            raise ValueError(f"{name} has {v.size} entries, expected {n}")
        return self.dev.upload(v.reshape(-1))

    def _rows8_in(self, x, name):
        if not isinstance(x, Rows8):
            raise TypeError(f"{name} must be 8-bit rows (Rows8), see quantize_rows")
        if x.dev is not self.dev:
            raise ValueError(f"{name} belongs to another context")
        return x

    def _rows8_out(self, out, shape, name="out"):
        if out is None:
            return Rows8.empty(self.dev, shape)
        if not isinstance(out, Rows8) or out.dev is not self.dev or out.shape != shape:
            self._rows8_in(out, name)
            raise ValueError(f"{name} has shape {out.shape}, expected {shape}")
        return out

    def _float_out(self, out, shape, dtype, name="out"):
        """``dtype``: the type of a new tensor, or of one that the caller brings (a tuple: the types it may have)."""
        if out is None:
            return self.dev.empty(shape, dtype)
        if not isinstance(out, DeviceTensor) or out.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
            raise ValueError(f"{name} must be a DeviceTensor of type {dtype}")
        if out.dev is not self.dev:
            raise ValueError(f"{name} belongs to another context")
        if out.shape != shape:
            raise ValueError(f"{name} has shape {out.shape}, expected {shape}")
        return out

    @staticmethod
    def _shape(x, name):
        shape = x.shape if isinstance(x, DeviceTensor) else tuple(map(int, np.shape(x)))
        if not shape or shape[-1] < 1:
            raise ValueError(f"{name} must be (..., features) with at least one feature, not {shape}")
        return shape

    # ---- operators --------------------------------------------------------------------------
    def quantize_rows(self, x, out=None) -> Rows8:
        """``x`` (..., features) in 8-bit rows: per row scale = max|x| / 127 (at least 2^-126) and x / scale rounded to the
        nearest integer, ties to even (a tie is one of x / (max|x| / 127); of fp32 values also what lies within 2^-18 of one),
        so q * scale is off by at most half a step and the scale's own rounding, (1/2 + 2^-16) scale. A row with a NaN or an
        infinity reads back as NaN. An activation's checkpoint, or a weight (out, in) with one scale per output channel for
        ``linear_q8``."""
        shape = self._shape(x, "x")
        y8 = self._rows8_out(out, shape)
        xd, _ = self._float_in(x, "x")
        self.dev.check(self.lib.grilly_quantize_rows(self.ctx, xd.ptr, y8.q.ptr, y8.scale.ptr, y8.rows, y8.features, y8.ld,
                                                     L.FLAG_IN_BF16 if xd.dtype == "bf16" else 0))
        return y8

    def dequantize_rows(self, x8: Rows8, dtype="f32", out=None) -> DeviceTensor:
        """The values of 8-bit rows as an 'f32' or 'bf16' DeviceTensor of their shape: the fp32 product q * scale, for bf16
        rounded to that."""
        self._rows8_in(x8, "x8")
        if dtype not in _FLOAT:
            raise ValueError("dtype must be 'f32' or 'bf16'")
        y = self._float_out(out, x8.shape, dtype if out is None else _FLOAT)
        self.dev.check(self.lib.grilly_dequantize_rows(self.ctx, x8.q.ptr, x8.scale.ptr, y.ptr, x8.rows, x8.features, x8.ld,
                                                       L.FLAG_OUT_BF16 if y.dtype == "bf16" else 0))
        return y

    def rmsnorm_residual_q8(self, x, residual=None, gamma=None, eps=1e-5, keep=False, out=None) -> NormQ8:
        """h = x + residual and RMSNorm(h) * gamma in 8-bit rows, in one pass over the rows (``residual`` then ``rmsnorm``,
        with 8 bits written instead of 32). ``keep`` also gives what ``rmsnorm_backward_q8`` needs: h in 8-bit rows and
        the rows' 1 / sqrt(mean(h^2) + eps). The statistics and y come from the unrounded fp32 sum. A row of y with a value
        that is not finite (by gamma, say) reads back as NaN; h, h8 and rstd depend on h alone.

        x and residual share shape and type; h has that type too. ``out`` = (y8, h, h8, rstd), each None for a new
        tensor; h may be x or residual (in place), h8 and rstd belong to ``keep``."""
        shape = self._shape(x, "x")
        F = shape[-1]
        if residual is not None and self._shape(residual, "residual") != shape:
            raise ValueError(f"residual must have shape {shape}")
        if not 0.0 < eps < math.inf:
            raise ValueError("eps must be positive and finite")
        if isinstance(residual, DeviceTensor) and isinstance(x, DeviceTensor) and residual.dtype != x.dtype:
            raise ValueError(f"x is {x.dtype} and residual {residual.dtype}: they must have one type")
        y8_out, h_out, h8_out, rstd_out = out if out is not None else (None,) * 4
        if not keep and (h8_out is not None or rstd_out is not None):
            raise ValueError("h8 and rstd are written with keep=True only")
        gd = self._f32_vector(gamma, F, "gamma")
        other = residual if isinstance(residual, DeviceTensor) else x
        host_dtype = other.dtype if isinstance(other, DeviceTensor) else "f32"
        xd, host_x = self._float_in(x, "x", host_dtype)
        rd, host_r = self._float_in(residual, "residual", host_dtype) if residual is not None else (None, False)
        y8 = self._rows8_out(y8_out, shape, "out y8")
        h = self._float_out(h_out, shape, xd.dtype, "out h")
        h8 = rstd = None
        if keep:
            h8 = self._rows8_out(h8_out, shape, "out h8")
            rstd = self._float_out(rstd_out, (y8.rows,), "f32", "out rstd")
            if h8.ld != y8.ld:
                raise ValueError("out y8 and h8 must have rows of the same length")
        self.dev.check(self.lib.grilly_rmsnorm_residual_q8(
            self.ctx, xd.ptr, _ptr(rd), _ptr(gd), h.ptr, y8.q.ptr, y8.scale.ptr, h8.q.ptr if keep else None,
            h8.scale.ptr if keep else None, _ptr(rstd), y8.rows, F, y8.ld, float(eps), L.FLAG_IN_BF16 if xd.dtype == "bf16" else 0))
        return NormQ8(y8, h.numpy() if (host_x or host_r) and h_out is None else h, h8, rstd)

    def linear_q8(self, x, weights, bias=None, act=None, dtype="f32", out=None):
        """act(x @ W.T + b) on 8-bit rows: int8 products, exact 32-bit sums, then the token's and the channel's scale, the
        bias and the activation (None, 'gelu', 'silu', 'relu') in fp32, rounded to ``dtype`` ('f32' or 'bf16') at the end.

        ``x`` and ``weights`` (out, in) are Rows8; an array or a floating DeviceTensor is quantised in this call (keep
        ``quantize_rows(weights)`` to do that once). At most 131071 input features; rows of |x| above 2^104 may leave fp32's
        range before the channel's scale brings them back."""
        if act not in _ACT:
            raise ValueError("act must be None, 'gelu', 'silu' or 'relu'")
        if dtype not in _FLOAT:
            raise ValueError("dtype must be 'f32' or 'bf16'")
        x_shape = self._rows8_in(x, "x").shape if isinstance(x, Rows8) else self._shape(x, "x")
        w_shape = self._rows8_in(weights, "weights").shape if isinstance(weights, Rows8) else self._shape(weights, "weights")
        if len(w_shape) != 2 or w_shape[0] < 1:
            raise ValueError("weights must be 2-D (out_features, in_features)")
        N, K = w_shape
        if x_shape[-1] != K:
            raise ValueError(f"input feature size {x_shape[-1]} does not match weights {tuple(w_shape)}")
        if K > 131071:
            raise ValueError("linear_q8 takes at most 131071 input features: more could overflow the 32-bit sums")
        bd = self._f32_vector(bias, N, "bias")
        y = self._float_out(out, x_shape[:-1] + (N,), dtype if out is None else _FLOAT)
        host = not isinstance(x, (Rows8, DeviceTensor))
        x8 = x if isinstance(x, Rows8) else self.quantize_rows(x)
        w8 = weights if isinstance(weights, Rows8) else self.quantize_rows(weights)
        self.dev.check(self.lib.grilly_linear_q8(self.ctx, x8.q.ptr, x8.scale.ptr, w8.q.ptr, w8.scale.ptr, _ptr(bd), y.ptr, x8.rows, N, K,
                                                 x8.ld, w8.ld, _ACT[act], L.FLAG_OUT_BF16 if y.dtype == "bf16" else 0))
        return y.numpy() if host and out is None else y

    def linear_backward_q8(self, grad_output, x8: Rows8, weights, dtype="bf16", out=None):
        """(grad_input, grad_weight, grad_bias) of y = x W^T + b (``linear_backward``) with the layer's input x kept in 8-bit
        rows. The products run in bf16 with fp32 sums: grad_output (..., out) and weights (out, in) are bf16 DeviceTensors
        or arrays (rounded to bf16 on the way in), x enters as its values rounded to bf16, which is far below the
        checkpoint's own half step. grad_input and grad_weight have type ``dtype``, grad_bias is fp32.

        ``out`` = (grad_input, grad_weight, grad_bias), each None for a new tensor."""
        self._rows8_in(x8, "x8")
        if dtype not in _FLOAT:
            raise ValueError("dtype must be 'f32' or 'bf16'")
        g_shape, w_shape = self._shape(grad_output, "grad_output"), self._shape(weights, "weights")
        if len(w_shape) != 2 or w_shape[0] < 1:
            raise ValueError("weights must be 2-D (out_features, in_features)")
        N, K = w_shape
        if x8.features != K:
            raise ValueError(f"input feature size {x8.features} does not match weights {tuple(w_shape)}")
        if g_shape != x8.shape[:-1] + (N,):
            raise ValueError(f"grad_output must have shape {x8.shape[:-1] + (N,)}")
        for t, name in ((grad_output, "grad_output"), (weights, "weights")):
            if isinstance(t, DeviceTensor) and t.dtype != "bf16":
                raise ValueError(f"{name} must be bf16, not {t.dtype}")
        gx_out, gw_out, gb_out = out if out is not None else (None,) * 3
        for t in (gx_out, gw_out):
            if isinstance(t, DeviceTensor):
                dtype = t.dtype
        if dtype not in _FLOAT:
            raise ValueError(f"out grad_input and grad_weight must be f32 or bf16, not {dtype}")
        gx = self._float_out(gx_out, x8.shape, dtype, "out grad_input")
        gw = self._float_out(gw_out, (N, K), dtype, "out grad_weight")
        gb = self._float_out(gb_out, (N,), "f32", "out grad_bias")
        god, host_g = self._float_in(grad_output, "grad_output", "bf16")
        wd, host_w = self._float_in(weights, "weights", "bf16")
        self.dev.check(self.lib.grilly_linear_backward_q8(self.ctx, god.ptr, x8.q.ptr, x8.scale.ptr, wd.ptr, gx.ptr, gw.ptr, gb.ptr, x8.rows, N, K,
                                                          x8.ld, L.FLAG_OUT_BF16 if dtype == "bf16" else 0))
        if (host_g or host_w) and out is None:
            return gx.numpy(), gw.numpy(), gb.numpy()
        return gx, gw, gb

    def rmsnorm_backward_q8(self, grad_output, h8: Rows8, rstd, gamma=None, grad_residual=None, out=None):
        """(grad_h, grad_gamma) of ``rmsnorm_residual_q8`` from its checkpoint (``keep=True``): with n = h rstd and
        g = grad_output gamma, grad_h = rstd (g - n mean(g n)) + grad_residual and grad_gamma = sum over rows of
        grad_output n. ``grad_residual`` is the gradient that reaches h past the norm; grad_h is the gradient of both x
        and residual. Types: grad_output, grad_residual and grad_h share one, grad_gamma is fp32.

        ``out`` = (grad_h, grad_gamma), each None for a new tensor; grad_h may be grad_output or grad_residual."""
        self._rows8_in(h8, "h8")
        shape, F = h8.shape, h8.features
        for t, name in ((grad_output, "grad_output"), (grad_residual, "grad_residual")):
            if t is not None and self._shape(t, name) != shape:
                raise ValueError(f"{name} must have shape {shape}")
        if isinstance(grad_residual, DeviceTensor) and isinstance(grad_output, DeviceTensor) and grad_residual.dtype != grad_output.dtype:
            raise ValueError(f"grad_output is {grad_output.dtype} and grad_residual {grad_residual.dtype}: they must have one type")
        gh_out, gg_out = out if out is not None else (None, None)
        if rstd is None:
            raise ValueError("rstd is required: rmsnorm_residual_q8 gives it with keep=True")
        rs = self._f32_vector(rstd, h8.rows, "rstd")
        gd = self._f32_vector(gamma, F, "gamma")
        other = grad_residual if isinstance(grad_residual, DeviceTensor) else grad_output
        host_dtype = other.dtype if isinstance(other, DeviceTensor) else "f32"
        god, host_g = self._float_in(grad_output, "grad_output", host_dtype)
        grd, host_r = self._float_in(grad_residual, "grad_residual", host_dtype) if grad_residual is not None else (None, False)
        gh = self._float_out(gh_out, shape, god.dtype, "out grad_h")
        gg = self._float_out(gg_out, (F,), "f32", "out grad_gamma")
        self.dev.check(self.lib.grilly_rmsnorm_backward_q8(
            self.ctx, god.ptr, h8.q.ptr, h8.scale.ptr, rs.ptr, _ptr(gd), _ptr(grd), gh.ptr, gg.ptr, h8.rows, F, h8.ld,
            L.FLAG_IN_BF16 if god.dtype == "bf16" else 0))
        if (host_g or host_r) and out is None:
            return gh.numpy(), gg.numpy()
        return gh, gg
