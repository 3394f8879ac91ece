"""Layer norm and RMS norm for B200, forward and backward (the gated RMSNorm of the gated-delta-net path is ``gdn.gated_rmsnorm``).

    y = (x - mean) * rstd * weight + bias,   rstd = 1 / sqrt(var + eps)                                  layer_norm
    h = round(x + residual),   y = h * rstd * weight,   rstd = 1 / sqrt(mean(h^2) + eps)                 rms_norm

over the last dimension (1 to 28672 elements).  ``x`` is bf16, fp16 or fp32; ``weight`` and ``bias`` have its dtype or fp32.  Sums and
statistics are fp32, results are rounded once.  Rows that are evenly spaced and contiguous are read as they are; others are copied first.
Rows of a whole number of 16-byte pieces on 16-byte boundaries take wide loads, others go element by element.  Errors are ValueError, as
in the reference's kernel library (python/avelang_kernels/amdgpu_gemm.py:463-486).  Rows that a bounded wait on the device has given up on are NaN in all their results, and so are
the columns of the gradients of weight and bias that miss elements of them; ``gdn.read_status()`` says so.  (The RMS norm's kernels wait for nothing but their own loads.)
"""
from __future__ import annotations

import torch

from . import _lib, torch_ops  # noqa: F401  (torch_ops declares the operators the native functions call)

__all__ = ["layer_norm", "layer_norm_backward", "LayerNormFunction", "rms_norm", "rms_norm_backward", "rms_norm_int8", "RmsNormFunction"]

_native = _lib.host
_lib.register_operators()


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, return_stats=False, out=None):
    """Returns ``y``, or with ``return_stats`` ``(y, mean, rstd)``, the statistics fp32 in the leading shape of ``x``.  ``out`` may be ``x``;
    one that shares some of its elements in another way is refused."""
    return _native.layer_norm(x, weight, bias, eps, return_stats, out)


def layer_norm_backward(d_y, x, mean, rstd, weight=None):
    """Gradients ``(dx, dweight, dbias)`` of ``layer_norm`` from its saved statistics; dweight and dbias, in the dtype of ``weight``, are
    sums over all rows in a fixed order (None without a weight)."""
    return _native.layer_norm_backward(d_y, x, mean, rstd, weight)


class LayerNormFunction(torch.autograd.Function):
    """``y = LayerNormFunction.apply(x, weight, bias, eps)``: ``layer_norm`` with its backward pass attached (weight and bias may be None).
    It can be differentiated once.  A step with its backward pass can be captured into a CUDA graph once the results of eager steps on the same leaves are gone."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = layer_norm(x, weight, bias, eps, return_stats=True)
        ctx.save_for_backward(x, mean, rstd, weight)
        ctx.has_bias = bias is not None
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y):
        x, mean, rstd, weight = ctx.saved_tensors
        dx, dw, db = layer_norm_backward(d_y, x, mean, rstd, weight)
        return dx, dw, db if ctx.has_bias else None, None


def rms_norm(x, weight=None, eps=1e-6, *, residual=None, zero_centered=False, return_stats=False, out=None, sum_out=None):
    """Returns ``y``; with ``residual`` (of the shape and dtype of ``x``) ``(y, h)``, where ``h`` is the sum as it is rounded to that dtype and
    as the norm takes it; with ``return_stats`` ``rstd`` (fp32, in the leading shape of ``x``) behind them.  ``zero_centered``: the weight is
    ``1 + weight``, the sum formed in fp32.  ``out`` and ``sum_out`` may each be ``x`` or ``residual``; those that share some of their elements
    in another way are refused."""
    return _native.rms_norm(x, weight, eps, residual, zero_centered, return_stats, out, sum_out)


def rms_norm_int8(x, weight=None, eps=1e-6, *, residual=None, zero_centered=False, sum_out=None):
    """``rms_norm`` with each row of the result in 8 bits: ``(q, scale)``, or ``(q, scale, h)`` with ``residual``, as
    ``gemm.gemm_int8_transposed_b`` takes them.  ``scale`` (fp32, in the leading shape of ``x``) is the row's largest ``|y|`` / 127, ``q`` (int8,
    rows a multiple of 16 bytes apart) is ``h * weight`` (in fp32) times 127 / its largest in the row, that factor rounded to fp32, to nearest,
    ties to even: ``y / scale`` but for the factor's rounding; ``y`` itself is not rounded in between.  A row that holds a NaN or an infinity has
    a NaN as its scale and zeros in ``q``; one whose scale would be below the smallest normal number, or whose largest ``|h * weight|`` is below
    3.8e-37, has zeros in both."""
    return _native.rms_norm_int8(x, weight, eps, residual, zero_centered, sum_out)


def rms_norm_backward(d_y, x, rstd, weight=None, *, d_sum=None, zero_centered=False):
    """Gradients ``(dx, dweight)`` of ``rms_norm`` from the rows that it has normalised (``h`` where there was a residual, else ``x``) and its
    ``rstd``.  ``d_sum``, the gradient that reaches ``h`` beside the norm, is added to ``dx``, which is the gradient of ``x`` and of the residual
    alike.  ``dweight``, in the dtype of ``weight``, is a sum over all rows in a fixed order (None without a weight)."""
    return _native.rms_norm_backward(d_y, x, rstd, weight, d_sum, zero_centered)


class RmsNormFunction(torch.autograd.Function):
    """``y, h = RmsNormFunction.apply(x, residual, weight, eps, zero_centered)``: ``rms_norm`` with its backward pass attached; with ``residual`` None it
    returns ``y`` alone (weight may be None).  It can be differentiated once.  A step with its backward pass can be captured into a CUDA graph once
    the results of eager steps on the same leaves are gone."""

    @staticmethod
    def forward(ctx, x, residual, weight, eps, zero_centered=False):
        ctx.set_materialize_grads(False)
        ctx.zero_centered = bool(zero_centered)
        got = rms_norm(x, weight, eps, residual=residual, zero_centered=zero_centered, return_stats=True)
        ctx.save_for_backward(x if residual is None else got[1], got[-1], weight)
        return got[0] if residual is None else got[:2]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y, d_h=None):
        x, rstd, weight = ctx.saved_tensors
        if d_y is None:  # only the sum was used
            return d_h, d_h, None, None, None
        dx, dw = rms_norm_backward(d_y, x, rstd, weight, d_sum=d_h, zero_centered=ctx.zero_centered)
        return dx, dx if ctx.needs_input_grad[1] else None, dw, None, None
