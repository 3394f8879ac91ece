"""Layer norm for B200, forward and backward (the gated RMSNorm of the gated-delta-net path is ``gdn.gated_rmsnorm``).

    y = (x - mean) * rstd * weight + bias,   rstd = 1 / sqrt(var + eps)

over the last dimension (1 to 28672 elements).  ``x`` is bf16, fp16 or fp32; ``weight`` and ``bias`` have its dtype or fp32.  Sums and
statistics are fp32, results are rounded once.  Rows that are evenly spaced and contiguous are read as they are; others are copied first.
Rows of a whole number of 16-byte pieces on 16-byte boundaries take wide loads, others go element by element.  Errors are ValueError, as
in the reference's kernel library (python/avelang_kernels/amdgpu_gemm.py:463-486).  Rows that a bounded wait on the device has given up on are NaN in all their results, and so are
the columns of the gradients of weight and bias that miss elements of them; ``gdn.read_status()`` says so.
"""
from __future__ import annotations

import torch

from . import _lib, torch_ops  # noqa: F401  (torch_ops declares the operators the native functions call)

__all__ = ["layer_norm", "layer_norm_backward", "LayerNormFunction"]

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
