"""Linear attention with a decay for each head for B200: chunked form for whole sequences, recurrent form for single tokens.

The state of one (sequence, value head) is an fp32 matrix M [dk, dv]:

    M <- exp(g_t) M + k_t v_t^T;  o_t = scale M^T q_t

the gated delta rule of ``gdn`` without its correction.  Entry points, layouts and errors are those of ``gdn`` (calling
convention of the reference's kernel library, python/avelang_kernels/amdgpu_gemm.py:458-494): q, k ``[B, T, Hk, dk]``; v, o
``[B, T, Hv, dv]``, bf16; value head h reads key head ``h // (Hv // Hk)``; dk and dv are 64 or 128 each; packed batches are
``B == 1`` with int32 ``cu_seqlens [N+1]`` on the device; states are fp32 ``[N or num_slots, Hv, dk, dv]``.

``g``, the logarithm of the decay, is fp32: ``[B, T, Hv]`` (one for every token and head), ``[Hv]`` (one a head) or None (no
decay).  It is meant to be <= 0; minus infinity empties the state.

A NaN or an infinity in a token of v reaches the outputs from that token on, and in the whole-sequence form also those of the tokens in front of it among its sixteen (counted from
the sequence's first): a masked score is an exact zero, but zero times a NaN is none.  In the gradients the same holds for k, q and d_o, on either side.  Other sequences are never reached.
"""
from __future__ import annotations

import torch

from . import _lib, torch_ops  # noqa: F401  (torch_ops declares the operators the native functions call)

__all__ = ["chunk_linear_attention", "fused_recurrent_linear_attention", "linear_attention_backward", "LinearAttentionFunction"]

_native = _lib.host
_lib.register_operators()


def chunk_linear_attention(q, k, v, g=None, scale=None, initial_state=None, output_final_state=False, cu_seqlens=None, *,
                           state_indices=None, inplace_state=True, chunk_size=64, out=None):
    """Whole sequences, 64 tokens at a time.  Returns ``(o, final_state or None)``; ``scale`` is ``dk ** -0.5`` unless given.

    With ``state_indices`` (int32 ``[N]``) the initial states are read from, and the final states written to, slots of the
    ``initial_state`` pool (in place unless ``inplace_state=False``); a negative slot skips the sequence (zero output, no state
    access).  Sequences that share a slot race for it.  A sequence of no tokens hands its initial state on.  Rows in front of
    the first offset of a packed batch and behind its last are left as they were.  ``out`` may be q, k or v."""
    return _native.linear_prefill(q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, state_indices, inplace_state, out,
                                  chunk_size, False)


def fused_recurrent_linear_attention(q, k, v, g=None, scale=None, initial_state=None, output_final_state=True, cu_seqlens=None, *,
                                     state_indices=None, inplace_state=True, out=None):
    """Token by token with the state on chip; ``T == 1`` with ``state_indices`` is the continuous-batching decode step: each state is
    read once from its slot of the ``initial_state`` pool and written once, in place unless ``inplace_state=False``.  A negative
    slot skips the sequence.  ``out`` may be q, k or v.  Returns ``(o, state)``."""
    return _native.linear_decode(q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, state_indices, inplace_state, out, 64)


def linear_attention_backward(q, k, v, g, d_o, scale=None, initial_state=None, d_final_state=None, cu_seqlens=None):
    """Gradients of ``chunk_linear_attention`` / ``fused_recurrent_linear_attention``.  ``d_o``: bf16, shaped like ``v``; ``d_final_state``:
    optional fp32 gradient of the final states; neither needs to lie on 16-byte boundaries.  Returns ``(dq, dk, dv, dg, d_initial_state)``: dq, dk bf16 in the shape of q, k (the
    value heads sharing a key head are summed in fp32), dv bf16, dg fp32 in the shape of g (None without one), ``d_initial_state``
    fp32 (None when no initial state was given).  Rows of a packed batch that belong to no sequence get zeros."""
    return _native.linear_backward(q, k, v, g, d_o, scale, initial_state, d_final_state, cu_seqlens)


class LinearAttentionFunction(torch.autograd.Function):
    """``o, final_state = LinearAttentionFunction.apply(q, k, v, g, scale, initial_state, cu_seqlens)``: the chunked forward pass with
    the chunked backward pass attached (g, scale, initial_state and cu_seqlens may be None).  Rows of a packed batch that belong to no sequence are zero, in the result and in the gradients.  It can be differentiated once.  A step with
    its backward pass can be captured into a CUDA graph once the results of eager steps on the same leaves are gone."""

    @staticmethod
    def forward(ctx, q, k, v, g, scale, initial_state, cu_seqlens):
        o, final = _native.linear_prefill(q, k, v, g, scale, initial_state, True, cu_seqlens, None, True, None, 64, True)
        ctx.save_for_backward(q, k, v, g, initial_state, cu_seqlens)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return o, final

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_final):
        q, k, v, g, s0, cu = ctx.saved_tensors
        d_o = torch.zeros_like(v) if d_o is None else d_o.to(torch.bfloat16).contiguous()
        d_final = None if d_final is None else d_final.float().contiguous()
        dq, dk, dv, dg, ds0 = linear_attention_backward(q, k, v, g, d_o, ctx.scale, s0, d_final, cu)
        return dq, dk, dv, dg, None, ds0, None
