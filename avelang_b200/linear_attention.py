"""Linear attention with a decay for each head for B200: chunked form for whole sequences, recurrent form for single tokens.

The state of one (sequence, value head) is an fp32 matrix M [dk, dv]:

    M <- exp(g_t) M + k_t v_t^T;  o_t = scale M^T q_t

the gated delta rule of ``gdn`` without its correction.  Entry points, layouts and errors are those of ``gdn`` (calling
convention of the reference's kernel library, python/avelang_kernels/amdgpu_gemm.py:458-494): q, k ``[B, T, Hk, dk]``; v, o
``[B, T, Hv, dv]``, bf16; value head h reads key head ``h // (Hv // Hk)``; dk and dv are 64 or 128 each; packed batches are
``B == 1`` with int32 ``cu_seqlens [N+1]`` on the device; states are fp32 ``[N or num_slots, Hv, dk, dv]``.

``g``, the logarithm of the decay, is fp32: ``[B, T, Hv]`` (one for every token and head), ``[Hv]`` (one a head) or None (no
decay).  It is meant to be <= 0; minus infinity empties the state.
"""
from __future__ import annotations

from . import _lib, torch_ops  # noqa: F401  (torch_ops declares the operators the native functions call)

__all__ = ["chunk_linear_attention", "fused_recurrent_linear_attention"]

_native = _lib.host
_lib.register_operators()


def chunk_linear_attention(q, k, v, g=None, scale=None, initial_state=None, output_final_state=False, cu_seqlens=None, *,
                           state_indices=None, inplace_state=True, chunk_size=64, out=None):
    """Whole sequences, 64 tokens at a time.  Returns ``(o, final_state or None)``; ``scale`` is ``dk ** -0.5`` unless given.

    With ``state_indices`` (int32 ``[N]``) the initial states are read from, and the final states written to, slots of the
    ``initial_state`` pool (in place unless ``inplace_state=False``); a negative slot skips the sequence (zero output, no state
    access).  Sequences that share a slot race for it.  A sequence of no tokens hands its initial state on.  Rows behind the last
    offset of a packed batch are left as they were."""
    return _native.linear_prefill(q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, state_indices, inplace_state, out,
                                  chunk_size)


def fused_recurrent_linear_attention(q, k, v, g=None, scale=None, initial_state=None, output_final_state=True, cu_seqlens=None, *,
                                     state_indices=None, inplace_state=True, out=None):
    """Token by token with the state on chip; ``T == 1`` with ``state_indices`` is the continuous-batching decode step: each state is
    read once from its slot of the ``initial_state`` pool and written once, in place unless ``inplace_state=False``.  A negative
    slot skips the sequence.  Returns ``(o, state)``."""
    return _native.linear_decode(q, k, v, g, scale, initial_state, output_final_state, cu_seqlens, state_indices, inplace_state, out, 64)
