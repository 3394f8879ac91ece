"""What the entry points of linear attention and layer norm refuse, and that each reaches its kernels through its operator (no GPU needed)."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from avelang_b200 import _lib
from test_dispatch import Recorder


def bf(*s):
    return torch.zeros(*s, dtype=torch.bfloat16, device="cuda:0")


def f32(*s):
    return torch.zeros(*s, device="cuda:0")


def i32(*s):
    return torch.zeros(*s, dtype=torch.int32, device="cuda:0")


CALLS = {
    "linear_prefill": lambda L, N: L.chunk_linear_attention(bf(1, 9, 2, 128), bf(1, 9, 2, 128), bf(1, 9, 4, 64), f32(4), output_final_state=True),
    "linear_decode": lambda L, N: L.fused_recurrent_linear_attention(bf(3, 1, 2, 64), bf(3, 1, 2, 64), bf(3, 1, 4, 128), f32(3, 1, 4), initial_state=f32(5, 4, 64, 128),
                                                                     state_indices=i32(3)),
    "linear_backward": lambda L, N: L.linear_attention_backward(bf(1, 9, 2, 128), bf(1, 9, 2, 128), bf(1, 9, 4, 64), f32(1, 9, 4), bf(1, 9, 4, 64)),
    "layer_norm": lambda L, N: N.layer_norm(bf(2, 3, 100), f32(100), f32(100), return_stats=True),
    "layer_norm_backward": lambda L, N: N.layer_norm_backward(bf(6, 100), bf(6, 100), f32(6), f32(6), bf(100)),
}


@pytest.mark.parametrize("name", list(CALLS))
def test_public_functions_call_their_operator(built_lib, name):
    from avelang_b200 import linear_attention, norm
    with FakeTensorMode(), Recorder(run=False) as mode:
        CALLS[name](linear_attention, norm)
    assert mode.seen == [name]


def test_namespace(built_lib):
    from avelang_kernels import linear_attention, norm
    import avelang_b200.linear_attention as a
    import avelang_b200.norm as b
    assert linear_attention is a and norm is b


@pytest.mark.parametrize("entry", ["chunk_linear_attention", "fused_recurrent_linear_attention"])
def test_linear_refusals(built_lib, entry):
    from avelang_b200 import linear_attention as L
    f = getattr(L, entry)
    q, v = lambda: bf(1, 9, 2, 128), lambda: bf(1, 9, 4, 128)
    with FakeTensorMode():
        for match, call in [
            ("q must have dtype torch.bfloat16", lambda: f(f32(1, 9, 2, 128), q(), v())),
            ("k must be a 4-D", lambda: f(q(), bf(9, 2, 128), v())),
            ("k must have shape", lambda: f(q(), bf(1, 8, 2, 128), v())),
            ("v must have leading shape", lambda: f(q(), q(), bf(1, 8, 4, 128))),
            ("multiple of key heads", lambda: f(q(), q(), bf(1, 9, 3, 128))),
            ("dk and dv must be 128 or 64", lambda: f(bf(1, 9, 2, 96), bf(1, 9, 2, 96), v())),
            ("dk and dv must be 128 or 64", lambda: f(q(), q(), bf(1, 9, 4, 256))),
            ("g must have dtype", lambda: f(q(), q(), v(), bf(1, 9, 4))),
            ("g must have shape", lambda: f(q(), q(), v(), f32(9, 4))),
            ("g must have shape", lambda: f(q(), q(), v(), f32(2))),
            ("contiguous in its last", lambda: f(q().transpose(2, 3).contiguous().transpose(2, 3), q(), v())),
            ("cu_seqlens requires B == 1", lambda: f(bf(2, 9, 2, 128), bf(2, 9, 2, 128), bf(2, 9, 4, 128), cu_seqlens=i32(3))),
            ("1-D int32", lambda: f(q(), q(), v(), cu_seqlens=torch.zeros(3, dtype=torch.int64, device="cuda:0"))),
            ("one state per sequence", lambda: f(q(), q(), v(), initial_state=f32(2, 4, 128, 128))),
            ("initial_state must have shape", lambda: f(q(), q(), v(), initial_state=f32(1, 4, 128, 64))),
            ("state_indices needs initial_state", lambda: f(q(), q(), v(), state_indices=i32(1))),
            ("state_indices must be int32", lambda: f(q(), q(), v(), initial_state=f32(5, 4, 128, 128), state_indices=i32(2))),
            ("out must have shape", lambda: f(q(), q(), v(), out=bf(1, 9, 4, 64))),
        ]:
            with pytest.raises(ValueError, match=match):
                call()
    with pytest.raises(ValueError, match="CUDA tensor"):
        z = torch.zeros(1, 9, 2, 128, dtype=torch.bfloat16)
        f(z, z, z)
    if entry == "chunk_linear_attention":
        with FakeTensorMode(), pytest.raises(ValueError, match="chunk_size must be 64"):
            f(q(), q(), v(), chunk_size=32)


def test_backward_refusals(built_lib):
    from avelang_b200 import linear_attention as L
    q, v = lambda: bf(1, 9, 2, 128), lambda: bf(1, 9, 4, 64)
    f = L.linear_attention_backward
    with FakeTensorMode():
        for match, call in [
            ("d_o must be a bf16", lambda: f(q(), q(), v(), None, f32(1, 9, 4, 64))),
            ("d_o must be a bf16", lambda: f(q(), q(), v(), None, bf(1, 9, 4, 128))),
            ("initial_state must be a contiguous", lambda: f(q(), q(), v(), None, v(), None, f32(1, 4, 64, 128))),
            ("d_final_state must be a contiguous", lambda: f(q(), q(), v(), None, v(), None, None, f32(2, 4, 128, 64))),
            ("g must have shape", lambda: f(q(), q(), v(), f32(3), v())),
            ("cu_seqlens requires B == 1", lambda: f(bf(2, 9, 2, 128), bf(2, 9, 2, 128), bf(2, 9, 4, 64), None, bf(2, 9, 4, 64), None, None, None, i32(2))),
        ]:
            with pytest.raises(ValueError, match=match):
                call()
    lib = _lib.load()
    a = _lib.LinearBwdArgs()
    assert lib.ave_linear_backward(None, None) == lib.ave_linear_backward(ctypes.byref(a), None) == _lib.INVALID_ARGUMENT
    a.struct_size = ctypes.sizeof(a)
    a.B, a.T, a.Hk, a.Hv, a.dk, a.dv, a.n_seqs = 1, 100, 2, 4, 128, 64, 1
    for n in ("q", "k", "v", "d_o", "d_q", "d_k", "d_v", "g", "d_g"):
        setattr(a, n, 0x1000)
    a.initial_state = 0x1000
    assert lib.ave_linear_backward(ctypes.byref(a), None) == _lib.INVALID_ARGUMENT  # its gradient has no place
    a.initial_state = None
    assert lib.ave_linear_backward(ctypes.byref(a), None) == _lib.INVALID_ARGUMENT  # no scratch
    a.workspace, a.workspace_bytes = 0x1000, 16
    assert lib.ave_linear_backward(ctypes.byref(a), None) == _lib.WORKSPACE_TOO_SMALL
    assert lib.ave_linear_backward_workspace_bytes(ctypes.byref(a)) > 0
    a.d_q = 0x1004
    assert lib.ave_linear_backward(ctypes.byref(a), None) == _lib.MISALIGNED


def test_norm_refusals(built_lib):
    from avelang_b200 import norm as N
    with FakeTensorMode():
        for match, call in [
            ("x must have dtype", lambda: N.layer_norm(torch.zeros(2, 4, dtype=torch.float64, device="cuda:0"))),
            ("must lie in", lambda: N.layer_norm(bf(2, 0))),
            ("must lie in", lambda: N.layer_norm(bf(2, 28673))),
            ("bias needs weight", lambda: N.layer_norm(bf(2, 8), None, f32(8))),
            ("weight must have shape", lambda: N.layer_norm(bf(2, 8), f32(7))),
            ("weight must have the dtype of x", lambda: N.layer_norm(bf(2, 8), torch.zeros(8, dtype=torch.float16, device="cuda:0"))),
            ("share a dtype", lambda: N.layer_norm(bf(2, 8), f32(8), bf(8))),
            ("out must be a", lambda: N.layer_norm(bf(2, 8), out=f32(2, 8))),
            ("out must be viewable", lambda: N.layer_norm(bf(2, 8), out=bf(8, 2).t())),
            ("d_y must be a", lambda: N.layer_norm_backward(f32(2, 8), bf(2, 8), f32(2), f32(2))),
            ("mean must be a contiguous fp32", lambda: N.layer_norm_backward(bf(2, 8), bf(2, 8), f32(3), f32(2))),
            ("rstd must be a contiguous fp32", lambda: N.layer_norm_backward(bf(2, 8), bf(2, 8), f32(2), bf(2))),
        ]:
            with pytest.raises(ValueError, match=match):
                call()
    with pytest.raises(ValueError, match="CUDA tensor"):
        N.layer_norm(torch.zeros(2, 8))


def test_c_abi_refusals(built_lib):
    lib = _lib.load()
    a = _lib.LinearArgs()
    assert lib.ave_linear_decode_step(None, None) == lib.ave_linear_decode_step(ctypes.byref(a), None) == _lib.INVALID_ARGUMENT
    a.struct_size = ctypes.sizeof(a)
    a.B, a.T, a.Hk, a.Hv, a.dk, a.dv, a.n_seqs = 1, 8, 2, 4, 128, 64, 1
    for f in (lib.ave_linear_decode_step, lib.ave_linear_chunk_prefill):
        assert f(ctypes.byref(a), None) == _lib.INVALID_ARGUMENT  # null tensors
        a.dv = 96
        assert f(ctypes.byref(a), None) == _lib.UNSUPPORTED
        a.dv = 64
    for n in ("q", "k", "v", "o"):
        setattr(a, n, 0x1000)
        for s in ("b", "t", "h"):
            setattr(a, f"{n}_stride_{s}", 512)
    a.v_stride_t = 516
    for f in (lib.ave_linear_decode_step, lib.ave_linear_chunk_prefill):
        assert f(ctypes.byref(a), None) == _lib.MISALIGNED
    a.T = 0
    for f in (lib.ave_linear_decode_step, lib.ave_linear_chunk_prefill):
        assert f(ctypes.byref(a), None) == _lib.OK
    n = _lib.LayerNormArgs()
    n.struct_size = ctypes.sizeof(n)
    n.rows, n.n, n.x_dtype, n.w_dtype = 2, 8, 0, 1
    assert lib.ave_layer_norm(ctypes.byref(n), None) == _lib.INVALID_ARGUMENT  # fp16 weights beside bf16 rows
    n.w_dtype, n.n = 2, 40000
    assert lib.ave_layer_norm(ctypes.byref(n), None) == _lib.UNSUPPORTED
    b = _lib.LayerNormBwdArgs()
    b.struct_size = ctypes.sizeof(b)
    b.rows, b.n, b.x_dtype, b.w_dtype = 2, 8, 0, 2
    for f in ("d_y", "x", "mean", "rstd", "d_x", "d_weight"):
        setattr(b, f, 0x1000)
    assert lib.ave_layer_norm_backward(ctypes.byref(b), None) == _lib.INVALID_ARGUMENT  # no scratch
    b.workspace, b.workspace_bytes = 0x1000, 16
    assert lib.ave_layer_norm_backward(ctypes.byref(b), None) == _lib.WORKSPACE_TOO_SMALL
    assert lib.ave_layer_norm_backward_workspace_bytes(ctypes.byref(b)) > 0


def test_struct_mirrors(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = [("AveLinearArgs", _lib.LinearArgs, "scale"), ("AveLinearBwdArgs", _lib.LinearBwdArgs, "scale"), ("AveLayerNormArgs", _lib.LayerNormArgs, "eps"), ("AveLayerNormBwdArgs", _lib.LayerNormBwdArgs, "w_dtype")]
    src = tmp_path / "sz.c"
    src.write_text('#include "ave_gdn.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){' + "".join(
        f'printf("%zu %zu\\n", sizeof({c}), offsetof({c}, {f}));' for c, _, f in names) + "return 0;}\n")
    exe = tmp_path / "sz"
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [x for _, m, f in names for x in (ctypes.sizeof(m), getattr(m, f).offset)]


def test_norm_refuses_results_that_overlap_their_input(built_lib):
    from avelang_b200 import norm as N
    with FakeTensorMode():
        buf = bf(9, 64)
        for x, out in ((buf[:8], buf[1:]), (buf[1:], buf[:8]), (buf[:, :40], buf[:, 20:60]), (buf.view(-1)[:512].view(8, 64), buf.view(-1)[32:544].view(8, 64)),
                       (buf[:8, :32], buf.view(-1)[:256].view(8, 32)), (buf[:1].expand(8, 64), buf[:8])):
            with pytest.raises(ValueError, match="itself or share no element"):
                N.layer_norm(x, out=out)
        with pytest.raises(ValueError, match="rows of out must not overlap"):
            N.layer_norm(bf(8, 64), out=buf[:1].expand(8, 64))
    with FakeTensorMode(), Recorder(run=False) as mode:
        buf = bf(9, 64)
        for x, out in ((buf, buf), (buf[:, :32], buf[:, 32:]), (buf[:, 40:], buf[:, :24]), (buf[:4], buf[4:8]), (buf[5:], buf[:4]), (buf[::2], buf[::2]), (buf[0], buf[0])):
            N.layer_norm(x, out=out)
    assert mode.seen == ["layer_norm"] * 7
