"""What the entry points of the RMS norm, of 8-bit rows and of their product refuse, and that each reaches its kernels through its operator (no GPU needed)."""
import ctypes
import os
import subprocess

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from avelang_b200 import _lib
from test_dispatch import Recorder


def bf(*s):
    return torch.zeros(*s, dtype=torch.bfloat16, device="cuda:0")


def f32(*s):
    return torch.zeros(*s, device="cuda:0")


def i8(*s):
    return torch.zeros(*s, dtype=torch.int8, device="cuda:0")


CALLS = {
    "rms_norm": [lambda G, N: N.rms_norm(bf(2, 3, 100), f32(100), residual=bf(2, 3, 100), return_stats=True),
                 lambda G, N: N.rms_norm_int8(bf(2, 3, 100), bf(100), residual=bf(2, 3, 100), zero_centered=True)],
    "rms_norm_backward": [lambda G, N: N.rms_norm_backward(bf(6, 100), bf(6, 100), f32(6), bf(100), d_sum=bf(6, 100))],
    "quantize_rows_int8": [lambda G, N: G.quantize_rows_int8(f32(3, 100))],
    "dequantize_rows_int8": [lambda G, N: G.dequantize_rows_int8(i8(3, 112)[:, :100], f32(3), torch.float16)],
    "gemm_int8_nt": [lambda G, N: G.gemm_int8_transposed_b(i8(3, 48)[:, :33], i8(5, 48)[:, :33], f32(3), f32(5), f32(5), out_dtype=torch.float16)],
}


@pytest.mark.parametrize("name", list(CALLS))
def test_public_functions_call_their_operator(built_lib, name):
    from avelang_b200 import gemm, norm
    for call in CALLS[name]:
        with FakeTensorMode(), Recorder(run=False) as mode:
            call(gemm, norm)
        assert mode.seen == [name]


def test_shapes_of_results(built_lib):
    from avelang_b200 import gemm, norm
    with FakeTensorMode(), Recorder(run=False):
        x, w = bf(2, 3, 100), f32(100)
        assert norm.rms_norm(x, w).shape == x.shape
        y, h = norm.rms_norm(x, w, residual=x)
        assert y.shape == h.shape == x.shape and h.dtype == torch.bfloat16
        y, rstd = norm.rms_norm(x, w, return_stats=True)
        assert rstd.shape == (2, 3) and rstd.dtype == torch.float32
        assert len(norm.rms_norm(x, residual=x, return_stats=True)) == 3
        q, scale = norm.rms_norm_int8(x)
        assert q.shape == x.shape and q.dtype == torch.int8 and q.stride() == (336, 112, 1) and scale.shape == (2, 3)
        q, scale, h = norm.rms_norm_int8(x, residual=x, sum_out=x)
        assert h is x
        q, scale = gemm.quantize_rows_int8(bf(100))
        assert q.shape == (100,) and scale.shape == ()
        assert gemm.dequantize_rows_int8(q, scale).dtype == torch.bfloat16
        assert gemm.gemm_int8_transposed_b(i8(3, 32), i8(5, 32), f32(3), f32(5)).dtype == torch.bfloat16
        out = torch.zeros(3, 5, dtype=torch.float16, device="cuda:0")
        assert gemm.gemm_int8_transposed_b(i8(3, 32), i8(5, 32), f32(3, 1), f32(5), out=out) is out


def test_norm_refusals(built_lib):
    from avelang_b200 import norm as N
    with FakeTensorMode(), Recorder(run=False):
        x, w = bf(4, 64), bf(64)
        wide = bf(8, 64)
        for match, call in [
            ("x must have dtype", lambda f: f(i8(4, 64))),
            ("x must have dtype", lambda f: f(x.double())),
            ("CUDA tensor", lambda f: f(torch.zeros(4, 64))),
            ("last dimension of x must lie in", lambda f: f(bf(4, 28673))),
            ("last dimension of x must lie in", lambda f: f(bf(4, 0))),
            ("weight must have shape", lambda f: f(x, bf(63))),
            ("weight must have the dtype of x", lambda f: f(x, w.half())),
            ("residual must be a torch.bfloat16 tensor of shape", lambda f: f(x, w, residual=bf(64))),
            ("residual must be a torch.bfloat16 tensor of shape", lambda f: f(x, w, residual=f32(4, 64))),
            ("sum_out needs residual", lambda f: f(x, w, sum_out=bf(4, 64))),
            ("sum_out must be a torch.bfloat16 tensor", lambda f: f(x, w, residual=x, sum_out=f32(4, 64))),
            ("sum_out must be viewable", lambda f: f(x, w, residual=x, sum_out=bf(64, 4).t())),
            ("the rows of sum_out must not overlap", lambda f: f(x, w, residual=x, sum_out=bf(64).expand(4, 64))),
            ("sum_out must be x or residual themselves", lambda f: f(wide[:4], w, residual=bf(4, 64), sum_out=wide[2:6])),
            ("sum_out must be x or residual themselves", lambda f: f(bf(4, 64), w, residual=wide[:4], sum_out=wide[2:6])),
            ("weight must be a tensor", lambda f: f(x, 1.0)),
        ]:
            for f in (N.rms_norm, N.rms_norm_int8):
                with pytest.raises(ValueError, match=match):
                    call(f)
        for match, call in [
            ("out must be a torch.bfloat16 tensor of shape", lambda: N.rms_norm(x, w, out=f32(4, 64))),
            ("out must be viewable", lambda: N.rms_norm(x, w, out=bf(64, 4).t())),
            ("the rows of out must not overlap", lambda: N.rms_norm(x, w, out=bf(64).expand(4, 64))),
            ("out must be x or residual themselves", lambda: N.rms_norm(wide[:4], w, out=wide[1:5])),
            ("out must be x or residual themselves", lambda: N.rms_norm(bf(4, 64), w, residual=wide[:4], out=wide[1:5])),
            ("out and sum_out must share no element", lambda: N.rms_norm(x, w, residual=bf(4, 64), out=x, sum_out=x)),
            ("out and sum_out must share no element", lambda: N.rms_norm(x, w, residual=x, out=wide[:4], sum_out=wide[3:7])),
            ("must share no memory with weight", lambda: N.rms_norm(x, wide[3], out=wide[:4])),
            ("must share no memory with weight", lambda: N.rms_norm(x, wide[3], residual=bf(4, 64), sum_out=wide[:4])),
            ("d_y must be a torch.bfloat16 tensor", lambda: N.rms_norm_backward(f32(4, 64), x, f32(4), w)),
            ("d_sum must be a torch.bfloat16 tensor", lambda: N.rms_norm_backward(x, x, f32(4), w, d_sum=bf(64))),
            ("rstd must be a contiguous fp32 tensor of 4", lambda: N.rms_norm_backward(x, x, f32(5), w)),
            ("rstd must be a contiguous fp32 tensor of 4", lambda: N.rms_norm_backward(x, x, bf(4), w)),
        ]:
            with pytest.raises(ValueError, match=match):
                call()
        N.rms_norm(x, w, residual=wide[:4], out=x, sum_out=wide[:4])       # each in the place of an input
        N.rms_norm(wide[:, :32], residual=bf(8, 32), out=wide[:, 32:])     # columns beside one another share nothing


def test_int8_refusals(built_lib):
    from avelang_b200 import gemm as G
    g = lambda a=None, b=None, sa=None, sb=None, *more, **kw: G.gemm_int8_transposed_b(i8(4, 64) if a is None else a, i8(6, 64) if b is None else b,
                                                                                      f32(4) if sa is None else sa, f32(6) if sb is None else sb, *more, **kw)
    with FakeTensorMode(), Recorder(run=False):
        pool = i8(4096)
        for match, call in [
            ("A must have dtype torch.int8", lambda: g(bf(4, 64))),
            ("B must have dtype torch.int8", lambda: g(None, i8(6, 64).to(torch.uint8))),
            ("must share K", lambda: g(i8(4, 32))),
            ("must share K", lambda: g(i8(1, 4, 64))),
            ("CUDA tensors on one device", lambda: g(torch.zeros(4, 64, dtype=torch.int8))),
            ("K must lie in", lambda: g(i8(4, 131072), i8(6, 131072))),
            ("K must lie in", lambda: g(i8(4, 0), i8(6, 0))),
            ("A must be contiguous in its last dimension, with rows a multiple of 16", lambda: g(i8(4, 72)[:, :64])),
            ("B must be contiguous in its last dimension, with rows a multiple of 16", lambda: g(None, i8(64, 6).t())),
            ("A must be contiguous in its last dimension, with rows a multiple of 16", lambda: g(i8(64).expand(4, 64))),
            ("a_scale must be a contiguous fp32 tensor of 4", lambda: g(None, None, f32(6))),
            ("b_scale must be a contiguous fp32 tensor of 6", lambda: g(None, None, None, bf(6))),
            ("b_scale must be a contiguous fp32 tensor of 6", lambda: g(None, None, None, f32(12)[::2])),
            ("bias must have shape", lambda: g(None, None, None, None, f32(4))),
            ("bias must have the dtype of the result", lambda: g(None, None, None, None, bf(6), out_dtype=torch.float16)),
            ("out_dtype must be a dtype", lambda: g(out_dtype="bf16")),
            ("out_dtype must be torch.bfloat16", lambda: g(out_dtype=torch.int8)),
            ("out must have shape", lambda: g(out=bf(6, 4))),
            ("out must have dtype", lambda: g(out=i8(4, 6))),
            ("out must have dtype out_dtype", lambda: g(out=bf(4, 6), out_dtype=torch.float32)),
            ("out must be contiguous", lambda: g(out=bf(6, 4).t())),
            ("out must be contiguous", lambda: g(out=bf(6).expand(4, 6))),
            ("out must not share memory with A", lambda: g(pool[:256].view(4, 64), out=pool[200:248].view(torch.bfloat16).view(4, 6))),
            ("out must not share memory with B", lambda: g(None, pool[:384].view(6, 64), out=pool[336:384].view(torch.bfloat16).view(4, 6))),
            ("x must have dtype", lambda: G.quantize_rows_int8(i8(4, 64))),
            ("last dimension of x must lie in", lambda: G.quantize_rows_int8(bf(1, 28673))),
            ("q must have dtype torch.int8", lambda: G.dequantize_rows_int8(bf(4, 64), f32(4))),
            ("scale must be a fp32 tensor of shape", lambda: G.dequantize_rows_int8(i8(4, 64), f32(5))),
            ("dtype must be torch.bfloat16", lambda: G.dequantize_rows_int8(i8(4, 64), f32(4), torch.int8)),
        ]:
            with pytest.raises(ValueError, match=match):
                call()
        g(pool[:256].view(4, 64), out=pool[256:304].view(torch.bfloat16).view(4, 6))  # behind it


def test_struct_mirrors_match_header(tmp_path):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pairs = {"AveRmsNormArgs": (_lib.RmsNormArgs, "eps"), "AveRmsNormBwdArgs": (_lib.RmsNormBwdArgs, "w_dtype"), "AveQuantRowsArgs": (_lib.QuantRowsArgs, "x_dtype"),
             "AveGemmInt8Args": (_lib.GemmInt8Args, "status")}
    src = tmp_path / "sz.c"
    src.write_text('#include "ave_gdn.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){' +
                   "".join(f'printf("%zu %zu ",sizeof({c}),offsetof({c},{last}));' for c, (_, last) in pairs.items()) + "return 0;}\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(tmp_path / "sz")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "sz")], check=True, capture_output=True, text=True).stdout.split()]
    assert got == [v for py, last in pairs.values() for v in (ctypes.sizeof(py), getattr(py, last).offset)]


def test_status_codes_without_a_device(built_lib):
    lib = _lib.load()

    def filled(cls, **kw):
        a = cls()
        a.struct_size = ctypes.sizeof(cls)
        for k, v in kw.items():
            setattr(a, k, v)
        return a

    norm = dict(x=0x1000, y=0x2000, rows=4, n=64, x_stride=64, y_stride=64, w_dtype=0)
    for want, change in [(_lib.INVALID_ARGUMENT, dict(struct_size=8)), (_lib.INVALID_ARGUMENT, dict(n=0)), (_lib.INVALID_ARGUMENT, dict(rows=-1)),
                         (_lib.UNSUPPORTED, dict(n=28673)), (_lib.INVALID_ARGUMENT, dict(w_dtype=1)), (_lib.INVALID_ARGUMENT, dict(x=None)),
                         (_lib.INVALID_ARGUMENT, dict(residual=0x3000)), (_lib.INVALID_ARGUMENT, dict(sum=0x3000)), (_lib.MISALIGNED, dict(x=0x1001)),
                         (_lib.INVALID_ARGUMENT, dict(flags=2)), (_lib.MISALIGNED, dict(flags=2, scale=0x4000, y=0x2008)),
                         (_lib.MISALIGNED, dict(flags=2, scale=0x4000, y_stride=72)), (_lib.MISALIGNED, dict(flags=2, scale=0x4002)), (_lib.OK, dict(rows=0, x=None))]:
        assert lib.ave_rms_norm(ctypes.byref(filled(_lib.RmsNormArgs, **{**norm, **change})), None) == want, change
    back = dict(d_y=0x1000, x=0x2000, rstd=0x3000, d_x=0x4000, rows=4, n=64)
    for want, change in [(_lib.INVALID_ARGUMENT, dict(rstd=None)), (_lib.INVALID_ARGUMENT, dict(d_weight=0x5000)),
                         (_lib.WORKSPACE_TOO_SMALL, dict(d_weight=0x5000, workspace=0x6000, workspace_bytes=64)), (_lib.MISALIGNED, dict(d_sum=0x7001)),
                         (_lib.OK, dict(rows=0))]:
        assert lib.ave_rms_norm_backward(ctypes.byref(filled(_lib.RmsNormBwdArgs, **{**back, **change})), None) == want, change
    assert lib.ave_rms_norm_backward_workspace_bytes(ctypes.byref(filled(_lib.RmsNormBwdArgs, **back))) == 0
    assert lib.ave_rms_norm_backward_workspace_bytes(ctypes.byref(filled(_lib.RmsNormBwdArgs, d_weight=0x5000, **back))) > 0
    quant = dict(x=0x1000, q=0x2000, scale=0x3000, rows=4, n=60, x_stride=60, q_stride=64)
    for call in (lib.ave_quantize_rows_int8, lib.ave_dequantize_rows_int8):
        for want, change in [(_lib.INVALID_ARGUMENT, dict(q=None)), (_lib.INVALID_ARGUMENT, dict(x_dtype=3)), (_lib.MISALIGNED, dict(q_stride=60)),
                             (_lib.MISALIGNED, dict(q_stride=48)), (_lib.MISALIGNED, dict(q=0x2004)), (_lib.UNSUPPORTED, dict(n=28673)), (_lib.OK, dict(rows=0))]:
            assert call(ctypes.byref(filled(_lib.QuantRowsArgs, **{**quant, **change})), None) == want, change
    prod = dict(a=0x1000, b=0x2000, c=0x3000, a_scale=0x4000, b_scale=0x5000, M=4, N=6, K=60, lda=64, ldb=64, ldc=6)
    for want, change in [(_lib.INVALID_ARGUMENT, dict(K=0)), (_lib.UNSUPPORTED, dict(K=131072)), (_lib.INVALID_ARGUMENT, dict(b_scale=None)),
                         (_lib.MISALIGNED, dict(lda=60)), (_lib.MISALIGNED, dict(ldb=48)), (_lib.MISALIGNED, dict(b=0x2008)), (_lib.MISALIGNED, dict(c=0x3001)),
                         (_lib.INVALID_ARGUMENT, dict(ldc=5)), (_lib.INVALID_ARGUMENT, dict(bias_dtype=1)), (_lib.OK, dict(M=0)), (_lib.OK, dict(N=0, b=None))]:
        assert lib.ave_gemm_int8_nt(ctypes.byref(filled(_lib.GemmInt8Args, **{**prod, **change})), None) == want, change
