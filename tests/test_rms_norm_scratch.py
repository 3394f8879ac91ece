"""The scratch of the RMS norm's gradients: a row of sums for each CTA that leaves some, and no CTA without a row."""
import ctypes

import pytest
import torch

from avelang_b200 import _lib


def arguments(rows, n, **more):
    a = _lib.RmsNormBwdArgs()
    a.struct_size, a.rows, a.n, a.d_weight = ctypes.sizeof(a), rows, n, 0x1000
    for k, v in more.items():
        setattr(a, k, v)
    return a


def test_follows_the_rows(built_lib):
    size = lambda rows, n: _lib.load().ave_rms_norm_backward_workspace_bytes(ctypes.byref(arguments(rows, n)))
    assert size(1, 28672) == 4 * 28672 and size(1, 1) == 4 and size(100, 2048) == 4 * 100 * 2048
    assert size(1 << 20, 2048) == size(2000, 2048) >= size(400, 2048)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,n", [(1, 28672), (2, 28671), (1, 8), (3, 64), (9, 63), (7, 1409), (30, 2048), (300, 8192), (299, 16384), (500, 28671), (600, 64), (700, 7)])
def test_nothing_behind_it(built_lib, rows, n, dtype):
    """With scratch of just that size, and a mark behind it, the gradients are those of the public call."""
    from avelang_b200 import norm
    gen = torch.Generator(device="cuda").manual_seed(rows + n)
    x, d_y = (torch.randn(rows, n, generator=gen, device="cuda").to(dtype) for _ in range(2))
    w, rstd = torch.rand(n, generator=gen, device="cuda") + 0.5, torch.rand(rows, generator=gen, device="cuda") + 0.5
    want = norm.rms_norm_backward(d_y, x, rstd, w, d_sum=x)
    dx, dw = torch.empty_like(x), torch.empty_like(w)
    a = arguments(rows, n, d_y=d_y.data_ptr(), x=x.data_ptr(), rstd=rstd.data_ptr(), weight=w.data_ptr(), d_sum=x.data_ptr(), d_x=dx.data_ptr(), d_weight=dw.data_ptr(),
                  dy_stride=n, x_stride=n, ds_stride=n, dx_stride=n, x_dtype=0 if dtype == torch.bfloat16 else 2, w_dtype=2)
    lib = _lib.load()
    a.workspace_bytes = lib.ave_rms_norm_backward_workspace_bytes(ctypes.byref(a))
    scratch = torch.full((a.workspace_bytes // 4 + 4096,), 7.0, device="cuda")
    a.workspace = scratch.data_ptr()
    assert lib.ave_rms_norm_backward(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == _lib.OK
    assert torch.equal(dx, want[0]) and torch.equal(dw, want[1])
    assert (scratch[a.workspace_bytes // 4:] == 7.0).all()
