"""What the whole numbers of 8-bit rows are, to the bit: each value times 127 / (the row's largest), that factor rounded to fp32, to nearest, ties to even."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def whole(f):
    """f: fp32 rows.  Products of two fp32 numbers are exact in 64 bits, and so is what they are rounded to."""
    factor = torch.full_like(f[:, 0], 127.0) / f.abs().amax(1)
    return torch.round(f.double() * factor.double()[:, None]).to(torch.int8)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,n", [(50, 64), (7, 100), (300, 2048), (40, 4097), (600, 4096), (3, 28672)])
def test_rows(built_lib, rows, n, dt):
    """Among the values are halves of the row's largest, 63.5 steps, and their neighbours."""
    from avelang_b200 import gemm
    gen = torch.Generator().manual_seed(rows + n)
    x = (torch.randn(rows, n, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen))).to(DT[dt])
    top = x.abs().amax(1)
    x[:, 1], x[:, 2], x[:, 3], x[:, 4] = top / 2, -top / 2, top / 4, (top.float() * (33.5 / 127)).to(DT[dt])
    x[:, 0] = top
    q, scale = gemm.quantize_rows_int8(x.cuda())
    assert torch.equal(q.cpu(), whole(x.float()))
    assert ((scale.cpu().double() * 127 / top.double() - 1).abs() <= 2 * 2.0 ** -24 * 1.01).all()  # (1 / 127 and the product rounded)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,n", [(1, 2048), (301, 2048), (60, 1409), (40, 8192)])
def test_norm(built_lib, rows, n, dt):
    from avelang_b200 import norm
    gen = torch.Generator().manual_seed(rows * n)
    x, res = (torch.randn(rows, n, generator=gen).to(DT[dt]) for _ in range(2))
    w = torch.randn(n, generator=gen) * 0.2
    for centered in (False, True):
        q, _, h = norm.rms_norm_int8(x.cuda(), w.cuda(), residual=res.cuda(), zero_centered=centered)
        assert torch.equal(q.cpu(), whole(h.cpu().float() * (w + 1.0 if centered else w)))
