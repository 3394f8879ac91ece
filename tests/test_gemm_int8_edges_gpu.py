"""The product of 8-bit integers where its tiles end: every number of columns that a chunk of 128 bytes can be left with, in rows on 16 bytes, off them and at odd addresses."""
import pytest
import torch

from test_gemm_int8_gpu import DT, check, device_rows, make

pytestmark = pytest.mark.gpu


def places(n):
    """First column and row distance of a result: at even and odd addresses, the rows' parity the same throughout and alternating, and on 16 bytes."""
    return [(first, first + n + more) for first in (0, 1, 2, 3) for more in (0, 1)] + [(16, -(-n // 16) * 16 + 32)]


def whole(m, n, k, dt, bias, layouts):
    """One product into each of the layouts: every element of the result is its own, everything beside it stays as it was."""
    from avelang_b200 import gemm
    aq, a, bq, b, sa, sb, bb = make(m, n, k, m + 3 * n + k, dt, bias)
    args = device_rows(aq, k), device_rows(bq, k), sa.cuda(), sb.cuda(), None if bb is None else bb.cuda()
    plain = gemm.gemm_int8_transposed_b(*args, out_dtype=DT[dt])
    check(plain, a, b, sa, sb, bb)
    for first, width in layouts:
        wide = torch.full((m + 2, width), float("nan"), dtype=DT[dt], device="cuda")
        out = wide[1:m + 1, first:first + n]
        gemm.gemm_int8_transposed_b(*args, out=out)
        assert torch.equal(out, plain), (first, width)
        out.fill_(float("nan"))
        assert torch.isnan(wide).all(), (first, width)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n", [1, 2, 3, 30, 31, 32, 33, 34, 35, 62, 63, 64, 65, 66, 67, 97, 98, 126, 127, 128, 129, 130, 131, 191, 193, 194, 258, 2050])
def test_what_is_left_of_a_chunk(built_lib, n, dt):
    whole(300, n, 40, dt, "own", places(n))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("m", [1, 2, 4, 20, 64, 128, 129, 3000])
def test_two_columns_of_the_last_chunk(built_lib, m, dt):
    for n in (2, 66, 130, 2050):
        whole(m, n, 33, dt, None, places(n))
