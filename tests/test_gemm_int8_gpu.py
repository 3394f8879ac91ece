"""The product of 8-bit integers against exact sums, rows in 8 bits and back, and a layer's step through norm, product and sum."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def rows8(gen, rows, n):
    q = torch.randint(-128, 128, (rows, -(-n // 16) * 16), generator=gen, dtype=torch.int8)
    return q, q[:, :n]


def device_rows(q, n):
    return q.cuda()[:, :n]


def exact(a, b, sa, sb, bias):
    """(value, |value without the bias|) in 64 bits; sums of whole numbers below 2^53 are exact."""
    c = (a.double() @ b.double().t()) * sa.double()[:, None] * sb.double()[None]
    return (c, c.abs()) if bias is None else (c + bias.double(), c.abs())


def check(got, a, b, sa, sb, bias):
    """The sum, its product with the first scale and the last step are rounded to fp32 each, the result once to its type."""
    want, size = exact(a, b, sa, sb, bias)
    e, t = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype)
    loss = 2.0 ** -24 * (2.01 * size + 1.01 * want.abs())
    lim = e * want.abs() + (1 + e) * loss + t.smallest_normal * t.eps
    assert ((got.cpu().double() - want).abs() <= lim).all()


def make(m, n, k, seed, dt, bias):
    gen = torch.Generator().manual_seed(seed)
    aq, a = rows8(gen, m, k)
    bq, b = rows8(gen, n, k)
    sa, sb = torch.rand(m, generator=gen) * 1e-3 + 1e-5, (torch.rand(n, generator=gen) - 0.3) * 1e-2
    bb = None if bias is None else torch.randn(n, generator=gen).to(torch.float32 if bias == "wide" else DT[dt])
    return aq, a, bq, b, sa, sb, bb


SIZES = [(1, 1, 1), (1, 16, 16), (1, 12352, 2048), (2, 130, 33), (3, 1544, 2048), (4, 100, 8192), (5, 7, 100), (8, 2048, 4096), (9, 257, 640), (16, 4096, 512), (17, 12352, 256), (33, 48, 1000),
         (64, 2048, 4096), (100, 1544, 127), (128, 256, 128), (129, 255, 129), (200, 12352, 384), (256, 512, 2048), (300, 1000, 1999), (1000, 1544, 200), (1003, 4104, 96), (2500, 300, 72), (4096, 2048, 256), (2900, 2571, 100),
         (5000, 1032, 513), (257, 20000, 64), (130, 19003, 1000), (10000, 1540, 33), (2, 40000, 64), (20, 40001, 80), (128, 38000, 48), (2560, 2304, 700), (2100, 2500, 130), (5120, 1050, 96), (4864, 1153, 40), (1300, 4100, 65)]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(built_lib, m, n, k):
    from avelang_b200 import gemm
    for i, (dt, bias) in enumerate((("bf16", None), ("fp16", "own"), ("fp32", "wide"), ("bf16", "wide"))):
        if i == 3 and m * n > 1 << 20:
            continue
        aq, a, bq, b, sa, sb, bb = make(m, n, k, m + n + k, dt, bias)
        call = lambda: gemm.gemm_int8_transposed_b(device_rows(aq, k), device_rows(bq, k), sa.cuda(), sb.cuda(), None if bb is None else bb.cuda(), out_dtype=DT[dt])
        got = call()
        assert got.shape == (m, n) and got.dtype == DT[dt]
        check(got, a, b, sa, sb, bb)
        assert torch.equal(got, call())
    from avelang_b200 import gdn
    assert gdn.read_status() == 0


def test_largest_sums(built_lib):
    """All operands at their lowest value, K at its limit: sums of 128 * 128 * 131071, just below 2^31."""
    from avelang_b200 import gemm
    for m, n, k in ((3, 20, 131071), (130, 40, 131071), (20, 600, 100003), (1030, 4000, 131071)):
        pitch = -(-k // 16) * 16
        aq, bq = torch.full((m, pitch), -128, dtype=torch.int8), torch.full((n, pitch), -128, dtype=torch.int8)
        bq[n // 2] = 127
        a, b = aq[:, :k], bq[:, :k]
        one = lambda c: torch.ones(c)
        got = gemm.gemm_int8_transposed_b(device_rows(aq, k), device_rows(bq, k), one(m).cuda(), one(n).cuda(), out_dtype=torch.float32)
        check(got, a, b, one(m), one(n), None)
        assert float(got[0, 0]) == float(torch.tensor(128.0 * 128 * k, dtype=torch.float64).float())


def test_rows_are_the_same_in_any_batch(built_lib):
    """A token's result does not depend on the batch that it is in."""
    from avelang_b200 import gemm
    aq, a, bq, b, sa, sb, bb = make(4000, 1544, 1000, 3, "bf16", "wide")
    A, B, sa, sb, bb = device_rows(aq, 1000), device_rows(bq, 1000), sa.cuda(), sb.cuda(), bb.cuda()
    whole = gemm.gemm_int8_transposed_b(A, B, sa, sb, bb)
    for lo, hi in ((0, 1), (5, 7), (100, 103), (300, 308), (17, 33), (1000, 1064), (700, 828), (60, 360), (1, 1100), (0, 3000)):
        assert torch.equal(gemm.gemm_int8_transposed_b(A[lo:hi], B, sa[lo:hi], sb, bb), whole[lo:hi])


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("m,n", [(1, 100), (5, 333), (70, 264), (300, 1000), (3000, 520), (9000, 600), (3000, 2001)])
def test_results_in_a_wider_tensor(built_lib, m, n, dt):
    """Results whose rows lie apart, on 16 bytes and off them; what lies beside them stays as it was."""
    from avelang_b200 import gemm
    aq, a, bq, b, sa, sb, _ = make(m, n, 96, m * n, dt, None)
    A, B, sc, sd = device_rows(aq, 96), device_rows(bq, 96), sa.cuda(), sb.cuda()
    want = gemm.gemm_int8_transposed_b(A, B, sc, sd, out_dtype=DT[dt])
    for first, width in ((16, -(-n // 16) * 16 + 32), (3, n + 7), (1, n + 1)):
        wide = torch.full((m + 2, width), 7.0, dtype=DT[dt], device="cuda")
        out = wide[1:m + 1, first:first + n]
        assert gemm.gemm_int8_transposed_b(A, B, sc, sd, out=out) is out
        assert torch.equal(out, want)
        assert (wide[0] == 7).all() and (wide[-1] == 7).all() and (wide[:, :first] == 7).all() and (wide[:, first + n:] == 7).all()


def test_what_lies_behind_a_row_is_not_read_into_it(built_lib):
    """Rows of 33 of 48 bytes: the 15 behind them hold something else, and so does what lies behind the last row of A and B."""
    from avelang_b200 import gemm
    for m, n, k in ((3, 50, 33), (40, 500, 33), (200, 3000, 250), (2600, 2050, 33)):
        aq, a, bq, b, sa, sb, _ = make(m, n, k, k, "fp32", None)
        outs = []
        for fill in (0, 77):
            pools = []
            for q, rows in ((aq, m), (bq, n)):
                pool = torch.full((rows + 130, q.shape[1]), fill, dtype=torch.int8)
                pool[:rows, :k] = q[:, :k]
                pools.append(pool.cuda()[:rows, :k])
            outs.append(gemm.gemm_int8_transposed_b(*pools, sa.cuda(), sb.cuda(), out_dtype=torch.float32))
        assert torch.equal(*outs)
        check(outs[0], a, b, sa, sb, None)


def test_scales(built_lib):
    """Scales of zero, NaN, infinity and of very different size; a NaN stays in its row or column."""
    from avelang_b200 import gemm
    for m in (4, 40, 400, 20000):
        aq, a, bq, b, sa, sb, _ = make(m, 300, 64, m, "fp32", None)
        plain = gemm.gemm_int8_transposed_b(device_rows(aq, 64), device_rows(bq, 64), sa.cuda(), sb.cuda(), out_dtype=torch.float32).cpu()
        sa[1], sa[2], sb[5], sb[7] = 0.0, float("nan"), float("nan"), 0.0
        sa[3], sb[9] = 1e30, 1e-30
        got = gemm.gemm_int8_transposed_b(device_rows(aq, 64), device_rows(bq, 64), sa.cuda(), sb.cuda(), out_dtype=torch.float32).cpu()
        assert torch.isnan(got[2]).all() and torch.isnan(got[:, 5]).all()
        cols = [c for c in range(300) if c not in (5, 7, 9)]
        assert (got[1, cols] == 0).all() and (got[[0, 1, 3], 7] == 0).all()
        assert torch.equal(got[0, cols], plain[0, cols])
        want = (a[3].double() @ b[9].double()) * float(sa[3]) * float(sb[9])
        assert abs(float(got[3, 9]) - float(want)) <= 4 * 2.0 ** -24 * abs(float(want))


@pytest.mark.parametrize("dt", list(DT))
def test_rows_and_back(built_lib, dt):
    from avelang_b200 import gemm
    gen = torch.Generator().manual_seed(8)
    for rows, n in ((1, 1), (3, 15), (700, 16), (9, 100), (40, 2048), (500, 4096), (4, 4100), (301, 1409), (2, 28672), (5, 28671), (0, 64)):
        x = (torch.randn(rows, n, generator=gen) * torch.exp(torch.randn(rows, 1, generator=gen))).to(DT[dt])
        q, scale = gemm.quantize_rows_int8(x.cuda())
        assert q.shape == (rows, n) and scale.shape == (rows,) and (rows <= 1 or q.stride(0) % 16 == 0)
        if rows:
            top = x.double().abs().amax(-1)
            s, d = scale.cpu().double(), q.cpu().double()
            assert ((s * 127 / top - 1).abs() <= 2.0 ** -22).all()
            assert ((d - x.double() * (127.0 / top)[:, None]).abs() <= 0.5 + 127 * 2.0 ** -22).all() and (d.abs().amax(-1) == 127).all()
        for to in DT.values():
            back = gemm.dequantize_rows_int8(q, scale, to)
            assert back.dtype == to and torch.equal(back, (q.float() * scale[:, None]).to(to))
        flat = q.contiguous()  # rows off 16 bytes
        assert torch.equal(gemm.dequantize_rows_int8(flat, scale), (q.float() * scale[:, None]).bfloat16())
    x = torch.randn(6, 200, generator=gen).to(DT[dt])
    x[0], x[2, 3], x[3, 199], x[4] = 0, float("inf"), float("nan"), torch.finfo(DT[dt]).smallest_normal
    for part in (x, x[:, :197]):
        q, scale = gemm.quantize_rows_int8(part.cuda())
        assert scale[0] == 0 and torch.isnan(scale[2]) and (q[[0, 2]] == 0).all()
        assert part is not x or (torch.isnan(scale[3]) and (q[3] == 0).all())
        assert (q[1].abs().max() == 127) and (dt == "fp16" or (scale[4] == 0 and (q[4] == 0).all()))
        back = gemm.dequantize_rows_int8(q, scale)
        assert torch.isnan(back[2]).all() and (back[0] == 0).all()
    stacked = torch.randn(2, 3, 70, generator=gen).to(DT[dt])
    q, scale = gemm.quantize_rows_int8(stacked.cuda())
    assert q.shape == (2, 3, 70) and scale.shape == (2, 3)
    assert torch.equal(gemm.dequantize_rows_int8(q, scale, torch.float32), q.float() * scale[..., None])
    q, scale = gemm.quantize_rows_int8(stacked[0, 0].cuda())
    assert q.shape == (70,) and scale.shape == () and gemm.dequantize_rows_int8(q, scale).shape == (70,)


def test_captured_and_on_other_streams(built_lib):
    """Products of every size captured into two graphs, replayed in turn on new operands, beside eager calls on a stream of their own."""
    from avelang_b200 import gdn, gemm, norm
    gen = torch.Generator().manual_seed(2)
    sizes = [(1, 512, 300), (64, 2048, 512), (700, 3000, 128), (2600, 2050, 200)]
    sets = [[torch.randn(m, k, generator=gen).bfloat16().cuda(), torch.randn(m, k, generator=gen).bfloat16().cuda(), *gemm.quantize_rows_int8(torch.randn(n, k, generator=gen).cuda())] for m, n, k in sizes]

    def step(x, res, wq, ws):
        q, scale, h = norm.rms_norm_int8(x, residual=res)
        return gemm.gemm_int8_transposed_b(q, wq, scale, ws), h

    def both():
        return [t for s in sets for t in step(*s)]

    both()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(both())
        graphs.append(g)
    for turn in range(3):
        for x, res, _, _ in sets:
            x.copy_(torch.randn_like(x))
            res.copy_(torch.randn_like(res))
        want = both()
        for t in outs[0] + outs[1]:
            t.zero_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = both()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b, c, d in zip(want, outs[0], outs[1], other):
            assert torch.equal(a, b) and torch.equal(a, c) and torch.equal(a, d)
    assert gdn.read_status() == 0


@pytest.mark.parametrize("tokens", [1, 7, 64, 500])
def test_a_layer_s_step(built_lib, tokens):
    """Norm with the residual to 8 bits, product, sum: against the same in 64 bits from the numbers that were stored."""
    from avelang_b200 import gemm, norm
    gen = torch.Generator().manual_seed(tokens)
    hidden, inner = 512, 1000
    x, res = torch.randn(tokens, hidden, generator=gen).bfloat16(), torch.randn(tokens, hidden, generator=gen).bfloat16()
    w_in, w_out, w = torch.randn(inner, hidden, generator=gen) * 0.05, torch.randn(hidden, inner, generator=gen) * 0.05, torch.rand(hidden, generator=gen) + 0.5
    bi, si = gemm.quantize_rows_int8(w_in.cuda())
    bo, so = gemm.quantize_rows_int8(w_out.bfloat16().cuda())
    q, s, h = norm.rms_norm_int8(x.cuda(), w.cuda(), residual=res.cuda())
    y = gemm.gemm_int8_transposed_b(q, bi, s, si)
    check(y, q.cpu(), bi.cpu(), s.cpu(), si.cpu(), None)
    q2, s2 = gemm.quantize_rows_int8(torch.tanh(y))
    out = gemm.gemm_int8_transposed_b(q2, bo, s2, so)
    check(out, q2.cpu(), bo.cpu(), s2.cpu(), so.cpu(), None)
    out, total = norm.rms_norm(out, residual=h, sum_out=h)
    # against the layer without rounding to 8 bits: operands within scale / 2 of their values, errors of K products that add like a walk
    hd = (x.double() + res.double()).bfloat16().double()
    yd = torch.tanh((hd / torch.sqrt(hd.square().mean(-1, keepdim=True) + 1e-6) * w.double()) @ w_in.double().t()) @ w_out.double().t()
    want = hd + yd
    assert float((total.cpu().double() - want).norm() / want.norm()) < 0.02


@pytest.mark.parametrize("n", [12352, 12351])
def test_offsets_beyond_32_bits(built_lib, n):
    """A result of more than 2^31 elements: its first and last rows, and those around the element 2^31."""
    from avelang_b200 import gemm
    m, k = 180000, 32
    gen = torch.Generator(device="cuda").manual_seed(n)
    a, b = (torch.randint(-128, 128, (r, k), generator=gen, dtype=torch.int8, device="cuda") for r in (m, n))
    sa, sb = torch.rand(m, generator=gen, device="cuda"), torch.rand(n, generator=gen, device="cuda")
    got = gemm.gemm_int8_transposed_b(a, b, sa, sb)
    for at in (0, (1 << 31) // n - 1, m - 3):
        rows = slice(at, at + 3)
        check(got[rows], a[rows].cpu(), b.cpu(), sa[rows].cpu(), sb.cpu(), None)


def test_rows_of_operands_beyond_32_bits(built_lib):
    """Rows of B more than 2^31 bytes apart from the first, in every form."""
    from avelang_b200 import gemm
    n, k, pitch = 40, 200, 1 << 26
    pool = torch.empty(n * pitch, dtype=torch.int8, device="cuda")
    b = pool.as_strided((n, k), (pitch, 1))
    b.copy_(torch.randint(-128, 128, (n, k), dtype=torch.int8, device="cuda"))
    sb = torch.rand(n, device="cuda") + 0.5
    for m in (1, 2, 30, 100, 300):
        a = torch.randint(-128, 128, (m, 208), dtype=torch.int8, device="cuda")[:, :k]
        sa = torch.rand(m, device="cuda") + 0.5
        got = gemm.gemm_int8_transposed_b(a, b, sa, sb, out_dtype=torch.float32)
        check(got, a.cpu(), b.cpu(), sa.cpu(), sb.cpu(), None)
    del b, pool
    torch.cuda.empty_cache()
