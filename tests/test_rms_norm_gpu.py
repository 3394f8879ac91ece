"""RMS norm with the residual's addition, its 8-bit form and its gradients, against the formulas in 64 bits.

U = 80 half steps of fp32: a sum over a row goes through at most 28 additions in a thread, 5 between the lanes, 32 between the warps, and each term is rounded; a sum of squares (no
cancellation) is then within U of itself, its root within U / 2, and three products behind it add as many half steps."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
U = 80 * 2.0 ** -24


def half(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return torch.finfo(dt).smallest_normal * torch.finfo(dt).eps


def make(rows, n, dt, wdt, seed, residual=True, plus_one=False):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, n, generator=gen) * 1.5).to(dt)
    res = (torch.randn(rows, n, generator=gen) * 2.0).to(dt) if residual else None
    w = None if wdt is None else (torch.randn(n, generator=gen) * 0.3 + (0.0 if plus_one else 1.0)).to(wdt)
    return x, res, w


def reference(x, res, w, plus_one, eps):
    h = x if res is None else (x.double() + res.double()).to(x.dtype)
    if res is not None and x.dtype != torch.float32:  # the kernel's sum is rounded to fp32 first; for these inputs that changes nothing
        assert torch.equal(h, (x.float() + res.float()).to(x.dtype))
    hd = h.double()
    rstd = 1.0 / torch.sqrt(hd.square().mean(-1) + eps)
    y = hd * rstd[..., None]
    return h, rstd, y if w is None else y * (w.double() + (1.0 if plus_one else 0.0))


def check_norm(got_y, got_h, got_rstd, x, res, w, plus_one, eps):
    h, rstd, y = reference(x, res, w, plus_one, eps)
    if res is not None:
        assert torch.equal(got_h.cpu(), h)
    if got_rstd is not None:
        assert got_rstd.shape == x.shape[:-1]
        assert ((got_rstd.cpu().double() / rstd - 1).abs() <= U).all()
    assert ((got_y.cpu().double() - y).abs() <= (half(x.dtype) + (1 + half(x.dtype)) * U) * y.abs() + tiny(x.dtype)).all()


def check_int8(q, scale, y):
    """scale within U of the row's largest / 127; q within half a step, and 127 U of one, of y / scale."""
    assert q.dtype == torch.int8 and q.shape == y.shape and scale.shape == y.shape[:-1]
    q, scale = q.cpu().double(), scale.cpu().double()
    top = y.abs().amax(-1)
    assert ((scale / (top / 127.0) - 1).abs() <= U).all()
    assert ((q * scale[..., None] - y).abs() <= scale[..., None] * (0.5 + 127 * U)).all()
    assert (q.abs().amax(-1) == 127).all() and (q >= -127).all()


# every form of the rows: pieces of 16 bytes or single elements, few rows and many
SIZES = [(1, 8), (3, 64), (700, 64), (5, 256), (400, 512), (1, 2048), (37, 2048), (301, 1024), (600, 2048), (300, 4096), (2, 8192), (299, 8192), (7, 16384), (3, 28672), (1, 1), (5, 7), (9, 63),
         (640, 100), (3, 513), (300, 1409), (2, 4097), (1, 28671)]


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,n", SIZES)
def test_forward(built_lib, rows, n, dt):
    from avelang_b200 import norm
    seed = rows * 31 + n
    for residual, wide, plus_one in ((True, True, False), (False, False, True), (True, None, False)):
        wdt = None if wide is None else torch.float32 if wide else DT[dt]
        x, res, w = make(rows, n, DT[dt], wdt, seed, residual, plus_one)
        args = dict(residual=None if res is None else res.cuda(), zero_centered=plus_one)
        xg, wg = x.cuda(), None if w is None else w.cuda()
        got = norm.rms_norm(xg, wg, 1e-6, return_stats=True, **args)
        check_norm(got[0], got[1], got[-1], x, res, w, plus_one, 1e-6)
        again = norm.rms_norm(xg, wg, 1e-6, **args)
        assert torch.equal(again[0] if residual else again, got[0])
        if n > 1:
            q, scale, *h = norm.rms_norm_int8(xg, wg, 1e-6, **args)
            ref_h, _, y = reference(x, res, w, plus_one, 1e-6)
            check_int8(q, scale, y)
            assert not residual or torch.equal(h[0].cpu(), ref_h)
        assert torch.equal(xg.cpu(), x) and (res is None or torch.equal(args["residual"].cpu(), res))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("n", [64, 96, 2048, 2049, 12288])
def test_special_rows(built_lib, n, dt):
    """Rows of zeros, with an infinity, with a NaN, of the largest and of the smallest numbers, beside ordinary ones, which they leave as they are."""
    from avelang_b200 import norm
    x, _, w = make(12, n, DT[dt], torch.float32, n, False)
    plain = norm.rms_norm(x.cuda(), w.cuda(), 1e-6, return_stats=True)
    q0, s0 = norm.rms_norm_int8(x.cuda(), w.cuda(), 1e-6)
    x[1] = 0
    x[3, n // 2] = float("inf")
    x[5, n - 1] = float("nan")
    x[7] = torch.finfo(DT[dt]).smallest_normal
    x[9] = 0
    x[9, n // 3] = 60000.0
    y, rstd = norm.rms_norm(x.cuda(), w.cuda(), 1e-6, return_stats=True)
    q, scale = norm.rms_norm_int8(x.cuda(), w.cuda(), 1e-6)
    for r in (0, 2, 4, 6, 8, 10, 11):
        assert torch.equal(y[r], plain[0][r]) and torch.equal(rstd[r], plain[1][r]) and torch.equal(q[r], q0[r]) and torch.equal(scale[r], s0[r])
    assert (y[1] == 0).all() and (q[1] == 0).all() and scale[1] == 0 and abs(float(rstd[1]) - 1000.0) < 1e-2
    assert rstd[3] == 0 and torch.isnan(y[3, n // 2]) and torch.isnan(scale[3]) and (q[3] == 0).all()
    assert torch.isnan(y[5]).all() and torch.isnan(scale[5]) and (q[5] == 0).all()
    check_norm(y[[7, 9]], None, rstd[[7, 9]], x[[7, 9]], None, w, False, 1e-6)
    if dt == "fp16":  # (bf16's and fp32's smallest normal number: below what a scale stands for)
        check_int8(q[[7]], scale[[7]], reference(x[[7]], None, w, False, 1e-6)[2])
    else:
        assert scale[7] == 0 and (q[7] == 0).all()
    check_int8(q[[9]], scale[[9]], reference(x[[9]], None, w, False, 1e-6)[2])
    w2 = w.clone()
    w2[2] = float("nan")
    q, scale = norm.rms_norm_int8(x[:1].cuda(), w2.cuda(), 1e-6)
    assert torch.isnan(scale[0]) and (q == 0).all()


@pytest.mark.parametrize("dt", list(DT))
def test_int8_of_a_plain_row(built_lib, dt):
    """Ties go to the even number: a row of 127 and halves has scale 1, exactly."""
    from avelang_b200 import gemm
    for n in (64, 100, 512, 5000):
        row = torch.arange(n, dtype=torch.float32) % 101 / 2.0 - 25.0
        row[n // 2] = -127.0
        x = row.to(DT[dt]).repeat(3, 1)
        q, scale = gemm.quantize_rows_int8(x.cuda())
        assert (scale == 1.0).all() and torch.equal(q.cpu().float(), row.round().repeat(3, 1))  # (torch rounds ties to even)
        assert torch.equal(gemm.dequantize_rows_int8(q, scale, torch.float32).cpu(), row.round().repeat(3, 1))


def test_layouts(built_lib):
    """Rows apart, off 16 bytes, expanded, transposed, of more dimensions; results in the place of inputs; guards beside the rows stay as they were."""
    from avelang_b200 import norm
    gen = torch.Generator().manual_seed(5)
    base = torch.randn(40, 600, generator=gen).bfloat16()
    w = (torch.randn(512, generator=gen) * 0.2 + 1).float()
    for x in (base[:, :512], base[:, 3:515], base[::2, 40:552], base[:1, :512].expand(9, 512), base[:, :512].reshape(5, 8, 512), base[3, :512], base[:0, :512]):
        xg = base.cuda().as_strided(x.size(), x.stride(), x.storage_offset()) if x.numel() else x.cuda()
        res = torch.randn(x.shape, generator=gen).bfloat16()
        y, h, rstd = norm.rms_norm(xg, w.cuda(), 1e-5, residual=res.cuda(), return_stats=True)
        assert y.shape == h.shape == x.shape and rstd.shape == x.shape[:-1]
        if x.numel():
            check_norm(y, h, rstd, x, res, w, False, 1e-5)
        q, scale, h2 = norm.rms_norm_int8(xg, w.cuda(), 1e-5, residual=res.cuda())
        if x.numel():
            check_int8(q, scale, reference(x, res, w, False, 1e-5)[2])
            assert torch.equal(h2, h)
    wide = torch.randn(30, 640, generator=gen).bfloat16()
    x, res = wide[:, 8:520], torch.randn(30, 512, generator=gen).bfloat16()
    for dst in ("new", "x", "residual", "both"):
        store, rg = wide.cuda(), res.cuda()
        xg = store[:, 8:520]
        kw = {"new": {}, "x": dict(out=xg), "residual": dict(sum_out=rg), "both": dict(out=rg, sum_out=xg)}[dst]
        y, h = norm.rms_norm(xg, w.cuda(), 1e-5, residual=rg, **kw)
        check_norm(y, h, None, x, res, w, False, 1e-5)
        assert torch.equal(store[:, :8].cpu(), wide[:, :8]) and torch.equal(store[:, 520:].cpu(), wide[:, 520:])
        assert dst not in ("x",) or y.data_ptr() == xg.data_ptr()
    t = torch.randn(512, 12, generator=gen).half()
    check_norm(norm.rms_norm(t.cuda().t(), w.cuda(), 1e-5), None, None, t.t().contiguous(), None, w, False, 1e-5)
    weights = torch.randn(513, generator=gen)  # a weight off 16 bytes
    y = norm.rms_norm(wide.cuda()[:, :512], weights.cuda()[1:], 1e-5)
    check_norm(y, None, None, wide[:, :512], None, weights[1:], False, 1e-5)


# ---------------------------------------------------------------------------------------------------------------- gradients
def gradients(d_y, x, rstd, w, d_sum, plus_one):
    """By the formula in 64 bits, with the terms that rounding is measured by."""
    xh, g = x.double() * rstd.double()[..., None], d_y.double()
    wd = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double() + (1.0 if plus_one else 0.0)
    gw = g * wd
    c, c_abs = (gw * xh).mean(-1, keepdim=True), (gw * xh).abs().mean(-1, keepdim=True)
    r = rstd.double()[..., None]
    dx = r * (gw - xh * c) + (0.0 if d_sum is None else d_sum.double())
    loss = r * (6 * 2.0 ** -24 * (gw.abs() + (xh * c).abs()) + U * xh.abs() * c_abs) + 2.0 ** -23 * (0.0 if d_sum is None else d_sum.double().abs())
    flat = (g * xh).reshape(-1, x.shape[-1])
    return dx, loss, flat.sum(0), flat.abs().sum(0)


def check_backward(dx, dw, d_y, x, rstd, w, d_sum, plus_one):
    ref, loss, dw_ref, dw_abs = gradients(d_y, x, rstd, w, d_sum, plus_one)
    e = half(x.dtype)
    assert ((dx.cpu().double() - ref).abs() <= e * ref.abs() + (1 + e) * loss + tiny(x.dtype)).all()
    if w is None:
        assert dw is None
        return
    assert dw.dtype == w.dtype
    ew, rows = half(w.dtype), x.numel() // x.shape[-1]
    # a column's terms: their own two roundings, at most rows / 148 + 64 additions in a thread and the groups, 56 between the CTAs and the warps
    assert ((dw.cpu().double() - dw_ref).abs() <= ew * dw_ref.abs() + (1 + ew) * (rows / 148 + 128) * 2.0 ** -24 * dw_abs + tiny(w.dtype)).all()


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("rows,n", SIZES + [(2000, 2048), (1001, 1409), (4000, 64)])
def test_backward(built_lib, rows, n, dt):
    from avelang_b200 import norm
    for add, wide, plus_one in ((True, True, False), (False, False, True), (True, None, False)):
        x, d_sum, w = make(rows, n, DT[dt], None if wide is None else torch.float32 if wide else DT[dt], rows * 7 + n, add, plus_one)
        d_y = torch.randn(rows, n, generator=torch.Generator().manual_seed(n)).to(DT[dt])
        rstd = (1.0 / torch.sqrt(x.double().square().mean(-1) + 1e-6)).float()
        call = lambda: norm.rms_norm_backward(d_y.cuda(), x.cuda(), rstd.cuda(), None if w is None else w.cuda(), d_sum=None if d_sum is None else d_sum.cuda(), zero_centered=plus_one)
        dx, dw = call()
        check_backward(dx, dw, d_y, x, rstd, w, d_sum, plus_one)
        dx2, dw2 = call()
        assert torch.equal(dx2, dx) and (dw is None or torch.equal(dw2, dw))  # (no atomics)


def test_gradient_against_differences(built_lib):
    """The directional derivative of sum(y a) + sum(h b) along random directions of x, residual and weight, by central differences in 64 bits."""
    from avelang_b200 import norm
    gen = torch.Generator().manual_seed(11)
    for n, plus_one in ((200, False), (37, True)):
        x, res, w = make(9, n, torch.float32, torch.float32, n, True, plus_one)
        a, b = torch.randn(9, n, generator=gen), torch.randn(9, n, generator=gen)

        def value(x, r, w):
            h = x + r
            return (h / torch.sqrt(h.square().mean(-1, keepdim=True) + 1e-6) * (w + (1.0 if plus_one else 0.0)) * a.double()).sum() + (h * b.double()).sum()

        leaves = [t.cuda().requires_grad_(True) for t in (x, res, w)]
        y, h = norm.RmsNormFunction.apply(*leaves, 1e-6, plus_one)
        torch.autograd.backward([y, h], [a.cuda(), b.cuda()])
        for i in range(3):
            d = torch.randn(leaves[i].shape, generator=gen).double()
            at = lambda t: value(*[v.double() + (t * d if k == i else 0.0) for k, v in enumerate((x, res, w))])
            want = float((at(1e-5) - at(-1e-5)) / 2e-5)  # (off by the third derivative * 2e-11)
            terms = (leaves[i].grad.cpu().double() * d).abs().sum()
            assert abs(float((leaves[i].grad.cpu().double() * d).sum()) - want) <= 1e-5 * float(terms) + 1e-6


def test_function(built_lib):
    from avelang_b200 import norm
    x, res, w = make(33, 256, torch.bfloat16, torch.float32, 3)
    rstd = lambda t: (1.0 / torch.sqrt(t.double().square().mean(-1) + 1e-6)).float()
    gen = torch.Generator().manual_seed(4)
    d_y, d_h = torch.randn(33, 256, generator=gen).bfloat16(), torch.randn(33, 256, generator=gen).bfloat16()
    leaves = lambda *t: [v.cuda().requires_grad_(True) for v in t]
    a, b, c = leaves(x, res, w)
    y, h = norm.RmsNormFunction.apply(a, b, c, 1e-6)
    torch.autograd.backward([y, h], [d_y.cuda(), d_h.cuda()])
    _, r, _ = norm.rms_norm(x.cuda(), w.cuda(), 1e-6, residual=res.cuda(), return_stats=True)[0:3]
    stats = norm.rms_norm(h.detach(), w.cuda(), 1e-6, return_stats=True)[1].cpu()
    check_backward(a.grad, c.grad, d_y, h.detach().cpu(), stats, w, d_h, False)
    assert torch.equal(a.grad, b.grad) and a.grad.data_ptr() != b.grad.data_ptr()
    a, b, c = leaves(x, res, w)  # only the norm, then only the sum
    y, h = norm.RmsNormFunction.apply(a, b, c, 1e-6)
    y.backward(d_y.cuda())
    check_backward(a.grad, c.grad, d_y, h.detach().cpu(), stats, w, None, False)
    a, b, c = leaves(x, res, w)
    y, h = norm.RmsNormFunction.apply(a, b, c, 1e-6)
    h.backward(d_h.cuda())
    assert torch.equal(a.grad.cpu(), d_h) and torch.equal(b.grad.cpu(), d_h) and c.grad is None
    a, c = leaves(x, w)  # no residual; the gradient of a sum has strides of zero
    y = norm.RmsNormFunction.apply(a, None, c, 1e-6, True)
    y.float().sum().backward()
    stats = norm.rms_norm(x.cuda(), w.cuda(), 1e-6, return_stats=True, zero_centered=True)[1].cpu()
    check_backward(a.grad, c.grad, torch.ones_like(x), x, stats, w, None, True)
    a, = leaves(x)
    y = norm.RmsNormFunction.apply(a, None, None, 1e-6)
    (g,) = torch.autograd.grad(y, a, d_y.cuda())
    check_backward(g, None, d_y, x, stats, None, None, False)
    a, = leaves(x[:0])
    y = norm.RmsNormFunction.apply(a, None, c, 1e-6)
    y.sum().backward()
    assert a.grad.shape == (0, 256)


def test_captured_steps_and_streams(built_lib):
    """Two captured steps of forward and backward pass, replayed in turn on new inputs, and the same calls on a stream of their own."""
    from avelang_b200 import norm
    shapes = [(300, 2048), (64, 1000)]
    made = []
    for rows, n in shapes:
        x, res, w = make(rows, n, torch.bfloat16, torch.float32, n)
        made.append([x.cuda(), res.cuda(), w.cuda(), torch.randn(rows, n, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()])

    def step(x, res, w, d_y):
        y, h, rstd = norm.rms_norm(x, w, 1e-6, residual=res, return_stats=True)
        q = norm.rms_norm_int8(x, w, 1e-6, residual=res)
        return [y, h, rstd, *q, *norm.rms_norm_backward(d_y, h, rstd, w, d_sum=d_y)]

    for m in made:
        step(*m)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for m in made:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*m))
        graphs.append(g)
    for turn in range(3):
        for m in made:
            for i in (0, 1, 3):
                m[i].copy_(torch.randn_like(m[i]))
        wants = [step(*m) for m in made]
        for o in outs:
            for t in o:
                t.zero_()
        for g in graphs:
            g.replay()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            sides = [step(*m) for m in made]
        torch.cuda.synchronize()
        for want, out, other in zip(wants, outs, sides):
            assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, out, other))


@pytest.mark.parametrize("n", [2048, 2047])
def test_offsets_beyond_32_bits(built_lib, n):
    """More than 2^31 elements: the first and the last rows, and those around the element 2^31, in the norm, its 8-bit form, its gradients and the way back from 8 bits."""
    from avelang_b200 import gemm, norm
    rows = 1050000
    gen = torch.Generator(device="cuda").manual_seed(n)
    x = torch.randn(rows, n, generator=gen, device="cuda", dtype=torch.bfloat16)
    w = torch.rand(n, generator=gen, device="cuda") + 0.5
    parts = [slice(at, at + 3) for at in (0, (1 << 31) // n - 1, rows - 3)]
    y, h, rstd = norm.rms_norm(x, w, residual=x, return_stats=True)
    for p in parts:
        check_norm(y[p], h[p], rstd[p], x[p].cpu(), x[p].cpu(), w.cpu(), False, 1e-6)
    q, scale = norm.rms_norm_int8(x, w)
    back = gemm.dequantize_rows_int8(q, scale)
    for p in parts:
        check_int8(q[p], scale[p], reference(x[p].cpu(), None, w.cpu(), False, 1e-6)[2])
        assert torch.equal(back[p], (q[p].float() * scale[p][:, None]).bfloat16())
    del q, back
    dx, _ = norm.rms_norm_backward(y, h, rstd, w, d_sum=x)
    for p in parts:
        ref, loss, _, _ = gradients(y[p].cpu(), h[p].cpu(), rstd[p].cpu(), w.cpu(), x[p].cpu(), False)
        e = half(x.dtype)
        assert ((dx[p].cpu().double() - ref).abs() <= e * ref.abs() + (1 + e) * loss + tiny(x.dtype)).all()
    del x, y, h, dx
    torch.cuda.empty_cache()
