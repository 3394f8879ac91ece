"""Layer norm and its gradients against the formulas in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(rows, n, dt, wdt, seed, shift=0.5):
    gen = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, n, generator=gen) * 1.5 + shift).to(dt)
    w, b = (torch.randn(n, generator=gen) * 0.3 + 1.0).to(wdt), (torch.randn(n, generator=gen) * 0.3).to(wdt)
    return x, w, b, torch.randn(rows, n, generator=gen).to(dt)


def reference(x, w, b, eps):
    xd = x.double()
    mean = xd.mean(-1)
    rstd = 1.0 / torch.sqrt(xd.var(-1, unbiased=False) + eps)
    xh = (xd - mean[..., None]) * rstd[..., None]
    y = xh if w is None else xh * w.double()
    return (y if b is None else y + b.double()), mean, rstd, xh


def check_forward(got, x, w, b, eps):
    """A sum of n numbers over a tree of partial sums loses at most (n / threads + log2 threads) half steps, 64 are enough up to 28672 columns; the mean's loss
    reaches y times rstd."""
    y, mean, rstd = got
    y_ref, m_ref, r_ref, xh = reference(x, w, b, eps)
    u = 64 * 2.0 ** -24
    top = x.double().abs().amax(-1)
    assert ((mean.cpu().double() - m_ref).abs() <= u * top).all()
    # (x - mean)^2 each within 2 u top |x - mean| + ..., relative to the variance: 4 u top rstd
    assert ((rstd.cpu().double() / r_ref - 1).abs() <= u + 4 * u * top * r_ref).all()
    scale = 1.0 if w is None else w.double().abs()
    loss = (u + 4 * u * top * r_ref)[..., None] * xh.abs() * scale + (u * top * r_ref)[..., None] * scale + 2.0 ** -23 * y_ref.abs()
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert ((y.cpu().double() - y_ref).abs() <= half * y_ref.abs() + (1 + half) * loss + tiny).all()


SHAPES = [(1, 1), (3, 2), (5, 7), (2, 64), (37, 65), (9, 255), (33, 256), (4, 257), (70, 512), (5, 1000), (3, 1409), (37, 2048), (2, 2047), (3, 4096), (2, 5000), (2, 8192),
          (2, 16384), (1, 20001), (2, 28672), (2, 25000), (1, 28671)]


@pytest.mark.parametrize("rows,n", SHAPES)
@pytest.mark.parametrize("dt,wdt", [("bf16", "fp32"), ("bf16", "bf16"), ("fp16", "fp16"), ("fp32", "fp32")])
def test_forward_and_gradients(built_lib, rows, n, dt, wdt):
    from avelang_b200 import norm
    x, w, b, dy = make(rows, n, DT[dt], DT[wdt], n)
    got = norm.layer_norm(x.cuda(), w.cuda(), b.cuda(), 1e-5, return_stats=True)
    check_forward(got, x, w, b, 1e-5)
    mean, rstd = got[1], got[2]
    dx, dw, db = norm.layer_norm_backward(dy.cuda(), x.cuda(), mean, rstd, w.cuda())
    md, rd = mean.cpu().double()[:, None], rstd.cpu().double()[:, None]
    xd, dyd, wd = x.double(), dy.double(), w.double()
    xh = (xd - md) * rd
    wdy = dyd * wd
    dx_ref = rd * (wdy - wdy.mean(-1, keepdim=True) - xh * (wdy * xh).mean(-1, keepdim=True))
    u = 64 * 2.0 ** -24
    top = xd.abs().amax(-1, keepdim=True) * rd  # x - mean loses at most half a step of what the larger of the two is, times rstd
    xh_loss = 2.0 ** -22 * (xh.abs() + top)
    loss = rd * (2.0 ** -22 * wdy.abs() + u * wdy.abs().mean(-1, keepdim=True) + (xh.abs() + xh_loss) * (u * (wdy * xh).abs() + wdy.abs() * xh_loss).mean(-1, keepdim=True)
                 + xh_loss * (wdy * xh).mean(-1, keepdim=True).abs() + 2.0 ** -22 * xh.abs() * (wdy * xh).mean(-1, keepdim=True).abs())
    half = torch.finfo(x.dtype).eps / 2
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert ((dx.cpu().double() - dx_ref).abs() <= half * dx_ref.abs() + (1 + half) * loss + tiny).all()
    # a column's sum: rows / CTAs and a tree of partial sums behind them
    whalf = torch.finfo(w.dtype).eps / 2
    for d, ref, mag in ((dw, (dyd * xh).sum(0), (dyd * xh).abs().sum(0) + (dyd.abs() * xh_loss).sum(0) / u), (db, dyd.sum(0), dyd.abs().sum(0))):
        assert d.dtype == w.dtype
        assert ((d.cpu().double() - ref).abs() <= whalf * ref.abs() + (1 + whalf) * u * mag + tiny).all()


@pytest.mark.parametrize("rows,n,dt", [(10700, 520, "bf16"), (10700, 1024, "fp16"), (4000, 1540, "fp32"), (11000, 1536, "bf16"), (5500, 4096, "bf16"), (2700, 8192, "bf16"), (1340, 8196, "fp32"),
                                       (10700, 264, "bf16"), (1400, 16384, "fp16")])
def test_rings_that_turn(built_lib, rows, n, dt):
    """More rows a group than its ring has slots: each slot is filled several times."""
    test_forward_and_gradients(built_lib, rows, n, dt, "fp32")


@pytest.mark.parametrize("rows,n", [(3000, 64), (5001, 100), (2500, 2048), (1300, 1409), (700, 8192)])
def test_many_rows(built_lib, rows, n):
    """Every CTA meets several rows; twice the same bits."""
    from avelang_b200 import norm
    x, w, b, dy = make(rows, n, torch.bfloat16, torch.float32, 3)
    xd, dyd = x.cuda(), dy.cuda()
    got = norm.layer_norm(xd, w.cuda(), b.cuda(), 1e-5, return_stats=True)
    check_forward(got, x, w, b, 1e-5)
    dx, dw, db = norm.layer_norm_backward(dyd, xd, got[1], got[2], w.cuda())
    xh = (x.double() - got[1].cpu().double()[:, None]) * got[2].cpu().double()[:, None]
    u = 64 * 2.0 ** -24
    for d, ref, mag in ((dw, (dy.double() * xh).sum(0), (dy.double() * xh).abs().sum(0) * 2), (db, dy.double().sum(0), dy.double().abs().sum(0))):
        assert ((d.cpu().double() - ref).abs() <= u * mag + 2.0 ** -24 * ref.abs()).all()
    again = norm.layer_norm_backward(dyd, xd, got[1], got[2], w.cuda())
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


def test_without_parameters_strides_shapes_and_in_place(built_lib):
    from avelang_b200 import norm
    x, w, b, dy = make(24, 512, torch.bfloat16, torch.float32, 5)
    xc = x.cuda()
    check_forward(norm.layer_norm(xc, return_stats=True), x, None, None, 1e-5)
    check_forward(norm.layer_norm(xc, w.cuda(), None, 1e-3, return_stats=True), x, w, None, 1e-3)
    y, m, r = norm.layer_norm(xc.view(2, 3, 4, 512), w.cuda(), b.cuda(), return_stats=True)
    assert y.shape == (2, 3, 4, 512) and m.shape == r.shape == (2, 3, 4)
    check_forward((y.view(24, 512), m.flatten(), r.flatten()), x, w, b, 1e-5)
    for lo, hi in ((128, 384), (3, 200)):  # columns of a wider matrix, on and off 16 bytes
        part, wp, bp = xc[:, lo:hi], w[lo:hi].cuda(), b[lo:hi].cuda()
        check_forward(norm.layer_norm(part, wp, bp, return_stats=True), x[:, lo:hi], w[lo:hi], b[lo:hi], 1e-5)
        _, m, r = norm.layer_norm(part, wp, bp, return_stats=True)
        a = norm.layer_norm_backward(dy.cuda()[:, lo:hi], part, m, r, wp)
        c = norm.layer_norm_backward(dy[:, lo:hi].contiguous().cuda(), part.contiguous(), m, r, wp)
        assert all(torch.allclose(p.float(), q.float(), rtol=2 ** -7, atol=1e-5) for p, q in zip(a, c))
    t = x.t().contiguous().cuda().t()  # rows that are not contiguous
    check_forward(norm.layer_norm(t, w.cuda(), b.cuda(), return_stats=True), x, w, b, 1e-5)
    z = xc.clone()
    want = norm.layer_norm(z, w.cuda(), b.cuda())
    assert norm.layer_norm(z, w.cuda(), b.cuda(), out=z).data_ptr() == z.data_ptr() and torch.equal(z, want)
    dx, dw, db = norm.layer_norm_backward(dy.cuda(), xc, *norm.layer_norm(xc, return_stats=True)[1:])
    assert dw is None and db is None


def test_constant_rows_a_large_mean_and_no_rows(built_lib):
    from avelang_b200 import norm
    w, b = torch.ones(1000, device="cuda"), torch.full((1000,), 0.25, device="cuda")
    y, m, r = norm.layer_norm(torch.full((3, 1000), 5.0, device="cuda"), w, b, return_stats=True)
    assert (y - 0.25).abs().max() <= 1e-3 and torch.allclose(m, torch.full_like(m, 5.0)) and torch.allclose(r, torch.full_like(r, 1e-5 ** -0.5), rtol=1e-3)
    x, w2, b2, _ = make(4, 1000, torch.float32, torch.float32, 6, shift=1e4)
    check_forward(norm.layer_norm(x.cuda(), w2.cuda(), b2.cuda(), return_stats=True), x, w2, b2, 1e-5)
    e = torch.empty(0, 1000, device="cuda")
    y, m, r = norm.layer_norm(e, w, b, return_stats=True)
    assert y.shape == (0, 1000) and m.shape == (0,)
    dx, dw, db = norm.layer_norm_backward(e, e, m, r, w)
    assert dx.shape == (0, 1000) and (dw == 0).all() and (db == 0).all()
    bad = torch.randn(3, 1000, device="cuda")
    bad[1, 5] = float("nan")
    y = norm.layer_norm(bad, w, b)
    assert y[1].isnan().all() and y[[0, 2]].isfinite().all()


def test_autograd_captured_steps_and_two_streams(built_lib):
    from avelang_b200 import norm
    x, w, b, dy = (t.cuda() for t in make(40, 384, torch.float32, torch.float32, 8))
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = norm.LayerNormFunction.apply(*leaves, 1e-5)
    got = torch.autograd.grad(y, leaves, dy)
    eps = 1e-2  # differences in 64 bits of the formula, along a random direction
    f = lambda a, c, d: (reference(a.cpu(), c.cpu(), d.cpu(), 1e-5)[0] * dy.cpu().double()).sum()
    for i, t in enumerate((x, w, b)):
        step = torch.randn_like(t, dtype=torch.float64)
        args = [u.double() for u in (x, w, b)]
        up, down = list(args), list(args)
        up[i], down[i] = args[i] + eps * step, args[i] - eps * step
        slope = (f(*up) - f(*down)) / (2 * eps)
        assert abs(float((got[i].double() * step).sum()) - float(slope)) <= 1e-3 * (abs(float(slope)) + float((got[i].double() * step).abs().sum()) * 1e-2)
    mean, rstd = norm.layer_norm(x, w, b, return_stats=True)[1:]
    want = norm.layer_norm_backward(dy, x, mean, rstd, w)
    graphs, outs = [], []
    for _ in range(2):  # two captured graphs with scratch of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(norm.layer_norm_backward(dy, x, mean, rstd, w))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(p, q) for p, q in zip(o, want))
