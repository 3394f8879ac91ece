"""Layer norm in a training step of a layer: its results and its gradients against the formulas in 64 bits, on what met it in the run."""
import pytest
import torch

import test_layer_norm_gpu as N
import test_linear_layers_gpu as M

pytestmark = pytest.mark.gpu


def check_gradients(got, dy, x, mean, rstd, w):
    """The bounds of tests/test_layer_norm_gpu.py: sums lose at most 64 half steps of their terms' absolute values, x - mean half a step of the larger of the two."""
    dx, dw, db = [t.cpu() for t in got]
    md, rd = mean.double()[:, None], rstd.double()[:, None]
    xd, dyd, wd = x.double(), dy.double(), w.double()
    xh = (xd - md) * rd
    wdy = dyd * wd
    dx_ref = rd * (wdy - wdy.mean(-1, keepdim=True) - xh * (wdy * xh).mean(-1, keepdim=True))
    u = 64 * 2.0 ** -24
    xh_loss = 2.0 ** -22 * (xh.abs() + xd.abs().amax(-1, keepdim=True) * rd)
    loss = rd * (2.0 ** -22 * wdy.abs() + u * wdy.abs().mean(-1, keepdim=True) + (xh.abs() + xh_loss) * (u * (wdy * xh).abs() + wdy.abs() * xh_loss).mean(-1, keepdim=True)
                 + (xh_loss + 2.0 ** -22 * xh.abs()) * (wdy * xh).mean(-1, keepdim=True).abs())
    half, tiny = torch.finfo(x.dtype).eps / 2, torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps
    assert dx.dtype == x.dtype and ((dx.double() - dx_ref).abs() <= half * dx_ref.abs() + (1 + half) * loss + tiny).all()
    whalf = torch.finfo(w.dtype).eps / 2
    for d, ref, mag in ((dw, (dyd * xh).sum(0), (dyd * xh).abs().sum(0) + (dyd.abs() * xh_loss).sum(0) / u), (db, dyd.sum(0), dyd.abs().sum(0))):
        assert d.dtype == w.dtype and ((d.double() - ref).abs() <= whalf * ref.abs() + (1 + whalf) * u * mag + tiny).all()


@pytest.mark.parametrize("lens", [None, [70, 1, 0, 57], [700, 3, 900]])
def test_norm_in_a_training_step(built_lib, lens):
    from avelang_b200 import gdn, linear_attention as L, norm
    nw, nb, w_in, w_gate, w_out = [t.requires_grad_() for t in M.weights(5)]
    B, T = (2, 100) if lens is None else (1, sum(lens))
    cu = None if lens is None else torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")
    x = (torch.randn(B, T, M.H, generator=torch.Generator().manual_seed(6)) * 2 + 0.3).bfloat16()
    xd = x.cuda().requires_grad_()
    y = norm.LayerNormFunction.apply(xd, nw, nb, 1e-5)
    y.retain_grad()
    q, k, v, z, g = M.heads(y, w_in, w_gate, lambda a, w: a @ w.t())
    o, state = L.LinearAttentionFunction.apply(q, k, v, g, None, None, cu)
    out = (o * torch.sigmoid(z)).reshape(B, T, M.HV * M.DV) @ w_out.t()
    (out.float().square().mean() + 0.01 * state.square().mean()).backward()
    assert gdn.read_status() == 0
    c = lambda t: t.detach().cpu().reshape(-1, t.shape[-1]) if t.dim() > 1 else t.detach().cpu()
    _, mean, rstd = norm.layer_norm(xd.detach(), return_stats=True)
    N.check_forward((c(y), mean.flatten().cpu(), rstd.flatten().cpu()), c(xd), c(nw), c(nb), 1e-5)
    check_gradients((c(xd.grad), nw.grad, nb.grad), c(y.grad), c(xd), mean.flatten().cpu(), rstd.flatten().cpu(), c(nw))


def test_the_bounds_see_a_wrong_formula():
    """On the CPU's side: gradients without the projection onto the row, and column sums without the statistics, are refused."""
    x, w, b, dy = N.make(40, 384, torch.float32, torch.float32, 7)
    _, mean, rstd, xh = N.reference(x, w, b, 1e-5)
    xd, wdy = xh, dy.double() * w.double()
    dx = rstd[:, None] * (wdy - wdy.mean(-1, keepdim=True) - xd * (wdy * xd).mean(-1, keepdim=True))
    right = [dx, (dy.double() * xh).sum(0), dy.double().sum(0)]
    check = lambda g: check_gradients([t.float() for t in g], dy, x, mean.float(), rstd.float(), w)
    check(right)
    for i, t in ((0, rstd[:, None] * (wdy - wdy.mean(-1, keepdim=True))), (1, (dy.double() * x.double()).sum(0)), (2, wdy.sum(0))):
        with pytest.raises(AssertionError):
            check(right[:i] + [t] + right[i + 1:])
