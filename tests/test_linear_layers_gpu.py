"""Layer norm and linear attention as a model runs them: a layer's prefill and decode steps over a pool of states, and a training step.  Every operator is held to its own bound on
the inputs that it met in the run."""
import pytest
import torch

import test_layer_norm_gpu as N
import test_linear_backward_gpu as BW
import test_linear_decode_gpu as D
import test_linear_prefill_gpu as P

pytestmark = pytest.mark.gpu
H, HK, HV, DK, DV = 512, 2, 4, 128, 64


def weights(seed):
    gen = torch.Generator().manual_seed(seed)
    wide = HK * DK * 2 + HV * DV * 2
    return ((torch.randn(H, generator=gen) * 0.1 + 1.0).cuda(), (torch.randn(H, generator=gen) * 0.1).cuda(), (torch.randn(wide, H, generator=gen) * H ** -0.5).bfloat16().cuda(),
            (torch.randn(HV, H, generator=gen) * H ** -0.5).bfloat16().cuda(), (torch.randn(H, HV * DV, generator=gen) * (HV * DV) ** -0.5).bfloat16().cuda())


def heads(y, w_in, w_gate, product):
    """q, k, v and z as column slices of one projection, and the decays."""
    B, T = y.shape[:2]
    p = product(y.reshape(B * T, H), w_in).view(B, T, -1)
    g = -torch.nn.functional.softplus((y.reshape(B * T, H) @ w_gate.t()).float()).view(B, T, HV) * 0.2
    q, k, v, z = p.split([HK * DK, HK * DK, HV * DV, HV * DV], -1)
    return q.view(B, T, HK, DK), k.view(B, T, HK, DK), v.view(B, T, HV, DV), z.view(B, T, HV, DV), g


def test_prefill_then_decode(built_lib):
    """A packed prompt into slots of a pool, then three tokens for each sequence."""
    from avelang_b200 import gdn, gemm, linear_attention as L, norm
    nw, nb, w_in, w_gate, w_out = weights(1)
    lens = [70, 1, 0, 200, 64]
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    idx = torch.tensor([4, 0, 6, 2, 5], dtype=torch.int32)
    gen = torch.Generator().manual_seed(2)
    pool = torch.randn(8, HV, DK, DV, generator=gen).cuda()
    xs = [torch.randn(1, sum(lens), H, generator=gen).bfloat16()] + [torch.randn(len(lens), 1, H, generator=gen).bfloat16() for _ in range(3)]
    for step, x in enumerate(xs):
        before = pool.cpu()
        xd = x.cuda()
        y, mean, rstd = norm.layer_norm(xd, nw, nb, return_stats=True)
        N.check_forward((y.view(-1, H), mean.flatten(), rstd.flatten()), x.view(-1, H), nw.cpu(), nb.cpu(), 1e-5)
        q, k, v, z, g = heads(y, w_in, w_gate, gemm.gemm_pipeline_transposed_b)
        if step == 0:
            o, state = L.chunk_linear_attention(q, k, v, g, None, pool, True, cu.cuda(), state_indices=idx.cuda())
        else:
            o, state = L.fused_recurrent_linear_attention(q, k, v, g, None, pool, state_indices=idx.cuda())
        assert state.data_ptr() == pool.data_ptr() and gdn.read_status() == 0
        (P if step == 0 else D).check(o, pool[idx.long().cuda()], *[t.cpu() for t in (q, k, v, g)], DK ** -0.5, before[idx.long()], *([cu] if step == 0 else []))
        assert torch.equal(pool.cpu()[[1, 3, 7]], before[[1, 3, 7]])
        n = gdn.gated_rmsnorm(o, z)
        nd = o.double() * torch.rsqrt((o.double() ** 2).mean(-1, keepdim=True) + 1e-6) * z.double() * torch.sigmoid(z.double())
        assert ((n.double() - nd).abs() <= 2.0 ** -8 * nd.abs() * (1 + 2.0 ** -8) + 64 * 2.0 ** -24 * nd.abs() + 1e-30).all()
        xd += gemm.gemm_pipeline_transposed_b(n.reshape(-1, HV * DV), w_out).view_as(xd)
        assert xd.isfinite().all()


@pytest.mark.parametrize("lens", [None, [70, 1, 0, 57]])
def test_training_step(built_lib, lens):
    """The gradient that each operator receives in the run, and the ones that it hands on."""
    from avelang_b200 import gdn, linear_attention as L, norm
    nw, nb, w_in, w_gate, w_out = weights(3)
    B, T = (2, 100) if lens is None else (1, sum(lens))
    cu = None if lens is None else torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    n_seqs = B if lens is None else len(lens)
    gen = torch.Generator().manual_seed(4)
    x = torch.randn(B, T, H, generator=gen).bfloat16()
    s0 = torch.randn(n_seqs, HV, DK, DV, generator=gen)
    xd, s0d = x.cuda().requires_grad_(), s0.cuda().requires_grad_()
    params = [t.requires_grad_() for t in (nw, nb, w_in, w_gate, w_out)]
    y = norm.LayerNormFunction.apply(xd, nw, nb, 1e-5)
    q, k, v, z, g = heads(y, w_in, w_gate, lambda a, w: a @ w.t())
    o, state = L.LinearAttentionFunction.apply(q, k, v, g, None, s0d, None if cu is None else cu.cuda())
    for t in (y, q, k, v, g, o, state):
        t.retain_grad()
    out = (o * torch.sigmoid(z)).reshape(B, T, HV * DV) @ w_out.t()
    (out.float().square().mean() + 0.01 * state.square().mean()).backward()
    assert gdn.read_status() == 0
    c = lambda t: t.detach().cpu()
    P.check(c(o), c(state), c(q), c(k), c(v), c(g), DK ** -0.5, s0, cu)
    BW.check([t.grad for t in (q, k, v, g, s0d)], c(q), c(k), c(v), c(g), DK ** -0.5, s0, cu, c(o.grad), c(state.grad))
    # the norm's gradients, from the gradient that reaches it, are those of a call of its own
    _, mean, rstd = norm.layer_norm(xd.detach(), nw.detach(), nb.detach(), return_stats=True)
    for a, b in zip((xd.grad, nw.grad, nb.grad), norm.layer_norm_backward(y.grad, xd.detach(), mean, rstd, nw.detach())):
        assert torch.equal(a, b)
    assert all(p.grad is not None and p.grad.isfinite().all() and p.grad.abs().max() > 0 for p in params)


def test_unused_results_have_no_gradient(built_lib):
    """Only the final states are used, or only the outputs."""
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = P.make(1, 90, 1, 2, 64, 128, "token", 5, 1, 0.1)
    for use in (0, 1):
        leaves = [t.cuda().requires_grad_() for t in (q, k, v, g, s0)]
        results = L.LinearAttentionFunction.apply(*leaves[:4], None, leaves[4], None)
        results[use].float().square().sum().backward()
        d = (2 * results[use].detach().float()).cpu()
        d_o, d_f = (d.bfloat16(), None) if use == 0 else (torch.zeros_like(v), d)
        BW.check([t.grad for t in leaves], q, k, v, g, 64 ** -0.5, s0, None, d_o, d_f)


def test_captured_training_step(built_lib):
    """Forward and backward captured into one graph and replayed on other inputs: the same bits as eager calls."""
    from avelang_b200 import linear_attention as L, norm

    def step(x, w, b, q, k, g):
        y = norm.LayerNormFunction.apply(x, w, b, 1e-5)
        o, s = L.LinearAttentionFunction.apply(q, k, y.view(1, 150, 2, 128), g, None, None, None)
        return torch.autograd.grad(o.float().square().sum() + s.sum(), (x, w, b, q, k, g))

    def inputs(seed):
        gen = torch.Generator().manual_seed(seed)
        q, k, _, g, _ = P.make(1, 150, 1, 2, 128, 128, "token", seed, 0, 0.1)
        return [torch.randn(150, 256, generator=gen).bfloat16(), torch.randn(256, generator=gen), torch.randn(256, generator=gen), q, k, g]

    held = [t.cuda().requires_grad_() for t in inputs(6)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*held)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(*held)
    for seed in (7, 8):
        new = inputs(seed)
        with torch.no_grad():
            for a, b in zip(held, new):
                a.copy_(b)
        graph.replay()
        eager = step(*[t.cuda().requires_grad_() for t in new])
        assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_two_streams_at_once(built_lib):
    """The same calls on two streams, scratch of each apart."""
    from avelang_b200 import linear_attention as L, norm
    args = [P.cuda(*P.make(1, 1500, 1, 2, 128, 128, "token", s, 1, 0.02)) for s in (9, 10)]
    rows = [torch.randn(2000, 1024, device="cuda").bfloat16() for _ in range(2)]
    w = torch.ones(1024, device="cuda")

    def work(i):
        q, k, v, g, s0 = args[i]
        o, s = L.chunk_linear_attention(q, k, v, g, None, s0, True)
        grads = L.linear_attention_backward(q, k, v, g, o, None, s0, s)
        y, m, r = norm.layer_norm(rows[i], w, w, return_stats=True)
        return [o, s, *grads, y, *norm.layer_norm_backward(y, rows[i], m, r, w)]

    alone = [work(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(work(i))
    torch.cuda.synchronize()
    for i in range(2):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, alone[i]))


def test_gradients_have_no_gradients(built_lib):
    from avelang_b200 import linear_attention as L, norm
    q, k, v, g, _ = [t.cuda().requires_grad_() if t is not None else None for t in P.make(1, 70, 1, 1, 64, 64, "token", 11)]
    o, _ = L.LinearAttentionFunction.apply(q, k, v, g, None, None, None)
    first = torch.autograd.grad(o.float().square().sum(), (q, k, v, g), create_graph=True)
    for t in first:
        with pytest.raises(RuntimeError, match="twice"):
            t.float().sum().backward(retain_graph=True)
    x = torch.randn(3, 64, device="cuda", requires_grad=True)
    dx, = torch.autograd.grad(norm.LayerNormFunction.apply(x, None, None, 1e-5).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="twice"):
        dx.sum().backward()


def test_refusals_of_the_differentiable_call(built_lib):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = P.cuda(*P.make(1, 70, 1, 1, 64, 64, "token", 12, 1))
    f = L.LinearAttentionFunction.apply
    for match, args in (("q must have dtype", (q.float(), k, v, g)), ("k must have shape", (q, k[:, :50], v, g)), ("g must have dtype", (q, k, v, g.double())),
                        ("one state per sequence", (q, k, v, g, None, s0.expand(2, -1, -1, -1).contiguous()))):
        with pytest.raises(ValueError, match=match):
            f(*args, *[None] * (7 - len(args)))
