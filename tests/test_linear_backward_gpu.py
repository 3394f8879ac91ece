"""Gradients of linear attention with a decay for each head, against autograd of the recurrence in 64 bits and against differences."""
import pytest
import torch

from oracle import linear_oracle as O
from test_linear_prefill_gpu import cuda, make

pytestmark = pytest.mark.gpu


def grads_in(shape_v, n, dk, seed, final):
    gen = torch.Generator().manual_seed(seed)
    d_o = torch.randn(shape_v, generator=gen).bfloat16()
    return d_o, torch.randn(n, shape_v[2], dk, shape_v[3], generator=gen) * 0.1 if final else None


def check(got, q, k, v, g, scale, s0, cu, d_o, d_final):
    """dq, dk and dv are scans like the forward pass and have its bound (2^-16 for the two-term operands, 2^-22 a rounding of the sums); the state's
    gradient has that of a state.  The gradient of g adds, token by token, sums A and B over pairs that are within 2^-18 of their terms' absolute values, so it is within
    that of all that was added."""
    ref = O.gradients(q, k, v, g, scale, s0, cu, d_o, d_final)
    mag = O.gradients(q.abs(), k.abs(), v.abs(), g, scale, None if s0 is None else s0.abs(), cu, d_o.abs(), None if d_final is None else d_final.abs())
    chunks = max([n for _, _, n in O.spans(q, cu)] + [0]) // 64 + 1
    es = (16 + chunks) * 2.0 ** -22
    eo = 2.0 ** -16 + es + 200 * 2.0 ** -24
    names = ("dq", "dk", "dv", "dg", "ds0")
    for name, x, r, m in zip(names, got, ref, mag):
        if r is None:
            assert x is None, name
            continue
        assert x.shape == r.shape, name
        x = x.cpu().double()
        assert x.isfinite().all(), name
        if name in ("dq", "dk", "dv"):
            tol = 2.0 ** -8 * r.abs() * (1 + 1e-3) + eo * m
        elif name == "ds0":
            tol = 2 * es * m
        else:
            # |A| + |B| of each token (the sums over the value heads of a key head are larger still)
            terms = ((q.double().abs() * mag[0]).sum(-1) + (k.double().abs() * mag[1]).sum(-1)).repeat_interleave(v.shape[2] // q.shape[2], 2)
            tol, mean = torch.zeros_like(r), torch.zeros_like(r)
            for b, t0, n in O.spans(q, cu):
                part = terms[b, t0:t0 + n]
                if g.dim() == 1:  # the sum over n tokens of such running sums: an error enters at most n of them
                    tol += n * part.sum(0)
                    mean += (n * part.norm(dim=0)) ** 2
                else:
                    tol[b, t0:t0 + n] = part.sum(0)
                    mean[b, t0:t0 + n] = part.norm(dim=0) ** 2
            tol = 2.0 ** -18 * (tol + m)
            # the errors of different tokens' sums are independent, so that they add like their squares
            assert ((x - r).abs() <= 2.0 ** -18 * (mean.sqrt() + m) + 1e-30).all(), name
        assert ((x - r).abs() <= tol + 1e-30).all(), (name, float(((x - r).abs() / (tol + 1e-30)).max()))


@pytest.mark.parametrize("T", [64, 1, 2, 63, 65, 200])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (128, 64), (64, 128)])
def test_lengths_and_head_dims(built_lib, T, dk, dv):
    from avelang_b200 import gdn, linear_attention as L
    q, k, v, g, s0 = make(2, T, 2, 2, dk, dv, "token", T, 2, 0.2)
    d_o, d_f = grads_in(v.shape, 2, dk, 7, True)
    got = L.linear_attention_backward(*cuda(q, k, v, g, d_o), None, s0.cuda(), d_f.cuda())
    assert gdn.read_status() == 0
    check(got, q, k, v, g, dk ** -0.5, s0, None, d_o, d_f)


@pytest.mark.parametrize("gate,rate", [("token", 4.0), ("token", 0.01), ("head", 1.0), ("head", 0.01), ("none", 1.0)])
@pytest.mark.parametrize("Hk,Hv", [(1, 1), (1, 6), (2, 4)])
@pytest.mark.parametrize("states", [True, False])
def test_gates_shared_heads_and_states(built_lib, gate, rate, Hk, Hv, states):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(1, 150, Hk, Hv, 128, 64, gate, 3, 1 if states else 0, rate)
    d_o, d_f = grads_in(v.shape, 1, 128, 8, states)
    got = L.linear_attention_backward(*cuda(q, k, v, g, d_o), 0.3, *cuda(s0, d_f))
    check(got, q, k, v, g, 0.3, s0, None, d_o, d_f)


@pytest.mark.parametrize("T,Hk,Hv,dk,dv,gate", [(2100, 1, 1, 128, 128, "token"), (1500, 1, 2, 64, 128, "head"), (1800, 2, 2, 128, 64, "none")])
def test_segments(built_lib, T, Hk, Hv, dk, dv, gate):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(1, T, Hk, Hv, dk, dv, gate, 4, 1, 0.02)
    d_o, d_f = grads_in(v.shape, 1, dk, 9, True)
    got = L.linear_attention_backward(*cuda(q, k, v, g, d_o), None, *cuda(s0, d_f))
    check(got, q, k, v, g, dk ** -0.5, s0, None, d_o, d_f)


@pytest.mark.parametrize("lens", [[64, 64], [0, 70, 0, 1, 129, 0], [900, 3, 700, 64]])
@pytest.mark.parametrize("gate", ["token", "head"])
def test_packed(built_lib, lens, gate):
    """What lies behind the last offset is NaN and has zero gradients."""
    from avelang_b200 import gdn, linear_attention as L
    T = sum(lens)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    q, k, v, g, s0 = make(1, T + 70, 1, 2, 128, 128, gate, 5, len(lens), 0.1)
    d_o, d_f = grads_in(v.shape, len(lens), 128, 10, True)
    for x in (q, k, v, d_o) + ((g,) if gate == "token" else ()):
        x[:, T:] = float("nan")
    got = list(L.linear_attention_backward(*cuda(q, k, v, g, d_o), None, s0.cuda(), d_f.cuda(), cu.cuda()))
    assert gdn.read_status() == 0
    for i in range(4 if gate == "token" else 3):
        assert (got[i][:, T:] == 0).all(), i
        got[i] = got[i][:, :T]
    check(got, q[:, :T], k[:, :T], v[:, :T], g[:, :T] if gate == "token" else g, 128 ** -0.5, s0, cu, d_o[:, :T], d_f)


def test_decays_of_zero(built_lib):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(1, 140, 1, 2, 128, 128, "token", 6, 1, 0.1)
    g[:, 30] = -1e30
    g[:, 70:72] = -float("inf")
    d_o, d_f = grads_in(v.shape, 1, 128, 11, True)
    got = L.linear_attention_backward(*cuda(q, k, v, g, d_o), None, *cuda(s0, d_f))
    want = O.gradients(q, k, v, torch.where(g < -1e6, torch.full_like(g, -1e6), g), 128 ** -0.5, s0, None, d_o, d_f)
    for x, r in zip(got, want):
        assert x.isfinite().all() and (x.cpu().double() - r).norm() <= 2.0 ** -8 * r.norm()
    assert (got[3][:, 30].abs() <= 1e-3).all() and (got[3][:, 70:72].abs() <= 1e-3).all()


def test_autograd_expanded_gradients_and_differences(built_lib):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(1, 100, 2, 4, 64, 64, "token", 7, 1, 0.2)
    leaves = [x.cuda().requires_grad_(True) for x in (q, k, v, g, s0)]
    o, final = L.LinearAttentionFunction.apply(*leaves[:4], None, leaves[4], None)
    got = torch.autograd.grad((o.float() * 0.5).sum() + final.sum(), leaves)  # gradients that are expanded scalars
    f = lambda a: (lambda r: 0.5 * r[0].sum() + r[1].sum())(O.recurrent(a[0], a[1], a[2], a[3], 64 ** -0.5, a[4]))
    gen = torch.Generator().manual_seed(12)
    at = [x.double() for x in (q, k, v, g, s0)]
    for i in range(5):
        step = torch.randn(at[i].shape, generator=gen, dtype=torch.float64)
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + 1e-4 * step, at[i] - 1e-4 * step
        slope = float((f(up) - f(down)) / 2e-4)
        mine = got[i].cpu().double() * step
        # each element within half a bf16 step: the errors of many add like their root of squares, 8 of which are allowed
        assert abs(float(mine.sum()) - slope) <= 8 * 2.0 ** -8 * float(mine.norm()) + 1e-5 * abs(slope)
    q1, v1 = q.cuda().requires_grad_(True), v.cuda()
    o, _ = L.LinearAttentionFunction.apply(q1, k.cuda(), v1, None, 0.5, None, None)
    o.float().sum().backward()
    assert q1.grad.isfinite().all()


def test_same_bits_twice_on_streams_and_captured(built_lib):
    from avelang_b200 import linear_attention as L
    ins = []
    for i in range(2):
        q, k, v, g, s0 = make(1, 1300, 1, 2, 128, 128, "token", 20 + i, 1, 0.02)
        d_o, d_f = grads_in(v.shape, 1, 128, 30 + i, True)
        ins.append(cuda(q, k, v, g, d_o) + [None] + cuda(s0, d_f))
    call = lambda x: L.linear_attention_backward(*x)
    want = [[t.clone() for t in call(x)] for x in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = []
        for s, x in zip(streams, ins):
            with torch.cuda.stream(s):
                got.append(call(x))
        torch.cuda.synchronize()
        assert all(torch.equal(p, r) for g, w in zip(got, want) for p, r in zip(g, w))
    graphs, outs = [], []
    for x in ins:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(x))
        graphs.append(graph)
    for _ in range(3):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, r) for g, w in zip(outs, want) for p, r in zip(g, w))


def test_no_tokens(built_lib):
    from avelang_b200 import linear_attention as L
    z = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")
    s0, d_f = torch.randn(2, 2, 64, 64, device="cuda"), torch.randn(2, 2, 64, 64, device="cuda")
    o, s = L.chunk_linear_attention(z(2, 0, 1, 64), z(2, 0, 1, 64), z(2, 0, 2, 64), None, None, s0, True)
    assert o.shape == (2, 0, 2, 64) and torch.equal(s, s0)
    got = L.linear_attention_backward(z(2, 0, 1, 64), z(2, 0, 1, 64), z(2, 0, 2, 64), torch.zeros(2, device="cuda"), z(2, 0, 2, 64), None, s0, d_f)
    assert (got[3] == 0).all() and torch.equal(got[4], d_f)
