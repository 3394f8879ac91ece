"""Linear attention on tensors that lie in ways which no kernel wants: off 16-byte boundaries, with odd distances in dimensions of one element, in one storage."""
import pytest
import torch

import test_linear_backward_gpu as BW
import test_linear_decode_gpu as D
import test_linear_prefill_gpu as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,T", [(1, 90), (2, 33)])
def test_gradients_off_16_bytes(built_lib, B, T):
    """The results go, with an odd number of others, into one vector: their gradients are views into its gradient."""
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = P.make(B, T, 1, 2, 128, 64, "token", 3, B, 0.1)
    leaves = [x.cuda().requires_grad_() for x in (q, k, v, g, s0)]
    o, s = L.LinearAttentionFunction.apply(*leaves[:4], None, leaves[4], None)
    n, gen = o.numel(), torch.Generator().manual_seed(4)
    w_o, w_s = torch.randn(n + 3, generator=gen).bfloat16(), torch.randn(s.numel() + 3, generator=gen)
    both = torch.cat([torch.zeros(3, dtype=torch.bfloat16, device="cuda"), o.flatten()]), torch.cat([torch.zeros(3, device="cuda"), s.flatten()])
    torch.autograd.backward(both, [w_o.cuda(), w_s.cuda()])
    BW.check([x.grad for x in leaves], q, k, v, g, 128 ** -0.5, s0, None, w_o[3:].view_as(v), w_s[3:].view_as(s0))


def test_a_gradient_of_every_alignment(built_lib):
    from avelang_b200 import linear_attention as L
    q, k, v, g, _ = P.cuda(*P.make(1, 70, 2, 4, 64, 128, "head", 5))
    d_o, d_f = P.cuda(*BW.grads_in(v.shape, 1, 64, 6, True))
    want = L.linear_attention_backward(q, k, v, g, d_o, None, None, d_f)
    for at in (1, 4, 8):
        a = torch.zeros(d_o.numel() + at, dtype=torch.bfloat16, device="cuda")[at:].view_as(d_o).copy_(d_o)
        b = torch.zeros(d_f.numel() + at, device="cuda")[at:].view_as(d_f).copy_(d_f)
        wide = torch.zeros(1, 70, 4, 128 + at, dtype=torch.bfloat16, device="cuda")[..., :128].copy_(d_o)
        for x in (a, wide):
            got = L.linear_attention_backward(q, k, v, g, x, None, None, b)
            assert all(p is r or torch.equal(p, r) for p, r in zip(got, want))


def test_one_of_a_kind_with_an_odd_distance(built_lib):
    """One batch row, one token or one head, cut out of buffers of odd width."""
    from avelang_b200 import linear_attention as L

    def cut(x, dim):  # the same values, with an odd distance in a dimension of one element
        strides = list(x.stride())
        assert x.size(dim) == 1
        strides[dim] = 1001
        return x.as_strided(x.shape, strides)

    for B, T, H, dim in ((1, 70, 2, 0), (3, 1, 2, 1), (2, 70, 1, 2)):
        q, k, v, g, s0 = P.make(B, T, H, H, 128, 128, "token", 7, B, 0.1)
        args = [cut(x.cuda(), dim) for x in (q, k, v)] + P.cuda(g, None, s0)
        out = cut(torch.zeros(v.shape, dtype=torch.bfloat16, device="cuda"), dim)
        o, s = L.chunk_linear_attention(*args, True, out=out)
        P.check(o, s, q, k, v, g, 128 ** -0.5, s0)
        o, s = L.fused_recurrent_linear_attention(*args)
        D.check(o, s, q, k, v, g, 128 ** -0.5, s0)
        d_o, d_f = BW.grads_in(v.shape, B, 128, 8, True)
        got = L.linear_attention_backward(*args[:4], cut(d_o.cuda(), dim), None, s0.cuda(), d_f.cuda())
        BW.check(got, q, k, v, g, 128 ** -0.5, s0, None, d_o, d_f)


@pytest.mark.parametrize("T", [90, 2100])
def test_results_in_the_place_of_inputs(built_lib, T):
    """Whole sequences, cut into segments or not, and the recurrent form, in the place of q, k or v."""
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = P.cuda(*P.make(1, T, 2, 2, 128, 128, "token", 9, 1, 0.05))
    want = L.chunk_linear_attention(q, k, v, g, None, s0, True)
    for i in range(3):
        x = [q.clone(), k.clone(), v.clone()]
        o, s = L.chunk_linear_attention(*x, g, None, s0, True, out=x[i])
        assert o.data_ptr() == x[i].data_ptr() and torch.equal(o, want[0]) and torch.equal(s, want[1])
    n = min(T, 90)
    x = [t[:, :n].contiguous() for t in (q, k, v)]
    want = L.fused_recurrent_linear_attention(*x, g[:, :n], None, s0)
    for i in range(3):
        y = [t.clone() for t in x]
        o, s = L.fused_recurrent_linear_attention(*y, g[:, :n], None, s0, out=y[i])
        assert o.data_ptr() == y[i].data_ptr() and torch.equal(o, want[0]) and torch.equal(s, want[1])
