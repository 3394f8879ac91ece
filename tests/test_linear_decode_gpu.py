"""Linear attention with a decay for each head, token by token, against the recurrence in 64 bits."""
import pytest
import torch

from oracle import linear_oracle as O

pytestmark = pytest.mark.gpu


def make(B, T, Hk, Hv, dk, dv, gate, seed, n_states=0):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, T, h, d, generator=gen).bfloat16() for h, d in ((Hk, dk), (Hk, dk), (Hv, dv)))
    g = {"token": -torch.rand(B, T, Hv, generator=gen) * 2.0, "head": -torch.rand(Hv, generator=gen), "none": None}[gate]
    s0 = torch.randn(n_states, Hv, dk, dv, generator=gen) if n_states else None
    return q, k, v, g, s0


def cuda(*xs):
    return [x.cuda() if x is not None else None for x in xs]


def check(o, s, q, k, v, g, scale, s0, cu=None):
    """A state takes a product, a multiplication by the decay and an addition a token, each within half a step (2^-24), and the decay itself within
    two steps of 2^-23: 8 T 2^-24 of the terms' absolute values.  The output adds dk products and a rounding to bf16 (2^-8)."""
    T = max(n for _, _, n in O.spans(q, cu)) if cu is None or cu.numel() > 1 else 0
    o_ref, s_ref = O.recurrent(q, k, v, g, scale, s0, cu)
    o_mag, s_mag = O.magnitudes(q, k, v, g, scale, s0, cu)
    eps = (8 * T + 8) * 2.0 ** -24
    if s is not None:
        assert ((s.cpu().double() - s_ref).abs() <= eps * s_mag + 1e-30).all()
    dk = q.shape[3]
    assert ((o.cpu().double() - o_ref).abs() <= (2.0 ** -8) * o_ref.abs() * (1 + 1e-3) + (eps + (dk + 8) * 2.0 ** -24) * o_mag + 1e-30).all()


@pytest.mark.parametrize("B,T,Hk,Hv,dk,dv", [(1, 1, 1, 1, 64, 64), (3, 1, 2, 4, 128, 128), (2, 1, 4, 4, 128, 64), (2, 1, 1, 8, 64, 128), (1, 7, 2, 4, 128, 128),
                                             (2, 33, 1, 2, 64, 64), (40, 1, 4, 8, 128, 128)])
@pytest.mark.parametrize("gate", ["token", "head", "none"])
def test_recurrent(built_lib, B, T, Hk, Hv, dk, dv, gate):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(B, T, Hk, Hv, dk, dv, gate, 1, B)
    qd, kd, vd, gd, sd = cuda(q, k, v, g, s0)
    o, s = L.fused_recurrent_linear_attention(qd, kd, vd, gd, initial_state=sd)
    check(o, s, q, k, v, g, dk ** -0.5, s0)
    o, s = L.fused_recurrent_linear_attention(qd, kd, vd, gd, 0.3)
    check(o, s, q, k, v, g, 0.3, None)


@pytest.mark.parametrize("n,slots,Hk,Hv,dk,dv", [(1, 2, 2, 4, 128, 128), (5, 9, 2, 4, 128, 128), (80, 100, 2, 4, 128, 128), (160, 200, 4, 8, 64, 128), (70, 80, 4, 8, 128, 64),
                                                 (300, 300, 1, 8, 64, 64)])
def test_pool_step(built_lib, n, slots, Hk, Hv, dk, dv):
    """Slots in any order, skipped rows, slots that nobody names left as they were, twice in a row."""
    from avelang_b200 import gdn, linear_attention as L
    q, k, v, g, pool = make(n, 1, Hk, Hv, dk, dv, "token", 2, slots)
    idx = torch.randperm(slots, generator=torch.Generator().manual_seed(3))[:n].to(torch.int32)
    if n > 3:
        idx[1], idx[3] = -1, -7
    live = idx >= 0
    at = idx[live].long()
    qd, kd, vd, gd, pd, idxd = cuda(q, k, v, g, pool, idx)
    ref = pool.clone()
    for _ in range(2):
        before = ref[at].clone()
        o, s = L.fused_recurrent_linear_attention(qd, kd, vd, gd, initial_state=pd, state_indices=idxd)
        assert s.data_ptr() == pd.data_ptr()
        check(o[live.cuda()], pd[at.cuda()], q[live], k[live], v[live], g[live], dk ** -0.5, before)
        assert (o[~live.cuda()] == 0).all()
        ref = pd.cpu()
    others = torch.ones(slots, dtype=torch.bool)
    others[at] = False
    assert torch.equal(pd.cpu()[others], pool[others])
    kept = pd.clone()
    o2, s2 = L.fused_recurrent_linear_attention(qd, kd, vd, gd, initial_state=pd, state_indices=idxd, inplace_state=False)
    assert torch.equal(pd, kept) and s2.data_ptr() != pd.data_ptr()
    check(o2[live.cuda()], s2[at.cuda()], q[live], k[live], v[live], g[live], dk ** -0.5, ref[at])
    assert gdn.read_status() == 0


def test_slot_beyond_the_pool_is_skipped_and_flagged(built_lib):
    from avelang_b200 import _lib, gdn, linear_attention as L
    q, k, v, g, pool = make(3, 1, 2, 4, 128, 128, "token", 4, 4)
    pd = pool.cuda()
    idx = torch.tensor([2, 4, 0], dtype=torch.int32).cuda()
    o, _ = L.fused_recurrent_linear_attention(*cuda(q, k, v, g), initial_state=pd, state_indices=idx)
    assert gdn.read_status() == _lib.DEV_BAD_SLOT
    assert (o[1] == 0).all() and torch.equal(pd[[1, 3]].cpu(), pool[[1, 3]])
    check(o[[0, 2]], pd[[2, 0]], q[[0, 2]], k[[0, 2]], v[[0, 2]], g[[0, 2]], 128 ** -0.5, pool[[2, 0]])


def test_packed_sequences_with_empty_ones(built_lib):
    from avelang_b200 import linear_attention as L
    cu = torch.tensor([0, 5, 5, 6, 17], dtype=torch.int32)
    q, k, v, g, s0 = make(1, 20, 2, 4, 128, 64, "head", 5, 4)
    out = torch.full((1, 20, 4, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    o, s = L.fused_recurrent_linear_attention(*cuda(q, k, v, g), None, s0.cuda(), True, cu.cuda(), out=out)
    assert o is out or o.data_ptr() == out.data_ptr()
    assert (out[:, 17:] == 7.0).all()
    check(o[:, :17], s, q[:, :17], k[:, :17], v[:, :17], g, 128 ** -0.5, s0, cu)
    assert torch.equal(s[1].cpu(), s0[1])


def test_strided_heads_and_decays_at_the_ends_of_the_range(built_lib):
    """Head-sharded slices of packed tensors; a decay of zero empties the state whatever it holds short of NaN."""
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(2, 4, 8, 8, 128, 128, "token", 6, 2)
    g[:, 1] = -float("inf")
    g[:, 2] = -1e30
    g[:, 3] = 0.0
    s0 = s0[:, 2:6].contiguous()
    sl = lambda x: x.cuda()[:, :, 2:6]
    gs = g.cuda()[:, :, 2:6]
    o, s = L.fused_recurrent_linear_attention(sl(q), sl(k), sl(v), gs, initial_state=s0.cuda())
    check(o, s, q[:, :, 2:6], k[:, :, 2:6], v[:, :, 2:6], g[:, :, 2:6], 128 ** -0.5, s0)


def test_another_stream_and_a_captured_step(built_lib):
    from avelang_b200 import linear_attention as L
    q, k, v, g, pool = make(6, 1, 2, 4, 128, 128, "token", 7, 6)
    idx = torch.arange(6, dtype=torch.int32).cuda()
    qd, kd, vd, gd = cuda(q, k, v, g)
    p0, p1 = pool.cuda(), pool.cuda()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [L.fused_recurrent_linear_attention(qd, kd, vd, gd, initial_state=p0, state_indices=idx)[0].clone() for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    out = torch.empty_like(vd)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.fused_recurrent_linear_attention(qd, kd, vd, gd, initial_state=p1, state_indices=idx, out=out)
    for w in want:
        graph.replay()
        assert torch.equal(out, w)
    assert torch.equal(p0, p1)
