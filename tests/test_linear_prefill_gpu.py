"""Chunked linear attention with a decay for each head over whole sequences, against the recurrence in 64 bits."""
import pytest
import torch

from oracle import linear_oracle as O

pytestmark = pytest.mark.gpu


def make(B, T, Hk, Hv, dk, dv, gate, seed, n_states=0, rate=1.0):
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, T, h, d, generator=gen).bfloat16() for h, d in ((Hk, dk), (Hk, dk), (Hv, dv)))
    g = {"token": -torch.rand(B, T, Hv, generator=gen) * 2.0 * rate, "head": -torch.rand(Hv, generator=gen) * rate, "none": None}[gate]
    s0 = torch.randn(n_states, Hv, dk, dv, generator=gen) if n_states else None
    return q, k, v, g, s0


def cuda(*xs):
    return [x.cuda() if x is not None else None for x in xs]


def bounds(q, k, v, g, scale, s0, cu=None):
    """Reference values and how far results may be off.  The increment's operands are carried to 24 bits, its sums are 12 MMA steps a chunk, each
    of which may lose 2^-22 of the terms' absolute values; a chunk more is a multiplication and an addition; factors are within 2^-22.  The scores and the
    state reach the output as two bf16 terms (2^-17 each at most), sums of dk + 64 products behind them; the output is rounded to bf16."""
    o, s = O.recurrent(q, k, v, g, scale, s0, cu)
    om, sm = O.magnitudes(q, k, v, g, scale, s0, cu)
    chunks = max([n for _, _, n in O.spans(q, cu)] + [0]) // 64 + 1
    es = (16 + chunks) * 2.0 ** -22
    eo = 2.0 ** -16 + es + (q.shape[3] + 72) * 2.0 ** -24
    return o, s, 2.0 ** -8 * o.abs() * (1 + 1e-3) + eo * om + 1e-30, es * sm + 1e-30


def check(o, s, *args):
    o_ref, s_ref, o_tol, s_tol = bounds(*args)
    assert ((o.cpu().double() - o_ref).abs() <= o_tol).all(), float(((o.cpu().double() - o_ref).abs() / o_tol).max())
    if s is not None:
        assert ((s.cpu().double() - s_ref).abs() <= s_tol).all(), float(((s.cpu().double() - s_ref).abs() / s_tol).max())


@pytest.mark.parametrize("T", [64, 1, 2, 63, 65, 128, 200])
@pytest.mark.parametrize("dk,dv", [(128, 128), (64, 64), (128, 64), (64, 128)])
def test_lengths_and_head_dims(built_lib, T, dk, dv):
    from avelang_b200 import gdn, linear_attention as L
    q, k, v, g, s0 = make(2, T, 2, 4, dk, dv, "token", T, 2, 0.2)
    o, s = L.chunk_linear_attention(*cuda(q, k, v, g, None, s0), True)
    assert gdn.read_status() == 0
    check(o, s, q, k, v, g, dk ** -0.5, s0)
    o, s = L.chunk_linear_attention(*cuda(q, k, v, g), 0.7)
    assert s is None
    check(o, None, q, k, v, g, 0.7, None)


@pytest.mark.parametrize("gate,rate", [("token", 1.0), ("token", 0.01), ("head", 1.0), ("head", 0.01), ("none", 1.0)])
@pytest.mark.parametrize("Hk,Hv", [(1, 1), (1, 8), (4, 4)])
def test_gates_and_shared_heads(built_lib, gate, rate, Hk, Hv):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(1, 150, Hk, Hv, 128, 128, gate, 3, 1, rate)
    o, s = L.chunk_linear_attention(*cuda(q, k, v, g, None, s0), True)
    check(o, s, q, k, v, g, 128 ** -0.5, s0)


@pytest.mark.parametrize("T,Hk,Hv,dk,dv,n", [(2100, 1, 1, 128, 128, 1), (3001, 2, 2, 64, 128, 0), (1500, 1, 2, 128, 64, 1)])
def test_segments(built_lib, T, Hk, Hv, dk, dv, n):
    """Few heads and a long sequence: segments side by side."""
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(1, T, Hk, Hv, dk, dv, "token", 4, n, 0.01)
    o, s = L.chunk_linear_attention(*cuda(q, k, v, g, None, s0), True)
    check(o, s, q, k, v, g, dk ** -0.5, s0)


@pytest.mark.parametrize("lens", [[1], [64, 64], [0, 70, 0, 1, 129, 0], [5, 300, 2], [1500, 3, 700, 64]])
def test_packed(built_lib, lens):
    """Rows in front of, between and behind sequences reach nobody: what lies behind the last offset is NaN, and stays as it was in the result."""
    from avelang_b200 import gdn, linear_attention as L
    T = sum(lens)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    q, k, v, g, s0 = make(1, T + 70, 2, 4, 128, 128, "token", 5, len(lens), 0.1)
    for x in (q, k, v, g):
        x[:, T:] = float("nan")
    out = torch.full((1, T + 70, 4, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    o, s = L.chunk_linear_attention(*cuda(q, k, v, g, None, s0), True, cu.cuda(), out=out)
    assert (out[:, T:] == 3.0).all() and gdn.read_status() == 0
    check(o[:, :T], s, q[:, :T], k[:, :T], v[:, :T], g[:, :T], 128 ** -0.5, s0, cu)


def test_a_sequence_with_nan_or_infinity_leaves_its_neighbours_alone(built_lib):
    from avelang_b200 import linear_attention as L
    cu = torch.tensor([0, 70, 150, 200], dtype=torch.int32)
    q, k, v, g, s0 = make(1, 200, 1, 2, 128, 64, "token", 6, 3, 0.1)
    for x in (q, k, v):
        x[:, 70:150] = float("nan")
    v[:, 140:150] = float("inf")
    o, s = L.chunk_linear_attention(*cuda(q, k, v, g, None, s0), True, cu.cuda())
    for n, (a, e) in ((0, (0, 70)), (2, (150, 200))):
        check(o[:, a:e], s[n:n + 1], q[:, a:e], k[:, a:e], v[:, a:e], g[:, a:e], 128 ** -0.5, s0[n:n + 1])


def test_pool_slots(built_lib):
    from avelang_b200 import _lib, gdn, linear_attention as L
    cu = torch.tensor([0, 70, 71, 90, 300], dtype=torch.int32)
    q, k, v, g, pool = make(1, 300, 2, 4, 128, 128, "token", 7, 9, 0.1)
    idx = torch.tensor([5, -1, 9, 0], dtype=torch.int32)
    pd = pool.cuda()
    args = cuda(q, k, v, g)
    o2, s2 = L.chunk_linear_attention(*args, None, pd, True, cu.cuda(), state_indices=idx.cuda(), inplace_state=False)
    assert gdn.read_status() == _lib.DEV_BAD_SLOT and torch.equal(pd.cpu(), pool)
    o, s = L.chunk_linear_attention(*args, None, pd, True, cu.cuda(), state_indices=idx.cuda())
    assert gdn.read_status() == _lib.DEV_BAD_SLOT and s.data_ptr() == pd.data_ptr()
    assert torch.equal(o, o2) and torch.equal(s, s2)
    assert (o[:, 70:90] == 0).all()
    assert torch.equal(pd.cpu()[[1, 2, 3, 4, 6, 7, 8]], pool[[1, 2, 3, 4, 6, 7, 8]])
    for n, sl in ((0, 5), (3, 0)):
        a, e = int(cu[n]), int(cu[n + 1])
        check(o[:, a:e], pd[sl:sl + 1], q[:, a:e], k[:, a:e], v[:, a:e], g[:, a:e], 128 ** -0.5, pool[sl:sl + 1])


@pytest.mark.parametrize("offsets", [[0, 80, 40, 100], [0, 50, 101], [-1, 50, 100]])
def test_bad_offsets_are_flagged_and_nothing_is_written(built_lib, offsets):
    from avelang_b200 import _lib, gdn, linear_attention as L
    cu = torch.tensor(offsets, dtype=torch.int32).cuda()
    q, k, v, g, s0 = make(1, 100, 1, 2, 64, 64, "token", 8, len(offsets) - 1)
    out = torch.full((1, 100, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    pool, idx = s0.cuda(), torch.arange(len(offsets) - 1, dtype=torch.int32).cuda()
    L.chunk_linear_attention(*cuda(q, k, v, g), None, pool, True, cu, state_indices=idx, out=out)
    assert gdn.read_status() == _lib.DEV_BAD_SEQLEN
    assert (out == 3.0).all() and torch.equal(pool.cpu(), s0)


def test_strides_expanded_inputs_and_decays_of_zero(built_lib):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(2, 140, 8, 8, 128, 128, "token", 9, 2, 0.1)
    g[:, 30] = -float("inf")
    g[:, 70:72] = -1e30
    sl = lambda x: x.cuda()[:, :, 2:6]
    packed = torch.cat([x.cuda() for x in (q, k, v)], dim=2)
    qs, ks, vs = packed[:, :, 2:6], packed[:, :, 10:14], packed[:, :, 18:22]
    out = torch.zeros(2, 140, 16, 128, dtype=torch.bfloat16, device="cuda")
    o, s = L.chunk_linear_attention(qs, ks, vs, sl(g), None, s0[:, 2:6].contiguous().cuda(), True, out=out[:, :, 3:7])
    check(o, s, q[:, :, 2:6], k[:, :, 2:6], v[:, :, 2:6], g[:, :, 2:6], 128 ** -0.5, s0[:, 2:6])
    assert (out[:, :, :3] == 0).all() and (out[:, :, 7:] == 0).all()
    one = q[:, :, :1]
    o, _ = L.chunk_linear_attention(one.cuda().expand(2, 140, 4, 128), sl(k), sl(v), sl(g))
    check(o, None, one.expand(2, 140, 4, 128), k[:, :, 2:6], v[:, :, 2:6], g[:, :, 2:6], 128 ** -0.5, None)
    heads_first = torch.zeros(2, 4, 140, 128, dtype=torch.bfloat16, device="cuda").transpose(1, 2)
    o, _ = L.chunk_linear_attention(qs, ks, vs, sl(g), out=heads_first)
    check(o, None, q[:, :, 2:6], k[:, :, 2:6], v[:, :, 2:6], g[:, :, 2:6], 128 ** -0.5, None)


def test_agrees_with_the_recurrent_form_and_continues_from_its_state(built_lib):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = make(1, 260, 2, 4, 128, 64, "head", 10, 1, 0.3)
    a = cuda(q, k, v, g, s0)
    _, s1 = L.chunk_linear_attention(a[0][:, :130], a[1][:, :130], a[2][:, :130], a[3], None, a[4], True)
    o2, s2 = L.fused_recurrent_linear_attention(a[0][:, 130:135], a[1][:, 130:135], a[2][:, 130:135], a[3], None, s1)
    o3, s3 = L.chunk_linear_attention(a[0][:, 135:], a[1][:, 135:], a[2][:, 135:], a[3], None, s2, True)
    o_ref, s_ref, o_tol, s_tol = bounds(q, k, v, g, 128 ** -0.5, s0)
    assert ((s3.cpu().double() - s_ref).abs() <= 3 * s_tol).all()  # three roundings of the state's path
    assert ((torch.cat([o2, o3], 1).cpu().double() - o_ref[:, 130:]).abs() <= 3 * o_tol[:, 130:]).all()


def test_streams_and_captured_calls(built_lib):
    """Two streams at once, and two captured graphs replayed beside one another, with segments (scratch) in both."""
    from avelang_b200 import linear_attention as L
    ins = [cuda(*make(1, 2300, 1, 2, 128, 128, "token", 20 + i, 1, 0.02)) for i in range(2)]
    call = lambda x: L.chunk_linear_attention(x[0], x[1], x[2], x[3], None, x[4], True)
    want = [[t.clone() for t in call(x)] for x in ins]
    streams = [torch.cuda.Stream() for _ in ins]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
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
    for _ in range(4):
        for s, graph in zip(streams, graphs):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, r) for g, w in zip(outs, want) for p, r in zip(g, w))


@pytest.mark.parametrize("n", [2, 256, 257])
def test_many_sequences_of_unequal_length(built_lib, n):
    """More work than SMs: up to 256 sequences run in the order of their lengths, ties in the batch's."""
    from avelang_b200 import gdn, linear_attention as L
    lens = torch.randint(0, 40, (n,), generator=torch.Generator().manual_seed(n)).tolist()
    lens[n // 2] = 200
    cu = torch.tensor([sum(lens[:i]) for i in range(n + 1)], dtype=torch.int32)
    q, k, v, g, s0 = make(1, int(cu[-1]), 1, 2, 64, 64, "token", 13, n, 0.1)
    o, s = L.chunk_linear_attention(*cuda(q, k, v, g, None, s0), True, cu.cuda())
    assert gdn.read_status() == 0
    check(o, s, q, k, v, g, 64 ** -0.5, s0, cu)


def test_pool_in_place_where_some_sequences_are_cut_into_segments(built_lib):
    """A sequence of one segment beside longer ones: its state is read before the final one takes its place."""
    from avelang_b200 import gdn, linear_attention as L
    lens = [1500, 3, 0, 700, 64]
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32)
    q, k, v, g, pool = make(1, sum(lens), 1, 2, 128, 128, "token", 14, 7, 0.05)
    idx = torch.tensor([4, 0, 6, 2, 5], dtype=torch.int32)
    args, pd = cuda(q, k, v, g), pool.cuda()
    apart = L.chunk_linear_attention(*args, None, pd, True, cu.cuda(), state_indices=idx.cuda(), inplace_state=False)
    assert torch.equal(pd.cpu(), pool)
    o, s = L.chunk_linear_attention(*args, None, pd, True, cu.cuda(), state_indices=idx.cuda())
    assert gdn.read_status() == 0 and s.data_ptr() == pd.data_ptr()
    assert torch.equal(o, apart[0]) and torch.equal(s, apart[1])
    check(o, s[idx.long().cuda()], q, k, v, g, 128 ** -0.5, pool[idx.long()], cu)
    assert torch.equal(s.cpu()[[1, 3]], pool[[1, 3]])
