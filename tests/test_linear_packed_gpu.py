"""Packed batches of linear attention whose sequences begin behind the first row or end in front of the last."""
import pytest
import torch

import test_linear_backward_gpu as BW
import test_linear_decode_gpu as D
import test_linear_prefill_gpu as P

pytestmark = pytest.mark.gpu
CUS = [[5, 70, 70, 135], [64, 128], [3, 3], [70, 1570, 1573, 2273], [129, 130]]
BEHIND = 67


def make(offsets, seed, gate="token", dims=(2, 4, 128, 128), outside=float("nan")):
    """Inputs whose rows outside all sequences hold `outside`, and those of the sequences alone with their offsets."""
    Hk, Hv, dk, dv = dims
    cu = torch.tensor(offsets, dtype=torch.int32)
    a, e = offsets[0], offsets[-1]
    q, k, v, g, s0 = P.make(1, e + BEHIND, Hk, Hv, dk, dv, gate, seed, len(offsets) - 1, 0.05)
    for x in (q, k, v) + ((g,) if gate == "token" else ()):
        x[:, :a] = outside
        x[:, e:] = outside
    inside = [x[:, a:e] for x in (q, k, v)] + [g[:, a:e] if gate == "token" else g, s0]
    return (q, k, v, g, s0), inside, cu, cu - a


@pytest.mark.parametrize("dims", [(2, 4, 128, 128), (1, 2, 64, 128)])
@pytest.mark.parametrize("offsets", CUS)
def test_rows_of_no_sequence_are_zero_in_a_differentiable_result(built_lib, offsets, dims):
    """The storage of the result held NaN before."""
    from avelang_b200 import gdn, linear_attention as L
    all_, inside, cu, own = make(offsets, 1, "token", dims)
    a, e = offsets[0], offsets[-1]
    for _ in range(3):
        junk = [torch.full_like(all_[2], float("nan"), device="cuda") for _ in range(4)]
        del junk
        leaves = [x.cuda().requires_grad_() for x in all_]
        o, s = L.LinearAttentionFunction.apply(*leaves[:4], None, leaves[4], cu.cuda())
        assert gdn.read_status() == 0
        assert (o[:, :a] == 0).all() and (o[:, e:] == 0).all()
    P.check(o[:, a:e].detach(), s.detach(), *inside[:4], dims[2] ** -0.5, inside[4], own)
    # the next layer multiplies every row: its weight's gradient is that of the sequences' rows
    w = torch.randn(8, dims[1] * dims[3], device="cuda", requires_grad=True)
    (o.flatten(2).float() @ w.t()).sum().backward()
    assert w.grad.isfinite().all() and all(x.grad[:, :a].eq(0).all() and x.grad[:, e:].eq(0).all() for x in leaves[:4])


def test_a_batch_without_sequences_or_with_bad_offsets_is_zero(built_lib):
    from avelang_b200 import _lib, gdn, linear_attention as L
    q, k, v, g, _ = P.cuda(*P.make(1, 90, 1, 2, 64, 64, "token", 2))
    for offsets, status in (([0], 0), ([0, 50, 40, 90], _lib.DEV_BAD_SEQLEN), ([0, 91], _lib.DEV_BAD_SEQLEN)):
        junk = [torch.full_like(v, float("nan")) for _ in range(4)]
        del junk
        o, _ = L.LinearAttentionFunction.apply(q, k, v, g, None, None, torch.tensor(offsets, dtype=torch.int32, device="cuda"))
        assert gdn.read_status() == status and (o == 0).all()


@pytest.mark.parametrize("form", ["whole", "recurrent"])
@pytest.mark.parametrize("gate", ["token", "head"])
@pytest.mark.parametrize("offsets", CUS)
def test_rows_outside_the_sequences_reach_nobody_and_stay(built_lib, offsets, gate, form):
    from avelang_b200 import gdn, linear_attention as L
    all_, inside, cu, own = make(offsets, 3, gate)
    a, e = offsets[0], offsets[-1]
    out = torch.full((1, e + BEHIND, 4, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    call = L.chunk_linear_attention if form == "whole" else L.fused_recurrent_linear_attention
    o, s = call(*P.cuda(*all_[:4], None, all_[4]), True, cu.cuda(), out=out)
    assert gdn.read_status() == 0 and o.data_ptr() == out.data_ptr()
    assert (out[:, :a] == 3.0).all() and (out[:, e:] == 3.0).all()
    (P if form == "whole" else D).check(o[:, a:e], s, *inside[:4], 128 ** -0.5, inside[4], own)


@pytest.mark.parametrize("gate", ["token", "head", "none"])
@pytest.mark.parametrize("offsets", CUS)
def test_gradients_of_rows_outside_the_sequences_are_zero(built_lib, offsets, gate):
    from avelang_b200 import gdn, linear_attention as L
    all_, inside, cu, own = make(offsets, 4, gate if gate != "none" else "head", (1, 2, 64, 128))
    if gate == "none":
        all_, inside = all_[:3] + (None, all_[4]), inside[:3] + [None, inside[4]]
    a, e = offsets[0], offsets[-1]
    d_o, d_f = BW.grads_in(all_[2].shape, len(offsets) - 1, 64, 5, True)
    d_o[:, :a] = d_o[:, e:] = float("nan")
    got = list(L.linear_attention_backward(*P.cuda(*all_[:4], d_o, None, all_[4], d_f, cu)))
    assert gdn.read_status() == 0
    for i in range(4 if gate == "token" else 3):
        assert (got[i][:, :a] == 0).all() and (got[i][:, e:] == 0).all()
        got[i] = got[i][:, a:e]
    if a == e:  # (autograd has no gradient for inputs that no sequence holds)
        assert all(x is None or x.numel() == 0 or (x == 0).all() for x in got[:4]) and torch.equal(got[4].cpu(), d_f)
    else:
        BW.check(got, *inside[:4], 64 ** -0.5, inside[4], own, d_o[:, a:e], d_f)


def test_slots_of_sequences_that_begin_behind_the_first_row(built_lib):
    from avelang_b200 import gdn, linear_attention as L
    offsets = [70, 1570, 1573, 1573, 2273]
    all_, inside, cu, own = make(offsets, 6)
    pool, idx = torch.randn(6, 4, 128, 128, generator=torch.Generator().manual_seed(7)), torch.tensor([4, 0, 3, 2], dtype=torch.int32)
    for form in ("whole", "recurrent"):
        pd = pool.cuda()
        call = L.chunk_linear_attention if form == "whole" else L.fused_recurrent_linear_attention
        o, s = call(*P.cuda(*all_[:4]), None, pd, True, cu.cuda(), state_indices=idx.cuda())
        assert gdn.read_status() == 0 and s.data_ptr() == pd.data_ptr()
        (P if form == "whole" else D).check(o[:, 70:2273], pd[idx.long().cuda()], *inside[:4], 128 ** -0.5, pool[idx.long()], own)
        assert torch.equal(pd.cpu()[[1, 5]], pool[[1, 5]])


def test_how_far_a_nan_reaches(built_lib):
    """Token 70 of a sequence that begins at row 5.  In q it stays in its token; in k it reaches what comes behind it; in v also those in front of it among its sixteen in the whole-sequence form,
    whose products of a masked score, zero, with it are no zeros."""
    from avelang_b200 import linear_attention as L
    cu, own = torch.tensor([5, 155], dtype=torch.int32), torch.tensor([0, 150], dtype=torch.int32)
    for value in (float("nan"), float("inf")):
        for form, call in ((P, L.chunk_linear_attention), (D, L.fused_recurrent_linear_attention)):
            for name in "qkv":
                x = dict(zip("qkvg", P.make(1, 155, 1, 2, 64, 64, "token", 8, 0, 0.1)))
                clean = {n: t[:, 5:].clone() for n, t in x.items()}
                x[name][:, 75] = value
                o, _ = call(*P.cuda(*x.values()), cu_seqlens=cu.cuda())
                ok = torch.ones(150, dtype=torch.bool)
                ok[70:71 if name == "q" else 150] = False
                assert not o[:, 5:][:, ~ok].isfinite().all(-1).any()
                if name == "v" and form is P:
                    ok[64:70] = False
                o = torch.where(ok[None, :, None, None], o[:, 5:].cpu(), torch.zeros((), dtype=torch.bfloat16))
                o_ref, _, o_tol, _ = P.bounds(*clean.values(), 64 ** -0.5, None, own)
                assert ((o.double() - o_ref).abs() <= o_tol)[:, ok].all()
