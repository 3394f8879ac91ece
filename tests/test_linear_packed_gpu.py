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
