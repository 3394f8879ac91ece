"""Linear attention with a negative scale and with a scale of zero.  A negative scale is a positive one with -q in q's place, so that results and bounds are those of that."""
import pytest
import torch

import test_linear_backward_gpu as BW
import test_linear_decode_gpu as D
import test_linear_prefill_gpu as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [-0.3, 0.0, -1.0])
@pytest.mark.parametrize("T,Hk,Hv,dk,dv", [(150, 2, 4, 128, 128), (1, 1, 1, 64, 64), (1500, 1, 2, 64, 128), (2100, 1, 1, 128, 64)])
def test_forward(built_lib, T, Hk, Hv, dk, dv, scale):
    """The long ones are cut into segments."""
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = P.make(1, T, Hk, Hv, dk, dv, "token", 1, 1, 0.05)
    for module, call in ((P, L.chunk_linear_attention), (D, L.fused_recurrent_linear_attention)):
        for states in (s0, None):
            o, s = call(*P.cuda(q, k, v, g), scale, None if states is None else states.cuda(), states is not None)
            module.check(o, s, q, k, v, g, scale, states)
            assert scale != 0.0 or (o == 0).all()


@pytest.mark.parametrize("scale", [-0.3, 0.0])
@pytest.mark.parametrize("gate", ["token", "head", "none"])
@pytest.mark.parametrize("T,Hk,Hv,dk,dv", [(150, 1, 2, 128, 128), (65, 2, 2, 64, 64), (1500, 1, 2, 64, 128)])
def test_gradients(built_lib, T, Hk, Hv, dk, dv, gate, scale):
    from avelang_b200 import linear_attention as L
    q, k, v, g, s0 = P.make(1, T, Hk, Hv, dk, dv, gate, 2, 1, 0.05)
    d_o, d_f = BW.grads_in(v.shape, 1, dk, 3, True)
    for states, final in ((s0, d_f), (None, None)):
        got = list(L.linear_attention_backward(*P.cuda(q, k, v, g, d_o), scale, *P.cuda(states, final)))
        if scale < 0:
            got[0] = -got[0]
        BW.check(got, -q if scale < 0 else q, k, v, g, abs(scale), states, None, d_o, final)
