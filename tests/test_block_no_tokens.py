"""The block and the layer around it on a batch without tokens: empty results of the right shape, with 8-bit projections and without."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from test_block_int8 import HIDDEN, make
from test_dispatch import Recorder


def run(int8):
    blk = make(int8=int8)
    x = torch.zeros(2, 0, HIDDEN, dtype=torch.bfloat16, device="cuda")
    for residual in (None, x):
        out, h = blk.layer(x, residual, torch.ones(HIDDEN, device="cuda"))
        assert out.shape == h.shape == x.shape and out.dtype == torch.bfloat16
    assert blk.forward(x).shape == x.shape


@pytest.mark.parametrize("int8", [False, True])
def test_calls(built_lib, int8):
    with FakeTensorMode(allow_non_fake_inputs=True), Recorder(run=False):
        run(int8)


@pytest.mark.gpu
@pytest.mark.parametrize("int8", [False, True])
def test_on_the_device(built_lib, int8):
    from avelang_b200 import gdn
    run(int8)
    assert gdn.read_status() == 0
