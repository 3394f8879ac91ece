"""What the public calls of linear attention hand to their operators, and calls that they refuse (no GPU needed)."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.utils._python_dispatch import TorchDispatchMode

from test_linear_norm_refusals import bf, f32, i32


class Calls(TorchDispatchMode):
    """The arguments of the library's operators, by name; none is run."""

    def __init__(self):
        super().__init__()
        self.made = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if func.namespace != "avelang_gdn":
            return func(*args, **(kwargs or {}))
        names = [a.name for a in func._schema.arguments]
        self.made.append((func._schema.name.split("::")[1], {**dict(zip(names, args)), **(kwargs or {})}))


def test_only_the_differentiable_call_clears_rows_of_no_sequence(built_lib):
    from avelang_b200 import linear_attention as L
    with FakeTensorMode(), Calls() as mode:
        x = bf(1, 9, 2, 64), bf(1, 9, 2, 64), bf(1, 9, 4, 64)
        L.chunk_linear_attention(*x, cu_seqlens=i32(3))
        L.LinearAttentionFunction.apply(*x, None, None, None, i32(3))
    assert [(n, a.get("zero_outside", False)) for n, a in mode.made] == [("linear_prefill", False), ("linear_prefill", True)]
