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


@pytest.mark.parametrize("name", ["q", "k", "v", "o"])
def test_distances_in_dimensions_of_one_element_may_be_anything(built_lib, name):
    """A batch of one cut out of a wider buffer, or a single token, or a single head.  (No call gets as far as a launch: scratch is missing.)"""
    import ctypes

    from avelang_b200 import _lib
    lib = _lib.load()

    def rc(dim, one):
        a, b = _lib.LinearArgs(), _lib.LinearBwdArgs()
        for args in (a, b):
            args.struct_size = ctypes.sizeof(args)
            args.B, args.T, args.Hk, args.Hv, args.dk, args.dv = 2, 8192, 2, 2, 64, 64
            if one:
                for field in {"b": ("B",), "t": ("T",), "h": ("Hk", "Hv")}[dim]:
                    setattr(args, field, 1)
            args.n_seqs, args.g = args.B, 0x1000
            for t in ("q", "k", "v", "o", "d_o", "d_q", "d_k", "d_v", "d_g"):
                if hasattr(args, t):
                    setattr(args, t, 0x1000)
                for d in "bth":
                    if hasattr(args, f"{t.replace('d_', 'd')}_stride_{d}"):
                        setattr(args, f"{t.replace('d_', 'd')}_stride_{d}", 1001 if d == dim and t.replace("d_", "") == name else 512)
        a.num_slots = a.n_seqs
        return lib.ave_linear_chunk_prefill(ctypes.byref(a), None) if dim != "t" or not one else None, lib.ave_linear_backward(ctypes.byref(b), None)

    for dim in "bth":
        assert rc(dim, False) == (_lib.MISALIGNED, _lib.MISALIGNED)
        forward, backward = rc(dim, True)
        assert backward == _lib.INVALID_ARGUMENT and forward in (None, _lib.INVALID_ARGUMENT)


@pytest.mark.parametrize("entry", ["chunk_linear_attention", "fused_recurrent_linear_attention"])
def test_results_that_lie_badly(built_lib, entry):
    """A result whose rows share memory is refused; where one takes the place of q or k, which the recurrent form's CTAs read while others write, that form reads a copy."""
    from avelang_b200 import linear_attention as L
    f = getattr(L, entry)
    with FakeTensorMode(), Calls() as mode:
        q, k, v = bf(2, 9, 4, 128), bf(2, 9, 4, 128), bf(2, 9, 4, 128)
        for out in (bf(1, 9, 4, 128).expand(2, 9, 4, 128), bf(2, 1, 4, 128).expand(2, 9, 4, 128), bf(2, 9, 1, 128).expand(2, 9, 4, 128)):
            with pytest.raises(ValueError, match="rows of out must not share memory"):
                f(q, k, v, out=out)
        assert not mode.made
        apart = lambda a: tuple(a[n].untyped_storage()._cdata != a["out"].untyped_storage()._cdata for n in "qk")
        for out, copied in ((q, (True, False)), (k, (False, True)), (q.view(2, 9, 4, 128), (True, False))):
            f(q, k, v, out=out)
            assert mode.made[-1][1]["out"] is out
            assert apart(mode.made[-1][1]) == ((True, True) if entry != "chunk_linear_attention" else tuple(not c for c in copied))
        wide = bf(2, 9, 16, 128)
        f(wide[:, :, :4], wide[:, :, 4:8], wide[:, :, 8:12], out=wide[:, :, 12:])
        f(q, k, v, out=v)
        assert mode.made[-1][1]["q"] is q and mode.made[-1][1]["k"] is k
        f(q[:1, :1, :1], k[:1, :1, :1], v[:1, :1, :1], out=bf(1, 1, 1, 128).expand(1, 1, 1, 128))
    assert len(mode.made) == 6
