"""The block with 8-bit projections and behind its norm: which operators it calls and what it refuses (no GPU needed), and on the GPU its results against the same
calls one by one, against its head shards and against the block in bf16."""
import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from test_block_gpu import _params
from test_dispatch import Recorder

HIDDEN, HK, HV, D = 256, 2, 4, 128


def weights(seed=4):
    p = _params(HIDDEN, HK, HV, D, seed=seed)
    w_out = 0.05 * torch.randn(HIDDEN, HV * D, generator=torch.Generator().manual_seed(seed + 1))
    return p, w_out


def make(cls="GdnBlockTP", int8=True, seed=4, **kw):
    from avelang_b200 import block
    p, w_out = weights(seed)
    more = (w_out,) if cls == "GdnBlockTP" else ()
    return getattr(block, cls)(*p, *more, Hk=HK, Hv=HV, dk=D, dv=D, int8=int8, **kw)


def test_calls_and_refusals(built_lib):
    with FakeTensorMode(allow_non_fake_inputs=True), Recorder(run=False) as mode:
        blk = make()
        assert mode.seen == ["quantize_rows_int8"] * 2
        assert blk.w.dtype == blk.w_out.dtype == torch.int8 and blk.w_scale.dtype == torch.float32
        x = torch.zeros(1, 9, HIDDEN, dtype=torch.bfloat16, device="cuda")
        w = torch.ones(HIDDEN, device="cuda")
        mode.seen.clear()
        out, h = blk.layer(x, x, w)
        assert out.shape == h.shape == x.shape
        assert mode.seen == ["rms_norm", "gemm_int8_nt", "conv1d_silu", "gate_beta", "chunk_prefill", "quantize_rows_int8", "gemm_int8_nt"]
        mode.seen.clear()
        blk.forward(x)
        assert mode.seen[:2] == ["quantize_rows_int8", "gemm_int8_nt"]
        plain = make(int8=False)
        mode.seen.clear()
        out, h = plain.layer(x, None, w)
        assert h is x and mode.seen[:2] == ["rms_norm", "gemm_bf16_nt"] and mode.seen[-1] == "gemm_bf16_nt"
        with pytest.raises(ValueError, match="int8=True"):
            plain.forward((torch.zeros(1, 9, HIDDEN, dtype=torch.int8, device="cuda"), torch.zeros(1, 9, device="cuda")))
        with pytest.raises(ValueError, match="fused_reduce"):
            make(rank=1, world=2).project(torch.zeros(9, HV * D // 2, dtype=torch.bfloat16, device="cuda"), fused_reduce=True)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [1, 70, 300])
def test_layer_is_its_calls(built_lib, T):
    """The layer's result bit for bit from its entry points, and near the layer in bf16: an 8-bit operand is off by 1 / sqrt(12) of a step of 1 / 127 of a row's largest value,
    about four deviations, so 0.009 of its size; two operands 0.013 a product, which the convolution, the gates and the second product pass on, together well below six times that."""
    from avelang_b200 import gdn, gemm, norm
    blk, plain = make(), make(int8=False)
    gen = torch.Generator().manual_seed(T)
    x, res = (torch.randn(2, T, HIDDEN, generator=gen).bfloat16().cuda() for _ in range(2))
    w = (1.0 + 0.1 * torch.randn(HIDDEN, generator=gen)).cuda()
    out, h = blk.layer(x, res, w, zero_centered=False)
    q, s, h2 = norm.rms_norm_int8(x, w, residual=res)
    assert torch.equal(h, h2)
    heads = blk.forward_local((q, s))
    q2, s2 = gemm.quantize_rows_int8(heads.reshape(2 * T, -1))
    assert torch.equal(out.reshape(2 * T, -1), gemm.gemm_int8_transposed_b(q2, blk.w_out, s2, blk.w_out_scale))
    y = gemm.gemm_int8_transposed_b(q.reshape(2 * T, -1), blk.w, s, blk.w_scale).cpu().double()
    exact = (q.reshape(2 * T, -1).cpu().double() @ blk.w.cpu().double().t()) * s.reshape(-1, 1).cpu().double() * blk.w_scale.cpu().double()
    assert ((y - exact).abs() <= (2.0 ** -8 + 4 * 2.0 ** -24) * exact.abs() + 2.0 ** -133).all()
    want, h3 = plain.layer(x, res, w)
    assert torch.equal(h, h3)
    assert float((out.float() - want.float()).norm() / want.float().norm()) < 0.078
    second, _ = blk.layer(out, h, w)  # the next layer on what this one has left
    assert torch.isfinite(second.float()).all()
    assert gdn.read_status() == 0


@pytest.mark.gpu
def test_head_shards_compose(built_lib):
    """A rank's columns are the same numbers with the same scales, and a token's scale is made of the whole row: the shards' heads are the unsharded block's."""
    x = torch.randn(2, 130, HIDDEN, generator=torch.Generator().manual_seed(3)).bfloat16().cuda()
    full = make("GdnBlockShard").forward(x)
    parts = [make("GdnBlockShard", rank=r, world=2).forward_local(x) for r in range(2)]
    err = (torch.cat(parts, 2).float() - full.float()).norm() / full.float().norm()
    assert float(err) < 1e-6


@pytest.mark.gpu
def test_captured_layer(built_lib):
    blk = make()
    x, res, w = torch.randn(3, 40, HIDDEN).bfloat16().cuda(), torch.randn(3, 40, HIDDEN).bfloat16().cuda(), torch.rand(HIDDEN).cuda() + 0.5
    blk.layer(x, res, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, h = blk.layer(x, res, w)
    for _ in range(2):
        x.copy_(torch.randn_like(x))
        want = blk.layer(x, res, w)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(h, want[1])
