"""Results that the library allocates itself: ordinary tensors of the mode, stream and device that they are made in."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def calls():
    from avelang_b200 import gdn, gemm, norm
    x, w = torch.randn(6, 128, device="cuda").bfloat16(), torch.rand(128, device="cuda")
    y, h, rstd = norm.rms_norm(x, w, residual=x, return_stats=True)
    q, s = gemm.quantize_rows_int8(x)
    return [y, h, rstd, q, s, gemm.gemm_int8_transposed_b(q, q, s, s), norm.layer_norm(x), gdn.gated_rmsnorm(x.view(1, 6, 1, 128), x.view(1, 6, 1, 128))]


def test_modes(built_lib):
    with torch.inference_mode():
        assert all(t.is_inference() for t in calls())
    with torch.no_grad():
        made = calls()
    assert not any(t.is_inference() or t.requires_grad for t in made)
    for t in made:  # their storage and version counter are their own
        before = t._version
        t.zero_()
        assert t._version == before + 1 and t.is_contiguous() and t.storage_offset() == 0
    assert len({t.untyped_storage().data_ptr() for t in made}) == len(made)


def test_deterministic_fill(built_lib):
    """With deterministic algorithms torch fills what it allocates; a result is written over it all the same."""
    torch.use_deterministic_algorithms(True)
    try:
        assert all(torch.isfinite(t.float()).all() for t in calls())
    finally:
        torch.use_deterministic_algorithms(False)


def test_memory_is_given_back_and_stays_with_its_stream(built_lib):
    from avelang_b200 import norm
    x = torch.randn(4096, 1024, device="cuda").bfloat16()
    norm.rms_norm(x)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    for _ in range(50):
        norm.rms_norm(x, return_stats=True)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == held
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = norm.rms_norm(x)
    side.synchronize()
    assert torch.equal(y, norm.rms_norm(x))
    blocks = [b for seg in torch.cuda.memory_snapshot() for b in seg["blocks"] if b["state"] == "active_allocated" and seg["stream"] == side.cuda_stream]
    assert any(b["size"] >= y.numel() * 2 for b in blocks)  # in the pool of the stream that it was made on
