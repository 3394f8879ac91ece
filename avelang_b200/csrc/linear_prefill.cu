// Chunked form of linear attention with a decay for each head over whole sequences: one scan, or, where sequences are cut into segments that
// run side by side, the segments' increments, their chain, and the scan from the states that enter them.  (32 heads of 128 over 16 key heads: 8192 tokens 118 to 129 us, of which
// increments 43, chain 6, scan 70 to 77; 203 tokens 13.5 us; 24 prompts of 65536 tokens 568 to 690 us by the draw of their lengths, 2.5 to 3.0 TB/s.)
#include "linear_scan_host.cuh"

namespace ave {

static lin::Plan prefill_plan(const AveLinearArgs& a) { return lin::plan_of(a.B, a.T, a.n_seqs, a.cu_seqlens != nullptr, a.Hv); }

size_t linear_prefill_workspace_bytes(const AveLinearArgs& a) { return lin::state_bytes(prefill_plan(a), a.Hv, a.dk, a.dv); }

int launch_linear_prefill(const AveLinearArgs& a, cudaStream_t stream) {
  lin::Args s{};
  s.cu_seqlens = a.cu_seqlens; s.status = a.status;
  s.B = a.B; s.T = a.T; s.Hv = a.Hv; s.n_seqs = a.n_seqs; s.num_slots = a.num_slots; s.state_indices = a.state_indices;
  s.x_div = s.y_div = a.Hv / a.Hk; s.w_div = s.e_div = 1;
  s.g = a.g; s.g_stride_b = a.g_stride_b; s.g_stride_t = a.g_stride_t;
  lin::set_scale(s, a.scale);
  s.scale_e = a.scale; s.scale_w = 1.f;
  s.o = a.o; s.o_stride_b = a.o_stride_b; s.o_stride_t = a.o_stride_t; s.o_stride_h = a.o_stride_h;
  s.zero_outside = a.cu_seqlens != nullptr && (a.flags & AVE_LINEAR_FLAG_ZERO_OUTSIDE) != 0;
  s.state_in = a.initial_state; s.state_out = a.final_state; s.st_y = a.dv; s.st_w = 1;
  s.plan = prefill_plan(a);
  if (s.plan.cut) {
    lin::place_states(s, a.workspace, a.dk, a.dv);
    s.final_by_chain = a.final_state != nullptr;
  }
  lin::Maps m{};
  int rc;
  if ((rc = lin::operand_map(&m.x, a.q, a.dk, a.Hk, a.B, a.T, a.q_stride_b, a.q_stride_t, a.q_stride_h))) return rc;
  if ((rc = lin::operand_map(&m.y, a.k, a.dk, a.Hk, a.B, a.T, a.k_stride_b, a.k_stride_t, a.k_stride_h))) return rc;
  if ((rc = lin::operand_map(&m.w, a.v, a.dv, a.Hv, a.B, a.T, a.v_stride_b, a.v_stride_t, a.v_stride_h))) return rc;
  m.o_ok = lin::result_map(&m.o, a.o, a.dv, a.Hv, a.B, a.T, a.o_stride_b, a.o_stride_t, a.o_stride_h);
  return lin::by_dims(a.dk, a.dv, [&](auto dk, auto dv) {
    if (s.plan.cut) {
      const int r = lin::launch_scan<dk, dv, lin::STATE>(s, m, stream);
      if (r != AVE_GDN_OK) return r;
      const int64_t grid = lin::chain_grid<dk, dv>(s);
      if (grid > 0x7fffffff) return (int)AVE_GDN_UNSUPPORTED;
      AVE_CUDA_TRY(launch_after(lin::chain_kernel<dk, dv>, (unsigned)grid, 256, 0, stream, s));
    }
    return s.state_out != nullptr && !s.final_by_chain ? lin::launch_scan<dk, dv, lin::OUT3>(s, m, stream) : lin::launch_scan<dk, dv, lin::OUT2>(s, m, stream);
  });
}

}  // namespace ave
