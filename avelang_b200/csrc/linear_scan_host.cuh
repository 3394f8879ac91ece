// Host side of the scans of linear attention: how a batch is cut into segments, tensor maps, launches.
#pragma once
#include <cmath>

#include "linear_scan.cuh"

namespace ave {
namespace {
namespace lin {

// One CTA walks a segment of one (sequence, value head).  Whole sequences need one pass; segments need their own increments first (a pass that reads Y and W alone) and the chain
// of them, so they pay where there are too few sequences and heads for the SMs, or where one sequence is so long that the others wait for it.  The lengths of packed sequences are
// not known here: the longest is taken to be four times the mean.  Unit: a chunk of the scan, 2.2 us on every SM; a chunk of the first pass takes 0.45 of that, a CTA's
// beginning and end 3 and 2.5, the chain and its launches 2.5 (8192 tokens x 32 heads, forward: whole 304 us, segments of 4096 tokens
// 212, of 2048 123; 24 prompts of 65536 tokens x 32 heads, one draw of their lengths: whole 568, segments of 5504 908;
// other draws, whole, up to 690.)
inline Plan plan_of(int B, int64_t T, int n_seqs, bool packed, int heads) {
  constexpr double SMS = 148;
  const double chunks = (double)((T * B + C - 1) / C);
  const double longest = packed ? (n_seqs > 1 ? fmin((double)T, 4.0 * T / n_seqs) : (double)T) / C : (double)((T + C - 1) / C);
  auto waves = [&](double units) { return packed ? units / SMS + 0.5 : (double)(int64_t)(units / SMS + 0.999999); };
  const double seqs = packed ? (double)n_seqs : (double)B;
  double best = packed ? fmax((chunks + 3.0 * seqs) * heads / SMS, longest + 3.0) + (n_seqs > MOST_IN_ORDER ? 0.25 * longest : 0.0) : waves(seqs * heads) * (longest + 3.0);
  int64_t len = 0;
  for (int parts = 2; parts <= 256; ++parts) {
    const int64_t each = (int64_t)((longest + parts - 1) / parts);
    if (each < 4) break;
    const double units = packed ? (chunks / (double)each + 0.5 * seqs) * heads : seqs * heads * (double)(((int64_t)longest + each - 1) / each);
    const double t = waves(units) * (1.45 * (double)each + 5.5) + 2.5 + 0.1 * parts;
    if (t < 0.95 * best) { best = t; len = each * C; }
  }
  Plan p;
  p.cut = len > 0;
  p.len = p.cut ? (int)len : 1 << 30;
  p.slots = p.cut ? T * B / len + n_seqs + 1 : n_seqs;
  return p;
}

inline void set_scale(Args& a, float scale) {  // of P'
  a.log_scale = (float)log2(fabs((double)scale));
  a.negative = scale < 0.f;
}

inline size_t state_bytes(const Plan& p, int heads, int dk, int dv) {  // increments and entering states, and the segments' decays
  return p.cut ? (size_t)p.slots * heads * ((size_t)dk * dv * 4) + (((size_t)p.slots * heads * 4 + 255) & ~(size_t)255) : 0;
}
inline void place_states(Args& a, void* ws, int dk, int dv) {
  a.seg_state = reinterpret_cast<float*>(ws);
  a.seg_decay = a.seg_state + (size_t)a.plan.slots * a.Hv * dk * dv;
}

// A head's features of 64 tokens of a [B, T, heads, d] tensor: 64 features after 64 features, so that a tile is one copy
inline int operand_map(CUtensorMap* m, const void* p, int d, int heads, int B, int T, int64_t sb, int64_t st, int64_t sh) {
  const uint32_t box[5] = {64, 64, (uint32_t)d / 64, 1, 1};
  const uint64_t dims[5] = {64, (uint64_t)T, (uint64_t)d / 64, (uint64_t)heads, (uint64_t)B};
  const uint64_t str[5] = {2, (uint64_t)(T > 1 ? st : d) * 2, 128, (uint64_t)(heads > 1 ? sh : d) * 2, (uint64_t)(B > 1 ? sb : d) * 2};
  return make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), 5, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

// 32 features of 64 tokens of the result; where its layout has no map, rows leave by 16-byte stores
inline bool result_map(CUtensorMap* m, void* p, int d, int heads, int B, int T, int64_t sb, int64_t st, int64_t sh) {
  const uint32_t box[4] = {32, 1, 64, 1};
  const uint64_t dims[4] = {(uint64_t)d, (uint64_t)heads, (uint64_t)T, (uint64_t)B};
  const uint64_t str[4] = {2, (uint64_t)(heads > 1 ? sh : d) * 2, (uint64_t)(T > 1 ? st : d) * 2, (uint64_t)(B > 1 ? sb : d) * 2};
  const int last_error = g_last_cuda_error;
  const bool ok = make_tmap(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, p, 4, dims, str, box, CU_TENSOR_MAP_SWIZZLE_64B) == AVE_GDN_OK;
  if (!ok) g_last_cuda_error = last_error;
  return ok;
}

// The register split of the roles counts on the registers that the kernel is launched with.
template <auto* kernel>
int scan_ready(int smem) {
  static std::atomic<bool> looked{false};
  if (!looked.load(std::memory_order_acquire)) {
    cudaFuncAttributes at;
    AVE_CUDA_TRY(cudaFuncGetAttributes(&at, kernel));
    if (at.numRegs != REGS_LAUNCH) return cuda_fail(cudaErrorInvalidKernelImage);
    looked.store(true, std::memory_order_release);
  }
  return allow_smem<kernel>(smem);
}
inline int64_t scan_grid(const Args& a) { return a.plan.slots * a.Hv; }
template <int DK, int DV, Mode kMode>
int launch_scan(const Args& a, const Maps& maps, cudaStream_t stream) {
  constexpr auto* kernel = &scan_kernel<DK, DV, false, kMode>;
  constexpr int smem = Cfg<kMode>::SMEM;
  const int rc = scan_ready<kernel>(smem);
  if (rc != AVE_GDN_OK) return rc;
  if (scan_grid(a) > 0x7fffffff) return AVE_GDN_UNSUPPORTED;
  AVE_CUDA_TRY(launch_after(kernel, (unsigned)scan_grid(a), THREADS, smem, stream, a, maps));
  return AVE_GDN_OK;
}
template <int DK, int DV>
int64_t chain_grid(const Args& a) { return (int64_t)a.n_seqs * a.Hv * (DK * DV / 1024); }

template <class F>
int by_dims(int dk, int dv, F f) {
  if (dk == 128) return dv == 128 ? f(std::integral_constant<int, 128>(), std::integral_constant<int, 128>())
                                  : f(std::integral_constant<int, 128>(), std::integral_constant<int, 64>());
  return dv == 128 ? f(std::integral_constant<int, 64>(), std::integral_constant<int, 128>())
                   : f(std::integral_constant<int, 64>(), std::integral_constant<int, 64>());
}

}  // namespace lin
}  // namespace
}  // namespace ave
