// Linear attention with a decay for each head, token by token:  M <- e^g M + k v^T,  o = scale M^T q.
//
// Bound by HBM: a state tile M[dk][dv] is read once and written once, whatever the number of tokens between.  A CTA holds COLS columns of
// one (sequence, value head) in registers; columns are independent of one another, so with few sequences a tile is shared out among
// several CTAs, and the sum over the dk rows is one pass through shared memory a token.  (256 sequences x 32 heads of 128 x 128, 1.08 GB of states: 165 us, the copy rate;
// one sequence: 5 us, a launch and one trip of a tile.  Tokens behind one another wait for their own q, k, v and g: 64 sequences x 32 heads, 1, 2, 4, 8, 16 tokens each,
// 51, 61, 78, 117 and 193 us, 256 sequences 172, 209, 275, 418 and 727, caches cold.)
#include "common.cuh"

namespace ave {
namespace {

__device__ __forceinline__ float decay_of(const float* g, int64_t at) {
  if (g == nullptr) return 1.f;
  const float x = g[at];
  return expf(x < -1e6f ? -1e6f : x);  // (a NaN stays one)
}

// 256 threads: a warp covers 128 / COLS rows at a time with one float4 a lane
template <int DK, int COLS>
__global__ void __launch_bounds__(256) linear_decode_kernel(const AveLinearArgs a) {
  constexpr int LANES = COLS / 4, RPL = 32 / LANES, LOADS = DK / (8 * RPL);
  static_assert(LOADS >= 1 && LOADS * 8 * RPL == DK, "rows");
  __shared__ float k_s[2][DK], q_s[2][DK];
  __shared__ __align__(16) float red[2][8][COLS];
  const int parts = a.dv / COLS;
  const int part = blockIdx.x % parts, unit = blockIdx.x / parts;
  const int n = unit / a.Hv, h = unit % a.Hv, hk = h / (a.Hv / a.Hk);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = (lane % LANES) * 4, row0 = warp * (DK / 8) + lane / LANES;

  pdl_trigger();
  pdl_wait();
  const SeqSpan sp = seq_span(a.cu_seqlens, n, a.T, a.status);
  if (!sp.ok) return;
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.o) + sp.b * a.o_stride_b + (int64_t)h * a.o_stride_h + part * COLS;
  int slot = n;
  if (a.state_indices != nullptr) {
    slot = a.state_indices[n];
    if (slot >= a.num_slots) {
      if (a.status != nullptr && threadIdx.x == 0) atomicOr(a.status, AVE_GDN_DEV_BAD_SLOT);
      slot = -1;
    }
    if (slot < 0) {  // no state access; the sequence's outputs are zero
      for (int t = 0; t < sp.len; ++t)
        if (threadIdx.x < COLS) o[(int64_t)(sp.t0 + t) * a.o_stride_t + threadIdx.x] = __float2bfloat16(0.f);
      return;
    }
  }
  const int64_t tile = ((int64_t)slot * a.Hv + h) * DK * a.dv + part * COLS;
  float4 S[LOADS];
  if (a.initial_state != nullptr) {
    const float* src = a.initial_state + tile;
    asm volatile("" : "+l"(src));  // keeps the streaming loads behind pdl_wait
#pragma unroll
    for (int i = 0; i < LOADS; ++i) S[i] = __ldcs(reinterpret_cast<const float4*>(src + (int64_t)(row0 + i * RPL) * a.dv + col));
  } else {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) S[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  const __nv_bfloat16* q = reinterpret_cast<const __nv_bfloat16*>(a.q) + sp.b * a.q_stride_b + (int64_t)hk * a.q_stride_h;
  const __nv_bfloat16* k = reinterpret_cast<const __nv_bfloat16*>(a.k) + sp.b * a.k_stride_b + (int64_t)hk * a.k_stride_h;
  const __nv_bfloat16* v = reinterpret_cast<const __nv_bfloat16*>(a.v) + sp.b * a.v_stride_b + (int64_t)h * a.v_stride_h + part * COLS;
  for (int t = 0; t < sp.len; ++t) {
    const int64_t tok = sp.t0 + t;
    const int turn = t & 1;  // the buffers of a token are written again two tokens later, behind the barriers of the next
    if (threadIdx.x < DK) k_s[turn][threadIdx.x] = bf2f(k[tok * a.k_stride_t + threadIdx.x]);
    else if (threadIdx.x < 2 * DK) q_s[turn][threadIdx.x - DK] = bf2f(q[tok * a.q_stride_t + threadIdx.x - DK]);
    float v4[4];
    unpack_bf16x4(*reinterpret_cast<const uint2*>(v + tok * a.v_stride_t + col), v4);
    const float decay = decay_of(a.g, sp.b * a.g_stride_b + tok * a.g_stride_t + h);
    __syncthreads();
    float p[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const float kr = k_s[turn][row0 + i * RPL], qr = q_s[turn][row0 + i * RPL];
      S[i].x = fmaf(decay, S[i].x, kr * v4[0]); S[i].y = fmaf(decay, S[i].y, kr * v4[1]);
      S[i].z = fmaf(decay, S[i].z, kr * v4[2]); S[i].w = fmaf(decay, S[i].w, kr * v4[3]);
      p[0] = fmaf(S[i].x, qr, p[0]); p[1] = fmaf(S[i].y, qr, p[1]); p[2] = fmaf(S[i].z, qr, p[2]); p[3] = fmaf(S[i].w, qr, p[3]);
    }
#pragma unroll
    for (int off = LANES; off < 32; off <<= 1)
#pragma unroll
      for (int c = 0; c < 4; ++c) p[c] += __shfl_xor_sync(0xffffffffu, p[c], off);
    if (lane < LANES) *reinterpret_cast<float4*>(&red[turn][warp][col]) = make_float4(p[0], p[1], p[2], p[3]);
    __syncthreads();
    if (threadIdx.x < COLS) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += red[turn][w][threadIdx.x];
      o[tok * a.o_stride_t + threadIdx.x] = __float2bfloat16(a.scale * s);
    }
  }
  if (a.final_state != nullptr) {
    float* dst = a.final_state + tile;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) __stcs(reinterpret_cast<float4*>(dst + (int64_t)(row0 + i * RPL) * a.dv + col), S[i]);
  }
}

}  // namespace

int launch_linear_decode(const AveLinearArgs& a, cudaStream_t stream) {
  const int64_t tiles = (int64_t)a.n_seqs * a.Hv;
  if (tiles == 0) return AVE_GDN_OK;
  // columns a CTA: a quarter of a tile where halves would leave SMs idle (32 heads, 128 x 128, quarters and halves: 1 sequence 2.9 and 3.0 us, 4 3.8 and 5.0,
  // 8 6.6 and 5.5, 64 49 and 42.5)
  const int cols = tiles * (a.dv / 64) < 2 * 148 ? 32 : 64;
  const int64_t grid = tiles * (a.dv / cols);
  if (grid > 0x7fffffff) return AVE_GDN_UNSUPPORTED;
  auto* kernel = a.dk == 128 ? (cols == 32 ? linear_decode_kernel<128, 32> : linear_decode_kernel<128, 64>)
                             : (cols == 32 ? linear_decode_kernel<64, 32> : linear_decode_kernel<64, 64>);
  AVE_CUDA_TRY(launch_after(kernel, (unsigned)grid, 256, 0, stream, a));
  return AVE_GDN_OK;
}

}  // namespace ave
