// Gradients of linear attention with a decay for each head.  With R_t the gradient of the state after token t,
//     R_t = scale q_t do_t^T + e^{g_{t+1}} R_{t+1},
//     dq_t = scale S_t do_t,   dk_t = R_t v_t,   dv_t = R_t^T k_t
// are scans of the forward pass's form: (do, v, k) forwards in time, (v, do, q) and (k, q, do) backwards.  The gradient of g_t is the sum over all pairs
// s < t <= u of m_us = e^{G_u - G_s} scale (q_u.k_s)(do_u.v_s) (the initial state counts as a token in front of all others, the final state's gradient as one
// behind them), so that with the strictly causal parts A_t = sum over s < t of m_ts and B_t = sum over u > t of m_ut
//     dg_{t+1} = dg_t - A_t + B_t,
// and dg at the first token of a segment is the product <S, R> of the state and the gradient that meet there.  The parts of A and B across chunks come with the
// scans for dq and dk, as q_t . (e_t S do_t) and k_t . (e_t R v_t) in front of the chunk's own terms; those inside a chunk are sums over the rows and the columns of one product,
// (q k^T) (do v^T) elementwise, in 32 bits.  The shorter formula with q.dq - k.dk would take the diagonal's terms, which are far larger where decays are strong, from both sides.
#include "linear_scan_host.cuh"

namespace ave {
namespace {
namespace lin {

// The scans of one call side by side: their CTAs fill the SMs together, the longest first.
struct Pass { Args a; Maps m; };
struct TwoPasses { Pass p[2]; };
struct ThreePasses { Pass p[3]; };
// Increments of the segments from the front, and from behind
template <int DK, int DV>
__global__ void __launch_bounds__(THREADS, 1) states_kernel(const __grid_constant__ TwoPasses t) {
  if (blockIdx.y == 0) scan<DK, DV, false, STATE>(t.p[0].a, t.p[0].m);
  else scan<DK, DV, true, STATE>(t.p[1].a, t.p[1].m);
}
template <int DK, int DV>
__global__ void __launch_bounds__(256) chains_kernel(const Args fwd, const Args rev) {
  if (blockIdx.y == 0) chain<DK, DV, false>(fwd);
  else chain<DK, DV, true>(rev);
}
// dq, dk, dv (kDq: the mode of the first two, kDv of the last).  2 x 4096 tokens, 32 heads: 335 us, one behind the other 337 (128 CTAs on 148 SMs each); with few heads the SMs fill:
// five documents of 3001 tokens, 8 heads, 48 us.
template <int DK, int DV, Mode kDq, Mode kDv>
__global__ void __launch_bounds__(THREADS, 1) grads_kernel(const __grid_constant__ ThreePasses t) {
  if (blockIdx.y == 0) scan<DV, DK, false, kDq>(t.p[0].a, t.p[0].m);
  else if (blockIdx.y == 1) scan<DV, DK, true, kDq>(t.p[1].a, t.p[1].m);
  else scan<DK, DV, true, kDv>(t.p[2].a, t.p[2].m);
}
template <int DK, int DV, Mode kDq, Mode kDv>
int launch_grads(const ThreePasses& t, cudaStream_t stream) {
  constexpr auto* kernel = &grads_kernel<DK, DV, kDq, kDv>;
  constexpr int smem = Cfg<kDq>::SMEM > Cfg<kDv>::SMEM ? Cfg<kDq>::SMEM : Cfg<kDv>::SMEM;
  const int rc = scan_ready<kernel>(smem);
  if (rc != AVE_GDN_OK) return rc;
  AVE_CUDA_TRY(launch_after(kernel, dim3((unsigned)scan_grid(t.p[0].a), 3), THREADS, smem, stream, t));
  return AVE_GDN_OK;
}

// The value heads of a key head, summed: out[row][hk][d] = sum over r of part[row][hk rep + r][d]; eight features a thread; dq, and dk.
// Bound by HBM and L2 (8192 tokens, 32 heads of 128 onto 16: 45 us for 335 MB).
__global__ void __launch_bounds__(256) sum_heads_kernel(const float* parts, int64_t apart, __nv_bfloat16* dq, __nv_bfloat16* dk, int64_t pieces, int d8, int hk, int rep) {
  const float* part = parts + blockIdx.y * apart;
  __nv_bfloat16* out = blockIdx.y == 0 ? dq : dk;
  pdl_wait();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (int64_t)gridDim.x * 256) {
    const int64_t head = i / d8;  // row * hk + key head
    const float* src = part + (head * rep * d8 + i % d8) * 8;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
    for (int r = 0; r < rep; ++r) {
      const float4 p = __ldcs(reinterpret_cast<const float4*>(src + (int64_t)r * d8 * 8)), q = __ldcs(reinterpret_cast<const float4*>(src + (int64_t)r * d8 * 8 + 4));
      x.x += p.x; x.y += p.y; x.z += p.z; x.w += p.w;
      y.x += q.x; y.y += q.y; y.z += q.z; y.w += q.w;
    }
    *reinterpret_cast<uint4*>(out + i * 8) = make_uint4(pack_bf16x2(x.x, x.y), pack_bf16x2(x.z, x.w), pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
  }
}

// m_ts of a chunk's pairs s < t, summed over s into a[t] and over t into b[s]: one CTA a (chunk, value head), as warp-level MMAs, one of the ten 16 x 16 blocks on and below the diagonal
// a warp, so that the CTA's time is a block's.  Bound by the four tiles it reads and the latencies in front of them
// (8192 tokens, 32 heads: 54 us for 201 MB of inputs; 77 with four warps of 16 rows each).
struct PairSums {
  const __nv_bfloat16 *q, *k, *v, *d_o;
  int64_t q_b, q_t, q_h, k_b, k_t, k_h, v_b, v_t, v_h, o_b, o_t, o_h;
  int rep;
  float scale;
  float *a, *b;  // [Hv][B T]
};
constexpr int PAIR_THREADS = 320;
template <int DK, int DV>
__global__ void __launch_bounds__(PAIR_THREADS) pair_sums_kernel(const Args s, const PairSums p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = tc::align1024(smem_raw);
  constexpr int KB = 2 * DK, VB = 2 * DV, Q0 = 0, K0 = 64 * KB, V0 = 2 * K0, O0 = V0 + 64 * VB;
  float2* G = reinterpret_cast<float2*>(smem + O0 + 64 * VB);  // [64]
  float *cols = reinterpret_cast<float*>(G + 64), *rows = cols + 256;  // [4][64] each: of the block's row for the columns, of its column for the rows
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_wait();
  if (!offsets_fit(s, false)) return;
  const int h = blockIdx.x % s.Hv, hk = h / p.rep;
  const Seg c = seg_of_slot(s, blockIdx.x / s.Hv);
  if (!c.ok || c.len == 0) return;
  const uint32_t base = tc::smem_u32(smem);
  if (warp < 8) {
    load_tile<64, DK / 8, 256>(base + Q0, p.q + c.b * p.q_b + (int64_t)c.t0 * p.q_t + hk * p.q_h, p.q_t, c.len, threadIdx.x);
    load_tile<64, DK / 8, 256>(base + K0, p.k + c.b * p.k_b + (int64_t)c.t0 * p.k_t + hk * p.k_h, p.k_t, c.len, threadIdx.x);
    cp_commit();
    load_tile<64, DV / 8, 256>(base + V0, p.v + c.b * p.v_b + (int64_t)c.t0 * p.v_t + h * p.v_h, p.v_t, c.len, threadIdx.x);
    load_tile<64, DV / 8, 256>(base + O0, p.d_o + c.b * p.o_b + (int64_t)c.t0 * p.o_t + h * p.o_h, p.o_t, c.len, threadIdx.x);
    cp_commit();
  } else if (warp == 8) {
    auto fetch = [&](int t) { return t < c.len ? s.g[c.b * s.g_stride_b + (int64_t)(c.t0 + t) * s.g_stride_t + h] : 0.f; };
    Two G0, G1;
    gate_scan(fetch(2 * lane), fetch(2 * lane + 1), lane, G0, G1);
    G[2 * lane] = make_float2(G0.h, G0.l);
    G[2 * lane + 1] = make_float2(G1.h, G1.l);
  }
  cp_wait<1>();
  __syncthreads();
  const int i = warp < 1 ? 0 : warp < 3 ? 1 : warp < 6 ? 2 : 3, j = warp - i * (i + 1) / 2, row = 16 * i + (lane >> 2);
  float x[2][4], y[2][4];
#pragma unroll
  for (int n = 0; n < 2; ++n) { zero(x[n]); zero(y[n]); }
#pragma unroll
  for (int k = 0; k < DK / 16; ++k) {
    uint32_t l[4], r[4];
    ldsm4(l, base + Q0 + at_a<KB>(16 * i, 2 * k, lane));
    ldsm4(r, base + K0 + at_b<KB>(16 * j, 2 * k, lane));
    mma_bf16(x[0], l, r[0], r[1]);
    mma_bf16(x[1], l, r[2], r[3]);
  }
  float own[2] = {0.f, 0.f};
  const float2 gt[2] = {G[row], G[row + 8]};
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = row + 8 * (e >> 1), col = 16 * j + 8 * n + 2 * (lane & 3) + (e & 1);
      const float2 gs = G[col];
      x[n][e] = col < t ? p.scale * ex2((gt[e >> 1].x - gs.x) + (gt[e >> 1].y - gs.y)) * x[n][e] : 0.f;
    }
  cp_wait<0>();
  __syncthreads();
#pragma unroll
  for (int k = 0; k < DV / 16; ++k) {
    uint32_t l[4], r[4];
    ldsm4(l, base + O0 + at_a<VB>(16 * i, 2 * k, lane));
    ldsm4(r, base + V0 + at_b<VB>(16 * j, 2 * k, lane));
    mma_bf16(y[0], l, r[0], r[1]);
    mma_bf16(y[1], l, r[2], r[3]);
  }
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = row + 8 * (e >> 1), col = 16 * j + 8 * n + 2 * (lane & 3) + (e & 1);
      const float m = col < t ? x[n][e] * y[n][e] : 0.f;
      own[e >> 1] += m;
      sum[e & 1] += m;
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], o);
      sum[1] += __shfl_xor_sync(0xffffffffu, sum[1], o);
    }
    if (lane < 4) *reinterpret_cast<float2*>(cols + 64 * i + 16 * j + 8 * n + 2 * lane) = make_float2(sum[0], sum[1]);
  }
#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    own[0] += __shfl_xor_sync(0xffffffffu, own[0], o);
    own[1] += __shfl_xor_sync(0xffffffffu, own[1], o);
  }
  if ((lane & 3) == 0) { rows[64 * j + row] = own[0]; rows[64 * j + row + 8] = own[1]; }
  __syncthreads();
  const int64_t at = ((int64_t)h * s.B + c.b) * s.T + c.t0;
  const int t = threadIdx.x & 63, block = t >> 4;
  if (t < c.len && threadIdx.x < 128) {
    const bool of_row = threadIdx.x < 64;
    float sum = 0.f;
    for (int n = of_row ? 0 : block; n <= (of_row ? block : 3); ++n) sum += (of_row ? rows : cols)[64 * n + t];
    (of_row ? p.a : p.b)[at + t] = sum;
  }
}

struct GateGrad {
  const float *inter_a, *intra_a, *inter_b, *intra_b;  // of the scans for dq and dk
  const float *seg_s, *seg_r;  // states that enter the segments, from the front and from behind
  const float *s0, *ds0;     // null: no initial state
  const float *sT, *dsT;     // null: the final states have no gradient
  float* dg;                 // [B, T, Hv], or null
  float* sums;               // [slot][Hv]: sums over the segment's tokens, or null
  int dk, dv;
};

template <int THREADS>
__device__ __forceinline__ double block_sum(double x, double* sm) {  // all threads get it
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sm[threadIdx.x >> 5] = x;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) s += sm[w];
  return s;
}

// One CTA a segment and head: the running sum of B - A from the segment's first token, in 64 bits.  Its end is known too, <S, R> of the next segment's beginning or of the final state and
// its gradient, or 0, and what is open there is spread evenly over the tokens: A and B are sums in 32 bits whose errors a running sum collects like a random walk, and a walk that is
// tied down at both ends strays 1.7 times less (2 x 4096 tokens in segments of 2048: 1.3e-6 of the gradient's norm without).  Bound by latencies: the next tokens are read while
// these are summed (20 us; 30 with 256 threads).
constexpr int GATE_THREADS = 512;
template <int PARTS>
__global__ void __launch_bounds__(GATE_THREADS) gate_grad_kernel(const Args a, const GateGrad q) {
  constexpr int N = GATE_THREADS;
  __shared__ double sm[N / 32], wsum[N / 32];
  pdl_wait();
  if (!offsets_fit(a, false)) return;
  const int h = blockIdx.x % a.Hv, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t slot = blockIdx.x / a.Hv;
  const Seg seg = seg_of_slot(a, slot);
  if (!seg.ok || seg.len == 0) {
    if (q.sums != nullptr && tid == 0) q.sums[slot * a.Hv + h] = 0.f;
    return;
  }
  const int64_t size = (int64_t)q.dk * q.dv;
  const float *x = nullptr, *y = nullptr;
  if (seg.j > 0) {
    x = q.seg_s + (slot * a.Hv + h) * size;
    y = q.seg_r + ((slot - 1) * a.Hv + h) * size;
  } else if (q.s0 != nullptr) {
    x = q.s0 + ((int64_t)seg.n * a.Hv + h) * size;
    y = q.ds0 + ((int64_t)seg.n * a.Hv + h) * size;
  }
  const float *xe = nullptr, *ye = nullptr;  // what meets behind the last token
  if (seg.j + 1 < seg.count) {
    xe = q.seg_s + ((slot + 1) * a.Hv + h) * size;
    ye = q.seg_r + (slot * a.Hv + h) * size;
  } else if (q.sT != nullptr) {
    xe = q.sT + ((int64_t)seg.n * a.Hv + h) * size;
    ye = q.dsT + ((int64_t)seg.n * a.Hv + h) * size;
  }
  auto product = [&](const float* x, const float* y) {
    double dot = 0.0;
    if (x != nullptr)
#pragma unroll 4
      for (int i = tid * 4; i < size; i += 4 * N) {
        const float4 u = *reinterpret_cast<const float4*>(x + i), v = *reinterpret_cast<const float4*>(y + i);
        dot += ((double)u.x * v.x + (double)u.y * v.y) + ((double)u.z * v.z + (double)u.w * v.w);
      }
    return dot;
  };
  const int64_t base = ((int64_t)h * a.B + seg.b) * a.T + seg.t0, plane = (int64_t)a.Hv * a.B * a.T;
  float va[PARTS + 1], vb[PARTS + 1];
  auto fetch = [&](int t) {
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
      va[p] = t < seg.len ? q.inter_a[p * plane + base + t] : 0.f;
      vb[p] = t < seg.len ? q.inter_b[p * plane + base + t] : 0.f;
    }
    va[PARTS] = t < seg.len ? q.intra_a[base + t] : 0.f;
    vb[PARTS] = t < seg.len ? q.intra_b[base + t] : 0.f;
  };
  auto step = [&] {  // B - A
    float ia = 0.f, ib = 0.f;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) { ia += va[p]; ib += vb[p]; }
    return ((double)ib - (double)ia) + ((double)vb[PARTS] - (double)va[PARTS]);
  };
  fetch(tid);
  double dot = product(x, y), open = product(xe, ye) - dot;  // dg of the first token; what the steps do not come to
  for (int t = tid; t < seg.len; t += N) {
    open -= step();
    fetch(t + N);
  }
  fetch(tid);
  double run = block_sum<N>(dot, sm), total = 0.0;
  open = block_sum<N>(open, sm) / seg.len;
  if (!isfinite(open)) open = 0.0;
  for (int t0 = 0; t0 < seg.len; t0 += N) {
    const int t = t0 + tid;
    const double d = step();
    fetch(t + N);
    double inc = d;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double u = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += u;
    }
    __syncthreads();
    if (lane == 31) wsum[warp] = inc;
    __syncthreads();
    double before = 0.0, whole = 0.0;
#pragma unroll
    for (int w = 0; w < N / 32; ++w) {
      if (w < warp) before += wsum[w];
      whole += wsum[w];
    }
    const double mine = run + before + inc - d + open * t;
    if (t < seg.len) {
      if (q.dg != nullptr) q.dg[((int64_t)seg.b * a.T + seg.t0 + t) * a.Hv + h] = (float)mine;
      total += mine;
    }
    run += whole;
  }
  if (q.sums != nullptr) {
    total = block_sum<N>(total, sm);
    if (tid == 0) q.sums[slot * a.Hv + h] = (float)total;
  }
}
// One decay a head: its gradient is the sum over all segments, in order
__global__ void __launch_bounds__(256) head_gate_grad_kernel(const Args a, const float* sums, float* dg) {
  __shared__ double sm[8];
  pdl_wait();
  if (!offsets_fit(a, false)) return;
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < a.plan.slots; i += 256) s += (double)sums[i * a.Hv + blockIdx.x];
  s = block_sum<256>(s, sm);
  if (threadIdx.x == 0) dg[blockIdx.x] = (float)s;
}

// Rows of a packed batch in front of its first offset and behind its last belong to no sequence: their gradients are zero.
__global__ void __launch_bounds__(128) clear_outside_kernel(const Args a, __nv_bfloat16* dq, __nv_bfloat16* dk, __nv_bfloat16* dv, float* dg, int wk, int wv) {
  pdl_wait();
  if (!offsets_fit(a, false)) return;
  const int lo = a.n_seqs > 0 ? a.cu_seqlens[0] : 0, hi = a.n_seqs > 0 ? a.cu_seqlens[a.n_seqs] : 0;
  const int outside = lo + (a.T - hi);
  for (int r = blockIdx.x; r < outside; r += gridDim.x) {
    const int64_t row = r < lo ? r : hi + (r - lo);
    for (int i = threadIdx.x; i < wk / 8; i += 128) {
      *reinterpret_cast<uint4*>(dq + row * wk + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
      *reinterpret_cast<uint4*>(dk + row * wk + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
    }
    for (int i = threadIdx.x; i < wv / 8; i += 128) *reinterpret_cast<uint4*>(dv + row * wv + 8 * i) = make_uint4(0u, 0u, 0u, 0u);
    if (dg != nullptr)
      for (int i = threadIdx.x; i < a.Hv; i += 128) dg[row * a.Hv + i] = 0.f;
  }
}

struct Layout {
  Plan plan;
  size_t s, s_decay, r, r_decay, part, inter_a, inter_b, intra_a, intra_b, sums, final, bytes;
};
Layout layout_of(const AveLinearBwdArgs& a) {
  Layout l{};
  l.plan = plan_of(a.B, a.T, a.n_seqs, a.cu_seqlens != nullptr, a.Hv);
  const size_t rows = (size_t)a.B * a.T * a.Hv;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t p = at;
    at += (bytes + 255) & ~(size_t)255;
    return p;
  };
  if (l.plan.cut) {
    const size_t tiles = (size_t)l.plan.slots * a.Hv;
    l.s = take(tiles * a.dk * a.dv * 4); l.s_decay = take(tiles * 4);
    l.r = take(tiles * a.dk * a.dv * 4); l.r_decay = take(tiles * 4);
  }
  if (a.Hv > a.Hk) l.part = take(2 * rows * a.dk * 4);
  if (a.g != nullptr) {
    l.inter_a = take(rows * (a.dk / 32) * 4); l.inter_b = take(rows * (a.dk / 32) * 4);
    l.intra_a = take(rows * 4); l.intra_b = take(rows * 4);
    l.sums = take((size_t)l.plan.slots * a.Hv * 4);
    if (a.d_final_state != nullptr) l.final = take((size_t)a.n_seqs * a.Hv * a.dk * a.dv * 4);
  }
  l.bytes = at;
  return l;
}

}  // namespace lin
}  // namespace

static const __nv_bfloat16* lin_bf(const void* p) { return reinterpret_cast<const __nv_bfloat16*>(p); }

size_t linear_backward_workspace_bytes(const AveLinearBwdArgs& a) { return lin::layout_of(a).bytes; }

int launch_linear_backward(const AveLinearBwdArgs& a, cudaStream_t stream) {
  const lin::Layout l = lin::layout_of(a);
  uint8_t* ws = reinterpret_cast<uint8_t*>(a.workspace);
  auto f32 = [&](size_t at) { return reinterpret_cast<float*>(ws + at); };
  const int rep = a.Hv / a.Hk;
  const bool grad = a.g != nullptr;
  int rc;
  CUtensorMap mq, mk, mv, mo;
  if ((rc = lin::operand_map(&mq, a.q, a.dk, a.Hk, a.B, a.T, a.q_stride_b, a.q_stride_t, a.q_stride_h))) return rc;
  if ((rc = lin::operand_map(&mk, a.k, a.dk, a.Hk, a.B, a.T, a.k_stride_b, a.k_stride_t, a.k_stride_h))) return rc;
  if ((rc = lin::operand_map(&mv, a.v, a.dv, a.Hv, a.B, a.T, a.v_stride_b, a.v_stride_t, a.v_stride_h))) return rc;
  if ((rc = lin::operand_map(&mo, a.d_o, a.dv, a.Hv, a.B, a.T, a.do_stride_b, a.do_stride_t, a.do_stride_h))) return rc;
  lin::Args base{};
  base.cu_seqlens = a.cu_seqlens; base.status = a.status;
  base.B = a.B; base.T = a.T; base.Hv = a.Hv; base.n_seqs = a.n_seqs; base.num_slots = a.n_seqs;
  base.g = a.g; base.g_stride_b = a.g_stride_b; base.g_stride_t = a.g_stride_t;
  base.x_div = base.y_div = base.w_div = base.e_div = 1;
  base.plan = l.plan;
  const int64_t part_floats = (int64_t)a.B * a.T * a.Hv * a.dk;
  lin::Args fwd = base, rev = base;  // states from the front, and their gradients from behind, as [dk][dv]
  fwd.y_div = rep; fwd.w_div = 1; fwd.scale_w = 1.f;
  fwd.state_in = a.initial_state; fwd.st_y = a.dv; fwd.st_w = 1;
  rev.y_div = rep; rev.w_div = 1; rev.scale_w = a.scale;
  rev.state_in = a.d_final_state; rev.st_y = a.dv; rev.st_w = 1;
  if (l.plan.cut) {
    fwd.seg_state = f32(l.s); fwd.seg_decay = f32(l.s_decay);
    rev.seg_state = f32(l.r); rev.seg_decay = f32(l.r_decay);
    rev.state_out = a.d_initial_state; rev.final_by_chain = a.d_initial_state != nullptr;
  }
  // gradient of q or k: dk features of Hk heads, summed over the value heads
  auto rows_of = [&](lin::Pass& p, void* out, int which) {
    lin::Args& s = p.a;
    s.o = out; s.o_stride_h = a.dk; s.o_stride_t = (int64_t)a.Hk * a.dk; s.o_stride_b = s.o_stride_t * a.T;
    if (rep == 1) {
      p.m.o_ok = lin::result_map(&p.m.o, out, a.dk, a.Hk, a.B, a.T, s.o_stride_b, s.o_stride_t, s.o_stride_h);
      return (int)AVE_GDN_OK;
    }
    s.o_part = f32(l.part) + which * part_floats;
    const uint64_t row = (uint64_t)a.Hv * a.dk * 4;
    const uint64_t dims[4] = {(uint64_t)a.dk, (uint64_t)a.Hv, (uint64_t)a.T, (uint64_t)a.B}, str[4] = {4, (uint64_t)a.dk * 4, row, row * a.T};
    const uint32_t box[4] = {32, 1, 64, 1};
    return make_tmap(&p.m.o, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, s.o_part, 4, dims, str, box, CU_TENSOR_MAP_SWIZZLE_128B);
  };
  rc = lin::by_dims(a.dk, a.dv, [&](auto dk, auto dv) {
    constexpr int DK = decltype(dk)::value, DV = decltype(dv)::value;
    int r;
    if (3 * lin::scan_grid(base) > 0x7fffffff) return (int)AVE_GDN_UNSUPPORTED;
    if (l.plan.cut) {
      lin::TwoPasses t{};
      t.p[0].a = fwd; t.p[0].m.y = mk; t.p[0].m.w = mv;
      t.p[1].a = rev; t.p[1].m.y = mq; t.p[1].m.w = mo;
      constexpr auto* states = &lin::states_kernel<DK, DV>;
      constexpr int smem = lin::Cfg<lin::STATE>::SMEM;
      if ((r = lin::scan_ready<states>(smem))) return r;
      AVE_CUDA_TRY(launch_after(states, dim3((unsigned)lin::scan_grid(base), 2), lin::THREADS, smem, stream, t));
      const int64_t grid = lin::chain_grid<DK, DV>(base);
      if (grid > 0x7fffffff) return (int)AVE_GDN_UNSUPPORTED;
      AVE_CUDA_TRY(launch_after(lin::chains_kernel<DK, DV>, dim3((unsigned)grid, 2), 256, 0, stream, fwd, rev));
    }
    lin::ThreePasses t{};
    {  // dq, and the final state
      lin::Args& s = t.p[0].a;
      lin::Maps& m = t.p[0].m;
      s = fwd;
      s.x_div = s.y_div = 1; s.w_div = s.e_div = rep; lin::set_scale(s, a.scale); s.scale_e = a.scale; s.st_y = 1; s.st_w = a.dv;
      m.x = mo; m.y = mv; m.w = mk; m.e = mq;
      if ((r = rows_of(t.p[0], a.d_q, 0))) return r;
      if (grad) {
        s.inter = f32(l.inter_a);
        if (a.d_final_state != nullptr) s.state_out = f32(l.final);
      }
    }
    {  // dk
      lin::Args& s = t.p[1].a;
      lin::Maps& m = t.p[1].m;
      s = rev;
      s.state_out = nullptr; s.final_by_chain = 0;
      s.x_div = s.y_div = 1; s.w_div = s.e_div = rep; lin::set_scale(s, a.scale); s.scale_e = 1.f; s.st_y = 1; s.st_w = a.dv;
      m.x = mv; m.y = mo; m.w = mq; m.e = mk;
      if ((r = rows_of(t.p[1], a.d_k, 1))) return r;
      if (grad) s.inter = f32(l.inter_b);
    }
    {  // dv, and the gradient of the initial state
      lin::Args& s = t.p[2].a;
      lin::Maps& m = t.p[2].m;
      s = rev;
      s.x_div = rep; lin::set_scale(s, a.scale); s.scale_e = 1.f;
      s.state_out = a.d_initial_state;
      m.x = mk; m.y = mq; m.w = mo;
      s.o = a.d_v; s.o_stride_h = a.dv; s.o_stride_t = (int64_t)a.Hv * a.dv; s.o_stride_b = s.o_stride_t * a.T;
      m.o_ok = lin::result_map(&m.o, a.d_v, a.dv, a.Hv, a.B, a.T, s.o_stride_b, s.o_stride_t, s.o_stride_h);
    }
    const bool exact = t.p[2].a.state_out != nullptr && !t.p[2].a.final_by_chain;
    if (grad) r = exact ? lin::launch_grads<DK, DV, lin::GRAD, lin::OUT3>(t, stream) : lin::launch_grads<DK, DV, lin::GRAD, lin::OUT2>(t, stream);
    else r = exact ? lin::launch_grads<DK, DV, lin::OUT2, lin::OUT3>(t, stream) : lin::launch_grads<DK, DV, lin::OUT2, lin::OUT2>(t, stream);
    if (r) return r;
    if (rep > 1) {
      const int64_t pieces = (int64_t)a.B * a.T * a.Hk * (a.dk / 8), ctas = (pieces + 255) / 256;
      AVE_CUDA_TRY(launch_after(lin::sum_heads_kernel, dim3((unsigned)(ctas < 148 * 8 ? ctas : 148 * 8), 2), 256, 0, stream, (const float*)f32(l.part), part_floats,
                                reinterpret_cast<__nv_bfloat16*>(a.d_q), reinterpret_cast<__nv_bfloat16*>(a.d_k), pieces, a.dk / 8, a.Hk, rep));
    }
    if (grad) {
      lin::Args s = base;
      s.plan = lin::Plan{lin::C, 1, (int64_t)a.B * a.T / lin::C + a.n_seqs + 1};
      const lin::PairSums p{lin_bf(a.q), lin_bf(a.k), lin_bf(a.v), lin_bf(a.d_o), a.q_stride_b, a.q_stride_t, a.q_stride_h, a.k_stride_b, a.k_stride_t, a.k_stride_h,
                            a.v_stride_b, a.v_stride_t, a.v_stride_h, a.do_stride_b, a.do_stride_t, a.do_stride_h, rep, a.scale, f32(l.intra_a), f32(l.intra_b)};
      constexpr auto* kernel = &lin::pair_sums_kernel<DK, DV>;
      constexpr int smem = 64 * 4 * (DK + DV) + 64 * 8 + 8 * 64 * 4 + 1024;
      if ((r = allow_smem<kernel>(smem))) return r;
      const int64_t grid = s.plan.slots * a.Hv;
      if (grid > 0x7fffffff) return (int)AVE_GDN_UNSUPPORTED;
      AVE_CUDA_TRY(launch_after(kernel, (unsigned)grid, lin::PAIR_THREADS, smem, stream, s, p));
    }
    return (int)AVE_GDN_OK;
  });
  if (rc != AVE_GDN_OK) return rc;
  const bool by_token = grad && (a.flags & AVE_LINEAR_FLAG_HEAD_GATE) == 0;
  if (grad) {
    lin::GateGrad q{};
    q.inter_a = f32(l.inter_a); q.inter_b = f32(l.inter_b); q.intra_a = f32(l.intra_a); q.intra_b = f32(l.intra_b);
    q.dk = a.dk; q.dv = a.dv;
    if (l.plan.cut) { q.seg_s = f32(l.s); q.seg_r = f32(l.r); }
    if (a.initial_state != nullptr) { q.s0 = a.initial_state; q.ds0 = a.d_initial_state; }
    if (a.d_final_state != nullptr) { q.sT = f32(l.final); q.dsT = a.d_final_state; }
    if (by_token) q.dg = a.d_g; else q.sums = f32(l.sums);
    const int64_t grid = l.plan.slots * a.Hv;
    AVE_CUDA_TRY(launch_after(a.dk == 128 ? lin::gate_grad_kernel<4> : lin::gate_grad_kernel<2>, (unsigned)grid, lin::GATE_THREADS, 0, stream, base, q));  // (scans give a sum for each 32 of dk)
    if (!by_token) AVE_CUDA_TRY(launch_after(lin::head_gate_grad_kernel, (unsigned)a.Hv, 256, 0, stream, base, (const float*)q.sums, a.d_g));
  }
  if (a.cu_seqlens != nullptr)
    AVE_CUDA_TRY(launch_after(lin::clear_outside_kernel, 148, 128, 0, stream, base, reinterpret_cast<__nv_bfloat16*>(a.d_q), reinterpret_cast<__nv_bfloat16*>(a.d_k),
                              reinterpret_cast<__nv_bfloat16*>(a.d_v), by_token ? a.d_g : (float*)nullptr, a.Hk * a.dk, a.Hv * a.dv));
  return AVE_GDN_OK;
}

}  // namespace ave
