// Layer norm over rows of n elements, and its gradients.
//
//   y = (x - m) r w + b,   m = mean(x),   r = 1 / sqrt(mean((x - m)^2) + eps)
//   dx = r (w dy - mean(w dy) - xh mean(w dy xh)),   xh = (x - m) r,   dw = sum over rows of dy xh,   db = sum over rows of dy
//
// Both are bound by HBM: the forward pass reads x and writes y, the backward pass reads x and dy and writes dx.  A row belongs to a group of threads, each of which keeps the same
// columns for every row it meets: the weights are read once a CTA, and the sums of the weight's gradient are registers too.  A CTA's sums go to scratch and a second kernel adds them
// in a fixed order.  Three forms by the row's length, figures for bf16 rows with fp32 weights, copy rate 6549 GB/s: rings of rows in shared memory for aligned rows of middle length
// (131072 x 2048: forward 179 to 187 us, 5.7 to 6.0 TB/s, through the public call 187 to 197, backward 267 to 272 us, 5.9 to 6.0 TB/s; 32768 x 8192: 203 and 262 us); rows in registers, U of them in flight a group, for short ones and for those
// that do not lie on 16 bytes (131072 x 64: 8.7 and 12.9 us; 30000 x 2047: 89 and 103 us, bound by the loads of single elements); and CTAs of 1024 threads for long ones
// (16384 x 16384 backward 567 us).
#include <cuda_fp16.h>

#include "common.cuh"
#include "tc.cuh"

namespace ave {
namespace {

template <class T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16(x); }
};
template <> struct Elem<__half> {
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
};
template <> struct Elem<float> {
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};

// VEC elements: 16 bytes, or one
template <class T, int VEC> struct alignas(sizeof(T) * VEC) Piece { T e[VEC]; };

template <class T, int VEC>
__device__ __forceinline__ Piece<T, VEC> raw_piece(const T* src, bool there) {
  Piece<T, VEC> p{};
  if (there) p = *reinterpret_cast<const Piece<T, VEC>*>(src);
  return p;
}
// A thread's elements are held as pairs, for packed arithmetic: with one element at a time the instructions come near the time of the copies.
// N: elements, an odd last one has a zero beside it.
template <int N> struct Pairs {
  static constexpr int H = (N + 1) / 2;
  float2 v[H];
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int i = 0; i < H; ++i) v[i] = make_float2(x, 2 * i + 1 < N ? x : 0.f);
  }
};
__device__ __forceinline__ float2 widen2(__nv_bfloat162 x) { return bf16x2_to_float2(*reinterpret_cast<const uint32_t*>(&x)); }
__device__ __forceinline__ float2 widen2(__half2 x) { return __half22float2(x); }
__device__ __forceinline__ float2 widen2(float2 x) { return x; }
__device__ __forceinline__ void narrow2(__nv_bfloat162& d, float2 x) { d = __floats2bfloat162_rn(x.x, x.y); }
__device__ __forceinline__ void narrow2(__half2& d, float2 x) { d = __floats2half2_rn(x.x, x.y); }
__device__ __forceinline__ void narrow2(float2& d, float2 x) { d = x; }
template <class T> struct Two;
template <> struct Two<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Two<__half> { using type = __half2; };
template <> struct Two<float> { using type = float2; };
// piece p of a thread's P pieces into, or out of, its elements
template <class T, int VEC, int N>
__device__ __forceinline__ void widen(Pairs<N>& f, int p, const Piece<T, VEC>& in) {
  if constexpr (VEC % 2 == 0) {
    const auto* two = reinterpret_cast<const typename Two<T>::type*>(in.e);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) f.v[p * VEC / 2 + i] = widen2(two[i]);
  } else {
    float& x = (p & 1) ? f.v[p / 2].y : f.v[p / 2].x;
    x = Elem<T>::up(in.e[0]);
  }
}
template <class T, int VEC, int N>
__device__ __forceinline__ void store(T* dst, int p, const Pairs<N>& f) {
  Piece<T, VEC> out;
  if constexpr (VEC % 2 == 0) {
    auto* two = reinterpret_cast<typename Two<T>::type*>(out.e);
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) narrow2(two[i], f.v[p * VEC / 2 + i]);
  } else {
    out.e[0] = Elem<T>::down((p & 1) ? f.v[p / 2].y : f.v[p / 2].x);
  }
  *reinterpret_cast<Piece<T, VEC>*>(dst) = out;
}
__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }
template <class T>
__device__ __forceinline__ float param(const void* p, bool wide, int64_t i) {
  return wide ? reinterpret_cast<const float*>(p)[i] : Elem<T>::up(reinterpret_cast<const T*>(p)[i]);
}

// Elements c .. c + VEC - 1 of a parameter as piece p; 16 bytes at a time where the caller says that they lie on them
template <class T, int VEC, int N>
__device__ __forceinline__ void params(Pairs<N>& f, int p, const void* src, bool wide, bool aligned, int64_t c, int64_t n, float otherwise) {
  if (VEC >= 4 && aligned && c < n && src != nullptr) {
    if (!wide) {
      widen<T, VEC, N>(f, p, raw_piece<T, VEC>(reinterpret_cast<const T*>(src) + c, true));
    } else {
#pragma unroll
      for (int i = 0; i < VEC; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(src) + c + i);
        f.v[(p * VEC + i) / 2] = make_float2(v.x, v.y);
        if constexpr (VEC >= 4) f.v[(p * VEC + i) / 2 + 1] = make_float2(v.z, v.w);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float& x = ((p * VEC + i) & 1) ? f.v[(p * VEC + i) / 2].y : f.v[(p * VEC + i) / 2].x;
    x = src != nullptr && c + i < n ? param<T>(src, wide, c + i) : otherwise;
  }
}

// U sums over the TPR threads of a group, every thread gets them.  With more than a warp to a group, all threads of the CTA call it and
// `smem` ([U][warps]) may be used again behind the next call's first barrier, so two calls in a row take two buffers.
template <int TPR, int U>
__device__ __forceinline__ void group_sum(float (&x)[U], float* smem) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] += __shfl_xor_sync(0xffffffffu, x[u], o);
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int warp = threadIdx.x >> 5, first = warp / W * W;
    const int warps = blockDim.x >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int u = 0; u < U; ++u) smem[u * warps + warp] = x[u];
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += smem[u * warps + first + w];
      x[u] = s;
    }
  }
}

template <class T, int VEC, int TPR, int P, int U>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) layer_norm_kernel(const AveLayerNormArgs a, bool aligned) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR, N = P * VEC, H = Pairs<N>::H;
  __shared__ float sums[2][U * 32];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const T* x = reinterpret_cast<const T*>(a.x);
  T* y = reinterpret_cast<T*>(a.y);
  pdl_wait();
  // the weights stay in registers, where a thread has few columns
  constexpr bool kKept = N <= 16;
  Pairs<kKept ? N : 1> w, b;
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
  if constexpr (kKept) {
    b.fill(0.f);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      params<T, VEC>(w, p, a.weight, wide, aligned, (int64_t)(p * TPR + sub) * VEC, a.n, 1.f);
      params<T, VEC>(b, p, a.bias, wide, aligned, (int64_t)(p * TPR + sub) * VEC, a.n, 0.f);
    }
  }
  const float inv_n = 1.f / (float)a.n;
  const int64_t step = (int64_t)gridDim.x * GROUPS * U;
  for (int64_t r0 = (int64_t)blockIdx.x * GROUPS * U; r0 < a.rows; r0 += step) {
    Piece<T, VEC> in[U][P];
    Pairs<N> f[U];
    float s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * GROUPS + group;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t c = (int64_t)(p * TPR + sub) * VEC;
        in[u][p] = raw_piece<T, VEC>(x + r * a.x_stride + c, r < a.rows && c < a.n);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      f[u].fill(0.f);
#pragma unroll
      for (int p = 0; p < P; ++p) widen<T, VEC, N>(f[u], p, in[u][p]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float2 t = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < H; ++i) t = __fadd2_rn(t, f[u].v[i]);
      s[u] = t.x + t.y;
    }
    group_sum<TPR, U>(s, sums[0]);
    float mean[U], q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // the squares are of differences from the mean: the sum of x^2 would lose what a large mean hides
      mean[u] = s[u] * inv_n;
      float2 t = make_float2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        float2 d = __fadd2_rn(f[u].v[i], splat(-mean[u]));
        if constexpr (VEC % 2 == 0) {
          if ((int64_t)(2 * i / VEC * TPR + sub) * VEC >= a.n) d = make_float2(0.f, 0.f);
        } else {
          if ((int64_t)(2 * i) * TPR + sub >= a.n) d.x = 0.f;
          if (2 * i + 1 >= N || (int64_t)(2 * i + 1) * TPR + sub >= a.n) d.y = 0.f;
        }
        f[u].v[i] = d;
        t = __ffma2_rn(d, d, t);
      }
      q[u] = t.x + t.y;
    }
    group_sum<TPR, U>(q, sums[1]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * GROUPS + group;
      if (r >= a.rows) continue;
      const float rstd = 1.f / sqrtf(q[u] * inv_n + a.eps);
      if (sub == 0) {
        if (a.mean != nullptr) a.mean[r] = mean[u];
        if (a.rstd != nullptr) a.rstd[r] = rstd;
      }
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float2 h = __fmul2_rn(f[u].v[i], splat(rstd));
        f[u].v[i] = kKept ? __ffma2_rn(h, w.v[kKept ? i : 0], b.v[kKept ? i : 0]) : h;
      }
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t c = (int64_t)(p * TPR + sub) * VEC;
        if (c >= a.n) continue;
        if constexpr (!kKept) {
          Pairs<VEC> wp, bp;
          bp.fill(0.f); wp.fill(1.f);
          params<T, VEC>(wp, 0, a.weight, wide, aligned, c, a.n, 1.f);
          params<T, VEC>(bp, 0, a.bias, wide, aligned, c, a.n, 0.f);
          if constexpr (VEC % 2 == 0) {
#pragma unroll
            for (int i = 0; i < VEC / 2; ++i) f[u].v[p * VEC / 2 + i] = __ffma2_rn(f[u].v[p * VEC / 2 + i], wp.v[i], bp.v[i]);
          } else {
            float& e = (p & 1) ? f[u].v[p / 2].y : f[u].v[p / 2].x;
            e = fmaf(e, wp.v[0].x, bp.v[0].x);
          }
        }
        store<T, VEC, N>(y + r * a.y_stride + c, p, f[u]);
      }
    }
  }
}

// Rows through a ring in shared memory: one CTA an SM, whose eight warps are 8 / G groups of G warps with a ring of `depth` rows each, filled by asynchronous copies, so that what is on
// its way does not depend on registers, and a thread's columns (P pieces) keep their weights, and in the backward pass their sums, in registers.  (131072 x 2048 bf16: forward 179 us; with
// rows in registers 296 us with eight warps a row, 230 with a warp a row, 352 with a warp a row and the next row fetched ahead, for which too few warps fit.  Backward 267; 418 in registers.)
// The groups meet at hardware barriers, whose waits have no limit, so a warp whose wait for a copy has expired goes on with the others.
constexpr int RING = 204800;  // bytes
template <int G>
__device__ __forceinline__ void group_barrier() {
  if constexpr (G > 1) asm volatile("bar.sync %0, %1;" ::"r"(1 + (int)(threadIdx.x >> 5) / G), "r"(32 * G) : "memory");
  else __syncwarp();
}
// N sums over the group, everybody gets them; `sm`: [N][8 warps]
template <int G, int N>
__device__ __forceinline__ void ring_sum(float (&x)[N], float* sm) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += __shfl_xor_sync(0xffffffffu, x[i], o);
  if constexpr (G > 1) {
    const int warp = threadIdx.x >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) sm[8 * i + warp] = x[i];
    group_barrier<G>();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float t = 0.f;
#pragma unroll
      for (int w = 0; w < G; ++w) t += sm[8 * i + warp / G * G + w];
      x[i] = t;
    }
  }
}
// The copies of a group's rows: `rows` arrays of n elements each a slot
template <class T, int G, int ARRAYS>
struct Ring {
  uint8_t* base;
  uint64_t* bars;
  uint32_t* flag;
  int depth, slot_bytes, row_bytes;
  bool leader, dead = false;
  int issued = 0, waited = 0, slot = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ float own(float sum) const { return dead ? __int_as_float(0x7fffffff) : sum; }  // what the thread adds to its row's sum
  __device__ __forceinline__ void issue(const T* a, const T* b) {  // into the slot that is free next
    if (leader && !dead) {
      const int s = issued % depth;
      uint64_t* bar = bars + s;
      tc::mbar_expect_tx(bar, (uint32_t)(ARRAYS * row_bytes));
      tc::bulk_load(base + s * slot_bytes, a, (uint32_t)row_bytes, bar);
      if constexpr (ARRAYS == 2) tc::bulk_load(base + s * slot_bytes + slot_bytes / 2, b, (uint32_t)row_bytes, bar);
    }
    ++issued;
  }
  // A wait that expires leaves the thread `dead`: from then on it adds NaN to its rows' sums, which makes them NaN for the whole group, it issues
  // nothing more, and the copies on their way are waited for once more, with a limit.
  __device__ __forceinline__ const uint8_t* wait() {
    if (!dead && !tc::mbar_wait(bars + slot, phase, flag)) {
      dead = true;
      if (leader)
        for (int i = 0; i < issued - waited; ++i) tc::drain(bars + (slot + i) % depth, slot + i < depth ? phase : phase ^ 1u);
    }
    return base + slot * slot_bytes;
  }
  __device__ __forceinline__ void report(uint32_t* status) const {  // behind all rows (where the wait expires, in their loop, 131072 x 2048 took 197 us, 193 to 194 here)
    if (dead && status != nullptr) atomicOr(status, AVE_GDN_DEV_WAIT_EXPIRED);
  }
  __device__ __forceinline__ void next() {
    ++waited;
    if (++slot == depth) { slot = 0; phase ^= 1u; }
  }
};
template <class T, int G, int ARRAYS>
__device__ __forceinline__ Ring<T, G, ARRAYS> make_ring(uint8_t* smem, uint64_t* bars, uint32_t* flag, int64_t n, int depth) {
  const int group = (int)(threadIdx.x >> 5) / G;
  Ring<T, G, ARRAYS> r;
  r.depth = depth;
  r.row_bytes = (int)(n * (int64_t)sizeof(T));
  r.slot_bytes = ARRAYS * ((r.row_bytes + 127) & ~127);
  r.base = smem + (size_t)group * depth * r.slot_bytes;
  r.bars = bars + 8 * group;
  r.flag = flag;
  r.leader = threadIdx.x % (32 * G) == 0;
  return r;
}

template <class T, int P, int G>
__global__ void __launch_bounds__(256, 1) layer_norm_ring_kernel(const AveLayerNormArgs a, int depth, bool aligned) {
  constexpr int VEC = 16 / sizeof(T), N = P * VEC, H = N / 2, GROUPS = 8 / G;
  extern __shared__ __align__(128) uint8_t ring_mem[];
  __shared__ float sums[2][2][8];
  __shared__ uint64_t bars[64];
  __shared__ uint32_t flag;
  const int sub = threadIdx.x % (32 * G), group = (int)(threadIdx.x >> 5) / G;
  const T* x = reinterpret_cast<const T*>(a.x);
  T* y = reinterpret_cast<T*>(a.y);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 64; ++i) tc::mbar_init(bars + i, 1);
    flag = 0;
    tc::fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  Ring<T, G, 1> ring = make_ring<T, G, 1>(ring_mem, bars, &flag, a.n, depth);
  const int64_t first = (int64_t)blockIdx.x * GROUPS + group, step = (int64_t)gridDim.x * GROUPS;
  int64_t ahead = first;
  for (int i = 0; i < depth && ahead < a.rows; ++i, ahead += step) ring.issue(x + ahead * a.x_stride, nullptr);
  Pairs<N> w, b;
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
  w.fill(1.f); b.fill(0.f);
#pragma unroll
  for (int p = 0; p < P; ++p) {
    params<T, VEC>(w, p, a.weight, wide, aligned, (int64_t)(p * 32 * G + sub) * VEC, a.n, 1.f);
    params<T, VEC>(b, p, a.bias, wide, aligned, (int64_t)(p * 32 * G + sub) * VEC, a.n, 0.f);
  }
  const float inv_n = 1.f / (float)a.n;
  const int n = (int)a.n;
  for (int64_t r = first; r < a.rows; r += step) {
    const T* row = reinterpret_cast<const T*>(ring.wait());
    Pairs<N> f;
    f.fill(0.f);
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = (p * 32 * G + sub) * VEC;
      if (c < n) widen<T, VEC, N>(f, p, *reinterpret_cast<const Piece<T, VEC>*>(row + c));
    }
    float2 t = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < H; ++i) t = __fadd2_rn(t, f.v[i]);
    float s[1] = {ring.own(t.x + t.y)};
    ring_sum<G, 1>(s, sums[0][0]);
    __syncwarp();  // the whole group has read the row
    if (ahead < a.rows) { ring.issue(x + ahead * a.x_stride, nullptr); ahead += step; }
    ring.next();
    const float mean = s[0] * inv_n;
    t = make_float2(0.f, 0.f);
#pragma unroll
    for (int p = 0; p < P; ++p)  // the squares are of differences from the mean: the sum of x^2 would lose what a large mean hides
      if ((p * 32 * G + sub) * VEC < n) {
#pragma unroll
        for (int i = p * VEC / 2; i < (p + 1) * VEC / 2; ++i) {
          f.v[i] = __fadd2_rn(f.v[i], splat(-mean));
          t = __ffma2_rn(f.v[i], f.v[i], t);
        }
      }
    s[0] = t.x + t.y;
    ring_sum<G, 1>(s, sums[1][0]);
    const float rstd = 1.f / sqrtf(s[0] * inv_n + a.eps);
    if (sub == 0) {
      if (a.mean != nullptr) a.mean[r] = mean;
      if (a.rstd != nullptr) a.rstd[r] = rstd;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = (p * 32 * G + sub) * VEC;
      if (c >= n) continue;
#pragma unroll
      for (int i = p * VEC / 2; i < (p + 1) * VEC / 2; ++i) f.v[i] = __ffma2_rn(__fmul2_rn(f.v[i], splat(rstd)), w.v[i], b.v[i]);
      store<T, VEC, N>(y + r * a.y_stride + c, p, f);
    }
  }
  ring.report(a.status);
}

// Sums of CTA c: partial[c][0][n] of dy xh, partial[c][1][n] of dy
template <class T, int VEC, int TPR, int P, int U>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) layer_norm_backward_kernel(const AveLayerNormBwdArgs a, float* partial, bool aligned) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR, N = P * VEC, H = Pairs<N>::H;
  __shared__ float sums[2][2 * U * 32];
  extern __shared__ float cols[];  // [GROUPS][2][TPR * P * VEC], with several groups to a CTA
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const T *x = reinterpret_cast<const T*>(a.x), *dy = reinterpret_cast<const T*>(a.d_y);
  T* dx = reinterpret_cast<T*>(a.d_x);
  pdl_wait();
  Pairs<N> w, dw, db;
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
  w.fill(1.f);
#pragma unroll
  for (int p = 0; p < P; ++p) params<T, VEC>(w, p, a.weight, wide, aligned, (int64_t)(p * TPR + sub) * VEC, a.n, 1.f);
  dw.fill(0.f); db.fill(0.f);
  const float inv_n = 1.f / (float)a.n;
  const int64_t step = (int64_t)gridDim.x * GROUPS * U;
  int turn = 0;
  // the next rows are on their way while these are reduced (where they fit: with many elements a thread the registers are the row's)
  constexpr bool kAhead = N <= 16;
  Piece<T, VEC> x_in[U][P], d_in[U][P];
  float m_in[U], r_in[U];
  auto fetch = [&](int64_t r0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * GROUPS + group;
      const bool there = r < a.rows;
      m_in[u] = there ? a.mean[r] : 0.f;
      r_in[u] = there ? a.rstd[r] : 0.f;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t c = (int64_t)(p * TPR + sub) * VEC;
        x_in[u][p] = raw_piece<T, VEC>(x + r * a.x_stride + c, there && c < a.n);
        d_in[u][p] = raw_piece<T, VEC>(dy + r * a.dy_stride + c, there && c < a.n);
      }
    }
  };
  const int64_t first = (int64_t)blockIdx.x * GROUPS * U;
  if (kAhead && first < a.rows) fetch(first);
  for (int64_t r0 = first; r0 < a.rows; r0 += step, turn ^= 1) {
    Pairs<N> xh[U], d[U];
    float s[2 * U], rstd[U], mean[U];
    if (!kAhead) fetch(r0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mean[u] = m_in[u];
      rstd[u] = r_in[u];
      xh[u].fill(0.f); d[u].fill(0.f);
#pragma unroll
      for (int p = 0; p < P; ++p) { widen<T, VEC, N>(xh[u], p, x_in[u][p]); widen<T, VEC, N>(d[u], p, d_in[u][p]); }
    }
    if (kAhead && r0 + step < a.rows) fetch(r0 + step);
#pragma unroll
    for (int u = 0; u < U; ++u) {  // (columns behind the row have dy = 0, so that what xh is there does not matter)
      float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
      for (int i = 0; i < H; ++i) {
        const float2 h = __fmul2_rn(__fadd2_rn(xh[u].v[i], splat(-mean[u])), splat(rstd[u])), g = d[u].v[i];
        dw.v[i] = __ffma2_rn(g, h, dw.v[i]);
        db.v[i] = __fadd2_rn(db.v[i], g);
        const float2 gw = __fmul2_rn(g, w.v[i]);
        s0 = __fadd2_rn(s0, gw);
        s1 = __ffma2_rn(gw, h, s1);
        xh[u].v[i] = h;
        d[u].v[i] = gw;
      }
      s[2 * u] = s0.x + s0.y;
      s[2 * u + 1] = s1.x + s1.y;
    }
    group_sum<TPR, 2 * U>(s, sums[turn]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * GROUPS + group;
      if (r >= a.rows) continue;
      const float c1 = s[2 * u] * inv_n, c2 = s[2 * u + 1] * inv_n;
#pragma unroll
      for (int i = 0; i < H; ++i)
        d[u].v[i] = __fmul2_rn(splat(rstd[u]), __ffma2_rn(xh[u].v[i], splat(-c2), __fadd2_rn(d[u].v[i], splat(-c1))));
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t c = (int64_t)(p * TPR + sub) * VEC;
        if (c < a.n) store<T, VEC, N>(dx + r * a.dx_stride + c, p, d[u]);
      }
    }
  }
  if (partial == nullptr) return;
  float* out = partial + (int64_t)blockIdx.x * 2 * a.n;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int64_t c = (int64_t)(p * TPR + sub) * VEC + i;
        const int e = p * VEC + i;
        if (c < a.n) { out[c] = e & 1 ? dw.v[e / 2].y : dw.v[e / 2].x; out[a.n + c] = e & 1 ? db.v[e / 2].y : db.v[e / 2].x; }
      }
  } else {
    constexpr int C = TPR * P * VEC;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = (p * TPR + sub) * VEC + i;
        const int e = p * VEC + i;
        cols[group * 2 * C + c] = e & 1 ? dw.v[e / 2].y : dw.v[e / 2].x;
        cols[group * 2 * C + C + c] = e & 1 ? db.v[e / 2].y : db.v[e / 2].x;
      }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * C; e += THREADS) {
      float t = 0.f;
      for (int g = 0; g < GROUPS; ++g) t += cols[g * 2 * C + e];
      const int c = e % C;
      if (c < a.n) out[(e / C) * a.n + c] = t;
    }
  }
}

// The same for the gradients: a slot holds a row of x and one of dy
template <class T, int P, int G>
__global__ void __launch_bounds__(256, 1) layer_norm_backward_ring_kernel(const AveLayerNormBwdArgs a, float* partial, int depth, bool aligned) {
  constexpr int VEC = 16 / sizeof(T), N = P * VEC, H = N / 2, GROUPS = 8 / G;
  extern __shared__ __align__(128) uint8_t ring_mem[];
  __shared__ float sums[2][2][8];
  __shared__ uint64_t bars[64];
  __shared__ uint32_t flag;
  const int sub = threadIdx.x % (32 * G), group = (int)(threadIdx.x >> 5) / G;
  const T *x = reinterpret_cast<const T*>(a.x), *dy = reinterpret_cast<const T*>(a.d_y);
  T* dx = reinterpret_cast<T*>(a.d_x);
  if (threadIdx.x == 0) {
    for (int i = 0; i < 64; ++i) tc::mbar_init(bars + i, 1);
    flag = 0;
    tc::fence_barrier_init();
  }
  __syncthreads();
  pdl_wait();
  Ring<T, G, 2> ring = make_ring<T, G, 2>(ring_mem, bars, &flag, a.n, depth);
  const int64_t first = (int64_t)blockIdx.x * GROUPS + group, step = (int64_t)gridDim.x * GROUPS;
  int64_t ahead = first;
  for (int i = 0; i < depth && ahead < a.rows; ++i, ahead += step) ring.issue(x + ahead * a.x_stride, dy + ahead * a.dy_stride);
  Pairs<N> w, dw, db;
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
  w.fill(1.f); dw.fill(0.f); db.fill(0.f);
#pragma unroll
  for (int p = 0; p < P; ++p) params<T, VEC>(w, p, a.weight, wide, aligned, (int64_t)(p * 32 * G + sub) * VEC, a.n, 1.f);
  const float inv_n = 1.f / (float)a.n;
  const int n = (int)a.n;
  float mean_next = first < a.rows ? a.mean[first] : 0.f, rstd_next = first < a.rows ? a.rstd[first] : 0.f;
  int turn = 0;
  for (int64_t r = first; r < a.rows; r += step, turn ^= 1) {
    const float mean = mean_next, rstd = rstd_next;
    if (r + step < a.rows) { mean_next = a.mean[r + step]; rstd_next = a.rstd[r + step]; }
    const uint8_t* slot = ring.wait();
    const T *row = reinterpret_cast<const T*>(slot), *grow = reinterpret_cast<const T*>(slot + ring.slot_bytes / 2);
    Pairs<N> xh, d;
    xh.fill(0.f); d.fill(0.f);
    float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = (p * 32 * G + sub) * VEC;
      if (c >= n) continue;
      widen<T, VEC, N>(xh, p, *reinterpret_cast<const Piece<T, VEC>*>(row + c));
      widen<T, VEC, N>(d, p, *reinterpret_cast<const Piece<T, VEC>*>(grow + c));
#pragma unroll
      for (int i = p * VEC / 2; i < (p + 1) * VEC / 2; ++i) {
        const float2 h = __fmul2_rn(__fadd2_rn(xh.v[i], splat(-mean)), splat(rstd)), g = d.v[i];
        dw.v[i] = __ffma2_rn(g, h, dw.v[i]);
        db.v[i] = __fadd2_rn(db.v[i], g);
        const float2 gw = __fmul2_rn(g, w.v[i]);
        s0 = __fadd2_rn(s0, gw);
        s1 = __ffma2_rn(gw, h, s1);
        xh.v[i] = h;
        d.v[i] = gw;
      }
    }
    float s[2] = {ring.own(s0.x + s0.y), ring.own(s1.x + s1.y)};
    ring_sum<G, 2>(s, sums[turn][0]);
    __syncwarp();  // the whole group has read the rows
    if (ahead < a.rows) { ring.issue(x + ahead * a.x_stride, dy + ahead * a.dy_stride); ahead += step; }
    ring.next();
    const float c1 = s[0] * inv_n, c2 = s[1] * inv_n;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = (p * 32 * G + sub) * VEC;
      if (c >= n) continue;
#pragma unroll
      for (int i = p * VEC / 2; i < (p + 1) * VEC / 2; ++i)
        d.v[i] = __fmul2_rn(splat(rstd), __ffma2_rn(xh.v[i], splat(-c2), __fadd2_rn(d.v[i], splat(-c1))));
      store<T, VEC, N>(dx + r * a.dx_stride + c, p, d);
    }
  }
  ring.report(a.status);
  if (partial == nullptr) return;
  if (ring.dead) { dw.fill(__int_as_float(0x7fffffff)); db.fill(__int_as_float(0x7fffffff)); }
  __syncthreads();  // all rows are done: the ring's memory takes the groups' sums, [GROUPS][2][n]
  float* cols = reinterpret_cast<float*>(ring_mem);
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = (p * 32 * G + sub) * VEC;
    if (c >= n) continue;
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) {
      *reinterpret_cast<float2*>(cols + (size_t)group * 2 * n + c + 2 * i) = dw.v[p * VEC / 2 + i];
      *reinterpret_cast<float2*>(cols + (size_t)group * 2 * n + n + c + 2 * i) = db.v[p * VEC / 2 + i];
    }
  }
  __syncthreads();
  float* out = partial + (int64_t)blockIdx.x * 2 * a.n;
  for (int e = threadIdx.x; e < 2 * n; e += 256) {
    float t = 0.f;
    for (int g = 0; g < GROUPS; ++g) t += cols[(size_t)g * 2 * n + e];
    out[e] = t;
  }
}

// Long rows: five numbers a column are more than the register file holds, so the column sums lie in shared memory (each thread's own place), the weights are read for every row, and the row
// stays as it was read.  (16384 rows of 16384 bf16: 567 us; 7.6 ms with everything in registers, which spill.  The longest still do, at 1024 threads: up to 184 bytes stored a thread above 24576 columns, up to
// 432 above 16384 off 16 bytes.  8192 rows, forward and backward us: of 20480 bf16 283 and 412, of 28672 334 and 590, fp32 369 and 882; off 16 bytes of 16383 250 and 602, 4096 of 28671 264 and 825.)
template <class T, int VEC, int P>
__global__ void __launch_bounds__(1024) layer_norm_backward_long_kernel(const AveLayerNormBwdArgs a, float* partial, bool aligned) {
  constexpr int TPR = 1024, HV = Pairs<VEC>::H;
  using A = typename std::conditional<VEC % 2 == 0, float2, float>::type;
  __shared__ float sums[2][2 * 32];
  extern __shared__ float2 acc_mem[];
  A* acc = reinterpret_cast<A*>(acc_mem);  // [2][P HV][TPR]: sums of dy xh, sums of dy
  const int sub = threadIdx.x;
  const T *x = reinterpret_cast<const T*>(a.x), *dy = reinterpret_cast<const T*>(a.d_y);
  T* dx = reinterpret_cast<T*>(a.d_x);
  pdl_wait();
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
#pragma unroll
  for (int i = 0; i < 2 * P * HV; ++i) acc[i * TPR + sub] = A{};
  const float inv_n = 1.f / (float)a.n;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
    Piece<T, VEC> x_in[P], d_in[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int64_t c = (int64_t)(p * TPR + sub) * VEC;
      x_in[p] = raw_piece<T, VEC>(x + r * a.x_stride + c, c < a.n);
      d_in[p] = raw_piece<T, VEC>(dy + r * a.dy_stride + c, c < a.n);
    }
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s[2] = {0.f, 0.f};
    Pairs<VEC> xh, d, w;
    auto piece = [&](int p) {
      xh.fill(0.f); d.fill(0.f); w.fill(1.f);
      widen<T, VEC, VEC>(xh, 0, x_in[p]);
      widen<T, VEC, VEC>(d, 0, d_in[p]);
      params<T, VEC>(w, 0, a.weight, wide, aligned, (int64_t)(p * TPR + sub) * VEC, a.n, 1.f);
#pragma unroll
      for (int i = 0; i < HV; ++i) xh.v[i] = __fmul2_rn(__fadd2_rn(xh.v[i], splat(-mean)), splat(rstd));
    };
#pragma unroll
    for (int p = 0; p < P; ++p) {
      piece(p);
      float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
      for (int i = 0; i < HV; ++i) {
        A* at = acc + (p * HV + i) * TPR + sub;
        if constexpr (VEC % 2 == 0) {
          at[0] = __ffma2_rn(d.v[i], xh.v[i], at[0]);
          at[P * HV * TPR] = __fadd2_rn(d.v[i], at[P * HV * TPR]);
        } else {
          at[0] = fmaf(d.v[i].x, xh.v[i].x, at[0]);
          at[P * HV * TPR] += d.v[i].x;
        }
        const float2 gw = __fmul2_rn(d.v[i], w.v[i]);
        s0 = __fadd2_rn(s0, gw);
        s1 = __ffma2_rn(gw, xh.v[i], s1);
      }
      s[0] += s0.x + s0.y;
      s[1] += s1.x + s1.y;
    }
    group_sum<TPR, 2>(s, sums[turn]);
    const float c1 = s[0] * inv_n, c2 = s[1] * inv_n;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int64_t c = (int64_t)(p * TPR + sub) * VEC;
      if (c >= a.n) continue;
      piece(p);
#pragma unroll
      for (int i = 0; i < HV; ++i)
        d.v[i] = __fmul2_rn(splat(rstd), __ffma2_rn(xh.v[i], splat(-c2), __ffma2_rn(d.v[i], w.v[i], splat(-c1))));
      store<T, VEC, VEC>(dx + r * a.dx_stride + c, 0, d);
    }
  }
  if (partial == nullptr) return;
  float* out = partial + (int64_t)blockIdx.x * 2 * a.n;
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int64_t c = (int64_t)(p * TPR + sub) * VEC + i;
      if (c >= a.n) continue;
      const A g = acc[(p * HV + i / 2) * TPR + sub], b = acc[(P * HV + p * HV + i / 2) * TPR + sub];
      if constexpr (VEC % 2 == 0) {
        out[c] = i & 1 ? g.y : g.x;
        out[a.n + c] = i & 1 ? b.y : b.x;
      } else {
        out[c] = g;
        out[a.n + c] = b;
      }
    }
}

// Adds the CTAs' sums: 32 columns a CTA, eight warps take every eighth row of sums
template <class T>
__global__ void __launch_bounds__(256) layer_norm_columns_kernel(const AveLayerNormBwdArgs a, const float* partial, int parts) {
  __shared__ float part[8][33];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;  // column of [dw | db]
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  if (c < 2 * a.n) {
    int i = warp;
    for (; i + 24 < parts; i += 32) {
      s0 += partial[(int64_t)i * 2 * a.n + c];
      s1 += partial[(int64_t)(i + 8) * 2 * a.n + c];
      s2 += partial[(int64_t)(i + 16) * 2 * a.n + c];
      s3 += partial[(int64_t)(i + 24) * 2 * a.n + c];
    }
    for (; i < parts; i += 8) s0 += partial[(int64_t)i * 2 * a.n + c];
  }
  part[warp][lane] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  if (warp != 0 || c >= 2 * a.n) return;
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) s += part[k][lane];
  void* dst = c < a.n ? a.d_weight : a.d_bias;
  const int64_t at = c < a.n ? c : c - a.n;
  if (dst == nullptr) return;
  if (a.w_dtype == AVE_DTYPE_FP32) reinterpret_cast<float*>(dst)[at] = s;
  else reinterpret_cast<T*>(dst)[at] = Elem<T>::down(s);
}

constexpr int BWD_CTAS = 148 * 3;
constexpr int64_t MAX_N = 28672;  // the gradients' column sums of a row, 8 bytes a column, lie in an SM's shared memory

inline int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

bool params_aligned(const void* w, const void* b) { return aligned16(w) && aligned16(b); }

template <class K>
int ctas_an_sm(K kernel, int threads, size_t smem) {
  int per = 1;
  return cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kernel, threads, smem) == cudaSuccess && per > 0 ? per : 1;
}

template <class T, int VEC, int TPR, int P, int U>
int run_forward(const AveLayerNormArgs& a, cudaStream_t stream) {
  constexpr int THREADS = TPR > 256 ? TPR : 256;
  const int64_t rows_cta = (int64_t)(THREADS / TPR) * U, ctas = (a.rows + rows_cta - 1) / rows_cta;
  static const int per = ctas_an_sm(layer_norm_kernel<T, VEC, TPR, P, U>, THREADS, 0);  // one wave, so that a CTA reads its weights once
  const int64_t most = (int64_t)sm_count() * per;
  AVE_CUDA_TRY(launch_after(layer_norm_kernel<T, VEC, TPR, P, U>, (unsigned)(ctas < most ? ctas : most), THREADS, 0, stream, a, params_aligned(a.weight, a.bias)));
  return AVE_GDN_OK;
}
// A ring's grid, its depth (as many rows as the shared memory holds or the group meets, eight at most), and its bytes
struct RingShape { int grid, depth, smem; };
inline RingShape ring_shape(int64_t rows, int64_t row_bytes, int arrays, int groups) {
  const int64_t slot = arrays * ((row_bytes + 127) & ~(int64_t)127), ctas = (rows + groups - 1) / groups, most = sm_count() < 148 ? sm_count() : 148;
  const int64_t grid = ctas < most ? ctas : most, turns = (rows + grid * groups - 1) / (grid * groups);
  int64_t depth = RING / (slot * groups);
  depth = depth < 8 ? depth : 8;
  depth = depth < turns ? depth : turns;
  return {(int)grid, (int)depth, (int)(depth * slot * groups)};
}
template <class T, int P, int G>
int run_forward_ring(const AveLayerNormArgs& a, cudaStream_t stream) {
  constexpr auto* kernel = &layer_norm_ring_kernel<T, P, G>;
  const int rc = allow_smem<kernel>(RING);
  if (rc != AVE_GDN_OK) return rc;
  const RingShape r = ring_shape(a.rows, a.n * (int64_t)sizeof(T), 1, 8 / G);
  AVE_CUDA_TRY(launch_after(kernel, (unsigned)r.grid, 256, (size_t)r.smem, stream, a, r.depth, params_aligned(a.weight, a.bias)));
  return AVE_GDN_OK;
}
template <class T, int P, int G>
int run_backward_ring(const AveLayerNormBwdArgs& a, cudaStream_t stream) {
  constexpr auto* kernel = &layer_norm_backward_ring_kernel<T, P, G>;
  const int rc = allow_smem<kernel>(RING);
  if (rc != AVE_GDN_OK) return rc;
  const RingShape r = ring_shape(a.rows, a.n * (int64_t)sizeof(T), 2, 8 / G);
  const int64_t cols = (int64_t)(8 / G) * 2 * a.n * 4;  // the groups' sums, at the end
  const bool sums = a.d_weight != nullptr || a.d_bias != nullptr;
  float* partial = sums ? reinterpret_cast<float*>(a.workspace) : nullptr;
  AVE_CUDA_TRY(launch_after(kernel, (unsigned)r.grid, 256, (size_t)(cols > r.smem ? cols : r.smem), stream, a, partial, r.depth, params_aligned(a.weight, nullptr)));
  if (sums) AVE_CUDA_TRY(launch_after(layer_norm_columns_kernel<T>, (unsigned)((2 * a.n + 31) / 32), 256, 0, stream, a, (const float*)partial, r.grid));
  return AVE_GDN_OK;
}

template <class T, int VEC, int TPR, int P, int U>
int run_backward(const AveLayerNormBwdArgs& a, cudaStream_t stream) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
  const size_t smem = GROUPS > 1 ? (size_t)GROUPS * 2 * TPR * P * VEC * 4 : 0;
  static_assert(GROUPS == 1 || (size_t)GROUPS * 2 * TPR * P * VEC * 4 <= 48 * 1024 - 2048, "column sums in the default shared memory");
  const int64_t rows_cta = (int64_t)GROUPS * U, ctas = (a.rows + rows_cta - 1) / rows_cta;
  static const int per = ctas_an_sm(layer_norm_backward_kernel<T, VEC, TPR, P, U>, THREADS, smem);
  int64_t most = (int64_t)sm_count() * per;
  if (most > BWD_CTAS) most = BWD_CTAS;
  const int grid = (int)(ctas < most ? ctas : most);
  const bool sums = a.d_weight != nullptr || a.d_bias != nullptr;
  float* partial = sums ? reinterpret_cast<float*>(a.workspace) : nullptr;
  AVE_CUDA_TRY(launch_after(layer_norm_backward_kernel<T, VEC, TPR, P, U>, (unsigned)grid, THREADS, smem, stream, a, partial, params_aligned(a.weight, nullptr)));
  if (sums) AVE_CUDA_TRY(launch_after(layer_norm_columns_kernel<T>, (unsigned)((2 * a.n + 31) / 32), 256, 0, stream, a, (const float*)partial, grid));
  return AVE_GDN_OK;
}

template <class T, int VEC, int P>
int run_backward_long(const AveLayerNormBwdArgs& a, cudaStream_t stream) {
  constexpr auto* kernel = &layer_norm_backward_long_kernel<T, VEC, P>;
  constexpr int smem = 2 * P * VEC * 4 * 1024;
  static_assert(smem <= 232448 - 1024, "shared memory of an SM");
  const int rc = allow_smem<kernel>(smem);
  if (rc != AVE_GDN_OK) return rc;
  const int64_t most = sm_count();
  const int grid = (int)(a.rows < most ? a.rows : most);
  const bool sums = a.d_weight != nullptr || a.d_bias != nullptr;
  float* partial = sums ? reinterpret_cast<float*>(a.workspace) : nullptr;
  AVE_CUDA_TRY(launch_after(kernel, (unsigned)grid, 1024, smem, stream, a, partial, params_aligned(a.weight, nullptr)));
  if (sums) AVE_CUDA_TRY(launch_after(layer_norm_columns_kernel<T>, (unsigned)((2 * a.n + 31) / 32), 256, 0, stream, a, (const float*)partial, grid));
  return AVE_GDN_OK;
}

// Threads a row and pieces a thread by the row's length; `f` is called with them and the rows in flight.
template <int TPR, int P, int U> struct Form { static constexpr int tpr = TPR, p = P, u = U; };
template <int VEC, class F>
int short_rows(int64_t n, F f) {  // up to 512 columns, whole pieces
  const int64_t pieces = n / VEC;
  if (pieces <= 8) return f(Form<8, 1, 2>());
  if (pieces <= 32) return f(Form<32, 1, 4>());
  if (VEC == 8 || pieces <= 64) return f(Form<32, 2, 2>());
  if constexpr (VEC == 4) return f(Form<256, 1, 4>());
  return AVE_GDN_UNSUPPORTED;
}
template <bool kLong, class F>
int by_element(int64_t n, F f) {
  if (n <= 8) return f(Form<8, 1, 2>());
  if (n <= 32) return f(Form<32, 1, 4>());
  if (n <= 64) return f(Form<32, 2, 2>());
  if (n <= 256) return f(Form<256, 1, 4>());
  if (n <= 512) return f(Form<256, 2, 2>());
  if (n <= 1024) return f(Form<256, 4, 2>());
  if (n <= 2048) return f(Form<256, 8, 1>());
  if constexpr (kLong) {
    if (n <= 4096) return f(Form<1024, 4, 1>());
    if (n <= 8192) return f(Form<1024, 8, 1>());
    if (n <= 16384) return f(Form<1024, 16, 1>());
    if (n <= MAX_N) return f(Form<1024, 28, 1>());
  }
  return AVE_GDN_UNSUPPORTED;
}
// Few rows: a row a CTA, two at most one behind the other.  (bf16 rows of 2048, forward and backward us: 37 rows 2.2 and 4.9, with a row a warp or two 4.1 and 6.0; 296 rows
// 3.1 and 6.3, 4.3 and 7.1; 592 rows 4.6 and 7.7, 4.3 and 7.6; 8192 rows 48 and 46, 14 and 25.)
bool few_rows(int64_t rows) { return rows <= 2 * 148; }
bool on16(int64_t stride, int size) { return (stride * size) % 16 == 0; }

template <class T>
int forward_t(const AveLayerNormArgs& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = a.n % V == 0 && aligned16(a.x) && aligned16(a.y) && on16(a.x_stride, sizeof(T)) && on16(a.y_stride, sizeof(T));
  // The ring from 513 columns on, 64 a thread or, with few rows, fewer (bf16, 16384 rows of 512: 20.4 us, 14.4 with rows in
  // registers; of 1024: 22.5 and 36.9; of 8192: 108 and 137)
  if (wide) {
    constexpr int P = 64 / V;
    if (a.n <= 512) return short_rows<V>(a.n, [&](auto f) { return run_forward<T, V, f.tpr, f.p, f.u>(a, stream); });
    const bool few = few_rows(a.rows);
    if (a.n <= 1024) return few ? run_forward_ring<T, P / 8, 8>(a, stream) : run_forward_ring<T, P / 2, 1>(a, stream);
    if (a.n <= 2048) return few ? run_forward_ring<T, P / 8, 8>(a, stream) : run_forward_ring<T, P, 1>(a, stream);
    if (a.n <= 4096) return few ? run_forward_ring<T, P / 4, 8>(a, stream) : run_forward_ring<T, P, 2>(a, stream);
    if (a.n <= 8192) return few ? run_forward_ring<T, P / 2, 8>(a, stream) : run_forward_ring<T, P, 4>(a, stream);
    if (a.n <= 16384) return run_forward_ring<T, P, 8>(a, stream);
    return run_forward<T, V, 1024, (MAX_N / V + 1023) / 1024, 1>(a, stream);
  }
  return by_element<true>(a.n, [&](auto f) { return run_forward<T, 1, f.tpr, f.p, f.u>(a, stream); });
}
template <class T>
int backward_t(const AveLayerNormBwdArgs& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = a.n % V == 0 && aligned16(a.x) && aligned16(a.d_y) && aligned16(a.d_x) && on16(a.x_stride, sizeof(T)) &&
                    on16(a.dy_stride, sizeof(T)) && on16(a.dx_stride, sizeof(T));
  if (wide) {
    // The ring from 257 columns on, 32 a thread (bf16, 16384 rows of 256: 20.5 us, 19.5 with rows in registers; of 512: 24.6 and 27.5; of 8192: 145 and 347)
    constexpr int P = 32 / V;
    if (a.n <= 256) return short_rows<V>(a.n, [&](auto f) { return run_backward<T, V, f.tpr, f.p, f.u>(a, stream); });
    const bool few = few_rows(a.rows);
    if (a.n <= 512) return few ? run_backward_ring<T, P / 4, 8>(a, stream) : run_backward_ring<T, P / 2, 1>(a, stream);
    if (a.n <= 1024) return few ? run_backward_ring<T, P / 4, 8>(a, stream) : run_backward_ring<T, P, 1>(a, stream);
    if (a.n <= 2048) return few ? run_backward_ring<T, P / 4, 8>(a, stream) : run_backward_ring<T, P, 2>(a, stream);
    if (a.n <= 4096) return few ? run_backward_ring<T, P / 2, 8>(a, stream) : run_backward_ring<T, P, 4>(a, stream);
    if (a.n <= 8192) return run_backward_ring<T, P, 8>(a, stream);
    if (a.n <= 16384) return run_backward_long<T, V, 16 / V>(a, stream);
    if (a.n <= 24576) return run_backward_long<T, V, 24 / V>(a, stream);
    return run_backward_long<T, 4, 7>(a, stream);
  }
  if (a.n > 2048) {
    if (a.n <= 8192) return run_backward_long<T, 1, 8>(a, stream);
    return a.n <= 16384 ? run_backward_long<T, 1, 16>(a, stream) : run_backward_long<T, 1, 28>(a, stream);
  }
  return by_element<false>(a.n, [&](auto f) { return run_backward<T, 1, f.tpr, f.p, f.u>(a, stream); });
}
}  // namespace

int64_t layer_norm_max_n() { return MAX_N; }

int launch_layer_norm(const AveLayerNormArgs& a, cudaStream_t stream) {
  switch (a.x_dtype) {
    case AVE_DTYPE_BF16: return forward_t<__nv_bfloat16>(a, stream);
    case AVE_DTYPE_FP16: return forward_t<__half>(a, stream);
    default: return forward_t<float>(a, stream);
  }
}
size_t layer_norm_backward_workspace_bytes(const AveLayerNormBwdArgs& a) {
  return (a.d_weight != nullptr || a.d_bias != nullptr) ? (size_t)BWD_CTAS * 2 * (size_t)a.n * 4 : 0;
}
int launch_layer_norm_backward(const AveLayerNormBwdArgs& a, cudaStream_t stream) {
  switch (a.x_dtype) {
    case AVE_DTYPE_BF16: return backward_t<__nv_bfloat16>(a, stream);
    case AVE_DTYPE_FP16: return backward_t<__half>(a, stream);
    default: return backward_t<float>(a, stream);
  }
}

}  // namespace ave
