// Gradients of the RMS norm.
//
//   xh = h r,   c = mean(w dy xh),   dx = r (w dy - xh c) + d_h,   dw = sum over rows of dy xh
//
// Bound by HBM: dy, h and d_h (the gradient that comes back beside the norm, where h is used further) are read once, dx is written once.  Rows come
// through a ring in shared memory as in the forward pass; a thread keeps its columns for every row it meets, so that the sums of the weight's
// gradient are registers.  A CTA's sums go to scratch and a second kernel adds them in a fixed order, 2.5 us behind the first.  bf16 with d_h: 131072 x 2048 308 us, 8192 x 2048 28
// us (21 at the copy rate), 8192 x 2047, element by element, 50; 1001 x 1409 fp32 7.1.
#include "rows.cuh"

namespace ave {
namespace {

using namespace rows;

constexpr int MAX_PARTS = 444;  // CTAs that leave sums: three an SM

// The groups' column sums of a CTA, added in the groups' order
template <int THREADS, int GROUPS>
__device__ __forceinline__ void add_groups(const float* cols, float* out, int n, int pitch) {
  __syncthreads();
  for (int c = threadIdx.x; c < n; c += THREADS) {
    float t = 0.f;
#pragma unroll 4
    for (int g = 0; g < GROUPS; ++g) t += cols[g * pitch + c];
    out[c] = t;
  }
}

template <class T, int THREADS, int TPR, int P, int S>
__global__ void __launch_bounds__(THREADS, 1) rms_backward_kernel(const AveRmsNormBwdArgs a, float* partial, bool aligned) {
  constexpr int GROUPS = THREADS / TPR, V = kVec<T>, H = V / 2;
  extern __shared__ uint4 ring[];
  __shared__ float sums[2][2 * THREADS / 32];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int bar = TPR > 32 && GROUPS > 1 ? 1 + group : 0;
  const T *dy = reinterpret_cast<const T*>(a.d_y), *x = reinterpret_cast<const T*>(a.x), *d_sum = reinterpret_cast<const T*>(a.d_sum);
  const bool add = d_sum != nullptr;
  const int arrays = add ? 3 : 2, n = (int)a.n;
  uint4* mine = ring + threadIdx.x;
  const int64_t first = (int64_t)blockIdx.x * GROUPS + group, step = (int64_t)gridDim.x * GROUPS;
  const int64_t turns = (a.rows - (int64_t)blockIdx.x * GROUPS + step - 1) / step;
  pdl_wait();
  auto fetch = [&](int64_t r, int stage) {
    if (r < a.rows) {
      uint4* to = mine + stage * arrays * P * THREADS;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int c = (p * TPR + sub) * V;
        if (c >= n) break;
        copy_async(to + p * THREADS, x + r * a.x_stride + c);
        copy_async(to + (P + p) * THREADS, dy + r * a.dy_stride + c);
        if (add) copy_async(to + (2 * P + p) * THREADS, d_sum + r * a.ds_stride + c);
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(first + s * step, s);
  const float inv_n = 1.f / (float)n, offset = (a.flags & AVE_RMS_FLAG_ZERO_CENTERED) ? 1.f : 0.f;
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
  constexpr bool kKept = P * V <= 32 && TPR < 1024;  // a thread's weights stay in registers
  float2 dw[P][H], kept[kKept ? P : 1][H];
#pragma unroll
  for (int p = 0; p < P; ++p) {
#pragma unroll
    for (int i = 0; i < H; ++i) dw[p][i] = splat(0.f);
    if constexpr (kKept)
      if ((p * TPR + sub) * V < n) params<T>(kept[p], a.weight, wide, aligned, (p * TPR + sub) * V, offset);
  }
  auto weights = [&](float2 (&w)[H], int p, int c) {
    if constexpr (kKept) {
#pragma unroll
      for (int i = 0; i < H; ++i) w[i] = kept[p][i];
    } else {
      params<T>(w, a.weight, wide, aligned, c, offset);
    }
  };
  int stage = 0;
  for (int64_t turn = 0; turn < turns; ++turn) {
    const int64_t r = first + turn * step;
    fetch(r + (S - 1) * step, stage == 0 ? S - 1 : stage - 1);  // (the stage that the turn before has read)
    const bool live = r < a.rows;
    const float rstd = live ? a.rstd[r] : 0.f;
    copy_wait<S - 1>();
    const uint4* row = mine + stage * arrays * P * THREADS;
    stage = stage == S - 1 ? 0 : stage + 1;
    float2 s2 = splat(0.f);
    if (live) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int c = (p * TPR + sub) * V;
        if (c >= n) break;
        float2 h[H], g[H], w[H];
        widen<T>(h, row[p * THREADS]);
        widen<T>(g, row[(P + p) * THREADS]);
        weights(w, p, c);
#pragma unroll
        for (int i = 0; i < H; ++i) s2 = __ffma2_rn(__fmul2_rn(g[i], w[i]), __fmul2_rn(h[i], splat(rstd)), s2);
      }
    }
    float sum = s2.x + s2.y, none = 0.f;
    group_reduce<TPR, false>(sum, none, sums[turn & 1], bar);
    if (!live) continue;
    const float c1 = sum * inv_n;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = (p * TPR + sub) * V;
      if (c >= n) break;
      float2 h[H], g[H], w[H], d[H];
      widen<T>(h, row[p * THREADS]);
      widen<T>(g, row[(P + p) * THREADS]);
      weights(w, p, c);
#pragma unroll
      for (int i = 0; i < H; ++i) {
        h[i] = __fmul2_rn(h[i], splat(rstd));
        dw[p][i] = __ffma2_rn(g[i], h[i], dw[p][i]);
        g[i] = __ffma2_rn(h[i], splat(-c1), __fmul2_rn(g[i], w[i]));
      }
      if (add) {
        widen<T>(d, row[(2 * P + p) * THREADS]);
#pragma unroll
        for (int i = 0; i < H; ++i) g[i] = __ffma2_rn(g[i], splat(rstd), d[i]);
      } else {
#pragma unroll
        for (int i = 0; i < H; ++i) g[i] = __fmul2_rn(g[i], splat(rstd));
      }
      *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.d_x) + r * a.dx_stride + c) = narrow<T>(g);
    }
  }
  if (partial == nullptr) return;
  pdl_trigger();
  float* out = partial + (int64_t)blockIdx.x * n;
  float* cols = GROUPS == 1 ? out : reinterpret_cast<float*>(ring) + group * TPR * P * V;
  if constexpr (GROUPS > 1) {
    copy_wait<0>();
    __syncthreads();  // all rows are done: the ring's memory takes the groups' sums
  }
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = (p * TPR + sub) * V;
    if (c >= n) break;
#pragma unroll
    for (int i = 0; i < H; ++i) {  // (a CTA's row of scratch may lie off 8 bytes)
      cols[c + 2 * i] = dw[p][i].x;
      cols[c + 2 * i + 1] = dw[p][i].y;
    }
  }
  if constexpr (GROUPS > 1) add_groups<THREADS, GROUPS>(reinterpret_cast<const float*>(ring), out, n, TPR * P * V);
}

// Rows that do not lie on 16 bytes: element by element, neighbouring threads on neighbouring columns, a row in registers
template <class T, int THREADS, int TPR, int P>
__global__ void __launch_bounds__(THREADS, 1) rms_backward_elements_kernel(const AveRmsNormBwdArgs a, float* partial) {
  constexpr int GROUPS = THREADS / TPR;
  __shared__ float sums[2][2 * THREADS / 32];
  extern __shared__ float cols[];  // [GROUPS][TPR * P], with several groups
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int bar = TPR > 32 && GROUPS > 1 ? 1 + group : 0;
  const T *dy = reinterpret_cast<const T*>(a.d_y), *x = reinterpret_cast<const T*>(a.x), *d_sum = reinterpret_cast<const T*>(a.d_sum);
  const bool wide = a.w_dtype == AVE_DTYPE_FP32, add = d_sum != nullptr;
  const float inv_n = 1.f / (float)a.n, offset = (a.flags & AVE_RMS_FLAG_ZERO_CENTERED) ? 1.f : 0.f;
  const int n = (int)a.n;
  pdl_wait();
  float w[P], dw[P];
#pragma unroll
  for (int p = 0; p < P; ++p) {
    w[p] = p * TPR + sub >= n ? 0.f : a.weight == nullptr ? 1.f : param<T>(a.weight, wide, p * TPR + sub) + offset;
    dw[p] = 0.f;
  }
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * GROUPS; r0 < a.rows; r0 += (int64_t)gridDim.x * GROUPS, turn ^= 1) {
    const int64_t r = r0 + group;
    const bool live = r < a.rows;
    const float rstd = live ? a.rstd[r] : 0.f;
    T h_in[P], g_in[P], d_in[P];
    const T zero = Elem<T>::down(0.f);
    auto fetch = [&](T (&v)[P], const T* row, bool wanted) {
#pragma unroll
      for (int p = 0; p < P; ++p) v[p] = wanted && live && p * TPR + sub < n ? row[p * TPR + sub] : zero;
    };
    fetch(h_in, x + r * a.x_stride, true);
    fetch(g_in, dy + r * a.dy_stride, true);
    fetch(d_in, d_sum + r * a.ds_stride, add);
    float sum = 0.f, none = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const float h = Elem<T>::up(h_in[p]) * rstd, g = Elem<T>::up(g_in[p]);
      dw[p] = fmaf(g, h, dw[p]);
      sum = fmaf(g * w[p], h, sum);
    }
    group_reduce<TPR, false>(sum, none, sums[turn], bar);
    if (!live) continue;
    const float c1 = sum * inv_n;
    T* to = reinterpret_cast<T*>(a.d_x) + r * a.dx_stride + sub;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (p * TPR + sub >= n) break;
      const float h = Elem<T>::up(h_in[p]) * rstd;
      to[p * TPR] = Elem<T>::down(fmaf(fmaf(h, -c1, Elem<T>::up(g_in[p]) * w[p]), rstd, Elem<T>::up(d_in[p])));  // (without d_sum plus zero)
    }
  }
  if (partial == nullptr) return;
  pdl_trigger();
  float* out = partial + (int64_t)blockIdx.x * n;
  float* sink = GROUPS == 1 ? out : cols + group * TPR * P;
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (p * TPR + sub < n) sink[p * TPR + sub] = dw[p];
  if constexpr (GROUPS > 1) add_groups<THREADS, GROUPS>(cols, out, n, TPR * P);
}

// Rows longer than those: a row a CTA, read again for the second pass
template <class T, int TPR, int P>
__global__ void __launch_bounds__(TPR, 1) rms_backward_long_kernel(const AveRmsNormBwdArgs a, float* partial) {
  __shared__ float sums[2][2 * TPR / 32];
  const int sub = threadIdx.x;
  const T *dy = reinterpret_cast<const T*>(a.d_y), *x = reinterpret_cast<const T*>(a.x), *d_sum = reinterpret_cast<const T*>(a.d_sum);
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
  const float inv_n = 1.f / (float)a.n, offset = (a.flags & AVE_RMS_FLAG_ZERO_CENTERED) ? 1.f : 0.f;
  const int n = (int)a.n;
  pdl_wait();
  auto weight = [&](int c) { return a.weight == nullptr ? 1.f : param<T>(a.weight, wide, c) + offset; };
  float dw[P];
#pragma unroll
  for (int p = 0; p < P; ++p) dw[p] = 0.f;
  int turn = 0;
  for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
    const float rstd = a.rstd[r];
    float sum = 0.f, none = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = p * TPR + sub;
      if (c >= n) break;
      const float g = Elem<T>::up(dy[r * a.dy_stride + c]), xh = Elem<T>::up(x[r * a.x_stride + c]) * rstd;
      dw[p] = fmaf(g, xh, dw[p]);
      sum = fmaf(g * weight(c), xh, sum);
    }
    group_reduce<TPR, false>(sum, none, sums[turn]);
    const float c1 = sum * inv_n;
#pragma unroll 4
    for (int c = sub; c < n; c += TPR) {
      const float g = Elem<T>::up(dy[r * a.dy_stride + c]) * weight(c), xh = Elem<T>::up(x[r * a.x_stride + c]) * rstd;
      const float d = fmaf(xh, -c1, g);
      reinterpret_cast<T*>(a.d_x)[r * a.dx_stride + c] = Elem<T>::down(d_sum != nullptr ? fmaf(d, rstd, Elem<T>::up(d_sum[r * a.ds_stride + c])) : d * rstd);
    }
  }
  if (partial == nullptr) return;
  pdl_trigger();
  float* out = partial + (int64_t)blockIdx.x * n;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const int c = p * TPR + sub;
    if (c < n) out[c] = dw[p];
  }
}

// Adds the CTAs' sums: 32 columns a CTA, each warp takes every 32nd row of sums
template <class T>
__global__ void __launch_bounds__(1024) rms_columns_kernel(const float* partial, void* d_weight, int w_dtype, int n, int parts) {
  __shared__ float part[32][33];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < n) {
    float v[4];  // four rows on their way
    for (int i = warp; i < parts; i += 128) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = i + 32 * k < parts ? partial[(int64_t)(i + 32 * k) * n + c] : 0.f;
      s += (v[0] + v[1]) + (v[2] + v[3]);
    }
  }
  part[warp][lane] = s;
  __syncthreads();
  if (warp != 0 || c >= n) return;
  float t[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int k = 0; k < 32; ++k) t[k & 3] += part[k][lane];
  const float sum = (t[0] + t[1]) + (t[2] + t[3]);
  if (w_dtype == AVE_DTYPE_FP32) reinterpret_cast<float*>(d_weight)[c] = sum;
  else reinterpret_cast<T*>(d_weight)[c] = Elem<T>::down(sum);
}

template <class T>
int add_columns(const AveRmsNormBwdArgs& a, int parts, cudaStream_t stream) {
  if (a.d_weight == nullptr) return AVE_GDN_OK;
  AVE_CUDA_TRY(launch_after(rms_columns_kernel<T>, (unsigned)((a.n + 31) / 32), 1024, 0, stream, (const float*)a.workspace, a.d_weight, a.w_dtype, (int)a.n, parts));
  return AVE_GDN_OK;
}
template <class T, int THREADS, int TPR, int P, int S>
int run_ring(const AveRmsNormBwdArgs& a, cudaStream_t stream) {
  constexpr int GROUPS = THREADS / TPR, ONE = S * P * THREADS * 16, MOST = 3 * ONE;
  static_assert(MOST <= 225 * 1024, "shared memory of an SM");
  static_assert(GROUPS == 1 || GROUPS * TPR * P * kVec<T> * 4 <= 2 * ONE, "the groups' sums lie in the ring");
  constexpr auto* kernel = &rms_backward_kernel<T, THREADS, TPR, P, S>;
  if constexpr (MOST > 47 * 1024) {
    const int rc = allow_smem<kernel>(MOST);
    if (rc != AVE_GDN_OK) return rc;
  }
  static const int per = ctas_an_sm(kernel, THREADS, MOST);
  const int64_t ctas = (a.rows + GROUPS - 1) / GROUPS, most = (int64_t)sm_count() * per < MAX_PARTS ? (int64_t)sm_count() * per : MAX_PARTS;
  const int grid = (int)(ctas < most ? ctas : most);
  float* partial = a.d_weight != nullptr ? reinterpret_cast<float*>(a.workspace) : nullptr;
  AVE_CUDA_TRY(launch_after(kernel, (unsigned)grid, THREADS, (size_t)(a.d_sum != nullptr ? MOST : MOST / 3 * 2), stream, a, partial, aligned16(a.weight)));
  return add_columns<T>(a, grid, stream);
}
template <class T, int THREADS, int TPR, int P>
int run_elements(const AveRmsNormBwdArgs& a, cudaStream_t stream) {
  constexpr int GROUPS = THREADS / TPR;
  constexpr size_t smem = GROUPS > 1 ? (size_t)THREADS * P * 4 : 0;
  static_assert(smem <= 40 * 1024, "column sums in the default shared memory");
  constexpr auto* kernel = &rms_backward_elements_kernel<T, THREADS, TPR, P>;
  static const int per = ctas_an_sm(kernel, THREADS, smem);
  const int64_t ctas = (a.rows + GROUPS - 1) / GROUPS, room = (int64_t)sm_count() * per, most = room < MAX_PARTS ? room : MAX_PARTS;
  const int grid = (int)(ctas < most ? ctas : most);
  float* partial = a.d_weight != nullptr ? reinterpret_cast<float*>(a.workspace) : nullptr;
  AVE_CUDA_TRY(launch_after(kernel, (unsigned)grid, THREADS, smem, stream, a, partial));
  return add_columns<T>(a, grid, stream);
}
template <class T>
int run_long(const AveRmsNormBwdArgs& a, cudaStream_t stream) {
  const int grid = (int)(a.rows < 2 * sm_count() && a.rows < MAX_PARTS ? a.rows : 2 * sm_count() < MAX_PARTS ? 2 * sm_count() : MAX_PARTS);
  float* partial = a.d_weight != nullptr ? reinterpret_cast<float*>(a.workspace) : nullptr;
  AVE_CUDA_TRY(launch_after(rms_backward_long_kernel<T, 1024, 28>, (unsigned)grid, 1024, 0, stream, a, partial));
  return add_columns<T>(a, grid, stream);
}

template <class T>
int backward_t(const AveRmsNormBwdArgs& a, cudaStream_t stream) {
  constexpr int V = kVec<T>, size = (int)sizeof(T);
  const bool wide = a.n % V == 0 && aligned16(a.x) && on16(a.x_stride, size) && aligned16(a.d_y) && on16(a.dy_stride, size) && aligned16(a.d_x) &&
                    on16(a.dx_stride, size) && aligned16(a.d_sum) && on16(a.ds_stride, size);
  const int64_t pieces = a.n / V;
  if (!wide && a.n <= 8192) {
    if (a.n <= 8) return run_elements<T, 256, 8, 1>(a, stream);
    if (a.n <= 64) return run_elements<T, 256, 32, 2>(a, stream);
    if (a.n <= 256) return run_elements<T, 512, 32, 8>(a, stream);
    if (a.n <= 512) return run_elements<T, 512, 64, 8>(a, stream);
    if (a.n <= 1024) return run_elements<T, 512, 128, 8>(a, stream);
    if (a.n <= 2048) return run_elements<T, 512, 256, 8>(a, stream);
    if (a.n <= 4096) return run_elements<T, 512, 512, 8>(a, stream);
    return run_elements<T, 1024, 1024, 8>(a, stream);
  }
  if (!wide || pieces > 4096) return run_long<T>(a, stream);
  if (pieces <= 8) return run_ring<T, 256, 8, 1, 3>(a, stream);
  if (pieces <= 32) return run_ring<T, 512, 32, 1, 3>(a, stream);
  if (a.rows <= 2 * 148) {
    if (pieces <= 256) return run_ring<T, 256, 256, 1, 2>(a, stream);
    if (pieces <= 1024) return run_ring<T, 512, 512, 2, 2>(a, stream);
  }
  if (pieces <= 64) return run_ring<T, 512, 32, 2, 2>(a, stream);
  if (pieces <= 128) return run_ring<T, 512, 32, 4, 2>(a, stream);
  if (pieces <= 256) return run_ring<T, 512, 64, 4, 2>(a, stream);
  if (pieces <= 512) return run_ring<T, 512, 128, 4, 2>(a, stream);
  if (pieces <= 1024) return run_ring<T, 512, 256, 4, 2>(a, stream);
  if (pieces <= 2048) return run_ring<T, 512, 512, 4, 2>(a, stream);
  return run_ring<T, 1024, 1024, 4, 1>(a, stream);
}

}  // namespace

size_t rms_norm_backward_workspace_bytes(const AveRmsNormBwdArgs& a) {  // (no CTA without a row)
  return a.d_weight != nullptr ? (size_t)(a.rows < MAX_PARTS ? a.rows : MAX_PARTS) * (size_t)a.n * 4 : 0;
}

int launch_rms_norm_backward(const AveRmsNormBwdArgs& a, cudaStream_t stream) {
  switch (a.x_dtype) {
    case AVE_DTYPE_BF16: return backward_t<__nv_bfloat16>(a, stream);
    case AVE_DTYPE_FP16: return backward_t<__half>(a, stream);
    default: return backward_t<float>(a, stream);
  }
}

}  // namespace ave
