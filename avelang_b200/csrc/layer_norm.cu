// Layer norm over rows of n elements, and its gradients.
//
//   y = (x - m) r w + b,   m = mean(x),   r = 1 / sqrt(mean((x - m)^2) + eps)
//   dx = r (w dy - mean(w dy) - xh mean(w dy xh)),   xh = (x - m) r,   dw = sum over rows of dy xh,   db = sum over rows of dy
//
// Both are bound by HBM: the forward pass reads x and writes y, the backward pass reads x and dy and writes dx.  A row belongs to a group of
// `TPR` threads, each of which keeps the same columns for every row it meets: the weights are read once a CTA, the row stays in
// registers between the reductions, and the sums of the weight's gradient are registers too.  U rows are in flight a group, which
// share the barriers of the reductions.  A CTA's sums go to scratch and a second kernel adds them in a fixed order.
#include <cuda_fp16.h>

#include "common.cuh"

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
__device__ __forceinline__ void load_piece(float (&f)[VEC], const T* src) {
  const Piece<T, VEC> p = *reinterpret_cast<const Piece<T, VEC>*>(src);
#pragma unroll
  for (int i = 0; i < VEC; ++i) f[i] = Elem<T>::up(p.e[i]);
}
template <class T, int VEC>
__device__ __forceinline__ void store_piece(T* dst, const float (&f)[VEC]) {
  Piece<T, VEC> p;
#pragma unroll
  for (int i = 0; i < VEC; ++i) p.e[i] = Elem<T>::down(f[i]);
  *reinterpret_cast<Piece<T, VEC>*>(dst) = p;
}
template <class T>
__device__ __forceinline__ float param(const void* p, bool wide, int64_t i) {
  return wide ? reinterpret_cast<const float*>(p)[i] : Elem<T>::up(reinterpret_cast<const T*>(p)[i]);
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
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) layer_norm_kernel(const AveLayerNormArgs a) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
  __shared__ float sums[2][U * 32];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const T* x = reinterpret_cast<const T*>(a.x);
  T* y = reinterpret_cast<T*>(a.y);
  pdl_wait();
  float w[P][VEC], b[P][VEC];
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int64_t c = (int64_t)(p * TPR + sub) * VEC + i;
      w[p][i] = a.weight != nullptr && c < a.n ? param<T>(a.weight, wide, c) : 1.f;
      b[p][i] = a.bias != nullptr && c < a.n ? param<T>(a.bias, wide, c) : 0.f;
    }
  const float inv_n = 1.f / (float)a.n;
  const int64_t step = (int64_t)gridDim.x * GROUPS * U;
  for (int64_t r0 = (int64_t)blockIdx.x * GROUPS * U; r0 < a.rows; r0 += step) {
    float f[U][P][VEC], s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * GROUPS + group;
      s[u] = 0.f;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t c = (int64_t)(p * TPR + sub) * VEC;
        if (r < a.rows && c < a.n) load_piece<T, VEC>(f[u][p], x + r * a.x_stride + c);
        else
#pragma unroll
          for (int i = 0; i < VEC; ++i) f[u][p][i] = 0.f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int i = 0; i < VEC; ++i) s[u] += f[u][p][i];
    group_sum<TPR, U>(s, sums[0]);
    float mean[U], q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // the squares are of differences from the mean: the sum of x^2 would lose what a large mean hides
      mean[u] = s[u] * inv_n;
      q[u] = 0.f;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const bool in = (int64_t)(p * TPR + sub) * VEC < a.n;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          f[u][p][i] -= mean[u];
          q[u] += in ? f[u][p][i] * f[u][p][i] : 0.f;
        }
      }
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
      for (int p = 0; p < P; ++p) {
        const int64_t c = (int64_t)(p * TPR + sub) * VEC;
        if (c >= a.n) continue;
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = fmaf(f[u][p][i] * rstd, w[p][i], b[p][i]);
        store_piece<T, VEC>(y + r * a.y_stride + c, o);
      }
    }
  }
}

// Sums of CTA c: partial[c][0][n] of dy xh, partial[c][1][n] of dy
template <class T, int VEC, int TPR, int P, int U>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256) layer_norm_backward_kernel(const AveLayerNormBwdArgs a, float* partial) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
  __shared__ float sums[2][2 * U * 32];
  extern __shared__ float cols[];  // [GROUPS][2][TPR * P * VEC], with several groups to a CTA
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const T *x = reinterpret_cast<const T*>(a.x), *dy = reinterpret_cast<const T*>(a.d_y);
  T* dx = reinterpret_cast<T*>(a.d_x);
  pdl_wait();
  float w[P][VEC], dw[P][VEC], db[P][VEC];
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
      const int64_t c = (int64_t)(p * TPR + sub) * VEC + i;
      w[p][i] = a.weight != nullptr && c < a.n ? param<T>(a.weight, wide, c) : 1.f;
      dw[p][i] = db[p][i] = 0.f;
    }
  const float inv_n = 1.f / (float)a.n;
  const int64_t step = (int64_t)gridDim.x * GROUPS * U;
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * GROUPS * U; r0 < a.rows; r0 += step, turn ^= 1) {
    float xh[U][P][VEC], d[U][P][VEC], s[2 * U], rstd[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * GROUPS + group;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t c = (int64_t)(p * TPR + sub) * VEC;
        if (r < a.rows && c < a.n) {
          load_piece<T, VEC>(xh[u][p], x + r * a.x_stride + c);
          load_piece<T, VEC>(d[u][p], dy + r * a.dy_stride + c);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) xh[u][p][i] = d[u][p][i] = 0.f;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * GROUPS + group;
      const float mean = r < a.rows ? a.mean[r] : 0.f;
      rstd[u] = r < a.rows ? a.rstd[r] : 0.f;
      s[2 * u] = s[2 * u + 1] = 0.f;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const bool in = (int64_t)(p * TPR + sub) * VEC < a.n;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          xh[u][p][i] = in ? (xh[u][p][i] - mean) * rstd[u] : 0.f;
          dw[p][i] += d[u][p][i] * xh[u][p][i];
          db[p][i] += d[u][p][i];
          d[u][p][i] *= w[p][i];
          s[2 * u] += d[u][p][i];
          s[2 * u + 1] += d[u][p][i] * xh[u][p][i];
        }
      }
    }
    group_sum<TPR, 2 * U>(s, sums[turn]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * GROUPS + group;
      if (r >= a.rows) continue;
      const float c1 = s[2 * u] * inv_n, c2 = s[2 * u + 1] * inv_n;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int64_t c = (int64_t)(p * TPR + sub) * VEC;
        if (c >= a.n) continue;
        float o[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) o[i] = rstd[u] * (d[u][p][i] - c1 - xh[u][p][i] * c2);
        store_piece<T, VEC>(dx + r * a.dx_stride + c, o);
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
        if (c < a.n) { out[c] = dw[p][i]; out[a.n + c] = db[p][i]; }
      }
  } else {
    constexpr int N = TPR * P * VEC;
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int c = (p * TPR + sub) * VEC + i;
        cols[group * 2 * N + c] = dw[p][i];
        cols[group * 2 * N + N + c] = db[p][i];
      }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * N; e += THREADS) {
      float t = 0.f;
      for (int g = 0; g < GROUPS; ++g) t += cols[g * 2 * N + e];
      const int c = e % N;
      if (c < a.n) out[(e / N) * a.n + c] = t;
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

constexpr int BWD_CTAS = 148 * 4;  // of sums in scratch, at most
constexpr int64_t MAX_N = 32768;

inline int sm_count() {
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  return sms;
}

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
  AVE_CUDA_TRY(launch_after(layer_norm_kernel<T, VEC, TPR, P, U>, (unsigned)(ctas < most ? ctas : most), THREADS, 0, stream, a));
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
  AVE_CUDA_TRY(launch_after(layer_norm_backward_kernel<T, VEC, TPR, P, U>, (unsigned)grid, THREADS, smem, stream, a, partial));
  if (sums) AVE_CUDA_TRY(launch_after(layer_norm_columns_kernel<T>, (unsigned)((2 * a.n + 31) / 32), 256, 0, stream, a, (const float*)partial, grid));
  return AVE_GDN_OK;
}

// Threads a row and pieces a thread by the row's length; `f` is called with them and the rows in flight.
template <int TPR, int P, int U> struct Form { static constexpr int tpr = TPR, p = P, u = U; };
template <int VEC, class F>
int by_length(int64_t n, F f) {
  const int64_t pieces = (n + VEC - 1) / VEC;
  if (pieces <= 8) return f(Form<8, 1, 2>());
  if (pieces <= 32) return f(Form<32, 1, 4>());
  if (pieces <= 64) return f(Form<32, 2, 2>());
  if (pieces <= 256) return f(Form<256, 1, 4>());
  if (pieces <= 512) return f(Form<256, 2, 2>());
  if (pieces <= 1024) return f(Form<256, 4, 1>());
  if constexpr (VEC >= 4) {
    if (pieces <= 4096) return f(Form<1024, 4, 1>());
    if constexpr (VEC == 4)
      if (pieces <= 8192) return f(Form<1024, 8, 1>());
  } else {
    if (pieces <= 4096) return f(Form<256, 16, 1>());
    if (pieces <= 32768) return f(Form<1024, 32, 1>());
  }
  return AVE_GDN_UNSUPPORTED;
}
bool on16(int64_t stride, int size) { return (stride * size) % 16 == 0; }

template <class T>
int forward_t(const AveLayerNormArgs& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = a.n % V == 0 && aligned16(a.x) && aligned16(a.y) && on16(a.x_stride, sizeof(T)) && on16(a.y_stride, sizeof(T));
  if (wide) return by_length<V>(a.n, [&](auto f) { return run_forward<T, V, f.tpr, f.p, f.u>(a, stream); });
  return by_length<1>(a.n, [&](auto f) { return run_forward<T, 1, f.tpr, f.p, f.u>(a, stream); });
}
template <class T>
int backward_t(const AveLayerNormBwdArgs& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = a.n % V == 0 && aligned16(a.x) && aligned16(a.d_y) && aligned16(a.d_x) && on16(a.x_stride, sizeof(T)) &&
                    on16(a.dy_stride, sizeof(T)) && on16(a.dx_stride, sizeof(T));
  if (wide) return by_length<V>(a.n, [&](auto f) { return run_backward<T, V, f.tpr, f.p, f.u>(a, stream); });
  return by_length<1>(a.n, [&](auto f) { return run_backward<T, 1, f.tpr, f.p, f.u>(a, stream); });
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
