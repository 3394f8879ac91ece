// RMS norm with the residual's addition, its form with 8-bit results, and rows in 8 bits and back.
//
//   h = round(x + residual),   y = h r w,   r = 1 / sqrt(mean(h^2) + eps)
//   scale = max|y| / 127,   q = round(y / scale) = round(h w (127 / max|h w|))    (the row's r cancels; the factor is rounded to fp32)
//
// All of it is bound by HBM: x and residual are read once, h and y are written once.  Rows of whole 16-byte pieces come through a ring in shared
// memory, filled by copies that each thread makes for itself (no barrier, nothing to wait for but its own copies), so that what is on its way does
// not depend on registers; the sum of squares, and the largest |h w|, are formed in one pass over the row's pieces, and a second pass over shared
// memory writes the results.  131072 x 2048 bf16: with a residual 355 to 361 us (6.0 TB/s of 6.5), to 8 bits 320 (5.9), 8-bit rows alone 139 (5.8) and back 132 (6.1); one row 1.7 to 1.9 us.
// Other rows go element by element (8192 x 2047 bf16 with a residual 35 us, 22 with 2048 columns).
#include "rows.cuh"

namespace ave {
namespace {

using namespace rows;

enum Mode { NORM, NORM8, QUANT };
constexpr int64_t FEW_ROWS = 2 * 148;  // a CTA a row, two at most one behind the other

// S stages of `arrays` (x, and the residual where there is one) x P pieces x THREADS
template <class T, int TPR, int P, int S, int MODE>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256, 1) rms_rows_kernel(const AveRmsNormArgs a, bool aligned) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR, V = kVec<T>, H = V / 2;
  extern __shared__ uint4 ring[];
  __shared__ float sums[2][2 * THREADS / 32];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int bar = TPR > 32 && GROUPS > 1 ? 1 + group : 0;
  const T *x = reinterpret_cast<const T*>(a.x), *residual = reinterpret_cast<const T*>(a.residual);
  const bool add = MODE != QUANT && residual != nullptr;
  const int arrays = add ? 2 : 1, n = (int)a.n;
  uint4* mine = ring + threadIdx.x;
  const int64_t first = (int64_t)blockIdx.x * GROUPS + group, step = (int64_t)gridDim.x * GROUPS;
  // every thread of a warp takes part in every turn, so the number of turns is that of the CTA's first row
  const int64_t turns = (a.rows - (int64_t)blockIdx.x * GROUPS + step - 1) / step;
  if (a.rows <= FEW_ROWS) pdl_trigger();  // a short kernel: the one behind it sets itself up beside it
  pdl_wait();
  auto fetch = [&](int64_t r, int stage) {
    if (r < a.rows) {
      uint4* to = mine + stage * arrays * P * THREADS;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int c = (p * TPR + sub) * V;
        if (c >= n) break;
        copy_async(to + p * THREADS, x + r * a.x_stride + c);
        if (add) copy_async(to + (P + p) * THREADS, residual + r * a.residual_stride + c);
      }
    }
    copy_commit();
  };
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(first + s * step, s);
  const float inv_n = 1.f / (float)n, offset = (a.flags & AVE_RMS_FLAG_ZERO_CENTERED) ? 1.f : 0.f;
  const bool wide = a.w_dtype == AVE_DTYPE_FP32;
  // a thread's columns are the same in every row: their weights stay in registers, but for the longest rows (read again for every row, from L1 and L2,
  // 131072 x 2048 with a residual to 8 bits took 423 us, 330 so)
  constexpr bool kKept = MODE != QUANT && P * V <= 32 && TPR < 1024;
  float2 kept[kKept ? P : 1][H];
  if constexpr (kKept)
#pragma unroll
    for (int p = 0; p < P; ++p)
      if ((p * TPR + sub) * V < n) params<T>(kept[p], a.weight, wide, aligned, (p * TPR + sub) * V, offset);
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
    copy_wait<S - 1>();
    const bool live = r < a.rows;
    uint4* row = mine + stage * arrays * P * THREADS;
    stage = stage == S - 1 ? 0 : stage + 1;
    float2 s2 = splat(0.f);
    float top = 0.f, top1 = 0.f;
    if (live) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        const int c = (p * TPR + sub) * V;
        if (c >= n) break;
        float2 f[H];
        widen<T>(f, row[p * THREADS]);
        if (add) {
          float2 g[H];
          widen<T>(g, row[(P + p) * THREADS]);
#pragma unroll
          for (int i = 0; i < H; ++i) f[i] = __fadd2_rn(f[i], g[i]);
          const uint4 h = narrow<T>(f);
          row[p * THREADS] = h;
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.sum) + r * a.sum_stride + c) = h;
          widen<T>(f, h);
        }
        if constexpr (MODE != QUANT) {
#pragma unroll
          for (int i = 0; i < H; ++i) s2 = __ffma2_rn(f[i], f[i], s2);
        }
        if constexpr (MODE == NORM8) {
          float2 w[H];
          weights(w, p, c);
#pragma unroll
          for (int i = 0; i < H; ++i) f[i] = __fmul2_rn(f[i], w[i]);
        }
        if constexpr (MODE != NORM) {
#pragma unroll
          for (int i = 0; i < H; ++i) { top = max_nan(top, fabsf(f[i].x)); top1 = max_nan(top1, fabsf(f[i].y)); }
        }
      }
    }
    float sum = s2.x + s2.y;
    top = max_nan(top, top1);
    group_reduce<TPR, MODE != NORM>(sum, top, sums[turn & 1], bar);
    if (!live) continue;
    const float rstd = MODE == QUANT ? 1.f : 1.f / sqrtf(sum * inv_n + a.eps);
    Scale sc;
    if constexpr (MODE != NORM) sc = row_scale(top, rstd);
    if (sub == 0) {
      if (MODE != QUANT && a.rstd != nullptr) a.rstd[r] = rstd;
      if constexpr (MODE != NORM) a.scale[r] = sc.scale;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = (p * TPR + sub) * V;
      if (c >= n) break;
      float2 f[H];
      widen<T>(f, row[p * THREADS]);
      float2 w[H];
      if constexpr (MODE != QUANT) weights(w, p, c);
      if constexpr (MODE == NORM) {
#pragma unroll
        for (int i = 0; i < H; ++i) f[i] = __fmul2_rn(__fmul2_rn(f[i], splat(rstd)), w[i]);
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.y) + r * a.y_stride + c) = narrow<T>(f);
      } else {
        uint32_t q[V / 4];
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
          if constexpr (MODE == NORM8) { f[2 * i] = __fmul2_rn(f[2 * i], w[2 * i]); f[2 * i + 1] = __fmul2_rn(f[2 * i + 1], w[2 * i + 1]); }
          q[i] = sc.inverse == 0.f ? 0u : pack_int8(f[2 * i], f[2 * i + 1], sc.inverse);
        }
        int8_t* to = reinterpret_cast<int8_t*>(a.y) + r * a.y_stride + c;
        if constexpr (V == 8) *reinterpret_cast<uint2*>(to) = make_uint2(q[0], q[1]);
        else *reinterpret_cast<uint32_t*>(to) = q[0];
      }
    }
  }
}

// Rows that do not lie on 16 bytes: element by element, neighbouring threads on neighbouring columns, a row in registers.  (Four columns a thread by the widest accesses
// that the row's address allows, or by aligned pieces that shuffles split and join, are slower: 8192 x 2047 bf16 with a residual 60 and 105 us, 35 so.)
template <class T, int TPR, int P, int MODE>
__global__ void __launch_bounds__(TPR > 256 ? TPR : 256, 1) rms_elements_kernel(const AveRmsNormArgs a) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
  __shared__ float sums[2][2 * THREADS / 32];
  const int sub = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int bar = TPR > 32 && GROUPS > 1 ? 1 + group : 0;
  const T *x = reinterpret_cast<const T*>(a.x), *residual = reinterpret_cast<const T*>(a.residual);
  const bool add = MODE != QUANT && residual != nullptr, wide = a.w_dtype == AVE_DTYPE_FP32;
  const float inv_n = 1.f / (float)a.n, offset = (a.flags & AVE_RMS_FLAG_ZERO_CENTERED) ? 1.f : 0.f;
  const int n = (int)a.n;
  if (a.rows <= FEW_ROWS) pdl_trigger();
  pdl_wait();
  auto weight = [&](int c) { return MODE == QUANT || a.weight == nullptr ? 1.f : param<T>(a.weight, wide, c) + offset; };
  constexpr bool kKept = MODE != QUANT && P <= 8;
  float kept[kKept ? P : 1];
  if constexpr (kKept)
#pragma unroll
    for (int p = 0; p < P; ++p) kept[p] = p * TPR + sub < n ? weight(p * TPR + sub) : 0.f;
  int turn = 0;
  for (int64_t r0 = (int64_t)blockIdx.x * GROUPS; r0 < a.rows; r0 += (int64_t)gridDim.x * GROUPS, turn ^= 1) {
    const int64_t r = r0 + group;
    const bool live = r < a.rows;
    const T *row = x + r * a.x_stride + sub, *other = residual + r * a.residual_stride + sub;
    T in[P], in2[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const bool there = live && p * TPR + sub < n;
      in[p] = there ? row[p * TPR] : Elem<T>::down(0.f);
      if (add) in2[p] = there ? other[p * TPR] : Elem<T>::down(0.f);
    }
    if (add) {
      T* to = reinterpret_cast<T*>(a.sum) + r * a.sum_stride + sub;
#pragma unroll
      for (int p = 0; p < P; ++p) {
        in[p] = Elem<T>::down(Elem<T>::up(in[p]) + Elem<T>::up(in2[p]));
        if (live && p * TPR + sub < n) to[p * TPR] = in[p];
      }
    }
    float sum = 0.f, top = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const float f = Elem<T>::up(in[p]);
      if constexpr (MODE != QUANT) sum = fmaf(f, f, sum);
      if constexpr (MODE == NORM8) top = max_nan(top, fabsf(f * (kKept ? kept[kKept ? p : 0] : p * TPR + sub < n ? weight(p * TPR + sub) : 0.f)));
      if constexpr (MODE == QUANT) top = max_nan(top, fabsf(f));
    }
    group_reduce<TPR, MODE != NORM>(sum, top, sums[turn], bar);
    if (!live) continue;
    const float rstd = MODE == QUANT ? 1.f : 1.f / sqrtf(sum * inv_n + a.eps);
    Scale sc;
    if constexpr (MODE != NORM) sc = row_scale(top, rstd);
    if (sub == 0) {
      if (MODE != QUANT && a.rstd != nullptr) a.rstd[r] = rstd;
      if constexpr (MODE != NORM) a.scale[r] = sc.scale;
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
      const int c = p * TPR + sub;
      if (c >= n) break;
      const float f = Elem<T>::up(in[p]), w = kKept ? kept[kKept ? p : 0] : weight(c);
      if constexpr (MODE == NORM) reinterpret_cast<T*>(a.y)[r * a.y_stride + c] = Elem<T>::down(f * rstd * w);
      else reinterpret_cast<int8_t*>(a.y)[r * a.y_stride + c] = sc.inverse == 0.f ? (int8_t)0 : to_int8(MODE == NORM8 ? f * w : f, sc.inverse);
    }
  }
}

// Values of 8-bit rows: a thread reads an aligned piece of a row (what lies in it behind the row's end, the last row's too, may be anything) and writes 16 bytes at a time, or, where the results do not lie on 16 bytes, one column and its neighbours the next ones (8192 x 2047
// 101 us with 16 columns a thread written one by one, 12 so)
template <class T>
__global__ void __launch_bounds__(256) dequantize_kernel(const AveQuantRowsArgs a, int pieces) {
  constexpr int V = kVec<T>, U = 4;
  const int stride = gridDim.x * 256, skip = stride / pieces, rest = stride - skip * pieces;  // (row and piece are stepped: a division costs more than the piece)
  pdl_wait();
  int64_t r = ((int64_t)blockIdx.x * 256 + threadIdx.x) / pieces;
  int piece = (int)((int64_t)blockIdx.x * 256 + threadIdx.x - r * pieces);
  while (r < a.rows) {
    uint32_t q[U][2];
    float s[U];
    T* to[U];
    int there[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {  // U pieces on their way
      there[u] = r < a.rows ? (int)a.n - piece * V : 0;
      to[u] = reinterpret_cast<T*>(a.x) + r * a.x_stride + piece * V;
      if (there[u] > 0) {
        const int8_t* from = reinterpret_cast<const int8_t*>(a.q) + r * a.q_stride + piece * V;
        s[u] = a.scale[r];
        if constexpr (V == 8) {
          const uint2 v = *reinterpret_cast<const uint2*>(from);
          q[u][0] = v.x; q[u][1] = v.y;
        } else {
          q[u][0] = *reinterpret_cast<const uint32_t*>(from);
        }
      }
      r += skip; piece += rest;
      if (piece >= pieces) { ++r; piece -= pieces; }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (there[u] <= 0) continue;
      float2 f[V / 2];
#pragma unroll
      for (int e = 0; e < V / 2; ++e)
        f[e] = make_float2((float)(int8_t)(q[u][e / 2] >> (16 * (e & 1))) * s[u], (float)(int8_t)(q[u][e / 2] >> (16 * (e & 1) + 8)) * s[u]);
      if (there[u] >= V) {
        *reinterpret_cast<uint4*>(to[u]) = narrow<T>(f);
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e < there[u]) to[u][e] = Elem<T>::down(e & 1 ? f[e / 2].y : f[e / 2].x);
      }
    }
  }
}
template <class T>
__global__ void __launch_bounds__(256) dequantize_elements_kernel(const AveQuantRowsArgs a, int blocks) {  // of 256 columns a row, a warp each
  pdl_wait();
  const int64_t total = a.rows * blocks;
  const int lane = threadIdx.x & 31, n = (int)a.n;
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < total; i += (int64_t)gridDim.x * 8) {
    const int64_t r = i / blocks;
    const int c = (int)(i - r * blocks) * 256 + lane;
    const int8_t* q = reinterpret_cast<const int8_t*>(a.q) + r * a.q_stride + c;
    T* to = reinterpret_cast<T*>(a.x) + r * a.x_stride + c;
    const float s = a.scale[r];
    int8_t v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + 32 * e < n ? q[32 * e] : (int8_t)0;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + 32 * e < n) to[32 * e] = Elem<T>::down((float)v[e] * s);
  }
}

constexpr int64_t MAX_N = 28672;

template <class T, int TPR, int P, int S, int MODE>
int run_rows(const AveRmsNormArgs& a, cudaStream_t stream) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR, ONE = S * P * THREADS * 16;
  constexpr int MOST = (MODE == QUANT ? 1 : 2) * ONE;
  static_assert(MOST <= 225 * 1024, "shared memory of an SM");
  constexpr auto* kernel = &rms_rows_kernel<T, TPR, P, S, MODE>;
  if constexpr (MOST > 47 * 1024) {
    const int rc = allow_smem<kernel>(MOST);
    if (rc != AVE_GDN_OK) return rc;
  }
  static const int per1 = ctas_an_sm(kernel, THREADS, ONE), per2 = ctas_an_sm(kernel, THREADS, MOST);
  const bool add = MODE != QUANT && a.residual != nullptr;
  const int64_t ctas = (a.rows + GROUPS - 1) / GROUPS, most = (int64_t)sm_count() * (add ? per2 : per1);
  const bool aligned = aligned16(a.weight);
  AVE_CUDA_TRY(launch_after(kernel, (unsigned)(ctas < most ? ctas : most), THREADS, (size_t)(add ? MOST : ONE), stream, a, aligned));
  return AVE_GDN_OK;
}
template <class T, int TPR, int P, int MODE>
int run_elements(const AveRmsNormArgs& a, cudaStream_t stream) {
  constexpr int THREADS = TPR > 256 ? TPR : 256, GROUPS = THREADS / TPR;
  constexpr auto* kernel = &rms_elements_kernel<T, TPR, P, MODE>;
  static const int per = ctas_an_sm(kernel, THREADS, 0);
  const int64_t ctas = (a.rows + GROUPS - 1) / GROUPS, most = (int64_t)sm_count() * per;
  AVE_CUDA_TRY(launch_after(kernel, (unsigned)(ctas < most ? ctas : most), THREADS, 0, stream, a));
  return AVE_GDN_OK;
}

template <class T, int MODE>
int forward(const AveRmsNormArgs& a, cudaStream_t stream) {
  constexpr int V = kVec<T>, size = (int)sizeof(T);
  const bool wide = a.n % V == 0 && aligned16(a.x) && on16(a.x_stride, size) && aligned16(a.residual) && on16(a.residual_stride, size) &&
                    aligned16(a.sum) && on16(a.sum_stride, size) && (MODE != NORM || (aligned16(a.y) && on16(a.y_stride, size)));
  if (!wide) {
    if (a.n <= 8) return run_elements<T, 8, 1, MODE>(a, stream);
    if (a.n <= 64) return run_elements<T, 32, 2, MODE>(a, stream);
    if (a.n <= 256) return run_elements<T, 32, 8, MODE>(a, stream);
    if (a.n <= 512) return run_elements<T, 64, 8, MODE>(a, stream);
    if (a.n <= 1024) return run_elements<T, 128, 8, MODE>(a, stream);
    if (a.n <= 2048) return run_elements<T, 256, 8, MODE>(a, stream);
    if (a.n <= 4096) return run_elements<T, 512, 8, MODE>(a, stream);
    if (a.n <= 8192) return run_elements<T, 1024, 8, MODE>(a, stream);
    if (a.n <= 16384) return run_elements<T, 1024, 16, MODE>(a, stream);
    return run_elements<T, 1024, 28, MODE>(a, stream);
  }
  const int pieces = (int)a.n / V;
  if (pieces <= 8) return run_rows<T, 8, 1, 2, MODE>(a, stream);
  if (pieces <= 32) return run_rows<T, 32, 1, 4, MODE>(a, stream);
  if (a.rows <= FEW_ROWS) {
    if (pieces <= 256) return run_rows<T, 256, 1, 2, MODE>(a, stream);
    if (pieces <= 1024) return run_rows<T, 512, 2, 2, MODE>(a, stream);
  }
  // Two stages, CTAs of 256 threads, two an SM: 131072 x 2048 bf16 with a residual 350 us, without 184, to 8 bits 322; three stages and four CTAs of 128 368, 193 and 330;
  // three CTAs of 256 with fewer registers 359, 190 and 324
  if (pieces <= 64) return run_rows<T, 32, 2, 4, MODE>(a, stream);
  if (pieces <= 128) return run_rows<T, 32, 4, 2, MODE>(a, stream);
  if (pieces <= 256) return run_rows<T, 64, 4, 2, MODE>(a, stream);
  if (pieces <= 512) return run_rows<T, 128, 4, 2, MODE>(a, stream);
  if (pieces <= 1024) return run_rows<T, 256, 4, 2, MODE>(a, stream);
  if (pieces <= 2048) return run_rows<T, 512, 4, 2, MODE>(a, stream);
  if (pieces <= 4096) return run_rows<T, 1024, 4, 1, MODE>(a, stream);
  if constexpr (size == 4) return run_rows<T, 1024, 7, 1, MODE>(a, stream);
  return AVE_GDN_UNSUPPORTED;
}
template <class T>
int forward_t(const AveRmsNormArgs& a, cudaStream_t stream) {
  return (a.flags & AVE_RMS_FLAG_INT8) ? forward<T, NORM8>(a, stream) : forward<T, NORM>(a, stream);
}
}  // namespace

int64_t rms_norm_max_n() { return MAX_N; }

int launch_rms_norm(const AveRmsNormArgs& a, cudaStream_t stream) {
  switch (a.x_dtype) {
    case AVE_DTYPE_BF16: return forward_t<__nv_bfloat16>(a, stream);
    case AVE_DTYPE_FP16: return forward_t<__half>(a, stream);
    default: return forward_t<float>(a, stream);
  }
}
int launch_quantize_rows(const AveQuantRowsArgs& q, cudaStream_t stream) {
  AveRmsNormArgs a{};
  a.struct_size = sizeof(a);
  a.x = q.x; a.y = q.q; a.scale = q.scale;
  a.rows = q.rows; a.n = q.n; a.x_stride = q.x_stride; a.y_stride = q.q_stride;
  a.x_dtype = a.w_dtype = q.x_dtype;
  switch (q.x_dtype) {
    case AVE_DTYPE_BF16: return forward<__nv_bfloat16, QUANT>(a, stream);
    case AVE_DTYPE_FP16: return forward<__half, QUANT>(a, stream);
    default: return forward<float, QUANT>(a, stream);
  }
}
template <class T>
int dequantize(const AveQuantRowsArgs& a, cudaStream_t stream) {
  const int64_t most = (int64_t)sm_count() * 8;
  if (aligned16(a.x) && on16(a.x_stride, (int)sizeof(T))) {
    const int pieces = (int)((a.n + kVec<T> - 1) / kVec<T>);
    const int64_t ctas = (a.rows * pieces + 255) / 256;
    AVE_CUDA_TRY(launch_after(dequantize_kernel<T>, (unsigned)(ctas < most ? ctas : most), 256, 0, stream, a, pieces));
  } else {
    const int blocks = (int)((a.n + 255) / 256);
    const int64_t ctas = (a.rows * blocks + 7) / 8;
    AVE_CUDA_TRY(launch_after(dequantize_elements_kernel<T>, (unsigned)(ctas < most ? ctas : most), 256, 0, stream, a, blocks));
  }
  return AVE_GDN_OK;
}
int launch_dequantize_rows(const AveQuantRowsArgs& a, cudaStream_t stream) {
  switch (a.x_dtype) {
    case AVE_DTYPE_BF16: return dequantize<__nv_bfloat16>(a, stream);
    case AVE_DTYPE_FP16: return dequantize<__half>(a, stream);
    default: return dequantize<float>(a, stream);
  }
}

}  // namespace ave
