// Rows in pieces of 16 bytes: what the kernels of the RMS norm and of rows in 8 bits share.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace ave {
namespace rows {

template <class T> struct Elem;
template <> struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16(x); }
  static __device__ __forceinline__ float2 up2(uint32_t x) { return bf16x2_to_float2(x); }
  static __device__ __forceinline__ uint32_t down2(float2 x) { return pack_bf16x2(x.x, x.y); }
};
template <> struct Elem<__half> {
  static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
  static __device__ __forceinline__ float2 up2(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
  static __device__ __forceinline__ uint32_t down2(float2 x) {
    const __half2 h = __floats2half2_rn(x.x, x.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <> struct Elem<float> {
  static __device__ __forceinline__ float up(float x) { return x; }
  static __device__ __forceinline__ float down(float x) { return x; }
};

// 16 bytes as pairs of fp32 and back
template <class T> constexpr int kVec = 16 / (int)sizeof(T);
template <class T>
__device__ __forceinline__ void widen(float2 (&f)[kVec<T> / 2], const uint4& v) {
  if constexpr (sizeof(T) == 4) {
    f[0] = make_float2(__uint_as_float(v.x), __uint_as_float(v.y));
    f[1] = make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
  } else {
    f[0] = Elem<T>::up2(v.x); f[1] = Elem<T>::up2(v.y); f[2] = Elem<T>::up2(v.z); f[3] = Elem<T>::up2(v.w);
  }
}
template <class T>
__device__ __forceinline__ uint4 narrow(const float2 (&f)[kVec<T> / 2]) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  else
    return make_uint4(Elem<T>::down2(f[0]), Elem<T>::down2(f[1]), Elem<T>::down2(f[2]), Elem<T>::down2(f[3]));
}
__device__ __forceinline__ float2 splat(float x) { return make_float2(x, x); }

// A weight of the rows' type or fp32
template <class T>
__device__ __forceinline__ float param(const void* p, bool wide, int64_t i) {
  return wide ? reinterpret_cast<const float*>(p)[i] : Elem<T>::up(reinterpret_cast<const T*>(p)[i]);
}
// The kVec of them that begin with element c, plus `offset`; where there is no weight, ones.  `aligned`: they lie on 16 bytes.
template <class T>
__device__ __forceinline__ void params(float2 (&w)[kVec<T> / 2], const void* p, bool wide, bool aligned, int64_t c, float offset) {
  constexpr int V = kVec<T>;
  if (p == nullptr) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = splat(1.f);
    return;
  }
  if (aligned && !wide) {
    widen<T>(w, *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(p) + c));
  } else if (aligned) {
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
      const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + c + 4 * i);
      w[2 * i] = make_float2(v.x, v.y);
      w[2 * i + 1] = make_float2(v.z, v.w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = make_float2(param<T>(p, wide, c + 2 * i), param<T>(p, wide, c + 2 * i + 1));
  }
#pragma unroll
  for (int i = 0; i < V / 2; ++i) w[i] = __fadd2_rn(w[i], splat(offset));
}

// The larger one, NaN where either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// A sum and a maximum over the TPR threads of a group; everybody gets them.  Groups beyond a warp are whole CTAs, or `bar` > 0 names the group's
// hardware barrier; `smem` ([2][warps of the CTA]) may be used again behind the next call's barrier, so two calls in a row take two buffers.
template <int TPR, bool kMax>
__device__ __forceinline__ void group_reduce(float& sum, float& top, float* smem, int bar = 0) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if constexpr (kMax) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, o));
  }
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int warp = threadIdx.x >> 5, first = warp / W * W;
    if ((threadIdx.x & 31) == 0) {
      smem[2 * warp] = sum;
      if constexpr (kMax) smem[2 * warp + 1] = top;
    }
    if (bar == 0) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(bar), "r"(TPR) : "memory");
    sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) sum += smem[2 * (first + w)];
    if constexpr (kMax) {
      top = smem[2 * first + 1];
#pragma unroll
      for (int w = 1; w < W; ++w) top = max_nan(top, smem[2 * (first + w) + 1]);
    }
  }
}

// 16 bytes into shared memory; a thread that reads what it has copied itself needs no barrier, only its own wait
__device__ __forceinline__ void copy_async(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// A row's scale, and what its values are multiplied with: 127 / top.  A largest value that is not finite gives a NaN, one whose scale would be
// below the smallest normal number, or whose 127 / top would be infinite, a zero; both with whole numbers of zero.
struct Scale { float scale, inverse; };
__device__ __forceinline__ Scale row_scale(float top, float factor) {  // of a row of values v with max|v factor| = top factor
  const float largest = top * factor, scale = largest * (1.f / 127.f);
  if (!(largest < __uint_as_float(0x7f800000u))) return {__uint_as_float(0x7fffffffu), 0.f};
  if (scale < 1.17549435e-38f || top < 3.8e-37f) return {0.f, 0.f};
  return {scale, 127.f / top};
}
// Four values as whole numbers, to nearest, ties to even: 1.5 * 2^23 leaves them in the low bits of the sum, which is rounded once
__device__ __forceinline__ uint32_t pack_int8(float2 a, float2 b, float inverse) {
  const float2 magic = splat(12582912.f), m = splat(inverse);
  a = __ffma2_rn(a, m, magic);
  b = __ffma2_rn(b, m, magic);
  const uint32_t lo = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040), hi = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
__device__ __forceinline__ int8_t to_int8(float x, float inverse) { return (int8_t)(__float_as_uint(fmaf(x, inverse, 12582912.f)) & 0xffu); }

inline bool on16(int64_t stride, int size) { return (stride * size) % 16 == 0; }
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

}  // namespace rows
}  // namespace ave
