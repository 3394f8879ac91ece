// C[M,N] = (A[M,K] * B[N,K]^T) a_scale[m] b_scale[n] + bias[n]: int8 operands, exact int32 sums in tensor memory (kind::i8), one rounding to bf16, fp16
// or fp32 behind fp32 scaling.  K is at most 131071, so that |sum| <= 128 * 128 * K stays below 2^31.
//
// One tile a cluster of `split` CTAs, each of which takes a contiguous share of K (split == 1 where there are tiles enough); the partial sums meet over
// distributed shared memory.  They are whole numbers: the result does not depend on the split.
#include <mutex>

#include "rows.cuh"
#include "tc.cuh"

namespace ave {
namespace {

using rows::Elem;

constexpr int BM = 128, BN = 256, BK = 128;  // BK: bytes of K a block, one swizzle span, four MMAs of 32
constexpr int THREADS = 192;
constexpr int STAGES = 10, RING = 200 * 1024;                    // ring depth limit and bytes
constexpr int SMEM = RING + BM * BK + 1024;                      // an MMA reads 128 rows of A wherever the tile ends

// instruction descriptor of kind::i8: signed operands, both K-major, int32 sums
__device__ __forceinline__ uint32_t idesc_i8(int m, int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24); }
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc),
               "r"(idesc), "r"(accumulate)
               : "memory");
}

struct Epilogue {  // what a sum becomes
  const float *a_scale, *b_scale;
  const void* bias;
  void* c;
  int64_t ldc;
  int bias_wide;
  int vector;  // rows of C lie on 16 bytes
};
template <class T>
__device__ __forceinline__ float bias_at(const Epilogue& e, int64_t n) { return e.bias == nullptr ? 0.f : rows::param<T>(e.bias, e.bias_wide != 0, n); }
// (sum * a_scale) * b_scale + bias: a sum of 24 bits and more is rounded to fp32 first, 2^-24 of its value
__device__ __forceinline__ float finish(int32_t sum, float a_scale, float b_scale, float bias) { return fmaf(__fmul_rn((float)sum, a_scale), b_scale, bias); }

struct Plan { int bn, split, stages, ks, a_rows; };  // tile width, CTAs a tile, ring depth, blocks of 128 a stage, rows of A

template <class T>
__global__ void __launch_bounds__(THREADS, 1)
gemm_int8_cluster_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Epilogue e, int64_t M, int64_t N, int64_t K,
                         uint32_t* status, const Plan plan, uint32_t tmem_cols) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = tc::align1024(smem_raw);
  __shared__ uint64_t full[STAGES], empty[STAGES], acc_full, drained;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile uint32_t abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bn = plan.bn, split = plan.split, stages = plan.stages;
  const int a_bytes = plan.a_rows * BK, b_bytes = bn * BK, stage_bytes = plan.ks * (a_bytes + b_bytes);
  const int nt = (int)((N + bn - 1) / bn), kb_count = (int)((K + plan.ks * BK - 1) / (plan.ks * BK));  // in stages of ks blocks
  const int rank = (int)(blockIdx.x % split), tile = (int)(blockIdx.x / split), tm = tile / nt, tn = tile % nt;
  const int per = (kb_count + split - 1) / split, kb0 = rank * per, kb1 = min(kb_count, kb0 + per);

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
    tc::mbar_init(&acc_full, 1);
    tc::mbar_init(&drained, 1);
    abort_flag = 0;
    tc::fence_barrier_init();
    tc::prefetch_tmap(&tmA);
    tc::prefetch_tmap(&tmB);
  }
  if (warp == 1) tc::tmem_alloc(&tmem_slot, tmem_cols);
  tc::tc_fence_before_sync();
  __syncthreads();
  tc::tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  pdl_wait();

  // Both issuing warps run their loops whole and elect a lane for the instructions themselves.  A stage holds `ks` blocks of 128 along K,
  // [A][A].. [B][B].., behind one barrier.
  if (warp == 0) {
    int s = 0; uint32_t ph = 0;
    int kb = kb0;
    for (; kb < kb1; ++kb) {
      if (!tc::mbar_wait_unrolled(&empty[s], ph ^ 1u, &abort_flag)) break;
      if (tc::elect_one()) {
        uint8_t* st = smem + s * stage_bytes;
        tc::mbar_expect_tx(&full[s], (uint32_t)stage_bytes);
        for (int j = 0; j < plan.ks; ++j) tc::tma_load_2d(st + plan.ks * a_bytes + j * b_bytes, &tmB, &full[s], (kb * plan.ks + j) * BK, tn * bn);
        for (int j = 0; j < plan.ks; ++j) tc::tma_load_2d(st + j * a_bytes, &tmA, &full[s], (kb * plan.ks + j) * BK, tm * BM);
      }
      __syncwarp();
      if (++s == stages) { s = 0; ph ^= 1u; }
    }
    if (abort_flag != 0u)  // the copies of the last `stages` turns may be on their way
      for (int i = max(kb0, kb - stages); i < kb; ++i) tc::drain(&full[(i - kb0) % stages], (uint32_t)((i - kb0) / stages) & 1u);
  } else if (warp == 1) {
    const uint32_t idesc = idesc_i8(BM, bn);
    int s = 0; uint32_t ph = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!tc::mbar_wait_unrolled(&full[s], ph, &abort_flag)) { ok = false; break; }
      tc::tc_fence_after_sync();
      if (tc::elect_one()) {
        // with fewer than 128 rows in the A tile the MMA reads whatever lies behind it: those lanes are never read back
        const uint32_t base = tc::smem_u32(smem) + (uint32_t)(s * stage_bytes);
        for (int j = 0; j < plan.ks; ++j) {
          const uint64_t da = tc::smem_desc_sw128(base + (uint32_t)(j * a_bytes), 16, 1024);
          const uint64_t db = tc::smem_desc_sw128(base + (uint32_t)(plan.ks * a_bytes + j * b_bytes), 16, 1024);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_i8(tmem_base, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), idesc, (kb > kb0 || j > 0 || k != 0) ? 1u : 0u);
        }
        tc::mma_commit(&empty[s]);
      }
      __syncwarp();
      if (++s == stages) { s = 0; ph ^= 1u; }
    }
    if (ok) {
      if (tc::elect_one()) tc::mma_commit(&acc_full);
    } else {
      tc::drain_mmas(&drained);
    }
  }
  __syncwarp();  // the other lanes of the issuing warps must not poll beside them
  // the accumulator is complete, so every operand tile has landed and been read
  const bool ok = tc::mbar_wait_unrolled(&acc_full, 0, &abort_flag);
  tc::tc_fence_after_sync();
  __syncwarp();
  tc::cluster_sync();  // ... in every CTA of the cluster: the rings may be overwritten
  const int rows = (int)min((int64_t)BM, M - (int64_t)tm * BM), slice = (rows + split - 1) / split, pitch = bn + 4;
  if (ok && warp >= 2) {
    const int row = (warp & 3) * 32 + lane;
    const bool live = row < rows;
    const int owner = live ? row / slice : 0;
    const uint32_t dst = tc::mapa(tc::smem_u32(smem) + (uint32_t)(((rank * slice + (row - owner * slice)) * pitch) * 4), (uint32_t)owner);
#pragma unroll 1
    for (int c = 0; c < bn; c += 16) {
      uint32_t r[16];
      tc::tmem_ld16(tmem_base + ((uint32_t)((warp & 3) * 32) << 16) + (uint32_t)c, r);
      tc::tmem_ld_wait();
      if (live) {
#pragma unroll
        for (int v = 0; v < 4; ++v) tc::st_cluster_v4(dst + (uint32_t)(c + 4 * v) * 4, r[4 * v], r[4 * v + 1], r[4 * v + 2], r[4 * v + 3]);
      }
    }
  }
  tc::tc_fence_before_sync();
  __syncwarp();
  tc::cluster_sync();
  {
    const int32_t* part = reinterpret_cast<const int32_t*>(smem);
    const int mine = min(slice, rows - rank * slice), vec = bn / 8;
    for (int i = threadIdx.x; i < mine * vec; i += THREADS) {
      const int r = i / vec, c = (i - r * vec) * 8;
      int32_t x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      for (int s = 0; s < split; ++s) {
        const int4 a = *reinterpret_cast<const int4*>(part + (s * slice + r) * pitch + c), b = *reinterpret_cast<const int4*>(part + (s * slice + r) * pitch + c + 4);
        x[0] += a.x; x[1] += a.y; x[2] += a.z; x[3] += a.w;
        x[4] += b.x; x[5] += b.y; x[6] += b.z; x[7] += b.w;
      }
      const int64_t col = (int64_t)tn * bn + c, at = (int64_t)tm * BM + rank * slice + r;
      const float a_scale = e.a_scale[at];
      T* dst = reinterpret_cast<T*>(e.c) + at * e.ldc + col;
      if (e.vector != 0 && col + 8 <= N) {
        float2 f[4];
#pragma unroll
        for (int v = 0; v < 4; ++v)
          f[v] = make_float2(finish(x[2 * v], a_scale, e.b_scale[col + 2 * v], bias_at<T>(e, col + 2 * v)),
                             finish(x[2 * v + 1], a_scale, e.b_scale[col + 2 * v + 1], bias_at<T>(e, col + 2 * v + 1)));
        constexpr int V = rows::kVec<T>;
#pragma unroll
        for (int p = 0; p < 8 / V; ++p) {
          float2 g[V / 2];
#pragma unroll
          for (int v = 0; v < V / 2; ++v) g[v] = f[p * V / 2 + v];
          reinterpret_cast<uint4*>(dst)[p] = rows::narrow<T>(g);
        }
      } else {
#pragma unroll
        for (int v = 0; v < 8; ++v)
          if (col + v < N) dst[v] = Elem<T>::down(finish(x[v], a_scale, e.b_scale[col + v], bias_at<T>(e, col + v)));
      }
    }
  }
  if (threadIdx.x == 0 && !ok && status != nullptr) atomicOr(status, AVE_GDN_DEV_WAIT_EXPIRED);
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after_sync();
    tc::tmem_dealloc(tmem_base, tmem_cols);
  }
}

// Tile width, K split and ring depth: among the cluster sizes that still give every tile its SMs, the one with the fewest bytes through the busiest SM
// (its operand tiles, plus what the exchange costs); tiles of full width, unsplit, where there are more of them than SMs.
// `clusters[s]`: clusters of s CTAs that run at once.
Plan make_plan(int64_t M, int64_t N, int64_t K, int sms, const int* clusters) {
  const int64_t mt = (M + BM - 1) / BM, kb = (K + BK - 1) / BK;
  const int64_t a_rows = M < BM ? (M + 7) / 8 * 8 : BM;
  auto depth = [&](int64_t stage) { return (int)(RING / stage < STAGES ? RING / stage : STAGES); };
  Plan best{};
  int64_t best_cost = INT64_MAX;
  for (int split = 1; split <= 8; ++split) {
    const int64_t tiles_n = clusters[split] / mt;
    if (tiles_n == 0) continue;
    const int64_t bn = ((N + tiles_n - 1) / tiles_n + 15) / 16 * 16, block = (a_rows + bn) * BK;
    if (bn > BN) continue;
    // blocks a stage: up to 48 KB a stage, at least three stages, no padding of K beyond one block a CTA
    int ks = 1;
    while (ks < 8 && 2 * ks * block <= 49152 && 2 * ks * split <= kb) ks *= 2;
    const int64_t steps = (kb + ks - 1) / ks, per = (steps + split - 1) / split;
    if ((split - 1) * per >= steps) continue;  // no CTA without work
    const int64_t stage = ks * block, exchange = split == 1 ? 0 : 65536 + a_rows * bn * 4;
    const int64_t least = ks > 2 ? ks * 8192 : 16384;
    const int64_t cost = per * (stage > least ? stage : least) + exchange;
    if (cost < best_cost) {
      best_cost = cost;
      best = {(int)bn, split, depth(stage), ks, (int)a_rows};
    }
  }
  if (best.bn == 0) {  // more tiles than SMs
    const int64_t nt = (N + BN - 1) / BN, bn = ((N + nt - 1) / nt + 15) / 16 * 16;
    best = {(int)bn, 1, depth((a_rows + bn) * BK), 1, (int)a_rows};
  }
  return best;
}

// Clusters of 1..8 CTAs of the kernel above that fit the device at once, asked once a device (nullptr: it would not say)
const int* cluster_counts(int dev, int sms) {
  static std::mutex mu;
  static int table[MAX_DEVICES][9] = {};
  if (dev < 0 || dev >= MAX_DEVICES) return nullptr;
  std::lock_guard<std::mutex> guard(mu);
  int* t = table[dev];
  if (t[0] == 0) {
    constexpr auto* kernel = &gemm_int8_cluster_kernel<__nv_bfloat16>;
    if (allow_smem<kernel>(SMEM) != AVE_GDN_OK) return nullptr;
    for (int s = 1; s <= 8; ++s) {
      cudaLaunchConfig_t cfg{};
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = (unsigned)s; at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3((unsigned)(s * sms)); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM;
      cfg.attrs = at; cfg.numAttrs = 1;
      int n = 0;
      if (s > 1 && cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) n = 0;
      t[s] = s == 1 ? sms : n;
    }
    (void)cudaGetLastError();
    t[0] = 1;
  }
  return t;
}

int operand_map(CUtensorMap* map, const void* base, int64_t rows, int64_t k, int64_t ld, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)k, (uint64_t)rows}, strides[2] = {1, (uint64_t)(rows > 1 ? ld : (k + 15) / 16 * 16)};  // (the distance of a single row says nothing)
  const uint32_t box[2] = {BK, (uint32_t)box_rows};
  return make_tmap(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, const_cast<void*>(base), 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <class T>
int launch_t(const AveGemmInt8Args& a, cudaStream_t stream) {
  int dev = 0, sms = 148;
  AVE_CUDA_TRY(cudaGetDevice(&dev));
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int size = (int)sizeof(T);
  const Epilogue e{a.a_scale, a.b_scale, a.bias, a.c, a.ldc, a.bias_dtype == AVE_DTYPE_FP32, aligned16(a.c) && rows::on16(a.ldc, size)};
  const int* clusters = cluster_counts(dev, sms);
  if (clusters == nullptr) return AVE_GDN_UNSUPPORTED;
  const Plan plan = make_plan(a.M, a.N, a.K, sms, clusters);
  CUtensorMap tmA, tmB;
  int rc = operand_map(&tmA, a.a, a.M, a.K, a.lda, plan.a_rows);
  if (rc != AVE_GDN_OK) return rc;
  rc = operand_map(&tmB, a.b, a.N, a.K, a.ldb, plan.bn);
  if (rc != AVE_GDN_OK) return rc;
  constexpr auto* kernel = &gemm_int8_cluster_kernel<T>;
  rc = allow_smem<kernel>(SMEM);
  if (rc != AVE_GDN_OK) return rc;
  uint32_t cols = 32;
  while ((int)cols < plan.bn) cols *= 2;
  const int64_t ctas = ((a.M + BM - 1) / BM) * ((a.N + plan.bn - 1) / plan.bn) * plan.split;
  if (ctas > INT32_MAX) return AVE_GDN_UNSUPPORTED;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = (unsigned)plan.split; at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)ctas); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM; cfg.stream = stream;
  cfg.attrs = at; cfg.numAttrs = 2;
  AVE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, tmA, tmB, e, a.M, a.N, a.K, a.status, plan, cols));
  return AVE_GDN_OK;
}

}  // namespace

int launch_gemm_int8_nt(const AveGemmInt8Args& a, cudaStream_t stream) {
  switch (a.c_dtype) {
    case AVE_DTYPE_BF16: return launch_t<__nv_bfloat16>(a, stream);
    case AVE_DTYPE_FP16: return launch_t<__half>(a, stream);
    default: return launch_t<float>(a, stream);
  }
}

}  // namespace ave
