// C[M,N] = (A[M,K] * B[N,K]^T) a_scale[m] b_scale[n] + bias[n]: int8 operands, exact int32 sums in tensor memory (kind::i8), one rounding to bf16, fp16
// or fp32 behind fp32 scaling.  K is at most 131071, so that |sum| <= 128 * 128 * K stays below 2^31.
//
// Three forms.  Persistent pairs of CTAs on tiles of 256 x bn (gemm_int8_pair_kernel).  Few rows: one tile of up to 128 rows a cluster of `split` CTAs, each of
// which takes a contiguous share of K; the partial sums meet over distributed shared memory (gemm_int8_cluster_kernel).  One or two rows, up to four where B
// is small: B streamed through the ordinary units (gemm_int8_stream_kernel).  Sums are whole numbers and all forms finish them in the same way: a result depends neither on the
// form nor on the split.
#include <mutex>
#include <type_traits>

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

__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem), "l"(a_desc), "l"(b_desc),
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

// ------------------------------------------------------------------------------------------------ pairs of CTAs
// A pair of CTAs works on a tile of 256 rows x bn columns (whole chunks of 128 bytes of the result, at most 256): each loads its 128 rows of A and bn / 2 rows of B, the leader issues
// MMAs of 256 x bn x 32 for both, and each finishes the 128 rows whose sums lie in its tensor memory, in one of two accumulators, while the next tile's products run.
//   warp 0      TMA producer: a ring of stages of 128 bytes of K, 5 of 32 KB with 256 columns, 9 with 64; the bytes of both CTAs are counted at the leader's barrier
//   warp 1      of the leader: MMAs; a stage is free in both CTAs when its products are done
//   warps 2..9  sums -> fp32 -> result, two warps a quarter of the rows, every other chunk of 128 bytes each: 32 rows of it through shared memory and out as one
//               TMA store, or element by element where the rows of C do not lie on 16 bytes
// Behind a wait that has expired every role leaves, the finishing warps write NaN where they have no sums, both CTAs meet, the leader makes up for copies that only one of them has asked
// for, both wait (with a limit) for copies, products and arrivals that are on their way, and they meet again before tensor memory is given back.
constexpr int PAIR_STAGES = 9, PAIR_RING = 184 * 1024, PAIR_THREADS = 320, PAIR_ROWS = 2 * BM;  // ring: depth limit and bytes of a CTA
constexpr int GROUP_M = 16;  // row tiles that are swept together, so that their rows of A stay in L2
constexpr int PAIR_OUT = PAIR_RING, PAIR_COLS = PAIR_OUT + 8 * 4096, PAIR_SMEM = PAIR_COLS + 8 * 1024 + 1024;

template <class T, int KS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
gemm_int8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const __grid_constant__ CUtensorMap tmC, const Epilogue e,
                      int64_t M, int64_t N, int64_t K, uint32_t* status, int bn, int stages, uint32_t whole) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = tc::align1024(smem_raw);
  __shared__ uint64_t full[PAIR_STAGES], empty[PAIR_STAGES], acc_full[2], acc_empty[2], drained;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile uint32_t abort_flag, issued[2], ended[2];  // stages whose copies the leader's and the other CTA's producer have asked for (kept by the leader); stages and tiles whose products the leader has issued
  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;  // (uniform to the compiler, and with it tiles, rows and addresses)
  const uint32_t rank = tc::cluster_rank();
  const int mt = (int)((M + PAIR_ROWS - 1) / PAIR_ROWS), nt = (int)((N + bn - 1) / bn), kb_count = (int)((K + KS * BK - 1) / (KS * BK));  // in stages of KS blocks
  const uint32_t b_bytes = (uint32_t)(bn / 2 * BK), stage_bytes = KS * (BM * BK + b_bytes);
  // Units of work: the first `whole` tiles, then the halves (of the columns) of those that are left.  B comes in boxes of half of a CTA's rows where there are halves.
  const uint32_t all_tiles = (uint32_t)mt * (uint32_t)nt, tiles = whole + 2 * (all_tiles - whole), first = blockIdx.x / 2, step = gridDim.x / 2;
  const bool halves = whole < all_tiles;
  auto width_at = [&](uint32_t unit) { return unit < whole ? bn : bn / 2; };
  auto tile_at = [&](uint32_t unit, int& m, int64_t& col, int& width) {
    const uint32_t tile = unit < whole ? unit : whole + (unit - whole) / 2, per = (uint32_t)(GROUP_M * nt), group = tile / per, r = tile - group * per,
                   rows = min((uint32_t)GROUP_M, (uint32_t)mt - group * GROUP_M), n = r / rows;
    m = (int)(group * GROUP_M + r - n * rows);
    width = width_at(unit);
    col = (int64_t)n * bn + (unit >= whole && ((unit - whole) & 1) != 0 ? width : 0);
  };
  auto landing = [&](int width) { return KS * (uint32_t)((BM + width / 2) * BK); };  // bytes of a stage of one CTA

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
    for (int b = 0; b < 2; ++b) { tc::mbar_init(&acc_full[b], 1); tc::mbar_init(&acc_empty[b], 16); }
    tc::mbar_init(&drained, 1);
    abort_flag = 0;
    issued[0] = issued[1] = ended[0] = ended[1] = 0;
    tc::fence_barrier_init();
    tc::prefetch_tmap(&tmA);
    tc::prefetch_tmap(&tmB);
  }
  if (warp == 1) tc::tmem_alloc_pair(&tmem_slot, 512);
  tc::tc_fence_before_sync();
  __syncthreads();
  tc::cluster_sync();  // both CTAs' barriers are there
  tc::tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  pdl_wait();

  if (warp == 0) {
    int s = 0; uint32_t ph = 0;
    uint32_t turns = 0;
    bool ok = true;
    for (uint32_t tile = first; tile < tiles && ok; tile += step) {
      int m, width;
      int64_t col;
      tile_at(tile, m, col, width);
      const int row_b = (int)col + (int)rank * (width / 2);
      const bool second = halves && width == bn;
      for (int kb = 0; kb < kb_count; ++kb) {
        if (!tc::mbar_wait_together(&empty[s], ph ^ 1u, &abort_flag)) { ok = false; break; }
        if (tc::elect_one()) {
          uint8_t* st = smem + s * (int)stage_bytes;
          const uint32_t bar = tc::mapa(tc::smem_u32(&full[s]), 0);
          if (rank == 0) tc::mbar_expect_tx(&full[s], 2 * landing(width));
#pragma unroll
          for (int j = 0; j < KS; ++j) {
            tc::tma_load_2d_pair(st + j * BM * BK, &tmA, bar, (kb * KS + j) * BK, m * PAIR_ROWS + (int)rank * BM);
            tc::tma_load_2d_pair(st + KS * BM * BK + j * (int)b_bytes, &tmB, bar, (kb * KS + j) * BK, row_b);
            if (second) tc::tma_load_2d_pair(st + KS * BM * BK + j * (int)b_bytes + bn / 4 * BK, &tmB, bar, (kb * KS + j) * BK, row_b + bn / 4);
          }
        }
        __syncwarp();
        ++turns;
        if (++s == stages) { s = 0; ph ^= 1u; }
      }
    }
    if (ok)  // the leader's last arrivals at this CTA's barriers (a stage that was never filled counts as free)
      for (int i = 0; i < stages; ++i) {
        if (!tc::mbar_wait_together(&empty[s], ph ^ 1u, &abort_flag)) break;
        if (++s == stages) { s = 0; ph ^= 1u; }
      }
    if (lane == 0) tc::st_cluster_u32(tc::mapa(tc::smem_u32(const_cast<uint32_t*>(&issued[rank])), 0), turns);
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t stage0 = (tc::smem_u32(smem) >> 4) | (uint32_t)tc::desc_lo(0, 16);
      constexpr uint32_t hi = tc::desc_hi(1024, true);
      int s = 0, local = 0; uint32_t ph = 0, blocks = 0;
      bool ok = true;
      for (uint32_t tile = first; tile < tiles; tile += step, ++local) {
        const int buf = local & 1;
        const uint32_t idesc = idesc_i8(PAIR_ROWS, width_at(tile));
        if (!tc::mbar_wait_together<true>(&acc_empty[buf], ((uint32_t)(local >> 1) & 1u) ^ 1u, &abort_flag)) { ok = false; break; }
        tc::tc_fence_after_sync();
        const uint32_t d = tmem_base + (uint32_t)buf * BN;
        for (int kb = 0; kb < kb_count; ++kb) {
          if (!tc::mbar_wait_together(&full[s], ph, &abort_flag)) { ok = false; break; }
          tc::tc_fence_after_sync();
          if (tc::elect_one()) {
            const uint32_t a_lo = stage0 + (uint32_t)s * (stage_bytes >> 4);  // low words of the descriptors; the high ones are constant
#pragma unroll
            for (int j = 0; j < KS; ++j)
#pragma unroll
              for (int k = 0; k < BK / 32; ++k)
                mma_i8_pair(d, tc::smem_desc(a_lo + (uint32_t)(j * BM * BK / 16 + 2 * k), hi), tc::smem_desc(a_lo + (uint32_t)(KS * BM * BK / 16 + 2 * k) + (uint32_t)j * (b_bytes >> 4), hi), idesc,
                            (kb | j | k) != 0 ? 1u : 0u);
            tc::mma_commit_pair(&empty[s]);
          }
          __syncwarp();
          ++blocks;
          if (++s == stages) { s = 0; ph ^= 1u; }
        }
        if (!ok) break;
        if (tc::elect_one()) tc::mma_commit_pair(&acc_full[buf]);
        __syncwarp();
      }
      if (lane < 4) tc::st_cluster_u32(tc::mapa(tc::smem_u32(const_cast<uint32_t*>(&ended[lane & 1])), (uint32_t)lane >> 1), (lane & 1) == 0 ? blocks : (uint32_t)local);
    }
  } else {
    const int quarter = warp & 3;  // tensor memory lanes this warp may touch
    constexpr int V = rows::kVec<T>, CW = 128 / (int)sizeof(T);  // columns a chunk
    const int half = (warp - 2) >> 2;  // which chunks
    uint8_t* out = smem + PAIR_OUT + (warp - 2) * 4096;
    float* cols = reinterpret_cast<float*>(smem + PAIR_COLS) + (warp - 2) * 256;  // scales and bias of this warp's columns, CW of a chunk behind those of the one before
    // The scales of a tile are fetched while the one before is finished (fetched and waited for in line they took 1600 to 1900 cycles a tile).
    float next_scale[4], next_bias[4], next_a = 0.f;
    int next_m = 0, next_width = 0;
    int64_t next_col = 0;
    auto prefetch = [&](uint32_t tile) {
      if (tile >= tiles) return;
      tile_at(tile, next_m, next_col, next_width);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = lane + 32 * j;
        const int64_t c = next_col + (i / CW * 2 + half) * CW + i % CW;
        next_scale[j] = c < N ? e.b_scale[c] : 0.f;
        next_bias[j] = c < N ? bias_at<T>(e, c) : 0.f;
      }
      const int64_t row = (int64_t)next_m * PAIR_ROWS + rank * BM + quarter * 32 + lane;
      next_a = row < M ? e.a_scale[row] : 0.f;
    };
    prefetch(first);
    int local = 0;
    uint32_t tile = first;
    for (; tile < tiles; tile += step, ++local) {
      const int m = next_m, width_now = next_width, buf = local & 1;
      const int64_t row0 = (int64_t)m * PAIR_ROWS + rank * BM + quarter * 32, col0 = next_col;
      const int n_left = (int)min((int64_t)width_now, N - col0);  // (of a second half possibly none)
      __syncwarp();
#pragma unroll
      for (int j = 0; j < 4; ++j) { cols[lane + 32 * j] = next_scale[j]; cols[128 + lane + 32 * j] = next_bias[j]; }
      const float a_scale = next_a;
      __syncwarp();
      prefetch(tile + step);
      if (!tc::mbar_wait_together(&acc_full[buf], (uint32_t)(local >> 1) & 1u, &abort_flag)) break;
      tc::tc_fence_after_sync();
      auto release = [&] {  // this warp's part of the accumulator is out of tensor memory
        tc::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive_cluster(tc::mapa(tc::smem_u32(&acc_empty[buf]), 0));
      };
      if (half * CW >= n_left) release();  // (a narrow last tile)
#pragma unroll 1
      for (int c = half * CW, at = 0; c < n_left; c += 2 * CW, at += CW) {
        uint32_t r[CW];
#pragma unroll
        for (int part = 0; part < CW; part += 32)
          tc::tmem_ld32(tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(buf * BN + c + part), *reinterpret_cast<uint32_t(*)[32]>(r + part));
        tc::tmem_ld_wait();
        if (c + 2 * CW >= n_left) release();
        uint4 packed[8];  // a row's 128 bytes
#pragma unroll
        for (int v = 0; v < CW; v += V) {
          float2 f[V / 2];
#pragma unroll
          for (int i = 0; i < V; i += 4) {
            const float4 sc = *reinterpret_cast<const float4*>(cols + at + v + i), bi = *reinterpret_cast<const float4*>(cols + 128 + at + v + i);
            const float2 x = __fmul2_rn(make_float2((float)(int32_t)r[v + i], (float)(int32_t)r[v + i + 1]), rows::splat(a_scale));
            const float2 y = __fmul2_rn(make_float2((float)(int32_t)r[v + i + 2], (float)(int32_t)r[v + i + 3]), rows::splat(a_scale));
            f[i / 2] = __ffma2_rn(x, make_float2(sc.x, sc.y), make_float2(bi.x, bi.y));
            f[i / 2 + 1] = __ffma2_rn(y, make_float2(sc.z, sc.w), make_float2(bi.z, bi.w));
          }
          packed[v / V] = rows::narrow<T>(f);
        }
        if (lane == 0) tc::bulk_wait_read<0>();  // the chunk before has left
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 8; ++j) *reinterpret_cast<uint4*>(out + lane * 128 + ((j ^ (lane & 7)) << 4)) = packed[j];
        if (e.vector != 0 && (c + CW <= n_left || n_left % V == 0)) {  // (a store writes whole 16 bytes: also those that begin inside the tensor and end behind it)
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < M) {
            tc::tma_store_2d(&tmC, out, (int)col0 + c, (int)row0);
            tc::bulk_commit();
          }
        } else {  // rows wherever they lie: a word a lane, 16-bit types as the aligned pairs of a row and what is left at its ends
          __syncwarp();
          const int live = (int)max((int64_t)0, min((int64_t)32, M - row0)), width = min(CW, n_left - c);
          T* dst = reinterpret_cast<T*>(e.c) + row0 * e.ldc + col0 + c;
          const bool odd0 = ((reinterpret_cast<uintptr_t>(dst) >> 1) & 1) != 0, flip = (e.ldc & 1) != 0;
          const uint32_t place = (uint32_t)(((lane >> 2) << 4) + (lane & 3) * 4);
          auto eight = [&](int i0, auto all) {  // rows i0 .. i0 + 7; `all`: each exists
            uint32_t w[8];  // (loads and stores of eight rows apart: one behind the other they wait for each other)
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = *reinterpret_cast<const uint32_t*>(out + (i0 + j) * 128 + (place ^ (uint32_t)(j << 4)));
            T* to = dst;
#pragma unroll
            for (int j = 0; j < 8; ++j, to += e.ldc) {
              const bool there = decltype(all)::value || i0 + j < live;
              if constexpr (sizeof(T) == 4) {
                if (lane < width && there) *reinterpret_cast<uint32_t*>(to + lane) = w[j];
              } else {
                const uint32_t behind = __shfl_down_sync(0xffffffffu, w[j], 1);
                const bool odd = odd0 != (flip && (j & 1) != 0);
                const int k = 2 * lane + (odd ? 1 : 0);
                const uint32_t v = __byte_perm(w[j], behind, odd ? 0x5432 : 0x3210);
                if (there) {
                  if (k + 1 < width) *reinterpret_cast<uint32_t*>(to + k) = v;
                  const bool begin = odd && lane == 0;
                  if (begin || k + 1 == width) *reinterpret_cast<uint16_t*>(to + (begin ? 0 : k)) = (uint16_t)(begin ? w[j] : v);
                }
              }
            }
          };
          if (sizeof(T) == 2 && width == 2) {  // at an odd address both are ends, and the first lane's: here a row a lane writes them.  (Two stores of ends in the loop: 32768 x 4001 x 600 122 -> 162 us.)
            const uint32_t both = *reinterpret_cast<const uint32_t*>(out + lane * 128 + ((lane & 7) << 4));
            uint16_t* to = reinterpret_cast<uint16_t*>(dst + lane * e.ldc);
            if (lane < live) { to[0] = (uint16_t)both; to[1] = (uint16_t)(both >> 16); }
          } else {
#pragma unroll 1
            for (int i0 = 0; i0 < live; i0 += 8, dst += 8 * e.ldc) {
              if (i0 + 8 <= live) eight(i0, std::true_type());
              else eight(i0, std::false_type());
            }
          }
          __syncwarp();
        }
      }
    }
    if (lane == 0) tc::bulk_wait_all();
    for (; tile < tiles; tile += step) {  // a wait has given up: what this warp leaves unwritten is NaN
      int m, width;
      int64_t col;
      tile_at(tile, m, col, width);
      const int64_t row = (int64_t)m * PAIR_ROWS + rank * BM + quarter * 32 + lane, n_left = min((int64_t)width, N - col);
      if (row < M)
        for (int c = 0; c < n_left; ++c)
          if ((c / CW & 1) == half) reinterpret_cast<T*>(e.c)[row * e.ldc + col + c] = Elem<T>::down(__uint_as_float(0x7fffffffu));
    }
  }

  __syncwarp();
  tc::tc_fence_before_sync();
  __syncthreads();
  if (threadIdx.x == 0 && abort_flag != 0u) {
    if (status != nullptr) atomicOr(status, AVE_GDN_DEV_WAIT_EXPIRED);
    tc::st_cluster_u32(tc::mapa(tc::smem_u32(const_cast<uint32_t*>(&abort_flag)), rank ^ 1u), 1u);
  }
  tc::cluster_sync();  // neither CTA ends, or gives tensor memory back, while the other may reach it
  if (abort_flag != 0u) {  // in both or in neither: copies and products may be on their way, all counted at the leader's barriers, and arrivals of finished products at either's
    if (threadIdx.x == 0) {
      const uint32_t blocks = ended[0], accs = ended[1];
      for (uint32_t i = blocks > (uint32_t)stages ? blocks - (uint32_t)stages : 0u; i < blocks; ++i) tc::drain(&empty[i % stages], i / stages & 1u);
      for (uint32_t i = accs > 2u ? accs - 2u : 0u; i < accs; ++i) tc::drain(&acc_full[i & 1u], i >> 1 & 1u);
    }
    if (rank == 0 && threadIdx.x == 0) {
      const uint32_t own = issued[0], other = issued[1], all = own > other ? own : other, begin = all > (uint32_t)stages ? all - (uint32_t)stages : 0u;
      auto bytes = [&](uint32_t i) { return landing(width_at(first + i / (uint32_t)kb_count * step)); };
      for (uint32_t i = own; i < other; ++i) tc::mbar_expect_tx(&full[i % stages], bytes(i));       // the other CTA's alone
      for (uint32_t i = other; i < own; ++i) tc::mbar_complete_tx(&full[i % stages], bytes(i));    // this one's alone
      for (uint32_t i = begin; i < all; ++i) tc::drain(&full[i % stages], i / stages & 1u);
    }
    if (warp == 1) {
      if (rank == 0 && tc::elect_one()) tc::mma_commit_pair(&drained);
      __syncwarp();
      tc::drain(&drained, 0u);
    }
    tc::cluster_sync();
  }
  if (warp == 1) {
    tc::tc_fence_after_sync();
    tc::tmem_dealloc_pair(tmem_base, 512);
  }
}

// ------------------------------------------------------------------------------------------------ few rows
struct Plan { int bn, split, stages, ks, a_rows; int64_t cost; };  // tile width, CTAs a tile, ring depth, blocks of 128 a stage, rows of A, bytes (see make_plan)

template <class T>
__global__ void __launch_bounds__(THREADS, 1)
gemm_int8_cluster_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Epilogue e, int64_t M, int64_t N, int64_t K,
                         uint32_t* status, const Plan plan, uint32_t tmem_cols) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = tc::align1024(smem_raw);
  __shared__ uint64_t full[STAGES], empty[STAGES], acc_full, drained;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile uint32_t abort_flag, failed;  // of this CTA; of any of the cluster
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int bn = plan.bn, split = plan.split, stages = plan.stages;
  const int a_bytes = plan.a_rows * BK, b_bytes = bn * BK, stage_bytes = plan.ks * (a_bytes + b_bytes);
  const int kb_count = (int)((K + plan.ks * BK - 1) / (plan.ks * BK));  // in stages of ks blocks
  const int rank = (int)(blockIdx.x % split), tn = (int)(blockIdx.x / split);
  const int per = (kb_count + split - 1) / split, kb0 = rank * per, kb1 = min(kb_count, kb0 + per);

  pdl_trigger();
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) { tc::mbar_init(&full[s], 1); tc::mbar_init(&empty[s], 1); }
    tc::mbar_init(&acc_full, 1);
    tc::mbar_init(&drained, 1);
    abort_flag = failed = 0;
    tc::fence_barrier_init();
    tc::prefetch_tmap(&tmA);
    tc::prefetch_tmap(&tmB);
  }
  if (warp == 1) tc::tmem_alloc(&tmem_slot, tmem_cols);
  tc::tc_fence_before_sync();
  __syncthreads();
  tc::tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  if (warp == 0 && lane == 0)  // the weights towards L2 while the kernel in front still runs (see gemm_int8_stream_kernel)
    for (int kb = kb0 * plan.ks; kb < min(kb1, kb0 + stages) * plan.ks; ++kb) tc::tma_prefetch_2d(&tmB, kb * BK, tn * bn);
  pdl_wait();

  // Both issuing warps run their loops whole and elect a lane for the instructions themselves.  A stage holds `ks` blocks of 128 along K,
  // [A][A].. [B][B].., behind one barrier.
  int turns = 0;  // stages that this warp has asked for, or issued the products of
  if (warp == 0) {
    int s = 0; uint32_t ph = 0;
    for (int kb = kb0; kb < kb1; ++kb, ++turns) {
      if (turns >= stages && !tc::mbar_wait_together(&empty[s], ph ^ 1u, &abort_flag)) break;
      if (tc::elect_one()) {
        uint8_t* st = smem + s * stage_bytes;
        tc::mbar_expect_tx(&full[s], (uint32_t)stage_bytes);
        for (int j = 0; j < plan.ks; ++j) tc::tma_load_2d(st + plan.ks * a_bytes + j * b_bytes, &tmB, &full[s], (kb * plan.ks + j) * BK, tn * bn);
        for (int j = 0; j < plan.ks; ++j) tc::tma_load_2d(st + j * a_bytes, &tmA, &full[s], (kb * plan.ks + j) * BK, 0);
      }
      __syncwarp();
      if (++s == stages) { s = 0; ph ^= 1u; }
    }
  } else if (warp == 1) {
    const uint32_t idesc = idesc_i8(BM, bn);
    int s = 0; uint32_t ph = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb, ++turns) {
      if (!tc::mbar_wait_together(&full[s], ph, &abort_flag)) { ok = false; break; }
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
    if (ok && tc::elect_one()) tc::mma_commit(&acc_full);
  }
  __syncwarp();  // the other lanes of the issuing warps must not poll beside them
  // the accumulator is complete, so every operand tile has landed and been read
  (void)tc::mbar_wait_unrolled(&acc_full, 0, &abort_flag);
  tc::tc_fence_after_sync();
  __syncwarp();
  tc::cluster_sync();  // ... in every CTA of the cluster: the rings may be overwritten
  if (warp < 2) {  // beside the exchange: nothing is on its way when the CTA ends
    const bool ok = abort_flag == 0u;  // (all waits are over: the same for the whole CTA, and one that has given up late has left its copies behind as well)
    auto last = [&](uint64_t* bars) {  // a stage a lane (one behind the other in front of the cluster's meeting: 8 x 12352 x 2048 8.1 -> 9.0 us)
      const int i = turns - 1 - lane;
      if (lane < stages && i >= 0) tc::drain(&bars[i % stages], (uint32_t)(i / stages) & 1u);
      __syncwarp();
    };
    if (warp == 1) last(empty);
    else if (!ok) {
      last(full);
      if (lane < split) tc::st_cluster_u32(tc::mapa(tc::smem_u32(const_cast<uint32_t*>(&failed)), (uint32_t)lane), 1u);
    }
    if (!ok && warp == 1) {
      if (turns == kb1 - kb0) tc::drain(&acc_full, 0u);
      tc::drain_mmas(&drained);
    }
  }
  const int rows = (int)M, slice = (rows + split - 1) / split, pitch = bn + 4;
  if (warp >= 2) {
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
    const bool whole = failed == 0u;
    for (int i = threadIdx.x; i < mine * vec; i += THREADS) {
      const int r = i / vec, c = (i - r * vec) * 8;
      int32_t x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
      for (int s = 0; s < split; ++s) {
        const int4 a = *reinterpret_cast<const int4*>(part + (s * slice + r) * pitch + c), b = *reinterpret_cast<const int4*>(part + (s * slice + r) * pitch + c + 4);
        x[0] += a.x; x[1] += a.y; x[2] += a.z; x[3] += a.w;
        x[4] += b.x; x[5] += b.y; x[6] += b.z; x[7] += b.w;
      }
      const int64_t col = (int64_t)tn * bn + c, at = rank * slice + r;
      const float a_scale = whole ? e.a_scale[at] : __uint_as_float(0x7fffffffu);  // (sums that miss a share: NaN)
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
  if (threadIdx.x == 0 && abort_flag != 0u && status != nullptr) atomicOr(status, AVE_GDN_DEV_WAIT_EXPIRED);
  __syncthreads();
  if (warp == 1) {
    tc::tc_fence_after_sync();
    tc::tmem_dealloc(tmem_base, tmem_cols);
  }
}

// Tile width, K split and ring depth for at most 128 rows: among the cluster sizes that still give every tile its SMs, the one with the fewest bytes through
// the busiest SM (its operand tiles, plus what the exchange costs).  `clusters[s]`: clusters of s CTAs that run at once.  No plan (bn == 0): more tiles than SMs.
Plan make_plan(int64_t M, int64_t N, int64_t K, const int* clusters) {
  const int64_t kb = (K + BK - 1) / BK, a_rows = (M + 7) / 8 * 8;
  Plan best{};
  best.cost = INT64_MAX;
  for (int split = 1; split <= 8; ++split) {
    const int64_t tiles = clusters[split];
    if (tiles == 0) continue;
    const int64_t bn = ((N + tiles - 1) / tiles + 15) / 16 * 16, block = (a_rows + bn) * BK;
    if (bn > BN) continue;
    // blocks a stage: up to 48 KB a stage, at least three stages, no padding of K beyond one block a CTA
    int ks = 1;
    while (ks < 8 && 2 * ks * block <= 49152 && 2 * ks * split <= kb) ks *= 2;
    const int64_t steps = (kb + ks - 1) / ks, per = (steps + split - 1) / split;
    if ((split - 1) * per >= steps) continue;  // no CTA without work
    const int64_t stage = ks * block, exchange = split == 1 ? 0 : 65536 + a_rows * bn * 4;
    const int64_t least = ks > 2 ? ks * 8192 : 16384;
    const int64_t cost = per * (stage > least ? stage : least) + exchange;
    if (cost < best.cost) best = {(int)bn, split, (int)(RING / stage < STAGES ? RING / stage : STAGES), ks, (int)a_rows, cost};
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

// ------------------------------------------------------------------------------------------------ one to four rows
// The time is that of streaming B and, from two rows on, of the products: four a lane and instruction (dp4a, of which an SM takes about 11 lanes a cycle).  A warp takes
// R rows of B, 16 loads of 512 bytes on their way, and MT rows of A from L1; with WK == 4 the warps of a CTA share the same rows of B, each a part of K.  The lanes' sums
// meet in one reduction each.  (The bytes of a piece behind K are cleared in A. They are read with the bytes in front of them in one aligned piece, behind the last row of an operand as well, and
// may be anything.)
template <class T, int MT, int R, int WK>
__global__ void __launch_bounds__(128) gemm_int8_stream_kernel(const int8_t* A, const int8_t* B, const Epilogue e, int M, int64_t N, int K, int64_t lda, int64_t ldb) {
  constexpr int PU = 16 / R;  // pieces of a row at a time
  __shared__ int32_t part[WK][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, turn = WK == 1 ? 0 : warp;
  const int64_t n0 = (WK == 1 ? (int64_t)blockIdx.x * 4 + warp : (int64_t)blockIdx.x) * R;
  pdl_trigger();
  // The weights towards L2 while the kernel in front still runs: nothing of them is read here, so it does not matter who writes them.  (A layer's two projections of one row
  // behind norm and rounding, weights from HBM: 13.3 us, 12.6 so, eight rows on clusters 18.6 and 17.6; with weights that L2 holds it costs a product 0.5 us, and so it does
  // in the pairs, which do without: 128 rows 22.8 and 23.3.)
  for (int r = 0; r < R; ++r)
    for (int k = turn * PU * 512 + lane * 128; k < K && n0 + r < N; k += WK * PU * 512)
      if (lane * 128 < PU * 512) asm volatile("prefetch.global.L2 [%0];" ::"l"(B + (n0 + r) * ldb + k));
  pdl_wait();
  if (n0 >= N) return;  // (the whole CTA, or with WK == 1 a warp, which meets no other)
  int32_t sum[MT][R] = {};
  const int8_t* b = B + n0 * ldb;
  for (int k0 = turn * PU * 512; k0 < K; k0 += WK * PU * 512) {
    uint4 w[R][PU];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int p = 0; p < PU; ++p) {
        const int k = k0 + p * 512 + lane * 16;
        w[r][p] = make_uint4(0, 0, 0, 0);
        if (k < K && n0 + r < N)
          asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[r][p].x), "=r"(w[r][p].y), "=r"(w[r][p].z), "=r"(w[r][p].w) : "l"(b + r * ldb + k));
      }
#pragma unroll
    for (int p = 0; p < PU; ++p) {
      const int k = k0 + p * 512 + lane * 16;
      if (k >= K) break;
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (m >= M) break;
        uint4 x = *reinterpret_cast<const uint4*>(A + m * lda + k);
        if (k + 16 > K) {
          uint32_t* words = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int there = K - k - 4 * i;  // bytes of this word in front of K
            words[i] = there >= 4 ? words[i] : there <= 0 ? 0u : words[i] & ((1u << (8 * there)) - 1u);
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          sum[m][r] = __dp4a((int)w[r][p].x, (int)x.x, sum[m][r]);
          sum[m][r] = __dp4a((int)w[r][p].y, (int)x.y, sum[m][r]);
          sum[m][r] = __dp4a((int)w[r][p].z, (int)x.z, sum[m][r]);
          sum[m][r] = __dp4a((int)w[r][p].w, (int)x.w, sum[m][r]);
        }
      }
    }
  }
  int32_t mine = 0;  // lane m R + r finishes row m, column r
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int32_t total = __reduce_add_sync(0xffffffffu, sum[m][r]);
      if (lane == m * R + r) mine = total;
    }
  if constexpr (WK > 1) {
    part[warp][lane] = mine;
    __syncthreads();
    if (warp != 0) return;
    mine = 0;
#pragma unroll
    for (int i = 0; i < WK; ++i) mine += part[i][lane];
  }
  const int m = lane / R;
  const int64_t n = n0 + lane % R;
  if (m < M && m < MT && n < N)
    reinterpret_cast<T*>(e.c)[m * e.ldc + n] = Elem<T>::down(finish(mine, e.a_scale[m], e.b_scale[n], bias_at<T>(e, n)));
}

template <class T, int MT, int WK>
int run_stream(const AveGemmInt8Args& a, const Epilogue& e, cudaStream_t stream) {
  constexpr int R = 4, columns = (WK == 1 ? 4 : 1) * R;  // (one or two rows of B a warp are slower, 12352 x 2048 5.8 and 10.1 us)
  AVE_CUDA_TRY(launch_after(gemm_int8_stream_kernel<T, MT, R, WK>, (unsigned)((a.N + columns - 1) / columns), 128, 0, stream, reinterpret_cast<const int8_t*>(a.a),
                            reinterpret_cast<const int8_t*>(a.b), e, (int)a.M, a.N, (int)a.K, a.lda, a.ldb));
  return AVE_GDN_OK;
}
// Up to two rows, up to four where there is little of B, whatever its shape.  (us, this form and clusters: 1 x 12352 x 2048 5.1 and 7.4, 2 rows 7.0 and 7.5, 4 rows 10.7 and 7.5;
// 2 x 4096 x 4096 6.3 and 6.1, 2 x 400 x 8192 3.6 and 5.1; 4 x 1544 x 2048 5.3 and 4.9, 4 x 12352 x 512 4.7 and 5.0, 4 x 1000 x 512 2.5 and 4.2.)
bool streams(const AveGemmInt8Args& a) {
  const int64_t whole = (a.K + 15) / 16 * 16;
  if ((a.M == 1 && a.lda < whole) || (a.N == 1 && a.ldb < whole)) return false;  // (a single row that ends inside a piece)
  return a.M <= 2 || (a.M <= 4 && a.K <= 1024 && a.N * a.K <= 1 << 23);
}
// K shared by a CTA's warps where there are few warps or long rows (us, shared and not: 1 x 400 x 8192 2.7 and 6.3, 1 x 2048 x 4096 3.0 and 4.0, 1 x 8192 x 8192 7.9 and 9.5,
// 1 x 4096 x 4096 4.8 and 4.4, 1 x 12352 x 2048 8.5 and 5.1)
template <class T>
int launch_stream(const AveGemmInt8Args& a, const Epilogue& e, cudaStream_t stream) {
  if (a.M > 2) return run_stream<T, 4, 1>(a, e, stream);
  if (a.K > 4096 || (a.K > 2048 && a.N < 4 * 592)) return a.M == 1 ? run_stream<T, 1, 4>(a, e, stream) : run_stream<T, 2, 4>(a, e, stream);
  return a.M == 1 ? run_stream<T, 1, 1>(a, e, stream) : run_stream<T, 2, 1>(a, e, stream);
}

// Width of the pairs' column tiles and what a product with it takes, in ns.  A block of 128 of K takes 112, 138, 194 and 265 ns with 64, 128, 192 and 256 columns where every
// pair has one tile at most (the narrow ones wait for their operands, 20 to 28 KB a CTA and block), and 208, 277, 347 and 417 where all are busy for longer (L2 and the power cap;
// 8192 x 2048 x 4096 with 256 columns 55 us, 61 with 192), a tile's results at least 9 ns a column, and launch, first operands and last results 4 us and 6 ns a column.
// `across`: rows of operands that do not lie on 128 bytes, whose blocks reach across two lines each (256 rows x 1544 x 2048 6.1 us, with 1999 of 2000 bytes 8.2).
struct Width { int bn; int64_t ns; bool halves; };  // halves: the last turn's tiles are taken as two each
Width pair_width(int64_t M, int64_t N, int64_t K, bool across, int pairs) {
  constexpr int alone_ns[4] = {112, 138, 194, 265}, busy_ns[4] = {208, 277, 347, 417};
  const int64_t mt = (M + PAIR_ROWS - 1) / PAIR_ROWS, kb = (K + BK - 1) / BK;
  Width best{0, INT64_MAX, false};
  for (int bn = BN; bn >= 64; bn -= 64) {
    const int64_t turns = (mt * ((N + bn - 1) / bn) + pairs - 1) / pairs, block = (turns > 1 ? busy_ns : alone_ns)[bn / 64 - 1];
    const int64_t products = kb * block * (across ? 4 : 3) / 3, results = 300 + 9 * bn;
    const int64_t turn = products > results ? products : results, left = mt * ((N + bn - 1) / bn) % pairs;
    // a last turn of at most half of the pairs in halves: their products take two thirds of the time (8192 x 2048 x 4096, 3.5 turns, 55 us, 50
    // so; 2048 x 12352 x 2048 43 and 41)
    const bool halves = bn == BN && turns > 1 && left > 0 && 2 * left <= pairs;
    const int64_t ns = 4000 + 6 * bn + turns * turn - (halves ? turn / 3 : 0);
    if (ns < best.ns) best = {bn, ns, halves};
  }
  return best;
}
template <class T>
int launch_pairs(const AveGemmInt8Args& a, const Epilogue& e, const Width& width, int pairs, cudaStream_t stream) {
  const int bn = width.bn;
  CUtensorMap tmA, tmB, tmC{};
  int rc = operand_map(&tmA, a.a, a.M, a.K, a.lda, BM);
  if (rc != AVE_GDN_OK) return rc;
  rc = operand_map(&tmB, a.b, a.N, a.K, a.ldb, width.halves ? bn / 4 : bn / 2);
  if (rc != AVE_GDN_OK) return rc;
  if (e.vector != 0) {
    const uint64_t size = sizeof(T), dims[2] = {(uint64_t)a.N, (uint64_t)a.M}, strides[2] = {size, (uint64_t)a.ldc * size};
    const uint32_t box[2] = {128 / (uint32_t)sizeof(T), 32};
    const CUtensorMapDataType dt = sizeof(T) == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16;
    rc = make_tmap(&tmC, dt, (int)size, a.c, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (rc != AVE_GDN_OK) return rc;
  }
  const int64_t tiles = ((a.M + PAIR_ROWS - 1) / PAIR_ROWS) * ((a.N + bn - 1) / bn);
  if (tiles > INT32_MAX) return AVE_GDN_UNSUPPORTED;
  const uint32_t whole = (uint32_t)(width.halves ? tiles / pairs * pairs : tiles);
  auto launch = [&](auto blocks) {
    constexpr int KS = decltype(blocks)::value;
    constexpr auto* kernel = &gemm_int8_pair_kernel<T, KS>;
    const int rc = allow_smem<kernel>(PAIR_SMEM);
    if (rc != AVE_GDN_OK) return rc;
    const int fit = PAIR_RING / (KS * (BM + bn / 2) * BK), stages = fit < PAIR_STAGES ? fit : PAIR_STAGES;
    AVE_CUDA_TRY(launch_after(kernel, (unsigned)(2 * (tiles < pairs ? tiles : pairs)), PAIR_THREADS, PAIR_SMEM, stream, tmA, tmB, tmC, e, a.M, a.N, a.K, a.status, bn, stages, whole));
    return (int)AVE_GDN_OK;
  };
  if (bn <= 128) return launch(std::integral_constant<int, 2>());
  return launch(std::integral_constant<int, 1>());
}

template <class T>
int launch_t(const AveGemmInt8Args& a, cudaStream_t stream) {
  int dev = 0, sms = 148;
  AVE_CUDA_TRY(cudaGetDevice(&dev));
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  const int size = (int)sizeof(T);
  const Epilogue e{a.a_scale, a.b_scale, a.bias, a.c, a.ldc, a.bias_dtype == AVE_DTYPE_FP32, aligned16(a.c) && rows::on16(a.ldc, size)};
  if (streams(a)) return launch_stream<T>(a, e, stream);
  const int* clusters = cluster_counts(dev, sms);
  if (clusters == nullptr || clusters[2] == 0) return AVE_GDN_UNSUPPORTED;
  // The pairs from 129 rows on, and from 64 where they take less by the two estimates: a cluster's 4.2 us and what comes through its busiest SM at 60 bytes a ns.
  // (us, clusters and pairs: N = 12352, K = 2048, 32 rows 8.2 and 9.5, 64 rows 9.7 and 8.4, 128 rows 13.7 and 8.6; N = 2048, K = 4096, 7.9 and 7.9, 7.7 and 7.9,
  // 10.3 and 7.9; N = 1544, K = 2048, 5.6 and 6.1, 5.6 and 6.1, 6.3 and 6.1.)
  const int pairs = clusters[2];
  const Width width = pair_width(a.M, a.N, a.K, a.lda % 128 != 0 || a.ldb % 128 != 0, pairs);
  Plan plan{};
  if (a.M <= BM) plan = make_plan(a.M, a.N, a.K, clusters);
  if (plan.bn == 0 || (a.M >= 64 && width.ns <= 4200 + plan.cost / 60)) return launch_pairs<T>(a, e, width, pairs, stream);
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
  const int64_t ctas = (a.N + plan.bn - 1) / plan.bn * plan.split;
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
