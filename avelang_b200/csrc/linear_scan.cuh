// The chunked scan of linear attention with a decay for each head, for one segment of one (sequence, value head):
//     H^T  state [dv lanes][dk], fp32 in registers, with bf16 images in TMEM
//     P    = X Y^T            masked and decayed: P'_ts = scale_p e^{G_t - G_s} P_ts for s <= t
//     O^T  = e_t (H^T X^T) + W^T P'^T
//     H^T <- decay H^T + W^T Yw,     Yw_s = w_s Y_s
// over chunks of 64 tokens, X, Y, W = q, k, v in the forward pass.  The gradients are scans of the same form: (do, v, k) forwards gives dq;
// (v, do, q) and (k, q, do) backwards in time give dk and dv, with the mask, the walk over the chunks and the decays' signs turned round.
// G is the sum of the decays' logarithms inside the chunk, so every exponent of a product that counts is <= 0 for g <= 0.
#pragma once
#include "common.cuh"
#include "tc.cuh"
#include "warpmma.cuh"

namespace ave {
namespace {
namespace lin {

constexpr int C = 64;       // tokens of a chunk
constexpr int TILE = 16384; // bytes of a tile: 64 tokens x 128 features (64 features: the first half)
constexpr int HALF = 8192;  // 64 tokens x 64 features

// Segments: sequence n's tokens are cut every `len` tokens, counted from its first.  Segment j of sequence n has slot
// floor(first token / len) + n + j: unique, and increasing with the sequence, while the offsets are monotone inside [0, T].
struct Plan {
  int len;       // a multiple of 64
  int cut;       // whether a sequence can have more than one segment
  int64_t slots; // of all sequences
};
struct Seg { int n, j, count, b, t0, len; bool ok; };  // t0, len: of the segment

// What a scan reads and writes.  Heads of an operand: value head h reads head h / div.
struct Args {
  const int32_t* cu_seqlens;
  uint32_t* status;
  int B, T, Hv, n_seqs, num_slots;
  const int32_t* state_indices;
  int x_div, y_div, w_div, e_div;
  const float* g;
  int64_t g_stride_b, g_stride_t;
  float scale_p, scale_e, scale_w;
  void* o;                         // bf16
  int64_t o_stride_b, o_stride_t, o_stride_h;
  float* o_part;                   // fp32 [B, T, Hv, dv] instead, for a sum over heads behind the scan
  const float* state_in;           // [slot, Hv, ..]: element (y feature, w feature) at y * st_y + w * st_w
  float* state_out;
  int st_y, st_w;
  float* seg_state;                // [segment slot, Hv, ..] likewise
  float* seg_decay;                // [segment slot, Hv]
  float* inter;                    // [dv / 32][Hv][B T]: e_t E_t . (H^T X_t), 32 features each      (for the gradient of g)
  float* intra;                    // [Hv][B T]: sum over s < t of P'_ts (E_t . W_s)
  Plan plan;
};
struct Maps { CUtensorMap x, y, w, e, o, o32; bool o_ok; };

__device__ __forceinline__ int64_t first_slot(const Args& a, int n) {
  return (a.cu_seqlens ? (int64_t)a.cu_seqlens[n] : (int64_t)n * a.T) / a.plan.len + n;
}
__device__ __forceinline__ Seg seg_of_slot(const Args& a, int64_t slot) {
  Seg s{0, 0, 0, 0, 0, 0, false};
  if (a.plan.cut) {
    int lo = 0, hi = a.n_seqs;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first_slot(a, mid) <= slot) lo = mid; else hi = mid;
    }
    s.n = lo;
    s.j = (int)(slot - first_slot(a, lo));
  } else {
    s.n = (int)slot;
  }
  const SeqSpan sp = seq_span(a.cu_seqlens, s.n, a.T, nullptr);
  const int64_t begin = (int64_t)s.j * a.plan.len;
  if (!sp.ok || s.j < 0 || (begin >= sp.len && s.j > 0)) return s;
  s.count = a.plan.cut ? max(1, (sp.len + a.plan.len - 1) / a.plan.len) : 1;
  s.b = sp.b; s.t0 = sp.t0 + (int)begin;
  s.len = a.plan.cut ? (int)min((int64_t)a.plan.len, sp.len - begin) : sp.len;
  s.ok = true;
  return s;
}
// A packed batch whose offsets are not monotone inside [0, T] is skipped as a whole.  Called by the whole CTA.
__device__ __forceinline__ bool offsets_fit(const Args& a, bool flag) {
  if (a.cu_seqlens == nullptr) return true;
  int bad = 0;
  for (int n = threadIdx.x; n < a.n_seqs; n += blockDim.x) {
    const int x = a.cu_seqlens[n], y = a.cu_seqlens[n + 1];
    bad |= (x < 0 || y < x || y > a.T) ? 1 : 0;
  }
  bad = __syncthreads_or(bad);
  if (bad && flag && threadIdx.x == 0 && a.status != nullptr) atomicOr(a.status, AVE_GDN_DEV_BAD_SEQLEN);
  return bad == 0;
}

// Shared memory: a ring of stages {X, Y, W, (E), gate vectors}, then the three terms of Yw and the two of P'
// Gate vectors of a chunk, floats: e[64] | w[64] | G hi[64] | G lo[64] | e^{-|G_i - G_31|}[64] (signs for g <= 0) | decay (and padding to 64 bytes)
constexpr int GATES = 1344;
constexpr int GV_E = 0, GV_W = 64, GV_H = 128, GV_L = 192, GV_F = 256, GV_TOT = 320;
template <bool kState, bool kGrad>
struct Cfg {
  static constexpr int TILES = kState ? 2 : kGrad ? 4 : 3;
  static constexpr int X = 0, Y = kState ? 0 : TILE, W = Y + TILE, E = W + TILE;
  static constexpr int STAGE = TILES * TILE;
  static constexpr int STAGES = kState ? 3 : kGrad ? 2 : 3;
  static constexpr int YW = STAGES * STAGE, PP = YW + 3 * TILE, GV = PP + (kState ? 0 : TILE), BARS = GV + STAGES * GATES;
  static constexpr int SMEM = BARS + 256 + 1024;
  static_assert(SMEM <= 232448, "shared memory of an SM");
  // TMEM columns; with the gradient of g the state has three terms, W^T P'^T takes the columns of P and H^T X^T has one accumulator
  static constexpr uint32_t P = 0, PE = 64, OI = kGrad ? 128 : 64, OA = kGrad ? 0 : 192, DS = kState ? 0 : kGrad ? 192 : 256, H = kGrad ? 320 : 384, COLS = kState ? 128 : 512;
  static constexpr int HT = kGrad ? 3 : 2;
  static constexpr uint32_t OI2 = kGrad ? 0 : 64;  // H^T X^T has a second accumulator
};

constexpr int THREADS = 640;  // warpgroups: P' (two warps, whose lanes are the chunk's rows), loader and gates, issuer; two for the state; outputs; Yw
constexpr int REGS_LAUNCH = 96, REGS_CTRL = 80, REGS_STATE = 112, REGS_OUT = 104, REGS_PREP = 72;
static_assert(REGS_CTRL + 2 * REGS_STATE + REGS_OUT + REGS_PREP <= 5 * REGS_LAUNCH, "register redistribution exceeds the launch allocation");
static_assert(THREADS * REGS_LAUNCH <= 65536, "launch allocation exceeds the register file");

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int DK, int DV, bool kRev, bool kState, bool kGrad>
__global__ void __launch_bounds__(THREADS, 1) scan_kernel(const Args a, const __grid_constant__ Maps maps) {
  using K = Cfg<kState, kGrad>;
  static_assert(!(kState && kGrad), "states alone have no outputs");
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = tc::align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + K::BARS);
  uint64_t* full = bars;           // [3] tiles of the stage landed
  uint64_t* gates = bars + 3;      // [3] its gate vectors written
  uint64_t* empty = bars + 6;      // [3] the stage is read
  uint64_t* p_full = bars + 9;     // P (and E W^T) accumulated
  uint64_t* pp_ready = bars + 10;  // P' written, P drained
  uint64_t* yw_ready = bars + 11;  // Yw written, W cleared behind the sequence
  uint64_t* ds_full = bars + 12;   // increment accumulated, Yw read
  uint64_t* ds_empty = bars + 13;  // increment drained
  uint64_t* h_ready = bars + 14;   // images of the state written
  uint64_t* h_read = bars + 15;    // H^T X^T accumulated
  uint64_t* o_full = bars + 16;    // both outputs accumulated, P' read
  uint64_t* o_empty = bars + 17;   // outputs drained
  uint64_t* mma_end = bars + 18;   // the MMAs are complete, when a wait has expired
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 19);
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < K::STAGES; ++i) {
      tc::mbar_init(&full[i], 1); tc::mbar_init(&gates[i], 1);
      tc::mbar_init(&empty[i], kState ? 9 : 12);  // the state's warps have read the decay, and: the issuer's commit, or the output warps
    }
    for (uint64_t* b : {p_full, ds_full, h_read, o_full, mma_end}) tc::mbar_init(b, 1);
    tc::mbar_init(pp_ready, 2); tc::mbar_init(yw_ready, 4);
    tc::mbar_init(ds_empty, 8); tc::mbar_init(h_ready, 8);
    tc::mbar_init(o_empty, 4);
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  pdl_wait();
  if (!offsets_fit(a, true)) return;
  const int h = blockIdx.x % a.Hv;
  const int64_t seg_slot = blockIdx.x / a.Hv;
  const Seg seg = seg_of_slot(a, seg_slot);
  if (!seg.ok) return;
  const bool last = kRev ? seg.j == 0 : seg.j == seg.count - 1;
  if (kState && last) return;  // nobody takes its state from here: the scan itself ends with it
  int slot = seg.n;
  if (a.state_indices != nullptr) {
    slot = a.state_indices[seg.n];
    if (slot >= a.num_slots) {
      if (a.status != nullptr && threadIdx.x == 0) atomicOr(a.status, AVE_GDN_DEV_BAD_SLOT);
      slot = -1;
    }
  }
  if (kState && slot < 0) return;
  const int64_t state_tile = ((int64_t)slot * a.Hv + h) * (DK * DV), seg_tile = (seg_slot * a.Hv + h) * (int64_t)(DK * DV);
  if constexpr (!kState) {
    __nv_bfloat16* og = reinterpret_cast<__nv_bfloat16*>(a.o) + seg.b * a.o_stride_b + (int64_t)h * a.o_stride_h;
    if (slot < 0) {  // skipped sequence: zero output, no state access
      for (int64_t e = threadIdx.x; e < (int64_t)seg.len * DV; e += THREADS) og[(seg.t0 + e / DV) * a.o_stride_t + e % DV] = __float2bfloat16(0.f);
      return;
    }
    if (seg.len == 0) {  // a sequence of no tokens hands its state on
      if (a.state_out != nullptr && a.state_out != a.state_in)
        for (int e = threadIdx.x; e < DK * DV; e += THREADS) a.state_out[state_tile + e] = a.state_in ? a.state_in[state_tile + e] : 0.f;
      return;
    }
  }
  const int n_chunks = (seg.len + C - 1) / C;
  auto chunk_at = [&](int c) { return kRev ? n_chunks - 1 - c : c; };  // place of the c-th chunk of the walk
  if (warp == 3) tc::tmem_alloc(tmem_slot, K::COLS);
  tc::tc_fence_before_sync();
  __syncthreads();
  tc::tc_fence_after_sync();
  const uint32_t tm = *tmem_slot;
  auto all = [](bool done) { return __all_sync(0xffffffffu, done) != 0; };

  if (warp < 4) {
    tc::reg_set<REGS_CTRL, REGS_LAUNCH>();
    if (warp < 2) {
      if constexpr (!kState) {
        // -------------------------------------------------------------- P': row t a lane
        const int t = 32 * warp + lane, r8 = lane & 7;
        const uint32_t lane_addr = tm + ((uint32_t)(32 * warp) << 16);
        int s = 0;
        uint32_t ph = 0;
        for (int c = 0; c < n_chunks; ++c) {
          const uint32_t cp = (uint32_t)c & 1u;
          const int at_tok = chunk_at(c) * C, len = min(C, seg.len - at_tok);
          if (!all(tc::mbar_wait3(p_full, cp, &gates[s], ph, o_full, cp ^ 1u, abort_flag))) break;
          tc::tc_fence_after_sync();
          const float* gv = reinterpret_cast<const float*>(smem + K::GV + s * GATES);
          uint8_t* row = smem + K::PP + t * 128;
          [[maybe_unused]] float sum = 0.f;
          // 16 columns from 16 k on, with factors f(column)
          auto step = [&](int k, auto factors, bool diagonal) {
            uint32_t x[16], hi[8], lo[8];
            [[maybe_unused]] uint32_t pe[16];
            tc::tmem_ld16(lane_addr + K::P + 16 * k, x);
            if constexpr (kGrad) tc::tmem_ld16(lane_addr + K::PE + 16 * k, pe);
            tc::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
              float p[4];
              factors(16 * k + i, p);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                p[j] *= __uint_as_float(x[i + j]);
                const int col = 16 * k + i + j;
                // what is masked may be anything; backwards also what lies behind the sequence
                if (diagonal && (kRev ? col < t : col > t)) p[j] = 0.f;
                if (kRev && col >= len) p[j] = 0.f;
                if constexpr (kGrad) {
                  const bool counts = !(diagonal && (kRev ? col <= t : col >= t)) && !(kRev && col >= len);
                  sum += counts ? p[j] * __uint_as_float(pe[i + j]) : 0.f;
                }
              }
              split_pair(make_float2(p[0], p[1]), hi[i / 2], lo[i / 2]);
              split_pair(make_float2(p[2], p[3]), hi[i / 2 + 1], lo[i / 2 + 1]);
            }
            *reinterpret_cast<uint4*>(row + (((2 * k) ^ r8) << 4)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            *reinterpret_cast<uint4*>(row + (((2 * k + 1) ^ r8) << 4)) = make_uint4(hi[4], hi[5], hi[6], hi[7]);
            *reinterpret_cast<uint4*>(row + HALF + (((2 * k) ^ r8) << 4)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            *reinterpret_cast<uint4*>(row + HALF + (((2 * k + 1) ^ r8) << 4)) = make_uint4(lo[4], lo[5], lo[6], lo[7]);
          };
          if (warp == (kRev ? 0 : 1)) {  // the 32 x 32 block off the diagonal: a factor a row and one a column, meeting at token 31
            const float r = a.scale_p * gv[GV_F + t];
#pragma unroll 1
            for (int k = kRev ? 2 : 0; k < (kRev ? 4 : 2); ++k)
              step(k, [&](int col, float (&p)[4]) {
                const float4 f = *reinterpret_cast<const float4*>(gv + GV_F + col);
                p[0] = r * f.x; p[1] = r * f.y; p[2] = r * f.z; p[3] = r * f.w;
              }, false);
          }
          const float gh = gv[GV_H + t], gl = gv[GV_L + t];
#pragma unroll 1
          for (int k = 2 * warp; k < 2 * warp + 2; ++k)
            step(k, [&](int col, float (&p)[4]) {
              const float4 h4 = *reinterpret_cast<const float4*>(gv + GV_H + col), l4 = *reinterpret_cast<const float4*>(gv + GV_L + col);
              p[0] = a.scale_p * ex2((gh - h4.x) + (gl - l4.x)); p[1] = a.scale_p * ex2((gh - h4.y) + (gl - l4.y));
              p[2] = a.scale_p * ex2((gh - h4.z) + (gl - l4.z)); p[3] = a.scale_p * ex2((gh - h4.w) + (gl - l4.w));
            }, true);
          tc::tc_fence_before_sync();
          tc::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(pp_ready);
          if constexpr (kGrad)
            if (t < len) a.intra[((int64_t)h * a.B + seg.b) * a.T + seg.t0 + at_tok + t] = sum;
          if (++s == K::STAGES) { s = 0; ph ^= 1u; }
        }
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- loader (one lane), and gate vectors, two tokens a lane; sums of logarithms in 64 bits
      if (lane == 0) {
        if (!kState) tc::prefetch_tmap(&maps.x);
        tc::prefetch_tmap(&maps.y); tc::prefetch_tmap(&maps.w);
      }
      constexpr double LOG2E = 1.4426950408889634;
      double seg_total = 0.0;
      const float* g = a.g != nullptr ? a.g + seg.b * a.g_stride_b + h : nullptr;
      auto fetch = [&](int c, int e) {
        const int t = chunk_at(c) * C + 2 * lane + e;
        if (g == nullptr || t >= seg.len) return 0.f;
        const float x = g[(int64_t)(seg.t0 + t) * a.g_stride_t];
        return x < -1e6f ? -1e6f : x;  // (a NaN stays one)
      };
      float n0 = fetch(0, 0), n1 = fetch(0, 1);
      int s = 0, issued = 0;
      uint32_t ph = 1;
      for (int c = 0; c < n_chunks; ++c) {
        if (c >= K::STAGES && !all(tc::mbar_wait(&empty[s], ph, abort_flag))) break;
        if (lane == 0) {
          uint8_t* st = smem + s * K::STAGE;
          const int tok = seg.t0 + chunk_at(c) * C;
          constexpr uint32_t bytes = (kState ? 1 : 2) * (DK / 64) * HALF + (kGrad ? 2 : 1) * (DV / 64) * HALF;
          tc::mbar_expect_tx(&full[s], bytes);
          auto load = [&](const CUtensorMap* m, int at, int halves, int head) {
#pragma unroll
            for (int i = 0; i < halves; ++i) tc::tma_load_4d(st + at + i * HALF, m, &full[s], 64 * i, head, tok, seg.b);
          };
          load(&maps.y, K::Y, DK / 64, h / a.y_div);
          load(&maps.w, K::W, DV / 64, h / a.w_div);
          if constexpr (!kState) load(&maps.x, K::X, DK / 64, h / a.x_div);
          if constexpr (kGrad) load(&maps.e, K::E, DV / 64, h / a.e_div);
        }
        __syncwarp();
        ++issued;
        const double x0 = (double)n0 * LOG2E, x1 = (double)n1 * LOG2E;
        if (c + 1 < n_chunks) { n0 = fetch(c + 1, 0); n1 = fetch(c + 1, 1); }
        double sum = x0 + x1;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double y = __shfl_up_sync(0xffffffffu, sum, o);
          if (lane >= o) sum += y;
        }
        const double total = __shfl_sync(0xffffffffu, sum, 31), mid = __shfl_sync(0xffffffffu, sum, 15);
        const double G0 = sum - x1, G1 = sum;
        seg_total += total;
        const int left = seg.len - chunk_at(c) * C - 2 * lane;  // tokens from this lane's first on
        const double sg = kRev ? -1.0 : 1.0;
        const float2 e = make_float2(a.scale_e * ex2((float)(kRev ? total - G0 : G0)), a.scale_e * ex2((float)(kRev ? total - G1 : G1)));
        float2 w = make_float2(a.scale_w * ex2((float)(kRev ? G0 : total - G0)), a.scale_w * ex2((float)(kRev ? G1 : total - G1)));
        if (left < 1) w.x = 0.f;
        if (left < 2) w.y = 0.f;
        const float2 hi = make_float2((float)(sg * G0), (float)(sg * G1)), lo = make_float2((float)(sg * G0 - hi.x), (float)(sg * G1 - hi.y));
        const bool behind = lane >= 16;
        const float2 f = make_float2(ex2((float)(behind ? G0 - mid : mid - G0)), ex2((float)(behind ? G1 - mid : mid - G1)));
        const float tot = (float)exp2(total);  // exact to the last bit: a state is multiplied by it once a chunk
        float* v = reinterpret_cast<float*>(smem + K::GV + s * GATES);
        reinterpret_cast<float2*>(v + GV_E)[lane] = e;
        reinterpret_cast<float2*>(v + GV_W)[lane] = w;
        reinterpret_cast<float2*>(v + GV_H)[lane] = hi;
        reinterpret_cast<float2*>(v + GV_L)[lane] = lo;
        reinterpret_cast<float2*>(v + GV_F)[lane] = f;
        if (lane == 0) v[GV_TOT] = tot;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&gates[s]);
        if (++s == K::STAGES) { s = 0; ph ^= 1u; }
      }
      if (kState && lane == 0) a.seg_decay[seg_slot * a.Hv + h] = (float)exp2(seg_total);
      // nothing is on its way into the shared memory of a CTA that ends, whatever became of those who wait for it
      if (lane == 0) {
#pragma unroll 1
        for (int c = max(0, issued - K::STAGES); c < issued; ++c) tc::drain(&full[c % K::STAGES], (uint32_t)(c / K::STAGES) & 1u);
      }
    } else {
      // ---------------------------------------------------------------- MMA issuer
      const uint32_t smem0 = tc::smem_u32(smem) >> 4;
      constexpr uint32_t hi_sw = tc::desc_hi(1024, true);
      auto scores = [&](uint32_t at) {  // lanes 0..63 are the chunk's rows; the others multiply what lies behind the tile, and nobody reads them
        if (tc::elect_one()) {
#pragma unroll
          for (int k = 0; k < DK / 16; ++k)
            tc::mma_ss(tm + K::P, tc::smem_desc(at + tc::desc_lo(K::X + (k >> 2) * HALF + 32 * (k & 3), 16), hi_sw),
                       tc::smem_desc(at + tc::desc_lo(K::Y + (k >> 2) * HALF + 32 * (k & 3), 16), hi_sw), tc::idesc_f16(128, 64, 1, 1, false, false), k != 0);
          if constexpr (kGrad) {
#pragma unroll
            for (int k = 0; k < DV / 16; ++k)
              tc::mma_ss(tm + K::PE, tc::smem_desc(at + tc::desc_lo(K::E + (k >> 2) * HALF + 32 * (k & 3), 16), hi_sw),
                         tc::smem_desc(at + tc::desc_lo(K::W + (k >> 2) * HALF + 32 * (k & 3), 16), hi_sw), tc::idesc_f16(128, 64, 1, 1, false, false), k != 0);
          }
          tc::mma_commit(p_full);
        }
        __syncwarp();
      };
      int s = 0;
      uint32_t ph = 0;
      bool ok = all(tc::mbar_wait(&full[0], 0u, abort_flag));
      if constexpr (!kState) {
        tc::tc_fence_after_sync();
        if (ok) scores(smem0);
      }
      for (int c = 0; c < n_chunks && ok; ++c) {
        const uint32_t cp = (uint32_t)c & 1u, at = smem0 + s * (K::STAGE >> 4);
        const int s_next = s + 1 == K::STAGES ? 0 : s + 1;
        const uint32_t ph_next = s_next == 0 ? ph ^ 1u : ph;
        // increment: the smallest terms first
        ok = all(tc::mbar_wait2(yw_ready, cp, ds_empty, cp ^ 1u, abort_flag));
        if (!ok) break;
        tc::tc_fence_after_sync();
        if (tc::elect_one()) {
#pragma unroll
          for (int t = 2; t >= 0; --t)
#pragma unroll
            for (int k = 0; k < 4; ++k)  // 16 tokens a step
              tc::mma_ss(tm + K::DS, tc::smem_desc(at + tc::desc_lo(K::W + 2048 * k, HALF), hi_sw),
                         tc::smem_desc(smem0 + tc::desc_lo(K::YW + t * TILE + 2048 * k, HALF), hi_sw), tc::idesc_f16(128, DK, 1, 1, true, true), !(t == 2 && k == 0));
          tc::mma_commit(ds_full);
          if constexpr (kState) tc::mma_commit(&empty[s]);
        }
        __syncwarp();
        if constexpr (!kState) {
          // (the accumulator that this takes was drained with the outputs of two chunks ago; with one accumulator o_empty has been waited for)
          ok = all(tc::mbar_wait(h_ready, cp, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
          if (tc::elect_one()) {
#pragma unroll
            for (int t = K::HT - 1; t >= 0; --t)
#pragma unroll
              for (int k = 0; k < DK / 16; ++k)
                tc::mma_ts(tm + K::OI + cp * K::OI2, tm + K::H + t * 64 + 8 * k, tc::smem_desc(at + tc::desc_lo(K::X + (k >> 2) * HALF + 32 * (k & 3), 16), hi_sw),
                           tc::idesc_f16(128, 64, 1, 1, false, false), !(t == K::HT - 1 && k == 0));
            tc::mma_commit(h_read);
          }
          __syncwarp();
          ok = all(tc::mbar_wait2(pp_ready, cp, o_empty, cp ^ 1u, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
          if (tc::elect_one()) {
            // only blocks of the triangle; the first step covers all tokens
#pragma unroll
            for (int t = 1; t >= 0; --t)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int k = kRev ? 3 - i : i, row = kRev ? 0 : 16 * k, n = kRev ? 16 * (k + 1) : 64 - 16 * k;
                tc::mma_ss(tm + K::OA + row, tc::smem_desc(at + tc::desc_lo(K::W + 2048 * k, HALF), hi_sw),
                           tc::smem_desc(smem0 + tc::desc_lo(K::PP + t * HALF + row * 128 + 32 * k, 16), hi_sw), tc::idesc_f16(128, n, 1, 1, true, false),
                           !(t == 1 && i == 0));
              }
            tc::mma_commit(o_full);
          }
          __syncwarp();
        }
        if (c + 1 < n_chunks) {
          if (kGrad) ok = all(tc::mbar_wait2(&full[s_next], ph_next, o_empty, cp, abort_flag));
          else ok = all(tc::mbar_wait(&full[s_next], ph_next, abort_flag));
          if constexpr (!kState) {
            tc::tc_fence_after_sync();
            if (ok) scores(smem0 + s_next * (K::STAGE >> 4));
          }
        }
        s = s_next; ph = ph_next;
      }
    }
  } else if (warp < 12) {
    tc::reg_set<REGS_STATE, REGS_LAUNCH>();
    // ------------------------------------------------------------------ state: group grp has half of the columns (features of Y)
    constexpr int HC = DK / 2;
    const int grp = (warp - 4) >> 2, d = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = tm + ((uint32_t)((warp & 3) * 32) << 16);
    const bool mine = d < DV;
    float2 S[HC / 2];
    {
      const float* src = kState ? nullptr : seg.count > 1 ? a.seg_state + seg_tile : a.state_in != nullptr ? a.state_in + state_tile : nullptr;
      asm volatile("" : "+l"(src));
#pragma unroll
      for (int i = 0; i < HC / 2; ++i) {
        S[i] = make_float2(0.f, 0.f);
        if (src != nullptr && mine) {
          const float* p = src + (int64_t)(HC * grp + 2 * i) * a.st_y + (int64_t)d * a.st_w;
          S[i] = make_float2(p[0], p[a.st_y]);
        }
      }
    }
    auto publish = [&]() {
#pragma unroll
      for (int q = 0; q < HC / 16; ++q) {  // 16 columns at a time
        uint32_t t0[8], t1[8], t2[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if constexpr (K::HT == 3) split3(S[8 * q + i], t0[i], t1[i], t2[i]);
          else split_pair(S[8 * q + i], t0[i], t1[i]);
        }
        const uint32_t at = lane_addr + K::H + (HC / 2) * grp + 8 * q;
        tc::tmem_st8(at, t0);
        tc::tmem_st8(at + 64, t1);
        if constexpr (K::HT == 3) tc::tmem_st8(at + 128, t2);
      }
      tc::tmem_st_wait();
      tc::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(h_ready);
    };
    if constexpr (!kState) publish();
    int s = 0;
    bool ok = true;
    for (int c = 0; c < n_chunks; ++c) {
      const uint32_t cp = (uint32_t)c & 1u;
      ok = all(tc::mbar_wait(ds_full, cp, abort_flag));  // (the gate vectors were there before Yw was)
      if (!ok) break;
      tc::tc_fence_after_sync();
      const float decay = reinterpret_cast<const float*>(smem + K::GV + s * GATES)[GV_TOT];
#pragma unroll
      for (int q = 0; q < HC / 16; ++q) {
        uint32_t x[16];
        tc::tmem_ld16(lane_addr + K::DS + HC * grp + 16 * q, x);
        tc::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          S[8 * q + i] = __ffma2_rn(make_float2(decay, decay), S[8 * q + i], make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])));
      }
      tc::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) { tc::mbar_arrive(ds_empty); tc::mbar_arrive(&empty[s]); }
      if (++s == K::STAGES) s = 0;
      if constexpr (!kState) {
        if (c + 1 < n_chunks) {
          ok = all(tc::mbar_wait(h_read, cp, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
          publish();
        }
      }
    }
    float* dst = kState ? a.seg_state + seg_tile : last && a.state_out != nullptr ? a.state_out + state_tile : nullptr;
    if (ok && mine && dst != nullptr) {
#pragma unroll
      for (int i = 0; i < HC / 2; ++i) {
        float* p = dst + (int64_t)(HC * grp + 2 * i) * a.st_y + (int64_t)d * a.st_w;
        p[0] = S[i].x; p[a.st_y] = S[i].y;
      }
    }
  } else if (warp < 16) {
    tc::reg_set<REGS_OUT, REGS_LAUNCH>();
    // ------------------------------------------------------------------ outputs: 32 features a warp, as accumulator fragments of warp-level MMAs, which matrix stores
    // transpose on their way into shared memory, in the place of the chunk's X (and Y, for 32-bit rows), whose readers are through
    if constexpr (!kState) {
      const int wq = warp & 3, gr = lane >> 2, t2 = 2 * (lane & 3), r8 = lane & 7, m4 = lane >> 3;
      const uint32_t lane_addr = tm + ((uint32_t)(wq * 32) << 16);
      const bool mine = 32 * wq < DV, f32 = a.o_part != nullptr;
      int s = 0;
      for (int c = 0; c < n_chunks; ++c) {
        const uint32_t cp = (uint32_t)c & 1u;
        if (!all(tc::mbar_wait(o_full, cp, abort_flag))) break;
        tc::tc_fence_after_sync();
        const float* gv = reinterpret_cast<const float*>(smem + K::GV + s * GATES);
        uint8_t* stage = smem + s * K::STAGE + wq * (f32 ? 8192 : 4096);
        const uint32_t stage_s = tc::smem_u32(stage);
        const int at_tok = chunk_at(c) * C, len = min(C, seg.len - at_tok);
        const int64_t tok0 = seg.t0 + at_tok;
        [[maybe_unused]] float xs[16];
        if constexpr (kGrad)
#pragma unroll
          for (int i = 0; i < 16; ++i) xs[i] = 0.f;
        if (mine) {
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {  // 16 features
            uint32_t oi[32], oa[32];
            tc::tmem_ld_frags(lane_addr + ((uint32_t)hf << 20) + K::OI + cp * K::OI2, oi);
            tc::tmem_ld_frags(lane_addr + ((uint32_t)hf << 20) + K::OA, oa);
            tc::tmem_ld_wait();
            if (hf == 1) {
              tc::tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) tc::mbar_arrive(o_empty);
            }
            if constexpr (kGrad) {  // E's pieces in the layout of the fragments
              const uint32_t e_s = tc::smem_u32(smem + s * K::STAGE + K::E) + (uint32_t)((wq >> 1) * HALF + (8 * (m4 >> 1) + r8) * 128 +
                                                                                      (((4 * (wq & 1) + 2 * hf + (m4 & 1)) ^ r8) << 4));
#pragma unroll
              for (int g = 0; g < 8; g += 2) {
                uint32_t e[4];
                ldsm4t(e, e_s + 1024 * g);
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                  const float2 f = bf16x2_to_float2(e[m]);
                  const int gg = g + (m >> 1);
                  xs[2 * gg] = fmaf(f.x, __uint_as_float(oi[4 * gg + 2 * (m & 1)]), xs[2 * gg]);
                  xs[2 * gg + 1] = fmaf(f.y, __uint_as_float(oi[4 * gg + 2 * (m & 1) + 1]), xs[2 * gg + 1]);
                }
              }
            }
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              const float2 e = *reinterpret_cast<const float2*>(gv + GV_E + 8 * g + t2);
#pragma unroll
              for (int rr = 0; rr < 2; ++rr) {
                uint32_t* x = &oa[4 * g + 2 * rr];
                const float2 y = __ffma2_rn(e, make_float2(__uint_as_float(oi[4 * g + 2 * rr]), __uint_as_float(oi[4 * g + 2 * rr + 1])),
                                            make_float2(__uint_as_float(x[0]), __uint_as_float(x[1])));
                x[0] = __float_as_uint(y.x); x[1] = __float_as_uint(y.y);
              }
            }
            auto pair = [&](int g, int rr) { return make_float2(__uint_as_float(oa[4 * g + 2 * rr]), __uint_as_float(oa[4 * g + 2 * rr + 1])); };
            if (f32) {  // [64 tokens][32 features] of 4 bytes, 128-byte swizzle
              const int c0 = (4 * hf) ^ (gr >> 2) ^ t2;
#pragma unroll
              for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int rr = 0; rr < 2; ++rr) {
                  float* p = reinterpret_cast<float*>(stage + (t2 + e) * 128 + (((2 * rr) ^ c0 ^ e) << 4)) + (gr & 3);
#pragma unroll
                  for (int g = 0; g < 8; ++g) p[256 * g] = __uint_as_float(oa[4 * g + 2 * rr + e]);
                }
            } else {  // of 2 bytes, 64-byte swizzle
              const uint32_t at = stage_s + (uint32_t)((8 * (m4 >> 1) + r8) * 64 + (((2 * hf + (m4 & 1)) ^ (r8 >> 1)) << 4));
#pragma unroll
              for (int g = 0; g < 8; g += 2) {
                uint32_t x[4];
#pragma unroll
                for (int m = 0; m < 4; ++m) { const float2 y = pair(g + (m >> 1), m & 1); x[m] = pack_bf16x2(y.x, y.y); }
                stsm4t(at + 512 * g, x[0], x[1], x[2], x[3]);
              }
            }
          }
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (!mine && lane == 0) tc::mbar_arrive(o_empty);
        if constexpr (kGrad) {
          // sums over the eight lanes of a token's features; lane (gr, t2 / 2) ends with the tokens 8 gr + t2, 8 gr + t2 + 1
#pragma unroll
          for (int w = 8; w >= 2; w >>= 1) {
            const int mask = 2 * w;  // 16, 8, 4: bit of gr
            const bool upper = (lane & mask) != 0;
#pragma unroll
            for (int i = 0; i < w; ++i) {
              const float send = upper ? xs[i] : xs[i + w];
              xs[i] = (upper ? xs[i + w] : xs[i]) + __shfl_xor_sync(0xffffffffu, send, mask);
            }
          }
          const int t = 8 * gr + t2;
          float* dst = a.inter + (((int64_t)wq * a.Hv + h) * a.B + seg.b) * a.T + tok0;
          if (mine && t < len) dst[t] = gv[GV_E + t] * xs[0];
          if (mine && t + 1 < len) dst[t + 1] = gv[GV_E + t + 1] * xs[1];
        }
        if (mine) {
          if (len == C && (f32 || maps.o_ok)) {
            if (lane == 0) tc::tma_store_4d(f32 ? &maps.o32 : &maps.o, stage, 32 * wq, h, (int)tok0, seg.b);
          } else if (f32) {
            float* dst = a.o_part + (((int64_t)seg.b * a.T + tok0) * a.Hv + h) * DV + 32 * wq + 4 * r8;
#pragma unroll 1
            for (int t = m4; t < len; t += 4) *reinterpret_cast<float4*>(dst + (int64_t)t * a.Hv * DV) = *reinterpret_cast<const float4*>(stage + t * 128 + ((r8 ^ (t & 7)) << 4));
            tc::fence_proxy_async_smem();
          } else {
            __nv_bfloat16* dst = reinterpret_cast<__nv_bfloat16*>(a.o) + seg.b * a.o_stride_b + (int64_t)h * a.o_stride_h + tok0 * a.o_stride_t + 32 * wq + 8 * (lane & 3);
#pragma unroll 1
            for (int t = lane >> 2; t < len; t += 8) *reinterpret_cast<uint4*>(dst + (int64_t)t * a.o_stride_t) = *reinterpret_cast<const uint4*>(stage + t * 64 + (((lane & 3) ^ ((t >> 1) & 3)) << 4));
            tc::fence_proxy_async_smem();
          }
        }
        if (lane == 0) {  // the next tiles of this stage come when it has been read
          tc::bulk_commit();
          tc::bulk_wait_read<0>();
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&empty[s]);
        if (++s == K::STAGES) s = 0;
      }
      if (lane == 0) tc::bulk_wait_all();
    }
  } else {
    tc::reg_set<REGS_PREP, REGS_LAUNCH>();
    {
      // ---------------------------------------------------------------- Yw: a piece (8 features of a token) at a time, in the places that Y's has
      constexpr int N = 128;
      const int tid = (warp - 16) * 32 + lane;
      int s = 0;
      uint32_t ph = 0;
      for (int c = 0; c < n_chunks; ++c) {
        const uint32_t cp = (uint32_t)c & 1u;
        const int len = min(C, seg.len - chunk_at(c) * C);
        if (!all(tc::mbar_wait3(&full[s], ph, &gates[s], ph, ds_full, cp ^ 1u, abort_flag))) break;
        const float* gv = reinterpret_cast<const float*>(smem + K::GV + s * GATES);
        uint8_t* st = smem + s * K::STAGE;
#pragma unroll 2
        for (int i = tid; i < (DK / 64) * 512; i += N) {
          const int tok = (i >> 3) & 63;
          const float w = gv[GV_W + tok];
          uint4 y = *reinterpret_cast<const uint4*>(st + K::Y + 16 * i);
          if (tok >= len) y = make_uint4(0u, 0u, 0u, 0u);  // (may be anything, and w is zero)
          const uint32_t in[4] = {y.x, y.y, y.z, y.w};
          uint32_t h0[4], h1[4], h2[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = bf16x2_to_float2(in[j]);
            split3(__fmul2_rn(f, make_float2(w, w)), h0[j], h1[j], h2[j]);
          }
          uint8_t* dst = smem + K::YW + 16 * i;
          *reinterpret_cast<uint4*>(dst) = make_uint4(h0[0], h0[1], h0[2], h0[3]);
          *reinterpret_cast<uint4*>(dst + TILE) = make_uint4(h1[0], h1[1], h1[2], h1[3]);
          *reinterpret_cast<uint4*>(dst + 2 * TILE) = make_uint4(h2[0], h2[1], h2[2], h2[3]);
        }
        // What lies behind the sequence in W's tile may be anything, and a product of zero with it need not be zero
        if (len < C)
#pragma unroll 1
          for (int i = 8 * len + tid; i < 512; i += N) {
            *reinterpret_cast<uint4*>(st + K::W + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
            if constexpr (DV == 128) *reinterpret_cast<uint4*>(st + K::W + HALF + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
          }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(yw_ready);
        if (++s == K::STAGES) { s = 0; ph ^= 1u; }
      }
    }
  }

  tc::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0u) {  // (the roles have ended: it stays as it is)
    if (threadIdx.x == 0 && a.status != nullptr) atomicOr(a.status, AVE_GDN_DEV_WAIT_EXPIRED);
    if (warp == 3) tc::drain_mmas(mma_end);
    tc::tc_fence_before_sync();
    __syncthreads();
  }
  if (warp == 3) {
    tc::tc_fence_after_sync();
    tc::tmem_dealloc(tm, K::COLS);
  }
}

// Between the two passes: seg_state goes from each segment's own increment to the state that enters it.
template <int DK, int DV, bool kRev>
__global__ void __launch_bounds__(256) chain_kernel(const Args a) {
  pdl_wait();
  if (!offsets_fit(a, false)) return;
  constexpr int PARTS = DK * DV / 1024;
  const int part = blockIdx.x % PARTS, h = blockIdx.x / PARTS % a.Hv, n = blockIdx.x / PARTS / a.Hv;
  const SeqSpan sp = seq_span(a.cu_seqlens, n, a.T, nullptr);
  const int count = (sp.len + a.plan.len - 1) / a.plan.len;
  if (!sp.ok || count < 2) return;
  int slot = n;
  if (a.state_indices != nullptr) slot = a.state_indices[n];
  if (slot < 0 || (a.state_indices != nullptr && slot >= a.num_slots)) return;
  const int64_t at = part * 1024 + threadIdx.x * 4, s0 = first_slot(a, n);
  float4 cur = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a.state_in != nullptr) cur = *reinterpret_cast<const float4*>(a.state_in + ((int64_t)slot * a.Hv + h) * (DK * DV) + at);
  float* base = a.seg_state + h * (int64_t)(DK * DV) + at;
  const int64_t step = (int64_t)a.Hv * (DK * DV);
  for (int i0 = 0; i0 < count; i0 += 4) {
    float4 own[4];
    float decay[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u < count - 1) {
        const int64_t sl = s0 + (kRev ? count - 1 - i0 - u : i0 + u);
        own[u] = *reinterpret_cast<const float4*>(base + sl * step);
        decay[u] = a.seg_decay[sl * a.Hv + h];
      }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u < count) {
        const int64_t sl = s0 + (kRev ? count - 1 - i0 - u : i0 + u);
        *reinterpret_cast<float4*>(base + sl * step) = cur;
        if (i0 + u < count - 1) {
          cur.x = fmaf(decay[u], cur.x, own[u].x); cur.y = fmaf(decay[u], cur.y, own[u].y);
          cur.z = fmaf(decay[u], cur.z, own[u].z); cur.w = fmaf(decay[u], cur.w, own[u].w);
        }
      }
  }
}

}  // namespace lin
}  // namespace
}  // namespace ave
