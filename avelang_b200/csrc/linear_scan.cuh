// The chunked scan of linear attention with a decay for each head, for one segment of one (sequence, value head):
//     H^T  state [dv lanes][dk], fp32 in registers, with bf16 images in TMEM
//     P    = X Y^T            masked and decayed: P'_ts = scale e^{G_t - G_s} P_ts for s <= t
//     O^T  = e_t (H^T X^T) + W^T P'^T
//     H^T <- decay H^T + (w W)^T Y,   w_s = e^{G_end - G_s}
// over chunks of 64 tokens, X, Y, W = q, k, v in the forward pass.  The gradients are scans of the same form: (do, v, k) forwards gives dq;
// (v, do, q) and (k, q, do) backwards in time give dk and dv, with the mask, the walk over the chunks and the decays' signs turned round.
// G is the sum of the decays' logarithms inside the chunk, so every exponent of a product that counts is <= 0 for g <= 0.
//
// All four products are tcgen05 MMAs with fp32 accumulators in tensor memory.  The inputs are bf16 and go in as they are; what is computed goes in as two or three bf16 terms, since
// one would leave 2^-9 of each number in a sum.  Tokens of a chunk come as one TMA copy an operand, three or four chunks ahead.  The state stays on chip from a segment's first chunk
// to its last, so HBM sees each input and output once; one CTA fills an SM.  What bounds a chunk is the chain of hand-overs between the roles (products, masking and decaying P, the
// state's update and its image for the next chunk), not the tensor pipe and not HBM: 2.3 us of outputs and state, 1.4 of the state alone, 3.9 with the gate gradient's terms.
// (d = 128, 148 heads x 2048 tokens: 72 us, 4.3 TB/s of the copy rate's 6.5,
// tensor pipe busy 0.42 of the cycles, DRAM 0.49, issue slots 0.52; the scans of a 2 x 4096 token, 32 head backward 335 us, of 49 heads x 2048 tokens 0.21, 0.26 and 0.33.)  64 tokens a chunk: with 128
// P is four times as large for twice the tokens, half of it masked, and two chunks' terms of it would not fit beside the stages.
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
  float log_scale;                 // P' carries scale as 2^log_scale, and the product W^T P'^T its sign
  int negative;
  float scale_e, scale_w;
  void* o;                         // bf16
  int64_t o_stride_b, o_stride_t, o_stride_h;
  int zero_outside;                // rows of no sequence become zero
  float* o_part;                   // fp32 [B, T, Hv, dv] instead, for a sum over heads behind the scan
  const float* state_in;           // [slot, Hv, ..]: element (y feature, w feature) at y * st_y + w * st_w
  float* state_out;
  int final_by_chain;              // chain_kernel writes state_out, for all sequences with tokens
  int st_y, st_w;
  float* seg_state;                // [segment slot, Hv, ..] likewise
  float* seg_decay;                // [segment slot, Hv]
  float* inter;                    // [dv / 32][Hv][B T]: e_t E_t . (H^T X_t), 32 features each      (for the gradient of g)
  Plan plan;
};
struct Maps {
  CUtensorMap x, y, w, e;  // 64 tokens of a head a copy
  CUtensorMap o;           // 32 features of 64 tokens, of the result or of o_part
  bool o_ok;               // the result's layout can be described by a map
};

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

// Whole sequences of a packed batch, the longest first, so that the SMs end together: the sequence whose turn it is.  Called by the whole CTA.  (24 prompts of 65536 tokens in all,
// 2 to 161 chunks each, 32 heads: 568 us, in the batch's order 777; other draws of the lengths take up to 690.)  Each sequence counts those in front of it, which takes a thread as many steps as there are sequences; where there are
// many, each is a small part of an SM's work and the batch's order serves.
constexpr int MOST_IN_ORDER = 256;
__device__ __forceinline__ int64_t longest_first(const Args& a, int64_t turn) {
  if (a.plan.cut || a.cu_seqlens == nullptr || a.n_seqs < 2 || a.n_seqs > MOST_IN_ORDER) return turn;
  __shared__ int lens[MOST_IN_ORDER], found;
  const int n = threadIdx.x;
  if (n < a.n_seqs) lens[n] = a.cu_seqlens[n + 1] - a.cu_seqlens[n];
  __syncthreads();
  if (n < a.n_seqs) {
    const int own = lens[n];
    int before = 0;
    for (int m = 0; m < a.n_seqs; ++m) before += (lens[m] > own || (lens[m] == own && m < n)) ? 1 : 0;
    if (before == turn) found = n;
  }
  __syncthreads();
  return found;
}

// Shared memory: a ring of stages {W, Y, (X), (E)} with their gate vectors, and the two terms of P'.
// Gate vectors of a chunk, floats: e[64] | w[64] | G hi[64] | G lo[64] | decay (and padding to 64 bytes)
constexpr int GATES = 1088;
constexpr int GV_E = 0, GV_W = 64, GV_H = 128, GV_L = 192, GV_TOT = 256;
// kMode: the state alone; outputs with a state in two terms (2) or three (3) bf16 terms an increment; and with what the gradient of g needs.
// A product of a weight and a bf16 number, two terms of it, is off by 2^-18 in the mean: enough for outputs that are rounded to bf16, not for a state that
// is itself a result, nor for the gradient of g.
enum Mode { STATE, OUT2, OUT3, GRAD };
template <Mode kMode>
struct Cfg {
  static constexpr bool kState = kMode == STATE, kGrad = kMode == GRAD;
  static constexpr int TERMS = kMode == OUT2 ? 2 : 3;  // of an increment
  static constexpr int HT = kGrad ? 3 : 2;             // of the state's image
  static constexpr int W = 0, Y = TILE, X = 2 * TILE, E = 3 * TILE;
  static constexpr int STAGE = (kState ? 2 : kGrad ? 4 : 3) * TILE;
  static constexpr int STAGES = kGrad ? 3 : 4;
  static constexpr int PP = STAGES * STAGE, GV = PP + (kState ? 0 : TILE), BARS = GV + STAGES * GATES;
  static constexpr int SMEM = BARS + 256 + 1024;
  static_assert(SMEM <= 232448, "shared memory of an SM");
  // TMEM columns.  With three terms W^T P'^T takes the columns of P, and with the gradient of g the increment's two halves (64 features of Y each) one another's.
  static constexpr bool kAlias = TERMS == 3;
  static constexpr uint32_t P = 0, OA = kAlias ? 0 : 64, OI = kAlias ? 64 : 128;
  // (For the state alone the chunks take two places in turn for their increments and their images.)
  static constexpr uint32_t DS = kState ? 0 : OI + 64, H = DS + (kGrad ? 64 : 128), IMG = kState ? 256 : H + 64 * HT;
  static constexpr uint32_t TURN_DS = kState ? 128 : 0, TURN_IMG = kState ? 32 * TERMS : 0, COLS = 512;
  static_assert(IMG + TURN_IMG + 32 * TERMS <= COLS, "tensor memory");
};

constexpr int THREADS = 640;  // warpgroups: loader, gate vectors and two issuers; two for the state and P'; outputs; images of W^T
constexpr int REGS_LAUNCH = 96, REGS_CTRL = 56, REGS_STATE = 128, REGS_OUT = 96, REGS_PREP = 72;
// (At 96 registers some roles spill: bytes stored and loaded a thread at d = 128, outputs 32 and 32, with an exact final state 32 and 32, the state alone 24 and 44; the backward's kernel of three
// scans 320 and 988, 116 and 508 without the gate gradient.)
static_assert(REGS_CTRL + 2 * REGS_STATE + REGS_OUT + REGS_PREP <= 5 * REGS_LAUNCH, "register redistribution exceeds the launch allocation");
static_assert(THREADS * REGS_LAUNCH <= 65536, "launch allocation exceeds the register file");

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Sums of the decays' base-2 logarithms as 64-bit integers in units of 2^-36: exact, and a step of a running sum is two shuffles and an addition.  (In 64-bit floating point a chunk's
// gate vectors took 3.8 k cycles, as sums of two floats 1.4 k.)  Logarithms are held inside +-1e6, so that 64 of them fit.
constexpr float FIXED = 68719476736.f;  // 2^36
struct Two { float h, l; };             // a number as the sum of two floats
__device__ __forceinline__ float diff(Two a, Two b) { return (a.h - b.h) + (a.l - b.l); }
__device__ __forceinline__ long long fixed_log2(float ln) {  // ln * log2(e); a NaN is the caller's to see
  constexpr float L = 1.44269504f, R = 1.925963033e-8f;
  ln = fminf(fmaxf(ln, -1e6f), 1e6f);
  const float p = ln * L;
  return __float2ll_rn(p * FIXED) + __float2ll_rn((fmaf(ln, L, -p) + ln * R) * FIXED);
}
__device__ __forceinline__ Two two(long long x) {
  const float h = __ll2float_rn(x);
  return Two{h * (1.f / FIXED), __ll2float_rn(x - __float2ll_rn(h)) * (1.f / FIXED)};
}
// Running sums over 64 tokens, two a lane, from the logarithms; returns the whole sum.  From a NaN on they are NaN.
__device__ __forceinline__ long long gate_scan(float n0, float n1, int lane, Two& G0, Two& G1) {
  const long long x0 = fixed_log2(n0), x1 = fixed_log2(n1);
  long long sum = x0 + x1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += y;
  }
  G1 = two(sum);
  G0 = two(sum - x1);
  const unsigned bad = __ballot_sync(0xffffffffu, isnan(n0) || isnan(n1));
  if (bad != 0u) {
    const int first = __ffs(bad) - 1;
    if (lane > first || (lane == first && isnan(n0))) G0.h = __int_as_float(0x7fffffff);
    if (lane >= first) G1.h = __int_as_float(0x7fffffff);
  }
  return __shfl_sync(0xffffffffu, sum, 31);
}
// 2^x to the last bit or two: a state is multiplied by the same number chunk after chunk, so that an error in it adds up.  Taylor's series of 2^r for |r| <= 1/2.
__device__ __forceinline__ float pow2(Two x) {
  const float n = rintf(x.h), r = ((x.h - n) + x.l) * 0.693147181f;
  float p = 1.f / 5040.f;
#pragma unroll
  for (int k = 0; k < 6; ++k) {
    constexpr float inv[6] = {1.f / 720.f, 1.f / 120.f, 1.f / 24.f, 1.f / 6.f, 0.5f, 1.f};
    p = fmaf(p, r, inv[k]);
  }
  p = fmaf(p, r, 1.f);
  if (n < -126.f) return 0.f;
  return n > 127.f ? p * __int_as_float(0x7f800000) : p * __int_as_float(((int)n + 127) << 23);  // (a NaN stays one)
}

// Rows of a packed batch in front of its first offset and behind its last, or all where the offsets are not monotone: the CTAs of a head share them out.
template <int D>
__device__ __forceinline__ void zero_outside(const Args& a, bool fit) {
  const int lo = fit ? a.cu_seqlens[0] : a.T, hi = fit ? a.cu_seqlens[a.n_seqs] : a.T;
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(a.o) + (int64_t)(blockIdx.x % a.Hv) * a.o_stride_h;
  const int64_t pieces = (int64_t)(lo + (a.T - hi)) * (D / 8), step = (int64_t)(gridDim.x / a.Hv) * THREADS;
  for (int64_t i = (int64_t)(blockIdx.x / a.Hv) * THREADS + threadIdx.x; i < pieces; i += step) {
    const int64_t r = i / (D / 8), t = r < lo ? r : hi + (r - lo);
    *reinterpret_cast<uint4*>(o + t * a.o_stride_t + 8 * (i % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
  }
}

template <int DK, int DV, bool kRev, Mode kMode>
__device__ __forceinline__ void scan(const Args& a, const Maps& maps) {
  using K = Cfg<kMode>;
  constexpr bool kState = K::kState, kGrad = K::kGrad;
  constexpr int FH = kGrad ? DK / 64 : 1;  // parts in which the increment comes: group g of the state's warps takes part g, or half of the only one
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = tc::align1024(smem_raw);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + K::BARS);
  uint64_t* full = bars;            // [4] tiles of the stage landed
  uint64_t* gates = bars + 4;       // [4] its gate vectors written
  uint64_t* empty = bars + 8;       // [4] the stage is read
  uint64_t* p_full = bars + 12;     // P accumulated
  uint64_t* pp_ready = bars + 13;   // P' written, P drained
  uint64_t* img_ready = bars + 14;  // [2] images of 32 tokens of W^T written
  uint64_t* img_read = bars + 16;   // [2] and read
  uint64_t* ds_full = bars + 18;    // [2] the increment accumulated; with the gradient of g one half after the other
  uint64_t* ds_empty = bars + 20;   // [2] and drained
  uint64_t* h_ready = bars + 22;    // images of the state written
  uint64_t* h_read = bars + 23;     // H^T X^T accumulated
  uint64_t* o_full = bars + 24;     // W^T P'^T accumulated, P' read
  uint64_t* o_empty = bars + 25;    // outputs drained
  uint64_t* cleared = bars + 26;    // what lies behind the sequence in the tiles of its last chunk cleared
  uint64_t* mma_end = bars + 27;    // [2] the MMAs of warps 3 and 1 are complete, when a wait has expired
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 29);
  // A wait sees only the parity of a barrier's phase, so no barrier may complete twice before each of its waiters has seen the first time.  All are ordered by the arrivals they
  // need: the products of a chunk by what is written for them, that by the products of the chunk before, and o_full, for which the output warps wait too, by o_empty of the
  // chunk before.
  volatile uint32_t* abort_flag = tmem_slot + 1;

  const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < K::STAGES; ++i) {
      tc::mbar_init(&full[i], 1); tc::mbar_init(&gates[i], 1);
      tc::mbar_init(&empty[i], kState ? 9 : 12);  // the state's warps have read the decay, and: the issuer's commit, or the output warps
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&img_ready[i], 4); tc::mbar_init(&img_read[i], 1);
      tc::mbar_init(&ds_full[i], 1); tc::mbar_init(&ds_empty[i], 8 / FH);
    }
    for (uint64_t* b : {p_full, h_read, o_full, &mma_end[0], &mma_end[1]}) tc::mbar_init(b, 1);
    tc::mbar_init(cleared, 4);
    tc::mbar_init(pp_ready, 6); tc::mbar_init(h_ready, 8); tc::mbar_init(o_empty, 4);
    *abort_flag = 0;
    tc::fence_barrier_init();
  }
  pdl_wait();
  const bool fit = offsets_fit(a, true);
  if constexpr (!kState && !kGrad && !kRev)
    if (a.zero_outside) zero_outside<DV>(a, fit);
  if (!fit) return;
  const int h = blockIdx.x % a.Hv;
  const int64_t seg_slot = longest_first(a, blockIdx.x / a.Hv);
  const Seg seg = seg_of_slot(a, seg_slot);
  if (!seg.ok) return;
  const bool last = kRev ? seg.j == 0 : seg.j == seg.count - 1;
  if (kState && last && !a.final_by_chain) return;  // nobody takes its state from here
  int slot = seg.n;
  if (a.state_indices != nullptr) {
    slot = a.state_indices[seg.n];
    if (slot >= a.num_slots) {
      if (a.status != nullptr && threadIdx.x == 0) atomicOr(a.status, AVE_GDN_DEV_BAD_SLOT);
      slot = -1;
    }
  }
  if (kState && (slot < 0 || seg.len == 0)) return;
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
    if (warp == 0) {
      // ---------------------------------------------------------------- loader
      if (lane == 0) {
        if (!kState) tc::prefetch_tmap(&maps.x);
        tc::prefetch_tmap(&maps.y); tc::prefetch_tmap(&maps.w);
        const int hx = h / a.x_div, hy = h / a.y_div, hw = h / a.w_div, he = h / a.e_div;
        int s = 0, issued = 0;
        uint32_t ph = 1;
#pragma unroll 1
        for (int c = 0; c < n_chunks; ++c) {
          if (c >= K::STAGES && !tc::mbar_wait(&empty[s], ph, abort_flag)) break;
          uint8_t* st = smem + s * K::STAGE;
          const int tok = seg.t0 + chunk_at(c) * C;
          constexpr uint32_t bytes = (kState ? 1 : 2) * (DK / 64) * HALF + (kGrad ? 2 : 1) * (DV / 64) * HALF;
          tc::mbar_expect_tx(&full[s], bytes);
          tc::tma_load_5d(st + K::Y, &maps.y, &full[s], 0, tok, 0, hy, seg.b);
          tc::tma_load_5d(st + K::W, &maps.w, &full[s], 0, tok, 0, hw, seg.b);
          if constexpr (!kState) tc::tma_load_5d(st + K::X, &maps.x, &full[s], 0, tok, 0, hx, seg.b);
          if constexpr (kGrad) tc::tma_load_5d(st + K::E, &maps.e, &full[s], 0, tok, 0, he, seg.b);
          ++issued;
          if (++s == K::STAGES) { s = 0; ph ^= 1u; }
        }
        // nothing is on its way into the shared memory of a CTA that ends, whatever became of those who wait for it
#pragma unroll 1
        for (int c = max(0, issued - K::STAGES); c < issued; ++c) tc::drain(&full[c % K::STAGES], (uint32_t)(c / K::STAGES) & 1u);
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------------- gate vectors, two tokens a lane
      [[maybe_unused]] Two seg_total{0.f, 0.f};
      const float* g = a.g != nullptr ? a.g + seg.b * a.g_stride_b + h : nullptr;
      auto fetch = [&](int c, int e) {
        const int t = chunk_at(c) * C + 2 * lane + e;
        if (g == nullptr || t >= seg.len) return 0.f;
        return g[(int64_t)(seg.t0 + t) * a.g_stride_t];
      };
      float n0 = fetch(0, 0), n1 = fetch(0, 1);
      int s = 0;
      uint32_t ph = 1;
      for (int c = 0; c < n_chunks; ++c) {
        if (c >= K::STAGES && !all(tc::mbar_wait(&empty[s], ph, abort_flag))) break;
        Two G0, G1;
        const long long whole = gate_scan(n0, n1, lane, G0, G1);
        if (c + 1 < n_chunks) { n0 = fetch(c + 1, 0); n1 = fetch(c + 1, 1); }  // (not looked at before the next round)
        Two total = two(whole);
        total.h += 0.f * __shfl_sync(0xffffffffu, G1.h, 31);  // (a NaN stays one)
        if constexpr (kState) seg_total = Two{seg_total.h + total.h, seg_total.l + total.l + ((seg_total.h - (seg_total.h + total.h)) + total.h)};
        const int left = seg.len - chunk_at(c) * C - 2 * lane;  // tokens from this lane's first on
        const float2 from0 = make_float2(ex2(G0.h + G0.l), ex2(G1.h + G1.l)), to_end = make_float2(ex2(diff(total, G0)), ex2(diff(total, G1)));
        const float2 e = __fmul2_rn(make_float2(a.scale_e, a.scale_e), kRev ? to_end : from0);
        float2 w = __fmul2_rn(make_float2(a.scale_w, a.scale_w), kRev ? from0 : to_end);
        if (left < 1) w.x = 0.f;
        if (left < 2) w.y = 0.f;
        const float sg = kRev ? -1.f : 1.f;
        const float2 hi = make_float2(sg * G0.h, sg * G1.h), lo = make_float2(sg * G0.l, sg * G1.l);
        const float tot = pow2(total);
        float* v = reinterpret_cast<float*>(smem + K::GV + s * GATES);
        reinterpret_cast<float2*>(v + GV_E)[lane] = e;
        reinterpret_cast<float2*>(v + GV_W)[lane] = w;
        reinterpret_cast<float2*>(v + GV_H)[lane] = hi;
        reinterpret_cast<float2*>(v + GV_L)[lane] = lo;
        if (lane == 0) v[GV_TOT] = tot;
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&gates[s]);
        if (++s == K::STAGES) { s = 0; ph ^= 1u; }
      }
      if (kState && lane == 0) a.seg_decay[seg_slot * a.Hv + h] = pow2(seg_total);
    } else if (warp == 3) {
      // ---------------------------------------------------------------- MMA issuer of the state: increments, H^T X^T
      const uint32_t smem0 = tc::smem_u32(smem) >> 4;
      constexpr uint32_t hi_sw = tc::desc_hi(1024, true);
      // 32 tokens' part of the increment, or of half f of it, the smallest terms first
      constexpr int N = kGrad ? 64 : DK;
      auto part = [&](int f, int q, uint32_t at, uint32_t turn) {
#pragma unroll
        for (int t = K::TERMS - 1; t >= 0; --t)
#pragma unroll
          for (int k = 2 * q; k < 2 * q + 2; ++k)  // 16 tokens a step
            tc::mma_ts(tm + K::DS + turn * K::TURN_DS, tm + K::IMG + turn * K::TURN_IMG + 32 * t + 8 * k,
                       tc::smem_desc(at + tc::desc_lo(K::Y + f * HALF + 2048 * k, HALF), hi_sw), tc::idesc_f16(128, N, 1, 1, false, true), !(q == 0 && t == K::TERMS - 1 && k == 0));
      };
      int s = 0;
      bool ok = true;
#pragma unroll 1
      for (int c = 0; c < n_chunks; ++c) {
        const uint32_t cp = (uint32_t)c & 1u, at = smem0 + s * (K::STAGE >> 4);
        if constexpr (kGrad && FH == 2) {  // one place for both halves of the increment: they come one after the other
          ok = all(tc::mbar_wait3(&ds_empty[1], cp ^ 1u, &img_ready[0], cp, &img_ready[1], cp, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
          if (tc::elect_one()) { part(0, 0, at, 0u); part(0, 1, at, 0u); tc::mma_commit(&ds_full[0]); }
          __syncwarp();
          ok = all(tc::mbar_wait(&ds_empty[0], cp, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
          if (tc::elect_one()) {
            part(1, 0, at, 0u); part(1, 1, at, 0u);
            tc::mma_commit(&img_read[0]); tc::mma_commit(&img_read[1]); tc::mma_commit(&ds_full[1]);
          }
          __syncwarp();
        } else if constexpr (kState) {
          const uint32_t turn = (uint32_t)(c >> 1) & 1u;
          ok = all(tc::mbar_wait2(&ds_empty[cp], turn ^ 1u, &img_ready[cp], turn, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
          if (tc::elect_one()) {
            part(0, 0, at, cp); part(0, 1, at, cp);
            tc::mma_commit(&ds_full[cp]); tc::mma_commit(&img_read[cp]); tc::mma_commit(&empty[s]);
          }
          __syncwarp();
        } else {  // the tokens by halves, as their images come, so that those of the next chunk are written beside it
          ok = all(tc::mbar_wait2(&ds_empty[0], cp ^ 1u, &img_ready[0], cp, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
          if (tc::elect_one()) { part(0, 0, at, 0u); tc::mma_commit(&img_read[0]); }
          __syncwarp();
          ok = all(tc::mbar_wait(&img_ready[1], cp, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
          if (tc::elect_one()) { part(0, 1, at, 0u); tc::mma_commit(&ds_full[0]); tc::mma_commit(&img_read[1]); }
          __syncwarp();
        }
        if constexpr (!kState) {
          ok = all(tc::mbar_wait2(h_ready, cp, o_empty, cp ^ 1u, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
          if (tc::elect_one()) {
#pragma unroll
            for (int t = K::HT - 1; t >= 0; --t)
#pragma unroll
              for (int k = 0; k < DK / 16; ++k)
                tc::mma_ts(tm + K::OI, tm + K::H + t * 64 + 8 * k, tc::smem_desc(at + tc::desc_lo(K::X + (k >> 2) * HALF + 32 * (k & 3), 16), hi_sw),
                           tc::idesc_f16(128, 64, 1, 1, false, false), !(t == K::HT - 1 && k == 0));
            tc::mma_commit(h_read);
          }
          __syncwarp();
        }
        if (++s == K::STAGES) s = 0;
      }
    } else if (!kState && warp == 1) {
      // ---------------------------------------------------------------- MMA issuer of the scores and of what they weigh: with one warp for all products its waits and issues, 4.1 k
      // cycles a chunk, were what a chunk took
      const uint32_t smem0 = tc::smem_u32(smem) >> 4;
      constexpr uint32_t hi_sw = tc::desc_hi(1024, true);
      const uint32_t neg = a.negative ? 1u << 13 : 0u;
      // Columns 0..31 of the scores have the chunk's rows in lanes 0..63, columns 32..63 in lanes 64..127 (the left operand begins 64 rows early): all lanes' warps take
      // a part of them.  The other halves multiply what lies in front of the tile and behind it, and nobody reads them.
      auto scores = [&](uint32_t at) {
        if (tc::elect_one()) {
#pragma unroll
          for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int k = 0; k < DK / 16; ++k)
              tc::mma_ss(tm + K::P + 32 * half, tc::smem_desc(at + tc::desc_lo(K::X - half * HALF + (k >> 2) * HALF + 32 * (k & 3), 16), hi_sw),
                         tc::smem_desc(at + tc::desc_lo(K::Y + half * 4096 + (k >> 2) * HALF + 32 * (k & 3), 16), hi_sw), tc::idesc_f16(128, 32, 1, 1, false, false), k != 0);
          tc::mma_commit(p_full);
        }
        __syncwarp();
      };
      int s = 0;
      uint32_t ph = 0;
      bool ok = all(tc::mbar_wait(&full[0], 0u, abort_flag));
      tc::tc_fence_after_sync();
      if (ok) scores(smem0);
#pragma unroll 1
      for (int c = 0; c < n_chunks && ok; ++c) {
        const uint32_t cp = (uint32_t)c & 1u, at = smem0 + s * (K::STAGE >> 4);
        if (++s == K::STAGES) { s = 0; ph ^= 1u; }
        ok = K::kAlias ? all(tc::mbar_wait(pp_ready, cp, abort_flag)) : all(tc::mbar_wait2(pp_ready, cp, o_empty, cp ^ 1u, abort_flag));
        if (ok && seg.len - chunk_at(c) * C < C) ok = all(tc::mbar_wait(cleared, 0u, abort_flag));
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
                         tc::smem_desc(smem0 + tc::desc_lo(K::PP + t * HALF + row * 128 + 32 * k, 16), hi_sw), tc::idesc_f16(128, n, 1, 1, true, false) | neg,
                         !(t == 1 && i == 0));
            }
          tc::mma_commit(o_full);
        }
        __syncwarp();
        if (c + 1 < n_chunks) {
          ok = K::kAlias ? all(tc::mbar_wait2(&full[s], ph, o_empty, cp, abort_flag)) : all(tc::mbar_wait(&full[s], ph, abort_flag));
          tc::tc_fence_after_sync();
          if (ok) scores(smem0 + s * (K::STAGE >> 4));
        }
      }
    }
  } else if (warp < 12) {
    tc::reg_set<REGS_STATE, REGS_LAUNCH>();
    // ------------------------------------------------------------------ state and P': group grp has half of the state's columns (features of Y)
    constexpr int HC = DK / 2;
    const int grp = (warp - 4) >> 2, half = FH == 2 ? grp : 0, d = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = tm + ((uint32_t)((warp & 3) * 32) << 16);
    const bool mine = d < DV;
    float2 S[HC / 2];
    {
      // (with the chain, which may have put the final state in the place of the initial one, every segment's)
      const float* src = kState ? nullptr : seg.count > 1 || a.final_by_chain ? a.seg_state + seg_tile : a.state_in != nullptr ? a.state_in + state_tile : nullptr;
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
    // P': 32 rows x 16 columns a warp, row t a lane.  Blocks in which no row has a part are neither written nor read: six warps are left.
    const int t = 32 * (warp & 1) + lane, col0 = 32 * ((warp & 3) >> 1) + 16 * grp;
    const bool has_part = kRev ? col0 + 15 >= 32 * (warp & 1) : col0 <= 32 * (warp & 1) + 31;
    auto weigh = [&](int c, int s, uint32_t ph) {
      const int at_tok = chunk_at(c) * C, len = min(C, seg.len - at_tok);
      if (has_part) {
        const uint32_t cp = (uint32_t)c & 1u;
        if (!all(tc::mbar_wait3(p_full, cp, &gates[s], ph, o_full, cp ^ 1u, abort_flag))) return false;
        tc::tc_fence_after_sync();
        const float* gv = reinterpret_cast<const float*>(smem + K::GV + s * GATES);
        uint8_t* row = smem + K::PP + t * 128;
        const float2 gh = make_float2(gv[GV_H + t], gv[GV_H + t]);
        const float gl1 = gv[GV_L + t] + a.log_scale;
        const float2 gl = make_float2(gl1, gl1);
        // eight columns at a time, in a loop that stays rolled: the code that a chunk runs has to fit the SM's instruction cache
#pragma unroll 1
        for (int k = col0; k < col0 + 16; k += 8) {
          uint32_t x[8], hi[4], lo[4];
          tc::tmem_ld8(lane_addr + K::P + k, x);
          tc::tmem_ld_wait();
          const int own = t - k, last = len - k;  // columns in front of own (forwards) or behind it have a part
#pragma unroll
          for (int i = 0; i < 8; i += 4) {
            const float4 h4 = *reinterpret_cast<const float4*>(gv + GV_H + k + i), l4 = *reinterpret_cast<const float4*>(gv + GV_L + k + i);
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
              const float2 d = __fadd2_rn(__fadd2_rn(gh, j ? make_float2(-h4.z, -h4.w) : make_float2(-h4.x, -h4.y)),
                                          __fadd2_rn(gl, j ? make_float2(-l4.z, -l4.w) : make_float2(-l4.x, -l4.y)));
              float2 p = __fmul2_rn(make_float2(ex2(d.x), ex2(d.y)), make_float2(__uint_as_float(x[i + j]), __uint_as_float(x[i + j + 1])));
              // what is masked may be anything; backwards also what lies behind the sequence
              if (kRev ? i + j < own || i + j >= last : i + j > own) p.x = 0.f;
              if (kRev ? i + j + 1 < own || i + j + 1 >= last : i + j + 1 > own) p.y = 0.f;
              split_pair(p, hi[(i + j) / 2], lo[(i + j) / 2]);
            }
          }
          uint8_t* piece = row + (((k >> 3) ^ (lane & 7)) << 4);
          *reinterpret_cast<uint4*>(piece) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
          *reinterpret_cast<uint4*>(piece + HALF) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        tc::tc_fence_before_sync();
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(pp_ready);
      }
      return true;
    };
    bool ok = true;
    int s = 0;
    uint32_t ph = 0;
#pragma unroll 1
    for (int c = 0; c < n_chunks; ++c) {
      const uint32_t cp = (uint32_t)c & 1u;
      const int s_c = s;
      const uint32_t ph_c = ph;
      if constexpr (!kState) {
        publish();
        if (!kGrad) ok = weigh(c, s_c, ph_c);  // (with the gradient of g the increment's second half waits for the first one to be taken)
        if (!ok) break;
      }
      ok = all(tc::mbar_wait(&ds_full[kState ? (int)cp : half], kState ? (uint32_t)(c >> 1) & 1u : cp, abort_flag));  // (the gate vectors were there before the images were)
      if (!ok) break;
      tc::tc_fence_after_sync();
      const float decay = reinterpret_cast<const float*>(smem + K::GV + s * GATES)[GV_TOT];
#pragma unroll
      for (int q = 0; q < HC / 16; ++q) {
        uint32_t x[16];
        tc::tmem_ld16(lane_addr + K::DS + cp * K::TURN_DS + (FH == 2 ? 0 : HC * grp) + 16 * q, x);
        tc::tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 8; ++i)
          S[8 * q + i] = __ffma2_rn(make_float2(decay, decay), S[8 * q + i], make_float2(__uint_as_float(x[2 * i]), __uint_as_float(x[2 * i + 1])));
      }
      tc::tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) { tc::mbar_arrive(&ds_empty[kState ? (int)cp : half]); tc::mbar_arrive(&empty[s]); }
      if (++s == K::STAGES) { s = 0; ph ^= 1u; }
      if constexpr (!kState) {
        if (kGrad) ok = weigh(c, s_c, ph_c);
        if (!ok) break;
        if (c + 1 < n_chunks) {  // the images may be written again
          ok = all(tc::mbar_wait(h_read, cp, abort_flag));
          if (!ok) break;
          tc::tc_fence_after_sync();
        }
      }
    }
    float* dst = kState ? a.seg_state + seg_tile : last && a.state_out != nullptr && !a.final_by_chain ? a.state_out + state_tile : nullptr;
    if (ok && mine && dst != nullptr) {
#pragma unroll
      for (int i = 0; i < HC / 2; ++i) {
        float* p = dst + (int64_t)(HC * grp + 2 * i) * a.st_y + (int64_t)d * a.st_w;
        p[0] = S[i].x; p[a.st_y] = S[i].y;
      }
    }
  } else if (!kState && warp < 16) {
    tc::reg_set<REGS_OUT, REGS_LAUNCH>();
    // ------------------------------------------------------------------ outputs: 32 features a warp, as accumulator fragments of warp-level MMAs, which matrix stores
    // transpose on their way into shared memory, in the place of the chunk's X (and Y, for 32-bit rows), whose readers are through; they leave by asynchronous copies
    if constexpr (!kState) {
      const int wq = warp & 3, gr = lane >> 2, t2 = 2 * (lane & 3), r8 = lane & 7, m4 = lane >> 3;
      const uint32_t lane_addr = tm + ((uint32_t)(wq * 32) << 16);
      const bool mine = 32 * wq < DV, f32 = a.o_part != nullptr;
      int before = -1;  // stage of the chunk before, whose rows may still be on their way out: its next tiles come when they have been read
      auto release = [&]() {
        if (lane == 0 && before >= 0) {
          tc::bulk_wait_read<0>();
          tc::mbar_arrive(&empty[before]);
        }
      };
      int s = 0;
      for (int c = 0; c < n_chunks; ++c) {
        const uint32_t cp = (uint32_t)c & 1u;
        if (!all(tc::mbar_wait2(o_full, cp, h_read, cp, abort_flag))) break;
        tc::tc_fence_after_sync();
        const float* gv = reinterpret_cast<const float*>(smem + K::GV + s * GATES);
        uint8_t* stage = smem + s * K::STAGE + (f32 ? K::Y + 8192 * wq : K::X + 4096 * wq);
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
            tc::tmem_ld_frags(lane_addr + ((uint32_t)hf << 20) + K::OI, oi);
            tc::tmem_ld_frags(lane_addr + ((uint32_t)hf << 20) + K::OA, oa);
            tc::tmem_ld_wait();
            if (hf == 1) {
              tc::tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) tc::mbar_arrive(o_empty);
              release();
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
        if (!mine) {
          if (lane == 0) tc::mbar_arrive(o_empty);
          release();
        }
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
            if (lane == 0) tc::tma_store_4d(&maps.o, stage, 32 * wq, h, (int)tok0, seg.b);
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
          __syncwarp();
          if (lane == 0) tc::bulk_commit();
        }
        before = s;
        if (++s == K::STAGES) s = 0;
      }
      if (lane == 0) tc::bulk_wait_all();
    }
  } else {
    tc::reg_set<REGS_PREP, REGS_LAUNCH>();
    // ------------------------------------------------------------------ images of W^T, each token times its weight, in bf16 terms: 32 features a warp, which matrix loads transpose into
    // pairs of tokens, the layout of a left operand.  (Y times the weights, in shared memory as right operand, was 64 KB more through shared memory a chunk, which
    // bounded it, and a third more instructions.)
    const int wq = warp & 3, r8 = lane & 7, m4 = lane >> 3, t2 = 2 * (lane & 3);
    // For the state alone the output's warps take every other chunk.
    constexpr int EACH = kState ? 2 : 1;
    int s = kState ? (warp >> 2) & 1 : 0;
    uint32_t ph = 0;
#pragma unroll 1
    for (int c = s; c < n_chunks; c += EACH) {
      const uint32_t cp = (uint32_t)c & 1u;
      const int len = min(C, seg.len - chunk_at(c) * C);
      bool ok = all(tc::mbar_wait2(&full[s], ph, &gates[s], ph, abort_flag));
      const float* gv = reinterpret_cast<const float*>(smem + K::GV + s * GATES);
      uint8_t* st = smem + s * K::STAGE;
      if (ok && len < C) {  // What lies behind the sequence in the tiles may be anything, and a product of zero with it need not be zero
        auto clear = [&](int at) { *reinterpret_cast<uint4*>(st + at) = make_uint4(0u, 0u, 0u, 0u); };
#pragma unroll 1
        for (int i = 8 * len + (threadIdx.x & 127); i < 512; i += 128) {
          clear(K::Y + 16 * i);
          if constexpr (DK == 128) clear(K::Y + HALF + 16 * i);
          if constexpr (!kState) clear(K::W + 16 * i);
          if constexpr (!kState && DV == 128) clear(K::W + HALF + 16 * i);
        }
        tc::fence_proxy_async_smem();
        __syncwarp();
        if (!kState && lane == 0) tc::mbar_arrive(cleared);
      }
#pragma unroll 1
      for (int q = 0; q < 2; ++q) {  // 32 tokens
        if (kState ? q == 0 : true) ok = ok && all(kState ? tc::mbar_wait(&img_read[cp], ((uint32_t)(c >> 1) & 1u) ^ 1u, abort_flag) : tc::mbar_wait(&img_read[q], cp ^ 1u, abort_flag));
        if (!ok) break;
        tc::tc_fence_after_sync();
        if (32 * wq < DV) {
          float2 w[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = *reinterpret_cast<const float2*>(gv + GV_W + 32 * q + 8 * i + t2);
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {  // 16 features
            const uint32_t w_s = tc::smem_u32(st + K::W) + (uint32_t)((wq >> 1) * HALF + (32 * q + 8 * (m4 >> 1) + r8) * 128 + (((4 * (wq & 1) + 2 * hf + (m4 & 1)) ^ r8) << 4));
            uint32_t x[8], terms[3][8];
            ldsm4t(reinterpret_cast<uint32_t(&)[4]>(x[0]), w_s);
            ldsm4t(reinterpret_cast<uint32_t(&)[4]>(x[4]), w_s + 2048);
            if (len < C)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                const int t = 32 * q + 8 * (i >> 1) + t2;
                if (t + 1 >= len) x[i] = t >= len ? 0u : x[i] & 0xffffu;
              }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float2 f = __fmul2_rn(bf16x2_to_float2(x[i]), w[i >> 1]);
              if constexpr (K::TERMS == 3) split3(f, terms[0][i], terms[1][i], terms[2][i]);
              else split_pair(f, terms[0][i], terms[1][i]);
            }
#pragma unroll
            for (int t = 0; t < K::TERMS; ++t) tc::tmem_st_pairs(tm + ((uint32_t)(32 * wq + 16 * hf) << 16) + K::IMG + cp * K::TURN_IMG + 32 * t + 16 * q, terms[t]);
          }
          tc::tmem_st_wait();
        }
        tc::tc_fence_before_sync();
        __syncwarp();
        if (lane == 0 && (!kState || q == 1)) tc::mbar_arrive(&img_ready[kState ? (int)cp : q]);
      }
      if (!ok) break;
      if ((s += EACH) >= K::STAGES) { s -= K::STAGES; ph ^= 1u; }
    }
  }

  tc::tc_fence_before_sync();
  __syncthreads();
  if (*abort_flag != 0u) {  // (the roles have ended: it stays as it is)
    if (threadIdx.x == 0 && a.status != nullptr) atomicOr(a.status, AVE_GDN_DEV_WAIT_EXPIRED);
    if (warp == 3 || (!kState && warp == 1)) tc::drain_mmas(&mma_end[warp == 1]);
    tc::tc_fence_before_sync();
    __syncthreads();
  }
  if (warp == 3) {
    tc::tc_fence_after_sync();
    tc::tmem_dealloc(tm, K::COLS);
  }
}

template <int DK, int DV, bool kRev, Mode kMode>
__global__ void __launch_bounds__(THREADS, 1) scan_kernel(const Args a, const __grid_constant__ Maps maps) {
  scan<DK, DV, kRev, kMode>(a, maps);
}

// Four numbers a thread, the next four segments read ahead; bound by their latency (8192 tokens x 32 heads in four segments: 6 us for 17 to 21 MB through L2).
// Between the two passes: seg_state goes from each segment's own increment to the state that enters it, and the last one's is the final state.
template <int DK, int DV, bool kRev>
__device__ __forceinline__ void chain(const Args& a) {
  pdl_wait();
  if (!offsets_fit(a, false)) return;
  constexpr int PARTS = DK * DV / 1024;
  const int part = blockIdx.x % PARTS, h = blockIdx.x / PARTS % a.Hv, n = blockIdx.x / PARTS / a.Hv;
  const SeqSpan sp = seq_span(a.cu_seqlens, n, a.T, nullptr);
  const int count = (sp.len + a.plan.len - 1) / a.plan.len;
  float* final = a.final_by_chain ? a.state_out : nullptr;
  if (!sp.ok || count < (final != nullptr ? 1 : 2)) return;
  int slot = n;
  if (a.state_indices != nullptr) slot = a.state_indices[n];
  if (slot < 0 || (a.state_indices != nullptr && slot >= a.num_slots)) return;
  const int64_t at = part * 1024 + threadIdx.x * 4, s0 = first_slot(a, n), tile = ((int64_t)slot * a.Hv + h) * (DK * DV) + at;
  float4 cur = make_float4(0.f, 0.f, 0.f, 0.f);
  if (a.state_in != nullptr) cur = *reinterpret_cast<const float4*>(a.state_in + tile);
  float* base = a.seg_state + h * (int64_t)(DK * DV) + at;
  const int64_t step = (int64_t)a.Hv * (DK * DV);
  const int own_until = final != nullptr ? count : count - 1;
  for (int i0 = 0; i0 < count; i0 += 4) {
    float4 own[4];
    float decay[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u < own_until) {
        const int64_t sl = s0 + (kRev ? count - 1 - i0 - u : i0 + u);
        own[u] = *reinterpret_cast<const float4*>(base + sl * step);
        decay[u] = a.seg_decay[sl * a.Hv + h];
      }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i0 + u < count) {
        const int64_t sl = s0 + (kRev ? count - 1 - i0 - u : i0 + u);
        *reinterpret_cast<float4*>(base + sl * step) = cur;
        if (i0 + u < own_until) {
          cur.x = fmaf(decay[u], cur.x, own[u].x); cur.y = fmaf(decay[u], cur.y, own[u].y);
          cur.z = fmaf(decay[u], cur.z, own[u].z); cur.w = fmaf(decay[u], cur.w, own[u].w);
        }
      }
  }
  if (final != nullptr) *reinterpret_cast<float4*>(final + tile) = cur;
}
template <int DK, int DV>
__global__ void __launch_bounds__(256) chain_kernel(const Args a) { chain<DK, DV, false>(a); }

}  // namespace lin
}  // namespace
}  // namespace ave
