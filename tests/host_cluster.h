// The CTAs of one cluster on the host, for kernels whose operands, products and results are on their way while warps wait for one another: each thread is a context of its own, the next one to run is
// drawn at random, and warps run at changing speeds.  Copies, products, arrivals of finished products and stores complete some time after they were asked for, late ones after so long that waits have
// given up; a wait gives up after a number of polls, each lane for itself.  Tensor maps, swizzled operands, tensor memory and mbarriers hold what the device's would hold.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <setjmp.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <ucontext.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <map>
#include <random>
#include <vector>

#include "ave_gdn.h"

#undef __global__
#undef __host__
#undef __device__
#undef __forceinline__
#undef __launch_bounds__
#undef __cluster_dims__
#undef __grid_constant__
#define __global__
#define __host__
#define __device__
#define __forceinline__ inline
#define __launch_bounds__(...)
#define __cluster_dims__(...)
#define __grid_constant__

namespace cta {
constexpr int CTAS = CLUSTER_CTAS, THREADS = CTA_THREADS, ALL = CTAS * THREADS;
constexpr uint32_t STATIC = 4096, BLOCK = 1u << 18, REMOTE = 1u << 24;  // bytes of a CTA's own variables, of all its shared memory, and a window of the cluster's
alignas(1024) uint8_t space[CTAS][BLOCK];
int32_t tensor[CTAS][128][512];
struct Map { uint8_t* base; int64_t cols, rows, pitch; int box; };  // bytes a row, rows, bytes from row to row, rows of a box of 128 bytes
std::vector<Map> maps;
struct Phase { int count, pending; long tx; uint32_t phase; };
struct Meeting { int here = 0; long turn = 0; };
struct State {
  std::mt19937 rng;
  std::multimap<long, std::function<void()>> events;
  Phase bars[CTAS][STATIC / 8];
  std::map<int, Meeting> meetings;
  int64_t words[ALL];
  bool done[ALL];
  int left[CTAS], flying[CTAS], columns[CTAS];
  std::vector<long> stores[ALL];  // when a thread's stores complete
  long now = 0, products[CTAS] = {};  // products: when the last one that a CTA has issued completes
  int limit = 0, late = 0;        // polls of a wait; of 1000 events so many are late,
  long far = 0;                   // by so many turns at most
  bool over = true;               // whether a CTA may not end while something is on its way into it
  const char* fault = nullptr;
} s;
struct Index { unsigned x; } thread, block, grid;
int rank, self;
ucontext_t contexts[ALL];
jmp_buf back, at[ALL];
std::function<void()> body;

inline void fail(const char* what) { if (s.fault == nullptr) s.fault = what; }
inline void yield() {
  if (_setjmp(at[self]) == 0) _longjmp(back, 1);
}
inline void meet(int id, int count) {
  Meeting& m = s.meetings[id];
  const long turn = m.turn;
  if (++m.here == count) { m.here = 0; ++m.turn; return; }
  while (m.turn == turn) yield();
}
enum { WARP = 1000, ELECT = 2000, LANES = 3000, TENSOR = 4000, CLUSTER = 5000 };  // lanes that wait for one another in different places do not meet
inline void warp(int kind) { meet(kind + self / 32, 32); }
template <class T> T exchange(T x, int from) {
  memcpy(&s.words[self], &x, sizeof(T));
  warp(LANES);
  T y;
  memcpy(&y, &s.words[(self & ~31) | from], sizeof(T));
  warp(LANES);
  return y;
}
inline void event(int to, long due, std::function<void()> what) {  // something on its way into CTA `to`
  ++s.flying[to];
  s.events.emplace(due, [=] { --s.flying[to]; what(); });
}
inline long later() {
  const long usual = (long)(s.rng() % 1500);
  return s.now + ((int)(s.rng() % 1000) < s.late ? (long)(s.rng() % s.far) : usual);
}
inline uint8_t* address(uint32_t a) {  // of this CTA's or, in the cluster's window, of another one's
  const int to = a >= REMOTE ? (int)(a / REMOTE) - 1 : rank;
  if (s.left[to] == 0 && s.over) fail("a CTA that has ended is reached");
  return space[to] + a % REMOTE;
}
inline uint32_t place(const void* p) { return (uint32_t)(((const uint8_t*)p - space[0]) % BLOCK); }
inline int owner(const void* p) { return (int)(((const uint8_t*)p - space[0]) / BLOCK); }
inline Phase& bar(const void* p) { return s.bars[owner(p)][place(p) / 8]; }
inline void settle(Phase& p) {
  if (p.pending == 0 && p.tx == 0) { p.pending = p.count; ++p.phase; }
}
inline void arrive(void* at, long expect = 0) {
  Phase& p = bar(at);
  if (p.pending <= 0) fail("an arrival too many");
  --p.pending;
  p.tx += expect;
  settle(p);
}
inline void count(void* at, long bytes) {
  bar(at).tx -= bytes;
  settle(bar(at));
}
inline bool wait(void* at, uint32_t parity, volatile uint32_t* flag) {
  for (int it = 0; it < s.limit; ++it) {
    if ((bar(at).phase & 1u) != parity) return true;
    if (*flag != 0u && it > 1) return false;
    yield();
  }
  *flag = 1u;
  return false;
}
inline uint32_t swizzled(uint32_t a) { return a ^ (((a >> 7) & 7u) << 4); }
inline void load(void* dst, const CUtensorMap* m, uint8_t* at, int x, int y) {
  const Map map = maps[*(const int*)m];
  uint8_t* to = (uint8_t*)dst;
  if (x % 16 != 0 || place(to) % 128 != 0) fail("a copy off 16 bytes");
  ++s.flying[owner(at)];  // where its bytes are counted
  event(owner(to), later(), [=] {
    for (int r = 0; r < map.box; ++r)
      for (int b = 0; b < 128; ++b) {
        const bool there = y + r < map.rows && x + b < map.cols;
        space[owner(to)][swizzled(place(to) + r * 128 + b)] = there ? map.base[(int64_t)(y + r) * map.pitch + x + b] : 0;
      }
    --s.flying[owner(at)];
    count(at, map.box * 128);
  });
}
inline void store(const CUtensorMap* m, const void* src, int x, int y, int size) {
  const Map map = maps[*(const int*)m];
  const std::vector<uint8_t> copy((const uint8_t*)src, (const uint8_t*)src + map.box * 128);
  const uint8_t* from = (const uint8_t*)src;
  const long due = later();
  s.stores[self].push_back(due);
  event(rank, due, [=] {
    if (memcmp(from, copy.data(), copy.size()) != 0) fail("results are overwritten before they have left");
    for (int r = 0; r < map.box; ++r)
      for (int b = 0; b < 128; b += 16)  // whole pieces that begin inside the tensor
        if (y + r < map.rows && (int64_t)x * size + b < map.cols)
          memcpy(map.base + (int64_t)(y + r) * map.pitch + (int64_t)x * size + b, space[owner(from)] + swizzled(place(from) + r * 128 + b), 16);
  });
}
// One product of `rows` x n x 32 bytes of 8-bit integers by `ctas` CTAs from CTA `first` on
inline void product(int first, int ctas, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  const int n = (int)((idesc >> 17) & 63u) * 8, m = (int)((idesc >> 24) & 31u) * 16, column = (int)(d & 0xffffu);
  const uint32_t from_a = (uint32_t)(a & 0x3fffu) << 4, from_b = (uint32_t)(b & 0x3fffu) << 4;
  if (m != 128 * ctas || n % 16 != 0 || n == 0 || n > 256 || (a >> 61) != 2 || ((a >> 32) & 0x3fffu) != 64) fail("a descriptor");
  long& last = s.products[first];
  last = std::max(last, later());
  for (int i = 1; i < ctas; ++i) ++s.flying[first + i];
  event(first, last, [=] {
    static int8_t rows[256][32], columns[256][32];
    for (int i = 1; i < ctas; ++i) --s.flying[first + i];
    for (int r = 0; r < m; ++r)
      for (int k = 0; k < 32; ++k) rows[r][k] = (int8_t)space[first + r / 128][swizzled(from_a + (uint32_t)(r % 128) * 128 + k) % BLOCK];
    for (int c = 0; c < n; ++c)
      for (int k = 0; k < 32; ++k) columns[c][k] = (int8_t)space[first + c / (n / ctas)][swizzled(from_b + (uint32_t)(c % (n / ctas)) * 128 + k) % BLOCK];
    for (int r = 0; r < m; ++r)
      for (int c = 0; c < n; ++c) {
        int32_t sum = 0;
        for (int k = 0; k < 32; ++k) sum += (int32_t)rows[r][k] * columns[c][k];
        int32_t& to = tensor[first + r / 128][r % 128][column + c];
        to = accumulate ? to + sum : sum;
      }
  });
}
// An arrival at the same barrier of `ctas` CTAs behind all products issued so far, at each of them some time of its own later
inline void commit(int first, int ctas, uint64_t* at) {
  const uint32_t where = place(at);
  for (int i = 0; i < ctas; ++i) event(first + i, std::max(s.products[first], later()), [=] { arrive(space[first + i] + where); });
}

inline void entry() {
  body();
  s.done[self] = true;
  if (--s.left[rank] == 0 && s.flying[rank] != 0 && s.over) fail("on their way into a CTA that has ended");
  _longjmp(back, 1);
}
// Runs the cluster whose first CTA is b of n; returns what went wrong, or nothing.
inline const char* run(int b, int n, unsigned seed, int limit, int late, long far, bool over, std::function<void()> kernel) {
  s = State();
  s.rng.seed(seed); s.limit = limit; s.late = late; s.far = far; s.over = over;
  memset(space, 0x55, sizeof(space));
  memset(tensor, 0x55, sizeof(tensor));
  grid.x = n;
  body = kernel;
  static std::vector<uint8_t> stacks((size_t)ALL * 65536);
  static int order[ALL], left, next;
  static bool begun[ALL];
  for (int& x : s.left) x = THREADS;
  for (int i = 0; i < ALL; ++i) {
    getcontext(&contexts[i]);
    contexts[i].uc_stack = {&stacks[(size_t)i * 65536], 0, 65536};
    contexts[i].uc_link = nullptr;
    makecontext(&contexts[i], entry, 0);
    order[i] = i;
    begun[i] = false;
  }
  left = ALL;
  static int speed[ALL / 32];
  auto slow = [] { const int among[] = {1, 1, 4, 30}; return among[s.rng() % 4]; };  // turns of a warp's that are passed over
  for (int& x : speed) x = slow();
  while (left > 0) {
    if (s.rng() % 8192 == 0) speed[s.rng() % (ALL / 32)] = slow();
    next = (int)(s.rng() % left);
    self = order[next];
    rank = self / THREADS; thread.x = self % THREADS; block.x = b + rank;
    ++s.now;
    if (speed[self / 32] > 1 && s.rng() % speed[self / 32] != 0) continue;
    if (_setjmp(back) == 0) {
      if (begun[self]) _longjmp(at[self], 1);
      begun[self] = true;
      setcontext(&contexts[self]);
    }
    if (s.done[order[next]]) order[next] = order[--left];
    while (!s.events.empty() && s.events.begin()->first <= s.now) {
      auto what = s.events.begin()->second;
      s.events.erase(s.events.begin());
      what();
    }
    if (s.now > 80000000) return s.fault ? s.fault : "the CTAs do not end";
    if (s.fault) return s.fault;
  }
  for (int c : s.columns) if (c != 0) fail("tensor memory is not given back");
  return s.fault;
}
}  // namespace cta
#define threadIdx cta::thread
#define blockIdx cta::block
#define gridDim cta::grid

inline void __syncthreads() { cta::meet(cta::rank, cta::THREADS); }
inline void __syncwarp() { cta::warp(cta::WARP); }
template <class T> T __shfl_sync(unsigned, T x, int from) { return cta::exchange(x, from & 31); }
template <class T> T __shfl_down_sync(unsigned, T x, int by) { const int lane = cta::self & 31; return cta::exchange(x, lane + by < 32 ? lane + by : lane); }
inline int __all_sync(unsigned, int x) {
  cta::s.words[cta::self] = x != 0;
  cta::warp(cta::LANES);
  int all = 1;
  for (int i = 0; i < 32; ++i) all &= (int)cta::s.words[(cta::self & ~31) | i];
  cta::warp(cta::LANES);
  return all;
}
inline float __uint_as_float(uint32_t x) { float f; memcpy(&f, &x, 4); return f; }
inline uint32_t __float_as_uint(float f) { uint32_t x; memcpy(&x, &f, 4); return x; }
inline float2 __fadd2_rn(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
inline float2 __fmul2_rn(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }
inline float2 __ffma2_rn(float2 a, float2 b, float2 c) { return make_float2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); }
inline float __fmul_rn(float a, float b) { return a * b; }
inline uint32_t __byte_perm(uint32_t a, uint32_t b, uint32_t s) {
  const uint64_t both = (uint64_t)b << 32 | a;
  uint32_t r = 0;
  for (int i = 0; i < 4; ++i) r |= (uint32_t)(both >> (8 * ((s >> (4 * i)) & 7u)) & 0xffu) << (8 * i);
  return r;
}
inline uint32_t atomicOr(uint32_t* p, uint32_t x) { const uint32_t was = *p; *p |= x; return was; }
using std::max;
using std::min;

namespace ave {
inline float2 bf16x2_to_float2(uint32_t raw) { return make_float2(__uint_as_float(raw << 16), __uint_as_float(raw & 0xffff0000u)); }
inline uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat16 pair[2] = {__float2bfloat16(lo), __float2bfloat16(hi)};
  uint32_t x;
  memcpy(&x, pair, 4);
  return x;
}
inline void pdl_wait() {}
inline void pdl_trigger() {}
namespace tc {
inline uint8_t* align1024(uint8_t* p) { return p; }
inline uint32_t smem_u32(const void* p) { return cta::place(p); }
inline uint32_t mapa(uint32_t a, uint32_t rank) { return (rank + 1) * cta::REMOTE + a; }
inline uint32_t cluster_rank() { return (uint32_t)cta::rank; }
inline void cluster_sync() { cta::meet(cta::CLUSTER, cta::ALL); }
inline bool elect_one() {
  cta::warp(cta::ELECT);
  return (cta::self & 31) == 0;
}
inline void mbar_init(uint64_t* bar, uint32_t count) { cta::bar(bar) = {(int)count, (int)count, 0, 0}; }
inline void fence_barrier_init() {}
inline void fence_proxy_async_smem() {}
inline void tc_fence_before_sync() {}
inline void tc_fence_after_sync() {}
inline void prefetch_tmap(const CUtensorMap*) {}
inline void tma_prefetch_2d(const CUtensorMap*, int, int) {}
inline void mbar_expect_tx(uint64_t* bar, uint32_t bytes) { cta::arrive(bar, bytes); }
inline void mbar_complete_tx(uint64_t* bar, uint32_t bytes) { cta::count(bar, bytes); }
inline void mbar_arrive_cluster(uint32_t bar) { cta::arrive(cta::address(bar)); }
inline bool mbar_wait_unrolled(uint64_t* bar, uint32_t parity, volatile uint32_t* flag) { return cta::wait(bar, parity, flag); }
template <bool kCluster = false> bool mbar_wait_together(uint64_t* bar, uint32_t parity, volatile uint32_t* flag) {
  for (int it = 0; it < cta::s.limit; ++it) {
    if (__all_sync(0xffffffffu, (cta::bar(bar).phase & 1u) != parity)) return true;
    if (it > 1 && !__all_sync(0xffffffffu, *flag == 0u)) return false;
    cta::yield();
  }
  *flag = 1u;
  return false;
}
inline void drain(uint64_t* bar, uint32_t parity) {
  while ((cta::bar(bar).phase & 1u) == parity) cta::yield();
}
inline void st_cluster_u32(uint32_t a, uint32_t x) { memcpy(cta::address(a), &x, 4); }
inline void st_cluster_v4(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  const uint32_t v[4] = {x, y, z, w};
  memcpy(cta::address(a), v, 16);
}
inline void tma_load_2d(void* dst, const CUtensorMap* m, uint64_t* bar, int x, int y) { cta::load(dst, m, (uint8_t*)bar, x, y); }
inline void tma_load_2d_pair(void* dst, const CUtensorMap* m, uint32_t bar, int x, int y) { cta::load(dst, m, cta::address(bar), x, y); }
inline void bulk_commit() {}
inline void bulk_wait_all() {
  for (;;) {
    bool any = false;
    for (long due : cta::s.stores[cta::self]) any = any || due >= cta::s.now;
    if (!any) break;
    cta::yield();
  }
  cta::s.stores[cta::self].clear();
}
template <int N> void bulk_wait_read() { bulk_wait_all(); }
inline void alloc(uint32_t* slot, uint32_t cols) {
  cta::warp(cta::TENSOR);
  *slot = 0;
  if ((cta::self & 31) == 0) cta::s.columns[cta::rank] += (int)cols;
}
inline void dealloc(uint32_t cols) {
  cta::warp(cta::TENSOR);
  if ((cta::self & 31) == 0) cta::s.columns[cta::rank] -= (int)cols;
}
inline void tmem_alloc(uint32_t* slot, uint32_t cols) { alloc(slot, cols); }
inline void tmem_alloc_pair(uint32_t* slot, uint32_t cols) { alloc(slot, cols); }
inline void tmem_dealloc(uint32_t, uint32_t cols) { dealloc(cols); }
inline void tmem_dealloc_pair(uint32_t, uint32_t cols) { dealloc(cols); }
template <int N> void tmem_ld(uint32_t at, uint32_t (&r)[N]) {
  cta::warp(cta::TENSOR);
  memcpy(r, &cta::tensor[cta::rank][(at >> 16) + (cta::self & 31)][at & 0xffffu], sizeof(r));
}
inline void tmem_ld16(uint32_t at, uint32_t (&r)[16]) { tmem_ld<16>(at, r); }
inline void tmem_ld32(uint32_t at, uint32_t (&r)[32]) { tmem_ld<32>(at, r); }
inline void tmem_ld_wait() {}
inline void mma_commit(uint64_t* bar) { cta::commit(cta::rank, 1, bar); }
inline void mma_commit_pair(uint64_t* bar) { cta::commit(0, 2, bar); }
inline void drain_mmas(uint64_t* bar) {
  if (elect_one()) mma_commit(bar);
  __syncwarp();
  drain(bar, 0u);
}
}  // namespace tc
}  // namespace ave
