// One CTA on the host, for kernels whose waits on asynchronous copies may expire: each of its threads is a context of its own, the next one to run is drawn at random, copies land
// some time after they were asked for (late ones after so many polls that some of those who wait have given up), and a wait gives up after a number of polls.  Shuffles, barriers and mbarriers do what the device's do.
#pragma once
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
#undef __shared__
#undef __forceinline__
#undef __launch_bounds__
#define __global__
#define __host__
#define __device__
#define __shared__ static
#define __forceinline__ inline
#define __launch_bounds__(...)

namespace cta {
#ifndef CTA_THREADS
#define CTA_THREADS 256
#endif
constexpr int THREADS = CTA_THREADS;
struct Copy { void* dst; const void* src; uint32_t bytes; uint64_t* bar; bool late; long due; };  // a turn, or a number of polls
struct Phase { int count, pending; long tx; uint32_t phase; long polls; };
struct Meeting { int here = 0; long turn = 0; };
struct State {
  std::mt19937 rng;
  std::vector<Copy> copies;
  std::map<uint64_t*, Phase> bars;
  std::map<int, Meeting> meetings;
  float lanes[THREADS];
  bool done[THREADS];
  long now = 0;
  int limit = 0, late = 0, pollers = 0;  // polls of a wait; of 1000 copies so many are late; threads that wait for a copy
  const char* fault = nullptr;
} s;
struct Index { unsigned x; } thread, block, grid, size{THREADS};
ucontext_t contexts[THREADS];  // a thread's first turn; from then on by jumps, which save no signal masks
jmp_buf back, at[THREADS];
std::function<void()> body;
alignas(1024) uint8_t memory[232448];

inline void yield() {
  if (_setjmp(at[thread.x]) == 0) _longjmp(back, 1);
}
inline void meet(int id, int count) {
  Meeting& m = s.meetings[id];
  const long turn = m.turn;
  if (++m.here == count) { m.here = 0; ++m.turn; return; }
  while (m.turn == turn) yield();
}
inline void warp() { meet(1000 + (int)(thread.x >> 5), 32); }
inline void complete(Phase& p) {
  if (p.pending == 0 && p.tx == 0) { p.pending = p.count; ++p.phase; p.polls = 0; }
}
inline void entry() {
  body();
  s.done[thread.x] = true;
  _longjmp(back, 1);
}
inline int slow() { const int among[] = {1, 1, 4, 30}; return among[s.rng() % 4]; }  // turns of a warp's that are passed over
// Runs CTA b of n; returns what went wrong, or nothing.
inline const char* run(int b, int n, unsigned seed, int limit, int late, int pollers, std::function<void()> kernel, std::function<bool()> step = nullptr) {
  s = State();
  s.rng.seed(seed); s.limit = limit; s.late = late; s.pollers = pollers;
  block.x = b; grid.x = n;
  body = kernel;
  static std::vector<uint8_t> stacks(THREADS * 65536);
  for (int i = 0; i < THREADS; ++i) {
    getcontext(&contexts[i]);
    contexts[i].uc_stack = {&stacks[(size_t)i * 65536], 0, 65536};
    contexts[i].uc_link = nullptr;
    makecontext(&contexts[i], entry, 0);
  }
  static int order[THREADS], left, next;
  static bool begun[THREADS];
  left = THREADS;
  for (int i = 0; i < THREADS; ++i) { order[i] = i; begun[i] = false; }
  int speed[THREADS / 32];
  for (int& x : speed) x = step ? slow() : 1;
  while (left > 0) {
    if (step && s.rng() % 4096 == 0) speed[s.rng() % (THREADS / 32)] = slow();
    next = (int)(s.rng() % left);
    thread.x = order[next];
    if (speed[thread.x >> 5] > 1 && s.rng() % speed[thread.x >> 5] != 0) { ++s.now; continue; }
    if (_setjmp(back) == 0) {
      if (begun[thread.x]) _longjmp(at[thread.x], 1);
      begun[thread.x] = true;
      setcontext(&contexts[thread.x]);
    }
    if (s.done[order[next]]) order[next] = order[--left];
    ++s.now;
    for (size_t i = 0; i < s.copies.size();) {
      Copy c = s.copies[i];
      Phase& p = s.bars[c.bar];
      if (c.due > (c.late ? p.polls : s.now)) { ++i; continue; }
      memcpy(c.dst, c.src, c.bytes);
      p.tx -= c.bytes;
      complete(p);
      s.copies.erase(s.copies.begin() + i);
    }
    if (step) step();
    if (s.now > 25000000) return s.fault ? s.fault : "the CTA does not end";
  }
  if (step && step()) return "copies or products on their way in a CTA that has ended";
  if (!s.copies.empty()) return "copies on their way into a CTA that has ended";
  return s.fault;
}
}  // namespace cta
#define threadIdx cta::thread
#define blockIdx cta::block
#define gridDim cta::grid
#define blockDim cta::size

inline void __syncthreads() { cta::meet(0, cta::THREADS); }
inline void __syncwarp() { cta::warp(); }
inline float __shfl_xor_sync(unsigned, float x, int mask) {
  const unsigned t = cta::thread.x;
  cta::s.lanes[t] = x;
  cta::warp();
  const float y = cta::s.lanes[t ^ (unsigned)mask];
  cta::warp();
  return y;
}
inline float __int_as_float(int x) { float f; memcpy(&f, &x, 4); return f; }
inline float __uint_as_float(uint32_t x) { float f; memcpy(&f, &x, 4); return f; }
inline float2 __fadd2_rn(float2 a, float2 b) { return make_float2(a.x + b.x, a.y + b.y); }
inline float2 __fmul2_rn(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }
inline float2 __ffma2_rn(float2 a, float2 b, float2 c) { return make_float2(fmaf(a.x, b.x, c.x), fmaf(a.y, b.y, c.y)); }
inline uint32_t atomicOr(uint32_t* p, uint32_t x) { const uint32_t was = *p; *p |= x; return was; }

namespace ave {
inline float2 bf16x2_to_float2(uint32_t raw) { return make_float2(__uint_as_float(raw << 16), __uint_as_float(raw & 0xffff0000u)); }
inline void pdl_wait() {}
namespace tc {
inline void mbar_init(uint64_t* bar, uint32_t count) { cta::s.bars[bar] = {(int)count, (int)count, 0, 0, 0}; }
inline void fence_barrier_init() {}
inline void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  cta::Phase& p = cta::s.bars[bar];
  if (p.tx != 0) cta::s.fault = "a slot is filled again before its copies have landed";
  --p.pending;
  p.tx += bytes;
}
inline void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  const bool late = (int)(cta::s.rng() % 1000) < cta::s.late;
  const long polls = (long)cta::s.limit * cta::s.pollers;
  cta::s.copies.push_back({dst, src, bytes, bar, late, late ? polls / 2 + (long)(cta::s.rng() % polls) : cta::s.now + (long)(cta::s.rng() % (32 * std::min(cta::s.limit, 8)))});
}
inline bool seen(uint64_t* bar, uint32_t parity) {
  ++cta::s.bars[bar].polls;
  return (cta::s.bars[bar].phase & 1u) != parity;
}
inline bool mbar_wait(uint64_t* bar, uint32_t parity, volatile uint32_t* abort_flag) {
  int left = cta::s.limit;
  while (!seen(bar, parity)) {
    if (*abort_flag != 0u || --left == 0) { *abort_flag = 1u; return false; }
    cta::yield();
  }
  return true;
}
inline void drain(uint64_t* bar, uint32_t parity) {
  while (!seen(bar, parity)) cta::yield();
}
}  // namespace tc
}  // namespace ave
