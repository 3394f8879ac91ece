"""The scan of linear attention on the CPU: the kernel's own source, compiled for the host with threads as contexts whose warps run at changing speeds, copies and MMAs that complete later than they
are issued, and waits that may give up.  Its numbers mean nothing here; that it ends, in step, with nothing on its way and its tensor memory given back, does."""
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "avelang_b200", "csrc")
CUDA = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")

DEVICE = r"""
#define CTA_THREADS 640
#include "host_cta.h"
#include <cuda.h>
namespace cta {
struct Store { unsigned thread; const uint8_t* src; long due; };
struct Commit { uint64_t* bar; long due; std::vector<uint32_t> reads; };
std::vector<Store> stores;
std::vector<Commit> commits[THREADS / 32];  // a warp's complete in order
std::vector<uint32_t> reads[THREADS / 32];  // shared memory that its MMAs since the last commit read: where each operand begins
std::map<const void*, uint32_t> boxes;      // bytes of a copy, by tensor map
int columns;                                // of tensor memory
int64_t words[THREADS];

inline long later() {
  const long usual = (long)(s.rng() % 1500);
  return s.now + ((int)(s.rng() % 1000) < s.late ? (long)(s.rng() % (8l * s.limit * THREADS)) : usual);
}
inline bool step() {  // what completes by now; whether anything is on its way
  bool any = false;
  for (auto& q : commits) {
    while (!q.empty() && q.front().due <= s.now) {
      Phase& p = s.bars[q.front().bar];
      --p.pending;
      complete(p);
      q.erase(q.begin());
    }
    any = any || !q.empty();
  }
  for (size_t i = 0; i < stores.size();) {
    if (stores[i].due <= s.now) stores.erase(stores.begin() + i); else ++i;
  }
  return any || !stores.empty();
}
inline void filled(const uint8_t* dst, uint32_t bytes) {
  const uint32_t a = (uint32_t)(dst - memory);
  auto in = [&](uint32_t x) { return x >= a && x < a + bytes; };
  for (auto& q : commits) for (auto& c : q) for (uint32_t x : c.reads) if (in(x)) s.fault = "a stage is filled while products read it";
  for (auto& r : reads) for (uint32_t x : r) if (in(x)) s.fault = "a stage is filled while products read it";
  for (auto& st : stores) if (in((uint32_t)(st.src - memory))) s.fault = "a stage is filled while rows leave it";
}
template <class T> T exchange(T x, int from) {
  const unsigned t = thread.x;
  memcpy(&words[t], &x, sizeof(T));
  warp();
  T y;
  memcpy(&y, &words[(t & ~31u) | (unsigned)from], sizeof(T));
  warp();
  return y;
}
}  // namespace cta
template <class T> T __shfl_sync(unsigned, T x, int from) { return cta::exchange(x, from & 31); }
template <class T> T __shfl_up_sync(unsigned, T x, int by) { const int lane = cta::thread.x & 31; return cta::exchange(x, lane >= by ? lane - by : lane); }
inline unsigned __ballot_sync(unsigned, bool x) {
  cta::words[cta::thread.x] = x;
  cta::warp();
  unsigned all = 0;
  for (unsigned i = 0; i < 32; ++i) all |= (unsigned)(cta::words[(cta::thread.x & ~31u) | i] != 0) << i;
  cta::warp();
  return all;
}
inline int __all_sync(unsigned m, bool x) { return __ballot_sync(m, x) == 0xffffffffu; }
inline int __syncthreads_or(int x) {
  static int sum;
  __syncthreads();
  if (cta::thread.x == 0) sum = 0;
  __syncthreads();
  sum |= x;
  __syncthreads();
  return sum;
}
inline int __ffs(unsigned x) { return __builtin_ffs((int)x); }
inline long long __float2ll_rn(float x) { return llrintf(x); }
inline float __ll2float_rn(long long x) { return (float)x; }
inline uint32_t __float_as_uint(float x) { uint32_t u; memcpy(&u, &x, 4); return u; }
using std::isnan;
using std::max;
using std::min;
namespace ave {
inline uint32_t pack_bf16x2(float, float) { return 0; }
inline void ldsm4t(uint32_t (&x)[4], uint32_t) { x[0] = x[1] = x[2] = x[3] = 0; }
inline void stsm4t(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) {}
inline void split_pair(float2, uint32_t& a, uint32_t& b) { a = b = 0; }
inline void split3(float2, uint32_t& a, uint32_t& b, uint32_t& c) { a = b = c = 0; }
namespace tc {
inline uint8_t* align1024(uint8_t* p) { return p; }
inline uint32_t smem_u32(const void* p) { return (uint32_t)((const uint8_t*)p - cta::memory); }
inline void mbar_arrive(uint64_t* bar) {
  cta::Phase& p = cta::s.bars[bar];
  if (p.pending <= 0) cta::s.fault = "an arrival too many";
  --p.pending;
  cta::complete(p);
}
inline bool mbar_wait2(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, volatile uint32_t* flag) { return mbar_wait(a, pa, flag) && mbar_wait(b, pb, flag); }
inline bool mbar_wait3(uint64_t* a, uint32_t pa, uint64_t* b, uint32_t pb, uint64_t* c, uint32_t pc, volatile uint32_t* flag) { return mbar_wait2(a, pa, b, pb, flag) && mbar_wait(c, pc, flag); }
inline void fence_proxy_async_smem() {}
inline void tc_fence_before_sync() {}
inline void tc_fence_after_sync() {}
inline void prefetch_tmap(const CUtensorMap*) {}
template <int A, int B> void reg_set() {}
inline bool elect_one() { return (cta::thread.x & 31) == 0; }
inline void tma_load_5d(void* dst, const CUtensorMap* m, uint64_t* bar, int, int, int, int, int) {
  const uint32_t bytes = cta::boxes[m];
  cta::filled((uint8_t*)dst, bytes);
  cta::s.copies.push_back({dst, dst, bytes, bar, false, cta::later()});
}
inline void tma_store_4d(const CUtensorMap*, const void* src, int, int, int, int) { cta::stores.push_back({cta::thread.x, (const uint8_t*)src, cta::s.now + (long)(cta::s.rng() % (cta::s.late == 0 ? 1000000 : 40000))}); }
inline void bulk_commit() {}
inline void bulk_wait_all() {
  for (;;) {
    bool mine = false;
    for (auto& st : cta::stores) mine = mine || st.thread == cta::thread.x;
    if (!mine) return;
    cta::yield();
  }
}
template <int N> void bulk_wait_read() { bulk_wait_all(); }
inline void tmem_alloc(uint32_t* slot, uint32_t cols) { *slot = 0; if (elect_one()) cta::columns += (int)cols; }
inline void tmem_dealloc(uint32_t, uint32_t cols) { if (elect_one()) cta::columns -= (int)cols; }
inline void tmem_ld8(uint32_t, uint32_t (&r)[8]) { memset(r, 0, sizeof(r)); }
inline void tmem_ld16(uint32_t, uint32_t (&r)[16]) { memset(r, 0, sizeof(r)); }
inline void tmem_ld_frags(uint32_t, uint32_t (&r)[32]) { memset(r, 0, sizeof(r)); }
inline void tmem_ld_wait() {}
inline void tmem_st8(uint32_t, const uint32_t (&)[8]) {}
inline void tmem_st_pairs(uint32_t, const uint32_t (&)[8]) {}
inline void tmem_st_wait() {}
inline void reading(uint64_t desc) { cta::reads[cta::thread.x >> 5].push_back((uint32_t)(desc & 0x3fffu) << 4); }
inline void mma_ss(uint32_t, uint64_t a, uint64_t b, uint32_t, uint32_t) { reading(a); reading(b); }
inline void mma_ts(uint32_t, uint32_t, uint64_t b, uint32_t, uint32_t) { reading(b); }
inline void mma_commit(uint64_t* bar) {
  auto& q = cta::commits[cta::thread.x >> 5];
  auto& own = cta::reads[cta::thread.x >> 5];
  long due = own.empty() ? cta::s.now : cta::later();  // (without products of its own it completes with those before)
  if (!q.empty()) due = std::max(due, q.back().due);
  q.push_back({bar, due, own});
  own.clear();
}
inline void drain_mmas(uint64_t* bar) {
  if (elect_one()) mma_commit(bar);
  __syncwarp();
  drain(bar, 0u);
}
"""
MAIN = r"""
using namespace ave;
template <class X> X* place(size_t n) { return (X*)aligned_alloc(128, (n * sizeof(X) + 127) / 128 * 128); }
template <int DK, int DV, bool kRev, lin::Mode kMode>
int walk() {
  using K = lin::Cfg<kMode>;
  constexpr int MOST = 64 * 8;
  int done = 0, expired = 0;
  lin::Args a{};
  a.B = a.Hv = a.n_seqs = a.num_slots = 1;
  a.x_div = a.y_div = a.w_div = a.e_div = 1;
  a.scale_e = a.scale_w = 1.f;
  float* g = place<float>(MOST);
  for (int t = 0; t < MOST; ++t) g[t] = -0.01f * (t % 7);
  a.g = g; a.g_stride_t = 1; a.g_stride_b = MOST;
  a.o = place<__nv_bfloat16>(MOST * DV); a.o_stride_t = a.o_stride_h = DV; a.o_stride_b = MOST * DV;
  a.state_out = place<float>(DK * DV); a.st_y = DV; a.st_w = 1;
  a.seg_state = place<float>(DK * DV); a.seg_decay = place<float>(1);
  a.inter = place<float>(4 * MOST);
  a.final_by_chain = kMode == lin::STATE;
  a.plan = lin::Plan{1 << 30, 0, 1};
  memset(a.seg_state, 0, DK * DV * 4);
  lin::Maps maps{};
  cta::boxes = {{&maps.x, DK * 128}, {&maps.y, DK * 128}, {&maps.w, DV * 128}, {&maps.e, DV * 128}};
  for (int late : {0, 5, 30})
    for (int seed = 1; seed <= 2; ++seed)
      for (int T : {1, 65, 500}) {
        uint32_t status = 0;
        a.T = T; a.status = &status;
        maps.o_ok = (seed + T) % 3 != 0;
        cta::columns = 0;
        cta::stores.clear();
        for (auto& q : cta::commits) q.clear();
        for (auto& r : cta::reads) r.clear();
        const char* fault = cta::run(0, 1, seed * 1000 + T, late == 0 ? 1 << 30 : 600, late, 32, [&] { lin::scan<DK, DV, kRev, kMode>(a, maps); }, cta::step);
        if (fault == nullptr && cta::columns != 0) fault = "tensor memory is not given back";
        if (fault == nullptr && status != 0 && (late == 0 || status != AVE_GDN_DEV_WAIT_EXPIRED)) fault = "the status word";
        if (fault != nullptr) { printf("T %d, seed %d, late %d: %s (status %u)\n", T, seed, late, fault, status); return 1; }
        if (status == 0) ++done; else ++expired;
      }
  printf("%d walks to the end, %d with an expiry\n", done, expired);
  return done > 0 && expired > 0 ? 0 : 1;
}
int main() { return walk<KEYS, VALUES, REVERSE, lin::MODE>(); }
"""


def program(scan, tc, common):
    cut = lambda text, a, b: text[text.index(a):text.index(b)]
    code = cut(scan, "constexpr int C = 64;", "template <int DK, int DV, bool kRev, Mode kMode>\n__global__ void")
    for device, host in (('asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));', "y = exp2f(x);"), ('asm volatile("" : "+l"(src));', ""),
                         ("extern __shared__ uint8_t smem_raw[];", "uint8_t* const smem_raw = cta::memory;")):
        assert code.count(device) == 1, device
        code = code.replace(device, host)
    assert "asm" not in code
    descriptors = cut(tc, "__host__ __device__ constexpr uint32_t desc_lo", "// ---------------------------------------------------------------- MMA")
    return DEVICE + descriptors + "}  // namespace tc\n" + cut(common, "struct SeqSpan {", "}  // namespace ave") + "namespace lin {\n" + code + "}  // namespace lin\n}  // namespace ave\n" + MAIN


def run(tmp_path, scan, mode, keys, values, reverse):
    read = lambda name: open(os.path.join(CSRC, name)).read()
    src, exe = tmp_path / "scan.cpp", tmp_path / "scan"
    src.write_text(program(scan, read("tc.cuh"), read("common.cuh")))
    define = dict(MODE=mode, KEYS=keys, VALUES=values, REVERSE=reverse)
    subprocess.run(["g++", "-std=c++17", "-O2", "-U_FORTIFY_SOURCE", "-w", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "tests"), "-I", CUDA,
                    *[f"-D{k}={v}" for k, v in define.items()], str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe)], capture_output=True, text=True, timeout=600)


SCAN = open(os.path.join(CSRC, "linear_scan.cuh")).read()


@pytest.mark.parametrize("mode,keys,values,reverse", [("STATE", 128, 64, "true"), ("OUT2", 128, 128, "false"), ("OUT3", 64, 128, "true"), ("GRAD", 128, 128, "false"),
                                                      ("GRAD", 64, 64, "true")])
def test_the_scan_ends_in_step_whatever_expires(tmp_path, mode, keys, values, reverse):
    done = run(tmp_path, SCAN, mode, keys, values, reverse)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.parametrize("mode,was,now,fault", [
    ("OUT2", "all(tc::mbar_wait2(pp_ready, cp, o_empty, cp ^ 1u, abort_flag))", "all(tc::mbar_wait(pp_ready, cp, abort_flag))", "does not end"),
    ("OUT2", "if (c >= K::STAGES && !tc::mbar_wait(&empty[s], ph, abort_flag)) break;", "", "is filled"),
    ("OUT2", "          tc::bulk_wait_read<0>();\n", "", "while rows leave it"),
    ("STATE", "for (int c = max(0, issued - K::STAGES); c < issued; ++c) tc::drain(", "for (int c = issued; c < issued; ++c) tc::drain(", "on their way"),
    ("STATE", "if (warp == 3 || (!kState && warp == 1)) tc::drain_mmas(&mma_end[warp == 1]);", "", "on their way")])
def test_the_walks_see_what_is_missing(tmp_path, mode, was, now, fault):
    """A wait that is left out of the source."""
    assert SCAN.count(was) == 1
    done = run(tmp_path, SCAN.replace(was, now), mode, 128, 128, "false")
    assert done.returncode == 1 and fault in done.stdout, done.stdout + done.stderr
