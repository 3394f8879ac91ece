"""The product of 8-bit integers on the CPU: the source of its pairs and clusters of CTAs, compiled for the host (tests/host_cluster.h), with operands, products, arrivals and results that take their time."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "avelang_b200", "csrc")
CUDA = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")

DEVICE = """inline void mma_i8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) { cta::product(cta::rank, 1, d, a, b, idesc, accumulate); }
inline void mma_i8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (cta::rank != 0) cta::fail("products issued by the other CTA");
  cta::product(0, 2, d, a, b, idesc, accumulate);
}
namespace tc {
inline void tma_store_2d(const CUtensorMap* m, const void* src, int x, int y) { cta::store(m, src, x, y, (int)sizeof(TYPE)); }
}
"""

MAIN = r"""
using namespace ave;
static float get(__nv_bfloat16 x) { return __bfloat162float(x); }
static float get(__half x) { return __half2float(x); }
static float get(float x) { return x; }
struct Case { int m, n, k, bn, more, whole, ldc, first; };  // more: stages of the ring, or the cluster's share in `bn` columns; whole: tiles in front of the halves; the result's row distance and first column
static int expired, ended;
static const char* walk(const Case& c, unsigned seed, int limit, int late, long far, int level) {
  const int pitch = (c.k + 15) / 16 * 16, guard = 64;
  std::vector<int8_t> a((size_t)c.m * pitch), b((size_t)c.n * pitch);
  std::mt19937 rng(seed * 7919 + c.n);
  for (auto& x : a) x = (int8_t)rng();  // (what lies behind K too)
  for (auto& x : b) x = (int8_t)rng();
  std::vector<float> sa(c.m), sb(c.n), bias(c.n);
  for (auto& x : sa) x = 0.001f * (1 + rng() % 100);
  for (auto& x : sb) x = 0.001f * (1 + rng() % 100);
  for (auto& x : bias) x = 0.1f * (rng() % 100);
  TYPE mark, *buffer = (TYPE*)aligned_alloc(128, (((size_t)c.m * c.ldc + 2 * guard) * sizeof(TYPE) + 127) / 128 * 128);
  const size_t all = (size_t)c.m * c.ldc + 2 * guard;
  memset(&mark, 0x7b, sizeof(mark));
  std::fill(buffer, buffer + all, mark);
  TYPE* const out = buffer + guard + c.first;
  Epilogue e{sa.data(), sb.data(), bias.data(), out, c.ldc, 1, ((uintptr_t)out % 16 == 0 && c.ldc * sizeof(TYPE) % 16 == 0) ? 1 : 0};
  uint32_t status = 0;
  CUtensorMap map[3];
  for (int i = 0; i < 3; ++i) memcpy(&map[i], &i, 4);
  const char* fault = nullptr;
#ifdef PAIR
  const int tiles = (c.m + 255) / 256 * ((c.n + c.bn - 1) / c.bn), pairs = tiles > 5 ? 2 : 1, whole = std::min(c.whole, tiles);
  cta::maps = {{(uint8_t*)a.data(), c.k, c.m, pitch, 128}, {(uint8_t*)b.data(), c.k, c.n, pitch, whole < tiles ? c.bn / 4 : c.bn / 2},
               {(uint8_t*)out, (int64_t)c.n * (int64_t)sizeof(TYPE), c.m, (int64_t)c.ldc * (int64_t)sizeof(TYPE), 32}};
  for (int p = 0; p < pairs && !fault; ++p) {
    fault = cta::run(2 * p, 2 * pairs, seed + p, limit, late, far, level > 0, [&] { gemm_int8_pair_kernel<TYPE, BLOCKS>(map[0], map[1], map[2], e, c.m, c.n, c.k, &status, c.bn, c.more, (uint32_t)whole); });
  }
#else
  const Plan plan{c.bn, cta::CTAS, c.more, BLOCKS, (c.m + 7) / 8 * 8, 0};
  const int tiles = (c.n + c.bn - 1) / c.bn;
  cta::maps = {{(uint8_t*)a.data(), c.k, c.m, pitch, plan.a_rows}, {(uint8_t*)b.data(), c.k, c.n, pitch, c.bn}, {}};
  for (int t = 0; t < tiles && !fault; ++t)
    fault = cta::run(t * cta::CTAS, tiles * cta::CTAS, seed + t, limit, late, far, level > 0, [&] { gemm_int8_cluster_kernel<TYPE>(map[0], map[1], e, c.m, c.n, c.k, &status, plan, 256); });
#endif
  long wrong = 0, none = 0, kept = 0, beside = 0;
  const size_t begin = guard + c.first;
  for (size_t i = 0; i < all; ++i) {
    const long r = i < begin ? -1 : (long)((i - begin) / c.ldc), col = i < begin ? -1 : (long)((i - begin) % c.ldc);
    const bool same = memcmp(&buffer[i], &mark, sizeof(mark)) == 0;
    if (r < 0 || r >= c.m || col >= c.n) { beside += !same; continue; }
    int32_t sum = 0;
    for (int k = 0; k < c.k; ++k) sum += (int32_t)a[(size_t)r * pitch + k] * b[(size_t)col * pitch + k];
    const TYPE want = Elem<TYPE>::down(finish(sum, sa[r], sb[col], bias[col]));
    if (memcmp(&buffer[i], &want, sizeof(want)) == 0) continue;
    if (std::isnan(get(buffer[i]))) ++none;
    else if (same) ++kept;
    else ++wrong;
  }
  free(buffer);
  status != 0 ? ++expired : ++ended;
  if (fault) return fault;
  if (beside) return "what lies beside the result has changed";
  if (status != 0 && (limit == 1 << 30 || status != AVE_GDN_DEV_WAIT_EXPIRED)) return "the status word";
  if (status == 0 && (wrong || none || kept)) { printf("%ld wrong, %ld NaN, %ld not written\n", wrong, none, kept); return "results"; }
  if (level > 1 && (wrong || kept)) { printf("%ld wrong, %ld not written, status %u\n", wrong, kept, status); return "results behind an expired wait"; }
  return nullptr;
}
int main(int argc, char** argv) {  // seeds, of 1000 events so many are late by so many turns at most, polls of a wait, and what is looked at: that it ends, with nothing on its way, and results behind an expired wait
  const int seeds = atoi(argv[1]), late = atoi(argv[2]), far = atoi(argv[3]), limit = atoi(argv[4]), level = atoi(argv[5]);
  const Case cases[] = {CASES};
  for (const Case& c : cases)
    for (int seed = 1; seed <= seeds; ++seed) {
      const char* fault = walk(c, seed * 100, limit, late, far, level);
      if (fault) { printf("%d x %d x %d, seed %d: %s\n", c.m, c.n, c.k, seed, fault); return 1; }
    }
  printf("%d to the end, %d with an expiry\n", ended, expired);
  return ended > 0 && (expired > 0) == (limit < 1 << 30) ? 0 : 1;
}
"""


def own(code):
    """Static shared memory as a structure in the CTA's part of the host's."""
    def local(match):
        lines = re.findall(r"__shared__ ([^;]+;)", match.group(0))
        names = [n for line in lines for n in re.findall(r"(\w+)(?:\[[^\]]*\])?\s*[,;]", line)]
        return "".join(["struct Own { ", *[line + " " for line in lines], "}; Own& own = *(Own*)cta::space[cta::rank]; static_assert(sizeof(Own) <= cta::STATIC, \"\");\n",
                        *[f"auto& {n} = own.{n};\n" for n in names]])
    code, n = re.subn(r"extern __shared__ uint8_t smem_raw\[\];", "uint8_t* const smem_raw = cta::space[cta::rank] + cta::STATIC;", code)
    code, m = re.subn(r"(?:[ \t]*__shared__ [^\n]*\n)+", local, code)
    assert (n, m) == (2, 2) and "__shared__" not in code and "asm" not in code
    return code


def program(source):
    read = lambda name: open(os.path.join(CSRC, name)).read()
    cut = lambda text, a, b: text[text.index(a):text.index(b)]
    tc, rows = read("tc.cuh"), read("rows.cuh")
    descriptors = (cut(tc, "__device__ __forceinline__ uint64_t smem_desc_sw128", "// The two words of such a descriptor")
                   + cut(tc, "__host__ __device__ constexpr uint32_t desc_lo", "// 32-bit instruction descriptor"))
    kernels = cut(source, "constexpr int BM = 128", "__device__ __forceinline__ void mma_i8(") + DEVICE + own(cut(source, "struct Epilogue {", "// Tile width, K split and ring depth"))
    return ('#include "host_cluster.h"\n#include <type_traits>\nnamespace ave {\nnamespace tc {\n' + descriptors + "}\nnamespace rows {\n"
            + cut(rows, "template <class T> struct Elem;", "// The larger one, NaN where either is") + "}\nusing rows::Elem;\n" + kernels + "}  // namespace ave\n" + MAIN)


def run(tmp_path, source, pair, dtype, blocks, cases, seeds, late=0, far=1, limit=1 << 30, level=2, ctas=2):
    src, exe = tmp_path / "product.cpp", tmp_path / "product"
    src.write_text(program(source))
    listed = ",".join("{" + ",".join(map(str, c)) + "}" for c in cases)
    define = dict(TYPE=dtype, BLOCKS=blocks, CASES=listed, CLUSTER_CTAS=ctas, CTA_THREADS=320 if pair else 192, **({"PAIR": 1} if pair else {}))
    subprocess.run(["g++", "-std=c++17", "-O3", "-U_FORTIFY_SOURCE", "-w", "-Wno-psabi", "-ffp-contract=off", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "tests"), "-I", CUDA,
                    *[f"-D{k}={v}" for k, v in define.items()], str(src), "-o", str(exe)], check=True)
    return subprocess.run([str(exe), str(seeds), str(late), str(far), str(limit), str(level)], capture_output=True, text=True, timeout=900)


SOURCE = open(os.path.join(CSRC, "gemm_int8.cu")).read()

# rows, columns, K, columns a tile, stages, tiles in front of the halves, row distance and first column of the result
PAIRS = {
    ("__nv_bfloat16", 2): [(300, 130, 600, 128, 3, 99, 131, 0), (256, 66, 100, 64, 9, 99, 80, 8)],
    ("__half", 1): [(520, 300, 300, 256, 5, 3, 301, 1), (40, 450, 385, 256, 2, 1, 456, 0)],
    ("float", 1): [(300, 386, 260, 256, 4, 2, 388, 0), (260, 193, 130, 192, 5, 99, 195, 1)],
}
# rows, columns, K, columns a tile, stages, nothing, row distance and first column of the result
CLUSTERS = {
    ("__nv_bfloat16", 1, 2): [(100, 70, 520, 64, 3, 0, 72, 0), (3, 33, 385, 48, 10, 0, 33, 0)],
    ("float", 2, 3): [(65, 100, 1500, 96, 2, 0, 101, 0), (2, 16, 700, 16, 4, 0, 16, 0)],
}


@pytest.mark.parametrize("dtype,blocks", list(PAIRS))
def test_pairs(tmp_path, dtype, blocks):
    done = run(tmp_path, SOURCE, True, dtype, blocks, PAIRS[dtype, blocks], 3)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.parametrize("dtype,blocks,ctas", list(CLUSTERS))
def test_clusters(tmp_path, dtype, blocks, ctas):
    done = run(tmp_path, SOURCE, False, dtype, blocks, CLUSTERS[dtype, blocks, ctas], 4, ctas=ctas)
    assert done.returncode == 0, done.stdout + done.stderr


def test_pairs_with_fewer_blocks_than_stages(tmp_path):
    """Arrivals of finished products that are as late as the whole tile: neither CTA ends in front of them."""
    done = run(tmp_path, SOURCE, True, "__nv_bfloat16", 2, [(256, 66, 100, 64, 9, 99, 80, 8), (200, 130, 300, 128, 4, 99, 130, 0)], 12, late=150, far=3000000)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.parametrize("dtype,blocks", list(PAIRS))
def test_pairs_behind_an_expired_wait(tmp_path, dtype, blocks):
    """Operands, products and arrivals that come late, waits that some lanes of a warp have given up and others have not: every CTA comes to its end, with
    nothing on its way into it, and results are right or NaN."""
    done = run(tmp_path, SOURCE, True, dtype, blocks, PAIRS[dtype, blocks], 8, late=4, far=4000000, limit=100)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.parametrize("dtype,blocks,ctas", list(CLUSTERS))
def test_clusters_behind_an_expired_wait(tmp_path, dtype, blocks, ctas):
    done = run(tmp_path, SOURCE, False, dtype, blocks, CLUSTERS[dtype, blocks, ctas], 8, late=4, far=4000000, limit=400, ctas=ctas)
    assert done.returncode == 0, done.stdout + done.stderr


def without(was, now, count=1):
    assert SOURCE.count(was) == count, was
    return SOURCE.replace(was, now)


ENDS = dict(seeds=16, late=4, far=4000000)
HALVES = [(256, 700, 385, 256, 5, 0, 704, 0)]
ONE = [(256, 256, 640, 256, 5, 9, 256, 0)]


def test_half_tiles_behind_an_expired_wait(tmp_path):
    """Copies that one CTA of a pair has asked for alone are made up for by the bytes of their own tile."""
    done = run(tmp_path, SOURCE, True, "__half", 1, HALVES, 16, late=4, far=4000000, limit=60)
    assert done.returncode == 0, done.stdout + done.stderr


@pytest.mark.parametrize("pair,key,cases,was,now,fault,more", [
    (True, ("__half", 1), None, "if (begin || k + 1 == width)", "if (begin)", "results", dict(seeds=1)),
    (True, ("__half", 1), ONE, "tc::mbar_wait_together(&acc_full[buf]", "tc::mbar_wait_unrolled(&acc_full[buf]", "do not end", dict(seeds=16, late=20, far=400000, limit=600)),
    (True, ("__half", 1), HALVES, "tc::mbar_complete_tx(&full[i % stages], bytes(i))", "tc::mbar_complete_tx(&full[i % stages], landing(bn))", "do not end", dict(ENDS, limit=60)),
    (True, ("__half", 1), HALVES, "tc::mbar_expect_tx(&full[i % stages], bytes(i))", "tc::mbar_expect_tx(&full[i % stages], landing(bn))", "do not end", dict(ENDS, limit=60)),
    (True, ("__half", 1), None, "tc::drain(&empty[i % stages], i / stages & 1u);\n", ";\n", "on their way", dict(ENDS, limit=100)),
    (True, ("float", 1), None, "for (; tile < tiles; tile += step) {  //", "for (; false;) {  //", "behind an expired wait", dict(ENDS, limit=100)),
    (False, ("float", 2, 3), None, "last(full);", ";", "on their way", dict(ENDS, limit=400)),
    (False, ("float", 2, 3), None, "whole ? e.a_scale[at] : __uint_as_float(0x7fffffffu)", "e.a_scale[at]", "behind an expired wait", dict(ENDS, limit=400))])
def test_the_walks_see_what_is_missing(tmp_path, pair, key, cases, was, now, fault, more):
    """A store, a wait, a count or a mark that is left out of the source."""
    done = run(tmp_path, without(was, now), pair, key[0], key[1], cases or (PAIRS if pair else CLUSTERS)[key], ctas=2 if pair else key[2], **more)
    assert done.returncode == 1 and fault in done.stdout, done.stdout + done.stderr
