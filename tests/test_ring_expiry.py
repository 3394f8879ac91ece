"""Layer norm's rings when a wait for a copy expires, on the CPU: the kernels' own source, compiled for the host with threads as contexts in a random order, copies that may be late and waits
that may give up.  A row is then right to the last bit or NaN in all of its results, a column of the weights' gradients likewise, the status word says so, no slot is filled while a copy into it is
on its way, and none is on its way into a CTA that has ended."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUDA = os.path.join(os.environ.get("CUDA_HOME", "/usr/local/cuda"), "include")

MAIN = r"""
using namespace ave;
static float value(int r, int c, int salt) { return (float)((r * 7919 + c * 104729 + salt * 1299709) % 2003) / 500.f - 2.f; }
template <class X> X* place(size_t n) { return (X*)aligned_alloc(128, (n * sizeof(X) + 127) / 128 * 128); }
static void put(__nv_bfloat16& x, float f) { x = __float2bfloat16(f); }
static void put(float& x, float f) { x = f; }
static float get(__nv_bfloat16 x) { return __bfloat162float(x); }
static float get(float x) { return x; }

template <class T>
struct Run {
  int rows, n;
  T *x, *dy, *y, *dx;
  float *w, *b, *mean, *rstd, *partial;
  uint32_t status = 0;
  Run(int rows, int n) : rows(rows), n(n), x(place<T>(rows * n)), dy(place<T>(rows * n)), y(place<T>(rows * n)), dx(place<T>(rows * n)), w(place<float>(n)), b(place<float>(n)),
        mean(place<float>(rows)), rstd(place<float>(rows)), partial(place<float>(2 * n)) {
    for (int r = 0; r < rows; ++r) {
      for (int c = 0; c < n; ++c) { put(x[r * n + c], value(r, c, 1)); put(dy[r * n + c], value(r, c, 2)); put(y[r * n + c], -77.f); put(dx[r * n + c], -77.f); }
      mean[r] = value(r, 0, 3); rstd[r] = 1.f + 0.1f * value(r, 0, 4);
    }
    for (int c = 0; c < n; ++c) { w[c] = value(0, c, 5); b[c] = value(0, c, 6); }
    for (int c = 0; c < 2 * n; ++c) partial[c] = -77.f;
  }
  template <int P, int G>
  const char* forward(unsigned seed, int depth, int limit, int late) {
    AveLayerNormArgs a{};
    a.struct_size = sizeof(a); a.x = x; a.y = y; a.weight = w; a.bias = b; a.mean = mean; a.rstd = rstd; a.rows = rows; a.n = n; a.x_stride = a.y_stride = n;
    a.w_dtype = AVE_DTYPE_FP32; a.eps = 1e-5f; a.status = &status;
    memset(cta::memory, 0x40, sizeof(cta::memory));  // (finite)
    return cta::run(0, 1, seed, limit, late, 32 * G, [=] { layer_norm_ring_kernel<T, P, G>(a, depth, true); });
  }
  template <int P, int G>
  const char* backward(unsigned seed, int depth, int limit, int late) {
    AveLayerNormBwdArgs a{};
    a.struct_size = sizeof(a); a.d_y = dy; a.x = x; a.mean = mean; a.rstd = rstd; a.weight = w; a.d_x = dx; a.rows = rows; a.n = n; a.dy_stride = a.x_stride = a.dx_stride = n;
    a.w_dtype = AVE_DTYPE_FP32; a.status = &status;
    memset(cta::memory, 0x40, sizeof(cta::memory));
    return cta::run(0, 1, seed, limit, late, 32 * G, [=] { layer_norm_backward_ring_kernel<T, P, G>(a, partial, depth, true); });
  }
};
static int all_nan, all_right, wrong;
template <class F> void tally(int count, F same) {  // same(i): 1 the right bits, 0 NaN, -1 neither
  int right = 0, nan = 0;
  for (int i = 0; i < count; ++i) { const int s = same(i); right += s == 1; nan += s == 0; }
  if (right == count) ++all_right; else if (nan == count) ++all_nan; else ++wrong;
}
static int compare(float got, float want) { return std::isnan(got) ? 0 : got == want ? 1 : -1; }

template <class T, int P, int G>
int whole(int rows, int n, int depth, int seeds) {
  int expired = 0;
  for (int pass = 0; pass < 2; ++pass) {
    Run<T> ref(rows, n);
    const char* fault = pass == 0 ? ref.template forward<P, G>(1, depth, 1 << 30, 0) : ref.template backward<P, G>(1, depth, 1 << 30, 0);
    if (fault != nullptr || ref.status != 0) { printf("undisturbed: %s, status %u\n", fault ? fault : "-", ref.status); return 1; }
    if (pass == 0)  // what the emulated CTA makes of a row
      for (int r = 0; r < rows; ++r) {
        double m = 0, v = 0;
        for (int c = 0; c < n; ++c) m += get(ref.x[r * n + c]) / n;
        for (int c = 0; c < n; ++c) v += (get(ref.x[r * n + c]) - m) * (get(ref.x[r * n + c]) - m) / n;
        if (std::fabs(ref.mean[r] - m) > 1e-5 || std::fabs(ref.rstd[r] - 1 / std::sqrt(v + 1e-5)) > 1e-5) { printf("undisturbed: row %d\n", r); return 1; }
      }
    for (int seed = 1; seed <= seeds; ++seed) {
      Run<T> got(rows, n);
      const int before = all_nan;
      fault = pass == 0 ? got.template forward<P, G>(seed, depth, 8, 30) : got.template backward<P, G>(seed, depth, 6, 100);
      if (fault != nullptr) { printf("seed %d: %s\n", seed, fault); return 1; }
      for (int r = 0; r < rows; ++r)
        tally(pass == 0 ? n + 2 : n, [&](int i) {
          if (pass == 1) return compare(get(got.dx[r * n + i]), get(ref.dx[r * n + i]));
          return i < n ? compare(get(got.y[r * n + i]), get(ref.y[r * n + i])) : i == n ? compare(got.mean[r], ref.mean[r]) : compare(got.rstd[r], ref.rstd[r]);
        });
      if (pass == 1)
        for (int c = 0; c < 2 * n; ++c) tally(1, [&](int) { return compare(got.partial[c], ref.partial[c]); });
      const bool nan = all_nan > before;
      if (got.status != (nan ? AVE_GDN_DEV_WAIT_EXPIRED : 0u)) { printf("seed %d, pass %d: status %u with %s\n", seed, pass, got.status, nan ? "NaN" : "no NaN"); return 1; }
      expired += nan;
    }
    if (wrong > 0) { printf("pass %d: %d rows or columns wrong beside %d right and %d NaN\n", pass, wrong, all_right, all_nan); return 1; }
  }
  printf("right %d NaN %d runs with an expiry %d of %d\n", all_right, all_nan, expired, 2 * seeds);
  return all_right > 0 && all_nan > 0 && expired > 0 && expired < 2 * seeds ? 0 : 1;
}
int main() { return whole<TYPE, PIECES, GROUP>(ROWS, COLUMNS, DEPTH, 30); }
"""


def kernels(text):
    """Rows' pieces and the ring kernels; what the host has no word for is put in its terms."""
    cut = lambda a, b: text[text.index(a):text.index(b)]
    code = (cut("template <class T> struct Elem;", "// U sums over the TPR threads") + cut("constexpr int RING", "// Sums of CTA c: partial")
            + cut("// The same for the gradients: a slot holds", "// Long rows: "))
    code, n = re.subn(r'asm volatile\("bar.sync %0, %1;" ::"r"\((.*?)\), "r"\((32 \* G)\) : "memory"\);', r"cta::meet(\1, \2);", code)
    code, m = re.subn(r"extern __shared__ __align__\(128\) uint8_t ring_mem\[\];", "uint8_t* const ring_mem = cta::memory;", code)
    assert (n, m) == (1, 2) and "asm" not in code
    return code


@pytest.mark.parametrize("dtype,pieces,group,rows,columns,depth", [("__nv_bfloat16", 1, 8, 12, 520, 3), ("__nv_bfloat16", 2, 1, 40, 264, 2), ("float", 2, 2, 24, 508, 8), ("float", 8, 4, 12, 2052, 2)])
def test_an_expired_wait_leaves_rows_right_or_nan(tmp_path, dtype, pieces, group, rows, columns, depth):
    source = open(os.path.join(ROOT, "avelang_b200", "csrc", "layer_norm.cu")).read()
    src, exe = tmp_path / "ring.cpp", tmp_path / "ring"
    src.write_text('#include "host_cta.h"\nnamespace ave {\n' + kernels(source) + "\n}  // namespace ave\n" + MAIN)
    define = dict(TYPE=dtype, PIECES=pieces, GROUP=group, ROWS=rows, COLUMNS=columns, DEPTH=depth)
    subprocess.run(["g++", "-std=c++17", "-O2", "-U_FORTIFY_SOURCE", "-w", "-ffp-contract=off", "-I", os.path.join(ROOT, "include"), "-I", os.path.join(ROOT, "tests"), "-I", CUDA,
                    *[f"-D{k}={v}" for k, v in define.items()], str(src), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stdout + done.stderr


def test_the_status_word_may_be_missing(built_lib):
    """Arguments that end in front of the status word are taken as before, shorter ones are not."""
    import ctypes

    from avelang_b200 import _lib
    lib = _lib.load()
    for args, call in ((_lib.LayerNormArgs, lib.ave_layer_norm), (_lib.LayerNormBwdArgs, lib.ave_layer_norm_backward)):
        assert args.status.offset + 8 == ctypes.sizeof(args)
        a = args()
        a.n, a.w_dtype = 8, 2
        for size, want in ((ctypes.sizeof(args), _lib.OK), (args.status.offset, _lib.OK), (args.status.offset - 8, _lib.INVALID_ARGUMENT), (0, _lib.INVALID_ARGUMENT)):
            a.struct_size = size
            assert call(ctypes.byref(a), None) == want  # (no rows)
    b = _lib.LayerNormBwdArgs()
    b.rows, b.n, b.d_weight = 2, 8, 0x1000
    sizes = []
    for b.struct_size in (ctypes.sizeof(b), _lib.LayerNormBwdArgs.status.offset):
        sizes.append(lib.ave_layer_norm_backward_workspace_bytes(ctypes.byref(b)))
    assert sizes[0] == sizes[1] > 0
