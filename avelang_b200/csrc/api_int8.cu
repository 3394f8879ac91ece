// extern "C" boundary of the RMS norm, of rows in 8 bits and of the product of 8-bit integers: argument validation and dispatch.  No device allocation, no
// synchronisation, nothing thrown across the boundary.
#include "common.cuh"

namespace ave {
int64_t rms_norm_max_n();
int launch_rms_norm(const AveRmsNormArgs& a, cudaStream_t stream);
size_t rms_norm_backward_workspace_bytes(const AveRmsNormBwdArgs& a);
int launch_rms_norm_backward(const AveRmsNormBwdArgs& a, cudaStream_t stream);
int launch_quantize_rows(const AveQuantRowsArgs& a, cudaStream_t stream);
int launch_dequantize_rows(const AveQuantRowsArgs& a, cudaStream_t stream);
int launch_gemm_int8_nt(const AveGemmInt8Args& a, cudaStream_t stream);

namespace {

constexpr int64_t MAX_K = 131071;  // 128 * 128 * K below 2^31
constexpr int64_t MAX_ROWS = (1ll << 31) - 1024;  // a tile's coordinates are 32-bit

bool dtype_ok(int x) { return x >= AVE_DTYPE_BF16 && x <= AVE_DTYPE_FP32; }
bool param_ok(int x, int w) { return dtype_ok(x) && (w == x || w == AVE_DTYPE_FP32); }
bool on_elem(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == AVE_DTYPE_FP32 ? 3u : 1u)) == 0; }
bool on_float(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 3u) == 0; }
// 8-bit rows: on 16 bytes, and so far apart that each has room for whole pieces (the distance of a single row says nothing)
bool int8_rows(const void* p, int64_t rows, int64_t n, int64_t stride) { return aligned16(p) && (rows <= 1 || (stride % 16 == 0 && stride >= n)); }

int validate_quant(const AveQuantRowsArgs* a) {
  if (a == nullptr || a->struct_size != sizeof(AveQuantRowsArgs) || a->rows < 0 || a->n <= 0 || !dtype_ok(a->x_dtype)) return AVE_GDN_INVALID_ARGUMENT;
  if (a->n > rms_norm_max_n()) return AVE_GDN_UNSUPPORTED;
  if (a->rows == 0) return AVE_GDN_OK;
  if (!a->x || !a->q || !a->scale) return AVE_GDN_INVALID_ARGUMENT;
  if (!on_elem(a->x, a->x_dtype) || !on_float(a->scale) || !int8_rows(a->q, a->rows, a->n, a->q_stride)) return AVE_GDN_MISALIGNED;
  return AVE_GDN_OK;
}

}  // namespace
}  // namespace ave

using namespace ave;

extern "C" {

int ave_rms_norm(const AveRmsNormArgs* a, void* stream) {
  if (a == nullptr || a->struct_size != sizeof(AveRmsNormArgs) || a->rows < 0 || a->n <= 0 || !param_ok(a->x_dtype, a->w_dtype)) return AVE_GDN_INVALID_ARGUMENT;
  if (a->n > rms_norm_max_n()) return AVE_GDN_UNSUPPORTED;
  if (a->rows == 0) return AVE_GDN_OK;
  const bool int8 = (a->flags & AVE_RMS_FLAG_INT8) != 0;
  if (!a->x || !a->y || (a->residual != nullptr) != (a->sum != nullptr) || (int8 && !a->scale)) return AVE_GDN_INVALID_ARGUMENT;
  if (!on_elem(a->x, a->x_dtype) || !on_elem(a->residual, a->x_dtype) || !on_elem(a->sum, a->x_dtype) || !on_elem(a->weight, a->w_dtype) ||
      !on_float(a->scale) || !on_float(a->rstd))
    return AVE_GDN_MISALIGNED;
  if (int8 ? !int8_rows(a->y, a->rows, a->n, a->y_stride) : !on_elem(a->y, a->x_dtype)) return AVE_GDN_MISALIGNED;
  return launch_rms_norm(*a, reinterpret_cast<cudaStream_t>(stream));
}

size_t ave_rms_norm_backward_workspace_bytes(const AveRmsNormBwdArgs* a) {
  if (a == nullptr || a->struct_size != sizeof(AveRmsNormBwdArgs) || a->rows <= 0 || a->n <= 0 || a->n > rms_norm_max_n()) return 0;
  return rms_norm_backward_workspace_bytes(*a);
}

int ave_rms_norm_backward(const AveRmsNormBwdArgs* a, void* stream) {
  if (a == nullptr || a->struct_size != sizeof(AveRmsNormBwdArgs) || a->rows < 0 || a->n <= 0 || !param_ok(a->x_dtype, a->w_dtype)) return AVE_GDN_INVALID_ARGUMENT;
  if (a->n > rms_norm_max_n()) return AVE_GDN_UNSUPPORTED;
  if (a->rows == 0) return AVE_GDN_OK;  // (a sum over no rows: the caller's)
  if (!a->d_y || !a->x || !a->rstd || !a->d_x) return AVE_GDN_INVALID_ARGUMENT;
  if (!on_elem(a->x, a->x_dtype) || !on_elem(a->d_y, a->x_dtype) || !on_elem(a->d_sum, a->x_dtype) || !on_elem(a->d_x, a->x_dtype) ||
      !on_elem(a->weight, a->w_dtype) || !on_elem(a->d_weight, a->w_dtype) || !on_float(a->rstd))
    return AVE_GDN_MISALIGNED;
  if (a->d_weight) {
    if (a->workspace == nullptr || !aligned16(a->workspace)) return AVE_GDN_INVALID_ARGUMENT;
    if (a->workspace_bytes < rms_norm_backward_workspace_bytes(*a)) return AVE_GDN_WORKSPACE_TOO_SMALL;
  }
  return launch_rms_norm_backward(*a, reinterpret_cast<cudaStream_t>(stream));
}

int ave_quantize_rows_int8(const AveQuantRowsArgs* a, void* stream) {
  const int rc = validate_quant(a);
  if (rc != AVE_GDN_OK || a->rows == 0) return rc;
  return launch_quantize_rows(*a, reinterpret_cast<cudaStream_t>(stream));
}

int ave_dequantize_rows_int8(const AveQuantRowsArgs* a, void* stream) {
  const int rc = validate_quant(a);
  if (rc != AVE_GDN_OK || a->rows == 0) return rc;
  return launch_dequantize_rows(*a, reinterpret_cast<cudaStream_t>(stream));
}

int ave_gemm_int8_nt(const AveGemmInt8Args* a, void* stream) {
  if (a == nullptr || a->struct_size != sizeof(AveGemmInt8Args) || a->M < 0 || a->N < 0 || a->K <= 0 || !param_ok(a->c_dtype, a->bias_dtype)) return AVE_GDN_INVALID_ARGUMENT;
  if (a->K > MAX_K || a->M > MAX_ROWS || a->N > MAX_ROWS) return AVE_GDN_UNSUPPORTED;
  if (a->M == 0 || a->N == 0) return AVE_GDN_OK;
  if (!a->a || !a->b || !a->c || !a->a_scale || !a->b_scale) return AVE_GDN_INVALID_ARGUMENT;
  if (a->ldc < a->N && a->M > 1) return AVE_GDN_INVALID_ARGUMENT;
  if (!int8_rows(a->a, a->M, a->K, a->lda) || !int8_rows(a->b, a->N, a->K, a->ldb) || !on_elem(a->c, a->c_dtype) || !on_elem(a->bias, a->bias_dtype) ||
      !on_float(a->a_scale) || !on_float(a->b_scale))
    return AVE_GDN_MISALIGNED;
  return launch_gemm_int8_nt(*a, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
