// extern "C" boundary of linear attention with a decay for each head and of layer norm: argument validation and dispatch.  No device
// allocation, no synchronisation, nothing thrown across the boundary.
#include <stddef.h>
#include <string.h>

#include "common.cuh"

namespace ave {
int launch_linear_decode(const AveLinearArgs& a, cudaStream_t stream);
int launch_linear_prefill(const AveLinearArgs& a, cudaStream_t stream);
size_t linear_prefill_workspace_bytes(const AveLinearArgs& a);
int launch_linear_backward(const AveLinearBwdArgs& a, cudaStream_t stream);
size_t linear_backward_workspace_bytes(const AveLinearBwdArgs& a);
int64_t layer_norm_max_n();
int launch_layer_norm(const AveLayerNormArgs& a, cudaStream_t stream);
size_t layer_norm_backward_workspace_bytes(const AveLayerNormBwdArgs& a);
int launch_layer_norm_backward(const AveLayerNormBwdArgs& a, cudaStream_t stream);

namespace {

bool head_dim(int d) { return d == 64 || d == 128; }
// (The distance of a dimension's elements says nothing where it has one only.)
template <class Args>
bool rows_on16(const Args& a, const void* p, int heads, int64_t sb, int64_t st, int64_t sh) {
  return aligned16(p) && (a.B <= 1 || sb % 8 == 0) && (a.T <= 1 || st % 8 == 0) && (heads <= 1 || sh % 8 == 0);
}

template <class Args>
int validate_shape(const Args* a) {
  if (a == nullptr || a->struct_size != sizeof(Args)) return AVE_GDN_INVALID_ARGUMENT;
  if (a->B < 0 || a->T < 0 || a->n_seqs < 0 || a->Hk <= 0 || a->Hv <= 0 || a->Hv % a->Hk != 0) return AVE_GDN_INVALID_ARGUMENT;
  if (!head_dim(a->dk) || !head_dim(a->dv)) return AVE_GDN_UNSUPPORTED;
  if (a->cu_seqlens != nullptr ? a->B != 1 : a->n_seqs != a->B) return AVE_GDN_INVALID_ARGUMENT;
  return AVE_GDN_OK;
}
template <class Args>
bool nothing_to_do(const Args& a) { return (int64_t)a.B * a.T == 0 || a.n_seqs == 0; }

int validate_linear(const AveLinearArgs* a) {
  const int rc = validate_shape(a);
  if (rc != AVE_GDN_OK) return rc;
  if (a->num_slots < 0) return AVE_GDN_INVALID_ARGUMENT;
  if (a->state_indices == nullptr && (a->initial_state || a->final_state) && a->num_slots < a->n_seqs) return AVE_GDN_INVALID_ARGUMENT;
  if (nothing_to_do(*a)) return AVE_GDN_OK;
  if (!a->q || !a->k || !a->v || !a->o) return AVE_GDN_INVALID_ARGUMENT;
  if (!rows_on16(*a, a->q, a->Hk, a->q_stride_b, a->q_stride_t, a->q_stride_h) || !rows_on16(*a, a->k, a->Hk, a->k_stride_b, a->k_stride_t, a->k_stride_h) ||
      !rows_on16(*a, a->v, a->Hv, a->v_stride_b, a->v_stride_t, a->v_stride_h) || !rows_on16(*a, a->o, a->Hv, a->o_stride_b, a->o_stride_t, a->o_stride_h))
    return AVE_GDN_MISALIGNED;
  if (!aligned16(a->initial_state) || !aligned16(a->final_state) || (reinterpret_cast<uintptr_t>(a->g) & 3u)) return AVE_GDN_MISALIGNED;
  return AVE_GDN_OK;
}

int validate_linear_bwd(const AveLinearBwdArgs* a) {
  const int rc = validate_shape(a);
  if (rc != AVE_GDN_OK) return rc;
  if (nothing_to_do(*a)) return AVE_GDN_OK;
  if (!a->q || !a->k || !a->v || !a->d_o || !a->d_q || !a->d_k || !a->d_v || (a->g && !a->d_g) || (a->initial_state && !a->d_initial_state)) return AVE_GDN_INVALID_ARGUMENT;
  if ((a->flags & AVE_LINEAR_FLAG_HEAD_GATE) && (a->g_stride_b != 0 || a->g_stride_t != 0)) return AVE_GDN_INVALID_ARGUMENT;
  if (!rows_on16(*a, a->q, a->Hk, a->q_stride_b, a->q_stride_t, a->q_stride_h) || !rows_on16(*a, a->k, a->Hk, a->k_stride_b, a->k_stride_t, a->k_stride_h) ||
      !rows_on16(*a, a->v, a->Hv, a->v_stride_b, a->v_stride_t, a->v_stride_h) || !rows_on16(*a, a->d_o, a->Hv, a->do_stride_b, a->do_stride_t, a->do_stride_h))
    return AVE_GDN_MISALIGNED;
  if (!aligned16(a->d_q) || !aligned16(a->d_k) || !aligned16(a->d_v) || !aligned16(a->initial_state) || !aligned16(a->d_final_state) || !aligned16(a->d_initial_state) ||
      ((reinterpret_cast<uintptr_t>(a->g) | reinterpret_cast<uintptr_t>(a->d_g)) & 3u))
    return AVE_GDN_MISALIGNED;
  return AVE_GDN_OK;
}

bool dtype_ok(int x, int w) { return x >= AVE_DTYPE_BF16 && x <= AVE_DTYPE_FP32 && (w == x || w == AVE_DTYPE_FP32); }
// Arguments whose status word, the last field, may be missing
template <class Args>
const Args* with_status(const Args* a, Args& own) {
  if (a == nullptr || a->struct_size == sizeof(Args)) return a;
  if (a->struct_size != offsetof(Args, status)) return nullptr;
  own = Args{};
  memcpy(&own, a, offsetof(Args, status));
  return &own;
}
bool on_elem(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == AVE_DTYPE_FP32 ? 3u : 1u)) == 0; }

}  // namespace
}  // namespace ave

using namespace ave;

extern "C" {

size_t ave_linear_prefill_workspace_bytes(const AveLinearArgs* a) {
  if (validate_linear(a) != AVE_GDN_OK || nothing_to_do(*a)) return 0;
  return linear_prefill_workspace_bytes(*a);
}

int ave_linear_chunk_prefill(const AveLinearArgs* a, void* stream) {
  const int rc = validate_linear(a);
  if (rc != AVE_GDN_OK) return rc;
  if (nothing_to_do(*a)) return AVE_GDN_OK;
  const size_t need = linear_prefill_workspace_bytes(*a);
  if (need > 0 && (a->workspace == nullptr || !aligned16(a->workspace))) return AVE_GDN_INVALID_ARGUMENT;
  if (a->workspace_bytes < need) return AVE_GDN_WORKSPACE_TOO_SMALL;
  return launch_linear_prefill(*a, reinterpret_cast<cudaStream_t>(stream));
}

int ave_linear_decode_step(const AveLinearArgs* a, void* stream) {
  const int rc = validate_linear(a);
  if (rc != AVE_GDN_OK) return rc;
  if (nothing_to_do(*a)) return AVE_GDN_OK;
  return launch_linear_decode(*a, reinterpret_cast<cudaStream_t>(stream));
}

size_t ave_linear_backward_workspace_bytes(const AveLinearBwdArgs* a) {
  if (validate_linear_bwd(a) != AVE_GDN_OK || nothing_to_do(*a)) return 0;
  return linear_backward_workspace_bytes(*a);
}

int ave_linear_backward(const AveLinearBwdArgs* a, void* stream) {
  const int rc = validate_linear_bwd(a);
  if (rc != AVE_GDN_OK) return rc;
  if (nothing_to_do(*a)) return AVE_GDN_OK;
  const size_t need = linear_backward_workspace_bytes(*a);
  if (need > 0 && (a->workspace == nullptr || !aligned16(a->workspace))) return AVE_GDN_INVALID_ARGUMENT;
  if (a->workspace_bytes < need) return AVE_GDN_WORKSPACE_TOO_SMALL;
  return launch_linear_backward(*a, reinterpret_cast<cudaStream_t>(stream));
}

int ave_layer_norm(const AveLayerNormArgs* args, void* stream) {
  AveLayerNormArgs own;
  const AveLayerNormArgs* a = with_status(args, own);
  if (a == nullptr || a->rows < 0 || a->n <= 0 || !dtype_ok(a->x_dtype, a->w_dtype)) return AVE_GDN_INVALID_ARGUMENT;
  if (a->n > layer_norm_max_n()) return AVE_GDN_UNSUPPORTED;
  if (a->rows == 0) return AVE_GDN_OK;
  if (!a->x || !a->y || (a->bias && !a->weight)) return AVE_GDN_INVALID_ARGUMENT;
  if (!on_elem(a->x, a->x_dtype) || !on_elem(a->y, a->x_dtype) || !on_elem(a->weight, a->w_dtype) || !on_elem(a->bias, a->w_dtype)) return AVE_GDN_MISALIGNED;
  return launch_layer_norm(*a, reinterpret_cast<cudaStream_t>(stream));
}

size_t ave_layer_norm_backward_workspace_bytes(const AveLayerNormBwdArgs* args) {
  AveLayerNormBwdArgs own;
  const AveLayerNormBwdArgs* a = with_status(args, own);
  if (a == nullptr || a->rows <= 0 || a->n <= 0 || a->n > layer_norm_max_n()) return 0;
  return layer_norm_backward_workspace_bytes(*a);
}

int ave_layer_norm_backward(const AveLayerNormBwdArgs* args, void* stream) {
  AveLayerNormBwdArgs own;
  const AveLayerNormBwdArgs* a = with_status(args, own);
  if (a == nullptr || a->rows < 0 || a->n <= 0 || !dtype_ok(a->x_dtype, a->w_dtype)) return AVE_GDN_INVALID_ARGUMENT;
  if (a->n > layer_norm_max_n()) return AVE_GDN_UNSUPPORTED;
  if (a->rows == 0) return AVE_GDN_OK;  // (sums over no rows: the caller's)
  if (!a->d_y || !a->x || !a->mean || !a->rstd || !a->d_x) return AVE_GDN_INVALID_ARGUMENT;
  if (!on_elem(a->x, a->x_dtype) || !on_elem(a->d_y, a->x_dtype) || !on_elem(a->d_x, a->x_dtype) || !on_elem(a->weight, a->w_dtype) ||
      !on_elem(a->d_weight, a->w_dtype) || !on_elem(a->d_bias, a->w_dtype))
    return AVE_GDN_MISALIGNED;
  if (a->d_weight || a->d_bias) {
    if (a->workspace == nullptr || !aligned16(a->workspace)) return AVE_GDN_INVALID_ARGUMENT;
    if (a->workspace_bytes < layer_norm_backward_workspace_bytes(*a)) return AVE_GDN_WORKSPACE_TOO_SMALL;
  }
  return launch_layer_norm_backward(*a, reinterpret_cast<cudaStream_t>(stream));
}

}  // extern "C"
