// extern "C" entry points of the learner's operators: argument checks.
#include <cuda_runtime.h>
#include <stdint.h>

#include "per_b200.h"
#include "per_internal.h"
#include "per_types.cuh"

namespace {

constexpr int64_t kMaxDim = (int64_t)1 << 30;

int check_norm(const per_norm_t* n) {
  if (!n) return PER_ERR_NULL_POINTER;
  if (!per_dtype_bytes(n->dtype)) return PER_ERR_INVALID_ARGUMENT;
  if (n->param_dtype != PER_F32 && n->param_dtype != n->dtype) return PER_ERR_INVALID_ARGUMENT;
  if (n->rows < 0 || n->dim < 1) return PER_ERR_INVALID_ARGUMENT;
  if (n->dim > kMaxDim || n->rows > ((int64_t)1 << 40)) return PER_ERR_TOO_LARGE;
  return PER_OK;
}

bool misaligned(const void* p, int64_t bytes) { return ((uintptr_t)p) % (uintptr_t)bytes != 0; }

// Whether [a, a + an) and [b, b + bn) share a byte.
bool overlap(const void* a, int64_t an, const void* b, int64_t bn) {
  const uintptr_t pa = (uintptr_t)a, pb = (uintptr_t)b;
  return pa < pb + (uintptr_t)bn && pb < pa + (uintptr_t)an;
}

// Bytes from the first value of the first row to the last value of the last.
int64_t span(const per_norm_t* n, int64_t stride) {
  return ((n->rows - 1) * stride + n->dim) * per_dtype_bytes(n->dtype);
}

// Rows with the same stride may interleave (columns of one packed buffer):
// they overlap only if their column ranges do.
bool rows_overlap(const per_norm_t* n, const void* a, int64_t as, const void* b, int64_t bs) {
  if (!overlap(a, span(n, as), b, span(n, bs))) return false;
  if (as != bs || as == 0) return true;
  const int64_t eb = per_dtype_bytes(n->dtype), pitch = as * eb, width = n->dim * eb;
  const int64_t d = (int64_t)((uintptr_t)b - (uintptr_t)a);
  const int64_t m = ((d % pitch) + pitch) % pitch;  // start of b's columns, seen from a's
  return m < width || m + width > pitch;
}

int check_tensors(const per_tensor_t* t, int64_t n) {
  if (n < 0) return PER_ERR_INVALID_ARGUMENT;
  if (n > 0 && !t) return PER_ERR_NULL_POINTER;
  if (n > ((int64_t)1 << 24)) return PER_ERR_TOO_LARGE;
  for (int64_t i = 0; i < n; ++i) {
    const int64_t eb = per_dtype_bytes(t[i].dtype);
    if (!eb || t[i].count < 0) return PER_ERR_INVALID_ARGUMENT;
    if (t[i].count > ((int64_t)1 << 44)) return PER_ERR_TOO_LARGE;
    if (t[i].count > 0 && !t[i].data) return PER_ERR_NULL_POINTER;
    if (misaligned(t[i].data, eb)) return PER_ERR_MISALIGNED;
  }
  return PER_OK;
}

int check_norm_call(const per_tensor_t* t, int64_t n, int32_t kind, const float* norm,
                    const void* workspace, int64_t workspace_bytes) {
  const int rc = check_tensors(t, n);
  if (rc) return rc;
  if (kind != PER_NORM_L1 && kind != PER_NORM_L2 && kind != PER_NORM_INF)
    return PER_ERR_INVALID_ARGUMENT;
  if (!norm || !workspace) return PER_ERR_NULL_POINTER;
  if (misaligned(norm, 4) || misaligned(workspace, 16)) return PER_ERR_MISALIGNED;
  if (workspace_bytes < per_grad_norm_bytes(n)) return PER_ERR_INVALID_ARGUMENT;
  return PER_OK;
}

}  // namespace

extern "C" {

int per_layer_norm(const per_norm_t* norm, const void* x, int64_t x_stride, const void* weight,
                   const void* bias, void* y, int64_t y_stride, float* stats, void* stream) {
  PerRange range("per_layer_norm");
  const int rc = check_norm(norm);
  if (rc) return rc;
  if (!(norm->eps >= 0.f)) return PER_ERR_INVALID_ARGUMENT;
  if (norm->rows == 0) return PER_OK;
  if (!x || !y) return PER_ERR_NULL_POINTER;
  if (x_stride < norm->dim || y_stride < norm->dim) return PER_ERR_INVALID_ARGUMENT;
  const int64_t eb = per_dtype_bytes(norm->dtype), pb = per_dtype_bytes(norm->param_dtype);
  if (misaligned(x, eb) || misaligned(y, eb) || misaligned(weight, pb) || misaligned(bias, pb) ||
      misaligned(stats, 16))
    return PER_ERR_MISALIGNED;
  if (rows_overlap(norm, x, x_stride, y, y_stride)) return PER_ERR_INVALID_ARGUMENT;
  return per_launch_layer_norm(*norm, x, x_stride, weight, bias, y, y_stride, stats,
                               (cudaStream_t)stream);
}

int64_t per_layer_norm_backward_workspace(const per_norm_t* norm) {
  if (check_norm(norm)) return -1;
  return per_layer_norm_backward_bytes(*norm);
}

int per_layer_norm_backward(const per_norm_t* norm, const void* dy, int64_t dy_stride,
                            const void* x, int64_t x_stride, const void* weight,
                            const float* stats, void* dx, int64_t dx_stride, void* dweight,
                            void* dbias, void* workspace, int64_t workspace_bytes, void* stream) {
  PerRange range("per_layer_norm_backward");
  const int rc = check_norm(norm);
  if (rc) return rc;
  if (!dx && !dweight && !dbias) return PER_OK;
  const int64_t eb = per_dtype_bytes(norm->dtype), pb = per_dtype_bytes(norm->param_dtype);
  if (misaligned(dweight, pb) || misaligned(dbias, pb) || misaligned(weight, pb) ||
      misaligned(dy, eb) || misaligned(x, eb) || misaligned(dx, eb) || misaligned(stats, 16) ||
       misaligned(workspace, 16))
    return PER_ERR_MISALIGNED;
  const cudaStream_t s = (cudaStream_t)stream;
  if (norm->rows == 0) {
    const size_t bytes = (size_t)(norm->dim * pb);
    for (void* p : {dweight, dbias}) {
      if (!p) continue;
      const cudaError_t e = cudaMemsetAsync(p, 0, bytes, s);
      if (e != cudaSuccess) return per_record_cuda(e);
    }
    return PER_OK;
  }
  if (!dy || !x || !stats) return PER_ERR_NULL_POINTER;
  if ((dy_stride != 0 && dy_stride < norm->dim) || x_stride < norm->dim ||
      (dx && dx_stride < norm->dim))
    return PER_ERR_INVALID_ARGUMENT;
  const int64_t need = per_layer_norm_backward_bytes(*norm);
  if (need > 0 && !workspace) return PER_ERR_NULL_POINTER;
  if (workspace_bytes < need) return PER_ERR_INVALID_ARGUMENT;
  if (dx && (rows_overlap(norm, x, x_stride, dx, dx_stride) ||
             rows_overlap(norm, dy, dy_stride, dx, dx_stride)))
    return PER_ERR_INVALID_ARGUMENT;
  return per_launch_layer_norm_backward(*norm, dy, dy_stride, x, x_stride, weight, stats, dx,
                                        dx_stride, dweight, dbias, workspace, s);
}

int64_t per_grad_norm_workspace(int64_t n) { return n < 0 ? -1 : per_grad_norm_bytes(n); }

int per_grad_norm(const per_tensor_t* tensors, int64_t n, int32_t kind, float* norm,
                  void* workspace, int64_t workspace_bytes, void* stream) {
  PerRange range("per_grad_norm");
  const int rc = check_norm_call(tensors, n, kind, norm, workspace, workspace_bytes);
  if (rc) return rc;
  return per_launch_grad_norm(tensors, n, kind, norm, workspace, (cudaStream_t)stream);
}

int per_scale_grads(const per_tensor_t* tensors, int64_t n, float max_norm, const float* norm,
                    void* stream) {
  PerRange range("per_scale_grads");
  const int rc = check_tensors(tensors, n);
  if (rc) return rc;
  if (!norm) return PER_ERR_NULL_POINTER;
  if (misaligned(norm, 4)) return PER_ERR_MISALIGNED;
  if (!(max_norm >= 0.f)) return PER_ERR_INVALID_ARGUMENT;
  return per_launch_scale_grads(tensors, n, max_norm, norm, (cudaStream_t)stream);
}

int per_clip_grad_norm(const per_tensor_t* tensors, int64_t n, int32_t kind, float max_norm,
                       float* norm, void* workspace, int64_t workspace_bytes, void* stream) {
  PerRange range("per_clip_grad_norm");
  const int rc = check_norm_call(tensors, n, kind, norm, workspace, workspace_bytes);
  if (rc) return rc;
  if (!(max_norm >= 0.f)) return PER_ERR_INVALID_ARGUMENT;
  return per_launch_clip_grad_norm(tensors, n, kind, max_norm, norm, workspace,
                                   (cudaStream_t)stream);
}

}  // extern "C"
