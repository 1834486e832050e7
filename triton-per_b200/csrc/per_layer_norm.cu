// Layer norm over rows, forward and backward.
//
// Forward, one row of D values: m = avg(x), v = avg((x - m)^2),
// r = 1 / sqrt(v + eps), h = (x - m) r, y = h w + b.
// Backward, with g = dy w: dx = r (g - avg(g) - h avg(g h)) per row, and over
// the rows dw = sum dy h, db = sum dy.
//
// Statistics are float32 sums around a first estimate of the mean: with
// s = fl(avg(x)), the sums of d = x - s and of d^2 give m = s + avg(d) and
// v = avg(d^2) - avg(d)^2. s lies within rounding of the mean, so the
// subtraction in v cancels nothing, and m is known to more than float32's
// precision; it is kept as float64 and used as a pair of float32 (s, avg(d)),
// because h loses |m| / sqrt(v) units of rounding to a mean held in float32.
#include <cuda_runtime.h>
#include <stdint.h>

#include "per_common.cuh"
#include "per_internal.h"
#include "per_types.cuh"

namespace {

constexpr int kThreads = 256;

struct Fwd {
  const void* x;
  const void* w;
  const void* b;
  void* y;
  double* mean;
  float* rstd;
  int64_t rows, x_stride, y_stride;
  int32_t dim;
  float eps;
};

struct Bwd {
  const void* dy;
  const void* x;
  const void* w;
  const double* mean;
  const float* rstd;
  void* dx;
  void* dw;
  void* db;
  float* part;  // [splits][2][dim]
  int64_t rows, dy_stride, x_stride, dx_stride;
  int32_t dim, splits;
};

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(PER_FULL_MASK, v, o);
  return v;
}

// Sums of a and b over the CTA, in a fixed order; every thread gets them.
__device__ __forceinline__ float2 block_sum2(float a, float b) {
  __shared__ float2 s[32];
  a = warp_sum(a);
  b = warp_sum(b);
  __syncthreads();  // the previous sums have been read
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = make_float2(a, b);
  __syncthreads();
  const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
  const float2 v = lane < warps ? s[lane] : make_float2(0.f, 0.f);
  return make_float2(warp_sum(v.x), warp_sum(v.y));
}

// ---- rows of any length: one CTA per row, the row read three times (from
// L2 after the first)
template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) per_layer_norm_long_kernel(const Fwd f) {
  per_wait_previous_grid();
  const float n = (float)f.dim;
  const P* w = static_cast<const P*>(f.w);
  const P* b = static_cast<const P*>(f.b);
  for (int64_t row = blockIdx.x; row < f.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(f.x) + row * f.x_stride;
    T* y = static_cast<T*>(f.y) + row * f.y_stride;
    float a = 0.f, q = 0.f;
    for (int64_t c = threadIdx.x; c < f.dim; c += kThreads) a += per_to_f32(x[c]);
    const float s = block_sum2(a, 0.f).x / n;
    a = 0.f;
    for (int64_t c = threadIdx.x; c < f.dim; c += kThreads) {
      const float d = per_to_f32(x[c]) - s;
      a += d;
      q = fmaf(d, d, q);
    }
    const float2 t = block_sum2(a, q);
    const float shift = t.x / n;
    const float r = rsqrtf(fmaxf(t.y / n - shift * shift, 0.f) + f.eps);
    for (int64_t c = threadIdx.x; c < f.dim; c += kThreads) {
      float h = (per_to_f32(x[c]) - s - shift) * r;
      if (w) h *= per_to_f32(w[c]);
      if (b) h += per_to_f32(b[c]);
      y[c] = per_from_f32<T>(h);
    }
    if (f.mean && threadIdx.x == 0) {
      f.mean[row] = (double)s + (double)shift;
      f.rstd[row] = r;
    }
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads) per_layer_norm_dx_long_kernel(const Bwd g) {
  per_wait_previous_grid();
  const float n = (float)g.dim;
  const P* w = static_cast<const P*>(g.w);
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(g.x) + row * g.x_stride;
    const T* dy = static_cast<const T*>(g.dy) + row * g.dy_stride;
    T* dx = static_cast<T*>(g.dx) + row * g.dx_stride;
    const double m = g.mean[row];
    const float hi = (float)m, lo = (float)(m - (double)hi), r = g.rstd[row];
    float a = 0.f, q = 0.f;
    for (int64_t c = threadIdx.x; c < g.dim; c += kThreads) {
      const float h = (per_to_f32(x[c]) - hi - lo) * r;
      const float gv = per_to_f32(dy[c]) * (w ? per_to_f32(w[c]) : 1.f);
      a += gv;
      q = fmaf(gv, h, q);
    }
    const float2 t = block_sum2(a, q);
    const float c1 = t.x / n, c2 = t.y / n;
    for (int64_t c = threadIdx.x; c < g.dim; c += kThreads) {
      const float h = (per_to_f32(x[c]) - hi - lo) * r;
      const float gv = per_to_f32(dy[c]) * (w ? per_to_f32(w[c]) : 1.f);
      dx[c] = per_from_f32<T>(r * (gv - c1 - h * c2));
    }
  }
}

// Column sums of one split of the rows: thread = column.
template <typename T>
__global__ void __launch_bounds__(kThreads) per_layer_norm_dw_long_kernel(const Bwd g) {
  per_wait_previous_grid();
  const int tiles = (g.dim - 1) / kThreads + 1;
  const int tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
  const int64_t c = (int64_t)tile * kThreads + threadIdx.x;
  if (c >= g.dim) return;
  const T* x = static_cast<const T*>(g.x) + c;
  const T* dy = static_cast<const T*>(g.dy) + c;
  float dw = 0.f, db = 0.f;
  for (int64_t row = split; row < g.rows; row += g.splits) {
    const double m = g.mean[row];
    const float hi = (float)m, lo = (float)(m - (double)hi), r = g.rstd[row];
    const float v = per_to_f32(dy[row * g.dy_stride]);
    dw = fmaf(v, (per_to_f32(x[row * g.x_stride]) - hi - lo) * r, dw);
    db += v;
  }
  g.part[(int64_t)split * 2 * g.dim + c] = dw;
  g.part[((int64_t)split * 2 + 1) * g.dim + c] = db;
}

// dw and db from the splits' sums, added in order.
template <typename P>
__global__ void __launch_bounds__(kThreads) per_layer_norm_join_kernel(const Bwd g) {
  per_wait_previous_grid();
  const int64_t c = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  if (c >= g.dim) return;
  float dw = 0.f, db = 0.f;
  for (int k = 0; k < g.splits; ++k) {
    dw += g.part[(int64_t)k * 2 * g.dim + c];
    db += g.part[((int64_t)k * 2 + 1) * g.dim + c];
  }
  if (g.dw) static_cast<P*>(g.dw)[c] = per_from_f32<P>(dw);
  if (g.db) static_cast<P*>(g.db)[c] = per_from_f32<P>(db);
}

int launch(const void* fn, int64_t grid, const void* arg, cudaStream_t stream) {
  void* args[] = {const_cast<void*>(arg)};
  const cudaError_t e = per_launch(fn, (unsigned)grid, kThreads, 0, stream, args, false);
  return e == cudaSuccess ? PER_OK : per_record_cuda(e);
}

int64_t row_grid(int64_t rows) { return rows < 65535 ? rows : 65535; }

// Row splits of the column sums.
int splits_of(int64_t rows, int64_t dim) {
  const int64_t tiles = (dim - 1) / kThreads + 1;
  int64_t s = 1184 / tiles;
  if (s > rows) s = rows;
  if (s > 256) s = 256;
  return s < 1 ? 1 : (int)s;
}

template <typename T, typename P>
int forward(const Fwd& f, cudaStream_t stream) {
  return launch((const void*)per_layer_norm_long_kernel<T, P>, row_grid(f.rows), &f, stream);
}

template <typename T, typename P>
int backward(const Bwd& g, cudaStream_t stream) {
  int rc = PER_OK;
  if (g.dx)
    rc = launch((const void*)per_layer_norm_dx_long_kernel<T, P>, row_grid(g.rows), &g, stream);
  if (rc || (!g.dw && !g.db)) return rc;
  const int64_t tiles = (g.dim - 1) / kThreads + 1;
  rc = launch((const void*)per_layer_norm_dw_long_kernel<T>, tiles * g.splits, &g, stream);
  if (rc) return rc;
  return launch((const void*)per_layer_norm_join_kernel<P>, tiles, &g, stream);
}

}  // namespace

// fn<T, P>(args) for the descriptor's types (checked: P is float or T)
#define PER_NORM_TYPES(n, fn, ...)                                                    \
  ((n).dtype == PER_F32    ? fn<float, float>(__VA_ARGS__)                            \
   : (n).dtype == PER_BF16 ? ((n).param_dtype == PER_F32                              \
                                  ? fn<__nv_bfloat16, float>(__VA_ARGS__)             \
                                  : fn<__nv_bfloat16, __nv_bfloat16>(__VA_ARGS__))    \
   : (n).param_dtype == PER_F32 ? fn<__half, float>(__VA_ARGS__)                      \
                                : fn<__half, __half>(__VA_ARGS__))

int per_launch_layer_norm(const per_norm_t& n, const void* x, int64_t x_stride, const void* weight,
                          const void* bias, void* y, int64_t y_stride, double* mean, float* rstd,
                          cudaStream_t stream) {
  const Fwd f{x, weight, bias, y, mean, rstd, n.rows, x_stride, y_stride, (int32_t)n.dim, n.eps};
  return PER_NORM_TYPES(n, forward, f, stream);
}

int64_t per_layer_norm_backward_bytes(const per_norm_t& n) {
  return (int64_t)splits_of(n.rows, n.dim) * 2 * n.dim * 4;
}

int per_launch_layer_norm_backward(const per_norm_t& n, const void* dy, int64_t dy_stride,
                                   const void* x, int64_t x_stride, const void* weight,
                                   const double* mean, const float* rstd, void* dx,
                                   int64_t dx_stride, void* dweight, void* dbias, void* workspace,
                                   cudaStream_t stream) {
  const Bwd g{dy, x, weight, mean, rstd, dx, dweight, dbias, static_cast<float*>(workspace),
              n.rows, dy_stride, x_stride, dx_stride, (int32_t)n.dim,
              splits_of(n.rows, n.dim)};
  return PER_NORM_TYPES(n, backward, g, stream);
}
