// The global norm of many tensors, and their scaling to at most a given norm.
//
// The tensors are cut into chunks that start on 16-byte boundaries of memory
// (the values before a tensor's first boundary go with its first chunk); each
// CTA takes an equal run of chunks and writes one partial sum in float64. The
// scaling kernel's CTAs each add all partial sums in the same fixed order, so
// no CTA waits for another and equal inputs give equal bits.
//
// Squares are summed in float32 per thread. A CTA whose sum is not finite, or
// so small that squares may have vanished below the float32 range, sums its
// values again in float64.
#include <cuda_runtime.h>
#include <stdint.h>

#include "per_common.cuh"
#include "per_internal.h"
#include "per_types.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kMaxCtas = 592;      // partial sums of one launch
constexpr int kSmallTable = 64;    // tensors of one launch: the table travels as a kernel
constexpr int kLargeTable = 1024;  // argument, of the size that the list needs

template <int N>
struct Table {
  void* data[N];
  int64_t count[N];
  uint32_t end[N];  // chunks of this and all earlier tensors
  uint8_t dtype[N];
  int32_t n;
  int32_t kind;
  int32_t chunk;        // values per chunk, a multiple of 8
  int32_t partials;     // of all launches of the call
  int32_t first_partial;
  float max_norm;
  double* part;
  float* norm;
};

template <typename T>
struct Span {  // one chunk: values [0, n) at p; [head, head + 16-byte vectors) aligned
  T* p;
  int64_t n;
  int head;
};

// Values before the first 16-byte boundary at or after p.
template <typename T>
__host__ __device__ int64_t head_of(const T* p, int64_t count) {
  const int64_t h = (int64_t)((16 - ((uintptr_t)p & 15)) & 15) / (int64_t)sizeof(T);
  return h < count ? h : count;
}

// Chunk k of a tensor: chunk 0 also holds the head.
template <typename T>
__device__ __forceinline__ Span<T> span_of(void* data, int64_t count, int64_t k, int chunk) {
  T* p = static_cast<T*>(data);
  const int64_t head = head_of(p, count);
  const int64_t lo = k == 0 ? 0 : head + k * chunk;
  const int64_t hi = head + (k + 1) * chunk;
  return Span<T>{p + lo, (hi < count ? hi : count) - lo, k == 0 ? (int)head : 0};
}

template <typename T>
union Vec {
  uint4 u;
  T t[16 / sizeof(T)];
};

// f(value) for every value of the span, by the whole CTA
template <typename T, typename F>
__device__ __forceinline__ void for_values(const Span<T>& s, F f) {
  constexpr int V = 16 / sizeof(T);
  if ((int)threadIdx.x < s.head) f(s.p[threadIdx.x]);
  const T* q = s.p + s.head;
  const int64_t nv = (s.n - s.head) / V;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < nv; i += kThreads) {
    Vec<T> v;
    v.u = reinterpret_cast<const uint4*>(q)[i];
#pragma unroll
    for (int j = 0; j < V; ++j) f(v.t[j]);
  }
  const int64_t c = nv * V + threadIdx.x;
  if (c < s.n - s.head) f(q[c]);
}

template <typename T>
__device__ __forceinline__ void scale_values(const Span<T>& s, float k) {
  constexpr int V = 16 / sizeof(T);
  if ((int)threadIdx.x < s.head)
    s.p[threadIdx.x] = per_from_f32<T>(per_to_f32(s.p[threadIdx.x]) * k);
  T* q = s.p + s.head;
  const int64_t nv = (s.n - s.head) / V;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < nv; i += kThreads) {
    Vec<T> v;
    v.u = reinterpret_cast<const uint4*>(q)[i];
#pragma unroll
    for (int j = 0; j < V; ++j) v.t[j] = per_from_f32<T>(per_to_f32(v.t[j]) * k);
    reinterpret_cast<uint4*>(q)[i] = v.u;
  }
  const int64_t c = nv * V + threadIdx.x;
  if (c < s.n - s.head) q[c] = per_from_f32<T>(per_to_f32(q[c]) * k);
}

// body(tensor, chunk of the tensor) for every chunk of this CTA's run
template <int N, typename F>
__device__ __forceinline__ void for_chunks(const Table<N>& t, F body) {
  if (t.n == 0) return;
  const uint32_t total = t.end[t.n - 1];
  const uint32_t lo = (uint32_t)((uint64_t)total * blockIdx.x / gridDim.x);
  const uint32_t hi = (uint32_t)((uint64_t)total * (blockIdx.x + 1) / gridDim.x);
  int a = 0, b = t.n - 1;  // the first tensor whose chunks reach past lo
  while (a < b) {
    const int m = (a + b) / 2;
    if (t.end[m] > lo) b = m; else a = m + 1;
  }
  for (uint32_t k = lo; k < hi; ++k) {
    while (t.end[a] <= k) ++a;
    body(a, (int64_t)(k - (a ? t.end[a - 1] : 0)));
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN wins
  return (a > b || a != a) ? a : b;
}

__device__ double block_join(double v, bool take_max) {
  __shared__ double s[kThreads / 32];
  for (int o = 16; o; o >>= 1) {
    const double u = __shfl_xor_sync(PER_FULL_MASK, v, o);
    v = take_max ? ((v > u || v != v) ? v : u) : v + u;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
  for (int k = 1; k < kThreads / 32; ++k) v = take_max ? ((v > s[k] || v != v) ? v : s[k]) : v + s[k];
  return v;
}

template <int N, typename F>
__device__ __forceinline__ void for_all(const Table<N>& t, F f) {
  for_chunks(t, [&](int a, int64_t k) {
    if (t.dtype[a] == PER_F32)
      for_values(span_of<float>(t.data[a], t.count[a], k, t.chunk), f);
    else if (t.dtype[a] == PER_BF16)
      for_values(span_of<__nv_bfloat16>(t.data[a], t.count[a], k, t.chunk), f);
    else
      for_values(span_of<__half>(t.data[a], t.count[a], k, t.chunk), f);
  });
}

template <int N, int KIND>
__global__ void __launch_bounds__(kThreads) per_norm_partial_kernel(const __grid_constant__ Table<N> t) {
  per_wait_previous_grid();
  float acc = 0.f;
  for_all(t, [&](auto v) {
    const float f = per_to_f32(v);
    if (KIND == PER_NORM_L2) acc = fmaf(f, f, acc);
    if (KIND == PER_NORM_L1) acc += fabsf(f);
    if (KIND == PER_NORM_INF) acc = max_nan(acc, fabsf(f));
  });
  double sum = block_join((double)acc, KIND == PER_NORM_INF);
  // 2^-60: a square lost below 2^-149 is under 2^-89 of such a sum
  if (KIND != PER_NORM_INF && !(sum <= 3.4e38 && sum >= 8.7e-19)) {
    double wide = 0.0;
    for_all(t, [&](auto v) {
      const double f = (double)per_to_f32(v);
      wide += KIND == PER_NORM_L2 ? f * f : fabs(f);
    });
    sum = block_join(wide, false);
  }
  if (threadIdx.x == 0) t.part[t.first_partial + blockIdx.x] = sum;
}

// The norm from all partial sums, the same bits in every thread that asks.
__device__ __forceinline__ float join_norm(const double* part, int n, int kind) {
  double v = 0.0;
  for (int k = threadIdx.x; k < n; k += kThreads) {
    const double u = part[k];
    v = kind == PER_NORM_INF ? ((v > u || v != v) ? v : u) : v + u;
  }
  v = block_join(v, kind == PER_NORM_INF);
  return (float)(kind == PER_NORM_L2 ? sqrt(v) : v);
}

__global__ void __launch_bounds__(kThreads)
    per_norm_join_kernel(const double* part, int n, int kind, float* norm) {
  per_wait_previous_grid();
  const float v = join_norm(part, n, kind);
  if (threadIdx.x == 0) *norm = v;
}

// part != NULL: the norm comes from the partial sums (and is written by the
// first launch's CTA 0), else it is read from t.norm.
template <int N>
__global__ void __launch_bounds__(kThreads) per_scale_kernel(const __grid_constant__ Table<N> t) {
  per_wait_previous_grid();
  float norm;
  if (t.part) {
    norm = join_norm(t.part, t.partials, t.kind);
    if (t.first_partial == 0 && blockIdx.x == 0 && threadIdx.x == 0) *t.norm = norm;
  } else {
    norm = *t.norm;
  }
  const float k = t.max_norm / (norm + 1e-6f);
  if (k >= 1.f) return;  // the factor is 1: nothing changes (NaN goes on)
  for_chunks(t, [&](int a, int64_t c) {
    if (t.dtype[a] == PER_F32)
      scale_values(span_of<float>(t.data[a], t.count[a], c, t.chunk), k);
    else if (t.dtype[a] == PER_BF16)
      scale_values(span_of<__nv_bfloat16>(t.data[a], t.count[a], c, t.chunk), k);
    else
      scale_values(span_of<__half>(t.data[a], t.count[a], c, t.chunk), k);
  });
}

int64_t launches_of(int64_t n) { return n <= kSmallTable ? 1 : (n - 1) / kLargeTable + 1; }

int64_t chunks_of(const per_tensor_t& t, int64_t chunk) {
  if (t.count == 0) return 0;
  const int64_t head = t.dtype == PER_F32 ? head_of(static_cast<float*>(t.data), t.count)
                                          : head_of(static_cast<__half*>(t.data), t.count);
  const int64_t body = t.count - head;
  return body <= chunk ? 1 : (body - 1) / chunk + 1;
}

// Fill the table of one launch; the grid, or -1 if the list is too large.
template <int N>
int64_t fill(Table<N>* t, const per_tensor_t* list, int64_t n) {
  int64_t total = 0;
  for (int64_t i = 0; i < n; ++i) total += list[i].count;
  int64_t chunk = 8192;
  while (total / chunk > ((int64_t)1 << 30)) chunk *= 2;
  t->chunk = (int32_t)chunk;
  int64_t end = 0;
  int k = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (list[i].count == 0) continue;
    t->data[k] = list[i].data;
    t->count[k] = list[i].count;
    t->dtype[k] = (uint8_t)list[i].dtype;
    end += chunks_of(list[i], chunk);
    if (end > 0xffffffffLL) return -1;
    t->end[k] = (uint32_t)end;
    ++k;
  }
  t->n = k;
  return end < 1 ? 1 : end < kMaxCtas ? end : kMaxCtas;
}

struct Call {
  int32_t kind;
  float max_norm;
  float* norm;
  double* part;
};

template <int N>
int partials(const per_tensor_t* list, int64_t n, const Call& c, int* first, cudaStream_t stream) {
  Table<N> t;
  const int64_t grid = fill(&t, list, n);
  if (grid < 0) return PER_ERR_TOO_LARGE;
  t.kind = c.kind;
  t.partials = 0;
  t.first_partial = *first;
  t.max_norm = 0.f;
  t.part = c.part;
  t.norm = c.norm;
  const void* fn = c.kind == PER_NORM_L2   ? (const void*)per_norm_partial_kernel<N, PER_NORM_L2>
                   : c.kind == PER_NORM_L1 ? (const void*)per_norm_partial_kernel<N, PER_NORM_L1>
                                           : (const void*)per_norm_partial_kernel<N, PER_NORM_INF>;
  void* args[] = {&t};
  const cudaError_t e = per_launch(fn, (unsigned)grid, kThreads, 0, stream, args, false);
  *first += (int)grid;
  return e == cudaSuccess ? PER_OK : per_record_cuda(e);
}

template <int N>
int scale(const per_tensor_t* list, int64_t n, const Call& c, int partial_count, int launch,
          cudaStream_t stream) {
  Table<N> t;
  const int64_t grid = fill(&t, list, n);
  if (grid < 0) return PER_ERR_TOO_LARGE;
  t.kind = c.kind;
  t.partials = partial_count;
  t.first_partial = launch;
  t.max_norm = c.max_norm;
  t.part = c.part;
  t.norm = c.norm;
  void* args[] = {&t};
  const cudaError_t e = per_launch((const void*)per_scale_kernel<N>, (unsigned)grid, kThreads, 0,
                                   stream, args, false);
  return e == cudaSuccess ? PER_OK : per_record_cuda(e);
}

int all_partials(const per_tensor_t* tensors, int64_t n, const Call& c, int* count,
                 cudaStream_t stream) {
  *count = 0;
  if (n <= kSmallTable) return partials<kSmallTable>(tensors, n, c, count, stream);
  for (int64_t i = 0; i < n; i += kLargeTable) {
    const int64_t m = n - i < kLargeTable ? n - i : kLargeTable;
    const int rc = partials<kLargeTable>(tensors + i, m, c, count, stream);
    if (rc) return rc;
  }
  return PER_OK;
}

int all_scales(const per_tensor_t* tensors, int64_t n, const Call& c, int partial_count,
               cudaStream_t stream) {
  if (n <= kSmallTable) return scale<kSmallTable>(tensors, n, c, partial_count, 0, stream);
  for (int64_t i = 0; i < n; i += kLargeTable) {
    const int64_t m = n - i < kLargeTable ? n - i : kLargeTable;
    const int rc = scale<kLargeTable>(tensors + i, m, c, partial_count, (int)(i / kLargeTable), stream);
    if (rc) return rc;
  }
  return PER_OK;
}

}  // namespace

int64_t per_grad_norm_bytes(int64_t n) {
  return launches_of(n) * kMaxCtas * (int64_t)sizeof(double);
}

int per_launch_grad_norm(const per_tensor_t* tensors, int64_t n, int32_t kind, float* norm,
                         void* workspace, cudaStream_t stream) {
  const Call c{kind, 0.f, norm, static_cast<double*>(workspace)};
  int count = 0;
  const int rc = all_partials(tensors, n, c, &count, stream);
  if (rc) return rc;
  double* part = c.part;
  void* args[] = {&part, &count, &kind, &norm};
  const cudaError_t e = per_launch((const void*)per_norm_join_kernel, 1, kThreads, 0, stream, args, false);
  return e == cudaSuccess ? PER_OK : per_record_cuda(e);
}

int per_launch_scale_grads(const per_tensor_t* tensors, int64_t n, float max_norm,
                           const float* norm, cudaStream_t stream) {
  const Call c{0, max_norm, const_cast<float*>(norm), nullptr};
  return all_scales(tensors, n, c, 0, stream);
}

int per_launch_clip_grad_norm(const per_tensor_t* tensors, int64_t n, int32_t kind, float max_norm,
                              float* norm, void* workspace, cudaStream_t stream) {
  const Call c{kind, max_norm, norm, static_cast<double*>(workspace)};
  int count = 0;
  const int rc = all_partials(tensors, n, c, &count, stream);
  if (rc) return rc;
  return all_scales(tensors, n, c, count, stream);
}
