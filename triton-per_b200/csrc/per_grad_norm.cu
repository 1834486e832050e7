// The global norm of many tensors, and their scaling to at most a given norm.
//
// N = sqrt(sum g^2) over every value of every tensor (or sum |g|, or max |g|),
// then g <- g min(1, max_norm / (N + 1e-6)): all values are read for the norm,
// and read and written again where the factor is below 1.
//
// The 16-byte vectors of the tensors' memory are cut into blocks of one vector
// per thread, and each CTA takes an equal run of blocks, with several blocks
// in flight whether they belong to one tensor or to many. The values outside
// whole vectors (up to 7 before the first 16-byte boundary of a tensor and up
// to 7 behind the last) are shared out over all threads of the launch. The
// host finds where each run begins, and the list travels with the launch as
// its argument, so no copy precedes it and nothing has to outlive it.
//
// First kernel: each CTA writes the sum of its run as one float64. Second
// kernel: every CTA adds all those sums in the same order, so no CTA waits for
// another (no counters to reset, nothing shared between calls but the
// workspace), and scales its run, last block first, because what the first
// kernel read last is what the L2 cache still holds. Under a programmatic
// launch the second kernel starts while the first one runs and fetches the
// values that it will scale first before it waits for the sums. A list of up
// to a megabyte goes through one kernel instead: a cluster of CTAs that keeps
// all values in registers between the norm and the scaling.
//
// Squares are summed in float32, in 16 sums per thread, and in float64 from
// there. A CTA whose sum is not finite, or so small that squares may have
// vanished below the float32 range, sums its run again in float64.
//
// DRAM bounds large lists (1.02 GB of bfloat16: 147 us for the norm, 7.0 TB/s
// read only, 498 us with the scaling, which the 469 us of its three passes at
// the copy rate bound from below), L2 and the chain of loads and sums the
// middle (155 MB of float32: norm 26.5 us; 11.4 MB in 100 tensors: 10 us), the
// launches and the exchange short ones (0.6 MB: 3.8 us in the one kernel, 4.9
// us in two).
#include <cuda_runtime.h>
#include <stdint.h>

#include "per_common.cuh"
#include "per_internal.h"
#include "per_types.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kMaxCtas = 296;   // of one launch: two per SM
constexpr int kUnroll = 8;      // vectors that a thread has in flight
constexpr int kCluster = 16;    // CTAs of the one-kernel form
constexpr int kHeld = 8;        // vectors that a thread keeps there
constexpr int kLoose = 16;      // threads per tensor for the values outside vectors

struct Entry {
  char* data;
  uint64_t count;  // values, and the type in the upper 8 bits
};

struct Start {  // where a run begins: block of a tensor of the list
  uint32_t block;
  uint32_t tensor;
};

// One launch's list: N tensors, runs of up to G CTAs. Three sizes, because a
// launch costs more with a larger argument.
template <int N, int G>
struct Table {
  static constexpr int kTensors = N, kCtas = G;
  Entry e[N];
  Start run[G + 1];  // the last one is the end of the list
  int32_t n;
  int32_t kind;
  int32_t partials;  // of all launches of the call
  int32_t first_partial;
  float max_norm;
  double* part;
  float* norm;
};
using Small = Table<64, kMaxCtas>;
using Medium = Table<256, kMaxCtas>;
using Large = Table<1536, kMaxCtas>;
static_assert(sizeof(Large) < 32000, "fits the arguments of a launch");

// A tensor as the kernels see it: `head` values, then whole vectors, then the
// rest.
struct View {
  char* data;
  int64_t count, vectors;
  int log2_bytes, dtype, head;
  __host__ __device__ __forceinline__ View(const Entry& e) {
    data = e.data;
    dtype = (int)(e.count >> 56);
    count = (int64_t)(e.count & ((1ull << 56) - 1));
    log2_bytes = dtype == PER_F32 ? 2 : 1;
    const int h = (16 - (int)((uintptr_t)data & 15)) & 15;
    head = (int)(h >> log2_bytes < count ? h >> log2_bytes : count);
    vectors = (count - head) >> (4 - log2_bytes);
  }
  __host__ __device__ __forceinline__ uint32_t blocks() const {
    return (uint32_t)((uint64_t)(vectors + kThreads - 1) / kThreads);
  }
  // value k of the (at most 14) values outside the vectors: 0 .. 6 lead, 8 .. 14 trail
  __device__ __forceinline__ char* loose(int k) const {
    const int64_t c = k < 8 ? k : head + (vectors << (4 - log2_bytes)) + (k - 8);
    return c < (k < 8 ? (int64_t)head : count) ? data + (c << log2_bytes) : nullptr;
  }
};

// f(T{}) with the type of a tensor
template <typename F>
__device__ __forceinline__ void with_type(int dtype, F f) {
  if (dtype == PER_F32)
    f(float{});
  else if (dtype == PER_BF16)
    f(__nv_bfloat16{});
  else
    f(__half{});
}

// The blocks of a CTA's run, in order (STEP 1) or from the last to the first
// (STEP -1).
template <typename TB, int STEP>
struct Walk {
  const TB& t;
  Start lo, hi;
  uint32_t tensor;       // current one
  int64_t at, end;       // next block there; the first one past this walk's share of it
  uint4* v;
  int64_t vectors;
  int dtype;
  bool more;

  __device__ __forceinline__ explicit Walk(const TB& table)
      : t(table), lo(table.run[blockIdx.x]), hi(table.run[blockIdx.x + 1]) {
    more = lo.tensor < hi.tensor || lo.block < hi.block;
    if (!more) return;
    tensor = STEP > 0 ? lo.tensor : hi.block > 0 ? hi.tensor : hi.tensor - 1;
    enter();
    skip();
  }
  __device__ __forceinline__ void enter() {
    const View e(t.e[tensor]);
    v = reinterpret_cast<uint4*>(e.data + (e.head << e.log2_bytes));
    vectors = e.vectors;
    dtype = e.dtype;
    const int64_t first = tensor == lo.tensor ? lo.block : 0;
    const int64_t last = tensor == hi.tensor ? hi.block : e.blocks();
    at = STEP > 0 ? first : last - 1;
    end = STEP > 0 ? last : first - 1;
  }
  // on to a tensor with blocks left
  __device__ __forceinline__ void skip() {
    while (at == end) {
      const bool was_last = STEP > 0 ? tensor + 1 > hi.tensor || (tensor + 1 == hi.tensor && hi.block == 0)
                                     : tensor == lo.tensor;
      if (was_last) {
        more = false;
        return;
      }
      tensor = STEP > 0 ? tensor + 1 : tensor - 1;
      enter();
    }
  }
  __device__ __forceinline__ int64_t left() const { return more ? (end - at) * STEP : 0; }
  // this thread's vector of the block, or NULL
  __device__ __forceinline__ uint4* vector(int64_t block) const {
    const int64_t i = block * kThreads + threadIdx.x;
    return i < vectors ? v + i : nullptr;
  }
  __device__ __forceinline__ void next() {
    at += STEP;
    skip();
  }
};

// The next K vectors of a walk (zeros where there is none). Their places and
// types are not kept: the same steps from the same point find them again.
template <int K, typename W>
__device__ __forceinline__ void fetch(W w, uint4 (&u)[K]) {
#pragma unroll
  for (int j = 0; j < K; ++j) {
    u[j] = make_uint4(0, 0, 0, 0);
    if (w.more) {
      if (const uint4* p = w.vector(w.at)) u[j] = __ldcg(p);
      w.next();
    }
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN wins
  return (a > b || a != a) ? a : b;
}

// 16 sums per thread of one kind
template <int KIND>
struct Sums {
  float2 s[8];
  __device__ __forceinline__ Sums() {
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = per_both(0.f);
  }
  __device__ __forceinline__ void add(float2& a, float2 v) {
    if (KIND == PER_NORM_L2) a = per_fma2(v, v, a);
    if (KIND == PER_NORM_L1) a = per_add2(a, make_float2(fabsf(v.x), fabsf(v.y)));
    if (KIND == PER_NORM_INF) a = make_float2(max_nan(a.x, fabsf(v.x)), max_nan(a.y, fabsf(v.y)));
  }
  template <typename T>
  __device__ __forceinline__ void add(uint4 u, int turn) {
    constexpr int P = 8 / (int)sizeof(T);  // pairs of a vector
#pragma unroll
    for (int i = 0; i < P; ++i) add(s[(turn * P + i) % 8], per_pair_of<T>(u, i));
  }
  template <typename T>
  __device__ __forceinline__ void add(T v) {
    add(s[0], make_float2(per_to_f32(v), 0.f));
  }
  __device__ __forceinline__ double total() const {
    if (KIND == PER_NORM_INF) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = max_nan(m, max_nan(s[i].x, s[i].y));
      return (double)m;
    }
    double t = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) t += (double)s[i].x + (double)s[i].y;
    return t;
  }
};

// the same in float64, for values whose squares leave float32
template <int KIND>
struct WideSum {
  double s = 0.0;
  template <typename T>
  __device__ __forceinline__ void add(T v) {
    const double f = (double)per_to_f32(v);
    s += KIND == PER_NORM_L2 ? f * f : fabs(f);
  }
  template <typename T>
  __device__ __forceinline__ void add(uint4 u, int) {
#pragma unroll
    for (int i = 0; i < 8 / (int)sizeof(T); ++i) {
      const float2 f = per_pair_of<T>(u, i);
      add(f.x);
      add(f.y);
    }
  }
};

__device__ __forceinline__ bool leaves_float32(double sum, int kind) {
  // 2^-60: a square lost below 2^-149 is under 2^-89 of such a sum
  return kind != PER_NORM_INF && !(sum <= 3.4e38 && sum >= 8.7e-19);
}

// f(address, type) for every loose value that is this thread's
template <typename TB, typename F>
__device__ __forceinline__ void for_loose(const TB& t, F f) {
  const int all = (int)gridDim.x * kThreads;
  for (int i = (int)(blockIdx.x * kThreads + threadIdx.x); i < t.n * kLoose; i += all) {
    const View e(t.e[i / kLoose]);
    if (char* p = e.loose(i % kLoose)) f(p, e.dtype);
  }
}

template <int K, typename W, typename S>
__device__ __forceinline__ void sum_fetched(W& w, const uint4 (&u)[K], S& acc) {
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (w.more) {
      with_type(w.dtype, [&](auto z) { acc.template add<decltype(z)>(u[j], j); });
      w.next();
    }
}

// A CTA's run into `acc`. The walk over it is the caller's, who can have found
// its way through the list before there is anything to read.
template <typename TB, typename S>
__device__ __forceinline__ void sum_run(const TB& t, Walk<TB, 1> w, S& acc) {
  for_loose(t, [&](char* p, int dtype) {
    with_type(dtype, [&](auto z) { acc.add(*reinterpret_cast<const decltype(z)*>(p)); });
  });
  while (w.more) {
    if (w.left() >= kUnroll) {  // blocks of one tensor
      const int64_t blocks = w.left() / kUnroll * kUnroll;
      with_type(w.dtype, [&](auto z) {
        using T = decltype(z);
        for (int64_t b = w.at; b < w.at + blocks; b += kUnroll) {
          const uint4* p = w.v + b * kThreads + threadIdx.x;
          const int64_t room = w.vectors - b * kThreads - threadIdx.x;
          uint4 u[kUnroll];
#pragma unroll
          for (int j = 0; j < kUnroll - 1; ++j) u[j] = p[j * kThreads];
          u[kUnroll - 1] = room > (kUnroll - 1) * kThreads ? p[(kUnroll - 1) * kThreads]
                                                          : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (int j = 0; j < kUnroll; ++j) acc.template add<T>(u[j], j);
        }
      });
      w.at += blocks;
      w.skip();
    } else {
      uint4 u[kUnroll];
      fetch(w, u);
      sum_fetched(w, u, acc);
    }
  }
}

__device__ __forceinline__ double join2(double a, double b, bool take_max) {
  return take_max ? ((a > b || a != a) ? a : b) : a + b;
}

// v of all threads joined in a fixed order; every thread gets the result
__device__ __forceinline__ double block_join(double v, bool take_max) {
  __shared__ double s[kThreads / 32];
#pragma unroll
  for (int o = 16; o; o >>= 1) v = join2(v, __shfl_xor_sync(PER_FULL_MASK, v, o), take_max);
  __syncthreads();  // an earlier join has been read
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int k = 1; k < kThreads / 32; ++k) v = join2(v, s[k], take_max);
  return v;
}

template <typename TB, int KIND>
__global__ void __launch_bounds__(kThreads, 2)
    per_norm_partial_kernel(const __grid_constant__ TB t) {
  const Walk<TB, 1> w(t);
  per_wait_previous_grid();
  Sums<KIND> acc;
  sum_run(t, w, acc);
  double sum = block_join(acc.total(), KIND == PER_NORM_INF);
  if (leaves_float32(sum, KIND)) {
    WideSum<KIND> wide;
    sum_run(t, Walk<TB, 1>(t), wide);
    sum = block_join(wide.s, false);
  }
  if (threadIdx.x == 0) t.part[t.first_partial + blockIdx.x] = sum;
}

// The norm from all partial sums, the same bits in every thread that asks.
__device__ __forceinline__ float root(double v, int kind) {
  return (float)(kind == PER_NORM_L2 ? sqrt(v) : v);
}
__device__ __forceinline__ float join_norm(const double* part, int n, int kind) {
  double v = 0.0;
  for (int k = threadIdx.x; k < n; k += kThreads)
    v = join2(v, __ldcg(part + k), kind == PER_NORM_INF);
  return root(block_join(v, kind == PER_NORM_INF), kind);
}

__global__ void __launch_bounds__(kThreads)
    per_norm_join_kernel(const double* part, int n, int kind, float* norm) {
  per_wait_previous_grid();
  const float v = join_norm(part, n, kind);
  if (threadIdx.x == 0) *norm = v;
}

template <typename T>
__device__ __forceinline__ uint4 scaled(uint4 u, float k) {
#pragma unroll
  for (int i = 0; i < 8 / (int)sizeof(T); ++i)
    per_set_pair<T>(u, i, per_mul2(per_pair_of<T>(u, i), per_both(k)));
  return u;
}

template <int K, typename W>
__device__ __forceinline__ void scale_fetched(W& w, const uint4 (&u)[K], float k) {
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (w.more) {
      if (uint4* p = w.vector(w.at))
        with_type(w.dtype, [&](auto z) { *p = scaled<decltype(z)>(u[j], k); });
      w.next();
    }
}

template <typename TB>
__device__ __forceinline__ void scale_loose(const TB& t, float k) {
  for_loose(t, [&](char* p, int dtype) {
    with_type(dtype, [&](auto z) {
      using T = decltype(z);
      T* q = reinterpret_cast<T*>(p);
      *q = per_from_f32<T>(per_to_f32(*q) * k);
    });
  });
}

// The factor, as torch.nn.utils.clip_grad_norm_ has it. 1 or above: nothing
// changes. NaN goes on.
__device__ __forceinline__ float factor(float max_norm, float norm) {
  return max_norm / (norm + 1e-6f);
}

// t.part: the norm comes from the partial sums (and the first launch's CTA 0
// writes it), else it is read from t.norm.
template <typename TB>
__global__ void __launch_bounds__(kThreads, 2) per_scale_kernel(const __grid_constant__ TB t) {
  uint4 u[kUnroll];
  // Nothing that runs beside this kernel writes the tensors: the kernel before
  // it in the stream is one of this call's, which lets this one start once it
  // has itself waited for all that came before.
  if (t.part) fetch(Walk<TB, -1>(t), u);
  per_wait_previous_grid();
  float norm;
  if (t.part) {
    norm = join_norm(t.part, t.partials, t.kind);
    if (t.first_partial == 0 && blockIdx.x == 0 && threadIdx.x == 0) *t.norm = norm;
  } else {
    norm = *t.norm;
  }
  const float k = factor(t.max_norm, norm);
  if (k >= 1.f) return;
  scale_loose(t, k);
  Walk<TB, -1> w(t);
  if (t.part) scale_fetched(w, u, k);
  while (w.more) {
    if (w.left() >= kUnroll) {
      const int64_t blocks = w.left() / kUnroll * kUnroll;
      with_type(w.dtype, [&](auto z) {
        using T = decltype(z);
        for (int64_t c = w.at; c > w.at - blocks; c -= kUnroll) {
          // blocks c - kUnroll + 1 .. c, of which only the last may be ragged
          uint4* p = w.v + (c - kUnroll + 1) * kThreads + threadIdx.x;
          const bool whole = w.vectors - c * kThreads > threadIdx.x;
#pragma unroll
          for (int j = 0; j < kUnroll; ++j)
            if (j < kUnroll - 1 || whole) u[j] = p[j * kThreads];
#pragma unroll
          for (int j = 0; j < kUnroll; ++j)
            if (j < kUnroll - 1 || whole) p[j * kThreads] = scaled<T>(u[j], k);
        }
      });
      w.at -= blocks;
      w.skip();
    } else {
      fetch(w, u);
      scale_fetched(w, u, k);
    }
  }
}

// The one-kernel form, for a short list of one type: one cluster, whose threads
// keep their vectors and loose values from the norm to the scaling. The host
// lists the blocks one by one (block b goes to CTA b mod kCluster), so every
// load of a thread can be issued at once.
struct Block {
  uint4* p;
  uint64_t n;  // vectors, up to kThreads
};
struct Short {
  static constexpr int kTensors = 64;
  Block b[kHeld * kCluster];
  Entry e[kTensors];
  int32_t n;
  float max_norm;  // < 0: only the norm is wanted
  float* norm;
};
static_assert(Short::kTensors * kLoose <= kCluster * kThreads, "one loose value per thread");

template <typename T, int KIND>
__global__ void __launch_bounds__(kThreads, 1) per_clip_short_kernel(const __grid_constant__ Short t) {
  __shared__ double sums[kCluster];
  // before a CTA writes into another one's shared memory, that one has to run
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  per_wait_previous_grid();
  uint4 u[kHeld];
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const Block& b = t.b[j * kCluster + blockIdx.x];
    u[j] = threadIdx.x < b.n ? __ldcg(b.p + threadIdx.x) : make_uint4(0, 0, 0, 0);
  }
  T* loose = nullptr;
  for_loose(t, [&](char* q, int) { loose = reinterpret_cast<T*>(q); });
  Sums<KIND> acc;
  if (loose) acc.add(*loose);
#pragma unroll
  for (int j = 0; j < kHeld; ++j) acc.template add<T>(u[j], j);
  double sum = block_join(acc.total(), KIND == PER_NORM_INF);
  if (leaves_float32(sum, KIND)) {
#pragma unroll
    for (int j = 0; j < kHeld; ++j)
      asm volatile("" : "+r"(u[j].x), "+r"(u[j].y), "+r"(u[j].z), "+r"(u[j].w));
    WideSum<KIND> wide;
    if (loose) wide.add(*loose);
#pragma unroll
    for (int j = 0; j < kHeld; ++j) wide.template add<T>(u[j], j);
    sum = block_join(wide.s, false);
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (threadIdx.x < kCluster) {
    const uint32_t local = (uint32_t)__cvta_generic_to_shared(&sums[blockIdx.x]);
    uint32_t remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(threadIdx.x));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(remote), "d"(sum) : "memory");
  }
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  double v = sums[0];
#pragma unroll
  for (int c = 1; c < kCluster; ++c) v = join2(v, sums[c], KIND == PER_NORM_INF);
  const float norm = root(v, KIND);
  if (blockIdx.x == 0 && threadIdx.x == 0) *t.norm = norm;
  if (t.max_norm < 0.f) return;
  const float k = factor(t.max_norm, norm);
  if (k >= 1.f) return;
#pragma unroll
  for (int j = 0; j < kHeld; ++j)  // held packed, not as the sums unpacked them
    asm volatile("" : "+r"(u[j].x), "+r"(u[j].y), "+r"(u[j].z), "+r"(u[j].w));
#pragma unroll
  for (int j = 0; j < kHeld; ++j) {
    const Block& b = t.b[j * kCluster + blockIdx.x];
    if (threadIdx.x < b.n) b.p[threadIdx.x] = scaled<T>(u[j], k);
  }
  if (loose) *loose = per_from_f32<T>(per_to_f32(*loose) * k);
}

// ---- host side

// Tensors of the list from `at` on that one launch takes.
int64_t batch_of(int64_t left) { return left < Large::kTensors ? left : Large::kTensors; }

// Fill the table of one launch for up to `most` CTAs; its grid (0: nothing to
// do, -1: too large).
template <typename TB>
int64_t fill(TB* t, const per_tensor_t* list, int64_t n, int64_t most) {
  int64_t blocks = 0;
  int k = 0;
  uint32_t per[TB::kTensors];
  for (int64_t i = 0; i < n; ++i) {
    if (list[i].count == 0) continue;
    t->e[k].data = static_cast<char*>(list[i].data);
    t->e[k].count = (uint64_t)list[i].count | ((uint64_t)list[i].dtype << 56);
    per[k] = View(t->e[k]).blocks();
    blocks += per[k++];
  }
  t->n = k;
  if (blocks > 0x7fffffff) return -1;
  if (k == 0) return 0;
  const int64_t grid = blocks < 1 ? 1 : blocks < most ? blocks : most;
  int64_t done = 0;  // blocks before tensor a
  int a = 0;
  for (int64_t c = 0; c <= grid; ++c) {
    const int64_t at = blocks * c / grid;
    while (a < k && done + per[a] <= at) done += per[a++];
    t->run[c].tensor = (uint32_t)a;
    t->run[c].block = (uint32_t)(at - done);
  }
  return grid;
}

struct Call {
  int32_t kind;
  float max_norm;
  float* norm;
  double* part;
};

template <typename TB>
void set_call(TB* t, const Call& c, int partials, int first) {
  t->kind = c.kind;
  t->partials = partials;
  t->first_partial = first;
  t->max_norm = c.max_norm;
  t->part = c.part;
  t->norm = c.norm;
}

int go(const void* fn, int64_t grid, void* table, cudaStream_t stream) {
  void* args[] = {table};
  const cudaError_t e = per_launch(fn, (unsigned)grid, kThreads, 0, stream, args, false);
  return e == cudaSuccess ? PER_OK : per_record_cuda(e);
}

template <typename TB>
int run_partials(TB* t, int64_t grid, const Call& c, int first, cudaStream_t stream) {
  set_call(t, c, 0, first);
  const void* fn = c.kind == PER_NORM_L2   ? (const void*)per_norm_partial_kernel<TB, PER_NORM_L2>
                   : c.kind == PER_NORM_L1 ? (const void*)per_norm_partial_kernel<TB, PER_NORM_L1>
                                           : (const void*)per_norm_partial_kernel<TB, PER_NORM_INF>;
  return go(fn, grid, t, stream);
}

int join(const Call& c, int count, cudaStream_t stream) {
  const double* part = c.part;
  int32_t kind = c.kind;
  float* norm = c.norm;
  void* args[] = {&part, &count, &kind, &norm};
  const cudaError_t e =
      per_launch((const void*)per_norm_join_kernel, 1, kThreads, 0, stream, args, false);
  return e == cudaSuccess ? PER_OK : per_record_cuda(e);
}

// partials: the norm is to be computed; scaling: the tensors are to be scaled.
// A list that one launch takes fills its table once for both kernels.
template <typename TB>
int one_table(TB* t, const per_tensor_t* list, int64_t n, const Call& c, bool partials, bool scaling,
              cudaStream_t stream) {
  const int64_t grid = fill(t, list, n, TB::kCtas);
  if (grid < 0) return PER_ERR_TOO_LARGE;
  int rc = PER_OK;
  if (partials && grid > 0) rc = run_partials(t, grid, c, 0, stream);
  if (rc) return rc;
  if (!scaling || grid == 0) return partials ? join(c, (int)grid, stream) : PER_OK;
  set_call(t, c, (int)grid, 0);
  return go((const void*)per_scale_kernel<TB>, grid, t, stream);
}

template <typename T>
const void* short_kernel(int32_t kind) {
  return kind == PER_NORM_L2   ? (const void*)per_clip_short_kernel<T, PER_NORM_L2>
         : kind == PER_NORM_L1 ? (const void*)per_clip_short_kernel<T, PER_NORM_L1>
                               : (const void*)per_clip_short_kernel<T, PER_NORM_INF>;
}

// One kernel for up to a megabyte of one type; false where the list is another.
bool one_kernel(const per_tensor_t* list, int64_t n, const Call& c, bool scaling,
                cudaStream_t stream, int* rc) {
  if (n < 1 || n > Short::kTensors) return false;
  Short t;
  t.n = 0;
  int blocks = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (list[i].dtype != list[0].dtype) return false;
    if (list[i].count == 0) continue;
    Entry& e = t.e[t.n++];
    e.data = static_cast<char*>(list[i].data);
    e.count = (uint64_t)list[i].count | ((uint64_t)list[i].dtype << 56);
    const View v(e);
    if (v.vectors > (int64_t)(kHeld * kCluster - blocks) * kThreads) return false;
    uint4* p = reinterpret_cast<uint4*>(v.data + (v.head << v.log2_bytes));
    for (int64_t left = v.vectors; left > 0; left -= kThreads, p += kThreads)
      t.b[blocks++] = Block{p, (uint64_t)(left < kThreads ? left : kThreads)};
  }
  if (t.n == 0) return false;
  for (; blocks < kHeld * kCluster; ++blocks) t.b[blocks] = Block{nullptr, 0};
  t.max_norm = scaling ? c.max_norm : -1.f;
  t.norm = c.norm;
  const int32_t dtype = list[0].dtype;
  const void* fn = dtype == PER_F32    ? short_kernel<float>(c.kind)
                   : dtype == PER_BF16 ? short_kernel<__nv_bfloat16>(c.kind)
                                       : short_kernel<__half>(c.kind);
  if (!per_cluster_fits(fn, kThreads, 0, kCluster)) return false;
  void* args[] = {&t};
  const cudaError_t e = per_launch_cluster(fn, kCluster, kThreads, 0, kCluster, stream, args);
  *rc = e == cudaSuccess ? PER_OK : per_record_cuda(e);
  return true;
}

int run(const per_tensor_t* list, int64_t n, const Call& c, bool partials, bool scaling,
        cudaStream_t stream) {
  int rc = PER_OK;
  if (partials && one_kernel(list, n, c, scaling, stream, &rc)) return rc;
  if (n <= Small::kTensors) {
    Small t;
    return one_table(&t, list, n, c, partials, scaling, stream);
  }
  if (n <= Medium::kTensors) {
    Medium t;
    return one_table(&t, list, n, c, partials, scaling, stream);
  }
  Large t;
  if (n <= Large::kTensors) return one_table(&t, list, n, c, partials, scaling, stream);
  int count = 0;
  for (int64_t i = 0; partials && i < n; i += Large::kTensors) {
    const int64_t grid = fill(&t, list + i, batch_of(n - i), Large::kCtas);
    if (grid < 0) return PER_ERR_TOO_LARGE;
    if (grid == 0) continue;
    rc = run_partials(&t, grid, c, count, stream);
    if (rc) return rc;
    count += (int)grid;
  }
  if (partials && (!scaling || count == 0)) return join(c, count, stream);
  bool first = true;
  for (int64_t i = 0; i < n; i += Large::kTensors) {
    const int64_t grid = fill(&t, list + i, batch_of(n - i), Large::kCtas);
    if (grid < 0) return PER_ERR_TOO_LARGE;
    if (grid == 0) continue;
    set_call(&t, c, count, first ? 0 : 1);
    rc = go((const void*)per_scale_kernel<Large>, grid, &t, stream);
    if (rc) return rc;
    first = false;
  }
  return PER_OK;
}

}  // namespace

int64_t per_grad_norm_bytes(int64_t n) {
  const int64_t launches = n <= Large::kTensors ? 1 : (n - 1) / Large::kTensors + 1;
  return launches * kMaxCtas * (int64_t)sizeof(double);
}

int per_launch_grad_norm(const per_tensor_t* tensors, int64_t n, int32_t kind, float* norm,
                         void* workspace, cudaStream_t stream) {
  return run(tensors, n, Call{kind, 0.f, norm, static_cast<double*>(workspace)}, true, false, stream);
}

int per_launch_scale_grads(const per_tensor_t* tensors, int64_t n, float max_norm,
                           const float* norm, cudaStream_t stream) {
  return run(tensors, n, Call{0, max_norm, const_cast<float*>(norm), nullptr}, false, true, stream);
}

int per_launch_clip_grad_norm(const per_tensor_t* tensors, int64_t n, int32_t kind, float max_norm,
                              float* norm, void* workspace, cudaStream_t stream) {
  return run(tensors, n, Call{kind, max_norm, norm, static_cast<double*>(workspace)}, true, true,
             stream);
}
