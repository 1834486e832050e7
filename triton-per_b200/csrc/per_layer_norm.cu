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
// precision; it is kept as the pair (s, avg(d)), because h loses
// |m| / sqrt(v) units of rounding to a mean held in one float32.
//
// Bytes: forward x read and y written once, backward x, dy read and dx written
// once, plus 16 bytes of statistics a row and the vectors; some 7 and 13
// operations a value, so that DRAM bounds every size beyond the L2 cache. What
// a row costs beyond its values (the sums over its threads, addresses, waits)
// decides how near a kernel comes, so rows are laid out by length (shape_of):
//   - up to 512 values, 16-bit ones up to 1,024 (512 in the backward pass of
//     whole vectors): LANES threads of a warp, several rows a warp;
//   - longer, whole vectors up to 8,192 values (16-bit forward: 16,384), rows that
//     start anywhere up to half of that: a group of warps of one CTA, rows copied
//     ahead into shared memory (forward, part of the upper half of whole vectors
//     goes to clusters of two, see shape_of);
//   - longer, up to 65,536 values (16-bit forward: 131,072): a cluster of up to 8
//     CTAs, each with a slice;
//   - longer: read from memory in each of two or three passes.
// The columns' sums dw and db: a thread keeps those of its columns in registers
// over all its rows; each CTA writes one partial row, and a second kernel adds
// these in a fixed order, so equal calls give equal bits.
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
  float4* stats;  // mean as a sum of two, rstd, 0
  int64_t rows, x_stride, y_stride;
  int32_t dim;
  float eps;
  int32_t group_threads;  // of a row that spans warps
};

struct Bwd {
  const void* dy;
  const void* x;
  const void* w;
  const float4* stats;
  void* dx;
  void* dw;
  void* db;
  float* part;  // [splits][2][padded]: sums of dw and db, in the order of `places`
  int64_t rows, dy_stride, x_stride, dx_stride;
  int32_t dim, splits;
  int32_t group_threads;  // of a row that spans warps
  int32_t joined;         // one cluster: no partial rows, its CTAs add their sums themselves
  struct Places {         // the order of the columns in a partial row, see store_columns()
    int32_t padded, slice, width, vec;
  } places;
};

// Sums of a and b over the CTA, in a fixed order; every thread gets them.
__device__ __forceinline__ double2 block_sum2(double a, double b) {
  __shared__ double2 s[32];
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    a += __shfl_xor_sync(PER_FULL_MASK, a, o);
    b += __shfl_xor_sync(PER_FULL_MASK, b, o);
  }
  __syncthreads();  // the previous sums have been read
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = make_double2(a, b);
  __syncthreads();
  double2 v = s[0];
  for (int k = 1; k < (int)(blockDim.x >> 5); ++k) v.x += s[k].x, v.y += s[k].y;
  return v;
}

// a / n for a count n, with inv = 1 / n: the first quotient corrected by its
// exact remainder, so that an exact quotient comes out exact.
__device__ __forceinline__ float over(float a, float n, float inv) {
  const float q = a * inv;
  return fmaf(fmaf(-q, n, a), inv, q);
}

// VEC values that are loaded and stored at once.
template <typename T, int VEC>
struct alignas(VEC * sizeof(T)) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load(const T* p) {
  Pack<T, VEC> r;
  if constexpr (VEC * sizeof(T) == 32) {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    reinterpret_cast<uint4*>(&r)[0] = a;
    reinterpret_cast<uint4*>(&r)[1] = b;
  } else if constexpr (VEC * sizeof(T) == 16) {
    *reinterpret_cast<uint4*>(&r) = *reinterpret_cast<const uint4*>(p);
  } else {
    static_assert(VEC == 1, "single values, or 16 and 32 bytes");
    r.v[0] = p[0];
  }
  return r;
}

template <typename T, int VEC>
__device__ __forceinline__ void store(T* p, const Pack<T, VEC>& r) {
  if constexpr (VEC == 1)
    p[0] = r.v[0];
  else
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(&r);
}

// The values of a thread, NV vectors of VEC, as pairs 0 .. NV VEC / 2, 16-bit
// ones by whole words.
template <typename T, int VEC, int NV>
__device__ __forceinline__ float2 get2(const Pack<T, VEC> (&p)[NV], int i) {
  if constexpr (sizeof(T) == 2 && VEC > 1)
    return per_unpack<T>(reinterpret_cast<const uint32_t*>(&p[2 * i / VEC])[i % (VEC / 2)]);
  else
    return make_float2(per_to_f32(p[2 * i / VEC].v[2 * i % VEC]),
                       per_to_f32(p[(2 * i + 1) / VEC].v[(2 * i + 1) % VEC]));
}
template <typename T, int VEC, int NV>
__device__ __forceinline__ void set2(Pack<T, VEC> (&p)[NV], int i, float2 f) {
  if constexpr (sizeof(T) == 2 && VEC > 1) {
    reinterpret_cast<uint32_t*>(&p[2 * i / VEC])[i % (VEC / 2)] = per_pack<T>(f);
  } else {
    p[2 * i / VEC].v[2 * i % VEC] = per_from_f32<T>(f.x);
    p[(2 * i + 1) / VEC].v[(2 * i + 1) % VEC] = per_from_f32<T>(f.y);
  }
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o; o >>= 1) v += __shfl_xor_sync(PER_FULL_MASK, v, o);
  return v;
}

// The sums of a and of b over LANES lanes, in the time of one: a first step
// leaves a to the even lanes and b to the odd ones. Even lanes return the sum
// of a, odd lanes that of b.
template <int LANES>
__device__ __forceinline__ float lanes_sum_split(float a, float b) {
  const bool odd = threadIdx.x & 1;
  float v = odd ? b : a;
  v += __shfl_xor_sync(PER_FULL_MASK, odd ? a : b, 1);
#pragma unroll
  for (int o = 2; o < LANES; o <<= 1) v += __shfl_xor_sync(PER_FULL_MASK, v, o);
  return v;
}
// both sums in every lane, from what lanes_sum_split() returned
__device__ __forceinline__ float2 join_split(float v) {
  const float o = __shfl_xor_sync(PER_FULL_MASK, v, 1);
  return (threadIdx.x & 1) ? make_float2(o, v) : make_float2(v, o);
}

// weight (or its absence as 1, bias as 0) of this thread's columns
template <typename P, int VEC, int NV>
__device__ __forceinline__ void load_columns(Pack<P, VEC> (&w)[NV], const void* p, float absent,
                                             int first, int width, int dim) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (first + k * width) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[k].v[j] = per_from_f32<P>(absent);
    if (c >= dim || !p) continue;
    const P* q = static_cast<const P*>(p) + c;
    if (VEC == 1 || (c + VEC <= dim && (uintptr_t)q % 16 == 0)) {
      w[k] = load<P, VEC>(q);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (c + j < dim) w[k].v[j] = q[j];
    }
  }
}

// Stops the compiler from holding 16-bit weights unpacked from row to row, in
// twice the registers.
template <typename P, int VEC, int NV>
__device__ __forceinline__ void keep_packed(Pack<P, VEC> (&w)[NV]) {
  if constexpr (sizeof(P) == 2 && VEC > 1) {
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
      for (int j = 0; j < VEC / 2; ++j)
        asm volatile("" : "+r"(reinterpret_cast<uint32_t*>(&w[k])[j]));
  }
}

// v -= s in the row's columns; the values beyond them, read as 0, stay at 0.
// The sums of v and of v^2.
template <int VEC, int NV>
__device__ __forceinline__ float2 centre(float2 (&v)[NV * VEC / 2], float s, int lane, int width,
                                         int dim) {
  const float2 m = per_both(-s);
#pragma unroll
  for (int i = 0; i < NV * VEC / 2; ++i) v[i] = per_add2(v[i], m);
  if ((lane + (NV - 1) * width + 1) * VEC > dim) {  // the end of the row is among this thread's
#pragma unroll
    for (int i = 0; i < NV * VEC / 2; ++i) {
      const int c0 = (lane + 2 * i / VEC * width) * VEC + 2 * i % VEC;
      const int c1 = VEC > 1 ? c0 + 1 : lane + (2 * i + 1) * width;
      if (c0 >= dim) v[i].x = 0.f;
      if (c1 >= dim) v[i].y = 0.f;
    }
  }
  float2 d1 = per_both(0.f), d2 = per_both(0.f);
#pragma unroll
  for (int i = 0; i < NV * VEC / 2; ++i) {
    d1 = per_add2(d1, v[i]);
    d2 = per_fma2(v[i], v[i], d2);
  }
  return make_float2(d1.x + d1.y, d2.x + d2.y);
}

// o = (v - shift) r w + b
template <typename T, typename P, int VEC, int NV>
__device__ __forceinline__ void normed(Pack<T, VEC> (&o)[NV], const float2 (&v)[NV * VEC / 2],
                                       float shift, float r, const Pack<P, VEC> (&w)[NV],
                                       const Pack<P, VEC> (&b)[NV]) {
  const float2 r2 = per_both(r), c2 = per_both(-shift * r);
#pragma unroll
  for (int i = 0; i < NV * VEC / 2; ++i) set2(o, i, per_fma2(per_fma2(v[i], r2, c2), get2(w, i), get2(b, i)));
}

template <typename T, int VEC, int NV>
__device__ __forceinline__ void store_row(T* y, const Pack<T, VEC> (&o)[NV], int lane, int width, int dim) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (lane + k * width) * VEC;
    if (c < dim) store<T, VEC>(y + c, o[k]);
  }
}

// Backward sums of a row's values in a thread: h = (x - mean) r, g = dy w, the
// column sums dw += dy h and db += dy, and the sums of g and of g h. Where
// dy is 0 nothing is added.
template <typename T, typename P, int VEC, int NV>
__device__ __forceinline__ float2 backward_sums(const Pack<T, VEC> (&qx)[NV], const Pack<T, VEC> (&qy)[NV],
                                                const Pack<P, VEC> (&w)[NV], float hi, float lo, float r,
                                                float2 (&h)[NV * VEC / 2], float2 (&g)[NV * VEC / 2],
                                                float2 (&aw)[NV * VEC / 2], float2 (&ab)[NV * VEC / 2]) {
  const float2 m2 = per_both(-hi), r2 = per_both(r), lor = per_both(-lo * r);
  float2 s1 = per_both(0.f), s2 = per_both(0.f);
#pragma unroll
  for (int i = 0; i < NV * VEC / 2; ++i) {
    const float2 d = get2(qy, i);
    h[i] = per_fma2(per_add2(get2(qx, i), m2), r2, lor);
    aw[i] = per_fma2(d, h[i], aw[i]);
    ab[i] = per_add2(ab[i], d);
    g[i] = per_mul2(d, get2(w, i));
    s1 = per_add2(s1, g[i]);
    s2 = per_fma2(g[i], h[i], s2);
  }
  return make_float2(s1.x + s1.y, s2.x + s2.y);
}

// o = r (g - sum g / n - h sum(g h) / n)
template <typename T, int VEC, int NV>
__device__ __forceinline__ void backward_values(Pack<T, VEC> (&o)[NV], const float2 (&h)[NV * VEC / 2],
                                                const float2 (&g)[NV * VEC / 2], float2 sums,
                                                float inv_n, float r) {
  const float2 r2 = per_both(r), k0 = per_both(-r * (sums.x * inv_n)),
               k1 = per_both(-r * (sums.y * inv_n));
#pragma unroll
  for (int i = 0; i < NV * VEC / 2; ++i) set2(o, i, per_fma2(h[i], k1, per_fma2(g[i], r2, k0)));
}

// A thread's column sums into a partial row: four neighbouring columns at a
// time, thread after thread, so that a warp's stores are whole lines (column by
// column a thread's stores lie 16 or 32 bytes from its neighbour's: the partial
// rows of 16384x8192 bfloat16 took 17 us to write and join, 7 us so). Columns
// beyond the row are stored too, and not looked at.
template <int VEC, int NV>
__device__ __forceinline__ void store_columns(float* part, const float2 (&a)[NV * VEC / 2], int lane,
                                              int width) {
  if constexpr (VEC > 1) {
#pragma unroll
    for (int q = 0; q < NV * VEC / 4; ++q)
      reinterpret_cast<float4*>(part)[q * width + lane] =
          make_float4(a[2 * q].x, a[2 * q].y, a[2 * q + 1].x, a[2 * q + 1].y);
  } else {
#pragma unroll
    for (int i = 0; i < NV / 2; ++i) {
      part[2 * i * width + lane] = a[i].x;
      part[(2 * i + 1) * width + lane] = a[i].y;
    }
  }
}
// The column that place p of a partial row holds.
__device__ __forceinline__ int column_at(const Bwd::Places& o, int p) {
  const int cta = p / o.slice, r = p % o.slice;
  if (o.vec == 1) return p;
  const int q = r / 4 / o.width, lane = r / 4 % o.width, per = o.vec / 4;
  return cta * o.slice + (lane + q / per * o.width) * o.vec + q % per * 4 + r % 4;
}

// The partial rows [groups][2][padded] of a CTA's groups, in shared memory,
// added into one.
__device__ __forceinline__ void add_groups(float* part, const float* sums, int groups, int padded) {
  for (int c = threadIdx.x; c < padded / 2; c += blockDim.x) {
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int q = 0; q < groups; ++q) {
      const float4 u = reinterpret_cast<const float4*>(sums)[q * (padded / 2) + c];
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
    reinterpret_cast<float4*>(part)[c] = v;
  }
}

// ---- clusters of CTAs
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t remote_address(const void* p, uint32_t cta) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
               : "=r"(r)
               : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(cta));
  return r;
}

// ---- short rows: LANES threads of a warp (a power of two) per row, several
// rows per warp, nothing but shuffles between the threads. Measured (back to
// back in a graph, new inputs): 65536x256 float32 24.5 us forward (5.5 TB/s),
// 35.5 us backward (5.7 TB/s); 8191x1001 half, single values, 12.3 and 19 us; 65536x32 columns of 74-value rows, forward, 7.0
// us; 1x256 1.25 us, of which the launch is most.

// A thread's own copies on their way into shared memory, STAGES rows ahead:
// it waits for and reads only what it has copied itself, so no barrier is
// needed. 16-byte vectors go by cp.async; single values are fetched into
// registers one row ahead. Where `in` is false the vector reads as zeros.
template <typename T, int VEC, int NV, int STAGES>
struct Ring {
  static constexpr bool kAsync = VEC * sizeof(T) == 16;
  static constexpr int kStages = kAsync ? STAGES : 1;
  static constexpr size_t kBytes = kAsync ? STAGES * NV * 16 : 0;  // per thread
  const uint4* mine;
  uint32_t at;
  Pack<T, VEC> reg[kAsync ? 1 : NV];

  __device__ __forceinline__ explicit Ring(const void* smem) {
    mine = static_cast<const uint4*>(smem) + threadIdx.x;
    at = (uint32_t)__cvta_generic_to_shared(mine);
  }
  __device__ __forceinline__ void fetch(int stage, int k, const T* p, bool in) {
    if constexpr (kAsync) {
      // a copy of 0 bytes reads nothing and fills the vector with zeros
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       at + (stage * NV + k) * blockDim.x * 16),
                   "l"(p), "r"(in ? 16 : 0)
                   : "memory");
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) reg[k].v[j] = per_from_f32<T>(0.f);
      if (in) reg[k] = load<T, VEC>(p);
    }
  }
  static __device__ __forceinline__ void commit() {
    if constexpr (kAsync) asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // the oldest stage has landed (one group per stage is in flight)
  static __device__ __forceinline__ void wait() {
    if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
  }
  __device__ __forceinline__ Pack<T, VEC> get(int stage, int k) {
    if constexpr (kAsync) {
      Pack<T, VEC> r;
      *reinterpret_cast<uint4*>(&r) = mine[(stage * NV + k) * blockDim.x];
      return r;
    } else {
      return reg[k];
    }
  }
};

constexpr int kWarpStages = 3;

template <typename T, typename P, int VEC, int NV, int LANES>
__global__ void __launch_bounds__(128) per_layer_norm_warp_kernel(const Fwd f) {
  extern __shared__ __align__(16) unsigned char dyn[];
  using R = Ring<T, VEC, NV, kWarpStages>;
  R ring(dyn);
  int stage = 0;
  const int lane = threadIdx.x % LANES, mine = (threadIdx.x & 31) / LANES;
  const int per_cta = blockDim.x / LANES;
  const int64_t step = (int64_t)gridDim.x * per_cta;
  const float n = (float)f.dim, inv_n = 1.f / n;
  const T* x = static_cast<const T*>(f.x);
  per_wait_previous_grid();
  auto fetch = [&](int st, int64_t row) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * LANES) * VEC;
      ring.fetch(st, k, x + row * f.x_stride + c, row < f.rows && c < f.dim);
    }
    R::commit();
  };
  int64_t base = (int64_t)blockIdx.x * per_cta + (threadIdx.x & ~31) / LANES;
#pragma unroll
  for (int k = 0; k < R::kStages; ++k) fetch(k, base + mine + k * step);
  Pack<P, VEC> w[NV], b[NV];
  load_columns(w, f.w, 1.f, lane, LANES, f.dim);
  load_columns(b, f.b, 0.f, lane, LANES, f.dim);
  for (; base < f.rows; base += step) {
    const int64_t row = base + mine;
    float2 v[NV * VEC / 2];
    float2 a = per_both(0.f);
    R::wait();
    {
      Pack<T, VEC> q[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) q[k] = ring.get(stage, k);
#pragma unroll
      for (int i = 0; i < NV * VEC / 2; ++i) {
        v[i] = get2(q, i);
        a = per_add2(a, v[i]);
      }
    }
    fetch(stage, row + R::kStages * step);
    stage = stage + 1 == R::kStages ? 0 : stage + 1;
    const float s = over(lanes_sum<LANES>(a.x + a.y), n, inv_n);
    const float2 e = centre<VEC, NV>(v, s, lane, LANES, f.dim);
    const float shift = over(lanes_sum<LANES>(e.x), n, inv_n);
    const float var = fmaf(-shift, shift, lanes_sum<LANES>(e.y) * inv_n);
    const float r = rsqrtf(fmaxf(var, 0.f) + f.eps);
    if (row < f.rows) {
      Pack<T, VEC> o[NV];
      normed<T, P, VEC, NV>(o, v, shift, r, w, b);
      store_row(static_cast<T*>(f.y) + row * f.y_stride, o, lane, LANES, f.dim);
      if (f.stats && lane == 0) f.stats[row] = make_float4(s, shift, r, 0.f);
    }
  }
}

constexpr int kJoinCtas = 16;  // of a launch that joins its own column sums

// Rows beyond the last read as dy = 0 and so add nothing to any sum.
template <typename T, typename P, int VEC, int NV, int LANES>
__global__ void __launch_bounds__(256) per_layer_norm_backward_warp_kernel(const Bwd g) {
  extern __shared__ __align__(16) unsigned char dyn[];
  using R = Ring<T, VEC, 2 * NV, kWarpStages>;
  R ring(dyn);
  int stage = 0;
  const int lane = threadIdx.x % LANES, mine = (threadIdx.x & 31) / LANES;
  const int per_cta = blockDim.x / LANES;
  const int64_t step = (int64_t)gridDim.x * per_cta;
  const float inv_n = 1.f / (float)g.dim;
  const T* x = static_cast<const T*>(g.x);
  const T* dy = static_cast<const T*>(g.dy);
  per_wait_previous_grid();
  auto fetch = [&](int st, int64_t row) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (lane + k * LANES) * VEC;
      const bool in = row < g.rows && c < g.dim;
      ring.fetch(st, k, x + row * g.x_stride + c, in);
      ring.fetch(st, NV + k, dy + row * g.dy_stride + c, in);
    }
    R::commit();
  };
  float2 nm = per_both(0.f);
  float nr = 0.f;
  auto fetch_stats = [&](int64_t row) {
    if (row >= g.rows) return;
    const float* st = reinterpret_cast<const float*>(g.stats + row);
    nm = *reinterpret_cast<const float2*>(st);
    nr = st[2];
  };
  int64_t base = (int64_t)blockIdx.x * per_cta + (threadIdx.x & ~31) / LANES;
#pragma unroll
  for (int k = 0; k < R::kStages; ++k) fetch(k, base + mine + k * step);
  fetch_stats(base + mine);
  Pack<P, VEC> w[NV];
  load_columns(w, g.w, 1.f, lane, LANES, g.dim);
  float2 aw[NV * VEC / 2], ab[NV * VEC / 2];
#pragma unroll
  for (int i = 0; i < NV * VEC / 2; ++i) aw[i] = ab[i] = per_both(0.f);
  for (; base < g.rows; base += step) {
    const int64_t row = base + mine;
    const float hi = nm.x, lo = nm.y, r = nr;
    float2 h[NV * VEC / 2], gv[NV * VEC / 2], e;
    R::wait();
    {
      Pack<T, VEC> qx[NV], qy[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        qx[k] = ring.get(stage, k);
        qy[k] = ring.get(stage, NV + k);
      }
      e = backward_sums(qx, qy, w, hi, lo, r, h, gv, aw, ab);
    }
    fetch(stage, row + R::kStages * step);
    fetch_stats(row + step);
    stage = stage + 1 == R::kStages ? 0 : stage + 1;
    if (!g.dx) continue;
    const float2 sums = join_split(lanes_sum_split<LANES>(e.x, e.y));
    if (row < g.rows) {
      Pack<T, VEC> o[NV];
      backward_values<T, VEC, NV>(o, h, gv, sums, inv_n, r);
      store_row(static_cast<T*>(g.dx) + row * g.dx_stride, o, lane, LANES, g.dim);
    }
  }
  if (!g.part && !g.joined) return;
  // the row groups of a warp by shuffles, then the warps through shared
  // memory, where the (empty) copies still in flight have ended
  constexpr int kPadded = LANES * NV * VEC;
  float* sums = reinterpret_cast<float*>(dyn);  // [warps][2][padded]
  float* own = sums + (threadIdx.x >> 5) * 2 * kPadded;
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NV * VEC / 2; ++i)
#pragma unroll
    for (int o = LANES; o < 32; o <<= 1) {
      aw[i].x += __shfl_xor_sync(PER_FULL_MASK, aw[i].x, o);
      aw[i].y += __shfl_xor_sync(PER_FULL_MASK, aw[i].y, o);
      ab[i].x += __shfl_xor_sync(PER_FULL_MASK, ab[i].x, o);
      ab[i].y += __shfl_xor_sync(PER_FULL_MASK, ab[i].y, o);
    }
  if (mine == 0) {
    store_columns<VEC, NV>(own, aw, lane, LANES);
    store_columns<VEC, NV>(own + kPadded, ab, lane, LANES);
  }
  __syncthreads();
  if (!g.joined) {
    add_groups(g.part + (int64_t)blockIdx.x * 2 * kPadded, sums, blockDim.x >> 5, kPadded);
    return;
  }
  // Few rows: the launch is one cluster, and each of its CTAs adds a share of the columns over all.
  float* all = sums + (blockDim.x >> 5) * 2 * kPadded;
  add_groups(all, sums, blockDim.x >> 5, kPadded);
  cluster_sync();
  const int ctas = (int)cluster_size();
  for (int p = (int)(cluster_rank() * blockDim.x + threadIdx.x); p < 2 * kPadded; p += ctas * blockDim.x) {
    float u[kJoinCtas];
#pragma unroll
    for (int c = 0; c < kJoinCtas; ++c) {  // every load on its way before the first is needed
      u[c] = 0.f;
      if (c < ctas)
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u[c]) : "r"(remote_address(all + p, c)));
    }
    float v = 0.f;
#pragma unroll
    for (int c = 0; c < kJoinCtas; ++c) v += u[c];
    const int c = column_at(g.places, p % kPadded);
    void* out = p < kPadded ? g.dw : g.db;
    if (out && c < g.dim) static_cast<P*>(out)[c] = per_from_f32<P>(v);
  }
  cluster_sync();  // no CTA ends while another may still read from it
}

// ---- longer rows: a group of warps per row (several groups in a CTA), or a
// cluster of CTAs per row, each with a slice of it.

constexpr int kMaxCluster = 8;
constexpr int kRowThreads = 512;  // of a CTA
constexpr int kMaxGroups = 8;

// A thread's place: `lane` of `width` threads that hold the values first ..
// first + dim of a row.
template <bool CLUSTER>
struct Group {
  int lane, width, index;  // index: of this CTA's groups
  int first, dim;          // this CTA's slice of the row
  int warps;               // of all CTAs of the row
  int64_t base, step;      // first row, rows between two turns
  __device__ __forceinline__ Group(int threads, int vec, int nv, int row_dim) {
    const int groups = CLUSTER ? 1 : blockDim.x / threads;
    index = CLUSTER ? 0 : threadIdx.x / threads;
    lane = threadIdx.x - index * threads;
    width = threads;
    first = 0;
    dim = row_dim;
    warps = width >> 5;
    base = (int64_t)blockIdx.x * groups + index;
    step = (int64_t)gridDim.x * groups;
    if constexpr (CLUSTER) {
      const int ctas = (int)cluster_size();
      base = blockIdx.x / ctas;
      step = gridDim.x / ctas;
      warps *= ctas;
      const int slice = threads * nv * vec;
      first = (int)cluster_rank() * slice;
      dim = row_dim - first;
      dim = dim < 0 ? 0 : dim > slice ? slice : dim;
    }
  }
};

// What the warps of a row hand to one another. In one CTA: each warp's words,
// then a barrier of the group. Over a cluster: each warp's words go to every
// CTA by st.async, which counts their bytes on a barrier word there that the
// CTA's threads wait for; a cluster barrier in its place also waits for the
// output rows that the threads have stored before.
// Two buffers by turns, so that one barrier per exchange is enough: a buffer is
// written again only in the next exchange but one, whose sender has waited for
// the exchange between, and with it for all readers of this one.
template <bool CLUSTER>
struct Exchange {
  static constexpr int kWarps = kRowThreads / 32 * (CLUSTER ? kMaxCluster : 1);
  float4 slot[2][kWarps];
  uint64_t arrived[2];  // CLUSTER
};

// The state of a thread in the exchanges of its row.
template <bool CLUSTER>
struct Turns {
  int turn = 0, parity = 0;
  bool failed = false;  // a wait has given up: nothing that follows is waited for
  // Once, by all threads of the CTA; a cluster barrier has to follow.
  __device__ __forceinline__ void begin(Exchange<CLUSTER>& e) {
    if constexpr (CLUSTER)
      if (threadIdx.x == 0) {
        per_mbar_init(&e.arrived[0], 1);
        per_mbar_init(&e.arrived[1], 1);
        per_fence_mbar_init();
      }
  }
  // The words that each warp sends (`bytes` of them) are here.
  __device__ __forceinline__ void wait(Exchange<CLUSTER>& e, int warps, int bytes) {
    if constexpr (CLUSTER) {
      if (threadIdx.x == 0 && !failed) per_mbar_arrive_expect_tx(&e.arrived[turn], warps * bytes);
      if (!failed) failed = !per_mbar_wait(&e.arrived[turn], parity, nullptr);
    }
  }
  __device__ __forceinline__ void next() {
    turn ^= 1;
    parity ^= turn ^ 1;  // flips when both buffers have had their turn
  }
};

// Among the threads of one CTA that share a row.
template <bool CLUSTER>
__device__ __forceinline__ void cta_part_sync(const Group<CLUSTER>& t) {
  __syncwarp();
  if (t.width > 32) asm volatile("bar.sync %0, %1;" ::"r"(t.index + 1), "r"(t.width) : "memory");
}
template <bool CLUSTER>
__device__ __forceinline__ void put(Exchange<CLUSTER>& e, Turns<CLUSTER>& turns, const Group<CLUSTER>& t,
                                    float4 v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if constexpr (!CLUSTER) {
    if (lane == 0) e.slot[turns.turn][warp] = v;
    cta_part_sync(t);
  } else {
    if (lane < (int)cluster_size()) {  // lane = the CTA that the warp's words go to
      const uint32_t to =
          remote_address(&e.slot[turns.turn][cluster_rank() * (blockDim.x >> 5) + warp], lane);
      asm volatile(
          "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(to),
          "r"(__float_as_uint(v.x)), "r"(__float_as_uint(v.y)), "r"(__float_as_uint(v.z)),
          "r"(__float_as_uint(v.w)), "r"(remote_address(&e.arrived[turns.turn], lane))
          : "memory");
    }
    turns.wait(e, t.warps, 16);
  }
}

// The warps of a row as a lane sees them in an exchange: lane l reads warps
// l mod span, + 32, ...; a butterfly over `span` lanes then joins them all.
template <bool CLUSTER>
struct Warps {
  static constexpr int kReads = Exchange<CLUSTER>::kWarps > 32 ? Exchange<CLUSTER>::kWarps / 32 : 1;
  int span, first, from;
  __device__ __forceinline__ explicit Warps(const Group<CLUSTER>& t) {
    span = 1;
    while (span < t.warps && span < 32) span *= 2;
    first = threadIdx.x & (span - 1);
    from = t.index * t.warps;
  }
  __device__ __forceinline__ float sum(float v) const {
    for (int o = span >> 1; o; o >>= 1) v += __shfl_xor_sync(PER_FULL_MASK, v, o);
    return v;
  }
};

// lanes_sum_split() of a warp in, that of the whole row out. `span`: lanes'
// worth of warps, a power of two up to 16.
template <bool CLUSTER>
__device__ __forceinline__ float exchange_split(Exchange<CLUSTER>& e, Turns<CLUSTER>& turns,
                                                const Group<CLUSTER>& t, int span, float v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  float* slots = reinterpret_cast<float*>(e.slot[turns.turn]);  // [warp][2]
  if constexpr (!CLUSTER) {
    if (lane < 2) slots[2 * warp + lane] = v;
    cta_part_sync(t);
  } else {
    if (lane < 2 * (int)cluster_size()) {  // lanes 2 c and 2 c + 1: to CTA c
      const uint32_t to = remote_address(
          &slots[2 * (cluster_rank() * (blockDim.x >> 5) + warp) + (lane & 1)], lane >> 1);
      asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to),
                   "r"(__float_as_uint(v)), "r"(remote_address(&e.arrived[turns.turn], lane >> 1))
                   : "memory");
    }
    turns.wait(e, t.warps, 8);
  }
  turns.next();
  const int first = 2 * t.index * t.warps, at = lane & (2 * span - 1);
  v = 0.f;
#pragma unroll
  for (int i = 0; i < (CLUSTER ? Exchange<CLUSTER>::kWarps / 16 : 1); ++i)
    if (at + 32 * i < 2 * t.warps) v += slots[first + at + 32 * i];
  for (int o = span; o > 1; o >>= 1) v += __shfl_xor_sync(PER_FULL_MASK, v, o);
  return v;
}

// One of the arrays whose rows a kernel reads: this CTA's slice of row r is the
// `dim` values from first + r stride on. [begin, end): what the rows of the
// array span.
template <typename T>
struct Array {
  const T* first;
  int64_t stride;
  uintptr_t begin, end;
  __device__ __forceinline__ Array(const void* p, int64_t row_stride, int64_t rows, int row_dim,
                                   int slice_first)
      : first(static_cast<const T*>(p) + slice_first), stride(row_stride) {
    begin = (uintptr_t)p;
    end = begin + (uintptr_t)((rows - 1) * row_stride + row_dim) * sizeof(T);
  }
  __device__ __forceinline__ const T* row(int64_t r) const { return first + r * stride; }
  // where row r starts between two 16-byte boundaries
  __device__ __forceinline__ int phase(int64_t r) const {
    return (int)(((uint32_t)(uintptr_t)first + (uint32_t)r * (uint32_t)(stride * (int64_t)sizeof(T))) & 15u);
  }
};

// 16 bytes from any element boundary of shared memory: vector i past `phase`
// bytes (0 .. 15) from a 16-byte boundary.
__device__ __forceinline__ uint4 window(const unsigned char* base, int i, int phase) {
  const uint4* p = reinterpret_cast<const uint4*>(base) + i;
  const uint4 a = p[0], b = p[1];
  uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  if (phase & 8)
#pragma unroll
    for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
  if (phase & 4)
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
  const int shift = (phase & 3) * 8;
  return make_uint4(__funnelshift_r(w[0], w[1], shift), __funnelshift_r(w[1], w[2], shift),
                    __funnelshift_r(w[2], w[3], shift), __funnelshift_r(w[3], w[4], shift));
}

// The rows of a group on their way into shared memory, STAGES of them, ARRAYS
// arrays each (plus, STATS, the 16 bytes of a row's statistics), by bulk copies
// that one thread issues, so that the others spend no instruction on
// addresses. A slot is filled again once every thread of the group is known to
// have read it: each has put what it read into the exchange that precedes.
//
// ANY false: rows are whole vectors on 16-byte boundaries. ANY: rows of any
// length that start anywhere; the copy takes the 16-byte blocks that hold a row
// (its neighbours' values come along and are masked), except where such a block
// would reach beyond the array, before its first row or behind its last: those
// rows are fetched value by value, by ordinary stores of all threads, which only
// a barrier orders before other threads' reads (and the Outbox's reads before
// its next row). Within one CTA the exchange has one; the st.async of a cluster's
// exchange orders nothing but its own bytes, so there the kernels add one.
template <typename T, int NV, int ARRAYS, int STAGES, bool STATS, bool ANY>
struct Rows {
  static constexpr int VEC = 16 / sizeof(T);
  unsigned char* slots;
  uint64_t* bars;
  int array_bytes, slot_bytes;
  int stage, parity;
  bool failed;  // a wait has given up: nothing that follows is waited for
  int phase[ARRAYS];

  // shared memory of one array's slice (ANY: a vector more than the slice, for
  // the phase, and one that window() reads), and of a group
  static __host__ __device__ int room(int width) { return width * NV * 16 + (ANY ? 32 : 0); }
  static __host__ __device__ size_t bytes(int width) {
    return (size_t)STAGES * (ARRAYS * room(width) + 16);
  }
  __device__ __forceinline__ Rows(unsigned char* smem, uint64_t* group_bars, int width) {
    slots = smem;
    bars = group_bars;
    array_bytes = room(width);
    slot_bytes = ARRAYS * array_bytes + 16;
    stage = parity = 0;
    failed = false;
#pragma unroll
    for (int a = 0; a < ARRAYS; ++a) phase[a] = 0;
  }
  // Once, before anything else, by all threads of the group: the barriers, and
  // zeros for the vectors beyond the slice, which no copy writes (ANY: get()
  // masks them). A barrier of the CTA has to follow.
  __device__ __forceinline__ void begin(int dim, int lane, int width) {
    if (lane == 0) {
      for (int k = 0; k < STAGES; ++k) per_mbar_init(bars + k, 1);
      per_fence_mbar_init();
    }
    if constexpr (!ANY) {
      for (int k = 0; k < STAGES * ARRAYS; ++k) {
        unsigned char* array = slots + k / ARRAYS * slot_bytes + k % ARRAYS * array_bytes;
        for (int i = dim * (int)sizeof(T) + lane * 16; i < array_bytes; i += width * 16)
          *reinterpret_cast<uint4*>(array + i) = make_uint4(0, 0, 0, 0);
      }
      per_fence_proxy_async_smem();
    }
  }
  // Fill slot `st` with row r (`in`: there is one). All threads of the group
  // call it.
  __device__ __forceinline__ void fetch(int st, const Array<T> (&arrays)[ARRAYS], const float4* stats,
                                        int64_t r, int dim, int lane, int width, bool in) {
    if (!in || failed) return;
    unsigned char* slot = slots + st * slot_bytes;
    if constexpr (!ANY) {
      if (lane) return;
      const uint32_t bytes = (uint32_t)dim * sizeof(T);
      per_mbar_arrive_expect_tx(bars + st, ARRAYS * bytes + (STATS ? 16 : 0));
#pragma unroll
      for (int a = 0; a < ARRAYS; ++a)
        if (bytes) per_bulk_load(slot + a * array_bytes, arrays[a].row(r), bytes, bars + st);
    } else {
      uint32_t bytes[ARRAYS], all = STATS ? 16 : 0;
      uintptr_t from[ARRAYS];
#pragma unroll
      for (int a = 0; a < ARRAYS; ++a) {
        const T* p = arrays[a].row(r);
        from[a] = (uintptr_t)p & ~(uintptr_t)15;
        const uintptr_t to = ((uintptr_t)(p + dim) + 15) & ~(uintptr_t)15;
        bytes[a] = dim ? (uint32_t)(to - from[a]) : 0;
        if (dim && (from[a] < arrays[a].begin || to > arrays[a].end)) {
          bytes[a] = 0;  // value by value
          T* out = reinterpret_cast<T*>(slot + a * array_bytes + ((uintptr_t)p & 15));
          for (int c = lane; c < dim; c += width) out[c] = p[c];
          per_fence_proxy_async_smem();  // before a later copy into the same slot
        }
        all += bytes[a];
      }
      if (lane) return;
      per_mbar_arrive_expect_tx(bars + st, all);
#pragma unroll
      for (int a = 0; a < ARRAYS; ++a)
        if (bytes[a])
          per_bulk_load(slot + a * array_bytes, reinterpret_cast<const void*>(from[a]), bytes[a],
                        bars + st);
    }
    if (STATS) per_bulk_load(slot + ARRAYS * array_bytes, stats + r, 16, bars + st);
  }
  // Wait for row r, the next one.
  __device__ __forceinline__ void wait(const Array<T> (&arrays)[ARRAYS], int64_t r) {
    if (!failed) failed = !per_mbar_wait(bars + stage, parity, nullptr);
    if constexpr (ANY)
#pragma unroll
      for (int a = 0; a < ARRAYS; ++a) phase[a] = arrays[a].phase(r);
  }
  // Vector `lane + k width` of the row's slice, zeros beyond its end.
  __device__ __forceinline__ Pack<T, VEC> get(int a, int k, int dim, int lane, int width) const {
    const unsigned char* array = slots + stage * slot_bytes + a * array_bytes;
    const int i = lane + k * width;
    Pack<T, VEC> q;
    if constexpr (!ANY) {
      *reinterpret_cast<uint4*>(&q) = *reinterpret_cast<const uint4*>(array + i * 16);
    } else {
      *reinterpret_cast<uint4*>(&q) = window(array, i, phase[a]);
      if ((i + 1) * VEC > dim) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (i * VEC + j >= dim) q.v[j] = per_from_f32<T>(0.f);
      }
    }
    return q;
  }
  __device__ __forceinline__ float4 get_stats() const {
    return *reinterpret_cast<const float4*>(slots + stage * slot_bytes + ARRAYS * array_bytes);
  }
  __device__ __forceinline__ void next() {
    if (++stage == STAGES) {
      stage = 0;
      parity ^= 1;
    }
  }
  // After the last row. Where a wait gave up, copies may still be on their way
  // into this CTA's memory: wait once more for each, within the same limit.
  __device__ __forceinline__ void end() {
    if (failed)
      for (int k = 0; k < STAGES; ++k)
        per_mbar_wait(bars + k, k < stage ? parity ^ 1 : parity, nullptr);
  }
};

// The way out for rows of any length that start anywhere: each thread puts its
// vectors into shared memory and takes those back that lie on 16-byte
// boundaries of the output; values at either end are stored one by one.
template <typename T, int NV>
struct Outbox {
  static constexpr int VEC = 16 / sizeof(T);
  static __host__ __device__ size_t bytes(int width) { return (size_t)width * NV * 16 + 48; }

  // Between two barriers of the group, of which the second is its own.
  template <bool CLUSTER>
  static __device__ __forceinline__ void store_row(unsigned char* box, T* y, const Pack<T, VEC> (&o)[NV],
                                                   const Group<CLUSTER>& t) {
    // the row begins one vector into the box
#pragma unroll
    for (int k = 0; k < NV; ++k)
      *reinterpret_cast<uint4*>(box + 16 + (t.lane + k * t.width) * 16) =
          *reinterpret_cast<const uint4*>(&o[k]);
    cta_part_sync(t);
    const int phase = (int)((uintptr_t)y & 15), first = -phase / (int)sizeof(T);
    unsigned char* out = reinterpret_cast<unsigned char*>(y) - phase;  // on a boundary
    const int skip = (16 - phase) >> 4;  // 1 where the row begins on one
#pragma unroll
    for (int k = 0; k <= NV; ++k) {
      const int i = t.lane + k * t.width;
      const int c = first + i * VEC;  // of the block's first value
      if (c >= t.dim || (k == NV && t.lane > 0)) continue;
      Pack<T, VEC> q;
      *reinterpret_cast<uint4*>(&q) = window(box, i + skip, (16 - phase) & 15);
      if (c >= 0 && c + VEC <= t.dim) {
        *reinterpret_cast<uint4*>(out + (int64_t)i * 16) = *reinterpret_cast<const uint4*>(&q);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (c + j >= 0 && c + j < t.dim) y[c + j] = q.v[j];
      }
    }
  }
};

// Rows ahead, of which more cost shared memory that nothing else needs: two
// are enough for the forward pass (16384x8192 bfloat16 93 us, three: 99) and for
// float32 rows backward (8192x16384: 238 us, three: 280); 16-bit rows backward,
// half the bytes, take three (16384x8192: 133 us, two: 146), unless an outbox
// has to fit beside them.
constexpr int kFwdStages = 2;
template <typename T, bool ANY>
constexpr int kBwdStages = ANY || sizeof(T) == 4 ? 2 : 3;

// Threads that a CTA is compiled for, which bounds a thread's registers. 32
// values of 16-bit rows with their weights and biases take some 144: CTAs of
// up to 192 threads get them (168 each, and as many CTAs per SM), since what
// the compiler spills at 128 costs up to half the time (32768x4096 bfloat16:
// 88 us without, 100 to 140 with). Larger CTAs keep 16-bit weights packed
// instead (16384x8192: 140 -> 104 us).
template <typename T, int NV>
constexpr bool kWide = sizeof(T) == 2 && NV == 4;
constexpr int kWideThreads = 384;

// Each thread holds its values in registers; two exchanges of the group's warps
// (mean, then squares) are one, because a warp's own mean and squares are
// enough to have the row's. Measured: 65536x4096 bfloat16 177 us (6.1 TB/s of
// the 6.5 TB/s of a copy; 193 us under a second's load, when the clocks fall),
// 16384x4096 float32 83 us (6.4 TB/s), 8192x16384 float32 in clusters of two
// 189 us (5.6 TB/s), 20000x1003 float32 34-37 us (4.4-4.7 TB/s).
template <typename T, typename P, int NV, bool CLUSTER, bool ANY, int THREADS>
__global__ void __launch_bounds__(THREADS) per_layer_norm_group_kernel(const Fwd f) {
  __shared__ Exchange<CLUSTER> ex;
  __shared__ __align__(8) uint64_t bars[kMaxGroups][kFwdStages];
  extern __shared__ __align__(16) unsigned char dyn[];
  constexpr int VEC = 16 / sizeof(T);
  using R = Rows<T, NV, 1, kFwdStages, false, ANY>;
  const Group<CLUSTER> t(f.group_threads, VEC, NV, f.dim);
  unsigned char* mine = dyn + t.index * (R::bytes(t.width) + (ANY ? Outbox<T, NV>::bytes(t.width) : 0));
  R rows(mine, bars[t.index], t.width);
  rows.begin(t.dim, t.lane, t.width);
  Turns<CLUSTER> turns;
  turns.begin(ex);
  const float n = (float)f.dim, inv_n = 1.f / n;
  const Array<T> x[1] = {Array<T>(f.x, f.x_stride, f.rows, f.dim, t.first)};
  T* y = static_cast<T*>(f.y) + t.first;

  // values of a warp of the row: this one's, and those of the warps that this
  // lane reads in an exchange
  const Warps<CLUSTER> all(t);
  auto values_of = [&](int warp) {
    const int per_cta = t.width >> 5, rank = CLUSTER ? warp / per_cta : 0;
    const int dim = f.dim - rank * t.width * NV * VEC;  // from that CTA's slice on
    int v = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int left = dim - ((warp - rank * per_cta) * 32 + k * t.width) * VEC;
      v += left < 0 ? 0 : left > 32 * VEC ? 32 * VEC : left;
    }
    return (float)v;
  };
  constexpr int Q = Warps<CLUSTER>::kReads;
  float mq[Q];
  const float own = values_of((t.lane >> 5) + (CLUSTER ? (int)cluster_rank() * (t.width >> 5) : 0));
#pragma unroll
  for (int i = 0; i < Q; ++i)
    mq[i] = all.first + 32 * i < t.warps ? values_of(all.first + 32 * i) : 0.f;
  const float inv_own = own > 0.f ? 1.f / own : 0.f;
  const int lead = t.dim - (t.lane & ~31) * VEC;  // values of the warp's first vectors
  const float inv_lead = lead > 0 ? 1.f / (float)(lead > 32 * VEC ? 32 * VEC : lead) : 0.f;

  if constexpr (CLUSTER)
    cluster_sync();  // before a CTA writes into another one's shared memory, that one has to run
  else
    __syncthreads();
  per_wait_previous_grid();
  auto fetch = [&](int st, int64_t row) {
    rows.fetch(st, x, nullptr, row, t.dim, t.lane, t.width, row < f.rows);
  };
  for (int k = 0; k < kFwdStages; ++k) fetch(k, t.base + k * t.step);
  if constexpr (ANY) cta_part_sync(t);  // values that were fetched one by one
  Pack<P, VEC> w[NV], b[NV];
  load_columns(w, f.w ? static_cast<const P*>(f.w) + t.first : nullptr, 1.f, t.lane, t.width, t.dim);
  load_columns(b, f.b ? static_cast<const P*>(f.b) + t.first : nullptr, 0.f, t.lane, t.width, t.dim);
  for (int64_t row = t.base; row < f.rows; row += t.step) {
    float2 v[NV * VEC / 2];
    float2 a = per_both(0.f);
    if constexpr (kWide<T, NV> && THREADS > kWideThreads) {
      keep_packed(w);
      keep_packed(b);
    }
    rows.wait(x, row);
    {
      Pack<T, VEC> q[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) q[k] = rows.get(0, k, t.dim, t.lane, t.width);
#pragma unroll
      for (int i = 0; i < NV * VEC / 2; ++i) v[i] = get2(q, i);
#pragma unroll
      for (int i = 0; i < VEC / 2; ++i) a = per_add2(a, v[i]);
    }
    // Distances from a mean of the warp's own first: of its first vectors alone, a part 1 / NV of
    // its values or more, whose mean lies within sqrt(NV - 1) standard deviations of the warp's,
    // so that the subtraction in its squares below loses no more than 2 bits (NV 4). Warp q of m_q
    // values then has the mean s_q + u_q with u_q = d1_q / m_q, and squares around it
    // d2_q - d1_q u_q. Seen from s_0 its mean lies at z_q; the row's at z = sum m_q z_q / n, and the
    // row's squares are the warps' plus m_q (z_q - z)^2 each.
    const float s = lanes_sum<32>(a.x + a.y) * inv_lead;
    const float2 e = centre<VEC, NV>(v, s, t.lane, t.width, t.dim);
    const float e1 = lanes_sum<32>(e.x), e2 = lanes_sum<32>(e.y);
    const float u = over(e1, own, inv_own);
    put(ex, turns, t, make_float4(s, u, fmaxf(fmaf(-e1, u, e2), 0.f), 0.f));
    if constexpr (CLUSTER && ANY) cta_part_sync(t);  // see Rows
    fetch(rows.stage, row + kFwdStages * t.step);
    const float s0 = ex.slot[turns.turn][all.from].x;
    float z = 0.f, sq = 0.f, zq[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i) {
      zq[i] = 0.f;
      if (mq[i] > 0.f) {
        const float4 o = ex.slot[turns.turn][all.from + all.first + 32 * i];
        zq[i] = (o.x - s0) + o.y;
        sq += o.z;
      }
      z = fmaf(mq[i], zq[i], z);
    }
    turns.next();
    z = over(all.sum(z), n, inv_n);
#pragma unroll
    for (int i = 0; i < Q; ++i) sq = fmaf(mq[i] * (zq[i] - z), zq[i] - z, sq);
    const float var = all.sum(sq) * inv_n;
    float r = rsqrtf(fmaxf(var, 0.f) + f.eps);
    if (rows.failed || turns.failed) r = __int_as_float(0x7fc00000);  // something never came: say so in the result
    Pack<T, VEC> o[NV];
    normed<T, P, VEC, NV>(o, v, z - (s - s0), r, w, b);
    if constexpr (ANY)
      Outbox<T, NV>::store_row(mine + R::bytes(t.width), y + row * f.y_stride, o, t);
    else
      store_row(y + row * f.y_stride, o, t.lane, t.width, t.dim);
    if (f.stats && t.lane == 0 && t.first == 0) f.stats[row] = make_float4(s0, z, r, 0.f);
    rows.next();
  }
  rows.end();
  if constexpr (CLUSTER) cluster_sync();  // no CTA ends while another may still write to it
}

// Measured: 65536x4096 bfloat16 250 us (6.4 TB/s), 16384x8192 bfloat16 132 us
// (6.1 TB/s, 7 us of it the join), 16384x4096 float32 135 us (6.0 TB/s),
// 8192x16384 float32 in clusters of two 238 us (6.8 TB/s). Rows that start
// anywhere cost two shifts and a mask more for each vector: 20000x1003 float32
// 47-49 us (4.9-5.1 TB/s), 9000x5001 bfloat16 104 us (2.6 TB/s).
// dx, and the column sums of this CTA's rows: each thread keeps the sums of
// its columns while its group walks down the rows; at the end the groups of a
// CTA are joined in shared memory and the CTA writes one partial row of dw and
// db. Columns beyond the row read as dy = 0 and so add nothing to any sum.
template <typename T, typename P, int NV, bool CLUSTER, bool ANY>
__global__ void __launch_bounds__(kRowThreads) per_layer_norm_backward_group_kernel(const Bwd g) {
  constexpr int VEC = 16 / sizeof(T), kStages = kBwdStages<T, ANY>;
  __shared__ Exchange<CLUSTER> ex;
  __shared__ __align__(8) uint64_t bars[kMaxGroups][kStages];
  extern __shared__ __align__(16) unsigned char dyn[];
  using R = Rows<T, NV, 2, kStages, true, ANY>;
  using O = Outbox<T, NV>;
  const Group<CLUSTER> t(g.group_threads, VEC, NV, g.dim);
  unsigned char* own = dyn + t.index * (R::bytes(t.width) + (ANY ? O::bytes(t.width) : 0));
  R rows(own, bars[t.index], t.width);
  rows.begin(t.dim, t.lane, t.width);
  Turns<CLUSTER> turns;
  turns.begin(ex);
  const float inv_n = 1.f / (float)g.dim;
  int span = 1;
  while (span < t.warps && span < 16) span *= 2;
  const Array<T> in[2] = {Array<T>(g.x, g.x_stride, g.rows, g.dim, t.first),
                          Array<T>(g.dy, g.dy_stride, g.rows, g.dim, t.first)};
  T* dx = static_cast<T*>(g.dx) + t.first;
  if constexpr (CLUSTER)
    cluster_sync();
  else
    __syncthreads();
  per_wait_previous_grid();
  auto fetch = [&](int st, int64_t row) {
    rows.fetch(st, in, g.stats, row, t.dim, t.lane, t.width, row < g.rows);
  };
  for (int k = 0; k < kStages; ++k) fetch(k, t.base + k * t.step);
  if constexpr (ANY) cta_part_sync(t);  // values that were fetched one by one
  Pack<P, VEC> w[NV];
  load_columns(w, g.w ? static_cast<const P*>(g.w) + t.first : nullptr, 1.f, t.lane, t.width, t.dim);
  float2 aw[NV * VEC / 2], ab[NV * VEC / 2];
#pragma unroll
  for (int i = 0; i < NV * VEC / 2; ++i) aw[i] = ab[i] = per_both(0.f);
  for (int64_t row = t.base; row < g.rows; row += t.step) {
    float2 h[NV * VEC / 2], gv[NV * VEC / 2], e;
    rows.wait(in, row);
    const float4 st = rows.get_stats();
    const bool failed = rows.failed || turns.failed;
    const float r = failed ? __int_as_float(0x7fc00000) : st.z;  // NaN: something never came
    {
      Pack<T, VEC> qx[NV], qy[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        qx[k] = rows.get(0, k, t.dim, t.lane, t.width);
        qy[k] = rows.get(1, k, t.dim, t.lane, t.width);
      }
      e = backward_sums(qx, qy, w, st.x, st.y, r, h, gv, aw, ab);
    }
    const float v = exchange_split(ex, turns, t, span, lanes_sum_split<32>(e.x, e.y));
    if constexpr (CLUSTER && ANY) cta_part_sync(t);  // see Rows
    fetch(rows.stage, row + kStages * t.step);
    if (g.dx) {
      Pack<T, VEC> o[NV];
      backward_values<T, VEC, NV>(o, h, gv, join_split(v), inv_n,
                                  turns.failed ? __int_as_float(0x7fc00000) : r);
      if constexpr (ANY)
        O::store_row(own + R::bytes(t.width), dx + row * g.dx_stride, o, t);
      else
        store_row(dx + row * g.dx_stride, o, t.lane, t.width, t.dim);
    }
    rows.next();
  }
  rows.end();
  if constexpr (CLUSTER) cluster_sync();  // no CTA ends while another may still write to it
  if (!g.part) return;
  const int slice = t.width * NV * VEC;  // places of this CTA's part of the row
  if (CLUSTER || t.width == (int)blockDim.x) {
    float* part = g.part + t.base * 2 * g.places.padded + t.first;
    store_columns<VEC, NV>(part, aw, t.lane, t.width);
    store_columns<VEC, NV>(part + g.places.padded, ab, t.lane, t.width);
  } else {
    float* sums = reinterpret_cast<float*>(dyn);  // [groups][2][padded], over the slots, all of them read
    __syncthreads();
    store_columns<VEC, NV>(sums + t.index * 2 * slice, aw, t.lane, t.width);
    store_columns<VEC, NV>(sums + t.index * 2 * slice + slice, ab, t.lane, t.width);
    __syncthreads();
    add_groups(g.part + (int64_t)blockIdx.x * 2 * slice, sums, blockDim.x / t.width, slice);
  }
}

// ---- rows of any length: one CTA per row, the row read three times (from
// L2 after the first). Rows of more than 65,536 to 131,072 values only. The
// loads of single values in flight bound it, so the launch bounds ask for the
// registers of 6 and 8 CTAs an SM (3000x303201 float32 forward 3.79 ms, with 5
// CTAs 4.38; 1000x140001 half backward 0.72 ms, with 6 CTAs 1.02). 512x200000
// float32: 566 us forward (1.4 TB/s), 914 us backward (1.3 TB/s); a single row
// of a million takes 1.2 ms, for which one CTA has no more loads to offer.

// Sums of f(i) = (a, b) over i = first, first + step, ... below end. A sum of
// millions of terms in float32 rounds each of them to the sum's own step (a row
// of 2^27 equal squares came out 0.7 % off), so float32 takes kRun terms at a
// time and float64 the rest.
constexpr int kRun = 32;
template <typename F>
__device__ __forceinline__ double2 long_sums(int64_t first, int64_t step, int64_t end, F f) {
  double2 sum = make_double2(0.0, 0.0);
  int64_t i = first;
  float2 v;
  for (; i + (kRun - 1) * step < end; sum.x += (double)v.x, sum.y += (double)v.y) {
    v = per_both(0.f);
#pragma unroll 8
    for (int k = 0; k < kRun; ++k, i += step) f(i, v);
  }
  for (v = per_both(0.f); i < end; i += step) f(i, v);
  sum.x += (double)v.x;
  sum.y += (double)v.y;
  return sum;
}

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads, 6) per_layer_norm_long_kernel(const Fwd f) {
  per_wait_previous_grid();
  const double n = (double)f.dim;
  const P* w = static_cast<const P*>(f.w);
  const P* b = static_cast<const P*>(f.b);
  for (int64_t row = blockIdx.x; row < f.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(f.x) + row * f.x_stride;
    T* y = static_cast<T*>(f.y) + row * f.y_stride;
    const double2 all = long_sums(threadIdx.x, kThreads, f.dim,
                                  [&](int64_t c, float2& v) { v.x += per_to_f32(x[c]); });
    const float s = (float)(block_sum2(all.x, 0.0).x / n);
    const double2 d = long_sums(threadIdx.x, kThreads, f.dim, [&](int64_t c, float2& v) {
      const float d = per_to_f32(x[c]) - s;
      v.x += d;
      v.y = fmaf(d, d, v.y);
    });
    const double2 t = block_sum2(d.x, d.y);
    const double off = t.x / n;
    const float shift = (float)off;
    const float r = rsqrtf((float)fmax(t.y / n - off * off, 0.0) + f.eps);
    for (int64_t c = threadIdx.x; c < f.dim; c += kThreads) {
      float h = (per_to_f32(x[c]) - s - shift) * r;
      if (w) h *= per_to_f32(w[c]);
      if (b) h += per_to_f32(b[c]);
      y[c] = per_from_f32<T>(h);
    }
    if (f.stats && threadIdx.x == 0) f.stats[row] = make_float4(s, shift, r, 0.f);
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kThreads, 8) per_layer_norm_dx_long_kernel(const Bwd g) {
  per_wait_previous_grid();
  const double n = (double)g.dim;
  const P* w = static_cast<const P*>(g.w);
  for (int64_t row = blockIdx.x; row < g.rows; row += gridDim.x) {
    const T* x = static_cast<const T*>(g.x) + row * g.x_stride;
    const T* dy = static_cast<const T*>(g.dy) + row * g.dy_stride;
    T* dx = static_cast<T*>(g.dx) + row * g.dx_stride;
    const float4 st = g.stats[row];
    const float hi = st.x, lo = st.y, r = st.z;
    const double2 sums = long_sums(threadIdx.x, kThreads, g.dim, [&](int64_t c, float2& v) {
      const float h = (per_to_f32(x[c]) - hi - lo) * r;
      const float gv = per_to_f32(dy[c]) * (w ? per_to_f32(w[c]) : 1.f);
      v.x += gv;
      v.y = fmaf(gv, h, v.y);
    });
    const double2 t = block_sum2(sums.x, sums.y);
    const float c1 = (float)(t.x / n), c2 = (float)(t.y / n);
    for (int64_t c = threadIdx.x; c < g.dim; c += kThreads) {
      const float h = (per_to_f32(x[c]) - hi - lo) * r;
      const float gv = per_to_f32(dy[c]) * (w ? per_to_f32(w[c]) : 1.f);
      dx[c] = per_from_f32<T>(r * (gv - c1 - h * c2));
    }
  }
}

// Column sums of one split of the rows: thread = column.
template <typename T>
__global__ void __launch_bounds__(kThreads, 8) per_layer_norm_dw_long_kernel(const Bwd g) {
  per_wait_previous_grid();
  const int tiles = (g.dim - 1) / kThreads + 1;
  const int tile = blockIdx.x % tiles, split = blockIdx.x / tiles;
  const int64_t c = (int64_t)tile * kThreads + threadIdx.x;
  if (c >= g.dim) return;
  const T* x = static_cast<const T*>(g.x) + c;
  const T* dy = static_cast<const T*>(g.dy) + c;
  const double2 sums = long_sums(split, g.splits, g.rows, [&](int64_t row, float2& v) {
    const float4 st = g.stats[row];
    const float d = per_to_f32(dy[row * g.dy_stride]);
    v.x = fmaf(d, (per_to_f32(x[row * g.x_stride]) - st.x - st.y) * st.z, v.x);
    v.y += d;
  });
  g.part[(int64_t)split * 2 * g.places.padded + c] = (float)sums.x;
  g.part[((int64_t)split * 2 + 1) * g.places.padded + c] = (float)sums.y;
}

// dw and db from the partial rows. A CTA adds 32 places: 8 threads take four
// each of a partial row, its 64 such teams every 64th row, so that most lists
// are read in a few loads per thread; the teams' sums are added in order.
constexpr int kJoinThreads = 512;
template <typename P>
__global__ void __launch_bounds__(kJoinThreads) per_layer_norm_join_kernel(const Bwd g) {
  __shared__ __align__(16) float s[kJoinThreads / 32][32];  // stored by float4
  per_wait_previous_grid();
  const int quad = threadIdx.x & 7, team = threadIdx.x >> 3;
  const int64_t all = 2 * (int64_t)g.places.padded;
  const int64_t at = (int64_t)blockIdx.x * 32 + quad * 4;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (at < all) {
#pragma unroll 4
    for (int k = team; k < g.splits; k += kJoinThreads / 8) {
      const float4 u = *reinterpret_cast<const float4*>(g.part + k * all + at);
      v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
    }
  }
#pragma unroll
  for (int o = 8; o < 32; o <<= 1) {
    v.x += __shfl_xor_sync(PER_FULL_MASK, v.x, o);
    v.y += __shfl_xor_sync(PER_FULL_MASK, v.y, o);
    v.z += __shfl_xor_sync(PER_FULL_MASK, v.z, o);
    v.w += __shfl_xor_sync(PER_FULL_MASK, v.w, o);
  }
  if ((threadIdx.x & 31) < 8) *reinterpret_cast<float4*>(&s[threadIdx.x >> 5][quad * 4]) = v;
  __syncthreads();
  const int64_t p = (int64_t)blockIdx.x * 32 + threadIdx.x;
  if (threadIdx.x >= 32 || p >= all) return;
  float sum = s[0][threadIdx.x];
#pragma unroll
  for (int q = 1; q < kJoinThreads / 32; ++q) sum += s[q][threadIdx.x];
  const bool second = p >= g.places.padded;
  const int c = column_at(g.places, (int)(second ? p - g.places.padded : p));
  void* out = second ? g.db : g.dw;
  if (out && c < g.dim) static_cast<P*>(out)[c] = per_from_f32<P>(sum);
}

int launch(const void* fn, int64_t grid, int threads, size_t smem, const void* arg,
           cudaStream_t stream, int cluster = 1) {
  void* args[] = {const_cast<void*>(arg)};
  const cudaError_t e = cluster > 1
                            ? per_launch_cluster(fn, (unsigned)grid, threads, smem, cluster, stream, args)
                            : per_launch(fn, (unsigned)grid, threads, smem, stream, args, false);
  return e == cudaSuccess ? PER_OK : per_record_cuda(e);
}

int64_t row_grid(int64_t rows) { return rows < 65535 ? rows : 65535; }

int sm_count() {
  static int sms[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (!sms[dev]) {
    int v = 0;
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) v = 148;
    sms[dev] = v;
  }
  return sms[dev];
}

// Row splits of the column sums of long rows, for some 8 CTAs an SM: half of that
// takes 1,765 us for 2000x131072 bfloat16 backward instead of 1,400; four times
// as many take 0 to 11 % less, and as many times the partial rows.
int splits_of(int64_t rows, int64_t dim) {
  const int64_t tiles = (dim - 1) / kThreads + 1;
  int64_t s = 1184 / tiles;
  if (s > rows) s = rows;
  return s < 1 ? 1 : (int)s;
}

// How a row is laid over threads: `lanes` of a warp, or a group of `threads`
// in each of `ctas` CTAs (lanes 0), with `nv` vectors per thread. ctas 0: too
// long for registers.
struct Shape {
  int lanes, nv, threads, ctas;
};

// Most vectors of a row that a thread holds. The sums over a row cost a thread
// some 100 instructions whatever it holds, so it should hold much; statistics,
// weights and (backward) two column sums per value have to fit its registers.
constexpr int kFwdVectors = 4;
template <typename T>
constexpr int kBwdVectors = sizeof(T) == 2 ? 2 : 4;
// Single values, in a warp: rows that start anywhere are faster so than by
// windows as long as a warp can hold them (50000x333 half 21 us against 40
// forward, 40 against 55 backward; 8191x1001 12 against 15 and 19 against 31;
// float32 only up to 16 a lane: 20000x1003 backward 54 against 47).
template <typename T>
constexpr int kSingles = sizeof(T) == 2 ? 32 : 16;

// Rows that a warp can hold stay in it, which needs no barrier; longer ones
// take a group of warps, and beyond one CTA a cluster of up to 8. In a warp,
// rows that start anywhere go by single values (vec 1).
Shape shape_of(int64_t dim, int vec, bool any, bool split, int singles, int full, int most_threads,
               int warp_threads) {
  const int small = any ? 4 : 1, most = any ? singles : full;
  const int64_t w = any ? dim : (dim + vec - 1) / vec;
  for (int lanes = 4; lanes <= 32; lanes *= 2)
    if (w <= lanes * small) return {lanes, small, warp_threads, 1};
  for (int nv = 2 * small; nv <= most; nv *= 2)
    if (w <= 32 * nv) return {32, nv, warp_threads, 1};
  const int64_t v = (dim + vec - 1) / vec;
  int ctas = 1;
  while (v > (int64_t)ctas * most_threads * full)
    if ((ctas *= 2) > kMaxCluster) return {0, 0, 0, 0};
  const auto threads = [&](int nv) { return (v + ctas * nv * 32 - 1) / (ctas * nv * 32) * 32; };
  // An SM has registers for some 512 threads: CTAs of more than 256 leave some
  // of them idle. Twice the CTAs then. Forward, with and without, us: 16384x5000 float32 (320 threads) 114 and 136,
  // 8192x10000 133 and 149, 8192x12288 bfloat16 (384) 79 and 90, but 16384x6000
  // float32 (384) 158 and 150, 8192x12000 198 and 163; from 448 threads on the
  // wider cluster costs more (8192x7600 float32 92 and 88, 4096x30000 266 and
  // 206). Rows that start anywhere, both passes, up to a full CTA: 3000x20001
  // bfloat16 backward 157 and 195, 8192x4201 float32 82 and 92, 106 and 119, but
  // 8192x6001 114 and 100, 136 and 128. In the backward pass of whole vectors the
  // wider cluster costs more (10000 float32 values: 153 -> 179 us).
  while (split && threads(full) > 256 && threads(full) < (any ? kRowThreads + 1 : 448) &&
         ctas < kMaxCluster)
    ctas *= 2;
  // As many vectors a thread as there may be, or half, where that leaves fewer
  // places empty: rows of 513 to 768 values, or twice that in the forward pass of
  // 16-bit ones. Few rows gain, us with half and with all: 512x768 float32 2.2
  // and 2.4 forward, 256x768 4.1 and 5.1 backward, 512x1200 bfloat16 2.3 and 2.8
  // forward. Of many, backward, 65536x768 float32 gains (95 and 102) and 65536x516
  // loses (80 and 74); forward they lose (8192x768 14.3 and 11.3, 65536x768 98
  // and 72).
  const int nv = threads(full / 2) <= most_threads && 8 * threads(full / 2) <= 13 * threads(full)
                     ? full / 2 : full;
  return {0, nv, (int)threads(nv), ctas};
}

// warp<T, P, VEC, NV, LANES>(...) or group<T, P, NV, CLUSTER, ANY>(...) for the
// shape, into rc; false where there is none. Half of F vectors a thread are for
// rows of up to 48 F vectors: never a cluster's, and where rows start anywhere
// only if these are more than a warp holds in single values.
#define PER_NORM_SHAPE(s, rc, warp, group, T, P, ANY, FULL, ...)                               \
  [&]() -> bool {                                                                              \
    constexpr int V = ANY ? 1 : 16 / sizeof(T), S = ANY ? 4 : 1, F = FULL;                     \
    constexpr int W = ANY ? kSingles<T> : F;                                                   \
    if (s.lanes == 4) return rc = warp<T, P, V, S, 4>(s, __VA_ARGS__), true;                   \
    if (s.lanes == 8) return rc = warp<T, P, V, S, 8>(s, __VA_ARGS__), true;                   \
    if (s.lanes == 16) return rc = warp<T, P, V, S, 16>(s, __VA_ARGS__), true;                 \
    if (s.lanes == 32 && s.nv == S) return rc = warp<T, P, V, S, 32>(s, __VA_ARGS__), true;    \
    if (s.lanes == 32 && s.nv == 2 * S)                                                        \
      return rc = warp<T, P, V, 2 * S, 32>(s, __VA_ARGS__), true;                              \
    if constexpr (W >= 4 * S)                                                                  \
      if (s.lanes == 32 && s.nv == 4 * S)                                                      \
        return rc = warp<T, P, V, 4 * S, 32>(s, __VA_ARGS__), true;                            \
    if constexpr (W >= 8 * S)                                                                  \
      if (s.lanes == 32) return rc = warp<T, P, V, 8 * S, 32>(s, __VA_ARGS__), true;           \
    if (s.ctas == 1 && s.nv == F)                                                              \
      return rc = group<T, P, F, false, ANY>(s, __VA_ARGS__), true;                            \
    if constexpr (!ANY || 3 * F * 16 / (int)sizeof(T) > 2 * W)                                 \
      if (s.ctas == 1) return rc = group<T, P, F / 2, false, ANY>(s, __VA_ARGS__), true;       \
    if (s.ctas > 1) return rc = group<T, P, F, true, ANY>(s, __VA_ARGS__), true;               \
    return false;                                                                              \
  }()

bool aligned(const void* p, int64_t stride, size_t elem) {
  return (uintptr_t)p % 16 == 0 && (stride * (int64_t)elem) % 16 == 0;
}

// CTAs (or clusters) that share `rows`: what is co-resident, or fewer.
int row_ctas(const void* fn, const Shape& s, int threads, size_t smem, int64_t rows, int64_t most,
             int64_t* out) {
  int rc = per_set_smem(fn, smem);
  if (rc) return rc;
  int ctas = 0;
  rc = per_coresident_clusters(fn, threads, smem, s.ctas, &ctas);
  if (rc) return rc;
  const int64_t per_cta = threads / (s.lanes ? s.lanes : s.threads);
  int64_t grid = (rows - 1) / per_cta + 1;
  if (grid > ctas) grid = ctas;
  if (most > 0 && grid > most) grid = most;
  *out = grid;
  return PER_OK;
}

template <typename T, typename P, int VEC, int NV, int LANES>
int forward_warp(const Shape& s, const Fwd& f, cudaStream_t stream) {
  const void* fn = (const void*)per_layer_norm_warp_kernel<T, P, VEC, NV, LANES>;
  const size_t smem = Ring<T, VEC, NV, kWarpStages>::kBytes * s.threads;
  int64_t grid = 0;
  const int rc = row_ctas(fn, s, s.threads, smem, f.rows, 0, &grid);
  return rc ? rc : launch(fn, grid, s.threads, smem, &f, stream);
}

template <typename T, typename P, int NV, bool CLUSTER, bool ANY>
int forward_group(const Shape& s, const Fwd& in, cudaStream_t stream) {
  Fwd f = in;
  f.group_threads = s.threads;
  const void* fn = (const void*)per_layer_norm_group_kernel<T, P, NV, CLUSTER, ANY, kRowThreads>;
  if constexpr (kWide<T, NV>)
    if (s.threads <= 192)
      fn = (const void*)per_layer_norm_group_kernel<T, P, NV, CLUSTER, ANY, kWideThreads>;
  // rows of few threads share a CTA of about 128
  const int groups = CLUSTER || s.threads > 64 ? 1 : 128 / s.threads;
  const size_t smem = groups * (Rows<T, NV, 1, kFwdStages, false, ANY>::bytes(s.threads) +
                                (ANY ? Outbox<T, NV>::bytes(s.threads) : 0));
  int64_t grid = 0;
  const int rc = row_ctas(fn, s, s.threads * groups, smem, f.rows, 0, &grid);
  return rc ? rc : launch(fn, grid * s.ctas, s.threads * groups, smem, &f, stream, s.ctas);
}

template <typename T, typename P, bool ANY>
int forward_rows(const Fwd& f, cudaStream_t stream) {
  constexpr int FULL = kFwdVectors;
  const Shape s = shape_of(f.dim, 16 / sizeof(T), ANY, true, kSingles<T>, FULL, kRowThreads, 128);
  int rc = PER_OK;
  if (PER_NORM_SHAPE(s, rc, forward_warp, forward_group, T, P, ANY, FULL, f, stream)) return rc;
  return launch((const void*)per_layer_norm_long_kernel<T, P>, row_grid(f.rows), kThreads, 0, &f,
                stream);
}

template <typename T, typename P>
int forward(const Fwd& f, cudaStream_t stream) {
  if (f.dim % (16 / sizeof(T)) == 0 && aligned(f.x, f.x_stride, sizeof(T)) &&
      aligned(f.y, f.y_stride, sizeof(T)) && aligned(f.w, 0, 1) && aligned(f.b, 0, 1))
    return forward_rows<T, P, false>(f, stream);
  return forward_rows<T, P, true>(f, stream);
}

// Most partial rows of dw and db: the workspace is sized before the pointers'
// alignment, and with it the kernel, is known. No less than the CTAs that an SM
// holds of any of them, so that it limits no grid (half and double of these
// measure the same at nine sizes from 65536x32 to 4096x8192).
int64_t most_partials(int64_t rows, int64_t dim) {
  const int64_t most = (int64_t)sm_count() * (dim <= 512 ? 8 : dim <= 2048 ? 4 : 2);
  return rows < most ? rows : most;
}

Bwd::Places long_places(int32_t dim) {
  const int32_t padded = (dim - 1) / 4 * 4 + 4;
  return {padded, padded, 1, 1};
}

// The order of the columns in a partial row.
Bwd::Places places_of(const Shape& s, int vec) {
  const int slice = (s.lanes ? s.lanes : s.threads) * s.nv * vec;
  return {s.ctas * slice, slice, s.lanes ? s.lanes : s.threads, vec};
}

// The row kernel, then the join of its partial rows where columns are wanted.
template <typename P>
int backward_run(const void* fn, const Shape& s, int threads, size_t smem, Bwd g, cudaStream_t stream) {
  int64_t grid = 0;
  int rc = row_ctas(fn, s, threads, smem, g.rows, most_partials(g.rows, g.dim), &grid);
  if (rc) return rc;
  const bool columns = g.dw || g.db;
  if (!columns) g.part = nullptr;
  rc = launch(fn, grid * s.ctas, threads, smem, &g, stream, s.ctas);
  if (rc || !columns) return rc;
  g.splits = (int32_t)grid;
  return launch((const void*)per_layer_norm_join_kernel<P>, (2 * (int64_t)g.places.padded - 1) / 32 + 1,
                kJoinThreads, 0, &g, stream);
}

template <typename T, typename P, int VEC, int NV, int LANES>
int backward_warp(const Shape& s, const Bwd& in, cudaStream_t stream) {
  Bwd g = in;
  g.places = places_of(s, VEC);
  const size_t ring = Ring<T, VEC, 2 * NV, kWarpStages>::kBytes * s.threads;
  const size_t sums = (size_t)(s.threads / 32) * 2 * g.places.padded * 4;
  const void* fn = (const void*)per_layer_norm_backward_warp_kernel<T, P, VEC, NV, LANES>;
  // Few rows (up to two turns of 16 CTAs): one launch, a cluster that joins its
  // own sums. In an eager step that saves 2 us of host time (256x256 float32: 62
  // to 60 us); longer ones would wait longer for 16 CTAs than a launch takes.
  const int64_t turn = s.threads / LANES;
  const size_t joined = sums + (size_t)2 * g.places.padded * 4;
  if ((g.dw || g.db) && g.rows <= 2 * kJoinCtas * turn && joined <= 100 * 1024) {
    int ctas = 1;
    while (ctas < kJoinCtas && ctas * turn < g.rows) ctas *= 2;
    const size_t smem = ring > joined ? ring : joined;
    const int rc = per_set_smem(fn, smem);
    if (rc) return rc;
    if (ctas <= 8 || per_cluster_fits(fn, s.threads, smem, ctas)) {
      g.joined = 1;
      g.part = nullptr;
      return launch(fn, ctas, s.threads, smem, &g, stream, ctas);
    }
  }
  return backward_run<P>(fn, s, s.threads, ring > sums ? ring : sums, g, stream);
}

template <typename T, typename P, int NV, bool CLUSTER, bool ANY>
int backward_group(const Shape& s, const Bwd& in, cudaStream_t stream) {
  Bwd g = in;
  g.group_threads = s.threads;
  // several groups share a CTA and its partial row
  int groups = CLUSTER ? 1 : kRowThreads / s.threads;
  groups = groups > kMaxGroups ? kMaxGroups : groups;
  size_t smem = groups * (Rows<T, NV, 2, kBwdStages<T, ANY>, true, ANY>::bytes(s.threads) +
                          (ANY ? Outbox<T, NV>::bytes(s.threads) : 0));
  g.places = places_of(s, 16 / sizeof(T));
  const size_t sums = groups > 1 ? (size_t)groups * 2 * g.places.padded * 4 : 0;
  smem = smem > sums ? smem : sums;
  return backward_run<P>((const void*)per_layer_norm_backward_group_kernel<T, P, NV, CLUSTER, ANY>, s,
                         s.threads * groups, smem, g, stream);
}

template <typename T, typename P, bool ANY>
int backward_rows(const Bwd& in, cudaStream_t stream) {
  constexpr int FULL = kBwdVectors<T>;
  const Shape s = shape_of(in.dim, 16 / sizeof(T), ANY, ANY, kSingles<T>, FULL, kRowThreads, 256);
  int rc = PER_OK;
  if (PER_NORM_SHAPE(s, rc, backward_warp, backward_group, T, P, ANY, FULL, in, stream)) return rc;
  Bwd g = in;
  g.splits = splits_of(g.rows, g.dim);
  g.places = long_places(g.dim);
  if (g.dx)
    rc = launch((const void*)per_layer_norm_dx_long_kernel<T, P>, row_grid(g.rows), kThreads, 0,
                &g, stream);
  if (rc || (!g.dw && !g.db)) return rc;
  const int64_t tiles = (g.dim - 1) / kThreads + 1;
  rc = launch((const void*)per_layer_norm_dw_long_kernel<T>, tiles * g.splits, kThreads, 0, &g,
              stream);
  if (rc) return rc;
  return launch((const void*)per_layer_norm_join_kernel<P>, (2 * (int64_t)g.places.padded - 1) / 32 + 1,
                kJoinThreads, 0, &g, stream);
}

template <typename T, typename P>
int backward(const Bwd& g, cudaStream_t stream) {
  if (g.dim % (16 / sizeof(T)) == 0 && aligned(g.x, g.x_stride, sizeof(T)) &&
      aligned(g.dy, g.dy_stride, sizeof(T)) && aligned(g.dx, g.dx_stride, sizeof(T)) &&
      aligned(g.w, 0, 1))
    return backward_rows<T, P, false>(g, stream);
  return backward_rows<T, P, true>(g, stream);
}

// Bytes of partial rows, whichever kernel the pointers' alignment asks for.
template <typename T, typename P>
int64_t backward_bytes(const per_norm_t& n) {
  if (n.rows == 0) return 0;
  constexpr int VEC = 16 / sizeof(T), FULL = kBwdVectors<T>;
  int64_t most = 0;
  for (const bool any : {false, true}) {
    if (!any && n.dim % VEC) continue;
    const Shape s = shape_of(n.dim, VEC, any, any, kSingles<T>, FULL, kRowThreads, 256);
    const int64_t bytes =
        s.ctas ? most_partials(n.rows, n.dim) * places_of(s, any && s.lanes ? 1 : VEC).padded
               : (int64_t)splits_of(n.rows, n.dim) * long_places((int32_t)n.dim).padded;
    most = bytes > most ? bytes : most;
  }
  return most * 2 * 4;
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
                          const void* bias, void* y, int64_t y_stride, float* stats,
                          cudaStream_t stream) {
  const Fwd f{x, weight, bias, y, reinterpret_cast<float4*>(stats), n.rows, x_stride, y_stride, (int32_t)n.dim, n.eps, 0};
  return PER_NORM_TYPES(n, forward, f, stream);
}

int64_t per_layer_norm_backward_bytes(const per_norm_t& n) {
  return PER_NORM_TYPES(n, backward_bytes, n);
}

int per_launch_layer_norm_backward(const per_norm_t& n, const void* dy, int64_t dy_stride,
                                   const void* x, int64_t x_stride, const void* weight,
                                   const float* stats, void* dx,
                                   int64_t dx_stride, void* dweight, void* dbias, void* workspace,
                                   cudaStream_t stream) {
  const Bwd g{dy, x, weight, reinterpret_cast<const float4*>(stats), dx, dweight, dbias,
              static_cast<float*>(workspace),
              n.rows, dy_stride, x_stride, dx_stride, (int32_t)n.dim, 0, 0, 0, {}};
  return PER_NORM_TYPES(n, backward, g, stream);
}
