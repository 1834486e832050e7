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
  int32_t group_threads;  // of a row that spans warps
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

// The values of a thread, NV vectors of VEC, as pairs 0 .. NV VEC / 2. WORDS:
// taken from and put into whole 32-bit words, which costs fewer instructions;
// the forward kernel goes by single values, because from words the compiler
// keeps weight and bias unpacked across rows and spills (65536x4096 bfloat16:
// 178 us by values, 203 by words; backward 304 us by values, 290 by words).
template <bool WORDS, typename T, int VEC, int NV>
__device__ __forceinline__ float2 get2(const Pack<T, VEC> (&p)[NV], int i) {
  if constexpr (WORDS && sizeof(T) == 2 && VEC > 1)
    return per_unpack<T>(reinterpret_cast<const uint32_t*>(&p[2 * i / VEC])[i % (VEC / 2)]);
  else
    return make_float2(per_to_f32(p[2 * i / VEC].v[2 * i % VEC]),
                       per_to_f32(p[(2 * i + 1) / VEC].v[(2 * i + 1) % VEC]));
}
template <bool WORDS, typename T, int VEC, int NV>
__device__ __forceinline__ void set2(Pack<T, VEC> (&p)[NV], int i, float2 f) {
  if constexpr (WORDS && sizeof(T) == 2 && VEC > 1) {
    reinterpret_cast<uint32_t*>(&p[2 * i / VEC])[i % (VEC / 2)] = per_pack<T>(f);
  } else {
    p[2 * i / VEC].v[2 * i % VEC] = per_from_f32<T>(f.x);
    p[(2 * i + 1) / VEC].v[(2 * i + 1) % VEC] = per_from_f32<T>(f.y);
  }
}

// The threads of a row: LANES of them (a power of two, several rows per
// warp), a group of warps (LANES 0, one or several groups in a CTA), or a
// cluster of CTAs (LANES -1, rows too long for one). Thread `lane` of `width`
// holds the vectors lane, lane + width, ..., NV of them at most.
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

template <int LANES>
struct Row {
  int lane, width;     // of this thread in its row
  int64_t base, step;  // first row of this warp, rows between two of its turns
  int mine;            // this thread's row is base + mine
  int group;           // of this CTA's groups
  int warps;           // of a row that spans warps
  __device__ __forceinline__ explicit Row(int group_threads) {
    mine = group = 0;
    warps = 1;
    if constexpr (LANES > 0) {
      const int per_cta = blockDim.x / LANES;
      lane = threadIdx.x % LANES;
      width = LANES;
      base = (int64_t)blockIdx.x * per_cta + (threadIdx.x & ~31) / LANES;
      step = (int64_t)gridDim.x * per_cta;
      mine = (threadIdx.x & 31) / LANES;
    } else if constexpr (LANES == 0) {
      const int groups = blockDim.x / group_threads;
      group = threadIdx.x / group_threads;
      lane = threadIdx.x - group * group_threads;
      width = group_threads;
      base = (int64_t)blockIdx.x * groups + group;
      step = (int64_t)gridDim.x * groups;
      warps = width >> 5;
    } else {
      const int ctas = (int)cluster_size();
      lane = threadIdx.x + (int)(cluster_rank() * blockDim.x);
      width = blockDim.x * ctas;
      base = blockIdx.x / ctas;
      step = gridDim.x / ctas;
      warps = width >> 5;
    }
  }
};

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = (LANES > 0 ? LANES : 32) / 2; o; o >>= 1) v += __shfl_xor_sync(PER_FULL_MASK, v, o);
  return v;
}

// What the warps of a row hand to one another: each warp's words go to every
// CTA of the row, then one barrier. Two buffers by turns, so that one barrier
// per exchange is enough: a buffer is written again only after the barrier of
// the next exchange, which follows every read of it.
constexpr int kMaxCluster = 8;
constexpr int kRowThreads = 512;  // of a CTA whose warps share rows
template <int LANES>
struct Exchange {
  float4 slot[2][LANES == 0 ? kRowThreads / 32 : kRowThreads / 32 * kMaxCluster];
};

template <int LANES>
__device__ __forceinline__ void put(Exchange<LANES>& e, int turn, const Row<LANES>& t, float4 v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if constexpr (LANES == 0) {
    if (lane == 0) e.slot[turn][warp] = v;
    __syncwarp();
    asm volatile("bar.sync %0, %1;" ::"r"(t.group + 1), "r"(t.width) : "memory");
  } else {
    if (lane < (int)cluster_size()) {  // lane = the CTA that the warp's words go to
      const float4* at = &e.slot[turn][cluster_rank() * (blockDim.x >> 5) + warp];
      const uint32_t local = (uint32_t)__cvta_generic_to_shared(at);
      uint32_t remote;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(lane));
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(remote), "f"(v.x),
                   "f"(v.y), "f"(v.z), "f"(v.w)
                   : "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// The warps of a row as a lane sees them in an exchange: lane l reads warps
// l mod span, + 32, ...; a butterfly over `span` lanes then joins them all.
template <int LANES>
struct Warps {
  static constexpr int kReads = LANES == 0 ? 1 : kRowThreads / 32 * kMaxCluster / 32;
  int span, first, from;
  __device__ __forceinline__ explicit Warps(const Row<LANES>& t) {
    span = 1;
    while (span < t.warps && span < 32) span *= 2;
    first = threadIdx.x & (span - 1);
    from = LANES == 0 ? t.group * t.warps : 0;
  }
  __device__ __forceinline__ float sum(float v) const {
    for (int o = span >> 1; o; o >>= 1) v += __shfl_xor_sync(PER_FULL_MASK, v, o);
    return v;
  }
};

// A thread's own copies on their way into shared memory, STAGES rows ahead:
// it waits for and reads only what it has copied itself, so no barrier is
// needed. 16-byte vectors go by cp.async; single values are fetched into
// registers one row ahead. Where `in` is false the vector reads as zeros.
template <typename T, int VEC, int NV, int STAGES>
struct Ring {
  static constexpr bool kAsync = VEC * sizeof(T) == 16;
  static constexpr int kStages = kAsync ? STAGES : 1;
  static constexpr size_t kBytes = kAsync ? STAGES * NV * 16 : 0;  // per thread
  uint32_t at;
  Pack<T, VEC> reg[kAsync ? 1 : NV];

  __device__ __forceinline__ explicit Ring(const void* smem) {
    at = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * 16;
  }
  // p is valid where `in` is true; base is always a valid address
  __device__ __forceinline__ void fetch(int stage, int k, const T* base, int64_t offset, bool in) {
    if constexpr (kAsync) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                       at + (stage * NV + k) * blockDim.x * 16),
                   "l"(in ? base + offset : base), "r"(in ? 16 : 0)
                   : "memory");
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) reg[k].v[j] = per_from_f32<T>(0.f);
      if (in) reg[k] = load<T, VEC>(base + offset);
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
      uint4 u;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                   : "r"(at + (stage * NV + k) * blockDim.x * 16)
                   : "memory");
      Pack<T, VEC> r;
      *reinterpret_cast<uint4*>(&r) = u;
      return r;
    } else {
      return reg[k];
    }
  }
};

// Before a CTA writes into another one's shared memory, that one has to run.
template <int LANES>
__device__ __forceinline__ void cluster_begins() {
  if constexpr (LANES < 0) {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
}

// weight (or its absence as 1, bias as 0) of this thread's columns
template <typename P, int VEC, int NV>
__device__ __forceinline__ void load_columns(Pack<P, VEC> (&w)[NV], const void* p, float absent,
                                             int lane, int width, int dim) {
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (lane + k * width) * VEC;
#pragma unroll
    for (int j = 0; j < VEC; ++j) w[k].v[j] = per_from_f32<P>(absent);
    if (c < dim && p) w[k] = load<P, VEC>(static_cast<const P*>(p) + c);
  }
}

constexpr int kFwdStages = 3;
constexpr int kBwdStages = 3;

// ---- forward, rows in registers
template <typename T, typename P, int VEC, int NV, int LANES>
__global__ void __launch_bounds__(LANES > 0 ? 128 : kRowThreads) per_layer_norm_kernel(const Fwd f) {
  __shared__ Exchange<LANES> ex;
  extern __shared__ __align__(16) unsigned char dyn[];
  const Row<LANES> t(blockDim.x);
  using R = Ring<T, VEC, NV, kFwdStages>;
  R ring(dyn);
  int turn = 0, stage = 0;
  constexpr int E2 = NV * VEC / 2;
  const float n = (float)f.dim, inv_n = 1.f / n;
  const T* x = static_cast<const T*>(f.x);
  T* y = static_cast<T*>(f.y);

  // values of a warp (of a row that spans warps): this one's, and those of the
  // warps that this lane reads in an exchange
  const Warps<LANES> all(t);
  auto values_of = [&](int warp) {
    int v = 0;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int left = f.dim / VEC - warp * 32 - k * t.width;
      v += left < 0 ? 0 : left > 32 ? 32 : left;
    }
    return (float)(v * VEC);
  };
  constexpr int Q = Warps<LANES>::kReads;
  float own = n, mq[Q];
  if constexpr (LANES <= 0) {
    own = values_of(t.lane >> 5);
#pragma unroll
    for (int i = 0; i < Q; ++i)
      mq[i] = all.first + 32 * i < t.warps ? values_of(all.first + 32 * i) : 0.f;
  }
  const float inv_own = own > 0.f ? 1.f / own : 0.f;

  cluster_begins<LANES>();
  per_wait_previous_grid();
  auto fetch = [&](int st, int64_t row) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (t.lane + k * t.width) * VEC;
      ring.fetch(st, k, x, row * f.x_stride + c, row < f.rows && c < f.dim);
    }
    R::commit();
  };
#pragma unroll
  for (int k = 0; k < R::kStages; ++k) fetch(k, t.base + t.mine + k * t.step);
  Pack<P, VEC> w[NV], b[NV];
  load_columns(w, f.w, 1.f, t.lane, t.width, f.dim);
  load_columns(b, f.b, 0.f, t.lane, t.width, f.dim);
  for (int64_t base = t.base; base < f.rows; base += t.step) {
    const int64_t row = base + t.mine;
    float2 v[E2];
    float2 a = per_both(0.f);
    R::wait();
    {
      Pack<T, VEC> q[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) q[k] = ring.get(stage, k);
#pragma unroll
      for (int i = 0; i < E2; ++i) {
        v[i] = get2<false>(q, i);
        a = per_add2(a, v[i]);
      }
    }
    fetch(stage, row + R::kStages * t.step);
    stage = stage + 1 == R::kStages ? 0 : stage + 1;
    // distances from a first mean: the row's, or (rows that span warps) the
    // warp's; columns beyond the row, read as 0, stay at 0
    const float s = over(lanes_sum<LANES>(a.x + a.y), own, inv_own);
    float2 d1 = per_both(0.f), d2 = per_both(0.f);
#pragma unroll
    for (int i = 0; i < E2; ++i) {
      const bool in0 = (t.lane + 2 * i / VEC * t.width) * VEC < f.dim;
      const bool in1 = VEC > 1 ? in0 : (t.lane + (2 * i + 1) * t.width) < f.dim;
      v[i] = per_add2(v[i], make_float2(in0 ? -s : 0.f, in1 ? -s : 0.f));
      d1 = per_add2(d1, v[i]);
      d2 = per_fma2(v[i], v[i], d2);
    }
    const float e1 = lanes_sum<LANES>(d1.x + d1.y);
    const float e2 = lanes_sum<LANES>(d2.x + d2.y);
    float shift, var;  // h = (v - shift) r
    double mean;
    if constexpr (LANES > 0) {
      shift = over(e1, n, inv_n);
      var = fmaf(-shift, shift, e2 * inv_n);
      mean = (double)s + (double)shift;
    } else {
      // Warp q of m_q values: mean s_q + u_q with u_q = d1_q / m_q, squares around it
      // d2_q - d1_q u_q. Seen from s_0 its mean lies at z_q; the row's at z = sum m_q z_q / n,
      // and the row's squares are the warps' plus m_q (z_q - z)^2 each.
      const float u = e1 * inv_own;
      put<LANES>(ex, turn, t, make_float4(s, u, fmaxf(fmaf(-e1, u, e2), 0.f), 0.f));
      const float s0 = ex.slot[turn][all.from].x;
      float z = 0.f, sq = 0.f, zq[Q];
#pragma unroll
      for (int i = 0; i < Q; ++i) {
        zq[i] = 0.f;
        if (mq[i] > 0.f) {
          const float4 o = ex.slot[turn][all.from + all.first + 32 * i];
          zq[i] = (o.x - s0) + o.y;
          sq += o.z;
        }
        z = fmaf(mq[i], zq[i], z);
      }
      turn ^= 1;
      z = over(all.sum(z), n, inv_n);
#pragma unroll
      for (int i = 0; i < Q; ++i) sq = fmaf(mq[i] * (zq[i] - z), zq[i] - z, sq);
      var = all.sum(sq) * inv_n;
      shift = z - (s - s0);
      mean = (double)s0 + (double)z;
    }
    const float r = rsqrtf(fmaxf(var, 0.f) + f.eps);
    const float2 r2 = per_both(r), c2 = per_both(-shift * r);
    if (row < f.rows) {
      Pack<T, VEC> o[NV];
#pragma unroll
      for (int i = 0; i < E2; ++i)
        set2<false>(o, i, per_fma2(per_fma2(v[i], r2, c2), get2<false>(w, i), get2<false>(b, i)));
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (t.lane + k * t.width) * VEC;
        if (c < f.dim) store<T, VEC>(y + row * f.y_stride + c, o[k]);
      }
      if (f.mean && t.lane == 0) {
        f.mean[row] = mean;
        f.rstd[row] = r;
      }
    }
  }
}

// ---- backward, rows in registers: dx, and the column sums of this CTA's
// rows. Each thread keeps the sums of its columns while its group walks down
// the rows; at the end the groups of a CTA are joined in shared memory and
// the CTA writes one partial row of dw and db. Columns beyond the row, and
// rows beyond the last, read as dy = 0 and so add nothing to any sum.
template <typename T, typename P, int VEC, int NV, int LANES>
__global__ void __launch_bounds__(LANES > 0 ? 256 : kRowThreads)
    per_layer_norm_backward_kernel(const Bwd g) {
  __shared__ Exchange<LANES> ex;
  extern __shared__ __align__(16) unsigned char dyn[];
  const Row<LANES> t(g.group_threads);
  using R = Ring<T, VEC, 2 * NV, kBwdStages>;
  R ring(dyn);
  int turn = 0, stage = 0;
  constexpr int E2 = NV * VEC / 2;
  const float inv_n = 1.f / (float)g.dim;
  const Warps<LANES> all(t);
  const T* x = static_cast<const T*>(g.x);
  const T* dy = static_cast<const T*>(g.dy);
  T* dx = static_cast<T*>(g.dx);
  cluster_begins<LANES>();
  per_wait_previous_grid();
  auto fetch = [&](int st, int64_t row) {
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (t.lane + k * t.width) * VEC;
      const bool in = row < g.rows && c < g.dim;
      ring.fetch(st, k, x, row * g.x_stride + c, in);
      ring.fetch(st, NV + k, dy, row * g.dy_stride + c, in);
    }
    R::commit();
  };
  double nm = 0.0;
  float nr = 0.f;
  auto fetch_stats = [&](int64_t row) {
    if (row >= g.rows) return;
    nm = g.mean[row];
    nr = g.rstd[row];
  };
#pragma unroll
  for (int k = 0; k < R::kStages; ++k) fetch(k, t.base + t.mine + k * t.step);
  fetch_stats(t.base + t.mine);
  Pack<P, VEC> w[NV];
  load_columns(w, g.w, 1.f, t.lane, t.width, g.dim);
  float2 aw[E2], ab[E2];
#pragma unroll
  for (int i = 0; i < E2; ++i) aw[i] = ab[i] = per_both(0.f);
  for (int64_t base = t.base; base < g.rows; base += t.step) {
    const int64_t row = base + t.mine;
    const float hi = (float)nm, r = nr;
    const float lo = (float)(nm - (double)hi);
    float2 h[E2], gv[E2];
    float2 s1 = per_both(0.f), s2 = per_both(0.f);
    R::wait();
    {
      Pack<T, VEC> qx[NV], qy[NV];
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        qx[k] = ring.get(stage, k);
        qy[k] = ring.get(stage, NV + k);
      }
#pragma unroll
      for (int i = 0; i < E2; ++i) {
        const float2 d = get2<true>(qy, i);
        h[i] = per_fma2(per_add2(get2<true>(qx, i), per_both(-hi)), per_both(r), per_both(-lo * r));
        aw[i] = per_fma2(d, h[i], aw[i]);
        ab[i] = per_add2(ab[i], d);
        gv[i] = per_mul2(d, get2<true>(w, i));
        s1 = per_add2(s1, gv[i]);
        s2 = per_fma2(gv[i], h[i], s2);
      }
    }
    fetch(stage, row + R::kStages * t.step);
    fetch_stats(row + t.step);
    stage = stage + 1 == R::kStages ? 0 : stage + 1;
    if (!g.dx) continue;
    float a = lanes_sum<LANES>(s1.x + s1.y), q = lanes_sum<LANES>(s2.x + s2.y);
    if constexpr (LANES <= 0) {
      put<LANES>(ex, turn, t, make_float4(a, q, 0.f, 0.f));
      a = q = 0.f;
#pragma unroll
      for (int i = 0; i < Warps<LANES>::kReads; ++i)
        if (all.first + 32 * i < t.warps) {
          const float4 o = ex.slot[turn][all.from + all.first + 32 * i];
          a += o.x;
          q += o.y;
        }
      turn ^= 1;
      a = all.sum(a);
      q = all.sum(q);
    }
    if (row < g.rows) {
      // r (g - a / n - h q / n)
      const float2 r2 = per_both(r), k0 = per_both(-r * (a * inv_n)), k1 = per_both(-r * (q * inv_n));
      Pack<T, VEC> o[NV];
#pragma unroll
      for (int i = 0; i < E2; ++i) set2<true>(o, i, per_fma2(h[i], k1, per_fma2(gv[i], r2, k0)));
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (t.lane + k * t.width) * VEC;
        if (c < g.dim) store<T, VEC>(dx + row * g.dx_stride + c, o[k]);
      }
    }
  }
  if (!g.part) return;
  if (LANES < 0 || (LANES == 0 && t.width == (int)blockDim.x)) {
    float* part = g.part + t.base * 2 * g.dim;
#pragma unroll
    for (int i = 0; i < E2; ++i) {
      const int c0 = (t.lane + 2 * i / VEC * t.width) * VEC + 2 * i % VEC;
      const int c1 = VEC > 1 ? c0 + 1 : t.lane + (2 * i + 1) * t.width;
      if (c0 < g.dim) part[c0] = aw[i].x, part[g.dim + c0] = ab[i].x;
      if (c1 < g.dim) part[c1] = aw[i].y, part[g.dim + c1] = ab[i].y;
    }
  } else if constexpr (LANES >= 0) {
    // the row groups of a warp by shuffles, then the groups through shared
    // memory, where the (empty) copies still in flight have ended
    float* part = g.part + (int64_t)blockIdx.x * 2 * g.dim;
    float* sums = reinterpret_cast<float*>(dyn);  // [groups][2][dim]
    const int group = LANES > 0 ? threadIdx.x >> 5 : t.group;
    const int groups = LANES > 0 ? blockDim.x >> 5 : blockDim.x / t.width;
    float* mine = sums + group * 2 * g.dim;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < E2; ++i) {
      if constexpr (LANES > 0) {
#pragma unroll
        for (int o = LANES; o < 32; o <<= 1) {
          aw[i].x += __shfl_xor_sync(PER_FULL_MASK, aw[i].x, o);
          aw[i].y += __shfl_xor_sync(PER_FULL_MASK, aw[i].y, o);
          ab[i].x += __shfl_xor_sync(PER_FULL_MASK, ab[i].x, o);
          ab[i].y += __shfl_xor_sync(PER_FULL_MASK, ab[i].y, o);
        }
      }
      const int c0 = (t.lane + 2 * i / VEC * t.width) * VEC + 2 * i % VEC;
      const int c1 = VEC > 1 ? c0 + 1 : t.lane + (2 * i + 1) * t.width;
      if (t.mine == 0 && c0 < g.dim) mine[c0] = aw[i].x, mine[g.dim + c0] = ab[i].x;
      if (t.mine == 0 && c1 < g.dim) mine[c1] = aw[i].y, mine[g.dim + c1] = ab[i].y;
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * g.dim; c += blockDim.x) {
      float v = 0.f;
      for (int q = 0; q < groups; ++q) v += sums[q * 2 * g.dim + c];
      part[c] = v;
    }
  }
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

// dw and db from the partial rows: a CTA adds 32 columns, each of its 8 warps
// every eighth partial row, then the warps' sums in order.
constexpr int kJoinThreads = 256;
template <typename P>
__global__ void __launch_bounds__(kJoinThreads) per_layer_norm_join_kernel(const Bwd g) {
  __shared__ float s[kJoinThreads / 32][32];
  per_wait_previous_grid();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;  // column of [dw, db]
  const int64_t cols = 2 * (int64_t)g.dim;
  float v = 0.f;
  if (c < cols) {
#pragma unroll 8
    for (int k = warp; k < g.splits; k += kJoinThreads / 32) v += g.part[k * cols + c];
  }
  s[warp][lane] = v;
  __syncthreads();
  if (warp || c >= cols) return;
#pragma unroll
  for (int q = 1; q < kJoinThreads / 32; ++q) v += s[q][lane];
  void* out = c < g.dim ? g.dw : g.db;
  if (out) static_cast<P*>(out)[c < g.dim ? c : c - g.dim] = per_from_f32<P>(v);
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

// Row splits of the column sums of long rows.
int splits_of(int64_t rows, int64_t dim) {
  const int64_t tiles = (dim - 1) / kThreads + 1;
  int64_t s = 1184 / tiles;
  if (s > rows) s = rows;
  if (s > 256) s = 256;
  return s < 1 ? 1 : (int)s;
}

// How a row is laid over threads: `lanes` of a warp with `nv` vectors each, or
// a group of `threads` of each of `ctas` CTAs (lanes 0). ctas 0: too long for
// registers.
struct Shape {
  int lanes, nv, threads, ctas;
};

// Most vectors of a row that a thread holds. The sums over a row cost a thread
// some 100 instructions whatever it holds, so it should hold much; statistics,
// weights and (backward) two column sums per value have to fit its registers.
template <typename T, int VEC>
constexpr int fwd_vectors() {
  return VEC == 1 ? 16 : 4;
}
template <typename T, int VEC>
constexpr int bwd_vectors() {
  return VEC == 1 ? 8 : sizeof(T) == 2 ? 2 : 4;
}

// Rows that a warp can hold stay in it, which needs no barrier; longer ones
// take a group of warps, and beyond one CTA a cluster of up to 8.
Shape shape_of(int64_t dim, int vec, int full, int warp_threads) {
  const int64_t v = (dim + vec - 1) / vec;
  const int small = vec == 1 ? 4 : 1;
  for (int lanes = 4; lanes <= 32; lanes *= 2)
    if (v <= lanes * small) return {lanes, small, warp_threads, 1};
  for (int nv = 2 * small; nv <= full; nv *= 2)
    if (v <= 32 * nv) return {32, nv, warp_threads, 1};
  for (int ctas = 1; ctas <= kMaxCluster; ctas *= 2)
    if (v <= (int64_t)ctas * kRowThreads * full) {
      const int64_t threads = (v + ctas * full - 1) / (ctas * full);
      return {0, full, (int)((threads + 31) / 32 * 32), ctas};
    }
  return {0, 0, 0, 0};
}

// go<T, P, VEC, NV, LANES>(shape, ...) for the shape into rc; false where
// there is none
#define PER_NORM_SHAPE(s, rc, go, T, P, VEC, FULL, ...)                                        \
  [&]() -> bool {                                                                              \
    constexpr int S = VEC == 1 ? 4 : 1, F = FULL;                                              \
    if (s.lanes == 4) return rc = go<T, P, VEC, S, 4>(s, __VA_ARGS__), true;                   \
    if (s.lanes == 8) return rc = go<T, P, VEC, S, 8>(s, __VA_ARGS__), true;                   \
    if (s.lanes == 16) return rc = go<T, P, VEC, S, 16>(s, __VA_ARGS__), true;                 \
    if (s.lanes == 32 && s.nv == S) return rc = go<T, P, VEC, S, 32>(s, __VA_ARGS__), true;    \
    if (s.lanes == 32 && s.nv == 2 * S)                                                        \
      return rc = go<T, P, VEC, 2 * S, 32>(s, __VA_ARGS__), true;                              \
    if constexpr (F >= 4 * S)                                                                  \
      if (s.lanes == 32) return rc = go<T, P, VEC, 4 * S, 32>(s, __VA_ARGS__), true;           \
    if (s.ctas == 1) return rc = go<T, P, VEC, F, 0>(s, __VA_ARGS__), true;                    \
    if (s.ctas > 1) return rc = go<T, P, VEC, F, -1>(s, __VA_ARGS__), true;                    \
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
  rc = per_coresident_ctas(fn, threads, smem, &ctas);
  if (rc) return rc;
  const int64_t per_cta = threads / (s.lanes ? s.lanes : s.threads);
  int64_t grid = (rows - 1) / per_cta + 1;
  const int64_t room = ctas / s.ctas > 0 ? ctas / s.ctas : 1;
  if (grid > room) grid = room;
  if (most > 0 && grid > most) grid = most;
  *out = grid;
  return PER_OK;
}

template <typename T, typename P, int VEC, int NV, int LANES>
int forward_go(const Shape& s, const Fwd& f, cudaStream_t stream) {
  const void* fn = (const void*)per_layer_norm_kernel<T, P, VEC, NV, LANES>;
  const size_t smem = Ring<T, VEC, NV, kFwdStages>::kBytes * s.threads;
  int64_t grid = 0;
  const int rc = row_ctas(fn, s, s.threads, smem, f.rows, 0, &grid);
  if (rc) return rc;
  return launch(fn, grid * s.ctas, s.threads, smem, &f, stream, s.ctas);
}

template <typename T, typename P, int VEC>
int forward_vec(const Fwd& f, cudaStream_t stream) {
  constexpr int FULL = fwd_vectors<T, VEC>();
  const Shape s = shape_of(f.dim, VEC, FULL, 128);
  int rc = PER_OK;
  if (PER_NORM_SHAPE(s, rc, forward_go, T, P, VEC, FULL, f, stream)) return rc;
  return launch((const void*)per_layer_norm_long_kernel<T, P>, row_grid(f.rows), kThreads, 0, &f,
                stream);
}

template <typename T, typename P>
int forward(const Fwd& f, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  if (f.dim % VEC == 0 && aligned(f.x, f.x_stride, sizeof(T)) &&
      aligned(f.y, f.y_stride, sizeof(T)) && aligned(f.w, 0, 1) && aligned(f.b, 0, 1))
    return forward_vec<T, P, VEC>(f, stream);
  return forward_vec<T, P, 1>(f, stream);
}

// Most partial rows of dw and db (the workspace is sized before the pointers'
// alignment is known, so this holds for every kernel).
int64_t most_partials(int64_t rows, int64_t dim) {
  const int64_t most = (int64_t)sm_count() * (dim <= 512 ? 8 : dim <= 2048 ? 4 : 2);
  return rows < most ? rows : most;
}

template <typename T, typename P, int VEC, int NV, int LANES>
int backward_go(const Shape& s, const Bwd& in, cudaStream_t stream) {
  Bwd g = in;
  const void* fn = (const void*)per_layer_norm_backward_kernel<T, P, VEC, NV, LANES>;
  // a CTA of about 256 threads: several groups share its partial row
  const int groups = LANES == 0 && s.threads <= 128 ? 256 / s.threads : 1;
  const int threads = s.threads * groups;
  g.group_threads = s.threads;
  size_t smem = Ring<T, VEC, 2 * NV, kBwdStages>::kBytes * threads;
  if (LANES > 0 || groups > 1) {
    const size_t sums = (size_t)(LANES > 0 ? threads / 32 : groups) * 2 * g.dim * 4;
    smem = smem > sums ? smem : sums;
  }
  int64_t grid = 0;
  int rc = row_ctas(fn, s, threads, smem, g.rows, most_partials(g.rows, g.dim), &grid);
  if (rc) return rc;
  const bool columns = g.dw || g.db;
  if (!columns) g.part = nullptr;
  rc = launch(fn, grid * s.ctas, threads, smem, &g, stream, s.ctas);
  if (rc || !columns) return rc;
  g.splits = (int32_t)grid;
  return launch((const void*)per_layer_norm_join_kernel<P>, (2 * (int64_t)g.dim - 1) / 32 + 1,
                kJoinThreads, 0, &g, stream);
}

template <typename T, typename P, int VEC>
int backward_vec(const Bwd& in, cudaStream_t stream) {
  constexpr int FULL = bwd_vectors<T, VEC>();
  const Shape s = shape_of(in.dim, VEC, FULL, 256);
  int rc = PER_OK;
  if (PER_NORM_SHAPE(s, rc, backward_go, T, P, VEC, FULL, in, stream)) return rc;
  Bwd g = in;
  g.splits = splits_of(g.rows, g.dim);
  if (g.dx)
    rc = launch((const void*)per_layer_norm_dx_long_kernel<T, P>, row_grid(g.rows), kThreads, 0,
                &g, stream);
  if (rc || (!g.dw && !g.db)) return rc;
  const int64_t tiles = (g.dim - 1) / kThreads + 1;
  rc = launch((const void*)per_layer_norm_dw_long_kernel<T>, tiles * g.splits, kThreads, 0, &g,
              stream);
  if (rc) return rc;
  return launch((const void*)per_layer_norm_join_kernel<P>, (2 * (int64_t)g.dim - 1) / 32 + 1,
                kJoinThreads, 0, &g, stream);
}

template <typename T, typename P>
int backward(const Bwd& g, cudaStream_t stream) {
  constexpr int VEC = 16 / sizeof(T);
  if (g.dim % VEC == 0 && aligned(g.x, g.x_stride, sizeof(T)) &&
      aligned(g.dy, g.dy_stride, sizeof(T)) && aligned(g.dx, g.dx_stride, sizeof(T)) &&
      aligned(g.w, 0, 1))
    return backward_vec<T, P, VEC>(g, stream);
  return backward_vec<T, P, 1>(g, stream);
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
  int64_t most = most_partials(n.rows, n.dim);
  const int64_t s = splits_of(n.rows, n.dim);
  if (most < s) most = s;
  return most * 2 * n.dim * 4;
}

int per_launch_layer_norm_backward(const per_norm_t& n, const void* dy, int64_t dy_stride,
                                   const void* x, int64_t x_stride, const void* weight,
                                   const double* mean, const float* rstd, void* dx,
                                   int64_t dx_stride, void* dweight, void* dbias, void* workspace,
                                   cudaStream_t stream) {
  const Bwd g{dy, x, weight, mean, rstd, dx, dweight, dbias, static_cast<float*>(workspace),
              n.rows, dy_stride, x_stride, dx_stride, (int32_t)n.dim, 0, 0};
  return PER_NORM_TYPES(n, backward, g, stream);
}
