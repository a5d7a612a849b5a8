// Distillation loss from a teacher's top logits, forward and backward.
//
// Row r has student logits z[0..V), K teacher logits t_k with ids i_k (a
// negative id marks an absent entry) and a weight w_r:
//   p_k  = softmax over the present entries of t_k / tau
//   q_v  = softmax over the vocabulary of z_v / tau
//   l_r  = tau^2 * sum_k p_k (log p_k - log q_{i_k})     (terms with p_k = 0 are 0)
//   dz_v = w_r * c_r * tau * (q_v * sum_k p_k - sum_{k: i_k = v} p_k)
// with c_r the upstream gradient times the reduction's factor.  A row without
// teacher entries, or with w_r = 0, has loss 0 and gradient 0 and its logits
// are not read.
//
// The pass is bound by HBM: every logit is read once and, when a gradient is
// wanted, every gradient element written once.  To read once, a row is held in
// shared memory while its maximum and sum are formed (one running maximum and
// sum per thread, fp32), spread over a cluster of up to 8 CTAs when it is
// longer than one CTA's share; the gradient is then written from the held row.
// The backward proper has nothing to do when the upstream gradient is 1 (a
// loss that is differentiated directly); for any other value it writes the
// gradient again from the logits and the row's statistics, so that each
// element is rounded once whatever the factor.
#include <algorithm>

#include "b2_common.cuh"

namespace b2 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxTop = 1024;        // teacher entries per row
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;

enum Reduction : int { kMean = 0, kSum = 1, kNone = 2 };

struct Args {
  const void* z;
  long long ldz;
  const void* t;
  long long ldt;
  int t_f32;
  const void* ids;
  long long ldi;
  int ids64;
  long long N, V;
  int K;
  float tau;
  const float* weight;  // [N] or null
  int reduction;
  float* loss;          // scalar, or [N] for kNone
  float* stats;         // [N][2] maximum and log2 of the sum, then the reduction's factor at [2N]
  float* row_loss;      // workspace [N] (kNone: the loss itself)
  unsigned* counter;    // workspace
  void* dz;             // null: no gradient
  long long lddz;
  const float* upstream;  // backward: scalar, or [N] for kNone
  int skip_ones;          // backward: a row whose upstream gradient is 1 is left as the forward wrote it
  long long slice;        // 16-byte vectors per CTA of the cluster
  long long tile;         // 16-byte vectors held in shared memory at once
  int* status;
};

// 2^x by the hardware's approximation (relative error about 2^-22, results
// below 2^-126 are 0): well inside the rounding of either logits type's
// statistics, and one instruction where two of them per logit are the
// arithmetic of the whole pass.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
struct Vec16 {
  static constexpr int N = 16 / sizeof(T);
  uint4 v;
  __device__ __forceinline__ float get(int i) const {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&v);
    if constexpr (sizeof(T) == 2) return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
    else return __uint_as_float(w[i]);
  }
};
template <typename T>
__device__ __forceinline__ float load1(const T* p) {
  if constexpr (sizeof(T) == 2) return bf2f(*p);
  else return *p;
}
template <typename T>
__device__ __forceinline__ void store1(T* p, float v) {
  if constexpr (sizeof(T) == 2) {
    __nv_bfloat16 h = __float2bfloat16_rn(v);
    *p = *reinterpret_cast<uint16_t*>(&h);
  } else {
    *p = v;
  }
}
__device__ __forceinline__ uint32_t cvt2(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ float ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Running maximum and sum of exponentials relative to it.  An empty pair is
// (-inf, 0); a maximum of -inf means that nothing above -inf was seen.
struct MaxSum {
  float m, s;
};
// (base-2 exponents: c = log2(e) / tau)
__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  // -inf - -inf would be NaN: a side that saw nothing keeps its sum of 0 (or a NaN that it saw)
  const float fa = a.m == m ? 1.f : ex2((a.m - m) * c);
  const float fb = b.m == m ? 1.f : ex2((b.m - m) * c);
  return {m, a.s * fa + b.s * fb};
}

template <typename F>
__device__ __forceinline__ float warp_reduce(float v, F f) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <typename F>
__device__ __forceinline__ float block_reduce(float v, float* scratch, F f) {
  v = warp_reduce(v, f);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int i = 1; i < kWarps; ++i) v = f(v, scratch[i]);
  return v;
}

// The row's teacher entries in dynamic shared memory, [K] each.
struct TeacherSmem {
  float* p;
  int* id;
  float* scratch;  // [kWarps]
};

struct Teacher {
  bool any;     // the row has an entry with a probability
  bool bad;     // an id is outside the vocabulary
  float m;      // maximum of the entries' logits
  float mass;   // sum of exp((t - m) / tau)
};

// The row's teacher: probabilities and ids into shared memory (absent entries:
// p = 0, id = -1).
__device__ __forceinline__ Teacher load_teacher(const Args& a, long long r, const TeacherSmem& sm) {
  Teacher t;
  float m = -INFINITY;
  int bad = 0, nan = 0;
  for (int k = threadIdx.x; k < a.K; k += kThreads) {
    const long long id = a.ids64 ? static_cast<const long long*>(a.ids)[r * a.ldi + k]
                                 : (long long)static_cast<const int*>(a.ids)[r * a.ldi + k];
    float v = -INFINITY;
    if (id >= 0) {
      const long long at = r * a.ldt + k;
      v = a.t_f32 ? static_cast<const float*>(a.t)[at] : bf2f(static_cast<const uint16_t*>(a.t)[at]);
      if (id >= a.V) bad = 1;
      if (v != v) nan = 1;
    }
    sm.id[k] = id >= 0 && id < a.V ? int(id) : -1;
    sm.p[k] = v;
    m = fmaxf(m, v);
  }
  t.bad = __syncthreads_or(bad);
  const bool has_nan = __syncthreads_or(nan);
  t.m = block_reduce(m, sm.scratch, [](float x, float y) { return fmaxf(x, y); });
  t.any = t.m > -INFINITY || has_nan;
  float s = 0.f;
  const float c = kLog2e / a.tau;
  for (int k = threadIdx.x; k < a.K; k += kThreads) {
    const float v = sm.p[k];
    const float e = v == -INFINITY ? 0.f : ex2((v - t.m) * c);
    sm.p[k] = e;
    s += e;
  }
  t.mass = block_reduce(s, sm.scratch, [](float x, float y) { return x + y; });
  const float inv = 1.f / t.mass;
  if (t.any)
    for (int k = threadIdx.x; k < a.K; k += kThreads) sm.p[k] *= inv;
  __syncthreads();
  return t;
}

// Probability the teacher gives to id (entries with the same id add up, in
// entry order), for entry k.
__device__ __forceinline__ float teacher_p(const TeacherSmem& sm, int K, int k) {
  const int id = sm.id[k];
  float p = 0.f;
  for (int j = 0; j < K; ++j)
    if (sm.id[j] == id) p += sm.p[j];
  return p;
}

// Vector-aligned parts of a row: `head` elements, then whole 16-byte vectors, then the rest.
template <typename T>
struct RowParts {
  int head, tail;
  long long vecs;
  __device__ __forceinline__ RowParts(const T* row, long long V) {
    constexpr int E = Vec16<T>::N;
    const int off = int((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    head = int(min((long long)((E - off) % E), V));
    vecs = (V - head) / E;
    tail = int(V - head - vecs * E);
  }
};

// The gradient of 16 bytes of logits: a * 2^((z - m) c - l2s)
template <typename T>
__device__ __forceinline__ uint4 grad_vec(const Vec16<T>& x, float m, float c, float l2s, float a) {
  constexpr int E = Vec16<T>::N;
  float g[E];
#pragma unroll
  for (int i = 0; i < E; ++i) g[i] = a * ex2((x.get(i) - m) * c - l2s);
  if constexpr (sizeof(T) == 2)
    return make_uint4(cvt2(g[0], g[1]), cvt2(g[2], g[3]), cvt2(g[4], g[5]), cvt2(g[6], g[7]));
  else
    return make_uint4(__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]), __float_as_uint(g[3]));
}

template <typename T>
__device__ __forceinline__ void put_vec(T* dst, const uint4& v, bool aligned) {
  if (aligned) {
    *reinterpret_cast<uint4*>(dst) = v;
  } else {
    const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
    for (int i = 0; i < Vec16<T>::N; ++i) dst[i] = e[i];
  }
}

// Factor of row r: its weight times the reduction's
__device__ __forceinline__ float row_factor(const Args& a, long long r) {
  const float w = a.weight ? a.weight[r] : 1.f;
  return a.reduction == kMean ? w * a.stats[2 * a.N] : w;
}

// Reduction factor (1 / sum of the weights, 0 if that is 0) and the arrival
// counter of the forward's last step.
__global__ void __launch_bounds__(1024) distill_begin_kernel(const Args a) {
  __shared__ double part[32];
  double s = 0;
  if (a.reduction == kMean && a.weight)
    for (long long i = threadIdx.x; i < a.N; i += 1024) s += a.weight[i];
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0;
    for (int i = 0; i < 32; ++i) total += part[i];
    if (!a.weight) total = double(a.N);
    a.stats[2 * a.N] = total == 0 ? 0.f : float(1.0 / total);
    *a.counter = 0;
  }
}

// Forward (GRAD: with the gradient for an upstream gradient of 1).  One
// cluster per row; CTA `rank` owns `slice` vectors of it (the first also the
// head, the last also the tail).
template <typename T, bool GRAD>
__global__ void __launch_bounds__(kThreads) distill_fwd_kernel(const Args a, int cluster) {
  constexpr int E = Vec16<T>::N;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint4* held = reinterpret_cast<uint4*>(smem_raw);
  __shared__ float teacher_scratch[kWarps];
  float* teacher_p0 = reinterpret_cast<float*>(held + a.tile);
  const TeacherSmem teacher{teacher_p0, reinterpret_cast<int*>(teacher_p0 + a.K), teacher_scratch};
  __shared__ uint64_t bar;
  __shared__ float share[2];          // this CTA's maximum and sum, read by the cluster
  __shared__ float scratch[2][kWarps];
  __shared__ int last_row;
  const int rank = cluster > 1 ? int(cluster_ctarank()) : 0;
  const long long r = blockIdx.x / cluster;
  const T* row = static_cast<const T*>(a.z) + r * a.ldz;
  T* out = GRAD ? static_cast<T*>(a.dz) + r * a.lddz : nullptr;
  const RowParts<T> part(row, a.V);
  const long long v0 = min(part.vecs, a.slice * rank), v1 = min(part.vecs, v0 + a.slice);
  const bool out_aligned = GRAD && (reinterpret_cast<uintptr_t>(out + part.head) & 15) == 0;
  const float w = row_factor(a, r);
  const bool skip_weight = w == 0.f;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar), 1);
    fence_barrier_init();
  }
  __syncthreads();
  const bool single = v1 - v0 <= a.tile;  // the slice stays in shared memory
  uint32_t parity = 0;
  auto fetch = [&](long long b) {  // start loading tile [b, b + tile)
    if (threadIdx.x == 0) {
      const uint32_t bytes = uint32_t(min(a.tile, v1 - b) * 16);
      mbar_arrive_expect_tx(smem_u32(&bar), bytes);
      const uint8_t* src = reinterpret_cast<const uint8_t*>(row + part.head) + b * 16;
      for (uint32_t at = 0; at < bytes; at += 16384)
        bulk_load_1d(smem_u32(held) + at, src + at, min(16384u, bytes - at), smem_u32(&bar));
    }
  };
  auto landed = [&] {
    const bool ok = mbar_wait(smem_u32(&bar), parity, a.status, nullptr);
    parity ^= 1;
    return ok;
  };
  if (!skip_weight && v1 > v0) fetch(v0);
  Teacher tch{};
  if (!skip_weight) tch = load_teacher(a, r, teacher);
  const bool skip = skip_weight || !(tch.any || tch.bad);
  float loss = 0.f;
  if (skip) {
    if (!skip_weight && v1 > v0) landed();  // no copy may be in flight when the CTA leaves
    if constexpr (GRAD) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      for (long long i = v0 + threadIdx.x; i < v1; i += kThreads) put_vec<T>(out + part.head + i * E, zero, out_aligned);
      if (rank == 0 && threadIdx.x < part.head) out[threadIdx.x] = T(0);
      if (rank == cluster - 1 && threadIdx.x < part.tail) out[part.head + part.vecs * E + threadIdx.x] = T(0);
    }
    if (rank == 0 && threadIdx.x == 0) {
      a.stats[2 * r] = 0.f;
      a.stats[2 * r + 1] = 0.f;
    }
  } else {
    const float c = kLog2e / a.tau;
    MaxSum ms{-INFINITY, 0.f};
    // one value: 2^0 of the sum if it is the maximum, NaN if it is +inf (inf - inf)
    auto add1 = [&](float x) { ms = merge(ms, {x, x == INFINITY ? __int_as_float(0x7fc00000) : 1.f}, c); };
    // the unaligned ends straight from memory
    float edge = 0.f;
    const bool has_head = rank == 0 && int(threadIdx.x) < part.head;
    const bool has_tail = rank == cluster - 1 && int(threadIdx.x) < part.tail;
    const T* edge_tail = row + part.head + part.vecs * E + threadIdx.x;
    if (has_head) {
      edge = load1(row + threadIdx.x);
      add1(edge);
    }
    float edge2 = 0.f;
    if (has_tail) {
      edge2 = load1(edge_tail);
      add1(edge2);
    }
    for (long long b = v0; b < v1; b += a.tile) {
      if (b > v0) {
        __syncthreads();  // everyone is done with the tile before
        fetch(b);
      }
      landed();
      const int n = int(min(a.tile, v1 - b));
      for (int i = threadIdx.x; i < n; i += kThreads) {
        Vec16<T> x;
        x.v = held[i];
        float mx = x.get(0);
#pragma unroll
        for (int j = 1; j < E; ++j) mx = fmaxf(mx, x.get(j));
        if (mx > ms.m) {
          ms.s *= ex2((ms.m - mx) * c);  // 0 * 2^-inf = 0 for the first
          ms.m = mx;
        }
        // nothing above -inf yet (or only NaN): exponents relative to 0, so that -inf gives 0 and NaN stays
        const float ref = ms.m == -INFINITY ? 0.f : ms.m;
#pragma unroll
        for (int j = 0; j < E; ++j) ms.s += ex2((x.get(j) - ref) * c);
      }
    }
    // this CTA's pair
    {
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        MaxSum other{__shfl_xor_sync(0xffffffffu, ms.m, o), __shfl_xor_sync(0xffffffffu, ms.s, o)};
        ms = merge(ms, other, c);
      }
      if ((threadIdx.x & 31) == 0) {
        scratch[0][threadIdx.x >> 5] = ms.m;
        scratch[1][threadIdx.x >> 5] = ms.s;
      }
      __syncthreads();
      ms = {scratch[0][0], scratch[1][0]};
#pragma unroll
      for (int i = 1; i < kWarps; ++i) ms = merge(ms, {scratch[0][i], scratch[1][i]}, c);
    }
    if (cluster > 1) {
      if (threadIdx.x == 0) {
        share[0] = ms.m;
        share[1] = ms.s;
      }
      cluster_sync();
      ms = {-INFINITY, 0.f};
      for (int i = 0; i < cluster; ++i) {
        const uint32_t at = mapa_shared(smem_u32(share), uint32_t(i));
        ms = merge(ms, {ld_cluster(at), ld_cluster(at + 4)}, c);
      }
      cluster_arrive();  // done reading the others; waited for before leaving
    }
    const float l2s = log2f(ms.s);
    if (rank == 0) {
      // the loss: sum over entries of p (log p - log q), in entry order per thread
      const float inv_tau = 1.f / a.tau;
      const float ln_mass = logf(tch.mass), ln_s = logf(ms.s);
      float sum = 0.f;
      for (int k = threadIdx.x; k < a.K; k += kThreads) {
        const float p = teacher.p[k];
        const int id = teacher.id[k];
        if (id < 0 || p == 0.f) continue;
        const long long at = r * a.ldt + k;
        const float tv = a.t_f32 ? static_cast<const float*>(a.t)[at] : bf2f(static_cast<const uint16_t*>(a.t)[at]);
        const float logp = (tv - tch.m) * inv_tau - ln_mass;
        const float logq = (load1(row + id) - ms.m) * inv_tau - ln_s;
        sum += p * (logp - logq);
      }
      loss = block_reduce(sum, scratch[0], [](float x, float y) { return x + y; }) * a.tau * a.tau;
      if (tch.bad) loss = __int_as_float(0x7fc00000);
      if (threadIdx.x == 0) {
        a.stats[2 * r] = ms.m;
        a.stats[2 * r + 1] = l2s;
        if (tch.bad) record_status(a.status, B2_ERR_INVALID);
      }
    }
    if constexpr (GRAD) {
      const float f = tch.bad ? __int_as_float(0x7fc00000) : w * a.tau;
      for (long long b = v0; b < v1; b += a.tile) {
        if (!single) {
          __syncthreads();
          fetch(b);
          landed();
        }
        const int n = int(min(a.tile, v1 - b));
        for (int i = threadIdx.x; i < n; i += kThreads) {
          Vec16<T> x;
          x.v = held[i];
          put_vec<T>(out + part.head + (b + i) * E, grad_vec<T>(x, ms.m, c, l2s, f), out_aligned);
        }
      }
      if (has_head) store1(out + threadIdx.x, f * ex2((edge - ms.m) * c - l2s));
      if (has_tail) store1(out + part.head + part.vecs * E + threadIdx.x, f * ex2((edge2 - ms.m) * c - l2s));
      __syncthreads();  // the entries' elements are written again, from both terms
      const long long lo = rank == 0 ? 0 : part.head + v0 * E;
      const long long hi = rank == cluster - 1 ? a.V : part.head + v1 * E;
      for (int k = threadIdx.x; k < a.K; k += kThreads) {
        const int id = teacher.id[k];
        if (id < lo || id >= hi) continue;
        const float q = ex2((load1(row + id) - ms.m) * c - l2s);
        store1(out + id, f * (q - teacher_p(teacher, a.K, k)));
      }
    }
    if (cluster > 1) cluster_wait();
  }
  if (rank != 0) return;
  // reduction: the last row to arrive adds all rows, in row order
  if (a.reduction == kNone) {
    if (threadIdx.x == 0) a.loss[r] = w * loss;
    return;
  }
  if (threadIdx.x == 0) {
    a.row_loss[r] = w == 0.f ? 0.f : w * loss;
    __threadfence();
    last_row = atomicAdd(a.counter, 1u) == unsigned(a.N - 1);
  }
  __syncthreads();
  if (!last_row) return;
  __threadfence();
  float sum = 0.f;
  for (long long i = threadIdx.x; i < a.N; i += kThreads) sum += __ldcg(a.row_loss + i);
  sum = block_reduce(sum, scratch[1], [](float x, float y) { return x + y; });
  if (threadIdx.x == 0) *a.loss = sum;
}

// Backward for any upstream gradient: the gradient again from the logits and
// the forward's statistics.  Work item: one of `pieces` pieces of a row.
template <typename T>
__global__ void __launch_bounds__(kThreads) distill_bwd_kernel(const Args a, int pieces) {
  constexpr int E = Vec16<T>::N;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ float teacher_scratch[kWarps];
  float* teacher_p0 = reinterpret_cast<float*>(smem_raw);
  const TeacherSmem teacher{teacher_p0, reinterpret_cast<int*>(teacher_p0 + a.K), teacher_scratch};
  const int tid = int(threadIdx.x);
  if (a.skip_ones && a.reduction != kNone && *a.upstream == 1.f) return;
  for (long long item = blockIdx.x; item < a.N * pieces; item += gridDim.x) {
    const long long r = item / pieces;
    const int piece = int(item - r * pieces);
    const float up = a.reduction == kNone ? a.upstream[r] : *a.upstream;
    if (a.skip_ones && up == 1.f) continue;
    const T* row = static_cast<const T*>(a.z) + r * a.ldz;
    T* out = static_cast<T*>(a.dz) + r * a.lddz;
    const RowParts<T> part(row, a.V);
    const long long v0 = min(part.vecs, a.slice * piece), v1 = min(part.vecs, v0 + a.slice);
    const bool first = piece == 0, last = piece == pieces - 1;
    const bool out_aligned = (reinterpret_cast<uintptr_t>(out + part.head) & 15) == 0;
    const float w = row_factor(a, r);
    __syncthreads();
    Teacher tch{};
    if (w != 0.f) tch = load_teacher(a, r, teacher);
    if (w == 0.f || !(tch.any || tch.bad)) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      for (long long i = v0 + tid; i < v1; i += kThreads) put_vec<T>(out + part.head + i * E, zero, out_aligned);
      if (first && tid < part.head) out[tid] = T(0);
      if (last && tid < part.tail) out[part.head + part.vecs * E + tid] = T(0);
      continue;
    }
    const float c = kLog2e / a.tau;
    const float m = a.stats[2 * r], l2s = a.stats[2 * r + 1];
    const float f = tch.bad ? __int_as_float(0x7fc00000) : up * w * a.tau;
    const uint4* src = reinterpret_cast<const uint4*>(row + part.head);
    constexpr int U = 4;
    for (long long i0 = v0 + tid; i0 < v1; i0 += U * kThreads) {
      Vec16<T> x[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * kThreads < v1) x[u].v = src[i0 + u * kThreads];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * kThreads < v1)
          put_vec<T>(out + part.head + (i0 + u * kThreads) * E, grad_vec<T>(x[u], m, c, l2s, f), out_aligned);
    }
    if (first && tid < part.head) store1(out + tid, f * ex2((load1(row + tid) - m) * c - l2s));
    if (last && tid < part.tail) {
      const long long i = part.head + part.vecs * E + tid;
      store1(out + i, f * ex2((load1(row + i) - m) * c - l2s));
    }
    __syncthreads();
    const long long lo = first ? 0 : part.head + v0 * E;
    const long long hi = last ? a.V : part.head + v1 * E;
    for (int k = tid; k < a.K; k += kThreads) {
      const int id = teacher.id[k];
      if (id < lo || id >= hi) continue;
      const float q = ex2((load1(row + id) - m) * c - l2s);
      store1(out + id, f * (q - teacher_p(teacher, a.K, k)));
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Shared memory a CTA holds of a row: up to 72 KB, so that three CTAs fit on an
// SM and one's loads overlap another's arithmetic; slices of rows that are
// longer than that times the largest cluster take up to 208 KB.
constexpr long long kSliceVecs = 72 * 1024 / 16;
constexpr long long kTileVecs = 208 * 1024 / 16;
constexpr size_t kTopBytes = size_t(kMaxTop) * 8;

b2_status check_args(const char* who, const Args& a, int dtype, int t_dtype, int ids_dtype) {
  if (a.N < 0 || a.V < 1 || a.K < 0) return set_error(B2_ERR_INVALID, "%s: bad shape", who);
  if (a.K > kMaxTop) return set_error(B2_ERR_UNSUPPORTED, "%s: at most %d teacher entries per row", who, kMaxTop);
  if (a.V >= INT32_MAX || a.N >= INT32_MAX / kMaxCluster)
    return set_error(B2_ERR_UNSUPPORTED, "%s: too many rows or logits", who);
  if (dtype != B2_BF16 && dtype != B2_F32) return set_error(B2_ERR_INVALID, "%s: bad logits dtype %d", who, dtype);
  if (t_dtype != B2_BF16 && t_dtype != B2_F32) return set_error(B2_ERR_INVALID, "%s: bad teacher dtype %d", who, t_dtype);
  if (ids_dtype != B2_I32 && ids_dtype != B2_I64) return set_error(B2_ERR_INVALID, "%s: ids must be int32 or int64", who);
  if (a.reduction < kMean || a.reduction > kNone) return set_error(B2_ERR_INVALID, "%s: bad reduction %d", who, a.reduction);
  if (!(a.tau > 0.f) || !(a.tau < INFINITY)) return set_error(B2_ERR_INVALID, "%s: temperature must be positive", who);
  if (a.ldz < a.V || (a.K > 0 && (a.ldt < a.K || a.ldi < a.K)) || (a.dz && a.lddz < a.V))
    return set_error(B2_ERR_INVALID, "%s: bad row stride", who);
  return B2_OK;
}

template <typename T, bool GRAD>
b2_status launch_fwd(Args a, cudaStream_t st) {
  int dev = 0;
  B2_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
  const long long vecs = (a.V * (long long)sizeof(T) + 15) / 16;
  int cluster = 1;
  // longer rows over more CTAs; so are few rows, down to 4 KB a CTA
  while (cluster < kMaxCluster && ((vecs + cluster - 1) / cluster > kSliceVecs ||
                                   (a.N * cluster < sm_count(dev) && vecs / cluster >= 512)))
    cluster *= 2;
  a.slice = (vecs + cluster - 1) / cluster;
  a.tile = std::min(a.slice, a.slice <= kSliceVecs ? kSliceVecs : kTileVecs);
  const size_t smem = size_t(a.tile) * 16 + size_t(a.K) * 8;
  auto kern = distill_fwd_kernel<T, GRAD>;
  static bool configured[64] = {};
  if (dev < 0 || dev >= 64) return set_error(B2_ERR_INVALID, "device index %d", dev);
  if (!configured[dev]) {
    B2_TRY(check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                           int(kTileVecs * 16 + kTopBytes)),
                      "cudaFuncSetAttribute(distill)"));
    configured[dev] = true;
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(a.N * cluster));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(cluster);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a, cluster), "distill forward launch");
}

template <typename T>
b2_status launch_bwd(Args a, cudaStream_t st) {
  int dev = 0;
  B2_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
  const long long vecs = (a.V * (long long)sizeof(T) + 15) / 16;
  const int pieces = int(std::max<long long>(1, std::min<long long>(64, vecs / 2048)));
  a.slice = (vecs + pieces - 1) / pieces;
  const long long grid = std::min<long long>(a.N * pieces, (long long)sm_count(dev) * 8);
  distill_bwd_kernel<T><<<unsigned(grid), kThreads, size_t(a.K) * 8, st>>>(a, pieces);
  return check_cuda(cudaGetLastError(), "distill backward launch");
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

size_t b2_distill_workspace_bytes(int64_t N) { return N > 0 ? size_t(N) * 4 + 16 : 16; }

b2_status b2_distill_loss_fwd(const void* z, int64_t ldz, int dtype, int64_t N, int64_t V, const void* t, int64_t ldt,
                              int t_dtype, const void* ids, int64_t ldi, int ids_dtype, int64_t K, float temperature,
                              const float* row_weight, int reduction, float* loss, float* stats, void* dz,
                              int64_t lddz, void* workspace, size_t workspace_bytes, void* stream) {
  Args a{};
  a.z = z;
  a.ldz = ldz;
  a.t = t;
  a.ldt = ldt;
  a.t_f32 = t_dtype == B2_F32;
  a.ids = ids;
  a.ldi = ldi;
  a.ids64 = ids_dtype == B2_I64;
  a.N = N;
  a.V = V;
  a.K = int(std::min<int64_t>(K, INT32_MAX));
  a.tau = temperature;
  a.weight = row_weight;
  a.reduction = reduction;
  a.loss = loss;
  a.stats = stats;
  a.dz = dz;
  a.lddz = lddz;
  B2_TRY(check_args("b2_distill_loss_fwd", a, dtype, t_dtype, ids_dtype));
  const auto st = static_cast<cudaStream_t>(stream);
  if (N == 0) {
    if (reduction == kNone) return B2_OK;
    if (!loss) return set_error(B2_ERR_INVALID, "b2_distill_loss_fwd: null pointer");
    return check_cuda(cudaMemsetAsync(loss, 0, 4, st), "distill loss memset");
  }
  if (!z || !loss || !stats || !workspace || (K > 0 && (!t || !ids)))
    return set_error(B2_ERR_INVALID, "b2_distill_loss_fwd: null pointer");
  const size_t need = b2_distill_workspace_bytes(N);
  if (workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(B2_ERR_WORKSPACE, "b2_distill_loss_fwd: workspace of %zu bytes (16-byte aligned) needed, got %zu",
                     need, workspace_bytes);
  a.counter = static_cast<unsigned*>(workspace);
  a.row_loss = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 16);
  a.status = device_status_ptr();
  if (reduction != kNone) {
    distill_begin_kernel<<<1, 1024, 0, st>>>(a);
    B2_TRY(check_cuda(cudaGetLastError(), "distill begin launch"));
  }
  if (dtype == B2_BF16) return dz ? launch_fwd<uint16_t, true>(a, st) : launch_fwd<uint16_t, false>(a, st);
  return dz ? launch_fwd<float, true>(a, st) : launch_fwd<float, false>(a, st);
}

b2_status b2_distill_loss_bwd(const void* z, int64_t ldz, int dtype, int64_t N, int64_t V, const void* t, int64_t ldt,
                              int t_dtype, const void* ids, int64_t ldi, int ids_dtype, int64_t K, float temperature,
                              const float* row_weight, int reduction, const float* stats, const float* upstream,
                              int skip_ones, void* dz, int64_t lddz, void* stream) {
  Args a{};
  a.z = z;
  a.ldz = ldz;
  a.t = t;
  a.ldt = ldt;
  a.t_f32 = t_dtype == B2_F32;
  a.ids = ids;
  a.ldi = ldi;
  a.ids64 = ids_dtype == B2_I64;
  a.N = N;
  a.V = V;
  a.K = int(std::min<int64_t>(K, INT32_MAX));
  a.tau = temperature;
  a.weight = row_weight;
  a.reduction = reduction;
  a.stats = const_cast<float*>(stats);
  a.upstream = upstream;
  a.skip_ones = skip_ones;
  a.dz = dz;
  a.lddz = lddz;
  B2_TRY(check_args("b2_distill_loss_bwd", a, dtype, t_dtype, ids_dtype));
  if (N == 0) return B2_OK;
  if (!z || !stats || !upstream || !dz || (K > 0 && (!t || !ids)))
    return set_error(B2_ERR_INVALID, "b2_distill_loss_bwd: null pointer");
  const auto st = static_cast<cudaStream_t>(stream);
  return dtype == B2_BF16 ? launch_bwd<uint16_t>(a, st) : launch_bwd<float>(a, st);
}

}  // extern "C"
