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
// Two kernels do that: distill_stream_kernel, persistent, loads rows ahead of
// the arithmetic and keeps the memory system busy through it (many long rows);
// distill_row_kernel gives every row CTAs of its own (few rows; many short rows,
// with fewer threads each; or rows that no cluster holds, which it reads twice).
//
// Products that go into a sum are written as fused multiply-adds or as rounded
// products, so that the kernels with and without the gradient round alike and
// give the same loss.
//
// Exponents are base 2: with c = log2(e) / tau and R = max * c (rounded), a
// thread's sum is sum 2^(z c - R), one fused multiply-add and one 2^x per logit;
// since every later use refers to the same rounded R, its rounding cancels.
// Where R is large (rows far from zero, or whose largest logit is the type's
// lowest value) or not finite, the difference is taken before the product: R's
// rounding, 2^-24 of it, then no longer is a small exponent (kPlain).
// The backward proper has nothing to do when the upstream gradient is 1 (a
// loss that is differentiated directly); for any other value it writes the
// gradient again from the logits and the row's statistics, so that each
// element is rounded once whatever the factor.
#include <algorithm>
#include <atomic>

#include "b2_common.cuh"

namespace b2 {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kShortThreads = 128;
constexpr int kMaxTop = 1024;        // teacher entries per row
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.69314718055994531f;
// Largest |R| of the plain form.  The bf16 gradient's exponent adds R to two other
// offsets, each sum rounded at 2^-17 up to here: 10^-5 of an element, where its own
// rounding is 2^-9; at |R| = 2^20 it would be a tenth, and from 2^31 on the rounding
// of R alone overflows 2^x.  4096 rows of 131072 bf16 logits take 484 us with the
// gradient in the plain form, 525 in the other (the loss alone 295 and 301).
constexpr float kPlain = 256.f;

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
  unsigned long long wait_ns;  // limit of a wait
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

// Maximum and the sum of exponentials relative to it (relative to its rounded R
// where that is finite).  An empty pair is (-inf, 0); a maximum of -inf means
// that nothing above -inf was seen.
struct MaxSum {
  float m, s;
};
// R = m c, rounded: never fused into what it is added to
__device__ __forceinline__ float offset_of(float m, float c) { return __fmul_rn(m, c); }
// log2 of the factor that brings a sum relative to `from` to one relative to `to`.
// (A sum of the plain form is relative to R, others to m c itself: where they meet,
// around kPlain, R's rounding of at most 2^-17 stays in the sum.)
__device__ __forceinline__ float rescale(float from, float to, float c) {
  const float a = offset_of(from, c), b = offset_of(to, c);
  return fabsf(a) < kPlain && fabsf(b) < kPlain ? a - b : (from - to) * c;
}
__device__ __forceinline__ MaxSum merge(MaxSum a, MaxSum b, float c) {
  const float m = fmaxf(a.m, b.m);
  // -inf - -inf would be NaN: a side that saw nothing keeps its sum of 0 (or a NaN that it saw)
  const float fa = a.m == m ? 1.f : ex2(rescale(a.m, m, c));
  const float fb = b.m == m ? 1.f : ex2(rescale(b.m, m, c));
  return {m, fmaf(a.s, fa, b.s * fb)};
}
// The pair of W neighbouring lanes' pairs, in each of them: the maximum first,
// then each lane's sum relative to it once, then the sum of those.
template <int W>
__device__ __forceinline__ MaxSum warp_pair(MaxSum v, float c) {
  float m = v.m;
#pragma unroll
  for (int o = W / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float s = v.m == m ? v.s : __fmul_rn(v.s, ex2(rescale(v.m, m, c)));
#pragma unroll
  for (int o = W / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return {m, s};
}
// One value: 2^0 of the sum if it is the maximum, NaN if it is +inf (inf - inf)
__device__ __forceinline__ MaxSum one_value(float x) {
  return {x, x == INFINITY ? __int_as_float(0x7fc00000) : 1.f};
}

// One look at a phase: parked by the hardware for up to kParkNs, or (PARK false)
// not at all.  CLUSTER: the phase is completed by other CTAs' arrivals, whose
// stores become visible.
constexpr uint32_t kParkNs = 1000000;
template <bool CLUSTER, bool PARK>
__device__ __forceinline__ bool mbar_look(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  if constexpr (!PARK)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
  else if constexpr (CLUSTER)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kParkNs)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(kParkNs)
        : "memory");
  return ok != 0;
}

// A wait that the first look did not end: false, with B2_ERR_TIMEOUT recorded,
// after `limit` ns, or when another warp of the CTA has given up (*gave_up, if
// there is one).  Out of line: it is rare, and in every wait its code cost 1 %.
template <bool CLUSTER>
__device__ __noinline__ bool mbar_wait_on(uint32_t bar, uint32_t parity, int* status, volatile int* gave_up,
                                          unsigned long long limit) {
  unsigned long long t0 = 0;
  for (;;) {
    if (limit < kParkNs ? mbar_look<CLUSTER, false>(bar, parity) : mbar_look<CLUSTER, true>(bar, parity)) return true;
    if (gave_up && *gave_up) return false;
    const unsigned long long t = globaltimer();
    if (t0 == 0) t0 = t;
    if (t - t0 > limit) {
      record_status(status, B2_ERR_TIMEOUT);
      if (gave_up) *gave_up = 1;
      return false;
    }
  }
}

// Waits of the persistent kernel's warps (all lanes call and get the same answer):
// parked instead of polling, since the pollers of one CTA would take the issue
// slots of the others on the SM (limits too short for that are polled).
template <bool CLUSTER>
__device__ __forceinline__ bool mbar_wait_parked(uint32_t bar, uint32_t parity, int* status, volatile int* gave_up,
                                                 unsigned long long limit) {
  bool ok = limit >= kParkNs && mbar_look<CLUSTER, true>(bar, parity);
  if (!ok) ok = mbar_wait_on<CLUSTER>(bar, parity, status, gave_up, limit);
  return __all_sync(0xffffffffu, ok);
}

template <typename F>
__device__ __forceinline__ float warp_reduce(float v, F f) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
template <int THREADS, typename F>
__device__ __forceinline__ float block_reduce(float v, float* scratch, F f) {
  v = warp_reduce(v, f);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  v = scratch[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) v = f(v, scratch[i]);
  return v;
}

// Teacher arrays in shared memory hold a multiple of four entries.
__host__ __device__ constexpr int padded_top(int K) { return (K + 3) / 4 * 4; }

// The row's teacher entries in dynamic shared memory.
struct TeacherSmem {
  float* p;
  int* id;
  float* scratch;  // a float a warp
};

struct Teacher {
  bool any;     // the row has an entry with a probability
  bool bad;     // an id is outside the vocabulary
  float m;      // maximum of the entries' logits
  float mass;   // sum of exp((t - m) / tau)
};

// The row's teacher: probabilities and ids into shared memory (absent entries:
// p = 0, id = -1).
template <int THREADS>
__device__ __forceinline__ Teacher load_teacher(const Args& a, long long r, const TeacherSmem& sm) {
  Teacher t;
  float m = -INFINITY;
  int bad = 0, nan = 0;
  for (int k = threadIdx.x; k < padded_top(a.K); k += THREADS) {
    long long id = -1;
    if (k < a.K)
      id = a.ids64 ? static_cast<const long long*>(a.ids)[r * a.ldi + k]
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
  t.m = block_reduce<THREADS>(m, sm.scratch, [](float x, float y) { return fmaxf(x, y); });
  t.any = t.m > -INFINITY || has_nan;
  float s = 0.f;
  const float c = kLog2e / a.tau;
  for (int k = threadIdx.x; k < a.K; k += THREADS) {
    const float v = sm.p[k];
    const float e = v == -INFINITY ? 0.f : ex2((v - t.m) * c);
    sm.p[k] = e;
    s += e;
  }
  t.mass = block_reduce<THREADS>(s, sm.scratch, [](float x, float y) { return x + y; });
  const float inv = 1.f / t.mass;
  if (t.any)
    for (int k = threadIdx.x; k < a.K; k += THREADS) sm.p[k] *= inv;
  __syncthreads();
  return t;
}

// Probability the teacher gives to entry k's id (entries with the same id add
// up, in entry order).  Ids are compared four at a time; the arrays hold a
// multiple of four entries, 16-byte aligned, absent ones with id -1.
__device__ __forceinline__ float teacher_p(const TeacherSmem& sm, int K, int k) {
  const int id = sm.id[k];
  float p = 0.f;
  const int4* ids = reinterpret_cast<const int4*>(sm.id);
  for (int j = 0; j < K; j += 4) {
    const int4 v = ids[j / 4];
    if (v.x == id) p += sm.p[j];
    if (v.y == id) p += sm.p[j + 1];
    if (v.z == id) p += sm.p[j + 2];
    if (v.w == id) p += sm.p[j + 3];
  }
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

// A thread's running pair over 16-byte vectors of logits.  The common case --
// its maximum so far times c is below kPlain -- is one multiply-add, one 2^x and one
// addition per logit; the test for it and for a new maximum is made once for up
// to 8 vectors (some lane of a warp sees a new maximum nearly every time, so its
// dozen instructions are the price of every test).
template <typename T>
struct Running {
  static constexpr int E = Vec16<T>::N;
  float c;
  MaxSum ms;
  float ref;    // ms.m * c
  bool plain;   // |ref| < kPlain
  __device__ __forceinline__ explicit Running(float c_) : c(c_), ms{-INFINITY, 0.f}, ref(-INFINITY), plain(false) {}
  __device__ __forceinline__ void grow(float m) {
    ms.s = __fmul_rn(ms.s, ex2(rescale(ms.m, m, c)));  // 0 * 2^-inf = 0 for the first
    ms.m = m;
    ref = offset_of(m, c);
    plain = fabsf(ref) < kPlain;
  }
  __device__ __forceinline__ void add1(float x) {
    ms = merge(ms, one_value(x), c);
    ref = offset_of(ms.m, c);
    plain = fabsf(ref) < kPlain;
  }
  template <int V>
  static __device__ __forceinline__ float max_of(const Vec16<T> (&x)[V]) {
    if constexpr (sizeof(T) == 2) {
      __nv_bfloat162 m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = reinterpret_cast<const __nv_bfloat162*>(&x[0].v)[i];
#pragma unroll
      for (int v = 1; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = __hmax2(m[i], reinterpret_cast<const __nv_bfloat162*>(&x[v].v)[i]);
      const __nv_bfloat162 all = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
      return fmaxf(__low2float(all), __high2float(all));
    } else {
      float m[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) m[i] = x[0].get(i);
#pragma unroll
      for (int v = 1; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) m[i] = fmaxf(m[i], x[v].get(i));
      return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    }
  }
  template <int V>
  __device__ __forceinline__ void add(const Vec16<T> (&x)[V]) {
    const float mx = max_of(x);
    if (mx > ms.m) grow(mx);
    if (plain) {
      float sum[4] = {ms.s, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < E; ++j) sum[j % 4] += ex2(fmaf(x[v].get(j), c, -ref));
      ms.s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    } else {
      // nothing above -inf yet (or only NaN): relative to 0, so that -inf gives 0 and NaN stays
      const float m = ms.m == -INFINITY ? 0.f : ms.m;
      float sum[4] = {ms.s, 0.f, 0.f, 0.f};
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < E; ++j) sum[j % 4] += ex2((x[v].get(j) - m) * c);
      ms.s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
    }
  }
  // vectors first, first + step, ... of src[0 .. n)
  template <int V>
  __device__ __forceinline__ int add_some(const uint4* src, int i, int n, int step) {
#pragma unroll 1
    for (; i + (V - 1) * step < n; i += V * step) {
      Vec16<T> x[V];
#pragma unroll
      for (int v = 0; v < V; ++v) x[v].v = src[i + v * step];
      add(x);
    }
    return i;
  }
  __device__ __forceinline__ void add_slice(const uint4* src, int first, int n, int step) {
    int i = add_some<8>(src, first, n, step);
    i = add_some<4>(src, i, n, step);
    add_some<1>(src, i, n, step);
  }
};

// A row's statistics as its gradient and loss use them: log2 q = z c - R - l2s.
template <typename T>
struct Prob {
  float c, m, l2s, ref;
  bool plain;
  __device__ __forceinline__ Prob(float c_, float m_, float l2s_)
      : c(c_), m(m_), l2s(l2s_), ref(offset_of(m_, c_)), plain(fabsf(ref) < kPlain) {}
  __device__ __forceinline__ float log2q(float z) const {
    return plain ? fmaf(z, c, -ref) - l2s : fmaf(z - m, c, -l2s);
  }
  // tau log q.  A finite logit whose z c leaves fp32's range (one masked with the
  // type's lowest value) has a finite one all the same: by z - m itself.
  __device__ __forceinline__ float tau_logq(float z, float tau) const {
    const float l = log2q(z), t = tau * kLn2;
    return l == -INFINITY && z > -INFINITY ? fmaf(-t, l2s, z - m) : __fmul_rn(t, l);
  }
  __device__ __forceinline__ float operator()(float z) const {
    if (plain) return fast(z);
    return ex2(log2q(z));
  }
  // `plain` rows.  bf16 results round at 2^-8: the two offsets are added up first
  // (an error of 2^-24 of their size, see kPlain); fp32 keeps z c - R exact where it
  // matters, near the top.
  __device__ __forceinline__ float fast(float z) const {
    if constexpr (sizeof(T) == 2) return ex2(fmaf(z, c, -(ref + l2s)));
    else return ex2(fmaf(z, c, -ref) - l2s);
  }
};

// The gradient of 16 bytes of logits, a * q.  PLAIN: a positive factor joins the
// exponent (off: its logarithm less the offsets), which saves the product.
template <typename T, bool PLAIN>
__device__ __forceinline__ uint4 grad_vec(const Vec16<T>& x, const Prob<T>& q, float a, float off) {
  constexpr int E = Vec16<T>::N;
  float g[E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if constexpr (!PLAIN) g[i] = a * ex2(q.log2q(x.get(i)));
    else if constexpr (sizeof(T) == 2) g[i] = ex2(fmaf(x.get(i), q.c, off));
    else g[i] = ex2(fmaf(x.get(i), q.c, -q.ref) + off);
  }
  if constexpr (sizeof(T) == 2)
    return make_uint4(cvt2(g[0], g[1]), cvt2(g[2], g[3]), cvt2(g[4], g[5]), cvt2(g[6], g[7]));
  else
    return make_uint4(__float_as_uint(g[0]), __float_as_uint(g[1]), __float_as_uint(g[2]), __float_as_uint(g[3]));
}
template <typename T>
__device__ __forceinline__ float grad_offset(const Prob<T>& q, float a) {
  return sizeof(T) == 2 ? log2f(a) - (q.ref + q.l2s) : log2f(a) - q.l2s;
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

// The gradient of vectors first, first + step, ... of src[0 .. n) to dst
template <typename T>
__device__ __forceinline__ void grad_slice(const uint4* src, T* dst, int first, int n, int step, const Prob<T>& q,
                                           float a) {
  if (q.plain && a > 0.f && (reinterpret_cast<uintptr_t>(dst) & 15) == 0) {
    const float off = grad_offset(q, a);
    uint4* d = reinterpret_cast<uint4*>(dst);
#pragma unroll 2
    for (int i = first; i < n; i += step) {
      Vec16<T> x;
      x.v = src[i];
      d[i] = grad_vec<T, true>(x, q, a, off);
    }
  } else {
#pragma unroll 1
    for (int i = first; i < n; i += step) {
      Vec16<T> x;
      x.v = src[i];
      put_vec<T>(dst + (long long)i * Vec16<T>::N, grad_vec<T, false>(x, q, a, 0.f),
                 (reinterpret_cast<uintptr_t>(dst) & 15) == 0);
    }
  }
}

// Factor of row r: its weight times the reduction's
__device__ __forceinline__ float row_factor(const Args& a, long long r) {
  const float w = a.weight ? a.weight[r] : 1.f;
  return a.reduction == kMean ? w * a.stats[2 * a.N] : w;
}

// Reduction factor (1 / sum of the weights, 0 if that is 0) and the arrival
// counter of the forward's last step.  One CTA, 8192 weights: 2 us.
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
// head, the last also the tail).  Few rows are bound by the latency of one, 8 us
// (one row of 32000 bf16 logits over 8 CTAs); 900 rows with the gradient take
// 34 us, 3.4 TB/s, in eight CTAs a SM.
template <typename T, bool GRAD, int THREADS>
__global__ void __launch_bounds__(THREADS) distill_row_kernel(const Args a, int cluster) {
  constexpr int E = Vec16<T>::N;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  uint4* held = reinterpret_cast<uint4*>(smem_raw);
  __shared__ float teacher_scratch[THREADS / 32];
  float* teacher_p0 = reinterpret_cast<float*>(held + a.tile);
  const TeacherSmem teacher{teacher_p0, reinterpret_cast<int*>(teacher_p0 + padded_top(a.K)), teacher_scratch};
  __shared__ uint64_t bar;
  __shared__ float share[2];          // this CTA's maximum and sum, read by the cluster
  __shared__ float scratch[2][THREADS / 32];
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
  // false: not in time; the copy has landed all the same before its shared memory
  // is used again or the CTA leaves
  auto landed = [&] {
    const bool ok = (a.wait_ns >= kParkNs && mbar_try_wait(smem_u32(&bar), parity)) ||
                    mbar_wait_on<false>(smem_u32(&bar), parity, a.status, nullptr, a.wait_ns);
    if (!ok) mbar_wait_on<false>(smem_u32(&bar), parity, a.status, nullptr, kWaitLimitNs);
    parity ^= 1;
    return ok;
  };
  if (!skip_weight && v1 > v0) fetch(v0);
  Teacher tch{};
  if (!skip_weight) tch = load_teacher<THREADS>(a, r, teacher);
  const bool skip = skip_weight || !(tch.any || tch.bad);
  float loss = 0.f;
  if (skip) {
    if (!skip_weight && v1 > v0) landed();  // no copy may be in flight when the CTA leaves
    if constexpr (GRAD) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      for (long long i = v0 + threadIdx.x; i < v1; i += THREADS) put_vec<T>(out + part.head + i * E, zero, out_aligned);
      if (rank == 0 && threadIdx.x < part.head) out[threadIdx.x] = T(0);
      if (rank == cluster - 1 && threadIdx.x < part.tail) out[part.head + part.vecs * E + threadIdx.x] = T(0);
    }
    if (rank == 0 && threadIdx.x == 0) {
      a.stats[2 * r] = 0.f;
      a.stats[2 * r + 1] = 0.f;
    }
  } else {
    const float c = kLog2e / a.tau;
    Running<T> run(c);
    // the unaligned ends straight from memory
    float edge = 0.f;
    const bool has_head = rank == 0 && int(threadIdx.x) < part.head;
    const bool has_tail = rank == cluster - 1 && int(threadIdx.x) < part.tail;
    const T* edge_tail = row + part.head + part.vecs * E + threadIdx.x;
    if (has_head) {
      edge = load1(row + threadIdx.x);
      run.add1(edge);
    }
    float edge2 = 0.f;
    if (has_tail) {
      edge2 = load1(edge_tail);
      run.add1(edge2);
    }
    bool lost = false;
    for (long long b = v0; b < v1; b += a.tile) {
      if (b > v0) {
        __syncthreads();  // everyone is done with the tile before
        fetch(b);
      }
      lost |= !landed();
      run.add_slice(held, int(threadIdx.x), int(min(a.tile, v1 - b)), THREADS);
    }
    MaxSum ms = run.ms;
    if (lost) ms.s = __int_as_float(0x7fc00000);  // a wait ran out: the row's loss and gradient are NaN
    // this CTA's pair
    {
      ms = warp_pair<32>(ms, c);
      if ((threadIdx.x & 31) == 0) {
        scratch[0][threadIdx.x >> 5] = ms.m;
        scratch[1][threadIdx.x >> 5] = ms.s;
      }
      __syncthreads();
      ms = warp_pair<THREADS / 32>({scratch[0][threadIdx.x % (THREADS / 32)], scratch[1][threadIdx.x % (THREADS / 32)]}, c);
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
      // the loss: sum over entries of p tau (log p - log q), in entry order per thread; times tau at the end
      const float ln_mass = logf(tch.mass);
      const Prob<T> qs(c, ms.m, l2s);
      float sum = 0.f;
      for (int k = threadIdx.x; k < a.K; k += THREADS) {
        const float p = teacher.p[k];
        const int id = teacher.id[k];
        if (id < 0 || p == 0.f) continue;
        const long long at = r * a.ldt + k;
        const float tv = a.t_f32 ? static_cast<const float*>(a.t)[at] : bf2f(static_cast<const uint16_t*>(a.t)[at]);
        const float tau_logp = fmaf(-a.tau, ln_mass, tv - tch.m);
        sum = fmaf(p, tau_logp - qs.tau_logq(load1(row + id), a.tau), sum);
      }
      loss = block_reduce<THREADS>(sum, scratch[0], [](float x, float y) { return x + y; }) * a.tau;
      if (tch.bad) loss = __int_as_float(0x7fc00000);
      if (threadIdx.x == 0) {
        a.stats[2 * r] = ms.m;
        a.stats[2 * r + 1] = l2s;
        if (tch.bad) record_status(a.status, B2_ERR_INVALID);
      }
    }
    if constexpr (GRAD) {
      const float f = tch.bad ? __int_as_float(0x7fc00000) : w * a.tau;
      const Prob<T> q(c, ms.m, l2s);
      for (long long b = v0; b < v1; b += a.tile) {
        float fb = f;
        if (!single) {
          __syncthreads();
          fetch(b);
          if (!landed()) fb = __int_as_float(0x7fc00000);
        }
        grad_slice<T>(held, out + part.head + b * E, int(threadIdx.x), int(min(a.tile, v1 - b)), THREADS, q, fb);
      }
      if (has_head) store1(out + threadIdx.x, f * q(edge));
      if (has_tail) store1(out + part.head + part.vecs * E + threadIdx.x, f * q(edge2));
      __syncthreads();  // the entries' elements are written again, from both terms
      const long long lo = rank == 0 ? 0 : part.head + v0 * E;
      const long long hi = rank == cluster - 1 ? a.V : part.head + v1 * E;
      for (int k = threadIdx.x; k < a.K; k += THREADS) {
        const int id = teacher.id[k];
        if (id < lo || id >= hi) continue;
        store1(out + id, f * (q(load1(row + id)) - teacher_p(teacher, a.K, k)));
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
#pragma unroll 8
  for (long long i = threadIdx.x; i < a.N; i += THREADS) sum += __ldcg(a.row_loss + i);
  sum = block_reduce<THREADS>(sum, scratch[1], [](float x, float y) { return x + y; });
  if (threadIdx.x == 0) *a.loss = sum;
}

// ---------------------------------------------------------------------------
// The persistent kernel.  Three CTAs a SM, so that one's copies, another's
// exponentials and a third's stores overlap; clusters of them walk the rows
// cluster by cluster, each CTA with a buffer for one slice.  Warp 8 runs ahead: it
// reads the next row's weight and teacher entries, starts the copy of its slice
// when the buffer is free unless the row is masked, meanwhile makes the teacher's probabilities
// and, from the slice's entries, its part of the loss.  Warps 0..7 form the
// slice's maximum and sum, exchange all that with the cluster's CTAs (a remote
// store and a remote arrival each) and write the gradient; then the entries'
// elements once more, from both terms.
//
// The loss in parts: with m_j the maximum of slice j, P_j the probability of the
// entries in it and lse the row's log-sum-exp of z / tau,
//   sum_k p_k tau (log p_k - log q_k) = sum_j [ sum_{k in j} p_k (tau log p_k -
//   (z_k - m_j)) + P_j (tau lse - m_j) ]
// whose slice sums need nothing of the other slices (and whose differences of
// logits, not divided by tau, are finite where the logits are).
//
// 8192 rows of 131072 bf16 logits with 64 entries, a seventh of them masked:
// 864 us with the gradient (4.6 TB/s of the 6.45 measured), 515 us the loss
// alone; a row's 10 us in a CTA are 2.5 of copy, 2.5 of sums, 0.7 of reduction,
// 1.6 of exchange, 2.1 of gradient and 0.9 of entries.  (One CTA of 16 warps a SM
// with a ring of three slices took 1610 us: a row at a time leaves the SM waiting
// in every reduction.  Slices of half the size, with a ring of two, 1130 us.)
//
// Statistics slots: a CTA's publication of its row i + 2 follows its end of row
// i + 1, which needed this CTA's publication of row i + 1, which this CTA made
// after its own end of row i: two slots are never overrun.
// ---------------------------------------------------------------------------
constexpr int kStreamWarps = 8;
constexpr int kStreamThreads = (kStreamWarps + 1) * 32;
constexpr int kStreamPerSm = 3;
constexpr int kSlots = 2;

// What the forward warp knows of the row in the buffer.
struct RowMeta {
  long long row;
  int skip, bad;
  float w, side, P, top;  // the slice's part of the loss over tau, relative to a logit of `top`; its entries' probability
  float head[8], tail[8];
};

// Logit `id` of a row, from this CTA's held slice (vectors from v0) or the row's unaligned ends.
template <typename T>
__device__ __forceinline__ float slice_logit(const uint4* slice, const RowMeta& mt, const RowParts<T>& parts,
                                             long long v0, int id) {
  const long long tail0 = parts.head + parts.vecs * Vec16<T>::N;
  return id < parts.head ? mt.head[id]
         : id >= tail0   ? mt.tail[id - tail0]
                         : load1(reinterpret_cast<const T*>(slice) + (id - parts.head - v0 * Vec16<T>::N));
}

// Barriers of the compute warps; the second is a vote: true if none of them has given up.
__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ bool compute_all(bool ok) {
  uint32_t all;
  __syncwarp();
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.and.pred q, 1, 256, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(all)
      : "r"(uint32_t(ok))
      : "memory");
  return all != 0;
}

template <typename T, bool GRAD>
__global__ void __launch_bounds__(kStreamThreads, kStreamPerSm) distill_stream_kernel(const Args a, int cluster) {
  constexpr int E = Vec16<T>::N;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ uint64_t full, top_full, empty, slot_bar[kSlots];
  __shared__ float4 slot[kSlots][kMaxCluster];  // a slice's maximum, sum, loss part and P
  __shared__ RowMeta meta;
  __shared__ float part[2][kStreamWarps][2];
  __shared__ float final_part[kStreamWarps];
  __shared__ int last_row;
  __shared__ int gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = int(threadIdx.x);
  const int rank = cluster > 1 ? int(cluster_ctarank()) : 0;
  const long long first = blockIdx.x / cluster, step = gridDim.x / cluster;
  const float c = kLog2e / a.tau;
  uint4* held = reinterpret_cast<uint4*>(smem_raw);
  float* top_p = reinterpret_cast<float*>(held + a.slice);
  const int Kp = padded_top(a.K);
  int* top_id = reinterpret_cast<int*>(top_p + 2 * Kp);  // two rows' entries
  const auto wait_for = [&](uint64_t& bar, uint32_t parity) {
    return mbar_wait_parked<false>(smem_u32(&bar), parity, a.status, &gave_up, a.wait_ns);
  };
  if (tid == 0) {
    gave_up = 0;
    mbar_init(smem_u32(&full), 1);
    mbar_init(smem_u32(&top_full), 1);
    mbar_init(smem_u32(&empty), kStreamWarps);
    for (int b = 0; b < kSlots; ++b) mbar_init(smem_u32(&slot_bar[b]), uint32_t(cluster));
    fence_barrier_init();
  }
  __syncthreads();
  if (cluster > 1) cluster_sync();  // every CTA's barriers exist before a remote arrival

  if (warp == kStreamWarps) {
    // ------------------------------ the forward warp ------------------------
    // A row's weight, teacher entries and unaligned ends, read before its buffer
    // is free, so that its copy starts the moment it is.
    struct Ahead {
      float w, m, edge;
      int bad;
      bool skip;
    };
    auto look = [&](long long r, int slot_at) {
      Ahead h{};
      const T* row = static_cast<const T*>(a.z) + r * a.ldz;
      const RowParts<T> parts(row, a.V);
      float* p = top_p + slot_at * Kp;
      int* ids = top_id + slot_at * Kp;
      h.w = row_factor(a, r);
      h.m = -INFINITY;
      h.skip = true;
      if (h.w == 0.f) return h;
      // lanes 0..7: the head, 8..15: the tail
      if (rank == 0 && lane < parts.head) h.edge = load1(row + lane);
      if (rank == cluster - 1 && lane >= 8 && lane - 8 < parts.tail)
        h.edge = load1(row + parts.head + parts.vecs * E + lane - 8);
      int nan = 0;
      for (int k = a.K + lane; k < Kp; k += 32) ids[k] = -1;
      for (int k = lane; k < a.K; k += 32) {
        const long long at = r * a.ldt + k;
        const long long id = a.ids64 ? static_cast<const long long*>(a.ids)[r * a.ldi + k]
                                     : (long long)static_cast<const int*>(a.ids)[r * a.ldi + k];
        float v = a.t_f32 ? static_cast<const float*>(a.t)[at] : bf2f(static_cast<const uint16_t*>(a.t)[at]);
        if (id < 0) v = -INFINITY;
        if (id >= a.V) h.bad = 1;
        if (v != v) nan = 1;
        ids[k] = id >= 0 && id < a.V ? int(id) : -1;
        p[k] = v;
        h.m = fmaxf(h.m, v);
      }
      h.bad = __any_sync(0xffffffffu, h.bad);
      nan = __any_sync(0xffffffffu, nan);
      h.m = warp_reduce(h.m, [](float x, float y) { return fmaxf(x, y); });
      h.skip = !(h.m > -INFINITY || nan || h.bad);
      return h;
    };
    long long n = 0, started = 0;  // rows whose slice is on its way or here
    Ahead next{};
    if (first < a.N) next = look(first, 0);
    for (long long r = first; r < a.N; r += step, ++n) {
      const int top_at = int(n & 1);
      const Ahead h = next;
      if (n > 0 && !wait_for(empty, uint32_t((n - 1) & 1))) break;
      const T* row = static_cast<const T*>(a.z) + r * a.ldz;
      const RowParts<T> parts(row, a.V);
      const long long v0 = min(parts.vecs, a.slice * rank), v1 = min(parts.vecs, v0 + a.slice);
      if (lane < 8) meta.head[lane] = h.edge;
      else if (lane < 16) meta.tail[lane - 8] = h.edge;
      if (lane == 0) {
        meta.row = r;
        meta.skip = h.skip;
        meta.bad = h.bad;
        meta.w = h.w;
      }
      __syncwarp();
      if (lane == 0) {
        const uint32_t bytes = h.skip ? 0u : uint32_t((v1 - v0) * 16);
        if (bytes) {
          mbar_arrive_expect_tx(smem_u32(&full), bytes);
          const uint8_t* src = reinterpret_cast<const uint8_t*>(row + parts.head) + v0 * 16;
          const uint32_t dst = smem_u32(held);
          for (uint32_t at = 0; at < bytes; at += 16384)
            bulk_load_1d(dst + at, src + at, min(16384u, bytes - at), smem_u32(&full));
        } else {
          mbar_arrive(smem_u32(&full));
        }
        if (h.bad && rank == 0) record_status(a.status, B2_ERR_INVALID);
      }
      started = n + 1;
      if (!h.skip) {
        float* p = top_p + top_at * Kp;
        float s = 0.f;
        for (int k = lane; k < a.K; k += 32) {
          const float v = p[k];
          const float e = v == -INFINITY ? 0.f : ex2((v - h.m) * c);
          p[k] = e;
          s += e;
        }
        s = warp_reduce(s, [](float x, float y) { return x + y; });
        const float inv = 1.f / s;
        // the entries of this slice, once it is here: their part of the loss
        const int* ids = top_id + top_at * Kp;
        const long long lo = rank == 0 ? 0 : parts.head + v0 * E;
        const long long hi = rank == cluster - 1 ? a.V : parts.head + v1 * E;
        const uint4* slice = held;
        if (!wait_for(full, uint32_t(n & 1))) break;
        float top = -INFINITY;
        for (int k = lane; k < a.K; k += 32) {
          const float pk = p[k] * inv;
          p[k] = pk;
          if (ids[k] >= lo && ids[k] < hi && pk != 0.f)
            top = fmaxf(top, slice_logit<T>(slice, meta, parts, v0, ids[k]));
        }
        top = warp_reduce(top, [](float x, float y) { return fmaxf(x, y); });
        if (!(fabsf(top) < INFINITY)) top = 0.f;
        float side = 0.f, P = 0.f;
        for (int k = lane; k < a.K; k += 32) {
          const float pk = p[k];
          if (ids[k] < lo || ids[k] >= hi || pk == 0.f) continue;
          const float z = slice_logit<T>(slice, meta, parts, v0, ids[k]);
          // a closed entry makes the loss infinite, also in a slice of nothing else
          side = z == -INFINITY ? INFINITY : fmaf(pk, fmaf(a.tau, logf(pk), top - z), side);
          P += pk;
        }
        side = warp_reduce(side, [](float x, float y) { return x + y; });
        P = warp_reduce(P, [](float x, float y) { return x + y; });
        if (lane == 0) {
          meta.side = side;
          meta.P = P;
          meta.top = top;
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&top_full));
      if (r + step < a.N) next = look(r + step, int((n + 1) & 1));
    }
    // every copy lands before the CTA goes away, also if someone gave up
    if (started > 0)
      mbar_wait_parked<false>(smem_u32(&full), uint32_t((started - 1) & 1), a.status, nullptr, kWaitLimitNs);
  } else {
    // ------------------------------ the compute warps -----------------------
    long long counted = 0;  // rows with statistics
    int flip = 0;
    // Statistics of the held row, its loss, its gradient; frees the buffer.
    auto finish = [&](long long n, MaxSum ms, float parts_m, float side, float P) {
      const RowMeta& mt = meta;
      const long long r = mt.row;
      const float l2s = log2f(ms.s);
      if (rank == 0 && warp == 0) {
        // lane j: slice j
        float part_loss = 0.f;
        if (lane < cluster)
          part_loss = P == 0.f ? side : fmaf(-P, Prob<T>(c, ms.m, l2s).tau_logq(parts_m, a.tau), side);
#pragma unroll
        for (int o = kMaxCluster / 2; o; o >>= 1) part_loss += __shfl_xor_sync(0xffffffffu, part_loss, o);
        side = part_loss;
      }
      if (rank == 0 && tid == 0) {
        const float loss = mt.bad ? __int_as_float(0x7fc00000) : a.tau * side;
        a.stats[2 * r] = ms.m;
        a.stats[2 * r + 1] = l2s;
        if (a.reduction == kNone) a.loss[r] = mt.w * loss;
        else a.row_loss[r] = mt.w * loss;
      }
      if constexpr (GRAD) {
        const T* row = static_cast<const T*>(a.z) + r * a.ldz;
        T* out = static_cast<T*>(a.dz) + r * a.lddz;
        const RowParts<T> parts(row, a.V);
        const long long v0 = min(parts.vecs, a.slice * rank), v1 = min(parts.vecs, v0 + a.slice);
        const int count = int(v1 - v0);
        const uint4* src = held;
        const float f = mt.bad ? __int_as_float(0x7fc00000) : mt.w * a.tau;
        const Prob<T> q(c, ms.m, l2s);
        T* dst = out + parts.head + v0 * E;
        grad_slice<T>(src, dst, tid, count, kStreamWarps * 32, q, f);
        const long long tail0 = parts.head + parts.vecs * E;
        if (rank == 0 && tid < parts.head) store1(out + tid, f * q(mt.head[tid]));
        if (rank == cluster - 1 && tid < parts.tail) store1(out + tail0 + tid, f * q(mt.tail[tid]));
        compute_sync();  // the entries' elements are written again, from both terms
        const long long lo = rank == 0 ? 0 : parts.head + v0 * E;
        const long long hi = rank == cluster - 1 ? a.V : parts.head + v1 * E;
        const int top_at = int(n & 1);
        const TeacherSmem top{top_p + top_at * Kp, top_id + top_at * Kp, nullptr};
        for (int k = tid; k < a.K; k += kStreamWarps * 32) {
          const int id = top.id[k];
          if (id < lo || id >= hi) continue;
          store1(out + id, f * (q(slice_logit<T>(src, mt, parts, v0, id)) - teacher_p(top, a.K, k)));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&empty));
    };
    // Leaving early: a warp whose wait ran out goes to the vote behind the loop and
    // meets the others at their next one (in the loop or behind it), where all of
    // them learn of it and leave.  So every warp comes to the same number of votes
    // (and of finish's barriers: one for every row whose vote passed).
    bool ok = true, all = true;  // this warp's waits were well; every warp's, by the last vote
    long long n = 0, r = first;
    for (; r < a.N; r += step, ++n) {
      ok = wait_for(full, uint32_t(n & 1));
      if (!ok) break;
      const RowMeta& mt = meta;
      const T* row = static_cast<const T*>(a.z) + r * a.ldz;
      const RowParts<T> parts(row, a.V);
      const long long v0 = min(parts.vecs, a.slice * rank), v1 = min(parts.vecs, v0 + a.slice);
      const int count = int(v1 - v0);
      if (mt.skip) {
        if constexpr (GRAD) {
          T* out = static_cast<T*>(a.dz) + r * a.lddz;
          T* dst = out + parts.head + v0 * E;
          const bool aligned = (reinterpret_cast<uintptr_t>(dst) & 15) == 0;
          for (int i = tid; i < count; i += kStreamWarps * 32)
            put_vec<T>(dst + (long long)i * E, make_uint4(0, 0, 0, 0), aligned);
          if (rank == 0 && tid < parts.head) out[tid] = T(0);
          if (rank == cluster - 1 && tid < parts.tail) out[parts.head + parts.vecs * E + tid] = T(0);
        }
        if (rank == 0 && tid == 0) {
          a.stats[2 * r] = a.stats[2 * r + 1] = 0.f;
          if (a.reduction == kNone) a.loss[r] = 0.f;
          else a.row_loss[r] = 0.f;
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&empty));
        continue;
      }
      const uint4* src = held;
      Running<T> run(c);
      if (rank == 0 && tid < parts.head) run.add1(mt.head[tid]);
      if (rank == cluster - 1 && tid < parts.tail) run.add1(mt.tail[tid]);
      run.add_slice(src, tid, count, kStreamWarps * 32);
      MaxSum ms = run.ms;
      ms = warp_pair<32>(ms, c);
      flip ^= 1;  // the last row's parts may still be read
      if (lane == 0) {
        part[flip][warp][0] = ms.m;
        part[flip][warp][1] = ms.s;
      }
      ok = wait_for(top_full, uint32_t(n & 1));
      all = compute_all(ok);
      if (!all) break;
      ms = warp_pair<kStreamWarps>({part[flip][lane % kStreamWarps][0], part[flip][lane % kStreamWarps][1]}, c);
      // the entries' part of the loss, now relative to the slice's maximum (in a closed slice it is infinite already)
      float side = mt.side, P = mt.P, slice_m = ms.m;
      if (P != 0.f && slice_m > -INFINITY) side = fmaf(P, slice_m - mt.top, side);
      if (cluster > 1) {
        const int at = int(counted % kSlots);
        if (warp == 0 && lane < cluster) {  // one lane per CTA of the cluster
          const uint32_t to = mapa_shared(smem_u32(&slot[at][rank]), uint32_t(lane));
          asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(ms.m), "f"(ms.s), "f"(side),
                       "f"(P)
                       : "memory");
          mbar_arrive_remote(mapa_shared(smem_u32(&slot_bar[at]), uint32_t(lane)));
        }
        __syncwarp();
        ok = mbar_wait_parked<true>(smem_u32(&slot_bar[at]), uint32_t(counted / kSlots) & 1u, a.status, &gave_up,
                                    a.wait_ns);
        if (!ok) {
          if constexpr (GRAD) compute_sync();  // finish's
          break;
        }
        float4 of{-INFINITY, 0.f, 0.f, 0.f};
        if (lane % kMaxCluster < cluster) of = slot[at][lane % kMaxCluster];
        ms = warp_pair<kMaxCluster>({of.x, of.y}, c);
        slice_m = of.x;
        side = of.z;
        P = of.w;
        ++counted;
      }
      finish(n, ms, slice_m, side, P);
    }
    if (all) all = compute_all(ok);
    if (!all && rank == 0 && tid == 0)  // rows without a loss
      for (float* to = a.reduction == kNone ? a.loss : a.row_loss; r < a.N; r += step) to[r] = __int_as_float(0x7fc00000);
  }
  __syncwarp();
  if (cluster > 1) cluster_sync();  // no CTA leaves while another may still write its slots
  if (a.reduction == kNone || rank != 0) return;
  // reduction: the last cluster to arrive adds all rows, in row order
  __syncthreads();
  if (tid == 0) {
    __threadfence();
    last_row = atomicAdd(a.counter, 1u) == unsigned(step - 1);
  }
  __syncthreads();
  if (!last_row) return;
  __threadfence();
  float sum = 0.f;
  if (warp < kStreamWarps)
    for (long long i = tid; i < a.N; i += kStreamWarps * 32) sum += __ldcg(a.row_loss + i);
  sum = warp_reduce(sum, [](float x, float y) { return x + y; });
  if (lane == 0 && warp < kStreamWarps) final_part[warp] = sum;
  __syncthreads();
  if (tid == 0) {
    sum = 0.f;
    for (int i = 0; i < kStreamWarps; ++i) sum += final_part[i];
    *a.loss = sum;
  }
}

// Backward for any upstream gradient: the gradient again from the logits and
// the forward's statistics.  Work item: one of `pieces` pieces of a row.  Bound
// by HBM: 8192 rows of 131072 bf16 logits 1040 us, 4.1 TB/s; 2 us when every
// upstream gradient is 1 and there is nothing to do.
template <typename T>
__global__ void __launch_bounds__(kThreads) distill_bwd_kernel(const Args a, int pieces) {
  constexpr int E = Vec16<T>::N;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ float teacher_scratch[kWarps];
  float* teacher_p0 = reinterpret_cast<float*>(smem_raw);
  const TeacherSmem teacher{teacher_p0, reinterpret_cast<int*>(teacher_p0 + padded_top(a.K)), teacher_scratch};
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
    if (w != 0.f) tch = load_teacher<kThreads>(a, r, teacher);
    if (w == 0.f || !(tch.any || tch.bad)) {
      const uint4 zero = make_uint4(0, 0, 0, 0);
      for (long long i = v0 + tid; i < v1; i += kThreads) put_vec<T>(out + part.head + i * E, zero, out_aligned);
      if (first && tid < part.head) out[tid] = T(0);
      if (last && tid < part.tail) out[part.head + part.vecs * E + tid] = T(0);
      continue;
    }
    const float c = kLog2e / a.tau;
    const Prob<T> q(c, a.stats[2 * r], a.stats[2 * r + 1]);
    const float f = tch.bad ? __int_as_float(0x7fc00000) : up * w * a.tau;
    const float off = f > 0.f ? grad_offset(q, f) : 0.f;
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
          put_vec<T>(out + part.head + (i0 + u * kThreads) * E,
                     q.plain && f > 0.f ? grad_vec<T, true>(x[u], q, f, off) : grad_vec<T, false>(x[u], q, f, 0.f),
                     out_aligned);
    }
    if (first && tid < part.head) store1(out + tid, f * q(load1(row + tid)));
    if (last && tid < part.tail) {
      const long long i = part.head + part.vecs * E + tid;
      store1(out + i, f * q(load1(row + i)));
    }
    __syncthreads();
    const long long lo = first ? 0 : part.head + v0 * E;
    const long long hi = last ? a.V : part.head + v1 * E;
    for (int k = tid; k < a.K; k += kThreads) {
      const int id = teacher.id[k];
      if (id < lo || id >= hi) continue;
      store1(out + id, f * (q(load1(row + id)) - teacher_p(teacher, a.K, k)));
    }
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// distill_row_kernel: shared memory a CTA holds of a row, up to 72 KB, so that
// three CTAs fit on an SM and one's loads overlap another's arithmetic; slices
// of rows that are longer than that times the largest cluster take up to 208 KB.
constexpr long long kSliceVecs = 72 * 1024 / 16;
constexpr long long kTileVecs = 208 * 1024 / 16;
constexpr size_t kTopBytes = size_t(kMaxTop) * 8;
// distill_stream_kernel: dynamic shared memory of a CTA, three to a SM.
constexpr size_t kStreamSmem = 73 * 1024;
// rows that distill_row_kernel takes with kShortThreads threads
constexpr long long kShortBytes = 48 * 1024;

// b2_distill_set_wait_limit
std::atomic<unsigned long long> g_wait_ns{kWaitLimitNs};

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

// Once per kernel and device (`done`: a static of the caller).
template <typename F>
b2_status allow_smem(F kern, size_t bytes, bool (&done)[64], int dev) {
  if (dev < 0 || dev >= 64) return set_error(B2_ERR_INVALID, "device index %d", dev);
  if (done[dev]) return B2_OK;
  B2_TRY(check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)),
                    "cudaFuncSetAttribute(distill)"));
  done[dev] = true;
  return B2_OK;
}

void cluster_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute& attr, long long clusters, int cluster, int threads,
                    size_t smem, cudaStream_t st) {
  cfg.gridDim = dim3(unsigned(clusters * cluster));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(cluster);
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
}

template <typename K, typename... A>
b2_status launch_clusters(K kern, long long clusters, int cluster, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  cluster_config(cfg, attr, clusters, cluster, threads, smem, st);
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, args...), "distill forward launch");
}

template <typename T, bool GRAD>
b2_status launch_fwd(Args a, cudaStream_t st) {
  int dev = 0;
  B2_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
  const int sms = sm_count(dev);
  const long long vecs = (a.V * (long long)sizeof(T) + 15) / 16;
  int cluster = 1;
  const size_t top = size_t(padded_top(a.K)) * 8;
  while (cluster < kMaxCluster && size_t((vecs + cluster - 1) / cluster) * 16 + 2 * top > kStreamSmem) cluster *= 2;
  a.slice = (vecs + cluster - 1) / cluster;
  const size_t held = size_t(a.slice) * 16 + 2 * top;
  const bool many = a.N * cluster >= 2LL * kStreamPerSm * sms;
  if (many && vecs * 16 <= kShortBytes) {
    // Many short rows: a CTA each, of half the threads, so that twice as many
    // rows overlap their latencies (8192 rows with the gradient: 2000 bf16 logits
    // 50 us, with all threads 81, in the persistent kernel 76; 16000 logits 121,
    // 143 and 146; 24000 logits 173 and 185 in the persistent one, 2000 rows of
    // 32000 68 and 64; 500 rows of 2000 11.1 us against 10.7 with all threads).
    a.slice = a.tile = vecs;
    auto kern = distill_row_kernel<T, GRAD, kShortThreads>;
    static bool configured[64] = {};
    B2_TRY(allow_smem(kern, kShortBytes + kTopBytes, configured, dev));
    return launch_clusters(kern, a.N, 1, kShortThreads, size_t(vecs) * 16 + top, st, a, 1);
  }
  // Persistent clusters where every CTA gets at least two slices, else CTAs of a
  // row's own (bf16, with the gradient): 8192 x 131072 864 us against 958; 300 x
  // 32000 18.4 against 17.1, 148 x 32000 13.3 against 12.5, where rows are too
  // few; the same at 1800 x 32000 (59).
  if (many && held <= kStreamSmem) {
    auto kern = distill_stream_kernel<T, GRAD>;
    static bool configured[64] = {};
    B2_TRY(allow_smem(kern, kStreamSmem, configured, dev));
    // as many clusters as are resident at once: a later one would run alone at the end
    static int resident[64][kMaxCluster + 1] = {};
    int& clusters = resident[dev][cluster];
    if (!clusters) {
      cudaLaunchConfig_t cfg{};
      cudaLaunchAttribute attr{};
      cluster_config(cfg, attr, kStreamPerSm * sms / cluster, cluster, kStreamThreads, kStreamSmem, st);
      int n = 0;
      B2_TRY(check_cuda(cudaOccupancyMaxActiveClusters(&n, kern, &cfg), "cudaOccupancyMaxActiveClusters"));
      if (n < 1) return set_error(B2_ERR_CUDA, "distill: no cluster of %d fits", cluster);
      clusters = std::min(n, kStreamPerSm * sms / cluster);
    }
    return launch_clusters(kern, clusters, cluster, kStreamThreads, held, st, a, cluster);
  }
  // longer rows over more CTAs; so are few rows, down to 4 KB a CTA
  cluster = 1;
  while (cluster < kMaxCluster && ((vecs + cluster - 1) / cluster > kSliceVecs ||
                                   (a.N * cluster < sms && vecs / cluster >= 512)))
    cluster *= 2;
  a.slice = (vecs + cluster - 1) / cluster;
  a.tile = std::min(a.slice, a.slice <= kSliceVecs ? kSliceVecs : kTileVecs);
  auto kern = distill_row_kernel<T, GRAD, kThreads>;
  static bool configured[64] = {};
  B2_TRY(allow_smem(kern, size_t(kTileVecs) * 16 + kTopBytes, configured, dev));
  return launch_clusters(kern, a.N, cluster, kThreads, size_t(a.tile) * 16 + top, st, a, cluster);
}

template <typename T>
b2_status launch_bwd(Args a, cudaStream_t st) {
  int dev = 0;
  B2_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
  const long long vecs = (a.V * (long long)sizeof(T) + 15) / 16;
  const int pieces = int(std::max<long long>(1, std::min<long long>(64, vecs / 2048)));
  a.slice = (vecs + pieces - 1) / pieces;
  const long long grid = std::min<long long>(a.N * pieces, (long long)sm_count(dev) * 8);
  distill_bwd_kernel<T><<<unsigned(grid), kThreads, size_t(padded_top(a.K)) * 8, st>>>(a, pieces);
  return check_cuda(cudaGetLastError(), "distill backward launch");
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

b2_status b2_distill_set_wait_limit(int64_t ns) {
  if (ns < 0) return set_error(B2_ERR_INVALID, "b2_distill_set_wait_limit: negative limit");
  g_wait_ns.store(ns ? (unsigned long long)ns : kWaitLimitNs, std::memory_order_relaxed);
  return B2_OK;
}

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
  a.wait_ns = g_wait_ns.load(std::memory_order_relaxed);
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
