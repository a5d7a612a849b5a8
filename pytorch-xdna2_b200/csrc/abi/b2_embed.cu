// Token embedding: scaled row lookup and its dense weight gradient.
//
//   forward   y[t][:]  = scale * W[id_t][:]
//   backward  dW[v][:] = scale * sum over the tokens t with id_t == v, in token
//             order, of dy[t][:]; rows without a token (and the padding row)
//             are zero
//
// Both are bound by HBM: the lookup moves T*D elements in and out, the
// gradient reads T*D elements of dy and writes all V*D of dW.
//
// The backward sorts the tokens by id (a stable least-significant-digit radix
// sort of (id, token) pairs, written here), so that a row's tokens are
// neighbours: every dy row is read once, every dW row is written once, the
// sums are fp32 in a fixed order (bit-reproducible, no atomics on values) and
// one frequent token spreads over many CTAs.  The sorted list is cut into
// pieces of kPiece tokens whatever their ids; a run of equal ids inside one
// piece is written directly, a run that crosses pieces leaves fp32 partial rows
// that a last kernel adds in piece order.
#include <algorithm>

#include "b2_common.cuh"

namespace b2 {
namespace {

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kDigitBits = 9;  // widest digit; 512 counters per warp
constexpr int kDigits = 1 << kDigitBits;
constexpr int kPiece = 32;     // sorted tokens per accumulation piece
constexpr int kAccThreads = 256;

template <int BYTES>
struct Vec;
template <>
struct Vec<16> { using type = uint4; };
template <>
struct Vec<8> { using type = uint2; };
template <>
struct Vec<4> { using type = uint32_t; };
template <>
struct Vec<2> { using type = uint16_t; };

// N consecutive elements (T: uint16_t = bf16 bits, or float) <-> fp32
template <typename T, int N>
struct Pack {
  using V = typename Vec<sizeof(T) * N>::type;
  union {
    V v;
    T e[N];
  };
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 2) return bf2f(e[i]);
    else return e[i];
  }
  __device__ __forceinline__ void set(int i, float f) {
    if constexpr (sizeof(T) == 2) {
      __nv_bfloat16 h = __float2bfloat16_rn(f);
      e[i] = *reinterpret_cast<uint16_t*>(&h);
    } else {
      e[i] = f;
    }
  }
};

__device__ __forceinline__ long long load_id(const void* ids, int is64, long long t) {
  return is64 ? static_cast<const long long*>(ids)[t] : (long long)static_cast<const int*>(ids)[t];
}

// ---------------------------------------------------------------------------
// forward: `lanes` threads (a power of two) walk one row, 256 / lanes rows per
// CTA, U rows' loads in flight per thread.  An id outside [0, V) gives a row of
// NaN and B2_ERR_INVALID in the device status word; nothing out of range is read.
// Bound by HBM: 65536 tokens of 131072 x 2048 bf16 rows 76 us (one row in flight a
// thread 87, eight 76), 0.54 GB with repeated rows; few tokens by latency (16 rows
// of 1024 bf16 in two CTAs 4 us), and where a row has more than 256 vectors their
// columns are spread over CTAs.
// ---------------------------------------------------------------------------
template <typename T, int N, int U>
__global__ void __launch_bounds__(256) embed_fwd_kernel(const void* __restrict__ ids, int is64, long long tokens,
                                                        const T* __restrict__ w, long long ldw, long long V,
                                                        int vecs, int log_lanes, float scale, T* __restrict__ y,
                                                        long long D, int* status) {
  const int lane = threadIdx.x & ((1 << log_lanes) - 1);
  const int rows_per_pass = 256 >> log_lanes;
  const long long t0 = (long long)blockIdx.x * rows_per_pass * U + (threadIdx.x >> log_lanes);
  long long id[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long t = t0 + (long long)u * rows_per_pass;
    id[u] = t < tokens ? load_id(ids, is64, t) : -1;
    if (t < tokens && (id[u] < 0 || id[u] >= V)) {
      id[u] = -1;
      if (lane == 0 && blockIdx.y == 0) record_status(status, B2_ERR_INVALID);
    }
  }
  for (int c = blockIdx.y * (1 << log_lanes) + lane; c < vecs; c += gridDim.y << log_lanes) {
    Pack<T, N> p[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (id[u] >= 0) p[u].v = reinterpret_cast<const typename Pack<T, N>::V*>(w + id[u] * ldw)[c];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long long t = t0 + (long long)u * rows_per_pass;
      if (t >= tokens) continue;
#pragma unroll
      for (int i = 0; i < N; ++i)
        p[u].set(i, id[u] >= 0 ? scale * p[u].get(i) : __int_as_float(0x7fc00000));
      reinterpret_cast<typename Pack<T, N>::V*>(y + t * D)[c] = p[u].v;
    }
  }
}

// ---------------------------------------------------------------------------
// the sort
// ---------------------------------------------------------------------------

// Sort key of a token: its id, or V for a token that contributes to no row
// (the padding id; an id out of range, reported by the forward).
__device__ __forceinline__ uint32_t key_of(const void* ids, int is64, long long t, long long V, long long pad) {
  const long long id = load_id(ids, is64, t);
  return (id < 0 || id >= V || id == pad) ? uint32_t(V) : uint32_t(id);
}

// Shared memory of a sorting CTA: per warp one counter per digit, then the
// digits' CTA-wide values.
struct SortSmem {
  uint32_t count[kSortWarps][kDigits];
  uint32_t digit[kDigits];
  uint32_t scan[kSortWarps];
};

// Exclusive prefix sum over 512 values held one per thread by threads 0..511
// (all threads call).
__device__ __forceinline__ uint32_t scan512(uint32_t v, uint32_t* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t n = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += n;
  }
  __syncthreads();
  if (lane == 31) scratch[warp] = x;
  __syncthreads();
  uint32_t before = 0;
  for (int i = 0; i < warp && i < 16; ++i) before += scratch[i];
  return before + x - v;
}

// Stable ranks of this CTA's items by one digit.  Item i of a thread sits at
// position warp * 32 * I + i * 32 + lane of the CTA's chunk.  On return rank[i]
// is the item's place among the warp's equal digits and s.count[w][d] the
// exclusive prefix over warps of digit d; the digit totals are in s.digit.
template <int I>
__device__ __forceinline__ void rank_items(SortSmem& s, const uint32_t (&key)[I], const bool (&valid)[I], int shift,
                                           uint32_t mask, uint32_t (&rank)[I]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int ndig = int(mask) + 1;
  for (int d = lane; d < ndig; d += 32) s.count[warp][d] = 0;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const uint32_t d = (key[i] >> shift) & mask;
    const uint32_t peers = __match_any_sync(0xffffffffu, valid[i] ? d : 0xffffffffu);
    const uint32_t before = __popc(peers & ((1u << lane) - 1));
    uint32_t base = 0;
    if (valid[i]) base = s.count[warp][d];
    __syncwarp();
    rank[i] = base + before;
    if (valid[i] && before == 0) s.count[warp][d] = base + __popc(peers);
    __syncwarp();
  }
  __syncthreads();
  for (int d = threadIdx.x; d < ndig; d += kSortThreads) {
    uint32_t run = 0;
#pragma unroll 8
    for (int w = 0; w < kSortWarps; ++w) {
      const uint32_t c = s.count[w][d];
      s.count[w][d] = run;
      run += c;
    }
    s.digit[d] = run;
  }
  __syncthreads();
}

// Up to kRankTokens tokens: a token's place is the number of smaller keys and of
// equal keys before it, counted over all keys in shared memory by kRankSplit
// threads a token.  Quadratic, but one launch over all SMs: 3000 tokens take 5 us,
// where a radix sort in one CTA took 10; 8192 tokens 16 us, the passes below 13.
constexpr int kRankTokens = 4096;
constexpr int kRankThreads = 256;
constexpr int kRankSplit = 8;
constexpr int kRankPerBlock = kRankThreads / kRankSplit;
__global__ void __launch_bounds__(kRankThreads)
    embed_rank_kernel(const void* __restrict__ ids, int is64, int tokens, long long V, long long pad,
                      uint32_t* __restrict__ key_out, uint32_t* __restrict__ tok_out) {
  __shared__ __align__(16) uint32_t keys[kRankTokens];
  chain_release();
  const int quads = (tokens + 3) / 4;
#pragma unroll 8
  for (int i = threadIdx.x; i < quads * 4; i += kRankThreads)
    keys[i] = i < tokens ? key_of(ids, is64, i, V, pad) : 0xffffffffu;
  __syncthreads();
  const int part = threadIdx.x % kRankSplit;
  const int first = blockIdx.x * kRankPerBlock;          // this CTA's tokens, a multiple of 4
  const int t = first + threadIdx.x / kRankSplit;
  const uint32_t mine = t < tokens ? keys[t] : 0;
  unsigned rank = 0;
  const uint4* q = reinterpret_cast<const uint4*>(keys);
  // keys before this CTA's tokens count when equal, keys behind them do not
  const int before = first / 4, behind = (first + kRankPerBlock) / 4;
#pragma unroll 4
  for (int i = part; i < before; i += kRankSplit) {
    const uint4 v = q[i];
    rank += unsigned(v.x <= mine) + unsigned(v.y <= mine) + unsigned(v.z <= mine) + unsigned(v.w <= mine);
  }
#pragma unroll 4
  for (int i = behind + part; i < quads; i += kRankSplit) {
    const uint4 v = q[i];
    rank += unsigned(v.x < mine) + unsigned(v.y < mine) + unsigned(v.z < mine) + unsigned(v.w < mine);
  }
  for (int i = first + part; i < min(first + kRankPerBlock, tokens); i += kRankSplit)
    rank += unsigned(keys[i] < mine || (keys[i] == mine && i < t));
#pragma unroll
  for (int o = 1; o < kRankSplit; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
  if (part == 0 && t < tokens) {
    key_out[rank] = mine;
    tok_out[rank] = uint32_t(t);
  }
}

// Many CTAs, one launch per digit.  table[p][b][d]: tokens of chunk b with
// digit d at the start of pass p.  This kernel fills pass 0's table and zeroes
// the later ones; each pass adds up the next one's while it scatters.  65536
// tokens, 131072 ids: 3 us here and 8 a pass, two of them.
__global__ void __launch_bounds__(kSortThreads)
    embed_hist_kernel(const void* __restrict__ ids, int is64, long long tokens, long long V, long long pad, int passes,
                      int bits, int chunk, uint32_t* __restrict__ table) {
  __shared__ uint32_t h[kDigits];
  chain_release();
  const uint32_t mask = (1u << bits) - 1;
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) h[d] = 0;
  __syncthreads();
  const long long t0 = (long long)blockIdx.x * chunk;
  const long long t1 = min(tokens, t0 + chunk);
  for (long long t = t0 + threadIdx.x; t < t1; t += kSortThreads)
    atomicAdd(&h[key_of(ids, is64, t, V, pad) & mask], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < kDigits; d += kSortThreads) {
    table[(long long)blockIdx.x * kDigits + d] = h[d];
    for (int p = 1; p < passes; ++p) table[((long long)p * gridDim.x + blockIdx.x) * kDigits + d] = 0;
  }
}

template <int I>
__global__ void __launch_bounds__(kSortThreads)
    embed_pass_kernel(const void* __restrict__ ids, int is64, long long tokens, long long V, long long pad, int pass,
                      int passes, int bits, uint32_t* __restrict__ table, const uint32_t* __restrict__ key_in,
                      const uint32_t* __restrict__ tok_in, uint32_t* __restrict__ key_out,
                      uint32_t* __restrict__ tok_out) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  SortSmem& s = *reinterpret_cast<SortSmem*>(smem_raw);
  chain_wait();
  chain_release();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int shift = pass * bits;
  const uint32_t mask = (1u << bits) - 1;
  constexpr int kChunk = kSortThreads * I;
  uint32_t key[I], tok[I], rank[I];
  bool valid[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const long long pos = (long long)blockIdx.x * kChunk + warp * 32 * I + i * 32 + lane;
    valid[i] = pos < tokens;
    key[i] = tok[i] = 0;
    if (valid[i]) {
      if (pass == 0) {
        tok[i] = uint32_t(pos);
        key[i] = key_of(ids, is64, pos, V, pad);
      } else {
        key[i] = key_in[pos];
        tok[i] = tok_in[pos];
      }
    }
  }
  // this chunk's first place for every digit: smaller digits of all chunks,
  // then the same digit in earlier chunks
  const uint32_t* tab = table + (long long)pass * gridDim.x * kDigits;
  uint32_t before = 0, total = 0;
  if (threadIdx.x <= mask) {
#pragma unroll 8
    for (int b = 0; b < int(gridDim.x); ++b) {
      const uint32_t c = tab[(long long)b * kDigits + threadIdx.x];
      total += c;
      if (b < int(blockIdx.x)) before += c;
    }
  }
  rank_items<I>(s, key, valid, shift, mask, rank);
  const uint32_t base = scan512(total, s.scan) + before;
  if (threadIdx.x <= mask) s.digit[threadIdx.x] = base;
  __syncthreads();
  uint32_t* next = table + (long long)(pass + 1) * gridDim.x * kDigits;
#pragma unroll
  for (int i = 0; i < I; ++i) {
    uint32_t pos = 0;
    if (valid[i]) {
      const uint32_t d = (key[i] >> shift) & mask;
      pos = s.digit[d] + s.count[warp][d] + rank[i];
      key_out[pos] = key[i];
      tok_out[pos] = tok[i];
    }
    if (pass + 1 < passes) {
      // one integer atomic per distinct (chunk, digit) of the warp
      const uint32_t slot = valid[i] ? (pos / kChunk) * kDigits + ((key[i] >> (shift + bits)) & mask) : 0xffffffffu;
      const uint32_t peers = __match_any_sync(0xffffffffu, slot);
      if (valid[i] && (peers & ((1u << lane) - 1)) == 0) atomicAdd(next + slot, uint32_t(__popc(peers)));
    }
  }
}

// ---------------------------------------------------------------------------
// accumulation.  CTAs [0, acc_blocks) add the pieces' rows; the CTAs behind
// them write zeros to the rows of dW that no token has.
// ---------------------------------------------------------------------------

// First position of the sorted keys with key >= want (all 256 threads call).
__device__ __forceinline__ long long lower_bound(const uint32_t* __restrict__ key, long long n, uint32_t want) {
  long long lo = 0;
  while (n > 0) {
    const long long step = (n + kAccThreads - 1) / kAccThreads;
    const long long at = (long long)(threadIdx.x + 1) * step - 1;
    const int below = __syncthreads_count(at < n && key[lo + at] < want);
    lo += below * step;
    // the answer lies in the first block whose last key is not below `want`
    // (if it has a last key), without that key itself when it has been tested
    n = min(step - 1, n - below * step);
    if (n < 0) n = 0;
  }
  return lo;
}

template <typename T, int N>
__device__ __forceinline__ void store_row(T* row, int c, const float (&acc)[N], float scale) {
  Pack<T, N> p;
#pragma unroll
  for (int i = 0; i < N; ++i) p.set(i, scale * acc[i]);
  reinterpret_cast<typename Pack<T, N>::V*>(row)[c] = p.v;
}

// Zeros to the rows of `base` (rows x width) that are not present (all threads of
// the CTA call).  The rows' elements are taken as one range: its whole 16-byte
// vectors, whatever the row length (a vector over two rows goes element by
// element).
template <typename T>
__device__ __forceinline__ void zero_absent(T* base, int rows, unsigned width, const uint8_t* present) {
  constexpr int E = 16 / sizeof(T);
  const unsigned total = unsigned(rows) * width;  // about 64 KB, or one row
  const unsigned head = min(total, unsigned((16 - (reinterpret_cast<uintptr_t>(base) & 15)) & 15) / unsigned(sizeof(T)));
  const unsigned whole = (total - head) / E;
  for (unsigned v = threadIdx.x; v < whole; v += kAccThreads) {
    const unsigned e0 = head + v * E;
    const unsigned first_row = e0 / width, last_row = (e0 + E - 1) / width;
    if (first_row == last_row) {
      if (!present[first_row]) *reinterpret_cast<uint4*>(base + e0) = make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (!present[(e0 + i) / width]) base[e0 + i] = T(0);
    }
  }
  const unsigned tail = head + whole * E;
  if (threadIdx.x < head && !present[threadIdx.x / width]) base[threadIdx.x] = T(0);
  if (threadIdx.x < total - tail && !present[(tail + threadIdx.x) / width]) base[tail + threadIdx.x] = T(0);
}

// The whole gradient in one launch for few tokens: CTAs [0, token_blocks) give
// every token 1 << log_warps warps (a warp for up to 32 vectors of columns); the
// first token of an id adds the rows of all tokens that have it, in token order,
// eight loads in flight.  The CTAs behind them zero the absent rows.  512 tokens,
// 20000 x 256 bf16: 5.2 us, 12 with the sort below, and two launches less on the
// host.  A frequent id's rows are added by one group of warps one batch after
// the other, which is why this ends at kSmallTokens: 512 tokens of one id take
// 26 us here, 14 there.
constexpr int kSmallTokens = 512;
template <int U>
struct Batch {
  static constexpr int value = U;
};

template <typename T, int N>
__global__ void __launch_bounds__(kAccThreads, 4)
    embed_small_kernel(const void* __restrict__ ids, int is64, int tokens, long long V, long long pad,
                       const T* __restrict__ dy, long long lddy, int vecs, int log_warps, long long D, float scale,
                       T* __restrict__ dw, int slabs, long long token_blocks, int zero_rows) {
  if ((long long)blockIdx.x >= token_blocks) {
    __shared__ uint8_t present[512];
    const long long r0 = ((long long)blockIdx.x - token_blocks) * zero_rows;
    const int rows = int(min((long long)zero_rows, V - r0));
    for (int i = threadIdx.x; i < rows; i += kAccThreads) present[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < tokens; i += kAccThreads) {
      const long long k = (long long)key_of(ids, is64, i, V, pad) - r0;
      if (k >= 0 && k < rows) present[k] = 1;  // (a token without a row has key V, behind every row)
    }
    __syncthreads();
    zero_absent(dw + r0 * D, rows, unsigned(D), present);
    return;
  }
  __shared__ uint32_t keys[kSmallTokens];
  const int padded = (tokens + 31) / 32 * 32;
  for (int i = threadIdx.x; i < padded; i += kAccThreads)
    keys[i] = i < tokens ? key_of(ids, is64, i, V, pad) : 0xffffffffu;
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = int(blockIdx.x / slabs) * ((kAccThreads / 32) >> log_warps) + (warp >> log_warps);
  if (t >= tokens) return;
  const uint32_t mine = keys[t];
  if (mine >= V) return;
  for (int base = 0; base < t; base += 32)
    if (__any_sync(0xffffffffu, base + lane < t && keys[base + lane] == mine)) return;  // not the id's first token
  // the id's tokens, in order
  __shared__ uint16_t lists[kAccThreads / 32][kSmallTokens];
  uint16_t* list = lists[warp];
  int count = 0;
  for (int base = t / 32 * 32; base < padded; base += 32) {
    const unsigned found = __ballot_sync(0xffffffffu, keys[base + lane] == mine);
    if (found >> lane & 1) list[count + __popc(found & ((1u << lane) - 1))] = uint16_t(base + lane);
    count += __popc(found);
  }
  __syncwarp();
  const int c = ((int(blockIdx.x % slabs) << log_warps) + (warp & ((1 << log_warps) - 1))) * 32 + lane;
  const int at = min(c, vecs - 1);
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  auto add = [&](int first, auto batch) {
    constexpr int U = decltype(batch)::value;
    Pack<T, N> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      v[u].v = reinterpret_cast<const typename Pack<T, N>::V*>(dy + (long long)list[first + u] * lddy)[at];
    __syncwarp();  // keeps the batch's loads together: the compiler otherwise takes them one by one to save registers
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += v[u].get(i);
  };
  int n = 0;
  for (; n + 8 <= count; n += 8) add(n, Batch<8>{});
  for (; n + 4 <= count; n += 4) add(n, Batch<4>{});
  for (; n < count; ++n) add(n, Batch<1>{});
  if (c < vecs) store_row<T, N>(dw + (long long)mine * D, c, acc, scale);
}

// Sums of the sorted tokens' rows, a piece of kPiece tokens and up to 256 vectors
// of columns per group of threads, four rows in flight a thread; the CTAs behind
// the pieces' zero the absent rows meanwhile.  Bound by HBM: 65536 tokens of
// 131072 x 2048 bf16 133 us for the 0.8 GB read and written, 6.1 TB/s; 3001 of
// 50001 x 1001 fp32 37 us, 5.7 TB/s.
template <typename T, int N>
__global__ void __launch_bounds__(kAccThreads)
    embed_acc_kernel(const uint32_t* __restrict__ key, const uint32_t* __restrict__ tok, long long tokens, long long V,
                     const T* __restrict__ dy, long long lddy, int vecs, int log_lanes, long long D, float scale,
                     T* __restrict__ dw, float* __restrict__ partial, long long pieces, int slabs,
                     long long acc_blocks, int zero_rows) {
  chain_wait();
  if ((long long)blockIdx.x >= acc_blocks) {
    __shared__ uint8_t present[512];
    const long long r0 = ((long long)blockIdx.x - acc_blocks) * zero_rows;
    const int rows = int(min((long long)zero_rows, V - r0));
    for (int i = threadIdx.x; i < rows; i += kAccThreads) present[i] = 0;
    const long long lo = lower_bound(key, tokens, uint32_t(r0));
    __syncthreads();
    long long p = lo + threadIdx.x;
    bool more = true;
    for (int turn = 0; turn < 8 && more; ++turn, p += kAccThreads) {
      const bool in = p < tokens && key[p] < uint32_t(r0 + rows);
      if (in) present[key[p] - r0] = 1;
      more = __syncthreads_or(in);
    }
    if (more) {
      // Frequent ids: a search for every row instead of all their keys (200000
      // tokens of a Zipf-like draw, 50000 x 768 bf16: the kernel takes 88 us, 224
      // when one CTA reads the 70000 keys of the first rows).
      for (int i = threadIdx.x; i < rows; i += kAccThreads) {
        long long a = lo, b = tokens;
        while (a < b) {
          const long long mid = (a + b) >> 1;
          if (key[mid] < uint32_t(r0 + i))
            a = mid + 1;
          else
            b = mid;
        }
        if (a < tokens && key[a] == uint32_t(r0 + i)) present[i] = 1;
      }
    }
    __syncthreads();
    zero_absent(dw + r0 * D, rows, unsigned(D), present);
    return;
  }
  const int per_block = kAccThreads >> log_lanes;
  const int slab = int(blockIdx.x % slabs);
  const long long piece = ((long long)blockIdx.x / slabs) * per_block + (threadIdx.x >> log_lanes);
  const int c = (slab << log_lanes) + (threadIdx.x & ((1 << log_lanes) - 1));
  if (piece >= pieces || c >= vecs) return;
  const long long p0 = piece * kPiece, p1 = min(tokens, p0 + kPiece);
  const uint32_t none = 0xffffffffu;
  const uint32_t prev = p0 > 0 ? key[p0 - 1] : none;
  const uint32_t next = p1 < tokens ? key[p1] : none;
  float acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  uint32_t cur = key[p0];
  bool begins = cur != prev;  // the current run starts in this piece
  constexpr int U = 4;
  for (long long p = p0; p < p1; p += U) {
    uint32_t k[U];
    Pack<T, N> v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      k[u] = p + u < p1 ? key[p + u] : none;
      if (k[u] < V) v[u].v = reinterpret_cast<const typename Pack<T, N>::V*>(dy + (long long)tok[p + u] * lddy)[c];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k[u] == none) break;
      if (k[u] != cur) {
        // the run of `cur` ends here
        if (begins)
          store_row<T, N>(dw + (long long)cur * D, c, acc, scale);
        else
#pragma unroll
          for (int i = 0; i < N; ++i) partial[(2 * piece) * D + (long long)c * N + i] = acc[i];
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = 0.f;
        cur = k[u];
        begins = true;
      }
      if (k[u] >= V) return;  // only tokens without a row follow
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] += v[u].get(i);
    }
  }
  if (begins && cur != next) {
    store_row<T, N>(dw + (long long)cur * D, c, acc, scale);
  } else {
    // slot 0: a run that came from the piece before; slot 1: one that starts here and goes on
    float* out = partial + (2 * piece + (begins ? 1 : 0)) * D + (long long)c * N;
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = acc[i];
  }
}

// Adds the partial rows of every run that crosses pieces, for 32 vectors of
// columns.  A warp looks after one piece: it finds the end of a run that starts
// there and goes on (32 pieces a look) and adds a short one's rows by itself, in
// piece order; a run over more than kShortRun pieces (a frequent token's has
// hundreds) is shared by the CTA's warps, every eighth piece each, and their
// sums are added in warp order.  65536 tokens of a Zipf-like draw: 17 us.
constexpr int kJoinWarps = kAccThreads / 32;
constexpr int kShortRun = 16;
template <typename T, int N>
__global__ void __launch_bounds__(kAccThreads)
    embed_join_kernel(const uint32_t* __restrict__ key, long long tokens, long long V, int vecs, long long D,
                      float scale, T* __restrict__ dw, const float* __restrict__ partial, long long pieces) {
  __shared__ float sums[kJoinWarps][N][32];
  __shared__ uint32_t long_key[kJoinWarps];
  __shared__ long long long_last[kJoinWarps];
  chain_wait();
  const uint32_t none = 0xffffffffu;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int c = blockIdx.y * 32 + lane;
  const long long first = (long long)blockIdx.x * kJoinWarps, piece = first + warp;
  const long long p0 = piece * kPiece, p1 = p0 + kPiece;
  uint32_t k = none;
  long long last = piece;  // the last piece of the run
  if (p1 < tokens) {  // the last piece's runs all end in it
    k = key[p1 - 1];
    const uint32_t next = key[p1], begin = key[p0], before = p0 > 0 ? key[p0 - 1] : none;
    if (k >= V || next != k || (begin == k && before == k)) k = none;  // none goes on, or it started earlier
  }
  if (k != none) {
    // 32 pieces a step, then the pieces of the last step
    for (;;) {
      const long long q = last + 32 * (lane + 1);
      const unsigned same = __ballot_sync(0xffffffffu, q < pieces && key[q * kPiece] == k);
      const int more = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
      last += 32 * more;
      if (more < 32) break;
    }
    for (;;) {
      const long long q = last + 1 + lane;
      const unsigned same = __ballot_sync(0xffffffffu, q < pieces && key[q * kPiece] == k);
      const int more = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
      last += more;
      if (more < 32) break;
    }
  }
  // slot 1 of the piece where the run starts, slot 0 of the others
  auto add = [&](float (&acc)[N], long long q, long long start) {
    const float* pp = partial + (2 * q + (q == start ? 1 : 0)) * D + (long long)c * N;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] += pp[i];
  };
  const bool is_long = k != none && last - piece >= kShortRun;
  if (k != none && !is_long && c < vecs) {
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
#pragma unroll 4
    for (long long q = piece; q <= last; ++q) add(acc, q, piece);
    store_row<T, N>(dw + (long long)k * D, c, acc, scale);
  }
  if (lane == 0) {
    long_key[warp] = is_long ? k : none;
    long_last[warp] = last;
  }
  if (!__syncthreads_or(is_long)) return;
  for (int j = 0; j < kJoinWarps; ++j) {
    const uint32_t kj = long_key[j];
    if (kj == none) continue;
    const long long start = first + j, end = long_last[j];
    float acc[N];
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] = 0.f;
    if (c < vecs)
#pragma unroll 8
      for (long long q = start + warp; q <= end; q += kJoinWarps) add(acc, q, start);
#pragma unroll
    for (int i = 0; i < N; ++i) sums[warp][i][lane] = acc[i];
    __syncthreads();
    if (warp == 0 && c < vecs) {
#pragma unroll
      for (int w = 1; w < kJoinWarps; ++w)
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] += sums[w][i][lane];
      store_row<T, N>(dw + (long long)kj * D, c, acc, scale);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

// Widest vector (elements of `size` bytes, at most 16 bytes) that divides the
// row length and strides and to which the pointers are aligned.
int vec_elems(int size, int64_t D, int64_t ld, const void* a, const void* b) {
  int n = 16 / size;
  while (n > 1 && (D % n || ld % n || reinterpret_cast<uintptr_t>(a) % (size_t(n) * size) ||
                   reinterpret_cast<uintptr_t>(b) % (size_t(n) * size)))
    n /= 2;
  return n;
}

int log_lanes_for(int vecs) {
  int l = 0;
  while (l < 8 && (1 << l) < vecs) ++l;
  return l;
}

// rows of dW a zeroing CTA looks after: about 64 KB
int zero_rows_for(int64_t D, size_t size) {
  return int(std::max<int64_t>(1, std::min<int64_t>(512, 65536 / (D * int64_t(size)))));
}

struct SortPlan {
  int passes, bits;
  bool one;      // by counting ranks, in one launch
  int items;     // tokens per thread
  int64_t blocks;
};

SortPlan sort_plan(int64_t T, int64_t V) {
  SortPlan p{};
  int bits = 1;
  while (bits < 32 && (int64_t(1) << bits) <= V) ++bits;  // keys 0 .. V
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.one = T <= kRankTokens;
  p.items = T <= 128 * 2 * kSortThreads ? 2 : 8;
  p.blocks = (T + int64_t(p.items) * kSortThreads - 1) / (int64_t(p.items) * kSortThreads);
  return p;
}

struct EmbedWs {
  size_t key0, tok0, key1, tok1, table, partial, total;
};

EmbedWs embed_ws(int64_t T, int64_t V, int64_t D) {
  const SortPlan p = sort_plan(T, V);
  EmbedWs w{};
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t r = at;
    at += (bytes + 255) / 256 * 256;
    return r;
  };
  w.key0 = take(size_t(T) * 4);
  w.tok0 = take(size_t(T) * 4);
  if (!p.one) {
    w.key1 = take(size_t(T) * 4);
    w.tok1 = take(size_t(T) * 4);
    w.table = take(size_t(p.passes) * size_t(p.blocks) * kDigits * 4);
  }
  const int64_t pieces = (T + kPiece - 1) / kPiece;
  w.partial = take(size_t(pieces) * 2 * size_t(D) * 4);
  w.total = at;
  return w;
}

// Once per kernel and device (`done`: a static of the caller).
template <typename F>
b2_status allow_smem(F kern, size_t bytes, bool (&done)[64]) {
  int dev = 0;
  B2_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
  if (dev < 0 || dev >= 64) return set_error(B2_ERR_INVALID, "device index %d", dev);
  if (done[dev]) return B2_OK;
  B2_TRY(check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes)),
                    "cudaFuncSetAttribute(embedding sort)"));
  done[dev] = true;
  return B2_OK;
}

template <int I>
b2_status sort_pass(const void* ids, int is64, int64_t T, int64_t V, int64_t pad, const SortPlan& p, int pass,
                    uint32_t* table, const uint32_t* ki, const uint32_t* ti, uint32_t* ko, uint32_t* to,
                    cudaStream_t st) {
  const size_t smem = sizeof(SortSmem);
  auto kern = embed_pass_kernel<I>;
  static bool configured[64] = {};
  B2_TRY(allow_smem(kern, smem, configured));
  return launch_chained(kern, dim3(unsigned(p.blocks)), kSortThreads, smem, st, "embedding sort pass launch", ids, is64, T,
                        V, pad, pass, p.passes, p.bits, table, ki, ti, ko, to);
}

template <typename T, int N>
b2_status run_fwd(const void* ids, int is64, int64_t tokens, const void* w, int64_t ldw, int64_t V, int64_t D,
                  float scale, void* y, cudaStream_t st) {
  constexpr int U = 4;
  const int vecs = int(D / N);
  const int ll = log_lanes_for(vecs);
  const int rows = (256 >> ll) * U;
  const int64_t bx = (tokens + rows - 1) / rows;
  // long rows of too few tokens for every SM: their columns over CTAs
  const int slabs = (vecs + (1 << ll) - 1) >> ll;
  int by = 1;
  if (slabs > 1) {
    int dev = 0;
    B2_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
    if (bx < sm_count(dev)) by = std::min(slabs, 64);
  }
  if (bx > INT32_MAX) return set_error(B2_ERR_UNSUPPORTED, "b2_embedding_fwd: too many tokens");
  embed_fwd_kernel<T, N, U><<<dim3(unsigned(bx), unsigned(by)), 256, 0, st>>>(
      ids, is64, tokens, static_cast<const T*>(w), ldw, V, vecs, ll, scale, static_cast<T*>(y), D,
      device_status_ptr());
  return check_cuda(cudaGetLastError(), "embedding forward launch");
}

template <typename T, int N>
b2_status run_acc(const uint32_t* key, const uint32_t* tok, int64_t tokens, int64_t V, const void* dy, int64_t lddy,
                  int64_t D, float scale, void* dw, float* partial, cudaStream_t st) {
  const int vecs = int(D / N);
  const int ll = log_lanes_for(vecs);
  const int slabs = (vecs + (1 << ll) - 1) >> ll;
  const int64_t pieces = (tokens + kPiece - 1) / kPiece;
  const int per_block = kAccThreads >> ll;
  const int64_t acc_blocks = (pieces + per_block - 1) / per_block * slabs;
  const int zr = zero_rows_for(D, sizeof(T));
  const int64_t blocks = acc_blocks + (V + zr - 1) / zr;
  if (blocks > INT32_MAX) return set_error(B2_ERR_UNSUPPORTED, "b2_embedding_bwd: too many rows");
  B2_TRY(launch_chained(embed_acc_kernel<T, N>, dim3(unsigned(blocks)), kAccThreads, 0, st, "embedding gradient launch",
                        key, tok, tokens, V, static_cast<const T*>(dy), lddy, vecs, ll, D, scale, static_cast<T*>(dw),
                        partial, pieces, slabs, acc_blocks, zr));
  if (pieces > 1) {
    B2_TRY(launch_chained(embed_join_kernel<T, N>, dim3(unsigned((pieces + kJoinWarps - 1) / kJoinWarps), unsigned((vecs + 31) / 32)),
                          kAccThreads, 0,
                          st, "embedding gradient join launch", key, tokens, V, vecs, D, scale, static_cast<T*>(dw),
                          static_cast<const float*>(partial), pieces));
  }
  return B2_OK;
}

template <typename T, int N>
b2_status run_small(const void* ids, int is64, int64_t tokens, int64_t V, int64_t pad, const void* dy, int64_t lddy,
                    int64_t D, float scale, void* dw, cudaStream_t st) {
  const int vecs = int(D / N);
  int lw = 0;
  while (lw < 3 && (32 << lw) < vecs) ++lw;
  const int slabs = (vecs + (32 << lw) - 1) / (32 << lw);
  const int per_block = (kAccThreads / 32) >> lw;
  const int64_t token_blocks = (tokens + per_block - 1) / per_block * slabs;
  const int zr = zero_rows_for(D, sizeof(T));
  const int64_t blocks = token_blocks + (V + zr - 1) / zr;
  if (blocks > INT32_MAX) return set_error(B2_ERR_UNSUPPORTED, "b2_embedding_bwd: too many rows");
  embed_small_kernel<T, N><<<unsigned(blocks), kAccThreads, 0, st>>>(ids, is64, int(tokens), V, pad,
                                                                      static_cast<const T*>(dy), lddy, vecs, lw, D,
                                                                      scale, static_cast<T*>(dw), slabs, token_blocks, zr);
  return check_cuda(cudaGetLastError(), "embedding gradient launch");
}

b2_status check_common(const char* who, int ids_dtype, int dtype, int64_t T, int64_t V, int64_t D, int64_t ld) {
  if (ids_dtype != B2_I32 && ids_dtype != B2_I64) return set_error(B2_ERR_INVALID, "%s: ids must be int32 or int64", who);
  if (dtype != B2_BF16 && dtype != B2_F32) return set_error(B2_ERR_INVALID, "%s: bad dtype %d", who, dtype);
  if (T < 0 || V < 0 || D < 0 || ld < D) return set_error(B2_ERR_INVALID, "%s: bad shape", who);
  if (T >= INT32_MAX || V >= INT32_MAX || D >= INT32_MAX)
    return set_error(B2_ERR_UNSUPPORTED, "%s: tokens, vocabulary and width must be below 2^31 - 1", who);
  return B2_OK;
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

b2_status b2_embedding_fwd(const void* ids, int ids_dtype, int64_t T, const void* weight, int64_t ldw, int dtype,
                           int64_t V, int64_t D, float scale, void* y, void* stream) {
  B2_TRY(check_common("b2_embedding_fwd", ids_dtype, dtype, T, V, D, ldw));
  if (T == 0 || D == 0) return B2_OK;
  if (!ids || !y || (!weight && V > 0)) return set_error(B2_ERR_INVALID, "b2_embedding_fwd: null pointer");
  const auto st = static_cast<cudaStream_t>(stream);
  const int is64 = ids_dtype == B2_I64;
  if (dtype == B2_BF16) {
    switch (vec_elems(2, D, ldw, weight, y)) {
      case 8: return run_fwd<uint16_t, 8>(ids, is64, T, weight, ldw, V, D, scale, y, st);
      case 4: return run_fwd<uint16_t, 4>(ids, is64, T, weight, ldw, V, D, scale, y, st);
      case 2: return run_fwd<uint16_t, 2>(ids, is64, T, weight, ldw, V, D, scale, y, st);
      default: return run_fwd<uint16_t, 1>(ids, is64, T, weight, ldw, V, D, scale, y, st);
    }
  }
  switch (vec_elems(4, D, ldw, weight, y)) {
    case 4: return run_fwd<float, 4>(ids, is64, T, weight, ldw, V, D, scale, y, st);
    case 2: return run_fwd<float, 2>(ids, is64, T, weight, ldw, V, D, scale, y, st);
    default: return run_fwd<float, 1>(ids, is64, T, weight, ldw, V, D, scale, y, st);
  }
}

size_t b2_embedding_bwd_workspace_bytes(int64_t T, int64_t V, int64_t D) {
  if (T <= kSmallTokens || V <= 0 || D <= 0 || T >= INT32_MAX || V >= INT32_MAX) return 0;
  return embed_ws(T, V, D).total;
}

b2_status b2_embedding_bwd(const void* ids, int ids_dtype, int64_t T, const void* dy, int64_t lddy, int dtype,
                           int64_t V, int64_t D, float scale, int64_t padding_idx, void* dw, void* workspace,
                           size_t workspace_bytes, void* stream) {
  B2_TRY(check_common("b2_embedding_bwd", ids_dtype, dtype, T, V, D, lddy));
  if (V == 0 || D == 0) return B2_OK;
  if (!dw) return set_error(B2_ERR_INVALID, "b2_embedding_bwd: null pointer");
  const auto st = static_cast<cudaStream_t>(stream);
  if (T == 0)
    return check_cuda(cudaMemsetAsync(dw, 0, size_t(V) * size_t(D) * (dtype == B2_BF16 ? 2 : 4), st),
                      "embedding gradient memset");
  if (!ids || !dy) return set_error(B2_ERR_INVALID, "b2_embedding_bwd: null pointer");
  if (T <= kSmallTokens) {
    const int wide = ids_dtype == B2_I64;
    if (dtype == B2_BF16) {
      switch (vec_elems(2, D, lddy, dy, dw)) {
        case 8: return run_small<uint16_t, 8>(ids, wide, T, V, padding_idx, dy, lddy, D, scale, dw, st);
        case 4: return run_small<uint16_t, 4>(ids, wide, T, V, padding_idx, dy, lddy, D, scale, dw, st);
        case 2: return run_small<uint16_t, 2>(ids, wide, T, V, padding_idx, dy, lddy, D, scale, dw, st);
        default: return run_small<uint16_t, 1>(ids, wide, T, V, padding_idx, dy, lddy, D, scale, dw, st);
      }
    }
    switch (vec_elems(4, D, lddy, dy, dw)) {
      case 4: return run_small<float, 4>(ids, wide, T, V, padding_idx, dy, lddy, D, scale, dw, st);
      case 2: return run_small<float, 2>(ids, wide, T, V, padding_idx, dy, lddy, D, scale, dw, st);
      default: return run_small<float, 1>(ids, wide, T, V, padding_idx, dy, lddy, D, scale, dw, st);
    }
  }
  if (!workspace) return set_error(B2_ERR_INVALID, "b2_embedding_bwd: null pointer");
  const EmbedWs w = embed_ws(T, V, D);
  if (workspace_bytes < w.total || reinterpret_cast<uintptr_t>(workspace) % 16)
    return set_error(B2_ERR_WORKSPACE, "b2_embedding_bwd: workspace of %zu bytes (16-byte aligned) needed, got %zu",
                     w.total, workspace_bytes);
  uint8_t* base = static_cast<uint8_t*>(workspace);
  auto u32 = [&](size_t off) { return reinterpret_cast<uint32_t*>(base + off); };
  const int is64 = ids_dtype == B2_I64;
  const SortPlan p = sort_plan(T, V);
  uint32_t *key = u32(w.key0), *tok = u32(w.tok0);
  if (p.one) {
    embed_rank_kernel<<<unsigned((T + kRankPerBlock - 1) / kRankPerBlock), kRankThreads, 0, st>>>(
        ids, is64, int(T), V, padding_idx, key, tok);
    B2_TRY(check_cuda(cudaGetLastError(), "embedding rank launch"));
  } else {
    uint32_t* table = u32(w.table);
    embed_hist_kernel<<<unsigned(p.blocks), kSortThreads, 0, st>>>(ids, is64, T, V, padding_idx, p.passes, p.bits,
                                                                   p.items * kSortThreads, table);
    B2_TRY(check_cuda(cudaGetLastError(), "embedding histogram launch"));
    uint32_t *ko = key, *to = tok, *ki = u32(w.key1), *ti = u32(w.tok1);
    for (int pass = 0; pass < p.passes; ++pass) {
      if (p.items == 2)
        B2_TRY(sort_pass<2>(ids, is64, T, V, padding_idx, p, pass, table, ki, ti, ko, to, st));
      else
        B2_TRY(sort_pass<8>(ids, is64, T, V, padding_idx, p, pass, table, ki, ti, ko, to, st));
      std::swap(ki, ko);
      std::swap(ti, to);
    }
    key = ki;
    tok = ti;
  }
  float* partial = reinterpret_cast<float*>(base + w.partial);
  if (dtype == B2_BF16) {
    switch (vec_elems(2, D, lddy, dy, dw)) {
      case 8: return run_acc<uint16_t, 8>(key, tok, T, V, dy, lddy, D, scale, dw, partial, st);
      case 4: return run_acc<uint16_t, 4>(key, tok, T, V, dy, lddy, D, scale, dw, partial, st);
      case 2: return run_acc<uint16_t, 2>(key, tok, T, V, dy, lddy, D, scale, dw, partial, st);
      default: return run_acc<uint16_t, 1>(key, tok, T, V, dy, lddy, D, scale, dw, partial, st);
    }
  }
  switch (vec_elems(4, D, lddy, dy, dw)) {
    case 4: return run_acc<float, 4>(key, tok, T, V, dy, lddy, D, scale, dw, partial, st);
    case 2: return run_acc<float, 2>(key, tok, T, V, dy, lddy, D, scale, dw, partial, st);
    default: return run_acc<float, 1>(key, tok, T, V, dy, lddy, D, scale, dw, partial, st);
  }
}

}  // extern "C"
