// Gated feed-forward block, forward and backward, on the tcgen05 tensor cores.
//
//   forward   g = x Wg^T, u = x Wu^T, h = act(g) * u, y = h Wd^T
//   backward  dh = dy Wd
//             dg = dh * u * act'(g), du = dh * act(g)
//             dx = dg Wg + du Wu
//             dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// x [M][D], Wg and Wu [F][D], Wd [E][F], y [M][E]; bf16 with fp32 sums.  Five
// products of the same size, 6 M D F operations forward and 12 M D F backward;
// all of them run in one kernel template, a persistent SM-pair GEMM
// (tcgen05.mma.cta_group::2, 256 x PBN output tiles) that differs in its
// epilogue:
//   kGate      both projections in one tile: the pair's first CTA brings PBN/2
//              rows of Wg as its half of the B operand, the second the same
//              rows of Wu, so a thread finds g and u of the same hidden unit in
//              its own accumulator row and writes h in one epilogue; for
//              training also the factors P = u act'(g) and A = act(g)
//   kGateBwd   the tile of dh with P and A of the same place: writes dg = dh P
//              and du = dh A
//   kStore     a plain product, up to three of them in one launch; the two
//              halves of dx are one reduction over 2F whose operands change in
//              the middle
// h, dg and du are rounded to bf16 once each, from fp32, as operands of the next
// product: a relative error of at most 2^-8, that of the tensors themselves.  P
// and A keep 16 bits of significand -- their upper halves as bf16 patterns, the
// next 8 bits of both in one 16-bit word R -- so that the backward adds no
// rounding of its own: with both as bf16 the errors of dx, dWg and dWu were 1.7
// times those of one rounding at the end, with g and u as bf16 (act' of a
// rounded g) those of dWd too.  Keeping the factors rather than g and u also
// leaves the backward's epilogue two products instead of an exponential.
//
// Everything is bound by the tensor pipe or, for few tokens, by reading the
// weights.  Reductions whose tiles would leave most SM pairs idle are split;
// the fp32 partial tiles are added in split order by a second kernel that then
// runs the same epilogue (bit-reproducible).
#include <algorithm>

#include "b2_common.cuh"

namespace b2 {
namespace {

constexpr int BK = 64;
constexpr int kThreads = 320;  // warp 0 TMA, warp 1 MMA, warps 2..9 epilogue
constexpr int kEpiWarps = 8;
constexpr int kABytes = 128 * BK * 2;
constexpr int kMaxProblems = 3;
constexpr int kGroupM = 8;     // row tiles walked together (operand reuse in L2)

enum Epi : int { kStore = 0, kGate = 1, kGateBwd = 2 };
enum Act : int { kSilu = 0, kGelu = 1, kRelu = 2 };

struct Problem {
  int tiles_m, tiles_n;
  int M, N;           // valid output rows / columns (kGate: N = F)
  int kb, kb_first;   // k-blocks; of these, the ones from the first operand pair
  int splits, kb_per_split;
  int item_begin;     // first work item
  int tma_out;
  uint16_t* out;
  long long ldo;
  float* partial;     // splits > 1: [tiles][splits] partial tiles
};

struct Maps {
  CUtensorMap a[kMaxProblems], b[kMaxProblems], o[kMaxProblems + 1];
};

struct Params {
  Problem p[kMaxProblems];
  int problems, items;
  int train;  // kGate: write the factors (kGateBwd reads P, A and R through maps.a[1], maps.b[1] and maps.o[0])
  int* status;
};

__device__ __forceinline__ uint32_t cvt2(float lo, float hi) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint16_t cvt1(float v) {
  __nv_bfloat16 h = __float2bfloat16_rn(v);
  return *reinterpret_cast<uint16_t*>(&h);
}

// act(g) and act'(g).  The activation is a template argument of every kernel
// that needs it: chosen at run time inside the unrolled element loops it put
// all three into them, and the epilogue of a 256-wide tile took 8 us instead of
// its 3.
template <int ACT>
__device__ __forceinline__ void act_both(float g, float& a, float& slope) {
  if constexpr (ACT == kSilu) {
    const float s = __fdividef(1.f, 1.f + __expf(-g));
    a = g * s;
    slope = s * (1.f + g * (1.f - s));
  } else if constexpr (ACT == kGelu) {
    const float cdf = 0.5f * (1.f + erff(g * 0.70710678118654752f));
    a = g * cdf;
    slope = cdf + g * 0.39894228040143268f * __expf(-0.5f * g * g);
  } else {
    a = g > 0.f || g != g ? g : 0.f;
    slope = g > 0.f ? 1.f : 0.f;
  }
}
template <int ACT>
__device__ __forceinline__ float act_value(float g) {
  float a, slope;
  act_both<ACT>(g, a, slope);
  return a;
}

// The factors P and A as stored: their upper halves (bf16 patterns, truncated)
// and the next 8 bits of each, P's above A's: 16 bits of significand, truncated
// (2^-15; rounding would cost the epilogue more instructions than the factors
// themselves).  A NaN stays one: results of arithmetic carry it in the upper half.
struct Factors2 {  // of two neighbouring columns
  uint32_t p, a, r;
};
__device__ __forceinline__ Factors2 pack_factors(float p0, float p1, float a0, float a1) {
  const uint32_t x0 = __float_as_uint(p0), x1 = __float_as_uint(p1), y0 = __float_as_uint(a0), y1 = __float_as_uint(a1);
  Factors2 f;
  f.p = __byte_perm(x0, x1, 0x7632);
  f.a = __byte_perm(y0, y1, 0x7632);
  // bytes: A0, P0, A1, P1 (byte 1 of each word)
  f.r = __byte_perm(__byte_perm(y0, x0, 0x0051), __byte_perm(y1, x1, 0x0051), 0x5410);
  return f;
}
__device__ __forceinline__ float factor_lo(uint32_t upper, uint32_t r, int byte) {  // column 0: upper's low half
  return __uint_as_float((upper << 16) | (((r >> (8 * byte)) & 0xffu) << 8));
}
__device__ __forceinline__ float factor_hi(uint32_t upper, uint32_t r, int byte) {  // column 1: upper's high half
  return __uint_as_float((upper & 0xffff0000u) | (((r >> (8 * byte)) & 0xffu) << 8));
}

template <int EPI, int PBN>
struct Config {
  static constexpr int kBHalf = PBN / 2;
  static constexpr int kStage = kABytes + kBHalf * BK * 2;
  // per epilogue warp: kStore two 32 x 64 boxes, kGate four 32 x 32 boxes, kGateBwd triples of 32 x 32 boxes.
  // Of these one beside a fifth stage at PBN 256 (dh of 8192 tokens, 4096 x 12288, in passes under the power cap: 700
  // us, 750 with two triples and four stages, 886 with three), two at 128 (512 tokens, 1024 x 4096: 13.3 us, 13.8 with one).
  static constexpr int kTriples = PBN == 256 ? 1 : 2;
  static constexpr int kEpiBytes = EPI == kGateBwd ? kTriples * 6144 : 2 * 4096;
  static constexpr int kStages = PBN == 256 ? 5 : (EPI == kGateBwd ? 5 : 6);
  static constexpr size_t kSmem = size_t(kStages) * kStage + kEpiWarps * kEpiBytes + 1024 + 512;
};

struct Item {
  int prob, mt, nt, split, kb0, kb1, tile;
};

__device__ __forceinline__ Item decode(const Params& p, int t) {
  Item it;
  int i = 0;
  while (i + 1 < p.problems && t >= p.p[i + 1].item_begin) ++i;
  const Problem& q = p.p[i];
  t -= q.item_begin;
  it.prob = i;
  // the splits of a tile are neighbours
  it.split = t % q.splits;
  t /= q.splits;
  it.tile = t;
  const int group = t / (kGroupM * q.tiles_n);
  const int first = group * kGroupM;
  const int rows = min(kGroupM, q.tiles_m - first);
  const int in = t - first * q.tiles_n;
  it.mt = first + in % rows;
  it.nt = in / rows;
  it.kb0 = it.split * q.kb_per_split;
  it.kb1 = min(q.kb, it.kb0 + q.kb_per_split);
  return it;
}

// Partial tiles: [tile][split][rank * 8 + warp][chunk][4-column group][lane]
// float4, so that a warp's accesses are contiguous.  Returns the float4 of
// 4-column group q of accumulator columns [32 j, 32 j + 32) of one warp.
template <int PBN>
__device__ __forceinline__ float4* partial_at(const Problem& q, int tile, int split, int region, int j, int lane) {
  return reinterpret_cast<float4*>(q.partial) +
         ((((long long)tile * q.splits + split) * 16 + region) * (PBN / 64) + j) * 256 + lane;
}

// A staged 32 x 64 box (128-byte rows, chunk c of row r at c ^ (r & 7)) to output
// rows that no TMA store can address: the warp writes row after row, 4-byte
// words in consecutive lanes where the row's parity allows, so that a row's 128
// bytes are one access (a thread writing its own row's elements took 17 us a
// tile).  All lanes call; cols, rows: what is inside the output.
__device__ __forceinline__ void store_box_rows(const uint8_t* box, uint16_t* dst, long long ld, int rows, int cols,
                                               int lane) {
  auto at = [&](int r, int c) {
    return *reinterpret_cast<const uint16_t*>(box + r * 128 + (((c >> 3) ^ (r & 7)) << 4) + (c & 7) * 2);
  };
  rows = min(rows, 32);
  cols = min(cols, 64);
#pragma unroll 4
  for (int r = 0; r < rows; ++r) {
    uint16_t* d = dst + r * ld;
    const int odd = int(reinterpret_cast<uintptr_t>(d) >> 1) & 1;
    const int c = 2 * lane + odd;
    if (c + 1 < cols)
      *reinterpret_cast<uint32_t*>(d + c) = uint32_t(at(r, c)) | (uint32_t(at(r, c + 1)) << 16);
    else if (c < cols)
      d[c] = at(r, c);
    if (odd && lane == 31) d[0] = at(r, 0);
  }
}

// 8192 tokens, 4096 x 12288, each launch by itself: gate 1130 us, down 531, dh 617,
// dx 1100, the three weight gradients 1737 -- 1.45 PFLOP/s over all five; in
// passes one after the other 5.64 ms, 1.32 PFLOP/s, under the power cap (the clock
// falls with it).  512 tokens, 1024 x
// 4096, forward and backward 78 us: there each product's launch, first tiles and
// epilogue (2.5, 2 and 4 us) outweigh its 3 us of tensor work.
template <int EPI, int PBN, bool A_MN, bool B_MN, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gated_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
  using C = Config<EPI, PBN>;
  constexpr int STAGES = C::kStages;
  constexpr uint32_t kIdesc = idesc_bf16_f32(256, PBN, A_MN, B_MN);
  constexpr uint32_t kTmemCols = 2 * PBN;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* epi_stage = smem + STAGES * C::kStage;
  uint64_t* bars = reinterpret_cast<uint64_t*>(epi_stage + kEpiWarps * C::kEpiBytes);
  uint64_t* full = bars;
  uint64_t* empty = bars + STAGES;
  uint64_t* tfull = bars + 2 * STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* mma_done = tempty + 2;
  uint64_t* factor_bars = mma_done + 1;  // kGateBwd: two per epilogue warp
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(factor_bars + 2 * kEpiWarps);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32;
  const int lane = threadIdx.x % 32;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int cluster = blockIdx.x >> 1;
  const int nclusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&tfull[a]), 1);
      mbar_init(smem_u32(&tempty[a]), 2 * kEpiWarps);
    }
    mbar_init(smem_u32(mma_done), 1);
    for (int i = 0; i < 2 * kEpiWarps; ++i) mbar_init(smem_u32(&factor_bars[i]), 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish_pair();
  } else if (warp == 0 && lane < 4) {
    // the tensor maps travel while the barriers are set up
    const bool two = EPI != kStore || p.problems > 1 || p.p[0].kb > p.p[0].kb_first;
    if (lane < (two ? 2 : 1)) tma_prefetch_desc(&maps.a[EPI == kGate ? 0 : lane]);
    if (lane < (two ? 2 : 1)) tma_prefetch_desc(&maps.b[lane]);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both CTAs' barriers initialized before any cross-CTA signal
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  chain_wait();
  chain_release();

  if (warp == 0) {
    if (lane == 0) {
      // ------------------------------ producer (both CTAs) -----------------
      int stage = 0;
      uint32_t phase = 0;
      int last_par[STAGES];
#pragma unroll
      for (int s = 0; s < STAGES; ++s) last_par[s] = -1;
      bool ok = true;
      for (int t = cluster; t < p.items && ok; t += nclusters) {
        const Item it = decode(p, t);
        const Problem& q = p.p[it.prob];
        const int row0 = it.mt * 256 + int(rank) * 128;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(smem_u32(&empty[stage]), phase ^ 1, p.status, abort_flag)) {
            ok = false;
            break;
          }
          const uint32_t fb_local = smem_u32(&full[stage]);
          if (leader) mbar_arrive_expect_tx(fb_local, 2 * C::kStage);
          last_par[stage] = int(phase);
          const uint32_t fb = mapa_shared(fb_local, 0);
          const uint32_t sa = smem_u32(smem + stage * C::kStage);
          const uint32_t sb = sa + kABytes;
          // the reduction's second half has operands of its own (dx)
          const bool second = kb >= q.kb_first;
          const int k0 = (second ? kb - q.kb_first : kb) * BK;
          const CUtensorMap* ma = &maps.a[it.prob + (second ? 1 : 0)];
          const CUtensorMap* mb = &maps.b[it.prob + (second ? 1 : 0)];
          // B: this CTA's half of the tile's columns; kGate: the tile's hidden units in Wg or Wu
          int n0 = it.nt * PBN + int(rank) * C::kBHalf;
          if constexpr (EPI == kGate) {
            mb = &maps.b[rank];
            n0 = it.nt * C::kBHalf;
          }
          if constexpr (A_MN) {
            tma_load_3d_pair(sa, ma, fb, row0, k0, 0);
            tma_load_3d_pair(sa + 8192, ma, fb, row0 + 64, k0, 0);
          } else {
            tma_load_3d_pair(sa, ma, fb, k0, row0, 0);
          }
          if constexpr (B_MN) {
#pragma unroll
            for (int h = 0; h < C::kBHalf / 64; ++h) tma_load_3d_pair(sb + h * 8192, mb, fb, n0 + h * 64, k0, 0);
          } else {
            tma_load_3d_pair(sb, mb, fb, k0, n0, 0);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok && leader) {  // let issued copies land before the CTA goes away
        for (int s = 0; s < STAGES; ++s)
          if (last_par[s] >= 0) mbar_wait(smem_u32(&full[s]), uint32_t(last_par[s]), p.status, nullptr);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ------------------------------ MMA issuer (leader CTA) --------------
      int stage = 0;
      uint32_t phase = 0;
      int acc = 0;
      uint32_t acc_phase = 0;
      bool ok = true;
      for (int t = cluster; t < p.items && ok; t += nclusters) {
        const Item it = decode(p, t);
        if (!mbar_wait(smem_u32(&tempty[acc]), acc_phase ^ 1, p.status, abort_flag)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + uint32_t(acc * PBN);
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(smem_u32(&full[stage]), phase, p.status, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * C::kStage);
          const uint32_t sb = sa + kABytes;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t ad =
                A_MN ? smem_desc_sw128(sa + k * 2048, 8192, 1024) : smem_desc_sw128(sa + k * 32, 16, 1024);
            const uint64_t bd =
                B_MN ? smem_desc_sw128(sb + k * 2048, 8192, 1024) : smem_desc_sw128(sb + k * 32, 16, 1024);
            tc_mma_pair(d_tmem, ad, bd, kIdesc, (kb > it.kb0 || k > 0) ? 1u : 0u);
          }
          tc_commit_pair_mc(smem_u32(&empty[stage]), uint16_t(0x3));
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (!ok) break;
        tc_commit_pair_mc(smem_u32(&tfull[acc]), uint16_t(0x3));
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1;
      }
      tc_commit_pair(smem_u32(mma_done));
      mbar_wait(smem_u32(mma_done), 0, p.status, nullptr);
    }
    __syncwarp();
  } else {
    // -------------------------------- epilogue (both CTAs) ------------------
    const int quarter = warp & 3;         // tensor-memory lane quarter this warp may read
    const int half = (warp - 2) >> 2;     // half of the accumulator's columns
    const int region = int(rank) * 8 + half * 4 + quarter;
    const uint32_t tempty_leader[2] = {mapa_shared(smem_u32(&tempty[0]), 0), mapa_shared(smem_u32(&tempty[1]), 0)};
    uint8_t* buf = epi_stage + (warp - 2) * C::kEpiBytes;
    int sel = 0;
    uint64_t* factor_bar = factor_bars + (warp - 2) * 2;  // one per box triple
    int factor_phase = 0;
    // loads a 32 x 32 box of each of P, A and R into box triple `which`, once the last store from it has read it
    auto fetch_factors = [&](int c0, int row, int which) {
      if (lane == 0) {
        bulk_wait_read<0>();
        const uint32_t bar = smem_u32(&factor_bar[which]);
        mbar_arrive_expect_tx(bar, 6144);
        tma_load_3d(smem_u32(buf + which * 6144), &maps.a[1], bar, c0, row, 0);
        tma_load_3d(smem_u32(buf + which * 6144 + 2048), &maps.b[1], bar, c0, row, 0);
        tma_load_3d(smem_u32(buf + which * 6144 + 4096), &maps.o[0], bar, c0, row, 0);
      }
      __syncwarp();
    };
    (void)factor_phase;
    (void)fetch_factors;
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int t = cluster; t < p.items; t += nclusters) {
      const Item it = decode(p, t);
      const Problem& q = p.p[it.prob];
      const int row0 = it.mt * 256 + int(rank) * 128 + quarter * 32;
      // kGateBwd: this warp's 32-column chunks of the tile; the first one's
      // factors travel while its product is still running
      int chunks = 0;
      if constexpr (EPI == kGateBwd) {
        const int f0 = it.nt * PBN + half * (PBN / 2);
        if (q.splits == 1 && row0 < q.M && f0 < q.N) chunks = min(PBN / 64, (q.N - f0 + 31) / 32);
        if (chunks > 0) fetch_factors(f0, row0, sel);
      }
      bool ok = mbar_wait(smem_u32(&tfull[acc]), acc_phase, p.status, abort_flag);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {  // the factors on their way land before the CTA goes away
        if (chunks > 0) mbar_wait(smem_u32(&factor_bar[sel]), uint32_t(factor_phase >> sel) & 1u, p.status, nullptr);
        break;
      }
      tc_fence_after();
      const uint32_t tacc = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(acc * PBN);
      const uint32_t thalf = tacc + uint32_t(half * (PBN / 2));
      if (q.splits > 1) {
        if (row0 < q.M) {
#pragma unroll 1
          for (int j = 0; j < PBN / 64; ++j) {
            uint32_t r[32];
            tmem_ld32(thalf + j * 32, r);
            tc_wait_ld();
            float4* dst = partial_at<PBN>(q, it.tile, it.split, region, j, lane);
#pragma unroll
            for (int c = 0; c < 8; ++c)
              dst[c * 32] = make_float4(__uint_as_float(r[4 * c]), __uint_as_float(r[4 * c + 1]),
                                        __uint_as_float(r[4 * c + 2]), __uint_as_float(r[4 * c + 3]));
          }
        }
      } else if constexpr (EPI == kStore) {
        // Boxes of 32 rows x 64 columns staged with the tensor map's 128-byte
        // swizzle (16-byte chunk c of row r at chunk c ^ (r & 7): the eight
        // rows of a store phase hit distinct banks) and written by the TMA
        // unit in whole rows, clipped at M and N; one box fills while the
        // other's store reads it.
#pragma unroll 1
        for (int j = 0; j < PBN / 128; ++j) {
          const int c0 = it.nt * PBN + half * (PBN / 2) + j * 64;
          if (c0 >= q.N || row0 >= q.M) break;
          uint32_t r[2][32];
          tmem_ld32(thalf + j * 64, r[0]);
          tmem_ld32(thalf + j * 64 + 32, r[1]);
          tc_wait_ld();
          if (lane == 0) bulk_wait_read<1>();
          __syncwarp();
          uint8_t* box = buf + sel * 4096;
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            const uint32_t* v = &r[c >> 2][(c & 3) * 8];
            *reinterpret_cast<uint4*>(box + lane * 128 + ((c ^ (lane & 7)) << 4)) =
                make_uint4(cvt2(__uint_as_float(v[0]), __uint_as_float(v[1])),
                           cvt2(__uint_as_float(v[2]), __uint_as_float(v[3])),
                           cvt2(__uint_as_float(v[4]), __uint_as_float(v[5])),
                           cvt2(__uint_as_float(v[6]), __uint_as_float(v[7])));
          }
          if (q.tma_out) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&maps.o[it.prob], smem_u32(box), c0, row0, 0);
              bulk_commit();
            }
          } else {
            __syncwarp();
            store_box_rows(box, q.out + (long long)row0 * q.ldo + c0, q.ldo, q.M - row0, q.N - c0, lane);
          }
          sel ^= 1;
        }
      } else {
        // gate epilogues: 32 hidden units at a time, staged in 32 x 32 boxes
        // (64-byte swizzle: chunk c of row r at chunk c ^ ((r >> 1) & 3))
        auto fill = [&](uint8_t* box, const uint32_t (&v)[16]) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<uint4*>(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
        };
        auto read = [&](const uint8_t* box, uint32_t (&v)[16]) {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint4 w = *reinterpret_cast<const uint4*>(box + lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4));
            v[4 * c] = w.x;
            v[4 * c + 1] = w.y;
            v[4 * c + 2] = w.z;
            v[4 * c + 3] = w.w;
          }
        };
        if constexpr (EPI == kGate) {
          const int f0 = it.nt * (PBN / 2) + half * (PBN / 4);
#pragma unroll 1
          for (int j = 0; j < PBN / 128; ++j) {
            const int c0 = f0 + j * 32;
            if (c0 >= q.N || row0 >= q.M) break;
            uint32_t g[32], u[32];
            tmem_ld32(tacc + uint32_t(half * (PBN / 4) + j * 32), g);
            tmem_ld32(tacc + uint32_t(PBN / 2 + half * (PBN / 4) + j * 32), u);
            tc_wait_ld();
            if (lane == 0) bulk_wait_read<0>();  // the boxes' last stores have read them
            __syncwarp();
            uint32_t h[16];
            if (p.train) {
              uint32_t fp[16], fa[16], fr[16];
#pragma unroll
              for (int c = 0; c < 16; ++c) {
                const float u0 = __uint_as_float(u[2 * c]), u1 = __uint_as_float(u[2 * c + 1]);
                float a0, s0, a1, s1;
                act_both<ACT>(__uint_as_float(g[2 * c]), a0, s0);
                act_both<ACT>(__uint_as_float(g[2 * c + 1]), a1, s1);
                h[c] = cvt2(a0 * u0, a1 * u1);
                const Factors2 f = pack_factors(s0 * u0, s1 * u1, a0, a1);
                fp[c] = f.p;
                fa[c] = f.a;
                fr[c] = f.r;
              }
              fill(buf + 2048, fp);
              fill(buf + 4096, fa);
              fill(buf + 6144, fr);
            } else {
#pragma unroll
              for (int c = 0; c < 16; ++c)
                h[c] = cvt2(act_value<ACT>(__uint_as_float(g[2 * c])) * __uint_as_float(u[2 * c]),
                            act_value<ACT>(__uint_as_float(g[2 * c + 1])) * __uint_as_float(u[2 * c + 1]));
            }
            fill(buf, h);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&maps.o[0], smem_u32(buf), c0, row0, 0);
              if (p.train) {
                tma_store_3d(&maps.o[1], smem_u32(buf + 2048), c0, row0, 0);
                tma_store_3d(&maps.o[2], smem_u32(buf + 4096), c0, row0, 0);
                tma_store_3d(&maps.o[3], smem_u32(buf + 6144), c0, row0, 0);
              }
              bulk_commit();
            }
          }
        } else {
          const int f0 = it.nt * PBN + half * (PBN / 2);
#pragma unroll 1
          for (int j = 0; j < chunks; ++j) {
            const int c0 = f0 + j * 32;
            // the other boxes take the next chunk's factors
            if (C::kTriples == 2 && j + 1 < chunks) fetch_factors(c0 + 32, row0, sel ^ 1);
            ok = mbar_wait(smem_u32(&factor_bar[sel]), uint32_t(factor_phase >> sel) & 1u, p.status, abort_flag);
            factor_phase ^= 1 << sel;
            uint32_t d[32];
            tmem_ld32(thalf + j * 32, d);
            tc_wait_ld();
            uint8_t* box = buf + sel * 6144;
            uint32_t pv[16], av[16], rv[16];
            read(box, pv);
            read(box + 2048, av);
            read(box + 4096, rv);
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              const float d0 = __uint_as_float(d[2 * c]), d1 = __uint_as_float(d[2 * c + 1]);
              pv[c] = cvt2(d0 * factor_lo(pv[c], rv[c], 1), d1 * factor_hi(pv[c], rv[c], 3));
              av[c] = cvt2(d0 * factor_lo(av[c], rv[c], 0), d1 * factor_hi(av[c], rv[c], 2));
            }
            // a lane writes its results over the factors that it read
            fill(box, pv);
            fill(box + 2048, av);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&maps.o[1], smem_u32(box), c0, row0, 0);
              tma_store_3d(&maps.o[2], smem_u32(box + 2048), c0, row0, 0);
              bulk_commit();
            }
            if (C::kTriples == 2)
              sel ^= 1;
            else if (j + 1 < chunks)
              fetch_factors(c0 + 32, row0, 0);
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (leader)
          mbar_arrive(smem_u32(&tempty[acc]));
        else
          mbar_arrive_remote(tempty_leader[acc]);
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
    if (lane == 0) bulk_wait_all();  // stores done before the CTA's shared memory goes away
    __syncwarp();
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync();  // no CTA leaves while its pair may still signal or read it
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
}

// Adds a problem's partial tiles in split order and finishes them with its
// epilogue.  Gate epilogues: a thread takes 8 columns of one row (kGate: of g and
// of u).  kStore: a warp takes 32 rows x COLS columns and writes them, staged,
// in whole rows (elements of unaligned rows straight from the threads that own
// the rows took 26 us for 777 x 1001 where this takes 6).  The lanes of a warp
// are 32 rows, so its partial reads are contiguous.
struct ReduceArgs {
  Problem q;
  int train;
  uint16_t *h, *o1, *o2, *o3;      // kGate: h, P, A, R; kGateBwd: -, dg, du, -
  const uint16_t *fp, *fa, *fr;
  long long ldh, ldo, ldf;
  int beside;
};

template <int PBN>
__device__ __forceinline__ void sum8(const Problem& q, int tile, int region, int j, int oct, int lane, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = 0.f;
#pragma unroll 4
  for (int s = 0; s < q.splits; ++s) {
    const float4* src = partial_at<PBN>(q, tile, s, region, j, lane) + oct * 64;
    const float4 a = __ldcg(src), b = __ldcg(src + 32);
    v[0] += a.x;
    v[1] += a.y;
    v[2] += a.z;
    v[3] += a.w;
    v[4] += b.x;
    v[5] += b.y;
    v[6] += b.z;
    v[7] += b.w;
  }
}

__device__ __forceinline__ void put8(uint16_t* dst, const float (&v)[8], int cols, bool vec) {
  if (vec && cols >= 8) {
    *reinterpret_cast<uint4*>(dst) = make_uint4(cvt2(v[0], v[1]), cvt2(v[2], v[3]), cvt2(v[4], v[5]), cvt2(v[6], v[7]));
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i < cols) dst[i] = cvt1(v[i]);
}

template <int PBN, int COLS>
__global__ void __launch_bounds__(256) gated_reduce_store_kernel(const __grid_constant__ ReduceArgs a) {
  __shared__ __align__(16) uint8_t boxes[8][32 * COLS * 2];
  // beside: what is added was complete before the kernel before this one began
  // (its chain_release stands after its chain_wait)
  if (!a.beside) chain_wait();
  const Problem& q = a.q;
  constexpr int kUnits = PBN / COLS, kVecs = COLS / 8;
  const int lane = threadIdx.x & 31;
  uint8_t* box = boxes[threadIdx.x >> 5];
  const long long units = (long long)q.tiles_m * q.tiles_n * 8 * kUnits;  // (tile, 32-row block, COLS columns)
  for (long long w = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5; w < units; w += (long long)gridDim.x * 8) {
    const int unit = int(w % kUnits);
    const long long rest = w / kUnits;
    const int rows = int(rest % 8);  // rank * 4 + quarter
    const int tile = int(rest / 8);
    const int group = tile / (kGroupM * q.tiles_n), first = group * kGroupM;
    const int gm = min(kGroupM, q.tiles_m - first), in = tile - first * q.tiles_n;
    const int row0 = (first + in % gm) * 256 + rows * 32, col0 = (in / gm) * PBN + unit * COLS;
    if (row0 >= q.M || col0 >= q.N) continue;
    const int chunk = unit * COLS / 32;
    const int half = chunk / (PBN / 64), j = chunk % (PBN / 64);
    const int region = (rows >> 2) * 8 + half * 4 + (rows & 3);
    const int skip = unit * COLS % 32 / 4 * 32;
    float4 v[2 * kVecs];
#pragma unroll
    for (int c = 0; c < 2 * kVecs; ++c) v[c] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll(COLS == 32 ? 2 : 8)
    for (int s = 0; s < q.splits; ++s) {
      const float4* src = partial_at<PBN>(q, tile, s, region, j, lane) + skip;
#pragma unroll
      for (int c = 0; c < 2 * kVecs; ++c) {
        const float4 x = __ldcg(src + c * 32);
        v[c].x += x.x;
        v[c].y += x.y;
        v[c].z += x.z;
        v[c].w += x.w;
      }
    }
    // 16-byte vector c of row r at c ^ ((r >> 1) & 3) of its 64 bytes
    const auto slot = [&](int r, int c) { return box + r * (COLS * 2) + ((kVecs == 4 ? c ^ ((r >> 1) & 3) : c) << 4); };
    __syncwarp();
#pragma unroll
    for (int c = 0; c < kVecs; ++c)
      *reinterpret_cast<uint4*>(slot(lane, c)) =
          make_uint4(cvt2(v[2 * c].x, v[2 * c].y), cvt2(v[2 * c].z, v[2 * c].w),
                     cvt2(v[2 * c + 1].x, v[2 * c + 1].y), cvt2(v[2 * c + 1].z, v[2 * c + 1].w));
    __syncwarp();
    const int nrows = min(32, q.M - row0), cols = min(COLS, q.N - col0);
    uint16_t* out = q.out + (long long)row0 * q.ldo + col0;
    if (q.tma_out && cols == COLS) {
      // aligned rows: a lane a vector
#pragma unroll
      for (int i = 0; i < kVecs; ++i) {
        const int r = i * (32 / kVecs) + lane / kVecs, c = lane % kVecs;
        if (r < nrows)
          *reinterpret_cast<uint4*>(out + (long long)r * q.ldo + c * 8) = *reinterpret_cast<const uint4*>(slot(r, c));
      }
    } else {
      const int c = lane % COLS;
#pragma unroll 4
      for (int r = lane / COLS; r < nrows; r += 32 / COLS)
        if (c < cols)
          out[(long long)r * q.ldo + c] = *reinterpret_cast<const uint16_t*>(slot(r, c >> 3) + (c & 7) * 2);
    }
  }
  if (a.beside) chain_wait();  // what waits for this kernel waits for the one before it too
}

template <int EPI, int PBN, int ACT>
__global__ void __launch_bounds__(256) gated_reduce_kernel(const __grid_constant__ ReduceArgs a) {
  chain_wait();
  const Problem& q = a.q;
  constexpr int kCols = EPI == kGate ? PBN / 2 : PBN;  // output columns of a tile
  constexpr int kOcts = kCols / 8;
  const int lane = threadIdx.x & 31;
  const long long units = (long long)q.tiles_m * q.tiles_n * 8 * kOcts;  // (tile, 32-row block, 8 columns)
  for (long long w = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5; w < units; w += (long long)gridDim.x * 8) {
    const int oc = int(w % kOcts);
    const long long rest = w / kOcts;
    const int rows = int(rest % 8);  // rank * 4 + quarter
    const int tile = int(rest / 8);
    const int group = tile / (kGroupM * q.tiles_n), first = group * kGroupM;
    const int gm = min(kGroupM, q.tiles_m - first), in = tile - first * q.tiles_n;
    const int mt = first + in % gm, nt = in / gm;
    const int row = mt * 256 + rows * 32 + lane;
    const int col = nt * kCols + oc * 8;
    if (row >= q.M || col >= q.N) continue;
    const int rank = rows >> 2, quarter = rows & 3;
    const int cols = q.N - col;
    float v[8];
    if constexpr (EPI == kGate) {
      float g[8];
      sum8<PBN>(q, tile, rank * 8 + quarter, oc / 4, oc & 3, lane, g);
      sum8<PBN>(q, tile, rank * 8 + 4 + quarter, oc / 4, oc & 3, lane, v);
      float h[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float act, slope;
        act_both<ACT>(g[i], act, slope);
        h[i] = act * v[i];
        v[i] *= slope;
        g[i] = act;
      }
      put8(a.h + (long long)row * a.ldh + col, h, cols, true);
      if (a.train) {
        // rows of the factors hold a multiple of 8 columns: whole vectors fit
        uint32_t fp[4], fa[4], fr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const Factors2 f = pack_factors(v[2 * i], v[2 * i + 1], g[2 * i], g[2 * i + 1]);
          fp[i] = f.p;
          fa[i] = f.a;
          fr[i] = f.r;
        }
        const long long at = (long long)row * a.ldo + col;
        *reinterpret_cast<uint4*>(a.o1 + at) = make_uint4(fp[0], fp[1], fp[2], fp[3]);
        *reinterpret_cast<uint4*>(a.o2 + at) = make_uint4(fa[0], fa[1], fa[2], fa[3]);
        *reinterpret_cast<uint4*>(a.o3 + at) = make_uint4(fr[0], fr[1], fr[2], fr[3]);
      }
    } else {
      const int half = oc / (PBN / 16), o = oc % (PBN / 16);
      sum8<PBN>(q, tile, rank * 8 + half * 4 + quarter, o / 4, o & 3, lane, v);
      const long long at = (long long)row * a.ldf + col;
      const uint4 pv = *reinterpret_cast<const uint4*>(a.fp + at);
      const uint4 av = *reinterpret_cast<const uint4*>(a.fa + at);
      const uint4 rv = *reinterpret_cast<const uint4*>(a.fr + at);
      const uint32_t pw[4] = {pv.x, pv.y, pv.z, pv.w}, aw[4] = {av.x, av.y, av.z, av.w}, rw[4] = {rv.x, rv.y, rv.z, rv.w};
      float dg[8], du[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        dg[2 * i] = v[2 * i] * factor_lo(pw[i], rw[i], 1);
        dg[2 * i + 1] = v[2 * i + 1] * factor_hi(pw[i], rw[i], 3);
        du[2 * i] = v[2 * i] * factor_lo(aw[i], rw[i], 0);
        du[2 * i + 1] = v[2 * i + 1] * factor_hi(aw[i], rw[i], 2);
      }
      put8(a.o1 + (long long)row * a.ldo + col, dg, cols, true);
      put8(a.o2 + (long long)row * a.ldo + col, du, cols, true);
    }
  }
}

// 16 bytes that start `shift` bits (a multiple of 16) into the 32 bytes lo, hi.
__device__ __forceinline__ uint4 shift_words(const uint4& lo, const uint4& hi, int shift) {
  const uint32_t v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  const int words = shift >> 5, bits = shift & 31;
  uint32_t o[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t x = words == 0 ? v[e] : words == 1 ? v[e + 1] : words == 2 ? v[e + 2] : v[e + 3];
    const uint32_t y = words == 0 ? v[e + 1] : words == 1 ? v[e + 2] : words == 2 ? v[e + 3] : v[e + 4];
    o[e] = __funnelshift_r(x, y, bits);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Copies of matrices whose rows no TMA map can address (a row stride that is
// not a multiple of 16 bytes, or a misaligned base) into rows that one can.  A
// warp takes a piece of a row (or several short rows, 1 << log_lanes lanes each)
// in aligned 16-byte words, kPadBatch on their way a lane; a lane's result is its
// word and the next one, which its neighbour has, shifted together.  What the
// last word of a row brings of the next row lands in the copy's padding, which no
// map covers.  2048 x 5461, 22 MB in and out: 9.3 us; a thread 16 bytes of the
// copy at a time, with both words of its own, took 11.5, whole rows a warp 12.2.
// (Beside the first product instead of before it: 127 -> 132 us for a training
// pass of 777 tokens, 1001 x 2730.)
constexpr int kPadBatch = 4;
struct PadArgs {
  const uint16_t* src[5];
  uint16_t* dst[5];
  long long lds[5];
  int rows[5], cols[5], ldd[5], log_lanes[5];
  long long begin[6];  // prefix sums of warps' units
  int n;
};
__global__ void __launch_bounds__(256) gated_pad_kernel(const __grid_constant__ PadArgs a) {
  chain_wait();
  constexpr int U = kPadBatch;
  const int lane = threadIdx.x & 31;
  for (long long unit = ((long long)blockIdx.x * 256 + threadIdx.x) >> 5; unit < a.begin[a.n]; unit += (long long)gridDim.x * 8) {
    int m = 0;
    while (unit >= a.begin[m + 1]) ++m;
    const int ll = a.log_lanes[m], L = 1 << ll, lw = lane & (L - 1);
    const int groups = a.ldd[m] / 8, segments = (groups + U * L - 1) / (U * L);
    const long long rows = (unit - a.begin[m]) / segments, row = rows * (32 >> ll) + (lane >> ll);
    const int j0 = int(unit - a.begin[m] - rows * segments) * U * L;
    const bool live = row < a.rows[m];
    const uint16_t* first = a.src[m];
    const uint16_t* end = first + (a.rows[m] - 1) * a.lds[m] + a.cols[m];
    const uintptr_t addr = reinterpret_cast<uintptr_t>(first + (live ? row : 0) * a.lds[m]);
    const int shift = int(addr & 15) * 8;
    const uint16_t* base = reinterpret_cast<const uint16_t*>(addr & ~uintptr_t(15));
    uint4* out = reinterpret_cast<uint4*>(a.dst[m] + (live ? row : 0) * a.ldd[m]);
    // the row's aligned word j; nothing outside the matrix is read
    auto word = [&](int j) {
      const uint16_t* p = base + (long long)j * 8;
      if (p >= first && p + 8 <= end) return __ldg(reinterpret_cast<const uint4*>(p));
      union {
        uint4 v;
        uint16_t e[8];
      } r;
#pragma unroll
      for (int e = 0; e < 8; ++e) r.e[e] = p + e >= first && p + e < end ? p[e] : uint16_t(0);
      return r.v;
    };
    uint4 w[U + 1];
#pragma unroll
    for (int u = 0; u < U; ++u)
      w[u] = live && j0 + u * L + lw <= groups ? word(j0 + u * L + lw) : make_uint4(0, 0, 0, 0);
    w[U] = live && lw == 0 && j0 + U * L <= groups ? word(j0 + U * L) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // the next word: the next lane's, or the first lane's of the next batch entry
      uint4 hi;
      const uint32_t* lo = &w[u].x;
      const uint32_t* up = &w[u + 1].x;
      uint32_t* h = &hi.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = __shfl_sync(0xffffffffu, lw == 0 ? up[i] : lo[i], (lw + 1) & (L - 1), L);
      // (lane 0 offers the next entry's word to the last lane; its own next word comes from lane 1)
      const int j = j0 + u * L + lw;
      if (live && j < groups) out[j] = shift_words(w[u], hi, shift);
    }
  }
}

// ---------------------------------------------------------------------------
// Few tokens (M <= kFewTokens): reading the weights once is everything, and a
// 256-row tile per token would idle most of the machine.  A CTA takes 16 weight
// rows (kGate: of Wg and of Wu), its 8 warps interleave the reduction in steps
// of 32, and a cluster of up to 8 CTAs shares a reduction of Wd.  The products
// run on mma.sync m16n8k16 with the weights as the 16-row operand and the tokens
// as the columns: a lane's 16 bytes of a weight row hold 8 consecutive k, which
// two instructions take in an order of their own (the same for both operands, so
// the sum is the same).  What bounds it is how much is on its way from memory:
// every lane copies its own 16 bytes ahead into a ring of 3 to 6 steps in shared
// memory (asynchronously, and read back by the same lane, so nothing has to be
// synchronized).  Partial sums are added in warp and CTA order.
//
// One token, D 1024, F 4096 (25 MB of weights): 10.2 us; 4096 x 12288 (302 MB):
// 57 us, 5.3 TB/s.  Loads straight to registers took 13 and 68 us; one
// cooperative kernel over both products with TMA boxes 18 and 67 us; 64 k a
// step, copied in whole 128-byte lines, 14 and 66 us.
// ---------------------------------------------------------------------------
constexpr int kFewThreads = 256;
constexpr int kFewWarps = kFewThreads / 32;
constexpr int kFewStages = 6;
constexpr int kFewTokens = 32;
// Up to this many tokens Wd's product takes h as two bf16 numbers, the rounded h
// and what the rounding left, as columns that the instruction has free: y's error
// is then that of its own rounding alone (1.4 times that otherwise).  One token,
// 1024 x 4096: 10.2 us, 9.6 without; 4096 x 12288 56.6 and 56.3; eight tokens would
// need a second column block, 64.8 and 59.4.
constexpr int kRestTokens = 4;

struct FewMat {
  const uint16_t* p;
  const uint16_t* end;  // one past the last element
  long long ld;
  int aligned;          // every row starts at 16 bytes
};
struct FewArgs {
  FewMat w[2];   // kGate: Wg, Wu; kStore: Wd
  FewMat x;      // [M][K]
  int M, rows, K;
  int early;     // the weights were not written by the kernel before this one
  uint16_t *out, *o1, *o2, *o3;  // kGate: h, P, A, R (or null); kStore: y
  long long ldo;            // of all of them
  uint16_t* rest;           // what rounding h left, [M][ldr], or null: kGate writes it, kStore's tokens go on with it
  long long ldr;
};

__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(src)) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Waits for the oldest of the S - 1 steps under way.
__device__ __forceinline__ void copy_wait_step(int S) {
  if (S == 3)
    copy_wait<1>();
  else if (S == 4)
    copy_wait<2>();
  else if (S == 5)
    copy_wait<3>();
  else
    copy_wait<4>();
}

// Starts this lane's copy of 8 consecutive elements of a row from k (zeros from K
// on) to its 16 bytes at `at`; rows at any alignment (WORDS 2): the two aligned
// words around them, 512 bytes apart, to be shifted when they are used.
template <int WORDS>
__device__ __forceinline__ void fetch8(const FewMat& m, const uint16_t* row, int k, int K, uint4* at) {
  const uintptr_t addr = reinterpret_cast<uintptr_t>(row + k);
  const uint16_t* first = reinterpret_cast<const uint16_t*>(WORDS == 2 ? addr & ~uintptr_t(15) : addr);
  const bool whole = k + 8 <= K && (WORDS == 2 ? first >= m.p && first + 16 <= m.end : m.aligned != 0);
  if (whole) {
#pragma unroll
    for (int w = 0; w < WORDS; ++w) copy16_async(smem_u32(at + w * 32), first + w * 8);
  } else {
    // at the ends of the row or the matrix: what is inside, element by element
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      union {
        uint4 v;
        uint16_t e[8];
      } r;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t* p = first + w * 8 + i;
        r.e[i] = p >= row + k && p < row + K ? __ldcg(p) : uint16_t(0);
      }
      at[w * 32] = r.v;
    }
  }
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16-byte slots of one step: weights, then tokens; 32 lanes each.
template <int EPI, int NT, bool ALIGNED>
struct FewConfig {
  static constexpr int kMats = EPI == kGate ? 2 : 1;
  static constexpr int kWords = ALIGNED ? 1 : 2;
  static constexpr int kSlots = kMats * 2 * kWords + NT;
  static constexpr size_t kStep = size_t(kFewWarps) * kSlots * 512;  // bytes of a stage
  static constexpr size_t kStatic = size_t(kFewWarps + 1) * kMats * 16 * 8 * NT * 4;  // red and total
  static constexpr int kMost = int((227 * 1024 - kStatic) / kStep) < kFewStages ? int((227 * 1024 - kStatic) / kStep) : kFewStages;
  static_assert(kMost >= 3, "a ring of three steps");
};

template <int EPI, int NT, int ACT, bool ALIGNED>
__global__ void __launch_bounds__(kFewThreads) gated_few_kernel(const __grid_constant__ FewArgs a, int cluster,
                                                                int S) {
  using C = FewConfig<EPI, NT, ALIGNED>;
  constexpr int kMats = C::kMats, kWords = C::kWords;
  constexpr int kOut = 16 * 8 * NT;   // sums per matrix
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ float red[kFewWarps][kMats][kOut];
  __shared__ float total[kMats][kOut];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, q = lane & 3;
  const int rank = cluster > 1 ? int(cluster_ctarank()) : 0;
  const int row0 = (blockIdx.x / cluster) * 16;
  uint4* ring = reinterpret_cast<uint4*>(smem_raw) + warp * S * C::kSlots * 32 + lane;
  const uint16_t* wrow[kMats][2];
  bool live[2];
  int shift[kMats][2];
  const int k_first = (rank * kFewWarps + warp) * 32 + q * 8;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    live[i] = row0 + g + 8 * i < a.rows;
#pragma unroll
    for (int m = 0; m < kMats; ++m) {
      wrow[m][i] = a.w[m].p + (long long)(live[i] ? row0 + g + 8 * i : row0) * a.w[m].ld;
      shift[m][i] = int(reinterpret_cast<uintptr_t>(wrow[m][i] + k_first) & 15) * 8;  // the same at every step
    }
  }
  const uint16_t* xrow[NT];
  bool xlive[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = n * 8 + g;
    const bool second = EPI == kStore && a.rest && r >= a.M;
    xlive[n] = r < (EPI == kStore && a.rest ? 2 * a.M : a.M);
    xrow[n] = second ? a.rest + (xlive[n] ? r - a.M : 0) * a.ldr : a.x.p + (long long)(xlive[n] ? r : 0) * a.x.ld;
  }
  float c[kMats][NT][4];
#pragma unroll
  for (int m = 0; m < kMats; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[m][n][i] = 0.f;
  const int stride = kFewWarps * cluster * 32;
  const int steps = (a.K - (k_first - q * 8) + stride - 1) / stride;  // of this warp; may be <= 0
  const uint4 zero = make_uint4(0, 0, 0, 0);
  // the copies of step t into stage `at`
  auto fetch_w = [&](int t, int at) {
    const int k = k_first + t * stride;
#pragma unroll
    for (int m = 0; m < kMats; ++m)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint4* slot = ring + (at * C::kSlots + (m * 2 + i) * kWords) * 32;
        if (k < a.K && live[i])
          fetch8<kWords>(a.w[m], wrow[m][i], k, a.K, slot);
        else
#pragma unroll
          for (int w = 0; w < kWords; ++w) slot[w * 32] = zero;
      }
  };
  auto fetch_x = [&](int t, int at) {
    const int k = k_first + t * stride;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint4* slot = ring + (at * C::kSlots + kMats * 2 * kWords + n) * 32;
      if (k < a.K && xlive[n])
        fetch8<1>(a.x, xrow[n], k, a.K, slot);
      else
        *slot = zero;
    }
  };
  if (!a.early) chain_wait();
  chain_release();
  for (int t = 0; t < S - 1; ++t)
    if (t < steps) fetch_w(t, t);
  if (a.early) chain_wait();  // the tokens' operand comes from the kernel before
  for (int t = 0; t < S - 1; ++t) {
    if (t < steps) fetch_x(t, t);
    copy_commit();
  }
  int at = 0;
  for (int t = 0; t < steps; ++t) {
    copy_wait_step(S);
    const uint4* slot = ring + at * C::kSlots * 32;
    uint4 xv[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) xv[n] = slot[(kMats * 2 * kWords + n) * 32];
#pragma unroll
    for (int m = 0; m < kMats; ++m) {
      uint4 w[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4* p = slot + (m * 2 + i) * kWords * 32;
        w[i] = ALIGNED ? p[0] : shift_words(p[0], p[(kWords - 1) * 32], shift[m][i]);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma16816(c[m][n], w[0].x, w[1].x, w[0].y, w[1].y, xv[n].x, xv[n].y);
        mma16816(c[m][n], w[0].z, w[1].z, w[0].w, w[1].w, xv[n].z, xv[n].w);
      }
    }
    // the stage of the step before is free
    const int next = at == 0 ? S - 1 : at - 1;
    if (t + S - 1 < steps) {
      fetch_w(t + S - 1, next);
      fetch_x(t + S - 1, next);
    }
    copy_commit();
    if (++at == S) at = 0;
  }
  copy_wait<0>();
#pragma unroll
  for (int m = 0; m < kMats; ++m)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        red[warp][m][(n * 8 + 2 * q + (i & 1)) * 16 + g + 8 * (i >> 1)] = c[m][n][i];
  __syncthreads();
  for (int t = threadIdx.x; t < kMats * kOut; t += kFewThreads) {
    const int m = t / kOut, o = t % kOut;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kFewWarps; ++w) v += red[w][m][o];
    total[m][o] = v;
  }
  if (cluster > 1)
    cluster_sync();
  else
    __syncthreads();
  if (rank == 0) {
    for (int t = threadIdx.x; t < kOut; t += kFewThreads) {
      const int row = row0 + (t & 15), token = t >> 4;
      if (row >= a.rows || token >= a.M) continue;
      auto cluster_total = [&](int m, int at) {
        float v = total[m][at];
        for (int r = 1; r < cluster; ++r) {
          float o;
          asm volatile("ld.shared::cluster.f32 %0, [%1];"
                       : "=f"(o)
                       : "r"(mapa_shared(smem_u32(&total[m][at]), uint32_t(r)))
                       : "memory");
          v += o;
        }
        return v;
      };
      float v[kMats];
#pragma unroll
      for (int m = 0; m < kMats; ++m) v[m] = cluster_total(m, t);
      const long long at = (long long)token * a.ldo + row;
      if constexpr (EPI == kGate) {
        float act, slope;
        act_both<ACT>(v[0], act, slope);
        const float h = act * v[1];
        const uint16_t hi = cvt1(h);
        a.out[at] = hi;
        if (a.rest) a.rest[token * a.ldr + row] = fabsf(bf2f(hi)) < INFINITY ? cvt1(h - bf2f(hi)) : uint16_t(0);
        if (a.o1) {
          const Factors2 f = pack_factors(slope * v[1], 0.f, act, 0.f);
          a.o1[at] = uint16_t(f.p);
          a.o2[at] = uint16_t(f.a);
          a.o3[at] = uint16_t(f.r);
        }
      } else {
        a.out[at] = cvt1(a.rest ? v[0] + cluster_total(0, t + 16 * a.M) : v[0]);
      }
    }
  }
  if (cluster > 1) cluster_sync();  // no CTA leaves while the first may read it
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

int64_t up8(int64_t n) { return (n + 7) / 8 * 8; }
bool tma_rows(const void* p, int64_t ld) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0; }

// A matrix in memory: rows x cols, row stride ld.
struct Mat {
  const void* p = nullptr;
  int64_t rows = 0, cols = 0, ld = 0;
};

b2_status map2d(CUtensorMap* m, const Mat& a, uint32_t box_cols, uint32_t box_rows, int swizzle) {
  const uint64_t dims[3] = {uint64_t(a.cols), uint64_t(a.rows), 1};
  const uint64_t strides[2] = {uint64_t(a.ld) * 2, uint64_t(a.ld) * 2 * uint64_t(a.rows)};
  const uint32_t box[3] = {box_cols, box_rows, 1};
  return encode_tmap_sw(m, a.p, 3, dims, strides, box, swizzle);
}

// One product: out[M][N] = A B with the operands as stored.  A: [M][K] or, MN
// (k-rows), [K][M]; B: [N][K] or [K][N].
struct Product {
  Mat a[2], b[2];   // the second pair continues the reduction (or, kGate, b[1] is Wu)
  int64_t M = 0, N = 0, K = 0;
  int pairs = 1;
  void* out = nullptr;
  int64_t ldo = 0;
};

struct Plan {
  int pbn = 256;
  int splits = 1;
  size_t partial_bytes = 0;
};

// Tile width and reduction splits of a product.  Cost in SM clocks of a pair
// on its busiest pair: a k-block of a 256-wide tile takes 512 clocks of the
// tensor pipe but about 800 to bring its operands from L2 when the clock is high
// (32 KB at 41 bytes a clock and SM; 24 KB of a 128-wide one: 600); each tile
// adds a pipeline fill and drain; a split adds writing and reading the fp32
// partials and the second kernel.
Plan plan_product(int64_t M, int64_t N, int64_t K, int pairs, bool gate, int sms) {
  const int clusters = std::max(1, sms / 2);
  const int64_t kb = (K + BK - 1) / BK * pairs;
  Plan best{};
  double best_cost = 1e300;
  for (int pbn : {256, 128}) {
    const int64_t cols = gate ? pbn / 2 : pbn;
    const int64_t tiles = ((M + 255) / 256) * ((N + cols - 1) / cols);
    for (int s = 1; s <= 16; ++s) {
      if (s > 1 && (kb / s < 4 || tiles * s > 2 * clusters)) break;
      const int64_t kps = (kb + s - 1) / s;
      const int64_t splits = (kb + kps - 1) / kps;
      if (splits != s) continue;
      const int64_t waves = (tiles * s + clusters - 1) / clusters;
      double cost = double(waves) * (double(kps) * (pbn == 256 ? 800 : 600) + 800) + 2500;
      // the epilogue writes the 32-row blocks that hold tokens
      const double rows = std::min<double>(double(M + 31) / 32 * 32, double((M + 255) / 256 * 256));
      if (s > 1) cost += 4000 + double(tiles) / double((M + 255) / 256) * rows * pbn * 4 * s * 2 / 2500.0;
      if (cost < best_cost) {
        best_cost = cost;
        best.pbn = pbn;
        best.splits = s;
        best.partial_bytes = s > 1 ? size_t(tiles) * s * 256 * pbn * 4 : 0;
      }
    }
  }
  return best;
}

template <int EPI, int PBN, bool A_MN, bool B_MN, int ACT>
b2_status launch_gemm(const Maps& maps, const Params& p, cudaStream_t st) {
  using C = Config<EPI, PBN>;
  auto kern = gated_kernel<EPI, PBN, A_MN, B_MN, ACT>;
  int dev = 0;
  B2_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
  static bool configured[64] = {};
  if (dev < 0 || dev >= 64) return set_error(B2_ERR_INVALID, "device index %d", dev);
  if (!configured[dev]) {
    B2_TRY(check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(C::kSmem)),
                      "cudaFuncSetAttribute(gated)"));
    configured[dev] = true;
  }
  const int clusters = std::min(p.items, sm_count(dev) / 2);
  return launch_chained(kern, dim3(2 * clusters), kThreads, C::kSmem, st, "gated product launch", maps, p);
}

// The gate epilogues' tensors.
struct Gate {
  int train = 0;
  Mat h, o1, o2, o3;             // written: h, P, A, R (kGate) or dg, du (kGateBwd)
  const uint16_t *fp = nullptr, *fa = nullptr, *fr = nullptr;
  int64_t ldf = 0;
};

int current_sms() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess ? sm_count(dev) : 148;
}

// Carves a workspace; with a null base it only counts.
struct Carve {
  uint8_t* base;
  size_t at = 0;
  explicit Carve(void* b) : base(static_cast<uint8_t*>(b)) {}
  void* take(size_t bytes) {
    void* r = base ? base + at : nullptr;
    at += (bytes + 255) / 256 * 256;
    return r;
  }
};

// Brings operands into TMA-addressable rows where they are not, in one launch.
struct Padder {
  PadArgs a{};
  void add(Mat& m, Carve& ws) {
    if (!m.p || m.rows == 0 || m.cols == 0) return;
    // room is reserved by the shape alone, so that the workspace size does not depend on the pointers
    if (tma_rows(m.p, m.ld)) return;
    const int64_t ld = up8(m.cols);
    void* d = ws.take(size_t(m.rows) * size_t(ld) * 2);
    const int i = a.n++;
    a.src[i] = static_cast<const uint16_t*>(m.p);
    a.dst[i] = static_cast<uint16_t*>(d);
    a.lds[i] = m.ld;
    a.rows[i] = int(m.rows);
    a.cols[i] = int(m.cols);
    a.ldd[i] = int(ld);
    int ll = 0;
    while (ll < 5 && (1 << ll) < ld / 8) ++ll;
    a.log_lanes[i] = ll;
    const int64_t words = int64_t(kPadBatch) << ll;
    a.begin[i + 1] = a.begin[i] + (m.rows + (32 >> ll) - 1) / (32 >> ll) * ((ld / 8 + words - 1) / words);
    m.p = d;
    m.ld = ld;
  }
  b2_status run(cudaStream_t st) {
    if (a.n == 0) return B2_OK;
    const unsigned blocks = unsigned(std::min<long long>((a.begin[a.n] + 7) / 8, current_sms() * 16LL));
    return launch_chained(gated_pad_kernel, dim3(blocks), 256, 0, st, "gated pad launch", a);
  }
};

b2_status launch_reduce_store(const ReduceArgs& r, int pbn, cudaStream_t st) {
  // Units of 8 columns where those of 32 would be fewer than 8 warps a SM (19
  // tokens, 1024 x 4096: a forward of 22 us against 27; 512 tokens, 4096 x 12288:
  // 131 us against 129 with the wide ones).
  const long long wide = (long long)(r.q.M + 31) / 32 * r.q.tiles_n * (pbn / 32);
  const bool narrow = wide < 8LL * current_sms();
  const long long units = (long long)r.q.tiles_m * r.q.tiles_n * 8 * (pbn / (narrow ? 8 : 32));
  const dim3 blocks(unsigned(std::min<long long>((units + 7) / 8, current_sms() * 16LL)));
  auto kern = pbn == 256 ? (narrow ? gated_reduce_store_kernel<256, 8> : gated_reduce_store_kernel<256, 32>)
                         : (narrow ? gated_reduce_store_kernel<128, 8> : gated_reduce_store_kernel<128, 32>);
  return launch_chained(kern, blocks, 256, 0, st, "gated reduce launch", r);
}

// Reductions of one product's partial tiles, put off until after the next
// product's launch, beside which they run.
struct Pending {
  ReduceArgs r[kMaxProblems];
  int pbn = 0, n = 0;
  void add(const ReduceArgs& a, int width) {
    r[n] = a;
    r[n].beside = 1;
    pbn = width;
    ++n;
  }
  b2_status run(cudaStream_t st) {
    for (int i = 0; i < n; ++i) B2_TRY(launch_reduce_store(r[i], pbn, st));
    n = 0;
    return B2_OK;
  }
};

template <int EPI, bool A_MN, bool B_MN, int ACT = kSilu>
b2_status run_products(const Product* pr, int n, const Plan& plan, void* partial, const Gate* gate, cudaStream_t st,
                       Pending* pending = nullptr, Pending* before = nullptr) {
  Maps maps;
  Params p{};
  p.problems = n;
  p.status = device_status_ptr();
  const int pbn = plan.pbn, bhalf = pbn / 2;
  uint8_t* part = static_cast<uint8_t*>(partial);
  for (int i = 0; i < n; ++i) {
    const Product& x = pr[i];
    Problem& q = p.p[i];
    const int cols = EPI == kGate ? pbn / 2 : pbn;
    q.tiles_m = int((x.M + 255) / 256);
    q.tiles_n = int((x.N + cols - 1) / cols);
    q.M = int(x.M);
    q.N = int(x.N);
    q.kb_first = int((x.K + BK - 1) / BK);
    q.kb = q.kb_first * x.pairs;
    q.splits = plan.splits;
    q.kb_per_split = (q.kb + q.splits - 1) / q.splits;
    q.splits = (q.kb + q.kb_per_split - 1) / q.kb_per_split;
    q.item_begin = p.items;
    q.out = static_cast<uint16_t*>(x.out);
    q.ldo = x.ldo;
    q.tma_out = EPI != kStore || tma_rows(x.out, x.ldo);
    const int tiles = q.tiles_m * q.tiles_n;
    if (q.splits > 1) {
      q.partial = reinterpret_cast<float*>(part);
      part += size_t(tiles) * q.splits * 256 * pbn * 4;
    }
    p.items += tiles * q.splits;
    const int operands = x.pairs;
    for (int k = 0; k < operands; ++k) {
      B2_TRY(A_MN ? map2d(&maps.a[i + k], x.a[k], 64, 64, 128) : map2d(&maps.a[i + k], x.a[k], 64, 128, 128));
      B2_TRY(B_MN ? map2d(&maps.b[i + k], x.b[k], 64, 64, 128)
                  : map2d(&maps.b[i + k], x.b[k], 64, uint32_t(bhalf), 128));
    }
    if (EPI == kGate) B2_TRY(map2d(&maps.b[1], x.b[1], 64, uint32_t(bhalf), 128));
    if (EPI == kStore && q.tma_out) B2_TRY(map2d(&maps.o[i], {x.out, x.M, x.N, x.ldo}, 64, 32, 128));
  }
  if (EPI != kStore) {
    p.train = gate->train;
    if (EPI == kGate) {
      B2_TRY(map2d(&maps.o[0], gate->h, 32, 32, 64));
    } else {
      B2_TRY(map2d(&maps.a[1], {gate->fp, pr[0].M, pr[0].N, gate->ldf}, 32, 32, 64));
      B2_TRY(map2d(&maps.b[1], {gate->fa, pr[0].M, pr[0].N, gate->ldf}, 32, 32, 64));
      B2_TRY(map2d(&maps.o[0], {gate->fr, pr[0].M, pr[0].N, gate->ldf}, 32, 32, 64));
    }
    if (EPI == kGateBwd || gate->train) {
      B2_TRY(map2d(&maps.o[1], gate->o1, 32, 32, 64));
      B2_TRY(map2d(&maps.o[2], gate->o2, 32, 32, 64));
    }
    if (EPI == kGate && gate->train) B2_TRY(map2d(&maps.o[3], gate->o3, 32, 32, 64));
  }
  B2_TRY((pbn == 256 ? launch_gemm<EPI, 256, A_MN, B_MN, ACT>(maps, p, st)
                     : launch_gemm<EPI, 128, A_MN, B_MN, ACT>(maps, p, st)));
  if (before) B2_TRY(before->run(st));
  for (int i = 0; i < n; ++i) {
    if (p.p[i].splits <= 1) continue;
    ReduceArgs r{};
    r.q = p.p[i];
    if (EPI != kStore) {
      r.train = gate->train;
      r.h = static_cast<uint16_t*>(const_cast<void*>(gate->h.p));
      r.o1 = static_cast<uint16_t*>(const_cast<void*>(gate->o1.p));
      r.o2 = static_cast<uint16_t*>(const_cast<void*>(gate->o2.p));
      r.o3 = static_cast<uint16_t*>(const_cast<void*>(gate->o3.p));
      r.fp = gate->fp;
      r.fa = gate->fa;
      r.fr = gate->fr;
      r.ldh = gate->h.ld;
      r.ldo = gate->o1.ld;
      r.ldf = gate->ldf;
    }
    if constexpr (EPI == kStore) {
      if (pending)
        pending->add(r, pbn);
      else
        B2_TRY(launch_reduce_store(r, pbn, st));
    } else {
      const long long units = (long long)r.q.tiles_m * r.q.tiles_n * 8 * ((EPI == kGate ? pbn / 2 : pbn) / 8);
      const dim3 blocks(unsigned(std::min<long long>((units + 7) / 8, current_sms() * 16LL)));
      auto kern = pbn == 256 ? gated_reduce_kernel<EPI, 256, ACT> : gated_reduce_kernel<EPI, 128, ACT>;
      B2_TRY(launch_chained(kern, blocks, 256, 0, st, "gated reduce launch", r));
    }
  }
  return B2_OK;
}

FewMat few_mat(const Mat& m) {
  const auto* p = static_cast<const uint16_t*>(m.p);
  return {p, p + (m.rows - 1) * m.ld + m.cols, m.ld, tma_rows(m.p, m.ld) ? 1 : 0};
}

template <int EPI, int NT, int ACT, bool ALIGNED>
b2_status launch_few_nt(const FewArgs& a, cudaStream_t st) {
  int dev = 0;
  B2_TRY(check_cuda(cudaGetDevice(&dev), "cudaGetDevice"));
  using C = FewConfig<EPI, NT, ALIGNED>;
  auto kern = gated_few_kernel<EPI, NT, ACT, ALIGNED>;
  static bool configured[64] = {};
  if (dev < 0 || dev >= 64) return set_error(B2_ERR_INVALID, "device index %d", dev);
  if (!configured[dev]) {
    B2_TRY(check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(C::kStep * C::kMost)),
                      "cudaFuncSetAttribute(gated few)"));
    configured[dev] = true;
  }
  const int groups = (a.rows + 15) / 16;
  const int steps = (a.K + 31) / 32;
  // The most steps on their way with every CTA resident; where not even the
  // smallest choice is resident, that one (more CTAs a SM leave less of the
  // machine idle in the last wave).  Only Wd's reductions are shared, whose rows
  // are few and whose copies start while h is still being computed; every warp
  // keeps three steps.
  int S = 3, cluster = 1;
  long long most = 0;
  for (int c = 1; c <= (EPI == kGate ? 1 : 8) && (c == 1 || steps >= 3 * kFewWarps * c); c *= 2)
    for (int n = 3; n <= C::kMost; ++n) {
      const long long resident = 228 * 1024 / (C::kStep * n + C::kStatic + 1024) * sm_count(dev);
      const long long under_way = (long long)groups * c * (n - 1);
      if ((long long)groups * c <= resident && under_way > most) {
        most = under_way;
        S = n;
        cluster = c;
      }
    }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(groups * cluster));
  cfg.blockDim = dim3(kFewThreads);
  cfg.dynamicSmemBytes = C::kStep * S;
  cfg.stream = st;
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return check_cuda(cudaLaunchKernelEx(&cfg, kern, a, cluster, S), "gated few-token launch");
}

template <int EPI, int ACT, bool ALIGNED>
b2_status launch_few_rows(const FewArgs& a, cudaStream_t st) {
  const int tokens = EPI == kStore && a.rest ? 2 * a.M : a.M;
  if (tokens <= 8) return launch_few_nt<EPI, 1, ACT, ALIGNED>(a, st);
  if (tokens <= 16) return launch_few_nt<EPI, 2, ACT, ALIGNED>(a, st);
  if (tokens <= 24) return launch_few_nt<EPI, 3, ACT, ALIGNED>(a, st);
  return launch_few_nt<EPI, 4, ACT, ALIGNED>(a, st);
}
template <int EPI, int ACT>
b2_status launch_few(const FewArgs& a, cudaStream_t st) {
  if constexpr (EPI == kGate)  // (takes_few)
    return launch_few_rows<EPI, ACT, true>(a, st);
  else
    return a.w[0].aligned ? launch_few_rows<EPI, ACT, true>(a, st) : launch_few_rows<EPI, ACT, false>(a, st);
}

// Which forwards take the few-token kernels.  Up to 16 tokens: 16 take 12 us
// (1024 x 4096), 27 us (2048 x 5464) and 74 us (4096 x 12288) there, 22, 30 and
// 78 us on the tensor-memory path, which does not grow with the tokens.  Up to
// 32 where the projections' CTAs are resident at once: 24 tokens 13 against 22 us
// (1024 x 4096), 32 tokens 8.4 against 14.7 us (512 x 1536); where they are
// not, 24 tokens take 33 against 31 us (2048 x 5464).  Rows of Wd at any
// alignment: one token 27 against 47 us with a padded copy (2048 x 5461), 16
// tokens 34 against 39.  Where x, Wg and Wu have them too, copies pay: 81 against
// 56 us (2045 x 5461).
template <int NT>
bool few_resident(int64_t rows) {
  using C = FewConfig<kGate, NT, true>;
  return (rows + 15) / 16 <= int64_t(228 * 1024 / (C::kStep * 3 + C::kStatic + 1024)) * current_sms();
}
bool takes_few(const Mat& x, const Mat& wg, const Mat& wu) {
  if (!tma_rows(x.p, x.ld) || !tma_rows(wg.p, wg.ld) || !tma_rows(wu.p, wu.ld)) return false;
  return x.rows <= 16 || (x.rows <= 24 && few_resident<3>(wg.rows)) ||
         (x.rows <= kFewTokens && few_resident<4>(wg.rows));
}

// The forward of few tokens: two launches, no padded copies.
b2_status few_forward(const Mat& x, const Mat& wg, const Mat& wu, const Mat& wd, int act, const Mat& h,
                      uint16_t* factors, int64_t apart, uint16_t* rest, void* y, int64_t ldy, cudaStream_t st) {
  FewArgs a{};
  a.w[0] = few_mat(wg);
  a.w[1] = few_mat(wu);
  a.x = few_mat(x);
  a.M = int(x.rows);
  a.rows = int(wg.rows);
  a.K = int(x.cols);
  a.out = static_cast<uint16_t*>(const_cast<void*>(h.p));
  if (factors) {
    a.o1 = factors;
    a.o2 = factors + apart;
    a.o3 = factors + 2 * apart;
  }
  a.ldo = h.ld;
  a.rest = rest;
  a.ldr = up8(h.cols);
  B2_TRY((act == kSilu   ? launch_few<kGate, kSilu>(a, st)
          : act == kGelu ? launch_few<kGate, kGelu>(a, st)
                         : launch_few<kGate, kRelu>(a, st)));
  FewArgs d{};
  d.w[0] = few_mat(wd);
  d.x = few_mat(h);
  d.M = a.M;
  d.rows = int(wd.rows);
  d.K = int(wd.cols);
  d.early = 1;
  d.rest = rest;
  d.ldr = a.ldr;
  d.out = static_cast<uint16_t*>(y);
  d.ldo = ldy;
  return launch_few<kStore, kSilu>(d, st);
}

struct Shape {
  int64_t M, D, F, E;
};

struct FwdPlan {
  Plan gate, down;
};
FwdPlan fwd_plan(const Shape& s, int sms) {
  return {plan_product(s.M, s.F, s.D, 1, true, sms), plan_product(s.M, s.E, s.F, 1, false, sms)};
}
struct BwdPlan {
  Plan dh, dx, dw;
};
BwdPlan bwd_plan(const Shape& s, int sms) {
  BwdPlan b;
  b.dh = plan_product(s.M, s.F, s.E, 1, false, sms);
  b.dx = plan_product(s.M, s.D, s.F, 2, false, sms);
  // the three weight gradients share one launch: their tiles together
  b.dw = plan_product(2 * s.F + s.E * s.F / std::max<int64_t>(1, s.D), s.D, s.M, 1, false, sms);
  return b;
}
size_t dw_partial_bytes(const Shape& s, const Plan& p) {
  if (p.splits <= 1) return 0;
  auto tiles = [&](int64_t m, int64_t n) { return size_t((m + 255) / 256) * size_t((n + p.pbn - 1) / p.pbn); };
  return (2 * tiles(s.F, s.D) + tiles(s.E, s.F)) * size_t(p.splits) * 256 * size_t(p.pbn) * 4;
}

size_t padded_bytes(int64_t rows, int64_t cols) { return size_t(rows) * size_t(up8(cols)) * 2 + 256; }

b2_status check_shape(const char* who, int64_t M, int64_t D, int64_t F, int64_t E, int act) {
  if (M < 0 || D < 1 || F < 1 || E < 1) return set_error(B2_ERR_INVALID, "%s: bad shape", who);
  if (act < kSilu || act > kRelu) return set_error(B2_ERR_INVALID, "%s: bad activation %d", who, act);
  const int64_t big = int64_t(1) << 30;
  if (M >= big || D >= big || F >= big || E >= big)
    return set_error(B2_ERR_UNSUPPORTED, "%s: sizes must be below 2^30", who);
  return B2_OK;
}

b2_status check_ws(const char* who, size_t need, const void* ws, size_t got) {
  if (!ws || got < need || reinterpret_cast<uintptr_t>(ws) % 256)
    return set_error(B2_ERR_WORKSPACE, "%s: workspace of %zu bytes (256-byte aligned) needed, got %zu", who, need, got);
  return B2_OK;
}

}  // namespace
}  // namespace b2

using namespace b2;

extern "C" {

size_t b2_gated_mlp_fwd_workspace_bytes(int64_t M, int64_t D, int64_t F, int64_t E) {
  if (M <= 0 || D <= 0 || F <= 0 || E <= 0) return 0;
  const FwdPlan p = fwd_plan({M, D, F, E}, current_sms());
  return padded_bytes(M, F) + padded_bytes(std::min<int64_t>(M, kRestTokens), F) + padded_bytes(M, D) +
         2 * padded_bytes(F, D) + padded_bytes(E, F) + std::max(p.gate.partial_bytes, p.down.partial_bytes) + 256;
}

b2_status b2_gated_mlp_fwd_bf16(const void* x, int64_t ldx, const void* w_gate, int64_t ldg, const void* w_up,
                                int64_t ldu, const void* w_down, int64_t ldd, int act, void* y, int64_t ldy,
                                void* saved, int64_t M, int64_t D, int64_t F, int64_t E, void* workspace, size_t workspace_bytes,
                                void* stream) {
  B2_TRY(check_shape("b2_gated_mlp_fwd_bf16", M, D, F, E, act));
  if (M == 0) return B2_OK;
  if (!x || !w_gate || !w_up || !w_down || !y) return set_error(B2_ERR_INVALID, "b2_gated_mlp_fwd_bf16: null pointer");
  if (ldx < D || ldg < D || ldu < D || ldd < F || ldy < E)
    return set_error(B2_ERR_INVALID, "b2_gated_mlp_fwd_bf16: bad row stride");
  if (saved && reinterpret_cast<uintptr_t>(saved) % 16)
    return set_error(B2_ERR_INVALID, "b2_gated_mlp_fwd_bf16: saved must be 16-byte aligned");
  B2_TRY(check_ws("b2_gated_mlp_fwd_bf16", b2_gated_mlp_fwd_workspace_bytes(M, D, F, E), workspace, workspace_bytes));
  const auto st = static_cast<cudaStream_t>(stream);
  const int sms = current_sms();
  const FwdPlan plan = fwd_plan({M, D, F, E}, sms);
  Carve ws(workspace);
  const int64_t Fp = up8(F);
  const Mat h = saved ? Mat{saved, M, F, 4 * Fp} : Mat{ws.take(size_t(M) * Fp * 2), M, F, Fp};
  Mat mx{x, M, D, ldx}, mg{w_gate, F, D, ldg}, mu{w_up, F, D, ldu}, md{w_down, E, F, ldd};
  if (takes_few(mx, mg, mu)) {
    uint16_t* keep = static_cast<uint16_t*>(saved);
    uint16_t* rest = M <= kRestTokens ? static_cast<uint16_t*>(ws.take(size_t(M) * Fp * 2)) : nullptr;
    return few_forward(mx, mg, mu, md, act, h, keep ? keep + Fp : nullptr, Fp, rest, y, ldy, st);
  }
  Padder pad;
  pad.add(mx, ws);
  pad.add(mg, ws);
  pad.add(mu, ws);
  pad.add(md, ws);
  B2_TRY(pad.run(st));
  void* partial = ws.take(std::max(plan.gate.partial_bytes, plan.down.partial_bytes));
  Gate gate;
  gate.train = saved != nullptr;
  gate.h = h;
  if (saved) {
    gate.o1 = {static_cast<uint16_t*>(saved) + Fp, M, F, 4 * Fp};
    gate.o2 = {static_cast<uint16_t*>(saved) + 2 * Fp, M, F, 4 * Fp};
    gate.o3 = {static_cast<uint16_t*>(saved) + 3 * Fp, M, F, 4 * Fp};
  }
  Product up;
  up.a[0] = mx;
  up.b[0] = mg;
  up.b[1] = mu;
  up.M = M;
  up.N = F;
  up.K = D;
  B2_TRY((act == kSilu   ? run_products<kGate, false, false, kSilu>(&up, 1, plan.gate, partial, &gate, st)
          : act == kGelu ? run_products<kGate, false, false, kGelu>(&up, 1, plan.gate, partial, &gate, st)
                         : run_products<kGate, false, false, kRelu>(&up, 1, plan.gate, partial, &gate, st)));
  Product down;
  down.a[0] = h;
  down.b[0] = md;
  down.M = M;
  down.N = E;
  down.K = F;
  down.out = y;
  down.ldo = ldy;
  return run_products<kStore, false, false>(&down, 1, plan.down, partial, nullptr, st);
}

size_t b2_gated_mlp_bwd_workspace_bytes(int64_t M, int64_t D, int64_t F, int64_t E) {
  if (M <= 0 || D <= 0 || F <= 0 || E <= 0) return 0;
  const Shape s{M, D, F, E};
  const BwdPlan p = bwd_plan(s, current_sms());
  return 2 * padded_bytes(M, F) + padded_bytes(M, D) + padded_bytes(M, E) + 2 * padded_bytes(F, D) +
         padded_bytes(E, F) +
         std::max(p.dh.partial_bytes, p.dx.partial_bytes) + dw_partial_bytes(s, p.dw) + 512;
}

b2_status b2_gated_mlp_bwd_bf16(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w_gate,
                                int64_t ldg, const void* w_up, int64_t ldu, const void* w_down, int64_t ldd, int act,
                                const void* saved, void* dx, void* dw_gate, void* dw_up, void* dw_down, int64_t M,
                                int64_t D, int64_t F, int64_t E, void* workspace, size_t workspace_bytes,
                                void* stream) {
  B2_TRY(check_shape("b2_gated_mlp_bwd_bf16", M, D, F, E, act));
  const auto st = static_cast<cudaStream_t>(stream);
  if (M == 0) {
    // no tokens: the weights' gradients are zero
    void* out[3] = {dw_gate, dw_up, dw_down};
    for (int i = 0; i < 3; ++i)
      if (out[i])
        B2_TRY(check_cuda(cudaMemsetAsync(out[i], 0, size_t(F) * size_t(i < 2 ? D : E) * 2, st), "gradient memset"));
    return B2_OK;
  }
  if (!dy || !x || !w_gate || !w_up || !w_down || !saved)
    return set_error(B2_ERR_INVALID, "b2_gated_mlp_bwd_bf16: null pointer");
  if (lddy < E || ldx < D || ldg < D || ldu < D || ldd < F)
    return set_error(B2_ERR_INVALID, "b2_gated_mlp_bwd_bf16: bad row stride");
  if (reinterpret_cast<uintptr_t>(saved) % 16)
    return set_error(B2_ERR_INVALID, "b2_gated_mlp_bwd_bf16: saved must be 16-byte aligned");
  B2_TRY(check_ws("b2_gated_mlp_bwd_bf16", b2_gated_mlp_bwd_workspace_bytes(M, D, F, E), workspace, workspace_bytes));
  const Shape s{M, D, F, E};
  const BwdPlan plan = bwd_plan(s, current_sms());
  Carve ws(workspace);
  const int64_t Fp = up8(F);
  const Mat h{saved, M, F, 4 * Fp};
  uint16_t* dgu = static_cast<uint16_t*>(ws.take(size_t(M) * Fp * 4));
  const Mat dg{dgu, M, F, 2 * Fp}, du{dgu + Fp, M, F, 2 * Fp};
  Mat mdy{dy, M, E, lddy}, mx{x, M, D, ldx}, mg{w_gate, F, D, ldg}, mu{w_up, F, D, ldu}, md{w_down, E, F, ldd};
  Padder pad;
  pad.add(mdy, ws);
  if (dw_gate || dw_up) pad.add(mx, ws);
  if (dx) {
    pad.add(mg, ws);
    pad.add(mu, ws);
  }
  pad.add(md, ws);
  B2_TRY(pad.run(st));
  void* partial =
      ws.take(std::max(plan.dh.partial_bytes, plan.dx.partial_bytes));
  void* dw_partial = ws.take(dw_partial_bytes(s, plan.dw));  // dx's are added later
  Gate gate;
  gate.o1 = dg;
  gate.o2 = du;
  gate.fp = static_cast<const uint16_t*>(saved) + Fp;
  gate.fa = gate.fp + Fp;
  gate.fr = gate.fa + Fp;
  gate.ldf = 4 * Fp;
  Product t;
  t.a[0] = mdy;
  t.b[0] = md;
  t.M = M;
  t.N = F;
  t.K = E;
  B2_TRY((run_products<kGateBwd, false, true>(&t, 1, plan.dh, partial, &gate, st)));
  Pending dx_sums;  // added while the weights' gradients are computed
  const bool weights = dw_gate || dw_up || dw_down;
  if (dx) {
    Product d;
    d.a[0] = dg;
    d.a[1] = du;
    d.b[0] = mg;
    d.b[1] = mu;
    d.pairs = 2;
    d.M = M;
    d.N = D;
    d.K = F;
    d.out = dx;
    d.ldo = D;
    B2_TRY((run_products<kStore, false, true>(&d, 1, plan.dx, partial, nullptr, st, weights ? &dx_sums : nullptr)));
  }
  Product w[3];
  int n = 0;
  auto weight = [&](void* out, const Mat& a, const Mat& b) {
    if (!out) return;
    Product& q = w[n++];
    q.a[0] = a;  // [M][rows]: the tokens are the reduction
    q.b[0] = b;
    q.M = a.cols;
    q.N = b.cols;
    q.K = M;
    q.out = out;
    q.ldo = b.cols;
  };
  weight(dw_gate, dg, mx);
  weight(dw_up, du, mx);
  weight(dw_down, mdy, h);
  if (n == 0) return B2_OK;
  return run_products<kStore, true, true>(w, n, plan.dw, dw_partial, nullptr, st, nullptr, &dx_sums);
}

}  // extern "C"
