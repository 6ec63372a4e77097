// Sparse attention over key tiles that a cheap score selects: rt_select_tiles
// turns a tile plan into a plan of fewer tiles, which the attention kernels
// run on unchanged.
//
//   kbar[h][t] = bf16(mean of the keys of tile t),  qbar[h][G] = bf16(mean of
//   the queries of group G)  (group consecutive queries; group = 1: q itself)
//   score[G][t] = sum over heads and dims of qbar kbar
//   candidates of G: tiles t other than G's own in which some query of G has
//   a live element of the plan
//   selected[G] = the own tile + the `keep` candidates of highest score
//   (equal scores: lowest tile first; NaN counts as -inf)
//   new mask = old mask, where selected[query's group][key's tile]
//
// The own tile always stays, and with it the diagonal, so every row keeps a
// live element (which the attention forward relies on).
//
// Means are quotients of 64-bit sums, rounded to fp32 and from there to bf16,
// so a score is a sum of products of bf16 numbers, and the choice goes by its
// exact value: the scores of 128 groups x all tiles are one tcgen05
// accumulation over the heads (fp32 in tensor memory), good to a bound that the
// norms give, and a group whose keep-th score has another within twice that
// bound is decided again, between those tiles alone, by 64-bit sums.
//
// Three kernels and the plan's lists: means (memory-bound: k once, and q once
// for group > 1), scores and choice (q or the means once; the scores never
// leave the SM), and the plan (element bits of the tiles that stay).
#include "rt_device.cuh"
#include "rt_internal.h"

namespace rt {
namespace select {

// Exact widening and one rounding, subnormal numbers among them: a cast would
// flush those to zero under --use_fast_math.
__device__ __forceinline__ double widen(float x) {
  double d;
  asm("cvt.f64.f32 %0, %1;" : "=d"(d) : "f"(x));
  return d;
}
__device__ __forceinline__ float narrow(double x) {
  float f;
  asm("cvt.rn.f32.f64 %0, %1;" : "=f"(f) : "d"(x));
  return f;
}

// A warp's means of 8 columns a lane: lane l holds columns 8 (l % CH) .. + 8
// of rows l / CH, + RL, ... of a run; sums in 64 bits.
template <int DH>
struct MeanLanes {
  static constexpr int CH = DH / 8, RL = 32 / CH;  // 8-column chunks of a row, rows of a warp's 16-byte step
  double acc[8];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.0;
  }
  __device__ __forceinline__ void add(const uint4& u) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack_bf16x2(w[i]);
      acc[2 * i] += widen(f.x);
      acc[2 * i + 1] += widen(f.y);
    }
  }
  // Adds up the STEP lanes (of consecutive rows) that share a column, divides
  // by `count` and returns the bf16 means; `sq` their sum of squares. WHOLE:
  // count is a power of two, whose reciprocal gives the quotient. For a run cut
  // short by the sequence's end one step more, of the remainder, does: with the
  // reciprocal correctly rounded so is the result (Markstein, 1990). Groups of 2
  // and 4 of 8 x 16 x 4096 x 64 took 54 and 58 us with quotients throughout,
  // instead of 44 and 45.
  template <int STEP, bool WHOLE>
  __device__ __forceinline__ uint4 means(int count, float& sq) {
    const double n = (double)max(count, 1), inv = 1.0 / n;
    float m[8];
    sq = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int off = 1; off < STEP; off *= 2) acc[e] += __shfl_xor_sync(0xFFFFFFFFu, acc[e], off * CH);
      double q = acc[e] * inv;
      if (!WHOLE) {
        const double rest = fma(-q, n, acc[e]);
        if (rest == rest) q = fma(rest, inv, q);  // of an infinite sum there is none
      }
      m[e] = __bfloat162float(__float2bfloat16_rn(narrow(q)));
      sq = fmaf(m[e], m[e], sq);
    }
    return make_uint4(pack_bf16x2(m[0], m[1]), pack_bf16x2(m[2], m[3]), pack_bf16x2(m[4], m[5]),
                      pack_bf16x2(m[6], m[7]));
  }
};

// Mean of one run of up to 128 rows, by a warp, 8 loads in flight per lane;
// with `norm2` also its sum of squares.
template <int DH>
__device__ __forceinline__ void long_mean(const uint16_t* __restrict__ src, int rows, uint16_t* __restrict__ dst,
                                          float* __restrict__ norm2, int lane) {
  using M = MeanLanes<DH>;
  M sum;
  sum.clear();
  const uint4* p = reinterpret_cast<const uint4*>(src) + lane;
  const int rl = lane / M::CH;
#pragma unroll 1
  for (int i0 = 0; i0 * M::RL < rows; i0 += 8) {
    uint4 u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u[i] = make_uint4(0u, 0u, 0u, 0u);
      if ((i0 + i) * M::RL + rl < rows) u[i] = p[(i0 + i) * 32];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum.add(u[i]);
  }
  float sq;
  const uint4 m = rows & (rows - 1) ? sum.template means<M::RL, false>(rows, sq)
                                    : sum.template means<M::RL, true>(rows, sq);
  if (rl == 0) reinterpret_cast<uint4*>(dst)[lane] = m;
  if (norm2 != nullptr) {
#pragma unroll
    for (int off = 1; off < M::CH; off *= 2) sq += __shfl_xor_sync(0xFFFFFFFFu, sq, off);
    if (lane == 0) *norm2 = sq;
  }
}

// Means of the runs of SIZE <= 32 rows among 32 rows (WHOLE), or fewer at the
// end of a sequence, by a warp that loads all of them first.
template <int DH, int SIZE, bool WHOLE>
__device__ __forceinline__ void short_means(const uint16_t* __restrict__ src, int rows, uint16_t* __restrict__ dst,
                                            int lane) {
  using M = MeanLanes<DH>;
  constexpr int N = 32 / M::RL;                         // 16-byte steps
  constexpr int PER = SIZE > M::RL ? SIZE / M::RL : 1;  // of a run
  constexpr int STEP = SIZE < M::RL ? SIZE : M::RL;     // row lanes of a run
  const uint4* p = reinterpret_cast<const uint4*>(src) + lane;
  const int chunk = lane % M::CH, rl = lane / M::CH;
  uint4 u[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    u[i] = make_uint4(0u, 0u, 0u, 0u);
    if (WHOLE || i * M::RL + rl < rows) u[i] = p[i * 32];
  }
#pragma unroll
  for (int i = 0; i < N; i += PER) {
    M sum;
    sum.clear();
#pragma unroll
    for (int j = 0; j < PER; ++j) sum.add(u[i + j]);
    const int run = (i * M::RL + rl) / SIZE, count = WHOLE ? SIZE : min(SIZE, rows - run * SIZE);
    float sq;
    const uint4 m = sum.template means<STEP, WHOLE>(count, sq);
    if (count > 0 && rl % STEP == 0) reinterpret_cast<uint4*>(dst + run * DH)[chunk] = m;
  }
}

// One warp per tile of k and, for SIZE > 1 (the group), per run of q or, of
// runs shorter than 32 rows, per 32 rows.
constexpr int kMeanWarps = 4;  // small blocks spread more evenly: 4096 tiles 16.0 us with 8 warps, 15.5 with 4

template <int DH, int SIZE>
__global__ void __launch_bounds__(32 * kMeanWarps, 32 / kMeanWarps) means_kernel(const uint16_t* __restrict__ q, const uint16_t* __restrict__ k,
                                                       long long BH, int S, int T, int groups,
                                                       uint16_t* __restrict__ qbar, uint16_t* __restrict__ kbar,
                                                       float* __restrict__ knorm2) {
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  long long task = (long long)blockIdx.x * kMeanWarps + (threadIdx.x >> 5);
  const long long tiles = BH * T;
  if (task < tiles) {
    const long long bh = task / T;
    const int t = (int)(task - bh * T);
    long_mean<DH>(k + (bh * S + t * RT_TILE) * DH, min(RT_TILE, S - t * RT_TILE), kbar + task * DH, knorm2 + task, lane);
  } else if (SIZE > 1) {
    constexpr int SPAN = SIZE < 32 ? 32 : SIZE;
    task -= tiles;
    const int parts = (S + SPAN - 1) / SPAN;
    const long long bh = task / parts;
    if (bh >= BH) return;  // a whole warp
    const int start = (int)(task - bh * parts) * SPAN, rows = min(SPAN, S - start);
    const uint16_t* src = q + (bh * S + start) * DH;
    uint16_t* dst = qbar + (bh * groups + start / SIZE) * DH;
    if constexpr (SIZE <= 32 && SIZE > 1) {
      if (rows == SPAN) short_means<DH, SIZE, true>(src, rows, dst, lane);
      else short_means<DH, SIZE, false>(src, rows, dst, lane);
    } else long_mean<DH>(src, rows, dst, nullptr, lane);
  }
}

// ---------------------------------------------------------------------------
// Scores and choice: one CTA per (128 groups, sample), 320 threads:
//   warp 0     producer: per head the groups' tile of q (or means) and the
//              tiles' means (TMA), into a ring of stages
//   warp 1     MMA: scores [128][T] += q_h kbar_h^T, in tensor memory
//   warps 2-5  one thread per group (TMEM lane): sum of squares of its row from
//              the ring while the MMAs run, then the choice
//   warps 6-9  meanwhile the groups' candidates, from the plan
// The choice of a thread: the keep-th largest score by bisection over the
// values (a pass over the T columns each, typically under ten), then the
// scores within twice the error bound of it.
// ---------------------------------------------------------------------------
constexpr int kSelThreads = 320;
constexpr int kSelMaxStages = 6;
constexpr int kMaxTiles = 512;

template <int DH>
struct SelCfg {
  static constexpr int kRowBytes = DH * 2;
  static constexpr int kTileBytes = RT_TILE * kRowBytes;
  static constexpr uint32_t kSwizzle = DH == 64 ? SW_128B : SW_64B;
  static constexpr int kSBO = 8 * kRowBytes;
};

// Shared memory behind the ring: the groups' candidate, chosen and ambiguous
// tiles as words, and each choosing warp's list of 64-bit scores.
struct SelLayout {
  int chunks, stages, stage_bytes, words, cand, chosen, close, exact, items, total;
};
inline __host__ __device__ SelLayout sel_layout(int T, int tile_bytes, int stages) {
  SelLayout l;
  l.chunks = (T + RT_TILE - 1) / RT_TILE;
  l.stage_bytes = (1 + l.chunks) * tile_bytes;
  l.stages = stages;
  l.words = (T + 31) / 32;
  const int words = RT_TILE * l.words * 4;
  l.cand = l.stages * l.stage_bytes;
  l.chosen = l.cand + words;
  l.close = l.chosen + words;
  l.exact = l.close + words;
  l.items = l.exact + 4 * T * 8;
  l.total = l.items + 4 * T * 2 + 1024;
  return l;
}
// Stages of the ring: three where CTAs share an SM (up to 128 tiles), as many
// as fit where there are fewer CTAs than SMs, which wait for their loads alone.
inline int sel_stages(int T, int tile_bytes, long long ctas) {
  const int chunks = (T + RT_TILE - 1) / RT_TILE;
  if (ctas > 148 && chunks == 1) return 3;
  int stages = kSelMaxStages;
  while (stages > 2 && sel_layout(T, tile_bytes, stages).total > 224 * 1024) --stages;
  return stages;
}

struct __align__(8) SelBarriers {
  uint64_t full[kSelMaxStages], empty[kSelMaxStages], done;
};

// Exact scores of up to 4 tiles for one group, by a warp (every lane gets them).
template <int DH>
__device__ __forceinline__ void exact_scores(const uint16_t* __restrict__ qrows, const uint16_t* __restrict__ kbar,
                                             int H, long long b, int g, int groups, int T, const int (&tile)[4], int n,
                                             int lane, double (&s)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = 0.0;
  constexpr int LW = DH / 2;  // 4-byte words of a row; DH = 32: two heads per step
  constexpr int HP = 32 / LW;
  const int col = lane % LW;
#pragma unroll 8
  for (int h0 = 0; h0 < H; h0 += HP) {
    const int h = h0 + lane / LW;
    if (h < H) {
      const float2 q = unpack_bf16x2(
          __ldg(reinterpret_cast<const uint32_t*>(qrows + ((b * H + h) * groups + g) * DH) + col));
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i < n) {
          const float2 k = unpack_bf16x2(
              __ldg(reinterpret_cast<const uint32_t*>(kbar + ((b * H + h) * T + tile[i]) * DH) + col));
          s[i] = fma(widen(q.x), widen(k.x), s[i]);
          s[i] = fma(widen(q.y), widen(k.y), s[i]);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s[i] += __shfl_xor_sync(0xFFFFFFFFu, s[i], off);
}

template <int DH>
__global__ void __launch_bounds__(kSelThreads, 2) select_kernel(
    const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
    const uint16_t* __restrict__ qrows, const uint16_t* __restrict__ kbar, const float* __restrict__ knorm2, int H,
    int stages, int group, int groups, int keep, rt_tile_plan plan, uint8_t* __restrict__ selected,
    uint32_t* __restrict__ chosen_bits) {
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  using C = SelCfg<DH>;
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ SelBarriers bars;
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_flag;
  __shared__ float s_kmax[4];
  __shared__ int s_undecided, s_need[RT_TILE];
  __shared__ uint8_t s_row[RT_TILE];
  const int T = plan.tiles, W = plan.words;
  const SelLayout L = sel_layout(T, C::kTileBytes, stages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int row0 = blockIdx.x * RT_TILE;
  const long long b = blockIdx.y;
  const uint32_t tmem_cols = L.chunks == 1 ? 128u : L.chunks == 2 ? 256u : 512u;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    s_undecided = 0;
    for (int i = 0; i < L.stages; ++i) {
      mbar_init(&bars.full[i], 1);
      mbar_init(&bars.empty[i], 1 + 4);
    }
    mbar_init(&bars.done, 1);
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&tmem_base_s, tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  if (warp == 0) {
    // ---------------- producer ----------------
    int h = 0;
    for (; h < H; ++h) {
      const int st = h % L.stages;
      if (h >= L.stages && !mbar_wait_warp(&bars.empty[st], ((h / L.stages) - 1) & 1, &abort_flag)) break;
      if (lane == 0) {
        uint8_t* at = smem + st * L.stage_bytes;
        mbar_arrive_expect_tx(&bars.full[st], L.stage_bytes);
        tma_load_3d(at, &tm_q, &bars.full[st], 0, row0, (int)(b * H + h));
        for (int c = 0; c < L.chunks; ++c)
          tma_load_3d(at + (1 + c) * C::kTileBytes, &tm_k, &bars.full[st], 0, c * RT_TILE, (int)(b * H + h));
      }
      __syncwarp();
    }
    // drain: every load issued must land before the CTA exits
    volatile int no_abort = 0;
    for (int i = max(0, h - L.stages); i < h; ++i) mbar_wait_warp(&bars.full[i % L.stages], (i / L.stages) & 1, &no_abort);
  } else if (warp == 1) {
    // ---------------- MMA: the whole warp waits, one elected lane issues ----------------
    const bool leader = elect_one_sync();
    for (int h = 0; h < H; ++h) {
      const int st = h % L.stages;
      if (!mbar_wait_warp(&bars.full[st], (h / L.stages) & 1, &abort_flag)) break;
      tc_fence_after();
      const uint8_t* at = smem + st * L.stage_bytes;
      const uint64_t qd = sdesc(smem_u32(at), 16, C::kSBO, C::kSwizzle);
      if (leader) {
        for (int c = 0; c < L.chunks; ++c) {
          const uint64_t kd = sdesc(smem_u32(at + (1 + c) * C::kTileBytes), 16, C::kSBO, C::kSwizzle);
          const uint32_t idesc = idesc_bf16_f32(128, min(128, (T - c * RT_TILE + 15) / 16 * 16), false, false);
#pragma unroll
          for (int ks = 0; ks < DH / 16; ++ks)
            mma_ss(tmem + c * 128, qd + ks * 2, kd + ks * 2, idesc, h > 0 || ks > 0 ? 1u : 0u);
        }
        mma_commit(&bars.empty[st]);
      }
      __syncwarp();
    }
    if (leader) mma_commit(&bars.done);
    __syncwarp();
    volatile int no_abort = 0;
    mbar_wait_warp(&bars.done, 0, &no_abort);
  } else if (warp >= 6) {
    // ---------------- candidates ----------------
    const int part = warp - 6, row = part * 32 + lane;  // of the CTA's groups
    const int g = row0 + row;
    const bool in = g < groups;
    uint32_t* cand = reinterpret_cast<uint32_t*>(smem + L.cand) + row * W;
    uint32_t* chosen = reinterpret_cast<uint32_t*>(smem + L.chosen) + row * W;
    uint32_t* close = reinterpret_cast<uint32_t*>(smem + L.close) + row * W;
    // candidates: live tiles of the group's query tile in which one of its queries has an element,
    // all of them for fully live tiles and for groups of a whole query tile
    const int first = in ? g * group : 0, qt = first / RT_TILE;
    for (int w = 0; w < W; ++w) {
      uint32_t mine = 0u;
      if (in) {
        const size_t at = ((size_t)b * T + qt) * W + w;
        mine = group == RT_TILE ? plan.live_bits[at] : plan.full_bits[at];
        if ((qt >> 5) == w) mine &= ~(1u << (qt & 31));
      }
      cand[w] = mine;
      chosen[w] = in && (qt >> 5) == w ? 1u << (qt & 31) : 0u;
      close[w] = 0u;
    }
    if (group < RT_TILE) {
      // the others by tile, shared out over the warps: a lane reads the element bits of 4 queries,
      // ballots make 128 bits of the queries that have some, and each group looks at its own
      asm volatile("bar.sync 2, 128;" ::: "memory");
      const int per = RT_TILE / group;  // groups of a query tile
      const int qt0 = row0 / per, qt1 = min(T, qt0 + group);
      uint32_t* all_cand = reinterpret_cast<uint32_t*>(smem + L.cand);
      // (query tile, word) pairs, 32 at a time; every fourth of their tiles, kBatch of them at once
      constexpr int kBatch = 2;
      const int pairs = (qt1 - qt0) * W;
      int turn = 0, n = 0;
      int tx[kBatch], tt[kBatch];  // query tile (relative) and key tile of the batch
#pragma unroll
      for (int k = 0; k < kBatch; ++k) tx[k] = tt[k] = 0;
      auto look = [&]() {
        uint4 e[kBatch][4];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          const uint4* m = reinterpret_cast<const uint4*>(plan.tile_masks) +
                           (((size_t)b * T + qt0 + tx[k]) * T + tt[k]) * RT_TILE + lane;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            e[k][i] = make_uint4(0u, 0u, 0u, 0u);
            if (k < n) e[k][i] = __ldg(m + 32 * i);
          }
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
          uint32_t some[4];
#pragma unroll
          for (int i = 0; i < 4; ++i)
            some[i] = __ballot_sync(kAll, (e[k][i].x | e[k][i].y | e[k][i].z | e[k][i].w) != 0u);
          for (int j = lane; j < per; j += 32) {
            const int at_q = j * group;
            uint32_t mine = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int lo = max(at_q - 32 * i, 0), hi = min(at_q + group - 32 * i, 32);  // of word i
              if (lo < hi) mine |= some[i] & (hi - lo == 32 ? kAll : ((1u << (hi - lo)) - 1u) << lo);
            }
            if (mine) atomicOr(all_cand + (tx[k] * per + j) * W + (tt[k] >> 5), 1u << (tt[k] & 31));
          }
        }
        n = 0;
      };
      for (int p0 = 0; p0 < pairs; p0 += 32) {
        const int mine = p0 + lane, x = mine / W, w = mine - x * W;
        uint32_t bits = 0u;
        if (mine < pairs) {
          const size_t at = ((size_t)b * T + qt0 + x) * W + w;
          bits = plan.live_bits[at] & ~plan.full_bits[at];
          if (((qt0 + x) >> 5) == w) bits &= ~(1u << ((qt0 + x) & 31));
        }
        uint32_t have = __ballot_sync(kAll, bits != 0u);
        while (have) {  // warp-uniform
          const int src = __ffs(have) - 1;
          have &= have - 1u;
          uint32_t left = __shfl_sync(kAll, bits, src);
          const int sx = __shfl_sync(kAll, x, src), sw = __shfl_sync(kAll, w, src);
          while (left) {
            const int u = __ffs(left) - 1;
            left &= left - 1u;
            if ((turn++ & 3) != part) continue;
#pragma unroll
            for (int k = 0; k < kBatch; ++k)
              if (k == n) {
                tx[k] = sx;
                tt[k] = sw * 32 + u;
              }
            if (++n == kBatch) look();
          }
        }
      }
      if (n) look();
    }
    __threadfence_block();
    asm volatile("bar.arrive 3, 256;" ::: "memory");
  } else {
    // ---------------- choice: one thread per group ----------------
    const int quad = warp & 3, part = warp - 2;
    const int row = quad * 32 + lane;  // of the CTA's groups, and the TMEM lane
    const int g = row0 + row;
    const bool in = g < groups;
    const uint32_t taddr = tmem + ((uint32_t)(quad * 32) << 16);
    uint32_t* cand = reinterpret_cast<uint32_t*>(smem + L.cand) + row * W;
    uint32_t* chosen = reinterpret_cast<uint32_t*>(smem + L.chosen) + row * W;
    uint32_t* close = reinterpret_cast<uint32_t*>(smem + L.close) + row * W;
    // Error bound of the scores. A step adds 16 products to the sum so far; with every addend cut off below
    // the 24 bits of the largest and the result below its own, 18 units of the largest addend. Neither that
    // nor the sum after it exceeds |q'| |kbar'|, the norms of all heads up to the step's (Cauchy-Schwarz), and
    // the sum of those products over the heads not sqrt(Q K), Q and K the sums of their squares.
    float kmax = 0.f;  // the largest K
    bool bad = false;
    for (int t = part * 32 + lane; t < T; t += 128) {
      float s = 0.f, k2 = 0.f;
#pragma unroll 8
      for (int h = 0; h < H; ++h) {
        k2 += knorm2[((size_t)b * H + h) * T + t];
        s += k2;
      }
      bad = bad || !(s < 1e30f);
      kmax = fmaxf(kmax, s);
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) kmax = fmaxf(kmax, __shfl_xor_sync(kAll, kmax, off));
    if (__any_sync(kAll, bad)) kmax = INFINITY;
    if (lane == 0) s_kmax[part] = kmax;
    asm volatile("bar.sync 1, 128;" ::: "memory");
    kmax = fmaxf(fmaxf(s_kmax[0], s_kmax[1]), fmaxf(s_kmax[2], s_kmax[3]));
    float q2 = 0.f, qsum = 0.f;  // |q'|^2, Q
    bool ok = true;
    for (int h = 0; h < H; ++h) {
      const int st = h % L.stages;
      if (!(ok = mbar_wait_warp(&bars.full[st], (h / L.stages) & 1, &abort_flag))) break;
      const uint4* at = reinterpret_cast<const uint4*>(smem + st * L.stage_bytes + row * C::kRowBytes);
#pragma unroll
      for (int c = 0; c < C::kRowBytes / 16; ++c) {  // any order of the row's chunks: one without bank conflicts
        const layer::F8 f = layer::unpack8(at[DH == 64 ? c ^ (lane & 7) : c ^ ((lane >> 1) & 3)]);
#pragma unroll
        for (int e = 0; e < 8; ++e) q2 = fmaf(f.v[e], f.v[e], q2);
      }
      qsum += q2;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bars.empty[st]);
    }
    // a little more for the fp32 sums Q and K themselves
    const float eps = 18.f * (DH / 16) * 1.1920929e-7f * (1.01f + (float)(H * DH) * 1.1920929e-7f);
    const bool bound = qsum > 1e-30f && qsum < 1e30f && kmax > 1e-30f && kmax < 1e30f;
    const float band = bound ? 2.f * (eps * sqrtf(qsum) * sqrtf(kmax) + 1e-35f) : INFINITY;
    asm volatile("bar.sync 3, 256;" ::: "memory");  // the candidates
    int n_cand = 0;
    for (int w = 0; w < W; ++w) n_cand += __popc(cand[w]);
    ok = ok && mbar_wait_warp(&bars.done, 0, &abort_flag);
    if (ok) {
      tc_fence_after();
      const bool all = n_cand <= keep;       // every candidate is kept
      const bool none = keep == 0 || n_cand == 0;
      bool exact = !all && !none && !bound;  // decided by 64-bit scores: the tiles in `close`
      bool search = !all && !none && bound;
      int need = keep;
      auto pass = [&](auto&& f) {  // the row's scores, 32 columns at a time
        for (int w = 0; w < W; ++w) {
          uint32_t r[32];
          tmem_ld32(taddr + w * 32, r);
          tmem_wait_ld();
          f(w, r);
        }
      };
      if (__any_sync(kAll, search)) {
        float lo = INFINITY, top = -INFINITY;
        pass([&](int w, const uint32_t(&r)[32]) {
          const uint32_t m = cand[w];
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if ((m >> e) & 1u) {
              lo = fminf(lo, __uint_as_float(r[e]));
              top = fmaxf(top, __uint_as_float(r[e]));
            }
        });
        // count(>= lo) >= keep > count(>= hi): the keep-th largest is in [lo, hi)
        float hi = top + fabsf(top) * 2.4e-7f + 1e-37f;
        bool going = search;
        while (__any_sync(kAll, going)) {  // three thresholds a pass
          const float mid = 0.5f * lo + 0.5f * hi, q1 = 0.5f * lo + 0.5f * mid, q3 = 0.5f * mid + 0.5f * hi;
          going = going && mid > lo && mid < hi;
          int n1 = 0, n2 = 0, n3 = 0;
          pass([&](int w, const uint32_t(&r)[32]) {
            const uint32_t m = cand[w];
            uint32_t g1 = 0u, g2 = 0u, g3 = 0u;
#pragma unroll
            for (int e = 0; e < 32; ++e) {
              const float x = __uint_as_float(r[e]);
              g1 |= x >= q1 ? 1u << e : 0u;
              g2 |= x >= mid ? 1u << e : 0u;
              g3 |= x >= q3 ? 1u << e : 0u;
            }
            n1 += __popc(g1 & m);
            n2 += __popc(g2 & m);
            n3 += __popc(g3 & m);
          });
          if (going) {
            if (n2 >= keep) {
              lo = n3 >= keep ? q3 : mid;
              hi = n3 >= keep ? hi : q3;
            } else {
              hi = n1 >= keep ? mid : q1;
              lo = n1 >= keep ? q1 : lo;
            }
            going = n1 != keep && n2 != keep && n3 != keep;
            if (n1 == keep) lo = q1;
            if (n2 == keep) lo = mid;
            if (n3 == keep) lo = q3;
          }
        }
        // the keep-th largest itself: the smallest score >= lo
        float kth = INFINITY;
        pass([&](int w, const uint32_t(&r)[32]) {
          const uint32_t m = cand[w];
#pragma unroll
          for (int e = 0; e < 32; ++e)
            if (((m >> e) & 1u) && __uint_as_float(r[e]) >= lo) kth = fminf(kth, __uint_as_float(r[e]));
        });
        int sure = 0, near = 0;
        pass([&](int w, const uint32_t(&r)[32]) {
          const uint32_t m = cand[w];
          uint32_t above = 0u, about = 0u;
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float d = __uint_as_float(r[e]) - kth;
            above |= d > band ? 1u << e : 0u;
            about |= fabsf(d) <= band ? 1u << e : 0u;
          }
          if (search) {
            chosen[w] |= above & m;
            close[w] = about & m;
          }
          sure += __popc(above & m);
          near += __popc(about & m);
        });
        if (search) {
          need = keep - sure;
          exact = near != need;
        }
      }
      // settled without another look: the close ones as well, or all candidates
      if (!exact) {
        for (int w = 0; w < W; ++w) {
          if (all) chosen[w] |= cand[w];
          else if (!none) chosen[w] |= close[w];
        }
      } else if (!bound) {
        for (int w = 0; w < W; ++w) close[w] = cand[w];
      }
      if (exact) {
        const int i = atomicAdd(&s_undecided, 1);
        s_row[i] = (uint8_t)row;
        s_need[i] = need;
      }
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");  // also by warps that gave up a wait
    // the undecided groups (in any order: they do not depend on one another), a warp each at a time
    double* score = reinterpret_cast<double*>(smem + L.exact) + part * T;
    uint16_t* item = reinterpret_cast<uint16_t*>(smem + L.items) + part * T;
    for (int at = part; ok && at < s_undecided; at += 4) {
      const int r = s_row[at], wanted = s_need[at];
      const uint32_t* m = reinterpret_cast<const uint32_t*>(smem + L.close) + r * W;
      int n = 0, have = 0, tile[4] = {0, 0, 0, 0};
      auto run = [&]() {
        double s[4];
        exact_scores<DH>(qrows, kbar, H, b, row0 + r, groups, T, tile, have, lane, s);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (lane == 0 && i < have) {
            score[n + i] = isnan(s[i]) ? -INFINITY : s[i];
            item[n + i] = (uint16_t)tile[i];
          }
        n += have;
        have = 0;
      };
      for (int w = 0; w < W; ++w) {
        uint32_t bits = m[w];
        while (bits) {  // warp-uniform
          const int t = w * 32 + __ffs(bits) - 1;
          bits &= bits - 1u;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i == have) tile[i] = t;
          if (++have == 4) run();
        }
      }
      if (have) run();
      __syncwarp();
      for (int i = lane; i < n; i += 32) {
        int before = 0;
        for (int j = 0; j < n; ++j) before += score[j] > score[i] || (score[j] == score[i] && j < i);
        if (before < wanted)
          atomicOr(reinterpret_cast<uint32_t*>(smem + L.chosen) + r * W + (item[i] >> 5), 1u << (item[i] & 31));
      }
      __syncwarp();
    }
    asm volatile("bar.sync 1, 128;" ::: "memory");
    if (ok) {
      // the CTA's rows of `selected` are contiguous
      const int rows_in = min(RT_TILE, groups - row0);
      const uint32_t* all_chosen = reinterpret_cast<const uint32_t*>(smem + L.chosen);
      const size_t base = ((size_t)b * groups + row0);
      const int id = part * 32 + lane;
      if (T % 4 == 0) {
        uint32_t* dst = reinterpret_cast<uint32_t*>(selected + base * T);
        for (int i = id; i < rows_in * (T / 4); i += 128) {
          const int r = i / (T / 4), t = i % (T / 4) * 4;
          const uint32_t four = all_chosen[r * W + (t >> 5)] >> (t & 31);
          dst[i] = (four & 1u) | (four & 2u) << 7 | (four & 4u) << 14 | (four & 8u) << 21;
        }
      } else {
        for (int i = id; i < rows_in * T; i += 128) {
          const int r = i / T, t = i % T;
          selected[base * T + i] = (uint8_t)((all_chosen[r * W + (t >> 5)] >> (t & 31)) & 1u);
        }
      }
      for (int i = id; i < rows_in * W; i += 128) chosen_bits[base * W + i] = all_chosen[i];
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem, tmem_cols);
  }
}

// The selected part of a plan: one block per (query tile, sample), a warp per
// key tile. Element bits of the tiles that stay partly live are written in
// both orientations, as the prepass does.
constexpr int kRefineWarps = 8;

__global__ void __launch_bounds__(kRefineWarps * 32) refine_plan_kernel(rt_tile_plan src, rt_tile_plan dst,
                                                                        const uint32_t* __restrict__ chosen_bits, int S,
                                                                        int group, int groups) {
  pdl_wait();  // the previous kernel on the stream has completed (launch_pdl)
  pdl_trigger();
  constexpr uint32_t kAll = 0xFFFFFFFFu;
  __shared__ uint32_t s_live[kMaxTiles / 32], s_full[kMaxTiles / 32];
  const int qt = blockIdx.x, b = blockIdx.y, T = src.tiles, W = src.words;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int w = threadIdx.x; w < W; w += blockDim.x) s_live[w] = s_full[w] = 0u;
  __syncthreads();
  const size_t row = (size_t)b * T + qt;
  // warps share out the words of tiles, or the tiles of a word where there are fewer words than warps
  const bool by_word = W >= kRefineWarps;
  int turn = 0;
  for (int word = by_word ? warp : 0; word < W; word += by_word ? kRefineWarps : 1) {
    uint32_t on[4], any_on = 0u;  // the tiles of this word that each of the lane's four queries keeps
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int i = qt * RT_TILE + 32 * m + lane;
      on[m] = i < S ? chosen_bits[((size_t)b * groups + i / group) * W + word] : 0u;
      any_on |= on[m];
    }
    uint32_t bits = src.live_bits[row * W + word] & __reduce_or_sync(kAll, any_on);
    const uint32_t full = src.full_bits[row * W + word];
    while (bits) {  // warp-uniform
      const int u = __ffs(bits) - 1, kt = word * 32 + u;
      bits &= bits - 1u;
      if (!by_word && (turn++ % kRefineWarps) != warp) continue;
      const bool was_full = (full >> u) & 1u;
      uint4 w[4];
      bool all = was_full;
      uint32_t any = 0u;
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const bool mine = (on[m] >> u) & 1u;
        w[m] = make_uint4(0u, 0u, 0u, 0u);
        if (mine)
          w[m] = was_full ? make_uint4(kAll, kAll, kAll, kAll)
                          : reinterpret_cast<const uint4*>(src.tile_masks)[(row * T + kt) * RT_TILE + 32 * m + lane];
        all = all && mine;
        any |= w[m].x | w[m].y | w[m].z | w[m].w;
      }
      if (!__any_sync(kAll, any != 0u)) continue;  // warp-uniform
      all = __all_sync(kAll, all);
      if (lane == 0) {
        atomicOr(&s_live[word], 1u << u);
        if (all) atomicOr(&s_full[word], 1u << u);
      }
      if (all) continue;  // warp-uniform
      uint4* dst_q = reinterpret_cast<uint4*>(dst.tile_masks) + (row * T + kt) * RT_TILE;
#pragma unroll
      for (int m = 0; m < 4; ++m) dst_q[32 * m + lane] = w[m];
      uint4* dst_k = reinterpret_cast<uint4*>(dst.tile_masks_t) + (((size_t)b * T + kt) * T + qt) * RT_TILE;
      auto put = [&](int kw, uint32_t a, uint32_t c, uint32_t d, uint32_t e) {
        dst_k[32 * kw + lane] = make_uint4(warp_transpose32(a, lane), warp_transpose32(c, lane),
                                           warp_transpose32(d, lane), warp_transpose32(e, lane));
      };
      put(0, w[0].x, w[1].x, w[2].x, w[3].x);
      put(1, w[0].y, w[1].y, w[2].y, w[3].y);
      put(2, w[0].z, w[1].z, w[2].z, w[3].z);
      put(3, w[0].w, w[1].w, w[2].w, w[3].w);
    }
  }
  __syncthreads();
  for (int w = threadIdx.x; w < W; w += blockDim.x) {
    dst.live_bits[row * W + w] = s_live[w];
    dst.full_bits[row * W + w] = s_full[w];
  }
}

struct Workspace {
  size_t kbar, knorm2, qbar, chosen, total;
};
Workspace workspace(int B, int H, int S, int Dh, int group) {
  const size_t T = (size_t)(S + RT_TILE - 1) / RT_TILE, G = (size_t)(S + group - 1) / group;
  Workspace w;
  w.kbar = 0;
  w.knorm2 = w.kbar + align_up(sizeof(uint16_t) * B * H * T * Dh);
  w.qbar = w.knorm2 + align_up(sizeof(float) * B * H * T);
  w.chosen = w.qbar + (group > 1 ? align_up(sizeof(uint16_t) * B * H * G * Dh) : 0);
  w.total = w.chosen + align_up(sizeof(uint32_t) * B * G * ((T + 31) / 32));
  return w;
}

template <int DH>
int launch(const uint16_t* q, const uint16_t* k, int B, int H, int S, const rt_tile_plan& plan, int keep, int group,
           const rt_tile_plan& out, uint8_t* selected, uint8_t* memory, cudaStream_t stream) {
  const Workspace ws = workspace(B, H, S, DH, group);
  const int T = plan.tiles, groups = (S + group - 1) / group;
  uint16_t* kbar = reinterpret_cast<uint16_t*>(memory + ws.kbar);
  uint16_t* qbar = reinterpret_cast<uint16_t*>(memory + ws.qbar);
  float* knorm2 = reinterpret_cast<float*>(memory + ws.knorm2);
  uint32_t* chosen = reinterpret_cast<uint32_t*>(memory + ws.chosen);
  const uint16_t* qrows = group > 1 ? qbar : q;
  const int span = std::max(32, group);
  const long long tasks = (long long)B * H * (T + (group > 1 ? (S + span - 1) / span : 0));
  if (tasks > (long long)kMeanWarps * INT32_MAX) return RT_ERR_INVALID_ARGUMENT;
  auto means = [&](auto kernel) {
    return launch_pdl("means_kernel launch", kernel, dim3((unsigned)((tasks + kMeanWarps - 1) / kMeanWarps)),
                      dim3(32 * kMeanWarps), 0, stream, q, k,
                      (long long)B * H, S, T, groups, qbar, kbar, knorm2);
  };
  const int st_means = group == 1    ? means(means_kernel<DH, 1>)
                       : group == 2  ? means(means_kernel<DH, 2>)
                       : group == 4  ? means(means_kernel<DH, 4>)
                       : group == 8  ? means(means_kernel<DH, 8>)
                       : group == 16 ? means(means_kernel<DH, 16>)
                       : group == 32 ? means(means_kernel<DH, 32>)
                       : group == 64 ? means(means_kernel<DH, 64>)
                                     : means(means_kernel<DH, 128>);
  if (st_means != RT_OK) return st_means;
  CUtensorMap tq, tk;
  if (make_qkv_tensor_map(&tq, qrows, B * H, groups, DH) != RT_OK || make_qkv_tensor_map(&tk, kbar, B * H, T, DH) != RT_OK)
    return RT_ERR_CUDA;  // detail recorded by make_qkv_tensor_map
  static bool configured[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    const cudaError_t e =
        cudaFuncSetAttribute(select_kernel<DH>, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024);
    if (e != cudaSuccess) return cuda_failure(e, "cudaFuncSetAttribute(select_kernel)");
    configured[dev] = true;
  }
  const int ctas = (groups + RT_TILE - 1) / RT_TILE;
  const int stages = sel_stages(T, SelCfg<DH>::kTileBytes, (long long)ctas * B);
  const SelLayout L = sel_layout(T, SelCfg<DH>::kTileBytes, stages);
  if (int st = launch_pdl("select_kernel launch", select_kernel<DH>, dim3(ctas, B),
                          dim3(kSelThreads), L.total, stream, tq, tk, qrows, kbar, knorm2, H, stages, group, groups, keep,
                          plan, selected, chosen))
    return st;
  if (int st = launch_pdl("refine_plan_kernel launch", refine_plan_kernel, dim3(T, B), dim3(kRefineWarps * 32), 0, stream,
                          plan, out, chosen, S, group, groups))
    return st;
  return launch_tile_lists(out, stream);
}

bool valid_shape(int32_t batch, int32_t heads, int32_t seq_len, int32_t group) {
  return batch >= 0 && heads >= 1 && seq_len >= 0 && seq_len <= 65536 && batch <= 65535 && heads <= 65535 &&
         (long long)batch * heads <= INT32_MAX &&
         group >= 1 && group <= RT_TILE && (group & (group - 1)) == 0;
}

}  // namespace select
}  // namespace rt

extern "C" size_t rt_select_tiles_workspace_bytes(int32_t batch, int32_t heads, int32_t seq_len, int32_t head_dim,
                                                  int32_t group) {
  if (!rt::select::valid_shape(batch, heads, seq_len, group) || head_dim <= 0) return 0;
  return rt::select::workspace(batch, heads, seq_len, head_dim, group).total;
}

extern "C" int rt_select_tiles(const uint16_t* q, const uint16_t* k, int32_t batch, int32_t heads, int32_t seq_len,
                               int32_t head_dim, const rt_tile_plan* plan, int32_t keep, int32_t group,
                               const rt_tile_plan* out, uint8_t* selected, void* workspace, size_t workspace_bytes,
                               void* stream) {
  using namespace rt;
  if (!select::valid_shape(batch, heads, seq_len, group) || keep < 0) return RT_ERR_INVALID_ARGUMENT;
  if (head_dim != 32 && head_dim != 64) return RT_ERR_UNSUPPORTED;
  if (batch == 0 || seq_len == 0) return RT_OK;
  if (!plan_matches(plan, batch, seq_len) || !plan_matches(out, batch, seq_len) || plan->live_bits == out->live_bits)
    return RT_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(k) || !q || !k || !selected || !aligned16(selected) || !workspace ||
      !aligned16(workspace))
    return RT_ERR_INVALID_ARGUMENT;
  const select::Workspace ws = select::workspace(batch, heads, seq_len, head_dim, group);
  if (workspace_bytes < ws.total) return RT_ERR_WORKSPACE;
  DeviceGuard guard(q);
  if (guard.status() != RT_OK) return guard.status();
  uint8_t* memory = static_cast<uint8_t*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return head_dim == 64
             ? select::launch<64>(q, k, batch, heads, seq_len, *plan, keep, group, *out, selected, memory, s)
             : select::launch<32>(q, k, batch, heads, seq_len, *plan, keep, group, *out, selected, memory, s);
}
