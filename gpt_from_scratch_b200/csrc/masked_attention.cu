// Masked attention, forward, and the kernel that makes its mask (head_dim 64 or 128, bf16; see masked_attention.cuh for
// the mask and the scores, masked_attention_bwd.cu for the gradients).
//
//   out_i = sum_j p_ij v_j,  p_ij = 2^(score_ij - lse_i) over the keys j that query i sees; a query that sees none: 0
//
// One pass over the keys with the running maximum and sum of the softmax; heads of q share the heads of k and v in groups.

#include "api.h"
#include "attention_tiles.cuh"
#include "masked_attention.cuh"

using namespace gfs;
using gfs_host::make_map;
using gfs_host::strides_ok;

namespace {

// ---------------------------------------------------------------------------
// The mask. One CTA per sequence: running maxima from the left (where a document starts, the last token that is not prefix)
// and running minima from the right (where it ends, the end of the prefix's run). Bound by latency, of the scans and of the few
// loads and stores of one CTA: us, 6 for 16 x 1024 tokens, 11 for 2 x 4096 under a window, 16 for 8192 with documents and prefixes.
// ---------------------------------------------------------------------------
constexpr int MASK_THREADS = 1024;

// Inclusive scan over the CTA's threads in order (RIGHT: from the last one), continued from `carry`; returns the inclusive
// value, `before` the exclusive one, and moves the carry on. tmp: 32 words.
template <bool RIGHT>
__device__ __forceinline__ int block_scan(int v, int& carry, int& before, int* tmp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto op = [](int a, int b) { return RIGHT ? min(a, b) : max(a, b); };
  constexpr int NONE = RIGHT ? 0x7fffffff : -1;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = RIGHT ? __shfl_down_sync(0xffffffffu, v, o) : __shfl_up_sync(0xffffffffu, v, o);
    if (RIGHT ? lane + o < 32 : lane >= o) v = op(v, u);
  }
  __syncthreads();
  if (lane == (RIGHT ? 0 : 31)) tmp[warp] = v;
  __syncthreads();
  int w = tmp[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = RIGHT ? __shfl_down_sync(0xffffffffu, w, o) : __shfl_up_sync(0xffffffffu, w, o);
    if (RIGHT ? lane + o < 32 : lane >= o) w = op(w, u);
  }
  const int src = RIGHT ? warp + 1 : warp - 1;
  int base = __shfl_sync(0xffffffffu, w, src & 31);
  base = op(src < 0 || src > 31 ? NONE : base, carry);
  const int near = RIGHT ? __shfl_down_sync(0xffffffffu, v, 1) : __shfl_up_sync(0xffffffffu, v, 1);
  before = lane == (RIGHT ? 31 : 0) ? base : op(base, near);
  carry = op(carry, __shfl_sync(0xffffffffu, w, RIGHT ? 0 : 31));
  return op(v, base);
}

struct MaskArgs {
  const void* ids;          // [B, S] or null
  const uint8_t* prefix;    // [B, S] or null
  int ids64, S, S_pad, window, causal;
  int *first, *last, *qfirst, *qlast, *padded, *positions;
  int4 *plan_q, *plan_k, *pairs;
};

// The tiles of a sequence in descending order of the rows between their ends (the work they are): kernels that start the
// heaviest first end together. Ranks by counting; a longer sequence than fits has enough tiles to even out by itself.
constexpr int MASK_SORT = 2048;
// ROWS: of a tile. `put` writes the entry of a tile at its rank.
template <int ROWS, typename Put>
__device__ __forceinline__ void sort_tiles(const int* lo, const int* hi, int S, int* weight, Put put) {
  const int n = (S + ROWS - 1) / ROWS;
  const bool sorted = n <= MASK_SORT;
  __syncthreads();
  for (int t = threadIdx.x; t < n; t += MASK_THREADS)
    if (sorted) weight[t] = hi[min((t + 1) * ROWS, S) - 1] - lo[t * ROWS];
  __syncthreads();
  for (int t = threadIdx.x; t < n; t += MASK_THREADS) {
    int rank = n - 1 - t;
    if (sorted) {
      rank = 0;
      const int mine = weight[t];
      for (int u = 0; u < n; ++u) rank += weight[u] > mine || (weight[u] == mine && u > t);
    }
    put(rank, t);
  }
}

// N: tokens per thread and step. A scan costs the same for 1,024 tokens as for 8,192 (1 -> 8 a thread, us: one sequence of 8192
// with a prefix 30 -> 16; up to 2,048 tokens one a thread has two steps at most, and needs no vectors).
template <int N>
__global__ void __launch_bounds__(MASK_THREADS) attention_mask_kernel(const MaskArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ int tmp[32];
  __shared__ int weight[MASK_SORT];
  const int b = blockIdx.x;
  const size_t row = static_cast<size_t>(b) * a.S;
  const size_t prow = static_cast<size_t>(b) * a.S_pad;
  const int chunks = (a.S_pad + MASK_THREADS * N - 1) / (MASK_THREADS * N);      // (i0 + N fits an int: S is checked)
  // what a thread's tokens hold: the first of a document, prefix, padding (bits)
  struct Tokens {
    unsigned starts, prefix, pad;
  };
  // (all loads of a thread are issued before the first is looked at)
  auto load = [&](int i0) {
    Tokens t = {0u, 0u, 0u};
    long long ids[N + 1] = {};
    uint8_t pre[N] = {};
    // whole vectors where rows of ids (prefix marks) begin at one: single elements of 1,024 threads, N apart, take N times the cycles
    const bool wide = N % 4 == 0 && !a.ids64 && (a.S & 3) == 0 && (reinterpret_cast<uintptr_t>(a.ids) & 15) == 0 && i0 + N <= a.S;
    const bool wide_p = N == 8 && (a.S & 7) == 0 && (reinterpret_cast<uintptr_t>(a.prefix) & 7) == 0 && i0 + N <= a.S;
    if (a.ids != nullptr && wide) {
      const int* from = static_cast<const int*>(a.ids) + row + i0;
      if (i0 > 0) ids[0] = from[-1];
#pragma unroll
      for (int e = 0; e + 3 < N; e += 4) {
        const int4 v = *reinterpret_cast<const int4*>(from + e);
        ids[e + 1] = v.x;
        ids[e + 2] = v.y;
        ids[e + 3] = v.z;
        ids[e + 4] = v.w;
      }
    } else if (a.ids != nullptr && a.ids64) {
#pragma unroll
      for (int e = -1; e < N; ++e)
        if (i0 + e >= 0 && i0 + e < a.S) ids[e + 1] = static_cast<const long long*>(a.ids)[row + i0 + e];
    } else if (a.ids != nullptr) {
#pragma unroll
      for (int e = -1; e < N; ++e)
        if (i0 + e >= 0 && i0 + e < a.S) ids[e + 1] = static_cast<const int*>(a.ids)[row + i0 + e];
    }
    if (a.prefix != nullptr && wide_p) {
      const uint2 v = *reinterpret_cast<const uint2*>(a.prefix + row + i0);
#pragma unroll
      for (int e = 0; e < N; ++e) pre[e] = static_cast<uint8_t>((e < 4 ? v.x : v.y) >> (8 * (e & 3)));
    } else if (a.prefix != nullptr) {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i0 + e < a.S) pre[e] = a.prefix[row + i0 + e];
    }
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const bool in = i0 + e < a.S;
      if (in && (i0 + e == 0 || ids[e + 1] != ids[e])) t.starts |= 1u << e;
      if (in && pre[e] != 0) t.prefix |= 1u << e;
      if (in && ids[e + 1] < 0) t.pad |= 1u << e;
    }
    return t;
  };
  // first stop at or behind a thread's first token, S where there is none
  auto first_of = [&](unsigned stops, int i0) { return stops ? i0 + __ffs(stops) - 1 : 0x7fffffff; };
  auto last_of = [&](unsigned stops, int i0) { return stops ? i0 + 31 - __clz(stops) : -1; };
  constexpr unsigned ALL = N == 32 ? 0xffffffffu : (1u << N) - 1u;
  // N numbers of a thread from or to a row of [B, S_pad]
  auto put = [&](int* to, int i0, const int (&v)[N]) {
    if (i0 >= a.S_pad) return;
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int e = 0; e < N; e += 4) *reinterpret_cast<int4*>(to + prow + i0 + e) = make_int4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) to[prow + i0 + e] = v[e];
    }
  };
  auto get = [&](const int* from, int i0, int (&v)[N]) {
    if (i0 >= a.S_pad) return;
    if constexpr (N % 4 == 0) {
#pragma unroll
      for (int e = 0; e < N; e += 4) {
        const int4 x = *reinterpret_cast<const int4*>(from + prow + i0 + e);
        v[e] = x.x;
        v[e + 1] = x.y;
        v[e + 2] = x.z;
        v[e + 3] = x.w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) v[e] = from[prow + i0 + e];
    }
  };
  // from the right: the end of the document, and the first token after this one that is not of the prefix's run. Of one chunk they stay
  // in registers, of several they wait in qlast and last.
  int carry = a.S, carry2 = a.S, any = 0;
  int ends[N], reaches[N] = {};
  auto from_right = [&](int i0, const Tokens& t) {
    const unsigned live = i0 >= a.S ? 0u : (a.S - i0 >= N ? ALL : (1u << (a.S - i0)) - 1u);
    const unsigned stops = t.starts | (~t.prefix & live);
    int end, reach = 0;
    block_scan<true>(first_of(t.starts, i0), carry, end, tmp);
    if (a.prefix != nullptr) block_scan<true>(first_of(stops, i0), carry2, reach, tmp);
#pragma unroll
    for (int e = N - 1; e >= 0; --e) {
      ends[e] = end;
      reaches[e] = reach;
      if ((t.starts >> e) & 1u) end = i0 + e;
      if ((stops >> e) & 1u) reach = i0 + e;
    }
  };
  auto from_left = [&](int i0, const Tokens& t) {
    int start, plain = -1;       // of the tokens before this thread's: the last start, the last token that is not prefix
    block_scan<false>(last_of(t.starts, i0), carry, start, tmp);
    if (a.prefix != nullptr) {
      const unsigned live = i0 >= a.S ? 0u : (a.S - i0 >= N ? ALL : (1u << (a.S - i0)) - 1u);
      block_scan<false>(last_of(~t.prefix & live, i0), carry2, plain, tmp);
    }
    if (t.pad != 0u) any = 1;
    int out[4][N], place[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int i = i0 + e;
      if ((t.starts >> e) & 1u) start = i;
      const bool p = (t.prefix >> e) & 1u;
      if (!p) plain = i;
      const bool lead = p && plain < start;
      int first = start, last = a.causal ? (lead ? reaches[e] : i + 1) : ends[e];
      int qfirst = a.causal && !lead ? i : start, qlast = ends[e];
      if (a.window > 0) {
        first = max(first, i - a.window + 1);
        qlast = min(qlast, i + a.window);
      }
      if ((t.pad >> e) & 1u) first = last = qfirst = qlast = i;      // wherever it does not widen a tile's range
      if (i >= a.S) first = last = qfirst = qlast = a.S;
      out[0][e] = first;
      out[1][e] = last;
      out[2][e] = qfirst;
      out[3][e] = qlast;
      place[e] = i - start;
    }
    put(a.first, i0, out[0]);
    put(a.last, i0, out[1]);
    put(a.qfirst, i0, out[2]);
    put(a.qlast, i0, out[3]);
    if (N % 4 == 0 && (a.S & 3) == 0 && i0 + N <= a.S) {
#pragma unroll
      for (int e = 0; e + 3 < N; e += 4)
        *reinterpret_cast<int4*>(a.positions + row + i0 + e) = make_int4(place[e], place[e + 1], place[e + 2], place[e + 3]);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (i0 + e < a.S) a.positions[row + i0 + e] = place[e];
    }
  };
  if (chunks == 1) {
    const int i0 = threadIdx.x * N;
    const Tokens t = load(i0);
    from_right(i0, t);
    carry = carry2 = -1;
    from_left(i0, t);
  } else {
    for (int c = chunks - 1; c >= 0; --c) {
      const int i0 = (c * MASK_THREADS + threadIdx.x) * N;
      from_right(i0, load(i0));
      put(a.qlast, i0, ends);
      put(a.last, i0, reaches);
    }
    carry = carry2 = -1;
    for (int c = 0; c < chunks; ++c) {
      const int i0 = (c * MASK_THREADS + threadIdx.x) * N;
      get(a.qlast, i0, ends);
      get(a.last, i0, reaches);
      from_left(i0, load(i0));
    }
  }
  any = __syncthreads_or(any);
  if (threadIdx.x == 0) a.padded[b] = any;
  const size_t tiles = static_cast<size_t>(b) * (a.S_pad / 128);
  const int *first = a.first + prow, *last = a.last + prow, *qfirst = a.qfirst + prow, *qlast = a.qlast + prow;
  auto end = [&](const int* hi, int t) { return hi[min(t * 128 + 127, a.S - 1)]; };
  sort_tiles<128>(first, last, a.S, weight, [&](int rank, int t) {
    a.plan_q[tiles + rank] = make_int4(t, first[t * 128], end(last, t), any);
  });
  sort_tiles<128>(qfirst, qlast, a.S, weight, [&](int rank, int t) {
    a.plan_k[tiles + rank] = make_int4(t, qfirst[t * 128], end(qlast, t), any);
  });
  int4* const pairs = a.pairs + static_cast<size_t>(b) * ((a.S_pad / 128 + 1) / 2) * 2;
  sort_tiles<256>(first, last, a.S, weight, [&](int rank, int t) {
    const bool two = t * 256 + 128 < a.S;
    const int la = first[t * 256], ha = end(last, 2 * t);
    const int lb = two ? first[t * 256 + 128] : 0, hb = two ? end(last, 2 * t + 1) : 0;
    int a0 = la >> 6, a1 = (ha + 63) >> 6, b0 = lb >> 6, b1 = (hb + 63) >> 6;
    // A row's range holds its own place or, of padding, ends there: only a tile of one row that is padding may have no block, the
    // last of a sequence. It gets one, which is masked whole; behind another tile that one's last, so that no gap comes between them.
    if (a1 <= a0) a1 = a0 + 1;
    if (two && b1 <= b0) {
      b0 = a1 - 1;
      b1 = a1;
    }
    pairs[2 * rank] = make_int4(t, a0, a1, b0);
    pairs[2 * rank + 1] = make_int4(b1, any, 0, 0);
  });
}

// ---------------------------------------------------------------------------
// Forward. An item is a CTA of the grid; those that run (one per SM) claim further ones, the widest first. It is two tiles
// of 128 queries that share the loads of their keys: two heads of a group at the same queries (groups of an even number), else
// neighbouring tiles of a head. Blocks of 64 keys, a thread per query row; scores double buffered in tensor memory, P over the
// scores that it was made from, O beside them (2 x 2 x 64 + 2 x D columns).
//
// Bound by the softmax warps, two per scheduler: their exponentials keep the special function unit (16 a clock and SM) busy for
// 45 % of the time, with a cap (2.25 operations a score) for 75 %; the rest is the length of their chains. us, and
// products at a share of the measured tensor rate: 16 heads (4 of k) of 8192 tokens, head_dim 128, documents with prefixes 91
// (0.41); 64 heads (16 of k) of 4096 under a window of 1024, capped 208 (0.35); 16 x 12 heads of 1024 tokens of head_dim 64 in
// documents of 200 tokens, where an item is five blocks and every fourth score is needed, 48 (100 MB: 15 at copy speed). What the backward
// needs is another half of the output: 5 to 8 more for the first and the last.
//
// What led here, us for the three: a CTA per tile, two per SM, blocks of 128 keys, each with its own loads 131, 263, 58 (a block's
// chain took 8,000 cycles, most of it its loads' latency at half of L2's rate); two tiles to a CTA and one warp that polls both
// tiles' events 168, 299, 68 (1,100 to 1,700 cycles late); an MMA warp per tile 155, 285, 63 (both tiles keep step, so
// both wait for their MMAs together); scores double buffered in blocks of 64: 100, 217, 58; items claimed, not dealt: 91, 208, 48. Slower
// than this: two threads to a row (sixteen softmax warps: a cap -6 %, the others +5 to 10 %), the next block's scores loaded ahead of
// this one's exponentials (+30 %), exponentials by polynomials on the FMA pipe for a half of them (+6 %), a delay to set the tiles out of step (0), four more warps
// that put the outputs out (+4 to 9 %), blocks classed by 32 rows and 32 keys, with no exponentials where nothing is seen (0 to +5 %).
// ---------------------------------------------------------------------------
struct MaskedFwdParams {
  float* lse;                  // [B, nh, S_pad], base 2; +inf for rows that see nothing; or null
  uint8_t* rest;               // with lse: [B, nh, S_pad, D], what O's rounding leaves out (bf16_rest)
  int S, S_pad, B, nh, group;
  int head_pairs;
  ScoreArgs score;
  MaskView mask;
  uint32_t* status;
};

constexpr int MFWD_FIRST_SW = 4;                    // warps 0: TMA, 1 and 2: the MMAs of a tile, 3: items and their queries; then the softmax warps
constexpr int MFWD_SW = 8;                          // four per tile, a row per thread
constexpr int MFWD_THREADS = 32 * (MFWD_FIRST_SW + MFWD_SW);
// 384 threads x 168 at the launch = 128 x 72 + 256 x 216: a softmax thread holds the scores of two blocks of its row.
constexpr int MFWD_REGS_IO = 72, MFWD_REGS_SOFTMAX = 216;
// A work item, as warp 3 puts it into shared memory when the one before has been taken: nobody else divides or waits for the plans.
struct alignas(16) FwdItem {
  uint4 claim;                 // what claim_cta answered
  int more;                    // 0: there are no further items
  int b, padded;
  int h[2], row[2];            // heads and first query rows of the two tiles
  int j0[2], j1[2];            // their blocks of 64 keys; j0 == j1: there is no second tile
  int lo_max[2], hi_min[2];    // what every row of a tile sees
  float slope2[2];             // - slope log2(e)
  int lo[2][128], hi[2][128];  // what the rows see
};
template <int D>
struct MFwdShape {
  static constexpr int DB = D / 64;
  static constexpr int Q_TILE = DB * 16384, KV_TILE = DB * 8192;    // 128 queries, 64 keys
  static constexpr int KS = D == 64 ? 8 : 4;        // stages of K and V
  static constexpr int STAGING = MFWD_SW * 4096;    // a warp's results on their way out: 32 rows of 64 columns
  static constexpr int SMEM = 2 * Q_TILE + 2 * KS * KV_TILE + STAGING + sizeof(FwdItem) + 512;
};
// Scores: as they are, capped with a bound that the running maximum may be left out for, capped.
enum Scores { PLAIN = 0, BOUNDED = 1, CAPPED = 2 };
// Up to this cap2 (caps up to 50) no maximum is needed: probabilities lie within 2^-73 and 2^73. What fp32 has beyond that is left to
// the values: sums over 2^20 keys stay below 2^128 for magnitudes up to 2^30, products above 2^-126 for those from 2^-40 on, and that is
// the range that masked_attention documents. With the maximum, us: 64 heads of 4096 under a window, cap 50, 221 -> 248.
constexpr float BOUNDED_CAP2 = 73.f;

template <int D, int SCORES, bool DIST>
__global__ void __launch_bounds__(MFWD_THREADS, 1)
masked_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                  const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to, const MaskedFwdParams p,
                  int n_levels) {
  using Shape = MFwdShape<D>;
  constexpr int DB = Shape::DB, Q_TILE = Shape::Q_TILE, KV_TILE = Shape::KV_TILE, KS = Shape::KS;
  constexpr uint32_t O_COL = 256;            // scores at [tile][buffer][64] before that; P takes the columns of its scores
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* Qs = smem_raw;                    // [2] tiles
  uint8_t* Ks = Qs + 2 * Q_TILE;             // [KS]
  uint8_t* Vs = Ks + KS * KV_TILE;           // [KS]
  uint8_t* staging = Vs + KS * KV_TILE;
  FwdItem& item = *reinterpret_cast<FwdItem*>(staging + Shape::STAGING);
  uint64_t* bars = reinterpret_cast<uint64_t*>(&item + 1);
  uint64_t* q_full = bars;                   // [tile]
  uint64_t* q_empty = bars + 2;
  uint64_t* k_full = bars + 4;               // [KS]
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;
  uint64_t* v_empty = v_full + KS;
  uint64_t* s_full = v_empty + KS;           // [tile][buffer]
  uint64_t* p_full = s_full + 4;
  uint64_t* o_full = p_full + 4;             // P V of the buffer is done
  uint64_t* o_empty = o_full + 4;            // [tile]
  uint64_t* i_full = o_empty + 2;
  uint64_t* i_empty = i_full + 1;
  uint64_t* i_claim = i_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(i_full + 3);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0) record_status(p.status, STATUS_BAD_ARGUMENT, 0x5a21u);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4; ++i) mbar_init(&bars[i], 1);
    for (int i = 0; i < KS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 2);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 2);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], MFWD_SW / 2);
      mbar_init(&o_full[i], 1);
    }
    for (int x = 0; x < 2; ++x) mbar_init(&o_empty[x], MFWD_SW / 2);
    mbar_init(i_full, 32);
    mbar_init(i_empty, 3 + MFWD_SW);
    mbar_init(i_claim, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
    tma_prefetch_desc(&to);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();       // set-up above may overlap the tail of the preceding kernel (programmatic launch)
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  WaitCtx wctx{abort_flag, p.status, GFS_WAIT_LIMIT_NS};

  // All barrier parities run on counters that continue across items. What a warp wants of the it-th item it copies out of the
  // slot, then it releases it.
  auto take_item = [&](int it) {        // false, for the whole warp: there are no more, or a wait has given up
    mbar_wait(i_full, it & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
    return !__any_sync(0xffffffffu, item.more == 0 || *abort_flag != 0);
  };
  auto release_item = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(i_empty);
  };
  struct Blocks {
    int u0, u1;      // all blocks of the item
  };
  auto blocks_of = [](const FwdItem& i) {
    return Blocks{i.j0[1] < i.j1[1] ? min(i.j0[0], i.j0[1]) : i.j0[0], max(i.j1[0], i.j1[1])};
  };

  if (warp < MFWD_FIRST_SW) {
    setmaxnreg_dec<MFWD_REGS_IO>();
    if (warp == 0) {
      int g = 0;      // key blocks loaded so far (ring position)
      for (int it = 0; take_item(it); ++it) {
        const int bb = item.b, kvh = item.h[0] / p.group;
        const Blocks u = blocks_of(item);
        if (lane == 0) {
          for (int j = u.u0; j < u.u1; ++j, ++g) {
            const int st = g % KS;
            const uint32_t par = ((g / KS) & 1) ^ 1u;
            mbar_wait(&k_empty[st], par, wctx, STATUS_TIMEOUT_PIPE_EMPTY);
            mbar_arrive_expect_tx(&k_full[st], KV_TILE);
#pragma unroll
            for (int db = 0; db < DB; ++db)
              tma_load_4d(Ks + st * KV_TILE + db * 8192, &tk, &k_full[st], db * 64, j * 64, kvh, bb);
            mbar_wait(&v_empty[st], par, wctx, STATUS_TIMEOUT_PIPE_EMPTY);
            mbar_arrive_expect_tx(&v_full[st], KV_TILE);
#pragma unroll
            for (int db = 0; db < DB; ++db)
              tma_load_4d(Vs + st * KV_TILE + db * 8192, &tv, &v_full[st], db * 64, j * 64, kvh, bb);
          }
        }
        // Only now may the next item be claimed: one that is claimed early waits here while other SMs have run out of work (us:
        // 64 heads of 4096 tokens under a window 224 -> 234 with the release at the start).
        release_item();
      }
      if (lane == 0) settle_copies(wctx);
    } else if (warp <= 2) {
      // The MMAs of tile x (whole warp, converged: the MMA / commit helpers elect the issuing lane). Each tile has a warp of its
      // own, which waits for nothing but its tile: one warp that polled the events of both came 1,100 to 1,700 cycles late. It
      // walks all blocks of the item; those that only the other tile sees are handed on.
      // Scores are double buffered: a block's are made while the softmax is at the block before, so neither waits for the other's
      // latency, nor do the two tiles meet in the same phase.
      constexpr uint32_t idesc_s = umma_idesc_bf16(128, 64, 0, 0);
      constexpr uint32_t idesc_o = umma_idesc_bf16(128, D, 0, 1);
      const int x = warp - 1;
      const uint32_t s_tmem = tmem_base + x * 128, o_tmem = tmem_base + O_COL + x * D;
      const uint32_t q_addr = smem_u32(Qs + x * Q_TILE);
      int g0 = 0;               // ring position of this item's first key block
      int cx = 0;               // this tile's blocks in earlier items (barrier phases)
      int had = 0;              // items in which it had blocks (phase of o_empty)
      for (int it = 0; take_item(it); ++it) {
        const int u0 = blocks_of(item).u0, u1 = blocks_of(item).u1;
        const int j0 = item.j0[x], j1 = item.j1[x];
        const bool padded = item.padded != 0;
        const int *first = p.mask.first + static_cast<size_t>(item.b) * p.S_pad, *last = p.mask.last + static_cast<size_t>(item.b) * p.S_pad;
        release_item();
        mbar_wait(&q_full[x], it & 1, wctx, STATUS_TIMEOUT_PIPE_FULL);
        auto scores = [&](int j) {
          const int g = g0 + j - u0, st = g % KS, n = cx + j - j0, buf = n & 1;
          mbar_wait(&k_full[st], (g / KS) & 1, wctx, STATUS_TIMEOUT_PIPE_FULL);
          if (j < j0 || j >= j1) {
            if (lane == 0) mbar_arrive(&k_empty[st]);
            return;
          }
          if (padded) zero_padding(Ks + st * KV_TILE, 64, DB, 8192, first + j * 64, last + j * 64, lane);
          if (n >= 2) mbar_wait(&o_full[2 * x + buf], ((n - 2) >> 1) & 1, wctx, STATUS_TIMEOUT_TMEM_FULL);   // its P has been read
          tc_fence_after();
          mma_kk<D / 16>(s_tmem + buf * 64, q_addr, 16384, smem_u32(Ks + st * KV_TILE), 8192, idesc_s, false);
          umma_commit_e(&s_full[2 * x + buf]);
          umma_commit_e(&k_empty[st]);
          if (j + 1 == j1) umma_commit_e(&q_empty[x]);      // the tile's last: the next item's queries may come
        };
        if (j1 <= j0) umma_commit_e(&q_empty[x]);
        auto values = [&](int j) {
          const int g = g0 + j - u0, st = g % KS, n = cx + j - j0, buf = n & 1;
          mbar_wait(&v_full[st], (g / KS) & 1, wctx, STATUS_TIMEOUT_PIPE_FULL);
          if (j < j0 || j >= j1) {
            if (lane == 0) mbar_arrive(&v_empty[st]);
            return;
          }
          if (padded) zero_padding(Vs + st * KV_TILE, 64, DB, 8192, first + j * 64, last + j * 64, lane);
          // the accumulator is overwritten once per item: the previous item's result has been read out of it
          if (j == j0) mbar_wait(&o_empty[x], (had & 1) ^ 1u, wctx, STATUS_TIMEOUT_SOFTMAX);
          mbar_wait(&p_full[2 * x + buf], (n >> 1) & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
          tc_fence_after();
          mma_tmn<4>(o_tmem, s_tmem + buf * 64, smem_u32(Vs + st * KV_TILE), 8192, idesc_o, j > j0);
          umma_commit_e(&o_full[2 * x + buf]);
          umma_commit_e(&v_empty[st]);
        };
        scores(u0);
        if (u0 + 1 < u1) scores(u0 + 1);
        for (int j = u0; j < u1; ++j) {
          values(j);
          if (j + 2 < u1) scores(j + 2);
        }
        g0 += u1 - u0;
        cx += j1 - j0;
        had += j1 > j0;
      }
    } else {
      const int heads = p.head_pairs ? p.nh / 2 : p.nh;
      const int BH = p.B * heads;
      for (int it = 0;; ++it) {
        mbar_wait(i_empty, (it & 1) ^ 1u, wctx, STATUS_TIMEOUT_PIPE_EMPTY);
        int w = blockIdx.x;
        bool more = true;
        if (it > 0) {
          if (lane == 0) claim_cta(&item.claim, i_claim);
          more = mbar_wait(i_claim, (it - 1) & 1, wctx, STATUS_TIMEOUT_PIPE_FULL) && claimed_cta(&item.claim, w);
          more = __all_sync(0xffffffffu, more);
          fence_proxy_async_smem();      // the next answer comes after everybody has read this one
        }
        if (more) {
          const int bh = w % BH, b = bh / heads, h = bh % heads;
          const size_t at = static_cast<size_t>(b) * n_levels + w / BH;
          int row[2], j0[2], j1[2], hh[2], padded;
          if (p.head_pairs) {
            const int4 e = p.mask.plan_q[at];
            hh[0] = 2 * h;
            hh[1] = 2 * h + 1;
            row[0] = row[1] = e.x * 128;
            j0[0] = j0[1] = e.y >> 6;
            j1[0] = j1[1] = max((e.z + 63) >> 6, j0[0] + 1);
            padded = e.w;
          } else {
            const int4 e = p.mask.pairs[2 * at], f = p.mask.pairs[2 * at + 1];
            hh[0] = hh[1] = h;
            row[0] = e.x * 256;
            row[1] = row[0] + 128;
            j0[0] = e.y;
            j1[0] = e.z;
            j0[1] = e.w;
            j1[1] = f.x;
            padded = f.y;
          }
          const int *first = p.mask.first + static_cast<size_t>(b) * p.S_pad, *last = p.mask.last + static_cast<size_t>(b) * p.S_pad;
          int lo[2][4], hi[2][4];
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int at_row = min(row[x], p.S_pad - 128) + 32 * i + lane;     // (no second tile: rows that nobody uses)
              lo[x][i] = first[at_row];
              hi[x][i] = last[at_row];
            }
          if (lane < 2) {
            const int x = lane, a = min(x == 0 ? row[0] : row[1], p.S_pad - 128);
            item.h[x] = x == 0 ? hh[0] : hh[1];
            item.row[x] = x == 0 ? row[0] : row[1];
            item.j0[x] = x == 0 ? j0[0] : j0[1];
            item.j1[x] = x == 0 ? j1[0] : j1[1];
            item.lo_max[x] = first[min(a + 127, p.S - 1)];
            item.hi_min[x] = last[a];
            item.slope2[x] = DIST ? -p.score.slopes[x == 0 ? hh[0] : hh[1]] * LOG2E_F : 0.f;
            item.b = b;
            item.padded = padded;
          }
#pragma unroll
          for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              item.lo[x][32 * i + lane] = lo[x][i];
              item.hi[x][32 * i + lane] = hi[x][i];
            }
        }
        if (lane == 0) item.more = more;
        __syncwarp();
        mbar_arrive(i_full);
        if (!more || __any_sync(0xffffffffu, *abort_flag != 0)) break;
        if (lane == 0) {
          for (int x = 0; x < 2; ++x) {        // (rows past S: zeros)
            mbar_wait(&q_empty[x], (it & 1) ^ 1u, wctx, STATUS_TIMEOUT_PIPE_EMPTY);  // the tile's score MMAs of the previous item are done
            mbar_arrive_expect_tx(&q_full[x], Q_TILE);
#pragma unroll
            for (int db = 0; db < DB; ++db)
              tma_load_4d(Qs + x * Q_TILE + db * 16384, &tq, &q_full[x], db * 64, item.row[x], item.h[x], item.b);
          }
        }
        __syncwarp();
      }
      if (lane == 0) settle_copies(wctx);
    }
  } else {
    setmaxnreg_inc<MFWD_REGS_SOFTMAX>();
    const int x = (warp - MFWD_FIRST_SW) >> 2;         // query tile of this warp
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_base + x * 128;
    const uint32_t o_addr = tmem_base + lane_base + O_COL + x * D;
    uint8_t* stage = staging + (warp - MFWD_FIRST_SW) * 4096;
    constexpr bool MAXED = SCORES != BOUNDED;
    const float sl2 = p.score.sl2, cap2 = p.score.cap2;
    const float k = SCORES != PLAIN || DIST ? 1.f : sl2;    // what turns the numbers in the registers into exponents
    const uint64_t k_2 = pack_f32x2(k, k), sl2_2 = pack_f32x2(sl2, sl2);
    const uint64_t cap_2 = pack_f32x2(cap2, cap2), m2cap_2 = pack_f32x2(-2.f * cap2, -2.f * cap2);
    struct Rows {
      int lo, hi, lo_max, hi_min;
      float slope2;
    };
    // bits [lo - col, hi - col) of 32: what the row sees
    auto live_bits = [](const Rows& q, int col) {
      const int a = max(q.lo - col, 0), z = q.hi - col;
      return (z >= 32 ? 0xffffffffu : (z <= 0 ? 0u : (1u << z) - 1u)) & (a >= 32 ? 0u : 0xffffffffu << a);
    };
    // 32 scores of a row from column col on -> exponents (plain ones: still to be scaled), dead ones -inf
    // (bounded ones: dead probabilities become 0 afterwards)
    auto transform = [&](uint32_t (&v)[32], int col, const Rows& q, int row, bool whole) {
      if (SCORES != PLAIN || DIST) {
        const uint64_t slope_2 = pack_f32x2(q.slope2, q.slope2);
        const float dist0 = static_cast<float>(row - col);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          uint64_t y[2] = {pack_u32x2(v[e], v[e + 1]), pack_u32x2(v[e + 2], v[e + 3])};
          if (SCORES != PLAIN) {
            uint64_t r0, r1;
            sigmoids(y[0], y[1], sl2_2, r0, r1);
            y[0] = fma_f32x2(r0, m2cap_2, cap_2);
            y[1] = fma_f32x2(r1, m2cap_2, cap_2);
          } else {
            y[0] = mul_f32x2(y[0], sl2_2);
            y[1] = mul_f32x2(y[1], sl2_2);
          }
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (DIST)
              y[u] = fma_f32x2(pack_f32x2(fabsf(dist0 - static_cast<float>(e + 2 * u)), fabsf(dist0 - static_cast<float>(e + 2 * u + 1))),
                               slope_2, y[u]);
            const float2 f = unpack_f32x2(y[u]);
            v[e + 2 * u] = __float_as_uint(f.x);
            v[e + 2 * u + 1] = __float_as_uint(f.y);
          }
        }
      }
      if (MAXED && !whole) {
        const uint32_t live = live_bits(q, col);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = (live >> e) & 1u ? v[e] : 0xff800000u;
      }
    };
    int cdone = 0;  // blocks of this tile processed in earlier items
    for (int it = 0; take_item(it); ++it) {
      const Rows q{item.lo[x][r], item.hi[x][r], item.lo_max[x], item.hi_min[x], item.slope2[x]};
      const int j0 = item.j0[x], j1 = item.j1[x], row = item.row[x] + r, b = item.b, h = item.h[x];
      release_item();
      float m = MAXED ? -INFINITY : 0.f;
      uint64_t l2 = 0, t2 = 0;                  // sums of the probabilities, as they are and as rounded to bf16
      // 32 exponents -> probabilities, packed, and their sums. They are rounded to bf16, v's type, since a product takes one type of 16 bits
      // (and has to be bf16: they go up to 2^73): up to 2^-8 of each, 1.7e-3 in the mean of squares. As two parts, P V would be made twice.
      auto probabilities = [&](const uint32_t (&v)[32], uint32_t (&packed)[16], uint64_t moff2, uint32_t live) {
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const uint64_t y2 = MAXED ? fma_f32x2(pack_u32x2(v[e], v[e + 1]), k_2, moff2) : pack_u32x2(v[e], v[e + 1]);
          const float2 y = unpack_f32x2(y2);
          float2 pr = make_float2(fast_exp2(y.x), fast_exp2(y.y));
          if (!MAXED && live != 0xffffffffu) {
            pr.x = (live >> e) & 1u ? pr.x : 0.f;
            pr.y = (live >> (e + 1)) & 1u ? pr.y : 0.f;
          }
          const uint32_t w = pack_bf16x2(pr.x, pr.y);
          l2 = add_f32x2(l2, pack_f32x2(pr.x, pr.y));
          t2 = add_f32x2(t2, pack_u32x2(w << 16, w & 0xffff0000u));
          packed[e >> 1] = w;
        }
      };
      for (int j = j0; j < j1; ++j) {
        const int c = cdone + j - j0, buf = c & 1;
        const bool whole = j * 64 >= q.lo_max && j * 64 + 64 <= q.hi_min;   // every row sees every key of the block
        const uint32_t at = s_addr + buf * 64;
        mbar_wait(&s_full[2 * x + buf], (c >> 1) & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
        tc_fence_after();
        uint32_t v0[32], v1[32], pk[16];
        tmem_ld_32x32(at, v0);
        tmem_ld_32x32(at + 32, v1);
        tmem_ld_wait_for(v0);
        tmem_ld_wait_for(v1);
        transform(v0, j * 64, q, row, whole);
        transform(v1, j * 64 + 32, q, row, whole);
        uint64_t moff2 = 0;
        if (MAXED) {
          float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            mx0 = fmax3(mx0, __uint_as_float(v0[e]), __uint_as_float(v0[e + 1]));
            mx1 = fmax3(mx1, __uint_as_float(v0[e + 2]), __uint_as_float(v0[e + 3]));
            mx2 = fmax3(mx2, __uint_as_float(v1[e]), __uint_as_float(v1[e + 1]));
            mx3 = fmax3(mx3, __uint_as_float(v1[e + 2]), __uint_as_float(v1[e + 3]));
          }
          const float m_new = fmax3(m, fmaxf(mx0, mx1), fmaxf(mx2, mx3));
          // The running maximum is raised only when it grew by more than 2^8 (or was still -inf): raising it rescales the
          // accumulator in tensor memory, which after the first blocks is rare.
          bool grow = false;
          float alpha = 1.f;
          if (m_new > m && (m == -INFINITY || (m_new - m) * k > 8.f)) {
            grow = true;
            alpha = (m == -INFINITY) ? 0.f : fast_exp2((m - m_new) * k);
          }
          if (j > j0 && __any_sync(0xffffffffu, grow && m != -INFINITY)) {
            // this warp's 32 accumulator rows (warp-collective accesses; rows whose maximum stays get factor 1, and so do those
            // that saw nothing yet: they hold zeros). P V of the previous block must be done.
            mbar_wait(&o_full[2 * x + (buf ^ 1)], ((c - 1) >> 1) & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
            tc_fence_after();
            const float a = grow && m != -INFINITY ? alpha : 1.f;
#pragma unroll 1
            for (int cc = 0; cc < D; cc += 32) {
              uint32_t wv[32];
              tmem_ld_32x32(o_addr + cc, wv);
              tmem_ld_wait_for(wv);
              uint32_t lo16[16], hi16[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                lo16[e] = __float_as_uint(__uint_as_float(wv[e]) * a);
                hi16[e] = __float_as_uint(__uint_as_float(wv[16 + e]) * a);
              }
              tmem_st_32x16(o_addr + cc, lo16);
              tmem_st_32x16(o_addr + cc + 16, hi16);
            }
            tmem_st_wait();
          }
          if (grow) {
            l2 = mul_f32x2(l2, pack_f32x2(alpha, alpha));
            t2 = mul_f32x2(t2, pack_f32x2(alpha, alpha));
            m = m_new;
          }
          const float moff = ((m == -INFINITY) ? 0.f : m) * k;
          moff2 = pack_f32x2(-moff, -moff);
        }
        // the probabilities go where the scores were: all of those are in registers
        probabilities(v0, pk, moff2, MAXED || whole ? 0xffffffffu : live_bits(q, j * 64));
        tmem_st_32x16(at, pk);
        probabilities(v1, pk, moff2, MAXED || whole ? 0xffffffffu : live_bits(q, j * 64 + 32));
        tmem_st_32x16(at + 16, pk);
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[2 * x + buf]);
      }
      if (j1 > j0) {
        // The output is normalised by the sum of the probabilities that it was made from, the rounded ones: a row that sees
        // little but one key has that key's value exactly. The backward recomputes them unrounded and gets the other sum.
        const float2 lp = unpack_f32x2(l2), tp = unpack_f32x2(t2);
        const float l = lp.x + lp.y, t = tp.x + tp.y;
        const bool seen = q.lo < q.hi;
        const float inv = seen && t > 0.f ? 1.f / t : 0.f;
        const int c_last = cdone + j1 - j0 - 1;
        mbar_wait(&o_full[2 * x + (c_last & 1)], (c_last >> 1) & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
        tc_fence_after();
        // Rows leave by TMA: a warp that stores them itself waits for its SM's share of the write rate (whole calls, us: 64 heads of
        // 4096 under a window 225 -> 219, 8192 tokens with prefixes 373 -> 368; what the backward needs is faster stored directly, 174 -> 170 for documents).
        const int row0 = row - lane;
#pragma unroll
        for (int cc = 0; cc < D / 32; ++cc) {
          uint32_t w[32], ow[16];
          if (cc % 2 == 0) {         // what was there has left
            if (lane == 0) bulk_wait_read_all();
            __syncwarp();
          }
          tmem_ld_32x32(o_addr + cc * 32, w);
          tmem_ld_wait_for(w);
          if (cc == D / 32 - 1) {    // the next item's first P V may overwrite the accumulator
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&o_empty[x]);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e)
            ow[e] = seen ? pack_bf16x2(__uint_as_float(w[2 * e]) * inv, __uint_as_float(w[2 * e + 1]) * inv) : 0u;
          if (p.lse != nullptr) {
            uint32_t rest[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float o[4] = {__uint_as_float(w[4 * e]) * inv, __uint_as_float(w[4 * e + 1]) * inv,
                                  __uint_as_float(w[4 * e + 2]) * inv, __uint_as_float(w[4 * e + 3]) * inv};
              rest[e] = seen ? bf16_rest(o, ow[2 * e], ow[2 * e + 1]) : 0u;
            }
            st_global_256(p.rest + ((static_cast<size_t>(b) * p.nh + h) * p.S_pad + row) * D + cc * 32, rest);   // a sector
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(stage + lane * 128 + ((((cc & 1) * 4 + i) ^ (lane & 7)) << 4)) =
                make_uint4(ow[4 * i], ow[4 * i + 1], ow[4 * i + 2], ow[4 * i + 3]);
          if (cc & 1) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && row0 < p.S) {        // (rows past the last token are cut off)
              tma_store_4d(&to, stage, (cc - 1) * 32, row0, h, b);
              bulk_commit();
            }
          }
        }
        if (p.lse != nullptr)
          p.lse[(static_cast<size_t>(b) * p.nh + h) * p.S_pad + row] =
              l > 0.f ? m * k + log2f(l) : (l == 0.f ? INFINITY : l);
      }
      cdone += j1 - j0;
    }
    if (lane == 0) bulk_wait_all();
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 512);
}

struct FwdMaps {
  const CUtensorMap *q, *k, *v, *o;
};

template <int D, int SCORES, bool DIST>
int launch_fwd(const FwdMaps& m, const MaskedFwdParams& p, cudaStream_t stream) {
  static gfs_host::SmemLimit limit;
  constexpr int smem = MFwdShape<D>::SMEM;
  if (!limit.raise(masked_fwd_kernel<D, SCORES, DIST>, smem)) return -10;
  const int tiles = p.S_pad / 128;
  const int n_levels = p.head_pairs ? tiles : (tiles + 1) / 2;
  const unsigned n_items = static_cast<unsigned>(n_levels) * p.B * (p.head_pairs ? p.nh / 2 : p.nh);
  gfs_host::launch_pdl(masked_fwd_kernel<D, SCORES, DIST>, dim3(n_items), dim3(MFWD_THREADS), smem, stream, *m.q,
                       *m.k, *m.v, *m.o, p, n_levels);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}
template <int D, bool DIST>
int launch_fwd_scores(const FwdMaps& m, const MaskedFwdParams& p, cudaStream_t stream) {
  if (p.score.cap2 <= 0.f) return launch_fwd<D, PLAIN, DIST>(m, p, stream);
  if constexpr (!DIST) {       // a bias has no bound: a slope may be negative
    if (p.score.cap2 <= BOUNDED_CAP2) return launch_fwd<D, BOUNDED, false>(m, p, stream);
  }
  return launch_fwd<D, CAPPED, DIST>(m, p, stream);
}

}  // namespace

extern "C" {

// The mask of B sequences of S tokens. ids (int32, or int64 with ids64; null: one document): a run of equal numbers is a
// document, one of negative numbers padding. prefix (bytes; null: none): the leading tokens of a document that are
// marked are seen by all of it. causal 0: every token sees its whole document. window (0: none): a query sees no key
// more than window - 1 tokens back. out: int32, laid out as masked_attention.cuh says (gfs_attention_mask_layout), 16-byte
// aligned.
int gfs_attention_mask(const void* ids, int ids64, const void* prefix, int B, int S, int causal, int window, void* out,
                       void* stream) {
  if (S < 0 || B < 0 || window < 0 || (!causal && (window > 0 || prefix != nullptr)) || S > 0x3fff0000) return -1;   // (i + window fits an int)
  if (S == 0 || B == 0) return 0;
  if (out == nullptr || reinterpret_cast<uintptr_t>(out) & 15) return -2;
  int* o = static_cast<int*>(out);
  const MaskLayout l = mask_layout(B, S);
  const MaskArgs a{ids, static_cast<const uint8_t*>(prefix), ids64, S, (S + 127) / 128 * 128, window > S ? 0 : window, causal,
                   o + l.first, o + l.last, o + l.qfirst, o + l.qlast, o + l.padded, o + l.positions,
                   reinterpret_cast<int4*>(o + l.plan_q), reinterpret_cast<int4*>(o + l.plan_k),
                   reinterpret_cast<int4*>(o + l.pairs)};
  gfs_host::launch_pdl(S > 2 * MASK_THREADS ? attention_mask_kernel<8> : attention_mask_kernel<1>, dim3(B), dim3(MASK_THREADS), 0,
                       static_cast<cudaStream_t>(stream), a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

// offsets[10]: where the buffer of a mask has first, last, qfirst, qlast, plan_q, plan_k, pairs, padded and positions, and its
// length.
void gfs_attention_mask_layout(int B, int S, long long* offsets) {
  const MaskLayout l = mask_layout(B, S);
  const size_t at[10] = {l.first, l.last, l.qfirst, l.qlast, l.plan_q, l.plan_k, l.pairs, l.padded, l.positions, l.end};
  for (int i = 0; i < 10; ++i) offsets[i] = static_cast<long long>(at[i]);
}

// q [B, nh, S, D], k and v [B, nkv, S, D], out like q; strides: 12 element strides {q, k, v, out} x {seq, batch, head}.
// mask: from gfs_attention_mask, of the same B and S. saved: for the backward, fp32 [B, nh, S_pad] (sums of exponentials, log base 2) and
// behind them bytes [B, nh, S_pad, D] (what out's rounding leaves out), 32-byte aligned; or null. cap 0: scores as they are.
// slopes: fp32 [nh] or null.
int gfs_masked_attention_fwd(const void* q, const void* k, const void* v, void* out, void* saved, const void* mask, int S,
                             int B, int nh, int nkv, int D, const long long* strides, float scale, float cap,
                             const void* slopes, void* stream_) {
  if ((D != 64 && D != 128) || !strides_ok(strides, 12) || nkv <= 0 || nh % nkv != 0) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) & 15 || reinterpret_cast<uintptr_t>(saved) & 31)
    return -2;
  if (S <= 0 || B <= 0 || nh <= 0) return 0;
  if (mask == nullptr) return -2;
  const int S_pad = (S + 127) / 128 * 128;
  if (static_cast<long long>(S_pad / 128) * B * nh > 0x7fffffffll) return -1;
  const FwdMaps m{make_map(q, D, S, nh, B, strides + 0, 128), make_map(k, D, S, nkv, B, strides + 3, 64),
                  make_map(v, D, S, nkv, B, strides + 6, 64), make_map(out, D, S, nh, B, strides + 9, 32)};
  if (!m.q || !m.k || !m.v || !m.o) return -3;
  MaskedFwdParams p;
  p.lse = static_cast<float*>(saved);
  p.rest = saved == nullptr ? nullptr : static_cast<uint8_t*>(saved) + 4 * static_cast<size_t>(B) * nh * S_pad;
  p.S = S; p.S_pad = S_pad; p.B = B; p.nh = nh; p.group = nh / nkv;
  p.head_pairs = p.group % 2 == 0;
  p.score.sl2 = cap > 0.f ? 2.f * scale * LOG2E_F / cap : scale * LOG2E_F;
  p.score.cap2 = cap * LOG2E_F;
  p.score.slopes = static_cast<const float*>(slopes);
  p.mask = mask_view(mask, B, S);
  p.status = gfs_host::status_words();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  if (slopes != nullptr)
    return D == 64 ? launch_fwd_scores<64, true>(m, p, stream) : launch_fwd_scores<128, true>(m, p, stream);
  return D == 64 ? launch_fwd_scores<64, false>(m, p, stream) : launch_fwd_scores<128, false>(m, p, stream);
}

}  // extern "C"
