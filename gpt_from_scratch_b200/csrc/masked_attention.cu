// Masked attention, forward, and the kernel that makes its mask (head_dim 64 or 128, bf16; see masked_attention.cuh for
// the mask and the scores, masked_attention_bwd.cu for the gradients).
//
//   out_i = sum_j p_ij v_j,  p_ij = 2^(score_ij - lse_i) over the keys j that query i sees; a query that sees none: 0
//
// One pass over the keys with the running maximum and sum of the softmax; heads of q share the heads of k and v in groups.
#include <algorithm>

#include "api.h"
#include "attention_tiles.cuh"
#include "masked_attention.cuh"

using namespace gfs;
using gfs_host::make_map;
using gfs_host::strides_ok;

namespace {

// ---------------------------------------------------------------------------
// The mask. One CTA per sequence, a thread per token and step: running maxima from the left (where a document starts, the last token
// that is not prefix) and running minima from the right (where it ends, the end of the prefix's run).
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
  int4 *plan_q, *plan_k;
};

// The tiles of a sequence in descending order of the rows between their ends (the work they are): kernels that start the
// heaviest first end together. Ranks by counting; a longer sequence than fits has enough tiles to even out by itself.
constexpr int MASK_SORT = 2048;
__device__ __forceinline__ void sort_tiles(const int* lo, const int* hi, int S, int4* plan, int* weight) {
  const int n = (S + 127) >> 7;
  const bool sorted = n <= MASK_SORT;
  __syncthreads();
  for (int t = threadIdx.x; t < n; t += MASK_THREADS)
    if (sorted) weight[t] = hi[min(t * 128 + 127, S - 1)] - lo[t * 128];
  __syncthreads();
  for (int t = threadIdx.x; t < n; t += MASK_THREADS) {
    int rank = n - 1 - t;
    if (sorted) {
      rank = 0;
      const int mine = weight[t];
      for (int u = 0; u < n; ++u) rank += weight[u] > mine || (weight[u] == mine && u > t);
    }
    plan[rank] = make_int4(t, lo[t * 128], hi[min(t * 128 + 127, S - 1)], 0);
  }
}

__global__ void __launch_bounds__(MASK_THREADS) attention_mask_kernel(const MaskArgs a) {
  pdl_wait();
  pdl_trigger();
  __shared__ int tmp[32];
  __shared__ int weight[MASK_SORT];
  const int b = blockIdx.x;
  const size_t row = static_cast<size_t>(b) * a.S;
  const size_t prow = static_cast<size_t>(b) * a.S_pad;
  auto id_of = [&](int i) -> long long {
    if (a.ids == nullptr) return 0;
    return a.ids64 ? static_cast<const long long*>(a.ids)[row + i] : static_cast<const int*>(a.ids)[row + i];
  };
  auto starts = [&](int i) { return i == 0 || id_of(i) != id_of(i - 1); };
  const int chunks = (a.S + MASK_THREADS - 1) / MASK_THREADS;
  // from the right: the end of the document, and the first token after this one that is not of the prefix's run
  int carry = a.S, carry2 = a.S;
  for (int c = chunks - 1; c >= 0; --c) {
    const int i = c * MASK_THREADS + threadIdx.x;
    const bool in = i < a.S;
    const bool edge = in && starts(i);
    int end, reach = 0;
    block_scan<true>(edge ? i : 0x7fffffff, carry, end, tmp);
    if (a.prefix != nullptr) block_scan<true>(in && (edge || !a.prefix[row + i]) ? i : 0x7fffffff, carry2, reach, tmp);
    if (in) {
      a.qlast[prow + i] = end;
      a.last[prow + i] = reach;
    }
  }
  carry = carry2 = -1;
  int any = 0;
  for (int c = 0; c < chunks; ++c) {
    const int i = c * MASK_THREADS + threadIdx.x;
    const bool in = i < a.S;
    int before;
    const int start = block_scan<false>(in && starts(i) ? i : -1, carry, before, tmp);
    bool lead = false;
    if (a.prefix != nullptr) {
      const bool p = in && a.prefix[row + i];
      const int plain = block_scan<false>(p ? -1 : i, carry2, before, tmp);   // the last token up to here that is not prefix
      lead = p && plain < start;
    }
    if (in) {
      const int end = a.qlast[prow + i];
      int first = start, last = a.causal ? (lead ? a.last[prow + i] : i + 1) : end;
      int qfirst = a.causal && !lead ? i : start, qlast = end;
      if (a.window > 0) {
        first = max(first, i - a.window + 1);
        qlast = min(qlast, i + a.window);
      }
      if (id_of(i) < 0) {
        first = last = qfirst = qlast = start;
        any = 1;
      }
      a.first[prow + i] = first;
      a.last[prow + i] = last;
      a.qfirst[prow + i] = qfirst;
      a.qlast[prow + i] = qlast;
      a.positions[row + i] = i - start;
    }
  }
  for (int i = a.S + threadIdx.x; i < a.S_pad; i += MASK_THREADS)
    a.first[prow + i] = a.last[prow + i] = a.qfirst[prow + i] = a.qlast[prow + i] = a.S;
  any = __syncthreads_or(any);
  if (threadIdx.x == 0) a.padded[b] = any;
  const size_t tiles = static_cast<size_t>(b) * (a.S_pad / 128);
  sort_tiles(a.first + prow, a.last + prow, a.S, a.plan_q + tiles, weight);
  sort_tiles(a.qfirst + prow, a.qlast + prow, a.S, a.plan_k + tiles, weight);
}

// ---------------------------------------------------------------------------
// Forward. A CTA has one tile of 128 queries of a head: TMA warp, MMA warp, eight softmax warps and half of the tensor memory (S | O),
// so two CTAs share an SM and each fills the other's waits. Two warps share the 32 rows of a quarter, 64 of a block's 128
// keys each, and exchange their row maxima through shared memory; P overwrites the scores that it was made from, in tensor memory.
// ---------------------------------------------------------------------------
struct MaskedFwdParams {
  __nv_bfloat16* O;
  long long o_ss, o_bs, o_hs;  // element strides: sequence, batch, head
  float* lse;                  // [B, nh, S_pad], base 2; +inf for rows that see nothing
  int S, S_pad, B, nh, group;
  ScoreArgs score;
  MaskView mask;
  uint32_t* status;
};

constexpr int MFWD_CW = 8;
constexpr int MFWD_THREADS = 32 * (2 + MFWD_CW);
template <int D>
struct MFwdShape {
  static constexpr int DB = D / 64;
  static constexpr int TILE = DB * 16384;
  static constexpr int KS = D == 64 ? 2 : 1;      // stages of K and V
  static constexpr int SMEM = TILE * (1 + 2 * KS) + 2048 + 256;
};

template <int D, bool CAP, bool DIST>
__global__ void __launch_bounds__(MFWD_THREADS, 2)
masked_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                  const __grid_constant__ CUtensorMap tv, const MaskedFwdParams p, int n_tiles) {
  using Shape = MFwdShape<D>;
  constexpr int DB = Shape::DB, TILE = Shape::TILE, KS = Shape::KS;
  constexpr uint32_t O_COL = 128, P_HALF = 64;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* Qs = smem_raw;
  uint8_t* Ks = Qs + TILE;
  uint8_t* Vs = Ks + KS * TILE;
  float* xch = reinterpret_cast<float*>(Vs + KS * TILE);     // [parity][half][row]
  uint64_t* bars = reinterpret_cast<uint64_t*>(xch + 512);
  uint64_t* q_full = bars;
  uint64_t* s_full = bars + 1;
  uint64_t* o_full = bars + 2;
  uint64_t* p_full = bars + 3;
  uint64_t* k_full = bars + 4;
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;
  uint64_t* v_empty = v_full + KS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_empty + KS);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0) record_status(p.status, STATUS_BAD_ARGUMENT, 0x5a21u);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4 + 4 * KS; ++i) mbar_init(&bars[i], i == 3 ? MFWD_CW : 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tq);
    tma_prefetch_desc(&tk);
    tma_prefetch_desc(&tv);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 256);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();       // set-up above may overlap the tail of the preceding kernel (programmatic launch)
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  WaitCtx wctx{abort_flag, p.status, GFS_WAIT_LIMIT_NS};

  const int BH = p.B * p.nh;
  const int level = static_cast<int>(blockIdx.x / BH);                // the tiles that see the most keys come first
  const int bh = static_cast<int>(blockIdx.x % BH);
  const int b = bh / p.nh, h = bh % p.nh, kvh = h / p.group;
  const TilePlan plan = load_plan(p.mask.plan_q + static_cast<size_t>(b) * n_tiles + level);
  const int* first = p.mask.first + static_cast<size_t>(b) * p.S_pad;
  const int* last = p.mask.last + static_cast<size_t>(b) * p.S_pad;
  const int row_a = plan.tile * 128, row_z = min(row_a + 127, p.S - 1);
  // blocks [j0, j1) of 128 keys; at least one, which may be masked whole
  const int j0 = plan.lo >> 7;
  const int j1 = max(j0 + 1, (plan.hi + 127) >> 7);

  if (warp == 0) {
    if (lane == 0) {
      auto load = [&](uint8_t* dst, const CUtensorMap& map, uint64_t* full, int row, int head) {
        mbar_arrive_expect_tx(full, TILE);
#pragma unroll
        for (int db = 0; db < DB; ++db) tma_load_4d(dst + db * 16384, &map, full, db * 64, row, head, b);   // rows past S: zeros
      };
      load(Qs, tq, q_full, row_a, h);
      for (int j = j0; j < j1; ++j) {
        const int g = j - j0, st = g % KS;
        const uint32_t par = ((g / KS) & 1) ^ 1u;
        mbar_wait(&k_empty[st], par, wctx, STATUS_TIMEOUT_PIPE_EMPTY);
        load(Ks + st * TILE, tk, &k_full[st], j * 128, kvh);
        mbar_wait(&v_empty[st], par, wctx, STATUS_TIMEOUT_PIPE_EMPTY);
        load(Vs + st * TILE, tv, &v_full[st], j * 128, kvh);
      }
      settle_copies(wctx);
    }
  } else if (warp == 1) {
    // whole warp, converged: the MMA / commit helpers elect the issuing lane
    constexpr uint32_t idesc_s = umma_idesc_bf16(128, 128, 0, 0);
    constexpr uint32_t idesc_o = umma_idesc_bf16(128, D, 0, 1);
    const bool padded = p.mask.padded[b] != 0;
    mbar_wait(q_full, 0, wctx, STATUS_TIMEOUT_PIPE_FULL);
    auto issue_s = [&](int j) {
      const int g = j - j0, st = g % KS;
      mbar_wait(&k_full[st], (g / KS) & 1, wctx, STATUS_TIMEOUT_PIPE_FULL);
      if (padded) zero_padding(Ks + st * TILE, 128, DB, 16384, first + j * 128, last + j * 128, lane);
      tc_fence_after();
      mma_kk<D / 16>(tmem_base, smem_u32(Qs), 16384, smem_u32(Ks + st * TILE), 16384, idesc_s, false);
      umma_commit_e(s_full);
      umma_commit_e(&k_empty[st]);
    };
    issue_s(j0);
    for (int j = j0; j < j1; ++j) {
      const int g = j - j0, st = g % KS;
      mbar_wait(&v_full[st], (g / KS) & 1, wctx, STATUS_TIMEOUT_PIPE_FULL);
      if (padded) zero_padding(Vs + st * TILE, 128, DB, 16384, first + j * 128, last + j * 128, lane);
      mbar_wait(p_full, g & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
      tc_fence_after();
      mma_tmn<8, P_HALF>(tmem_base + O_COL, tmem_base, smem_u32(Vs + st * TILE), 16384, idesc_o, j > j0);
      umma_commit_e(o_full);
      umma_commit_e(&v_empty[st]);
      if (j + 1 < j1) {
        mbar_wait(o_full, g & 1, wctx, STATUS_TIMEOUT_TMEM_FULL);   // P, where the next scores go, has been read
        issue_s(j + 1);
      }
    }
  } else {
    const int half = (warp - 2) >> 2;                       // keys [64 half, + 64) of every block
    const int quarter = warp & 3;
    const int r = quarter * 32 + lane;
    const int row = row_a + r;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_addr = tmem_base + lane_base + half * 64;
    const uint32_t o_addr = tmem_base + lane_base + O_COL + half * (D / 2);
    const uint32_t p_addr = tmem_base + lane_base + half * P_HALF;
    float* const xch_own = xch + half * 128 + r;            // + 256 * parity
    const float* const xch_other = xch + (half ^ 1) * 128 + r;
    const int lo = first[row], hi = last[row];
    const int lo_max = first[row_z], hi_min = last[row_a];  // a block between these is seen whole by every row
    const float slope2 = DIST ? p.score.slopes[h] * LOG2E_F : 0.f;
    const float k = CAP || DIST ? 1.f : p.score.sl2;        // what turns the numbers in v[] into exponents
    const uint64_t k_2 = pack_f32x2(k, k);
    uint32_t xpar = 0;
    auto exchange = [&](float v) {
      xch_own[xpar * 256] = v;
      named_barrier_sync(1 + quarter, 64);                  // the two warps that share these rows
      const float o = xch_other[xpar * 256];
      xpar ^= 1u;
      return o;
    };
    float m = -INFINITY;
    uint64_t l2 = 0;                                        // two partial sums of this thread's exponentials
    for (int j = j0; j < j1; ++j) {
      const int g = j - j0;
      const int col0 = j * 128 + half * 64;
      mbar_wait(s_full, g & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
      tc_fence_after();
      uint32_t v[2][32];
      tmem_ld_32x32(s_addr, v[0]);
      tmem_ld_32x32(s_addr + 32, v[1]);
      tmem_ld_wait_for(v[0]);
      tmem_ld_wait_for(v[1]);
      if (CAP || DIST) {
        const float dist0 = static_cast<float>(row - col0);
#pragma unroll
        for (int e = 0; e < 64; e += 4) {
          float x[4], y[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) x[u] = __uint_as_float(v[e >> 5][(e & 31) + u]);
          if (CAP) {
            float rr[4];
            sigmoids(x, p.score.sl2, rr);
#pragma unroll
            for (int u = 0; u < 4; ++u) y[u] = fmaf(rr[u], -2.f * p.score.cap2, p.score.cap2);
          } else {
#pragma unroll
            for (int u = 0; u < 4; ++u) y[u] = x[u] * p.score.sl2;
          }
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if (DIST) y[u] = fmaf(fabsf(dist0 - static_cast<float>(e + u)), -slope2, y[u]);
            v[e >> 5][(e & 31) + u] = __float_as_uint(y[u]);
          }
        }
      }
      if (j * 128 < lo_max || j * 128 + 128 > hi_min) {
        // some row does not see some key: dead scores become -inf in the registers, then the block takes the same code as every other
        const int a = lo - col0;
        const unsigned n = static_cast<unsigned>(hi - lo);
#pragma unroll
        for (int e = 0; e < 64; ++e)
          v[e >> 5][e & 31] = static_cast<unsigned>(e - a) < n ? v[e >> 5][e & 31] : 0xff800000u;
      }
      float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
      for (int e = 0; e < 32; e += 2) {
        mx0 = fmax3(mx0, __uint_as_float(v[0][e]), __uint_as_float(v[0][e + 1]));
        mx1 = fmax3(mx1, __uint_as_float(v[1][e]), __uint_as_float(v[1][e + 1]));
      }
      const float mx = fmaxf(mx0, mx1);
      const float m_new = fmax3(m, mx, exchange(mx));
      // the maximum of all keys so far: both threads of a row raise it alike
      const bool grow = m_new > m;
      float alpha = 1.f;
      if (grow) {
        alpha = (m == -INFINITY) ? 0.f : fast_exp2((m - m_new) * k);
        l2 = mul_f32x2(l2, pack_f32x2(alpha, alpha));
        m = m_new;
      }
      const float moff = ((m == -INFINITY) ? 0.f : m) * k;
      const uint64_t moff2 = pack_f32x2(-moff, -moff);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 32; e += 2) {
          const float2 a = unpack_f32x2(fma_f32x2(pack_u32x2(v[c][e], v[c][e + 1]), k_2, moff2));
          const float p0 = fast_exp2(a.x), p1 = fast_exp2(a.y);
          l2 = add_f32x2(l2, pack_f32x2(p0, p1));
          pk[e >> 1] = pack_bf16x2(p0, p1);
        }
        tmem_st_32x16(p_addr + 16 * c, pk);
      }
      if (g > 0 && __any_sync(0xffffffffu, grow)) {
        // rescale this warp's 32 accumulator rows in tensor memory (warp-collective accesses; rows whose maximum stays get
        // factor 1), its half of the columns. P V of the previous block is done: this block's scores were issued after it.
        mbar_wait(o_full, (g - 1) & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
        tc_fence_after();
        uint32_t wv[D / 32][16];
#pragma unroll
        for (int c = 0; c < D / 32; ++c) tmem_ld_32x16(o_addr + 16 * c, wv[c]);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) tmem_ld_wait_for16(wv[c]);
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
#pragma unroll
          for (int e = 0; e < 16; ++e) wv[c][e] = __float_as_uint(__uint_as_float(wv[c][e]) * alpha);
          tmem_st_32x16(o_addr + 16 * c, wv[c]);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(p_full);
    }
    const float2 lp = unpack_f32x2(l2);
    float l = lp.x + lp.y;
    l += exchange(l);
    const float inv_l = (l > 0.f) ? 1.f / l : 0.f;
    mbar_wait(o_full, (j1 - j0 - 1) & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
    tc_fence_after();
    uint32_t o[D / 64][32];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) tmem_ld_32x32(o_addr + 32 * c, o[c]);
#pragma unroll
    for (int c = 0; c < D / 64; ++c) tmem_ld_wait_for(o[c]);
    if (row < p.S) {
      const bool seen = lo < hi;
      __nv_bfloat16* dst = p.O + row * p.o_ss + b * p.o_bs + h * p.o_hs + half * (D / 2);
      auto two = [&](int c, int e) {
        return seen ? pack_bf16x2(__uint_as_float(o[c][e]) * inv_l, __uint_as_float(o[c][e + 1]) * inv_l) : 0u;
      };
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
#pragma unroll
        for (int e = 0; e < 32; e += 8)
          *reinterpret_cast<uint4*>(dst + 32 * c + e) = make_uint4(two(c, e), two(c, e + 2), two(c, e + 4), two(c, e + 6));
      }
    }
    if (half == 0 && p.lse != nullptr)
      p.lse[static_cast<size_t>(bh) * p.S_pad + row] = l > 0.f ? m * k + log2f(l) : (l == 0.f ? INFINITY : l);
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, 256);
}

template <int D, bool CAP, bool DIST>
int launch_fwd(const CUtensorMap* tq, const CUtensorMap* tk, const CUtensorMap* tv, const MaskedFwdParams& p,
               cudaStream_t stream) {
  static gfs_host::SmemLimit limit;
  constexpr int smem = MFwdShape<D>::SMEM;
  if (!limit.raise(masked_fwd_kernel<D, CAP, DIST>, smem)) return -10;
  const int n_tiles = p.S_pad / 128;
  gfs_host::launch_pdl(masked_fwd_kernel<D, CAP, DIST>, dim3(static_cast<unsigned>(n_tiles) * p.B * p.nh),
                       dim3(MFWD_THREADS), smem, stream, *tq, *tk, *tv, p, n_tiles);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}
template <int D>
int launch_fwd_scores(const CUtensorMap* tq, const CUtensorMap* tk, const CUtensorMap* tv, const MaskedFwdParams& p,
                      bool cap, cudaStream_t stream) {
  const bool dist = p.score.slopes != nullptr;
  if (cap) return dist ? launch_fwd<D, true, true>(tq, tk, tv, p, stream) : launch_fwd<D, true, false>(tq, tk, tv, p, stream);
  return dist ? launch_fwd<D, false, true>(tq, tk, tv, p, stream) : launch_fwd<D, false, false>(tq, tk, tv, p, stream);
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
  if (S < 0 || B < 0 || window < 0 || (!causal && (window > 0 || prefix != nullptr)) || S > 0x7fffff00) return -1;
  if (S == 0 || B == 0) return 0;
  if (reinterpret_cast<uintptr_t>(out) & 15) return -2;
  int* o = static_cast<int*>(out);
  const MaskLayout l = mask_layout(B, S);
  const MaskArgs a{ids, static_cast<const uint8_t*>(prefix), ids64, S, (S + 127) / 128 * 128, window > S ? 0 : window, causal,
                   o + l.first, o + l.last, o + l.qfirst, o + l.qlast, o + l.padded, o + l.positions,
                   reinterpret_cast<int4*>(o + l.plan_q), reinterpret_cast<int4*>(o + l.plan_k)};
  gfs_host::launch_pdl(attention_mask_kernel, dim3(B), dim3(MASK_THREADS), 0, static_cast<cudaStream_t>(stream), a);
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

// offsets[9]: where the buffer of a mask has first, last, qfirst, qlast, plan_q, plan_k, padded and positions, and its length.
void gfs_attention_mask_layout(int B, int S, long long* offsets) {
  const MaskLayout l = mask_layout(B, S);
  const size_t at[9] = {l.first, l.last, l.qfirst, l.qlast, l.plan_q, l.plan_k, l.padded, l.positions, l.end};
  for (int i = 0; i < 9; ++i) offsets[i] = static_cast<long long>(at[i]);
}

// q [B, nh, S, D], k and v [B, nkv, S, D], out like q; strides: 12 element strides {q, k, v, out} x {seq, batch, head}.
// mask: from gfs_attention_mask, of the same B and S. lse: fp32 [B, nh, S_pad], base 2, or null (no backward will follow). cap 0: scores as they are.
// slopes: fp32 [nh] or null.
int gfs_masked_attention_fwd(const void* q, const void* k, const void* v, void* out, void* lse, const void* mask, int S,
                             int B, int nh, int nkv, int D, const long long* strides, float scale, float cap,
                             const void* slopes, void* stream_) {
  if ((D != 64 && D != 128) || !strides_ok(strides, 12) || nkv <= 0 || nh % nkv != 0) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out)) & 15)
    return -2;
  if (S <= 0 || B <= 0 || nh <= 0) return 0;
  const int S_pad = (S + 127) / 128 * 128;
  if (static_cast<long long>(S_pad / 128) * B * nh > 0x7fffffffll) return -1;
  const CUtensorMap* tq = make_map(q, D, S, nh, B, strides + 0, 128);
  const CUtensorMap* tk = make_map(k, D, S, nkv, B, strides + 3, 128);
  const CUtensorMap* tv = make_map(v, D, S, nkv, B, strides + 6, 128);
  if (!tq || !tk || !tv) return -3;
  MaskedFwdParams p;
  p.O = static_cast<__nv_bfloat16*>(out);
  p.o_ss = strides[9]; p.o_bs = strides[10]; p.o_hs = strides[11];
  p.lse = static_cast<float*>(lse);
  p.S = S; p.S_pad = S_pad; p.B = B; p.nh = nh; p.group = nh / nkv;
  p.score.sl2 = cap > 0.f ? 2.f * scale * LOG2E_F / cap : scale * LOG2E_F;
  p.score.cap2 = cap * LOG2E_F;
  p.score.slopes = static_cast<const float*>(slopes);
  p.mask = mask_view(mask, B, S);
  p.status = gfs_host::status_words();
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  return D == 64 ? launch_fwd_scores<64>(tq, tk, tv, p, cap > 0.f, stream)
                 : launch_fwd_scores<128>(tq, tk, tv, p, cap > 0.f, stream);
}

}  // extern "C"
