// Masked attention, backward (head_dim 64 or 128, bf16; the mask and the scores: masked_attention.cuh).
//
//   P = 2^(score - lse), dP = dO V^T, dvec = rowsum(dO * O), dS = P (dP - dvec) (times 1 - tanh^2 of capped scores)
//   dV = P^T dO, dK = scale dS^T Q (both summed over the heads of q that share them), dQ = scale dS K
//
// Two kernels from one template, deterministic, no atomics, after a pre-pass for dvec:
//   mode 0: items of 128 keys    -> dK, dV, streaming 64-query tiles of every head of the group
//   mode 1: items of 128 queries -> dQ,     streaming 64-key tiles
// Only the streamed tiles between the item's first and last visible row are visited. Both modes recompute P from two score MMAs
// (X = R1 T1^T, Y = R2 T2^T) and hand P / dS to the gradient MMAs through tensor memory, rounded to bf16, the type of q, k and dO that
// they meet there (up to 2^-8 of each; errors of gradients 2.4 to 2.5e-3, of documents of a few tokens up to 3.4e-3, with 1.7e-3 for the
// results' own rounding; in two parts each product would be made twice); the streamed tile is
// consumed twice from the same shared-memory bytes, K-major and MN-major.
#include <algorithm>

#include "api.h"
#include "attention_tiles.cuh"
#include "masked_attention.cuh"

using namespace gfs;
using gfs_host::make_map;
using gfs_host::strides_ok;

namespace {

// ---------------------------------------------------------------------------
// Pre-pass (25 MB + 25 MB + 13 MB: 16 us): dvec[b, h, s] = sum_d dO * O, O with what its rounding left out, 0 for padding (whatever its
// dO holds) and for rows S .. S_pad. Eight threads per row, 16 bytes (head_dim 128: twice) of dO and O, four rows (two: four leave
// room for two CTAs per SM, 4 us more) a thread with all loads issued first; rows in the memory order of O (heads or tokens
// fastest), one division by a constant of the launch per row.
// ---------------------------------------------------------------------------
constexpr int dvec_rows(int D) { return 256 / D; }
struct DvecArgs {
  const __nv_bfloat16 *dO, *O;
  const uint8_t* rest;         // [B, nh, S_pad, D]: what O's rounding left out
  float* dvec;
  const int *first, *last, *padded;
  int S, S_pad, nh;
  long long do_ss, do_bs, do_hs, o_ss, o_bs, o_hs;
  unsigned inner;              // length of the faster index: S_pad (tokens) or nh (heads)
  unsigned long long magic;    // floor(2^40 / inner) + 1: row / inner = row * magic >> 40 for row < 2^24, inner <= 2^16; or 0
  int s_fastest;
};
template <int D>
__global__ void __launch_bounds__(256) masked_dvec_kernel(const DvecArgs a) {
  pdl_wait();
  pdl_trigger();
  constexpr int V = D / 64;                     // 16-byte vectors a thread
  constexpr int ROWS = dvec_rows(D);
  const int sub = threadIdx.x & 7, b = blockIdx.y;
  const unsigned total = static_cast<unsigned>(a.S_pad) * a.nh;
  const unsigned row0 = blockIdx.x * (32u * ROWS) + (threadIdx.x >> 3);
  uint4 x[ROWS][V], y[ROWS][V];
  uint2 z[ROWS][V];
  unsigned at[ROWS], token[ROWS];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const unsigned row = row0 + 32u * i;
    const unsigned outer = a.magic != 0 ? static_cast<unsigned>((row * a.magic) >> 40) : row / a.inner;
    const unsigned rest = row - outer * a.inner;
    const unsigned s = a.s_fastest ? rest : outer, h = a.s_fastest ? outer : rest;
    at[i] = h * a.S_pad + s;
    token[i] = min(s, static_cast<unsigned>(a.S_pad) - 1u);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      x[i][v] = y[i][v] = make_uint4(0, 0, 0, 0);
      z[i][v] = make_uint2(0, 0);
    }
    if (row < total && s < static_cast<unsigned>(a.S)) {
      const __nv_bfloat16* px = a.dO + s * a.do_ss + b * a.do_bs + h * a.do_hs + sub * 8;
      const __nv_bfloat16* py = a.O + s * a.o_ss + b * a.o_bs + h * a.o_hs + sub * 8;
      const uint8_t* pz = a.rest + (static_cast<size_t>(b) * a.nh * a.S_pad + at[i]) * D + sub * 8;
#pragma unroll
      for (int v = 0; v < V; ++v) {
        x[i][v] = *reinterpret_cast<const uint4*>(px + 64 * v);
        y[i][v] = *reinterpret_cast<const uint4*>(py + 64 * v);
        z[i][v] = *reinterpret_cast<const uint2*>(pz + 64 * v);
      }
    }
  }
  const bool padded = a.padded[b] != 0;       // (after the loads: they do not wait for it)
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    float acc = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const uint32_t xw[4] = {x[i][v].x, x[i][v].y, x[i][v].z, x[i][v].w};
      const uint32_t yw[4] = {y[i][v].x, y[i][v].y, y[i][v].z, y[i][v].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 a2 = unpack_bf16x2(xw[e]), b2 = with_rest(yw[e], e < 2 ? z[i][v].x : z[i][v].y, 2 * (e & 1));
        acc += a2.x * b2.x + a2.y * b2.y;
      }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
    const size_t m = static_cast<size_t>(b) * a.S_pad + token[i];
    if (padded && a.first[m] >= a.last[m]) acc = 0.f;
    if (row0 + 32u * i < total && sub == 0) a.dvec[static_cast<size_t>(b) * a.nh * a.S_pad + at[i]] = acc;
  }
}

// ---------------------------------------------------------------------------
// Main kernel
// ---------------------------------------------------------------------------
struct MaskedBwdParams {
  float* partial;       // mode 0, parts > 1: fp32 [parts][dK, dV][B, nkv, S_pad, D]
  int parts;            // the heads of a group are dealt to this many items
  const float* lse;   // [B, nh, S_pad], base 2
  const float* dvec;  // [B, nh, S_pad]
  int S, S_pad, B, nh, group;
  float scale;
  ScoreArgs score;
  MaskView mask;
  uint32_t* status;
};

constexpr int MBWD_CW = 16;                         // compute warps
constexpr int MBWD_FIRST_CW = 4;                    // warps 0-2: TMA, score MMAs, gradient MMAs; 3: items
constexpr int MBWD_THREADS = 32 * (MBWD_FIRST_CW + MBWD_CW);

// A work item, as warp 3 puts it into shared memory when the one before has been taken: nobody else divides or waits for the plans. At
// head_dim 64 there is room for what the resident rows see and (mode 1) their statistics too.
struct alignas(16) BwdItem {
  uint4 claim;                 // what claim_cta answered
  int more;                    // 0: there are no further items
  int b, h, rt, part, padded;
  int t_begin, n_t;            // streamed tiles per head (at least one, which may be masked whole)
};
struct BwdRows {
  int lo[128], hi[128];
  float lse[128], dvec[128];
};

template <int D, int MODE>
struct MBwdShape {
  // Stages of the streamed-tile ring. A stage is only released when the gradient MMAs that read it have
  // finished and the score MMAs run two tiles ahead, so the TMA of a tile has (TS - 2) tile periods to land.
  static constexpr int TS = D == 64 ? 7 : 4;
  static constexpr int STAGE_BYTES = 2048;          // per compute warp, to transpose its output rows through
  static constexpr int STAGING = MBWD_CW * STAGE_BYTES;
  static constexpr bool ROWS = D == 64;             // BwdRows beside the items
  static constexpr int ITEMS = static_cast<int>(sizeof(BwdItem) + (ROWS ? sizeof(BwdRows) : 0));
  static constexpr int SMEM = 2 * (D / 64) * 16384 + 2 * TS * (D / 64) * 8192 + STAGING + (MODE == 0 ? TS * 512 : 0) + ITEMS + 256;
};

// Sixteen compute warps: two groups of eight take alternate streamed tiles (group = X/Y buffer); within a group two warps
// share the 32 rows of a quarter, 32 streamed columns each (no exchange is needed: the statistics are inputs). The
// MMAs are issued by two warps (1: scores, 2: gradients), so neither order waits for the other. P / dS go to columns of their own
// where there is room, for dK / dV at head_dim 128 to the columns of the scores they were made from.
//
// Bound, at head_dim 128, by shared memory feeding the tensor pipe: a score MMA of 128 x 64 x 16 reads 6 KB for 32 cycles of
// multiplication, so that it takes 48, and with the gradients' a streamed tile needs 1,280 (dQ: 1,024) cycles of 1,790 (1,350); with
// a cap by the chain of its 2.25 special function operations a score. us, dK / dV with dQ beside them (each alone): 16 heads (4
// of k) of 8192 tokens, head_dim 128, documents with prefixes 232 (166, 114); 4 x 16 heads (4) of 2048, capped 181 (134, 89); 16 x 12
// heads of 1024, head_dim 64, in documents of 200 tokens, four streamed tiles an item, 98 (62, 48): there items' ends weigh as much
// as their tiles. What items cost was cut by a warp that prepares them (their plans, and the rows' statistics), by claiming them,
// by not parting groups of heads where there is an item for every SM (the first case 280 -> 232), and by results that leave by TMA
// (whole calls 368 -> 362, 284 -> 279, 170 -> 166); not by loading the
// next resident tiles early nor by prefetching rows into registers. Handing P over before dS is made, so that dV's products
// start earlier, made registers spill: 146 -> 151 and 102 -> 162.
template <int D, int MODE, bool CAP, bool DIST>
__global__ void __launch_bounds__(MBWD_THREADS, 1)
masked_bwd_kernel(const __grid_constant__ CUtensorMap tr1, const __grid_constant__ CUtensorMap tr2,
                  const __grid_constant__ CUtensorMap tt1, const __grid_constant__ CUtensorMap tt2,
                  const __grid_constant__ CUtensorMap to1, const __grid_constant__ CUtensorMap to2,     // mode 0: dK, dV; mode 1: dQ, -
                  const MaskedBwdParams p, int n_rt) {
  using Shape = MBwdShape<D, MODE>;
  constexpr int DB = D / 64;
  constexpr int TS = Shape::TS;
  constexpr int R_BYTES = DB * 16384;  // resident [128 x D]
  constexpr int T_BYTES = DB * 8192;   // streamed [64 x D]
  constexpr uint32_t TMEM_COLS = 512;
  constexpr uint32_t Y_COL = 128;      // X tiles at [0, 128), Y tiles after them
  constexpr uint32_t ACC1 = 256, ACC2 = 256 + D;
  constexpr bool OVERLAY = (D == 128 && MODE == 0);   // P over X, dS over Y
  constexpr uint32_t PT_COL = 384;     // else: [buffer][P 32 cols | dS 32 cols]
  constexpr int EPI_WARPS = (MODE == 1 && D == 64) ? MBWD_CW / 2 : MBWD_CW;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* R1 = smem_raw;
  uint8_t* R2 = R1 + R_BYTES;
  uint8_t* T1 = R2 + R_BYTES;
  uint8_t* T2 = T1 + TS * T_BYTES;
  uint8_t* staging = T2 + TS * T_BYTES;
  float* stats = reinterpret_cast<float*>(staging + Shape::STAGING);  // mode 0: [TS stages][lse 64 | dvec 64]
  BwdItem* slot = reinterpret_cast<BwdItem*>(reinterpret_cast<uint8_t*>(stats) + (MODE == 0 ? TS * 512 : 0));
  BwdRows* rows = reinterpret_cast<BwdRows*>(slot + 1);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(slot) + Shape::ITEMS);
  uint64_t* r_full = bars;
  uint64_t* t_full = bars + 1;             // [TS]
  uint64_t* t_empty = t_full + TS;         // [TS]
  uint64_t* xy_full = t_empty + TS;
  uint64_t* xy_empty = xy_full + 2;
  uint64_t* m_full = xy_empty + 2;
  uint64_t* m_empty = m_full + 2;
  uint64_t* acc_full = m_empty + 2;
  uint64_t* acc_empty = acc_full + 1;
  uint64_t* r_empty = acc_full + 2;
  uint64_t* i_full = acc_full + 3;
  uint64_t* i_empty = i_full + 1;
  uint64_t* i_claim = i_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(i_full + 3);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (smem_u32(smem_raw) & 1023u) {
    if (threadIdx.x == 0) record_status(p.status, STATUS_BAD_ARGUMENT, 0x5a23u);
    return;
  }
  // the rows that a resident row sees: queries of a key, keys of a query
  const int* const lo_all = MODE == 0 ? p.mask.qfirst : p.mask.first;
  const int* const hi_all = MODE == 0 ? p.mask.qlast : p.mask.last;
  // An item (resident tile, batch * head * part) is a CTA of the grid, the heaviest first; those that run (one per SM) claim
  // further ones. Barrier phases run on counters that continue across items, so the next item's loads and first score MMAs overlap
  // this one's epilogue.
  const int hpi = MODE == 0 ? p.group / p.parts : 1;    // heads per item

  if (threadIdx.x == 0) {
    mbar_init(r_full, 1);
    for (int i = 0; i < TS; ++i) {
      mbar_init(&t_full[i], 1);
      mbar_init(&t_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&xy_full[i], 1);
      mbar_init(&xy_empty[i], MBWD_CW / 2);
      mbar_init(&m_full[i], MBWD_CW / 2);
      mbar_init(&m_empty[i], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, EPI_WARPS);
    mbar_init(r_empty, 1);
    mbar_init(i_full, 32);
    mbar_init(i_empty, 3 + MBWD_CW);
    mbar_init(i_claim, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tr1);
    tma_prefetch_desc(&tr2);
    tma_prefetch_desc(&tt1);
    tma_prefetch_desc(&tt2);
    tma_prefetch_desc(&to1);
    if (MODE == 0) tma_prefetch_desc(&to2);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Set-up above may overlap the tail of the preceding kernel (programmatic launch). The dQ kernel reads nothing that the
  // preceding dK / dV kernel writes, and that one had waited for everything before it when it let this one start: it
  // waits at its end, so that its completion means that of both (launch_hints.h).
  if (MODE == 0) pdl_wait();
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;
  WaitCtx wctx{abort_flag, p.status, GFS_WAIT_LIMIT_NS};
  // The it-th item is copied out of the slot and the slot released; false, for the whole warp: there are no more, or a wait has
  // given up.
  auto take_item = [&](int it, BwdItem& item) {
    mbar_wait(i_full, it & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
    item = *slot;
    return !__any_sync(0xffffffffu, item.more == 0 || *abort_flag != 0);
  };
  auto release_item = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(i_empty);
  };

  if (warp == 0) {
    {
      int g = 0;  // streamed tiles loaded so far (ring position)
      BwdItem item;
      for (int it = 0; take_item(it, item); ++it, release_item()) {     // released, so the next one claimed, after the loads
        if (lane != 0) continue;
        const int rt = item.rt, b = item.b, h = item.h, t_begin = item.t_begin, n_t = item.n_t;
        mbar_wait(r_empty, (it & 1) ^ 1u, wctx, STATUS_TIMEOUT_PIPE_EMPTY);  // previous item's score MMAs done
        mbar_arrive_expect_tx(r_full, 2 * R_BYTES);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          tma_load_4d(R1 + db * 16384, &tr1, r_full, db * 64, rt * 128, h, b);
          tma_load_4d(R2 + db * 16384, &tr2, r_full, db * 64, rt * 128, h, b);
        }
        for (int hh = 0; hh < hpi; ++hh) {
          const int th = MODE == 0 ? h * p.group + item.part * hpi + hh : h / p.group;   // head of the streamed tiles
          for (int t = 0; t < n_t; ++t, ++g) {
            const int st = g % TS;
            const int ti = t_begin + t;
            mbar_wait(&t_empty[st], ((g / TS) & 1) ^ 1u, wctx, STATUS_TIMEOUT_PIPE_EMPTY);
            mbar_arrive_expect_tx(&t_full[st], 2 * T_BYTES + (MODE == 0 ? 512 : 0));
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              tma_load_4d(T1 + st * T_BYTES + db * 8192, &tt1, &t_full[st], db * 64, ti * 64, th, b);
              tma_load_4d(T2 + st * T_BYTES + db * 8192, &tt2, &t_full[st], db * 64, ti * 64, th, b);
            }
            if (MODE == 0) {
              const size_t off = (static_cast<size_t>(b) * p.nh + th) * p.S_pad + ti * 64;
              bulk_load_1d(stats + st * 128, p.lse + off, 256, &t_full[st]);
              bulk_load_1d(stats + st * 128 + 64, p.dvec + off, 256, &t_full[st]);
            }
          }
        }
      }
      if (lane == 0) settle_copies(wctx);
    }
  } else if (warp == 1) {
    // Score MMAs (whole warp, converged: the MMA / commit helpers elect the issuing lane); runs ahead as
    // far as the X/Y buffers and the streamed-tile ring allow.
    constexpr uint32_t idesc_xy = umma_idesc_bf16(128, 64, 0, 0);
    const uint32_t r1 = smem_u32(R1), r2 = smem_u32(R2);
    int g = 0;
    BwdItem item;
    for (int it = 0; take_item(it, item); ++it) {
      release_item();
      const int b = item.b, t_begin = item.t_begin, n_t = item.n_t;
      const bool padded = item.padded != 0;
      const int n = n_t * hpi;
      mbar_wait(r_full, it & 1, wctx, STATUS_TIMEOUT_PIPE_FULL);
      for (int t = 0; t < n; ++t, ++g) {
        const int st = g % TS, sb = g & 1;
        mbar_wait(&t_full[st], (g / TS) & 1, wctx, STATUS_TIMEOUT_PIPE_FULL);
        if (padded) {
          const size_t at = static_cast<size_t>(b) * p.S_pad + (t_begin + t % n_t) * 64;
          zero_padding(T1 + st * T_BYTES, 64, DB, 8192, p.mask.first + at, p.mask.last + at, lane);
          zero_padding(T2 + st * T_BYTES, 64, DB, 8192, p.mask.first + at, p.mask.last + at, lane);
        }
        mbar_wait(OVERLAY ? &m_empty[sb] : &xy_empty[sb], ((g >> 1) & 1) ^ 1u, wctx, STATUS_TIMEOUT_SOFTMAX);
        tc_fence_after();
        mma_kk<D / 16>(tmem_base + sb * 64, r1, 16384, smem_u32(T1 + st * T_BYTES), 8192, idesc_xy, false);
        mma_kk<D / 16>(tmem_base + Y_COL + sb * 64, r2, 16384, smem_u32(T2 + st * T_BYTES), 8192, idesc_xy, false);
        umma_commit_e(&xy_full[sb]);
      }
      umma_commit_e(r_empty);
    }
  } else if (warp == 2) {
    // gradient MMAs
    constexpr uint32_t idesc_acc = umma_idesc_bf16(128, D, 0, 1);
    int g = 0;
    BwdItem item;
    for (int it = 0; take_item(it, item); ++it) {
      release_item();
      const int n = item.n_t * hpi;
      for (int t = 0; t < n; ++t, ++g) {
        const int st = g % TS, sb = g & 1;
        mbar_wait(&m_full[sb], (g >> 1) & 1, wctx, STATUS_TIMEOUT_SOFTMAX);
        if (t == 0) mbar_wait(acc_empty, (it & 1) ^ 1u, wctx, STATUS_TIMEOUT_TMEM_EMPTY);  // previous epilogue done
        tc_fence_after();
        const uint32_t pt = tmem_base + (OVERLAY ? sb * 64 : PT_COL + sb * 64);
        const uint32_t ds = OVERLAY ? pt + Y_COL : pt + 32;
        constexpr int HALF = OVERLAY ? 32 : 16;   // columns from the first to the second half of P / dS
        if (MODE == 0) {
          mma_tmn<4, HALF>(tmem_base + ACC1, pt, smem_u32(T2 + st * T_BYTES), 8192, idesc_acc, t > 0);   // dV += P^T dO
          mma_tmn<4, HALF>(tmem_base + ACC2, ds, smem_u32(T1 + st * T_BYTES), 8192, idesc_acc, t > 0);   // dK += dS^T Q
        } else {
          mma_tmn<4, HALF>(tmem_base + ACC1, ds, smem_u32(T1 + st * T_BYTES), 8192, idesc_acc, t > 0);   // dQ += dS K
        }
        umma_commit_e(&t_empty[st]);
        umma_commit_e(&m_empty[sb]);
      }
      umma_commit_e(acc_full);
    }
  } else if (warp == 3) {
    const int heads = MODE == 0 ? p.nh / p.group : p.nh;
    const int BHP = p.B * heads * p.parts;
    const int4* const plans = MODE == 0 ? p.mask.plan_k : p.mask.plan_q;
    for (int it = 0;; ++it) {
      mbar_wait(i_empty, (it & 1) ^ 1u, wctx, STATUS_TIMEOUT_PIPE_EMPTY);
      int w = blockIdx.x;
      bool more = true;
      if (it > 0) {
        if (lane == 0) claim_cta(&slot->claim, i_claim);
        more = mbar_wait(i_claim, (it - 1) & 1, wctx, STATUS_TIMEOUT_PIPE_FULL) && claimed_cta(&slot->claim, w);
        more = __all_sync(0xffffffffu, more);
        fence_proxy_async_smem();      // the next answer comes after everybody has read this one
      }
      int4 plan = make_int4(0, 0, 0, 0);
      int b = 0, h = 0, part = 0;
      int lo[4], hi[4];
      float lse[4] = {}, dvec[4] = {};
      if (more) {
        const int level = w / BHP;
        int q = w - level * BHP;
        part = q % p.parts;
        q /= p.parts;
        b = q / heads;
        h = q - b * heads;
        plan = plans[static_cast<size_t>(b) * n_rt + level];
        if (Shape::ROWS) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = plan.x * 128 + 32 * i + lane;
            lo[i] = lo_all[static_cast<size_t>(b) * p.S_pad + row];
            hi[i] = hi_all[static_cast<size_t>(b) * p.S_pad + row];
            if (MODE == 1) {
              lse[i] = p.lse[(static_cast<size_t>(b) * p.nh + h) * p.S_pad + row];
              dvec[i] = p.dvec[(static_cast<size_t>(b) * p.nh + h) * p.S_pad + row];
            }
          }
        }
      }
      if (more && Shape::ROWS) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          rows->lo[32 * i + lane] = lo[i];
          rows->hi[32 * i + lane] = hi[i];
          if (MODE == 1) {
            rows->lse[32 * i + lane] = lse[i];
            rows->dvec[32 * i + lane] = dvec[i];
          }
        }
      }
      if (lane == 0) {
        const int t_begin = plan.y >> 6;
        slot->more = more;
        slot->b = b;
        slot->h = h;
        slot->rt = plan.x;
        slot->part = part;
        slot->padded = plan.w;
        slot->t_begin = t_begin;
        slot->n_t = max(((plan.z + 63) >> 6) - t_begin, 1);
      }
      __syncwarp();
      mbar_arrive(i_full);
      if (!more || __any_sync(0xffffffffu, *abort_flag != 0)) break;
    }
    if (lane == 0) settle_copies(wctx);
  } else {
    const int cw = warp - MBWD_FIRST_CW;
    const int quarter = warp & 3;
    const int half = (cw >> 2) & 1;     // 32 of the 64 streamed columns
    const int group = cw >> 3;          // parity of the streamed tiles of this warp
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = static_cast<uint32_t>(quarter * 32) << 16;
    const float sl2 = p.score.sl2, cap2 = p.score.cap2;
    const uint64_t neg_sl2 = pack_f32x2(-sl2, -sl2), neg_one = pack_f32x2(-1.f, -1.f);
    const uint32_t x_addr = tmem_base + lane_base + group * 64 + half * 32;
    const uint32_t y_addr = x_addr + Y_COL;
    const uint32_t p_addr = OVERLAY ? x_addr : tmem_base + lane_base + PT_COL + group * 64 + half * 16;
    const uint32_t ds_addr = OVERLAY ? y_addr : p_addr + 32;
    uint8_t* stage = staging + cw * Shape::STAGE_BYTES;
    bool acc_pending = false;           // the previous item's acc_full phase has not been waited for
    int g0 = 0;
    BwdItem item;
    for (int it = 0; take_item(it, item); ++it) {
      const int rt = item.rt, b = item.b, h = item.h, t_begin = item.t_begin, n_t = item.n_t;
      const int head0 = MODE == 0 ? h * p.group + item.part * hpi : h;   // query head of the item's first tiles
      const int n = n_t * hpi;
      const int row_g = rt * 128 + r;  // mode 0: key position, mode 1: query position
      int lo, hi;
      float row_lse = 0.f, row_dvec = 0.f;
      if (Shape::ROWS) {
        lo = rows->lo[r];
        hi = rows->hi[r];
        if (MODE == 1) {
          row_lse = rows->lse[r];
          row_dvec = rows->dvec[r];
        }
      } else {
        const size_t at = static_cast<size_t>(b) * p.S_pad + row_g;
        lo = lo_all[at];
        hi = hi_all[at];
        if (MODE == 1) {
          row_lse = p.lse[(static_cast<size_t>(b) * p.nh + h) * p.S_pad + row_g];
          row_dvec = p.dvec[(static_cast<size_t>(b) * p.nh + h) * p.S_pad + row_g];
        }
      }
      release_item();
      const int row0 = rt * 128 + quarter * 32;
      // what every row of this warp sees, and what any of them does (a warp past the end: nothing)
      const int z = max(min(31, p.S - 1 - row0), 0);
      const int lo_min = __shfl_sync(0xffffffffu, lo, 0), hi_min = __shfl_sync(0xffffffffu, hi, 0);
      const int lo_max = __shfl_sync(0xffffffffu, lo, z), hi_max = __shfl_sync(0xffffffffu, hi, z);
      for (int t = (g0 + group) & 1; t < n; t += 2) {
        const int g = g0 + t;
        const int st = g % TS;                      // streamed-tile stage (for the column statistics)
        const uint32_t par = (g >> 1) & 1;
        const int hh = MODE == 0 ? t / n_t : 0;
        const int col0 = (t_begin + t - hh * n_t) * 64 + half * 32;       // position of this warp's first column
        const int kind = col0 > hi_max - 1 || col0 + 31 < lo_min || hi_max <= lo_min ? 2      // nothing is seen
                         : (col0 >= lo_max && col0 + 32 <= hi_min ? 0 : 1);                   // everything; some
        mbar_wait(&xy_full[group], par, wctx, STATUS_TIMEOUT_SOFTMAX);
        tc_fence_after();
        uint32_t pp[16], dd[16];
        if (kind == 2) {
#pragma unroll
          for (int e = 0; e < 16; ++e) pp[e] = dd[e] = 0u;
          if (!OVERLAY && lane == 0) mbar_arrive(&xy_empty[group]);
        } else {
          uint32_t xv[32], yv[32];
          tmem_ld_32x32(x_addr, xv);
          tmem_ld_32x32(y_addr, yv);
          tmem_ld_wait_for(xv);
          tmem_ld_wait_for(yv);
          if (!OVERLAY) {
            // X / Y are in registers: hand the buffer back now so the next scores can be computed
            // into it while this block's math runs
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&xy_empty[group]);
          }
          const float slope2 = DIST ? p.score.slopes[head0 + hh] * LOG2E_F : 0.f;
          const float dist0 = static_cast<float>(row_g - col0);
          const int a = lo - col0;
          const unsigned width = static_cast<unsigned>(hi - lo);
          // Chunks seen in part turn their dead scores into -inf in the registers, which makes both P and dS exact
          // zeros (dvec and dP are finite: padding was zeroed), and run the same code as the others.
          if (!CAP && kind == 1) {
#pragma unroll
            for (int e = 0; e < 32; ++e) xv[e] = static_cast<unsigned>(e - a) < width ? xv[e] : 0xff800000u;
          }
          const float* st_lse = stats + st * 128 + half * 32;
          const float* st_dv = st_lse + 64;
#pragma unroll
          for (int e = 0; e < 32; e += 4) {
            uint64_t ls[2], dv[2];
            if (MODE == 0) {   // per-column statistics of the streamed query tile (same address in all lanes)
              const float4 l4 = *reinterpret_cast<const float4*>(st_lse + e);
              const float4 d4 = *reinterpret_cast<const float4*>(st_dv + e);
              ls[0] = pack_f32x2(l4.x, l4.y); ls[1] = pack_f32x2(l4.z, l4.w);
              dv[0] = pack_f32x2(d4.x, d4.y); dv[1] = pack_f32x2(d4.z, d4.w);
            } else {
              ls[0] = ls[1] = pack_f32x2(row_lse, row_lse);
              dv[0] = dv[1] = pack_f32x2(row_dvec, row_dvec);
            }
            uint64_t r[2];             // of capped scores: their derivative is 4 r (1 - r)
            if (CAP) sigmoids(pack_u32x2(xv[e], xv[e + 1]), pack_u32x2(xv[e + 2], xv[e + 3]), pack_f32x2(sl2, sl2), r[0], r[1]);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              // lse - score, formed negated (the exponential turns the sign back), two columns per instruction
              uint64_t z = CAP ? fma_f32x2(r[u], pack_f32x2(2.f * cap2, 2.f * cap2), add_f32x2(ls[u], pack_f32x2(-cap2, -cap2)))
                               : fma_f32x2(pack_u32x2(xv[e + 2 * u], xv[e + 2 * u + 1]), neg_sl2, ls[u]);
              if (DIST) {
                const float at = dist0 - static_cast<float>(e + 2 * u);
                z = fma_f32x2(pack_f32x2(fabsf(at), fabsf(at - 1.f)), pack_f32x2(slope2, slope2), z);
              }
              float2 zz = unpack_f32x2(z);
              if (CAP && kind == 1) {    // (other scores are made -inf before)
                zz.x = static_cast<unsigned>(e + 2 * u - a) < width ? zz.x : INFINITY;
                zz.y = static_cast<unsigned>(e + 2 * u + 1 - a) < width ? zz.y : INFINITY;
              }
              const float p0 = fast_exp2(-zz.x), p1 = fast_exp2(-zz.y);
              const uint64_t dy = fma_f32x2(dv[u], neg_one, pack_u32x2(yv[e + 2 * u], yv[e + 2 * u + 1]));
              uint64_t d2 = mul_f32x2(pack_f32x2(p0, p1), dy);
              if (CAP) d2 = mul_f32x2(d2, fma_f32x2(mul_f32x2(r[u], neg_one), r[u], r[u]));   // its 4: in the result's scale
              const float2 d = unpack_f32x2(d2);
              if (MODE == 0) pp[(e >> 1) + u] = pack_bf16x2(p0, p1);
              dd[(e >> 1) + u] = pack_bf16x2(d.x, d.y);
            }
          }
        }
        // columns of this row -> 16 packed columns of the P / dS tensor-memory tiles
        if (!OVERLAY) {
          mbar_wait(&m_empty[group], par ^ 1u, wctx, STATUS_TIMEOUT_SOFTMAX);
          tc_fence_after();
        }
        if (MODE == 0) tmem_st_32x16(p_addr, pp);
        tmem_st_32x16(ds_addr, dd);
        if (acc_pending) {   // before the arrival that lets the next phase of acc_full complete
          mbar_wait(acc_full, (it - 1) & 1, wctx, STATUS_TIMEOUT_TMEM_FULL);
          acc_pending = false;
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m_full[group]);
      }
      g0 += n;
      // Epilogue: accumulators -> global. dK / dV: one group of warps each, a half of the columns per warp.
      // dQ: a quarter of the columns per warp at head_dim 128; at head_dim 64 the group that does not own
      // the next item's first tile does it all and the other one goes on.
      if (EPI_WARPS != MBWD_CW && group == (g0 & 1)) {
        acc_pending = true;
        continue;
      }
      constexpr int NC = (MODE == 0) ? D / 64 : 1;    // 32-column chunks per warp
      const int c0 = (MODE == 0) ? half * (D / 2) : (D == 128 ? group * 64 + half * 32 : half * 32);
      const bool is_dv = MODE == 0 && group == 1;
      const float out_scale = is_dv ? 1.f : (CAP ? 4.f : 1.f) * p.scale;
      const uint32_t acc = tmem_base + lane_base + (MODE == 0 && !is_dv ? ACC2 : ACC1);
#pragma unroll
      for (int ci = 0; ci < NC; ++ci) {
        const int c = c0 + 32 * ci;
        if (ci == 0) {
          mbar_wait(acc_full, it & 1, wctx, STATUS_TIMEOUT_TMEM_FULL);
          tc_fence_after();
        }
        uint32_t v[32], wv[16];
        tmem_ld_32x32(acc + c, v);
        tmem_ld_wait_for(v);
        if (ci == NC - 1) {      // the accumulators may be overwritten by the next item
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(acc_empty);
        }
        if (item.padded != 0 && lo >= hi) {    // padding: zeros, whatever its own rows held
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0u;
        }
        if (MODE == 0 && p.parts > 1) {
          // fp32, one part of the sum: 16 columns at a time, the width of a staged row
          float* to = p.partial + (((static_cast<size_t>(item.part) * 2 + is_dv) * p.B + b) * (p.nh / p.group) + h) * p.S_pad * D +
                      static_cast<size_t>(row0) * D + c;
#pragma unroll
          for (int c2 = 0; c2 < 2; ++c2) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              wv[e] = __float_as_uint(__uint_as_float(v[16 * c2 + e]) * out_scale);
            store_rows_32x32(stage, wv, lane, reinterpret_cast<__nv_bfloat16*>(to + 16 * c2), 2 * D, p.S - row0);
          }
        } else {
          const uint64_t scale2 = pack_f32x2(out_scale, out_scale);
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            const float2 o = unpack_f32x2(mul_f32x2(pack_u32x2(v[2 * e], v[2 * e + 1]), scale2));
            wv[e] = pack_bf16x2(o.x, o.y);
          }
          if (lane == 0) bulk_wait_read_all();       // what was staged there has left
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((i ^ ((lane >> 1) & 3)) << 4)) =
                make_uint4(wv[4 * i], wv[4 * i + 1], wv[4 * i + 2], wv[4 * i + 3]);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && row0 < p.S) {             // (rows past the last token are cut off)
            tma_store_4d(is_dv ? &to2 : &to1, stage, c, row0, h, b);
            bulk_commit();
          }
        }
      }
    }
  }

  if (warp >= MBWD_FIRST_CW && lane == 0) bulk_wait_all();
  if (MODE == 1) pdl_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem_base, TMEM_COLS);
}

// dK and dV from the parts' sums, added in their order. D / 8 threads per row of [B, nkv, S].
__global__ void __launch_bounds__(256)
masked_dkv_kernel(const float* partial, int parts, __nv_bfloat16* __restrict__ dk, __nv_bfloat16* __restrict__ dv, int S,
                  int S_pad, int B, int nkv, int D, long long k_ss, long long k_bs, long long k_hs, long long v_ss,
                  long long v_bs, long long v_hs) {
  pdl_wait();
  pdl_trigger();
  const int tpr = D >> 3;
  const size_t n = static_cast<size_t>(B) * nkv * S_pad * D;     // elements of one tensor of one part
  const unsigned total = 2u * B * nkv * S;
  for (unsigned row = blockIdx.x * (256 / tpr) + threadIdx.x / tpr; row < total; row += gridDim.x * (256 / tpr)) {
    const int c = (threadIdx.x % tpr) * 8;
    const unsigned is_dv = row >= total / 2;
    const unsigned r = row - is_dv * (total / 2);
    const unsigned s = r % S, bh = r / S;
    const float* from = partial + is_dv * n + (static_cast<size_t>(bh) * S_pad + s) * D + c;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f), z = a;
    for (int i = 0; i < parts; ++i) {
      const float4 x = *reinterpret_cast<const float4*>(from + 2 * n * i), y = *reinterpret_cast<const float4*>(from + 2 * n * i + 4);
      a.x += x.x; a.y += x.y; a.z += x.z; a.w += x.w;
      z.x += y.x; z.y += y.y; z.z += y.z; z.w += y.w;
    }
    const unsigned b = bh / nkv, h = bh % nkv;
    __nv_bfloat16* to = is_dv ? dv + s * v_ss + b * v_bs + h * v_hs : dk + s * k_ss + b * k_bs + h * k_hs;
    *reinterpret_cast<uint4*>(to + c) = make_uint4(pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(z.x, z.y),
                                                   pack_bf16x2(z.z, z.w));
  }
}

// Into how many parts the heads of a group are dealt for dK and dV: until there is an item for every SM. Parts cost a pass over
// fp32 sums; with more items than SMs the uneven end of this kernel is filled by dQ's, which starts beside it. us, forward
// and backward, causal, 1 part -> 2 -> 4: [1, 32 heads (4), 2048, 128] (64 items) 333 -> ... -> 197, [1, 16 (1), 8192, 128] (64) 2511 -> ... ->
// 1134, [1, 32 (4), 4096, 128] (128) 743 -> 612 -> 631, [1, 32 (8), 2048, 128] (128) 202 -> 202 -> 218; 256 items, [1, 32 (4), 8192, 128] 2205 ->
// 2316 -> 2331, in documents [1, 16 (4), 8192, 128] 365 -> 395 -> 430.
int group_parts(int tiles, int B, int nkv, int group) {
  int parts = 1;
  while (parts < 4 && group % (2 * parts) == 0 && static_cast<long long>(tiles) * B * nkv * parts < gfs_host::sm_count())
    parts *= 2;
  return tiles > 1 ? parts : 1;
}

struct BwdMaps {
  const CUtensorMap *q128, *k128, *v128, *do128, *q64, *k64, *v64, *do64, *dq, *dk, *dv;
};

template <int D, bool CAP, bool DIST>
int launch_bwd(const BwdMaps& m, const MaskedBwdParams& p0, const MaskedBwdParams& p1, cudaStream_t stream) {
  static gfs_host::SmemLimit limit0, limit1;
  const int n_rt = p0.S_pad / 128;
  const int items0 = n_rt * p0.B * (p0.nh / p0.group) * p0.parts, items1 = n_rt * p0.B * p0.nh;
  constexpr int smem0 = MBwdShape<D, 0>::SMEM, smem1 = MBwdShape<D, 1>::SMEM;
  if (!limit0.raise(masked_bwd_kernel<D, 0, CAP, DIST>, smem0) || !limit1.raise(masked_bwd_kernel<D, 1, CAP, DIST>, smem1))
    return -10;
  gfs_host::launch_pdl(masked_bwd_kernel<D, 0, CAP, DIST>, dim3(items0), dim3(MBWD_THREADS), smem0, stream, *m.k128,
                       *m.v128, *m.q64, *m.do64, *m.dk, *m.dv, p0, n_rt);
  if (cudaGetLastError() != cudaSuccess) return -12;
  gfs_host::launch_pdl(masked_bwd_kernel<D, 1, CAP, DIST>, dim3(items1), dim3(MBWD_THREADS), smem1, stream, *m.q128,
                       *m.do128, *m.k64, *m.v64, *m.dq, *m.dq, p1, n_rt);
  return cudaGetLastError() == cudaSuccess ? 0 : -13;
}
template <int D>
int launch_bwd_scores(const BwdMaps& m, const MaskedBwdParams& p0, const MaskedBwdParams& p1, bool cap, cudaStream_t s) {
  const bool dist = p0.score.slopes != nullptr;
  if (cap) return dist ? launch_bwd<D, true, true>(m, p0, p1, s) : launch_bwd<D, true, false>(m, p0, p1, s);
  return dist ? launch_bwd<D, false, true>(m, p0, p1, s) : launch_bwd<D, false, false>(m, p0, p1, s);
}

}  // namespace

extern "C" {

// fp32 elements of the scratch `partial` of the backward (0: none)
long long gfs_masked_attention_scratch(int S, int B, int nh, int nkv, int D) {
  if (S <= 0 || B <= 0 || nh <= 0 || nkv <= 0) return 0;
  const int tiles = (S + 127) / 128;
  const int parts = group_parts(tiles, B, nkv, nh / nkv);
  return parts > 1 ? 2ll * parts * B * nkv * tiles * 128 * D : 0;
}

// strides: 24 element strides for {q, k, v, out, dout, dq, dk, dv} x {seq, batch, head}; lse (from the forward) and dvec
// (scratch): fp32 [B, nh, S_pad]; partial: partial_floats of scratch, the size above on the same device or more (fewer are
// refused: the parts depend on its SMs); the rest as for gfs_masked_attention_fwd. dq shares no memory with anything that is read
// for dk and dv, nor with them: its kernel runs beside theirs.
int gfs_masked_attention_bwd(const void* q, const void* k, const void* v, const void* out, const void* dout,
                             const void* saved, void* dvec, void* partial, long long partial_floats, void* dq, void* dk,
                             void* dv, const void* mask, int S, int B, int nh, int nkv, int D, const long long* strides,
                             float scale, float cap, const void* slopes, void* stream_) {
  if ((D != 64 && D != 128) || !strides_ok(strides, 24) || nkv <= 0 || nh % nkv != 0) return -1;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
       reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(dout) | reinterpret_cast<uintptr_t>(dq) |
       reinterpret_cast<uintptr_t>(dk) | reinterpret_cast<uintptr_t>(dv) | reinterpret_cast<uintptr_t>(saved)) & 15)
    return -2;
  if (S <= 0 || B <= 0 || nh <= 0) return 0;
  const int S_pad = (S + 127) / 128 * 128;
  if (static_cast<long long>(S_pad) * nh > 0x3fffffffll || B > 65535) return -1;   // 32-bit row numbers in the pre-pass
  if (static_cast<long long>(S_pad / 128) * B * nh > 0x7fffffffll) return -1;
  if (saved == nullptr || dvec == nullptr || mask == nullptr) return -2;
  const long long scratch = gfs_masked_attention_scratch(S, B, nh, nkv, D);
  if (scratch > 0 && (partial == nullptr || reinterpret_cast<uintptr_t>(partial) & 15 || partial_floats < scratch)) return -4;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const long long *sq = strides, *sk = strides + 3, *sv = strides + 6, *so = strides + 9, *sdo = strides + 12,
                  *sdq = strides + 15, *sdk = strides + 18, *sdv = strides + 21;
  MaskedBwdParams p = {};
  p.mask = mask_view(mask, B, S);
  {
    const int s_fastest = so[0] < so[2] ? 1 : 0;
    const unsigned inner = s_fastest ? S_pad : nh, rows = static_cast<unsigned>(S_pad) * nh;
    const unsigned per_block = 32 * dvec_rows(D);
    const DvecArgs a{static_cast<const __nv_bfloat16*>(dout), static_cast<const __nv_bfloat16*>(out),
                     static_cast<const uint8_t*>(saved) + 4 * static_cast<size_t>(B) * nh * S_pad, static_cast<float*>(dvec),
                     p.mask.first, p.mask.last, p.mask.padded, S, S_pad, nh, sdo[0], sdo[1], sdo[2], so[0], so[1], so[2], inner,
                     rows + per_block < (1u << 24) && inner <= (1u << 16) ? (1ull << 40) / inner + 1 : 0ull, s_fastest};
    const dim3 grid((rows + per_block - 1) / per_block, B);
    gfs_host::launch_pdl(D == 64 ? masked_dvec_kernel<64> : masked_dvec_kernel<128>, grid, dim3(256), 0, stream, a);
    if (cudaGetLastError() != cudaSuccess) return -11;
  }
  const BwdMaps maps{make_map(q, D, S, nh, B, sq, 128), make_map(k, D, S, nkv, B, sk, 128),
                     make_map(v, D, S, nkv, B, sv, 128), make_map(dout, D, S, nh, B, sdo, 128),
                     make_map(q, D, S, nh, B, sq, 64), make_map(k, D, S, nkv, B, sk, 64),
                     make_map(v, D, S, nkv, B, sv, 64), make_map(dout, D, S, nh, B, sdo, 64),
                     make_map(dq, D, S, nh, B, sdq, 32, 32), make_map(dk, D, S, nkv, B, sdk, 32, 32),
                     make_map(dv, D, S, nkv, B, sdv, 32, 32)};
  if (!maps.q128 || !maps.k128 || !maps.v128 || !maps.do128 || !maps.q64 || !maps.k64 || !maps.v64 || !maps.do64 ||
      !maps.dq || !maps.dk || !maps.dv)
    return -3;
  p.lse = static_cast<const float*>(saved);
  p.dvec = static_cast<const float*>(dvec);
  p.S = S; p.S_pad = S_pad; p.B = B; p.nh = nh; p.group = nh / nkv; p.scale = scale;
  p.score.sl2 = cap > 0.f ? 2.f * scale * LOG2E_F / cap : scale * LOG2E_F;
  p.score.cap2 = cap * LOG2E_F;
  p.score.slopes = static_cast<const float*>(slopes);
  p.status = gfs_host::status_words();
  p.parts = 1;
  MaskedBwdParams p0 = p;
  p0.parts = group_parts(S_pad / 128, B, nkv, nh / nkv);
  p0.partial = static_cast<float*>(partial);
  const int rc = D == 64 ? launch_bwd_scores<64>(maps, p0, p, cap > 0.f, stream)
                         : launch_bwd_scores<128>(maps, p0, p, cap > 0.f, stream);
  if (rc != 0 || p0.parts == 1) return rc;
  const long long rows = 2ll * B * nkv * S;
  const int rows_per_block = 256 / (D >> 3);
  const dim3 grid(static_cast<unsigned>(std::min<long long>((rows + rows_per_block - 1) / rows_per_block, gfs_host::sm_count() * 32)));
  gfs_host::launch_pdl(masked_dkv_kernel, grid, dim3(256), 0, stream, static_cast<const float*>(partial), p0.parts,
                       static_cast<__nv_bfloat16*>(dk), static_cast<__nv_bfloat16*>(dv), S, S_pad, B, nkv, D, sdk[0], sdk[1],
                       sdk[2], sdv[0], sdv[1], sdv[2]);
  return cudaGetLastError() == cudaSuccess ? 0 : -14;
}

}  // extern "C"
