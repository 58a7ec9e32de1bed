// What the attention kernels share: matrix products of tiles in shared and tensor memory, epilogue stores, tensor maps
// of strided [B, heads, S, D] tensors.
#pragma once
#include "common.cuh"

namespace gfs {

constexpr float LOG2E_F = 1.4426950408889634f;

// three-input maximum (one instruction on sm_100)
__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A K-major [rows x K] (64-column blocks a_blk bytes apart), B K-major [N x K] (blocks b_blk apart).
// The shared-memory descriptors are built once per call and advanced by adding the byte offset
// (in 16-byte units) to their start-address field: the tiles are 1024-byte aligned and the
// offsets small, so the 14-bit field never carries. The issuing thread competes with the
// compute warps for issue slots, so every instruction saved per MMA shortens the chain.
template <int KSTEPS>
__device__ __forceinline__ void mma_kk(uint32_t d, uint32_t a, uint32_t a_blk, uint32_t b, uint32_t b_blk,
                                       uint32_t idesc, bool accumulate) {
  const uint64_t ad0 = umma_desc_sw128(a, 16, 1024);
  const uint64_t bd0 = umma_desc_sw128(b, 16, 1024);
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) {
    const uint64_t ad = ad0 + (((ks >> 2) * a_blk + (ks & 3) * 32) >> 4);
    const uint64_t bd = bd0 + (((ks >> 2) * b_blk + (ks & 3) * 32) >> 4);
    umma_ss_e(d, ad, bd, idesc, (accumulate || ks > 0) ? 1u : 0u);
  }
}
// A K-major; B MN-major: stored as [K rows x N] in 64-column blocks b_blk bytes apart
// (each block: K rows of 128 B).
template <int KSTEPS>
__device__ __forceinline__ void mma_kmn(uint32_t d, uint32_t a, uint32_t a_blk, uint32_t b, uint32_t b_blk,
                                        uint32_t idesc, bool accumulate) {
  const uint64_t ad0 = umma_desc_sw128(a, 16, 1024);
  const uint64_t bd0 = umma_desc_sw128(b, b_blk, 1024);
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) {
    const uint64_t ad = ad0 + (((ks >> 2) * a_blk + (ks & 3) * 32) >> 4);
    const uint64_t bd = bd0 + ((ks * 2048) >> 4);
    umma_ss_e(d, ad, bd, idesc, (accumulate || ks > 0) ? 1u : 0u);
  }
}

// A in tensor memory (8 columns per 16-wide K step; the second half of the K steps starts HALF columns
// after the first); B MN-major as in mma_kmn.
template <int KSTEPS, int HALF = KSTEPS * 4>
__device__ __forceinline__ void mma_tmn(uint32_t d, uint32_t a_tmem, uint32_t b, uint32_t b_blk, uint32_t idesc,
                                        bool accumulate) {
  const uint64_t bd0 = umma_desc_sw128(b, b_blk, 1024);
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ++ks) {
    const uint64_t bd = bd0 + ((ks * 2048) >> 4);
    const uint32_t a = a_tmem + (ks / (KSTEPS / 2)) * HALF + (ks % (KSTEPS / 2)) * 8;
    umma_ts_e(d, a, bd, idesc, (accumulate || ks > 0) ? 1u : 0u);
  }
}

// ---------------------------------------------------------------------------
// Epilogue stores. An accumulator row lives in one thread, so a direct store instruction writes 16
// bytes to each of 32 different rows: 32 passes through the load/store unit per instruction, which
// made the epilogues of these kernels LSU-bound (about 1,000 cycles per 128 x 64 output tile). The
// rows are therefore transposed through a per-warp staging area in shared memory (XOR-swizzled, free
// of bank conflicts both ways) and leave as whole 64- or 128-byte row segments.
// ---------------------------------------------------------------------------
// 32 rows x 32 bf16 columns; w = this lane's row (16 packed words); stage: 2 KB of this warp.
__device__ __forceinline__ void store_rows_32x32(uint8_t* stage, const uint32_t (&w)[16], int lane,
                                                 __nv_bfloat16* g0, long long row_stride, int rows_valid) {
#pragma unroll
  for (int q4 = 0; q4 < 4; ++q4)
    *reinterpret_cast<uint4*>(stage + lane * 64 + ((q4 ^ ((lane >> 1) & 3)) << 4)) =
        make_uint4(w[4 * q4], w[4 * q4 + 1], w[4 * q4 + 2], w[4 * q4 + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = (lane >> 2) + 8 * i;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + row * 64 + (((lane & 3) ^ ((row >> 1) & 3)) << 4));
    if (row < rows_valid) *reinterpret_cast<uint4*>(g0 + row * row_stride + (lane & 3) * 8) = v;
  }
  __syncwarp();
}

// 32 rows x 64 bf16 columns; w = this lane's row (32 packed words); stage: 4 KB of this warp.
__device__ __forceinline__ void store_rows_32x64(uint8_t* stage, const uint32_t (&w)[32], int lane,
                                                 __nv_bfloat16* g0, long long row_stride, int rows_valid) {
#pragma unroll
  for (int ch = 0; ch < 8; ++ch)
    *reinterpret_cast<uint4*>(stage + lane * 128 + ((ch ^ (lane & 7)) << 4)) =
        make_uint4(w[4 * ch], w[4 * ch + 1], w[4 * ch + 2], w[4 * ch + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = (lane >> 3) + 4 * i;
    const uint4 v = *reinterpret_cast<const uint4*>(stage + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
    if (row < rows_valid) *reinterpret_cast<uint4*>(g0 + row * row_stride + (lane & 7) * 8) = v;
  }
  __syncwarp();
}

}  // namespace gfs

namespace gfs_host {

inline const CUtensorMap* make_map(const void* base, int D, int S, int nh, int B, const long long* st, uint32_t box_rows,
                                  uint32_t box_cols = 64) {
  // st = {seq, batch, head} element strides
  uint64_t dims[4] = {static_cast<uint64_t>(D), static_cast<uint64_t>(S), static_cast<uint64_t>(nh),
                      static_cast<uint64_t>(B)};
  uint64_t strides[4] = {2, static_cast<uint64_t>(st[0]) * 2, static_cast<uint64_t>(st[2]) * 2,
                         static_cast<uint64_t>(st[1]) * 2};
  uint32_t box[4] = {box_cols, box_rows, 1, 1};
  return tmap_nd_cached(base, 4, dims, strides, box);
}

inline bool strides_ok(const long long* st, int n) {
  for (int i = 0; i < n; ++i)
    if (st[i] & 7) return false;
  return true;
}

}  // namespace gfs_host
