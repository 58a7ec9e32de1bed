// The mask and the scores of masked attention (masked_attention.cu, masked_attention_bwd.cu).
//
// Every query sees one range of keys, [first, last), and both ends grow or stay from query to query of a sequence:
// documents, a prefix, a window and padding all have that form. So the queries that see a key are a range too, the ends of a tile's
// first and last row bound the whole tile, and a block of scores is skipped, masked or taken whole by comparing numbers.
#pragma once
#include <stdint.h>

#include "common.cuh"

namespace gfs {

// What gfs_attention_mask writes; int32, S_pad = S rounded up to a multiple of 128. A token whose two ranges are empty is
// padding: it sees nothing and nothing sees it, and what its rows of q, k, v and the gradients hold does not matter.
// Rows S .. S_pad are empty.
struct MaskView {
  const int *first, *last;     // [B, S_pad]: the keys that a query sees
  const int *qfirst, *qlast;   // [B, S_pad]: the queries that see a key
  const int4 *plan_q, *plan_k; // [B, S_pad / 128]: the tiles of 128 queries (keys), those that see (are seen by) most first
  const int4* pairs;           // [B, ceil(S_pad / 256), 2]: the same for pairs of query tiles
  const int* padded;           // [B]: the sequence has padding
};
// An entry of a plan: {tile, the first row that any of its rows sees (for keys: is seen by), one past the last, padded}.
// Of the pairs: {pair, blocks [a0, a1) of 64 keys of its first tile, b0}, {b1 of its second tile, padded, 0, 0}; the blocks of both
// are one stretch without a gap, at least one each; b0 == b1: there is no second tile.

// The parts of the buffer that gfs_attention_mask fills: int32 offsets.
struct MaskLayout {
  size_t first, last, qfirst, qlast, plan_q, plan_k, pairs, padded, positions, end;
};
__host__ __device__ inline MaskLayout mask_layout(int B, int S) {
  const size_t S_pad = (static_cast<size_t>(S) + 127) / 128 * 128;
  const size_t n = B * S_pad, plan = B * (S_pad / 128) * 4;
  MaskLayout l;
  l.first = 0;
  l.last = n;
  l.qfirst = 2 * n;
  l.qlast = 3 * n;
  l.plan_q = 4 * n;
  l.plan_k = l.plan_q + plan;
  l.pairs = l.plan_k + plan;
  l.positions = l.pairs + B * ((S_pad / 128 + 1) / 2) * 8;
  l.padded = l.positions + static_cast<size_t>(B) * S;
  l.end = l.padded + B;
  return l;
}
inline MaskView mask_view(const void* buffer, int B, int S) {
  const int* m = static_cast<const int*>(buffer);
  const MaskLayout l = mask_layout(B, S);
  return MaskView{m + l.first, m + l.last, m + l.qfirst, m + l.qlast, reinterpret_cast<const int4*>(m + l.plan_q),
                  reinterpret_cast<const int4*>(m + l.plan_k), reinterpret_cast<const int4*>(m + l.pairs), m + l.padded};
}

// The softmax's exponents are base 2: score = log2(e) (scale q k, or cap tanh(scale q k / cap)) - slope log2(e) |i - j|.
struct ScoreArgs {
  float sl2;            // scale log2(e); capped: 2 scale log2(e) / cap, so that tanh(..) = 1 - 2 / (1 + 2^(sl2 q k))
  float cap2;           // cap log2(e)
  const float* slopes;  // [heads], or null
};

__device__ __forceinline__ float min_nan(float a, float b) {
  float d;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// r = 1 / (1 + 2^(sl2 x)) of four scores, as two pairs: tanh = 1 - 2 r, its derivative 4 r (1 - r). The absolute error counts
// here (the score is an exponent), and it is that of r, a few 2^-24: the approximate tanh instruction is off by up to
// 2^-11 of the value, 0.02 for a score of 40. Four exponentials and one reciprocal, of the product of the four denominators: it
// stays in range as exponents are cut off at 30, where tanh is 1 to 32 bits. In pairs (one instruction of the FMA pipe for
// two scores) 5 instructions a score.
__device__ __forceinline__ void sigmoids(uint64_t x0, uint64_t x1, uint64_t sl2, uint64_t& r0, uint64_t& r1) {
  const float2 u0 = unpack_f32x2(mul_f32x2(x0, sl2)), u1 = unpack_f32x2(mul_f32x2(x1, sl2));
  const uint64_t one = pack_f32x2(1.f, 1.f);
  const uint64_t d0 = add_f32x2(pack_f32x2(fast_exp2(min_nan(u0.x, 30.f)), fast_exp2(min_nan(u0.y, 30.f))), one);
  const uint64_t d1 = add_f32x2(pack_f32x2(fast_exp2(min_nan(u1.x, 30.f)), fast_exp2(min_nan(u1.y, 30.f))), one);
  const float2 pr = unpack_f32x2(mul_f32x2(d0, d1));
  const float inv = fast_rcp(pr.x * pr.y);
  const uint64_t q = pack_f32x2(inv * pr.y, inv * pr.x);      // 1 / (d0 d1), elementwise
  r0 = mul_f32x2(q, d1);
  r1 = mul_f32x2(q, d0);
}

// What the rounding of outputs to bf16 leaves out, for the backward: dvec = sum dO O takes the place of sum P dP there, and in rows
// that see a few keys, whose P (dP - dvec) is small against both, half a step of O (up to 2^-8) is more than all else that is rounded:
// errors of dQ and dK are 2.7 to 3.2e-3 with it and 2.4 to 2.5e-3 without, in documents of 4 to 100 tokens up to 5.5e-3 and 2.5 to 3.4e-3.
// A signed byte per number, the next eight bits of its pattern as the difference from the rounded one (patterns grow with magnitudes, so
// exponents and signs do not matter); it leaves 2^-15. Costs: half of O written and read once more, 4 to 5 % of a training call.
__device__ __forceinline__ uint32_t bf16_rest(const float (&o)[4], uint32_t r01, uint32_t r23) {
  const uint32_t r[4] = {r01 << 16, r01 & 0xffff0000u, r23 << 16, r23 & 0xffff0000u};
  int left[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) left[e] = static_cast<int>(__float_as_uint(o[e]) - r[e] + 128u) >> 8;
  uint32_t upper, packed;       // saturating: half a step up is 128 (and of a NaN any byte does)
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(upper) : "r"(left[3]), "r"(left[2]));
  asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(packed) : "r"(left[1]), "r"(left[0]), "r"(upper));
  return packed;
}
__device__ __forceinline__ void st_global_256(void* at, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
// Two bf16 with the bytes `at` and `at` + 1 of four of those
__device__ __forceinline__ float2 with_rest(uint32_t rounded, uint32_t rest, int at) {
  const int lo = static_cast<int>(rest << (24 - 8 * at)) >> 24, hi = static_cast<int>(rest << (16 - 8 * at)) >> 24;
  return make_float2(__uint_as_float((rounded << 16) + (static_cast<uint32_t>(lo) << 8)),
                     __uint_as_float((rounded & 0xffff0000u) + (static_cast<uint32_t>(hi) << 8)));
}

// Zeros in the rows of a tile (swizzled blocks of 64 columns, `rows` rows of 128 bytes, `blocks` of them block_bytes apart) whose
// tokens are padding: their probabilities are 0, but 0 times what they hold might not be. The whole warp.
__device__ __forceinline__ void zero_padding(uint8_t* tile, int rows, int blocks, int block_bytes, const int* first,
                                             const int* last, int lane) {
  for (int r0 = 0; r0 < rows; r0 += 32) {
    unsigned dead = __ballot_sync(0xffffffffu, first[r0 + lane] >= last[r0 + lane]);
    while (dead != 0u) {
      const int r = r0 + __ffs(dead) - 1;
      dead &= dead - 1;
      for (int c = lane; c < blocks * 8; c += 32)
        *reinterpret_cast<uint4*>(tile + (c >> 3) * block_bytes + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
  }
  fence_proxy_async_smem();
  __syncwarp();
}

}  // namespace gfs
