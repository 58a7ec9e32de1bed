// Rotary positions in general form, alone or after a norm of every head of q and k.
//
//   rotation    (a, b) -> (a cos - b sin, a sin + b cos) for the R / 2 pairs of a head's first R dimensions: pairs
//               side by side (2i, 2i + 1) or half of R apart (i, i + R / 2); the other D - R dimensions stay.
//               cos and sin: rows of an fp32 table, row s or positions[b][s] for the token (s, b).
//   norm        n = x / sqrt(mean(x^2) + eps) over a head's D dimensions, z = n w, then the rotation of z
//   backward    dz = the transposed rotation of dy (sin -> -sin), dw = sum over tokens and heads of dz n,
//               dx = rstd (dz w - n mean(dz w n))
//
// Everything between the load of an element and its store is fp32, rounded once.
//
// An element is read once and written once, so memory is the floor; about ten instructions an element come close to the issue
// rate (0.68 of it in the norm's forward), which is why numbers are converted in pairs and norms computed in pairs of fp32.
// us, and GB/s: rotation of 64 of 128 dimensions of 16 heads of 8192 tokens, bf16, 13 (5,100); norm and rotation of 24 heads of
// 16384 tokens, head_dim 64, bf16, forward 22 (4,600), backward 45 (4,450); of 40 heads of 8192 tokens, head_dim 128, fp16, 34 (4,900)
// and 64 (4,400). Two backward blocks of 128 registers an SM with four steps of loads each (three blocks and three steps 60 for 45, two steps
// 70), a token's chunks in one warp's loop 54.
//
// A row (the head of a token) belongs to a group of 8, 16 or 32 lanes, eight elements each (one 16-byte load of a 16-bit type); a
// partner half a head away is in another lane of the group, and the norm's sums stay in it. A group takes a few rows
// of one token, so that the table's entries are loaded once for them and the loads of all rows are in flight together.
// What no 16-byte access can reach (odd strides or addresses, head sizes no multiple of 8), and rotated dimensions whose halves or
// pairs would part a lane's eight elements (no multiple of 16, or of 8 in pairs), go to kernels that give a row a warp, an
// element at a time: right for everything, and far from memory's rate. us (beside them the 16-byte path's): 16 heads of 8192 tokens,
// bf16, 40 of 80 halves apart 41 (all 80: 16), 24 of 96 47 (18); with norms and k's heads 100 (31), with the backward 496 (88).
#include <cuda_fp16.h>

#include <algorithm>

#include "api.h"
#include "common.cuh"

using namespace gfs;

namespace {

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// Eight elements as they lie in memory.
template <typename T>
struct alignas(16) Vec8 {
  T v[8];
};
template <typename T>
__device__ __forceinline__ Vec8<T> load_vec(const T* p) {
  Vec8<T> r;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(Vec8<T>) / 16); ++i)
    reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
  return r;
}
// pairs of 16-bit numbers at a time: one conversion instruction for two
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __nv_bfloat16) { return pack_bf16x2(lo, hi); }
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, __half) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack_pair(uint32_t u, __nv_bfloat16) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack_pair(uint32_t u, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = make_uint4(pack_pair(f[0], f[1], T()), pack_pair(f[2], f[3], T()), pack_pair(f[4], f[5], T()),
                                              pack_pair(f[6], f[7], T()));
  } else {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
}
template <typename T>
__device__ __forceinline__ void to_floats(const Vec8<T>& x, float (&f)[8]) {
  if constexpr (sizeof(T) == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(&x);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 v = unpack_pair(w[e], T());
      f[2 * e] = v.x;
      f[2 * e + 1] = v.y;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = to_f32(x.v[e]);
  }
}

// A tensor [S, B, heads, D], its dimensions contiguous.
struct Part {
  void* p;
  long long ss, bs, hs;   // element strides: sequence, batch, head
  __device__ long long at(int s, int b, int h) const { return s * ss + b * bs + h * hs; }
};

struct RotaryArgs {
  Part x;                 // heads [0, n1) are q's, [n1, n1 + n2) k's, then (backward) n2 of v
  Part y1, y2, y3;        // forward: where q and k go; backward: their gradients, and v's
  Part dx;                // backward: the gradient of x
  const void *w1, *w2;    // norm weights of q and k (null: no norm)
  float* dw;              // backward: fp32 [blocks][2][D]
  const float *cos, *sin;  // [rows, R / 2]
  const void* positions;  // [B, S] or null
  int pos64, rows;
  int S, B, n1, n2, n3, D, R;
  int inverse;            // rotate the other way
  float eps, inv_D;
  uint32_t* status;
};

// Row of the table for the token (s, b). One outside of it is reported and taken from the border.
__device__ __forceinline__ int table_row(const RotaryArgs& a, int s, int b) {
  if (a.positions == nullptr) return s;
  const size_t at = static_cast<size_t>(b) * a.S + s;
  const long long p = a.pos64 ? static_cast<const long long*>(a.positions)[at] : static_cast<const int*>(a.positions)[at];
  if (p < 0 || p >= a.rows) {
    record_status(a.status, STATUS_BAD_ARGUMENT, 0xf05u);
    return p < 0 ? 0 : a.rows - 1;
  }
  return static_cast<int>(p);
}

// The table's entries for a lane's eight elements: four pairs side by side, or eight elements of one half.
template <bool HALF>
struct Turn {
  float c[HALF ? 8 : 4], s[HALF ? 8 : 4];
};
template <bool HALF>
__device__ __forceinline__ Turn<HALF> load_turn(const RotaryArgs& a, int row, int e0) {
  Turn<HALF> t;
  constexpr int N = HALF ? 8 : 4;
  if (e0 >= a.R) {
#pragma unroll
    for (int i = 0; i < N; ++i) t.c[i] = t.s[i] = 0.f;
    return t;
  }
  const int half = a.R >> 1;
  const int col = HALF ? (e0 < half ? e0 : e0 - half) : e0 >> 1;
  const size_t at = static_cast<size_t>(row) * half + col;
#pragma unroll
  for (int i = 0; i < N; i += 4) {
    const float4 c = *reinterpret_cast<const float4*>(a.cos + at + i);
    const float4 s = *reinterpret_cast<const float4*>(a.sin + at + i);
    t.c[i] = c.x; t.c[i + 1] = c.y; t.c[i + 2] = c.z; t.c[i + 3] = c.w;
    t.s[i] = s.x; t.s[i + 1] = s.y; t.s[i + 2] = s.z; t.s[i + 3] = s.w;
  }
  const bool flip = a.inverse != (HALF && e0 < half);   // an element of the first half gets minus its partner times sin
  if (flip) {
#pragma unroll
    for (int i = 0; i < N; ++i) t.s[i] = -t.s[i];
  }
  return t;
}
// All lanes of the warp call this (the partner half a head away is in another lane of the group).
template <bool HALF, int LANES>
__device__ __forceinline__ void rotate(float (&f)[8], const Turn<HALF>& t, int e0, int R) {
  if (HALF) {
    const int lane = (threadIdx.x & (LANES - 1));
    const int partner = e0 < R ? (e0 < (R >> 1) ? lane + (R >> 4) : lane - (R >> 4)) : lane;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float o = __shfl_sync(0xffffffffu, f[e], partner, LANES);
      if (e0 < R) f[e] = f[e] * t.c[HALF ? e : 0] + o * t.s[HALF ? e : 0];
    }
  } else if (e0 < R) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float x = f[2 * i], y = f[2 * i + 1];
      f[2 * i] = x * t.c[i] - y * t.s[i];
      f[2 * i + 1] = x * t.s[i] + y * t.c[i];
    }
  }
}
template <int LANES>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o, LANES);
  return v;
}

constexpr int ROT_THREADS = 256;
constexpr int ROT_WARPS = ROT_THREADS / 32;

// A work item is a warp's: up to STEPS * 32 / LANES heads of one kind (q's, k's or v's) of a token. In a step the groups of the
// warp have neighbouring heads, so a step's load is contiguous; all steps' loads are issued before the first is used.
template <int LANES, int STEPS>
struct Items {
  static constexpr int GROUPS = 32 / LANES;
  static constexpr int ROWS = GROUPS * STEPS;
  static constexpr int of(int heads) { return (heads + ROWS - 1) / ROWS; }
};
template <typename T>
constexpr int bwd_steps() { return sizeof(T) == 2 ? 4 : 2; }   // two inputs of up to 16 (32-bit types: 32) bytes a lane and step
constexpr int FWD_STEPS = 4;

// f32x2 lanes of a vector: eight elements as four pairs.
__device__ __forceinline__ void to_pairs(const float (&f)[8], uint64_t (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack_f32x2(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ float pair_sum(uint64_t v) {
  const float2 f = unpack_f32x2(v);
  return f.x + f.y;
}

// Forward (and the rotation's own backward).
template <typename T, int LANES, bool HALF, bool NORM>
__global__ void __launch_bounds__(ROT_THREADS)
rotary_kernel(const RotaryArgs a, unsigned n_items, unsigned items_per_token, int items_q) {
  pdl_wait();
  pdl_trigger();
  using I = Items<LANES, FWD_STEPS>;
  const unsigned item = blockIdx.x * ROT_WARPS + (threadIdx.x >> 5);
  if (item >= n_items) return;
  const int group = (threadIdx.x & 31) / LANES;
  const int e0 = (threadIdx.x & (LANES - 1)) * 8;
  const bool lane_on = e0 < a.D;
  const unsigned token = item / items_per_token;
  int c = static_cast<int>(item - token * items_per_token);
  const int s = static_cast<int>(token / a.B), b = static_cast<int>(token % a.B);
  const bool is_q = c < items_q;
  if (!is_q) c -= items_q;
  const int heads = is_q ? a.n1 : a.n2, h0 = c * I::ROWS + group;
  const T* x = static_cast<const T*>(a.x.p) + a.x.at(s, b, (is_q ? 0 : a.n1) + h0) + e0;
  Vec8<T> in[FWD_STEPS];
#pragma unroll
  for (int i = 0; i < FWD_STEPS; ++i)
    if (lane_on && h0 + i * I::GROUPS < heads) in[i] = load_vec(x + i * I::GROUPS * a.x.hs);
  uint64_t w[4];
  if (NORM) {
    float f[8] = {};
    if (lane_on) to_floats(load_vec(static_cast<const T*>(is_q ? a.w1 : a.w2) + e0), f);
    to_pairs(f, w);
  }
  Turn<HALF> t = {};
  if (lane_on) t = load_turn<HALF>(a, table_row(a, s, b), e0);
  const Part& out = is_q ? a.y1 : a.y2;
  T* y = static_cast<T*>(out.p) + out.at(s, b, h0) + e0;
#pragma unroll
  for (int i = 0; i < FWD_STEPS; ++i) {
    if (h0 - group + i * I::GROUPS >= heads) break;      // the whole warp is past the last head
    const bool on = lane_on && h0 + i * I::GROUPS < heads;
    float f[8] = {};
    if (on) to_floats(in[i], f);
    if (NORM) {
      uint64_t v[4], ss = 0;
      to_pairs(f, v);
#pragma unroll
      for (int e = 0; e < 4; ++e) ss = fma_f32x2(v[e], v[e], ss);
      const float rstd = rsqrtf(group_sum<LANES>(pair_sum(ss)) * a.inv_D + a.eps);
      const uint64_t r2 = pack_f32x2(rstd, rstd);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 z = unpack_f32x2(mul_f32x2(mul_f32x2(v[e], r2), w[e]));
        f[2 * e] = z.x;
        f[2 * e + 1] = z.y;
      }
    }
    rotate<HALF, LANES>(f, t, e0, a.R);
    if (on) store_vec(y + i * I::GROUPS * out.hs, f);
  }
}

// Backward of norm and rotation, of q's and k's heads; v's gradient is copied into its place. A grid of the warps that fit
// strides over the items; the weights' gradients stay in registers until the end: a sum per block, added up in a fixed
// order by qk_norm_dw_kernel.
template <typename T, int LANES, bool HALF, bool NORM>
__global__ void __launch_bounds__(ROT_THREADS, 2)
qk_norm_rope_bwd_kernel(const RotaryArgs a, unsigned n_items, unsigned items_per_token, int items_q, int items_k) {
  pdl_wait();
  pdl_trigger();
  constexpr int STEPS = bwd_steps<T>();
  using I = Items<LANES, STEPS>;
  const int group = (threadIdx.x & 31) / LANES;
  const int e0 = (threadIdx.x & (LANES - 1)) * 8;
  const bool lane_on = e0 < a.D;
  uint64_t dw1[4] = {}, dw2[4] = {};
  for (unsigned item = blockIdx.x * ROT_WARPS + (threadIdx.x >> 5); item < n_items; item += gridDim.x * ROT_WARPS) {
    const unsigned token = item / items_per_token;
    int c = static_cast<int>(item - token * items_per_token);
    const int s = static_cast<int>(token / a.B), b = static_cast<int>(token % a.B);
    const int kind = c < items_q ? 0 : (c < items_q + items_k ? 1 : 2);
    c -= kind == 0 ? 0 : (kind == 1 ? items_q : items_q + items_k);
    const int heads = kind == 0 ? a.n1 : (kind == 1 ? a.n2 : a.n3), h0 = c * I::ROWS + group;
    const int head0 = (kind == 0 ? 0 : (kind == 1 ? a.n1 : a.n1 + a.n2)) + h0;
    const Part& from = kind == 0 ? a.y1 : (kind == 1 ? a.y2 : a.y3);
    const T* g = static_cast<const T*>(from.p) + from.at(s, b, h0) + e0;
    const T* x = static_cast<const T*>(a.x.p) + a.x.at(s, b, head0) + e0;
    T* dx = static_cast<T*>(a.dx.p) + a.dx.at(s, b, head0) + e0;
    Vec8<T> gv[STEPS], xv[STEPS];
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (lane_on && h0 + i * I::GROUPS < heads) {
        gv[i] = load_vec(g + i * I::GROUPS * from.hs);
        if (NORM && kind != 2) xv[i] = load_vec(x + i * I::GROUPS * a.x.hs);
      }
    if (kind == 2) {
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
        if (lane_on && h0 + i * I::GROUPS < heads)
#pragma unroll
          for (int u = 0; u < static_cast<int>(sizeof(Vec8<T>) / 16); ++u)
            reinterpret_cast<uint4*>(dx + i * I::GROUPS * a.dx.hs)[u] = reinterpret_cast<const uint4*>(&gv[i])[u];
      continue;
    }
    uint64_t w[4], dw[4] = {};
    if (NORM) {
      float f[8] = {};
      if (lane_on) to_floats(load_vec(static_cast<const T*>(kind == 0 ? a.w1 : a.w2) + e0), f);
      to_pairs(f, w);
    }
    Turn<HALF> t = {};
    if (lane_on) t = load_turn<HALF>(a, table_row(a, s, b), e0);
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
      if (h0 - group + i * I::GROUPS >= heads) break;
      const bool on = lane_on && h0 + i * I::GROUPS < heads;
      float f[8] = {};
      if (on) to_floats(gv[i], f);
      rotate<HALF, LANES>(f, t, e0, a.R);
      if (NORM) {
        uint64_t dz[4], v[4], zw[4], ss = 0, dot = 0;
        to_pairs(f, dz);
        float xf[8] = {};
        if (on) to_floats(xv[i], xf);
        to_pairs(xf, v);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          zw[e] = mul_f32x2(dz[e], w[e]);
          ss = fma_f32x2(v[e], v[e], ss);
          dot = fma_f32x2(zw[e], v[e], dot);
        }
        // (groups past the last head hold zeros, whose factor without eps would be infinite)
        const float mean = group_sum<LANES>(pair_sum(ss)) * a.inv_D + a.eps;
        const float rstd = on ? rsqrtf(mean) : 0.f;
        const float m = group_sum<LANES>(pair_sum(dot)) * rstd * rstd * a.inv_D;      // mean(dz w n) rstd
        const uint64_t r2 = pack_f32x2(rstd, rstd), m2 = pack_f32x2(-m, -m);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t n = mul_f32x2(v[e], r2);
          dw[e] = fma_f32x2(dz[e], n, dw[e]);
          const float2 o = unpack_f32x2(fma_f32x2(n, m2, mul_f32x2(zw[e], r2)));
          f[2 * e] = o.x;
          f[2 * e + 1] = o.y;
        }
      }
      if (on) store_vec(dx + i * I::GROUPS * a.dx.hs, f);
    }
    if (NORM) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (kind == 0) dw1[e] = add_f32x2(dw1[e], dw[e]);
        else dw2[e] = add_f32x2(dw2[e], dw[e]);
      }
    }
  }
  if (NORM) {
    constexpr int GROUPS = ROT_THREADS / LANES;
    __shared__ float part[GROUPS][LANES * 8];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 d = unpack_f32x2(which == 0 ? dw1[e] : dw2[e]);
        part[threadIdx.x / LANES][e0 + 2 * e] = d.x;
        part[threadIdx.x / LANES][e0 + 2 * e + 1] = d.y;
      }
      __syncthreads();
      for (int d = threadIdx.x; d < a.D; d += ROT_THREADS) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < GROUPS; ++i) sum += part[i][d];
        a.dw[(static_cast<size_t>(blockIdx.x) * 2 + which) * a.D + d] = sum;
      }
    }
  }
}

// The same two, a warp per row and an element per lane and step: any even R, any D up to 256, any strides and addresses.
constexpr int ROT_MAX_D = 256;
constexpr int ROT_STEPS = ROT_MAX_D / 32;
template <bool HALF>
__device__ __forceinline__ float turned(const RotaryArgs& a, int row, int d, float own, float other) {
  const int half = a.R >> 1;
  const int col = HALF ? (d < half ? d : d - half) : d >> 1;
  const bool first = HALF ? d < half : (d & 1) == 0;
  const float c = a.cos[static_cast<size_t>(row) * half + col], s = a.sin[static_cast<size_t>(row) * half + col];
  return own * c + other * (first != (a.inverse != 0) ? -s : s);
}
template <bool HALF>
__device__ __forceinline__ int partner_of(int d, int R) {
  return HALF ? (d < (R >> 1) ? d + (R >> 1) : d - (R >> 1)) : d ^ 1;
}

template <typename T, bool HALF, bool NORM>
__global__ void __launch_bounds__(ROT_THREADS)
rotary_any_kernel(const RotaryArgs a, unsigned n_rows) {
  pdl_wait();
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const unsigned heads = a.n1 + a.n2;
  for (unsigned r = blockIdx.x * (ROT_THREADS / 32) + (threadIdx.x >> 5); r < n_rows; r += gridDim.x * (ROT_THREADS / 32)) {
    const unsigned token = r / heads;
    const int h = static_cast<int>(r - token * heads);
    const int s = static_cast<int>(token / a.B), b = static_cast<int>(token % a.B);
    const T* x = static_cast<const T*>(a.x.p) + a.x.at(s, b, h);
    const T* w = static_cast<const T*>(h < a.n1 ? a.w1 : a.w2);
    T* y = h < a.n1 ? static_cast<T*>(a.y1.p) + a.y1.at(s, b, h) : static_cast<T*>(a.y2.p) + a.y2.at(s, b, h - a.n1);
    const int row = table_row(a, s, b);
    float rstd = 1.f;
    if (NORM) {
      float ss = 0.f;
      for (int d = lane; d < a.D; d += 32) ss += to_f32(x[d]) * to_f32(x[d]);
      rstd = rsqrtf(warp_sum(ss) * a.inv_D + a.eps);
    }
    auto z = [&](int d) { return NORM ? to_f32(x[d]) * (rstd * to_f32(w[d])) : to_f32(x[d]); };
    for (int d = lane; d < a.D; d += 32)
      y[d] = from_f32<T>(d < a.R ? turned<HALF>(a, row, d, z(d), z(partner_of<HALF>(d, a.R))) : z(d));
  }
}

template <typename T, bool HALF, bool NORM>
__global__ void __launch_bounds__(ROT_THREADS)
qk_norm_rope_bwd_any_kernel(const RotaryArgs a, unsigned n_rows) {
  pdl_wait();
  pdl_trigger();
  constexpr int WARPS = ROT_THREADS / 32;
  const int lane = threadIdx.x & 31;
  const unsigned heads = a.n1 + a.n2 + a.n3;
  float dw[2][ROT_STEPS] = {};
  for (unsigned r = blockIdx.x * WARPS + (threadIdx.x >> 5); r < n_rows; r += gridDim.x * WARPS) {
    const unsigned token = r / heads;
    const int h = static_cast<int>(r - token * heads);
    const int s = static_cast<int>(token / a.B), b = static_cast<int>(token % a.B);
    const int k = h < a.n1 ? 0 : (h < a.n1 + a.n2 ? 1 : 2);
    const T* g = k == 0 ? static_cast<const T*>(a.y1.p) + a.y1.at(s, b, h)
               : k == 1 ? static_cast<const T*>(a.y2.p) + a.y2.at(s, b, h - a.n1)
                        : static_cast<const T*>(a.y3.p) + a.y3.at(s, b, h - a.n1 - a.n2);
    T* dx = static_cast<T*>(a.dx.p) + a.dx.at(s, b, h);
    if (k == 2) {
      for (int d = lane; d < a.D; d += 32) dx[d] = g[d];
      continue;
    }
    const int row = table_row(a, s, b);
    const T* x = static_cast<const T*>(a.x.p) + a.x.at(s, b, h);
    const T* w = static_cast<const T*>(k == 0 ? a.w1 : a.w2);
    float dz[ROT_STEPS];
    float ss = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < ROT_STEPS; ++i) {
      const int d = lane + 32 * i;
      if (d < a.D) {
        dz[i] = to_f32(g[d]);
        if (d < a.R) dz[i] = turned<HALF>(a, row, d, dz[i], to_f32(g[partner_of<HALF>(d, a.R)]));
        if (NORM) {
          const float f = to_f32(x[d]);
          ss += f * f;
          dot += dz[i] * to_f32(w[d]) * f;
        }
      }
    }
    float rstd = 1.f, m = 0.f;
    if (NORM) {
      rstd = rsqrtf(warp_sum(ss) * a.inv_D + a.eps);
      m = warp_sum(dot) * rstd * rstd * a.inv_D;
    }
#pragma unroll
    for (int i = 0; i < ROT_STEPS; ++i) {
      const int d = lane + 32 * i;
      if (d < a.D) {
        float o = dz[i];
        if (NORM) {
          const float n = to_f32(x[d]) * rstd;
          if (k == 0) dw[0][i] += dz[i] * n;
          else dw[1][i] += dz[i] * n;
          o = rstd * dz[i] * to_f32(w[d]) - n * m;
        }
        dx[d] = from_f32<T>(o);
      }
    }
  }
  if (NORM) {
    __shared__ float part[WARPS][ROT_MAX_D];
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
#pragma unroll
      for (int i = 0; i < ROT_STEPS; ++i) part[threadIdx.x >> 5][lane + 32 * i] = dw[which][i];
      __syncthreads();
      for (int d = threadIdx.x; d < a.D; d += ROT_THREADS) {
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < WARPS; ++i) sum += part[i][d];
        a.dw[(static_cast<size_t>(blockIdx.x) * 2 + which) * a.D + d] = sum;
      }
    }
  }
}

// dw1, dw2 [D] from the blocks' partial sums [blocks][2][D]: 32 columns a block, 32 threads to a column.
template <typename T>
__global__ void __launch_bounds__(1024)
qk_norm_dw_kernel(const float* parts, int blocks, int D, T* __restrict__ dw1, T* __restrict__ dw2) {
  pdl_wait();
  pdl_trigger();
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), sub = threadIdx.x >> 5;
  float sum = 0.f;
  if (col < 2 * D)
    for (int i = sub; i < blocks; i += 32) sum += parts[static_cast<size_t>(i) * 2 * D + col];
  __shared__ float s[32][33];
  s[threadIdx.x & 31][sub] = sum;
  __syncthreads();
  sum = warp_sum(s[sub][threadIdx.x & 31]);
  const int c = blockIdx.x * 32 + sub;
  if ((threadIdx.x & 31) == 0 && c < 2 * D) {
    if (c < D) dw1[c] = from_f32<T>(sum);
    else dw2[c - D] = from_f32<T>(sum);
  }
}

bool aligned(const Part& t, int elem) {
  if (t.p == nullptr) return true;
  const long long per = 16 / elem;
  return (reinterpret_cast<uintptr_t>(t.p) & 15) == 0 && t.ss % per == 0 && t.bs % per == 0 && t.hs % per == 0;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// 16-byte accesses reach everything, and no pair is split between the eight elements of a lane and its neighbour's.
bool vectors(const RotaryArgs& a, int elem, int half) {
  if (a.D % 8 != 0 || a.R % (half ? 16 : 8) != 0) return false;
  return aligned(a.x, elem) && aligned(a.y1, elem) && aligned(a.y2, elem) && aligned(a.y3, elem) && aligned(a.dx, elem) &&
         aligned16(a.cos) && aligned16(a.sin) && aligned16(a.w1) && aligned16(a.w2);
}

template <typename T, bool HALF, bool NORM>
int launch_forward(const RotaryArgs& a, bool vec, cudaStream_t stream) {
  const unsigned long long tokens = static_cast<unsigned long long>(a.S) * a.B;
  const int heads = a.n1 + a.n2;
  if (tokens * heads > 0x7fffffffull) return -1;
  if (!vec) {
    const unsigned rows = static_cast<unsigned>(tokens * heads);
    const unsigned blocks = std::min<unsigned>((rows + 7) / 8, gfs_host::sm_count() * 32);
    gfs_host::launch_pdl(rotary_any_kernel<T, HALF, NORM>, dim3(blocks), dim3(ROT_THREADS), 0, stream, a, rows);
  } else {
    const int lanes = a.D <= 64 ? 8 : (a.D <= 128 ? 16 : 32);
    const int rows = FWD_STEPS * 32 / lanes;
    const int items_q = (a.n1 + rows - 1) / rows, per = items_q + (a.n2 + rows - 1) / rows;
    const unsigned items = static_cast<unsigned>(tokens) * per;
    auto kern = lanes == 8 ? rotary_kernel<T, 8, HALF, NORM>
                           : (lanes == 16 ? rotary_kernel<T, 16, HALF, NORM> : rotary_kernel<T, 32, HALF, NORM>);
    gfs_host::launch_pdl(kern, dim3((items + ROT_WARPS - 1) / ROT_WARPS), dim3(ROT_THREADS), 0, stream, a, items,
                         static_cast<unsigned>(per), items_q);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : -11;
}

int bwd_blocks() { return gfs_host::sm_count() * 2; }   // what is resident

template <typename T, bool HALF, bool NORM>
int launch_backward(const RotaryArgs& a, bool vec, T* dw1, T* dw2, cudaStream_t stream) {
  const unsigned long long tokens = static_cast<unsigned long long>(a.S) * a.B;
  const int heads = a.n1 + a.n2 + a.n3;
  if (tokens * heads > 0x7fffffffull) return -1;
  unsigned blocks;
  if (!vec) {
    const unsigned rows = static_cast<unsigned>(tokens * heads);
    blocks = std::min<unsigned>((rows + 7) / 8, bwd_blocks());
    gfs_host::launch_pdl(qk_norm_rope_bwd_any_kernel<T, HALF, NORM>, dim3(blocks), dim3(ROT_THREADS), 0, stream, a, rows);
  } else {
    const int lanes = a.D <= 64 ? 8 : (a.D <= 128 ? 16 : 32);
    const int rows = bwd_steps<T>() * 32 / lanes;
    const int items_q = (a.n1 + rows - 1) / rows, items_k = (a.n2 + rows - 1) / rows;
    const int per = items_q + items_k + (a.n3 + rows - 1) / rows;
    const unsigned items = static_cast<unsigned>(tokens) * per;
    blocks = std::min<unsigned>((items + ROT_WARPS - 1) / ROT_WARPS, bwd_blocks());
    auto kern = lanes == 8 ? qk_norm_rope_bwd_kernel<T, 8, HALF, NORM>
                           : (lanes == 16 ? qk_norm_rope_bwd_kernel<T, 16, HALF, NORM>
                                          : qk_norm_rope_bwd_kernel<T, 32, HALF, NORM>);
    gfs_host::launch_pdl(kern, dim3(blocks), dim3(ROT_THREADS), 0, stream, a, items, static_cast<unsigned>(per), items_q,
                         items_k);
  }
  if (cudaGetLastError() != cudaSuccess) return -11;
  if (NORM) {
    gfs_host::launch_pdl(qk_norm_dw_kernel<T>, dim3((2 * a.D + 31) / 32), dim3(1024), 0, stream,
                         static_cast<const float*>(a.dw), static_cast<int>(blocks), a.D, dw1, dw2);
    if (cudaGetLastError() != cudaSuccess) return -12;
  }
  return 0;
}

template <typename T>
int dispatch(const RotaryArgs& a, int half, bool norm, bool backward, void* dw1, void* dw2, cudaStream_t stream) {
  const bool vec = vectors(a, sizeof(T), half);
  T *d1 = static_cast<T*>(dw1), *d2 = static_cast<T*>(dw2);
  if (backward) {
    if (half) return norm ? launch_backward<T, true, true>(a, vec, d1, d2, stream)
                          : launch_backward<T, true, false>(a, vec, d1, d2, stream);
    return norm ? launch_backward<T, false, true>(a, vec, d1, d2, stream)
                : launch_backward<T, false, false>(a, vec, d1, d2, stream);
  }
  if (half) return norm ? launch_forward<T, true, true>(a, vec, stream) : launch_forward<T, true, false>(a, vec, stream);
  return norm ? launch_forward<T, false, true>(a, vec, stream) : launch_forward<T, false, false>(a, vec, stream);
}

int dispatch_type(const RotaryArgs& a, int dtype, int half, bool norm, bool backward, void* dw1, void* dw2,
                  cudaStream_t stream) {
  switch (dtype) {
    case 0: return dispatch<__nv_bfloat16>(a, half, norm, backward, dw1, dw2, stream);
    case 1: return dispatch<__half>(a, half, norm, backward, dw1, dw2, stream);
    case 2: return dispatch<float>(a, half, norm, backward, dw1, dw2, stream);
    default: return -1;
  }
}

bool sizes_ok(int S, int B, int n, int D, int R, int rows, const void* positions) {
  return S >= 0 && B >= 0 && n >= 0 && D > 0 && D <= ROT_MAX_D && R > 0 && R % 2 == 0 && R <= D &&
         (positions != nullptr ? rows > 0 : rows >= S);
}

Part part(const void* p, const long long* st) { return Part{const_cast<void*>(p), st[0], st[1], st[2]}; }

}  // namespace

extern "C" {

// y = rotation of x, both [S, B, nh, D]. strides: 6 element strides {x, y} x {seq, batch, head}. cos, sin: fp32
// [rows, R / 2]; positions: null (token s takes row s) or [B, S], int32 or (pos64) int64: one outside [0, rows) puts
// STATUS_BAD_ARGUMENT into the status words. half: pairs (i, i + R / 2), else (2i, 2i + 1). inverse: the transposed
// rotation. dtype: 0 bf16, 1 fp16, 2 fp32. D <= 256.
int gfs_rotary(const void* x, void* y, const long long* strides, const void* cosb, const void* sinb, const void* positions,
               int pos64, int rows, int S, int B, int nh, int D, int R, int half, int inverse, int dtype, void* stream) {
  if (!sizes_ok(S, B, nh, D, R, rows, positions)) return -1;
  if (S == 0 || B == 0 || nh == 0) return 0;
  RotaryArgs a = {};
  a.x = part(x, strides);
  a.y1 = part(y, strides + 3);
  a.cos = static_cast<const float*>(cosb);
  a.sin = static_cast<const float*>(sinb);
  a.positions = positions; a.pos64 = pos64; a.rows = rows;
  a.S = S; a.B = B; a.n1 = nh; a.D = D; a.R = R; a.inverse = inverse != 0;
  a.status = gfs_host::status_words();
  return dispatch_type(a, dtype, half, false, false, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

// q [S, B, n1, D] and k [S, B, n2, D], contiguous, from the packed projection x [S, B, n1 + 2 n2, D] (the last n2 heads
// are v's and not read): norm with the weights w1, w2 [D] (null: none), then the rotation as above. strides: 3 of x.
int gfs_qk_norm_rope_fwd(const void* x, const long long* strides, const void* w1, const void* w2, void* q, void* k,
                         const void* cosb, const void* sinb, const void* positions, int pos64, int rows, int S, int B,
                         int n1, int n2, int D, int R, int half, float eps, int dtype, void* stream) {
  if (!sizes_ok(S, B, n1 + n2, D, R, rows, positions)) return -1;
  if ((w1 == nullptr) != (w2 == nullptr)) return -1;
  if (S == 0 || B == 0 || n1 + n2 == 0) return 0;
  RotaryArgs a = {};
  a.x = part(x, strides);
  a.y1 = Part{q, static_cast<long long>(B) * n1 * D, static_cast<long long>(n1) * D, D};
  a.y2 = Part{k, static_cast<long long>(B) * n2 * D, static_cast<long long>(n2) * D, D};
  a.w1 = w1; a.w2 = w2;
  a.cos = static_cast<const float*>(cosb);
  a.sin = static_cast<const float*>(sinb);
  a.positions = positions; a.pos64 = pos64; a.rows = rows;
  a.S = S; a.B = B; a.n1 = n1; a.n2 = n2; a.D = D; a.R = R; a.eps = eps; a.inv_D = 1.f / D;
  a.status = gfs_host::status_words();
  return dispatch_type(a, dtype, half, w1 != nullptr, false, nullptr, nullptr, static_cast<cudaStream_t>(stream));
}

// fp32 elements of the scratch `dw` of the backward
long long gfs_qk_norm_rope_scratch(int D) { return static_cast<long long>(bwd_blocks()) * 2 * D; }

// dx (packed like x) from dq, dk, dv, and the weights' gradients dw1, dw2 [D] (with w1, w2 only). strides: 15 element
// strides {x, dq, dk, dv, dx} x {seq, batch, head}.
int gfs_qk_norm_rope_bwd(const void* x, const void* dq, const void* dk, const void* dv, void* dx, const long long* strides,
                         const void* w1, const void* w2, void* dw1, void* dw2, void* dw, const void* cosb,
                         const void* sinb, const void* positions, int pos64, int rows, int S, int B, int n1, int n2, int D,
                         int R, int half, float eps, int dtype, void* stream) {
  if (!sizes_ok(S, B, n1 + n2, D, R, rows, positions)) return -1;
  if ((w1 == nullptr) != (w2 == nullptr) || S == 0 || B == 0 || n1 + n2 == 0) return -1;
  if (w1 != nullptr && (dw1 == nullptr || dw2 == nullptr || dw == nullptr)) return -1;
  RotaryArgs a = {};
  a.x = part(x, strides);
  a.y1 = part(dq, strides + 3);
  a.y2 = part(dk, strides + 6);
  a.y3 = part(dv, strides + 9);
  a.dx = part(dx, strides + 12);
  a.w1 = w1; a.w2 = w2;
  a.dw = static_cast<float*>(dw);
  a.cos = static_cast<const float*>(cosb);
  a.sin = static_cast<const float*>(sinb);
  a.positions = positions; a.pos64 = pos64; a.rows = rows;
  a.S = S; a.B = B; a.n1 = n1; a.n2 = n2; a.n3 = n2; a.D = D; a.R = R; a.inverse = 1; a.eps = eps; a.inv_D = 1.f / D;
  a.status = gfs_host::status_words();
  return dispatch_type(a, dtype, half, w1 != nullptr, true, dw1, dw2, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
