// kanjoos_amd/csrc/knj_pages_attn.h -- what the attention kernels over 4-bit pages share.
#pragma once

#include <type_traits>

#include "knj_pages.h"
#include "knj_tree.h"

namespace knj {
namespace tree {

typedef float f32x2 __attribute__((ext_vector_type(2)));

// Eight f16 at an LDS address.
__device__ __forceinline__ h16x8 lds_h8(uint32_t p) {
  typedef __attribute__((address_space(3))) const h16x8 lds_v8;
  return *(lds_v8*)(uintptr_t)p;
}

// Eight weights as f16 high parts and remainders, two to an instruction; a remainder in one
// (w - hi with hi read as f16: the factor is kept out of the compiler's sight, which else
// makes it a conversion, of an upper half at half the rate, and a difference).
__device__ __forceinline__ void split8(const float (&w)[8], h16x8& hi, h16x8& lo) {
  float minus = -1.0f;
  asm("" : "+s"(minus));
#pragma unroll
  for (int i = 0; i < 8; i += 2) {
    const hx2 h = __builtin_convertvector(f32x2{w[i], w[i + 1]}, hx2);
    const f32x2 r = {fmaf((float)h[0], minus, w[i]), fmaf((float)h[1], minus, w[i + 1])};
    const hx2 l = __builtin_convertvector(r, hx2);
    hi[i] = h[0];
    hi[i + 1] = h[1];
    lo[i] = l[0];
    lo[i + 1] = l[1];
  }
}

// The halves of a word that are infinite or NaN (0x7C00 and up) replaced by zero; the sign
// bits of those that were.  `signs` has both halves' sign bits, or none: then nothing is.
__device__ __forceinline__ uint32_t clear_nonfinite(uint32_t& w, uint32_t signs) {
  const uint32_t m = ((w & 0x7FFF7FFFu) + 0x04000400u) & signs;
  w &= ~(m | (m - (m >> 15)));
  return m;
}

// Eight queries from element `at` on as f32.
template <bool SPLIT>
__device__ __forceinline__ void queries8(const TreeArgs& a, uint64_t at, float4& x, float4& y) {
  if constexpr (SPLIT) {
    x = ld4<KNJ_TYPE_F32>(a.q, at);
    y = ld4<KNJ_TYPE_F32>(a.q, at + 4);
  } else if (a.type == KNJ_TYPE_F16) {
    x = ld4<KNJ_TYPE_F16>(a.q, at);
    y = ld4<KNJ_TYPE_F16>(a.q, at + 4);
  } else {
    x = ld4<KNJ_TYPE_BF16>(a.q, at);
    y = ld4<KNJ_TYPE_BF16>(a.q, at + 4);
  }
}
__device__ __forceinline__ float largest8(const float4& x, const float4& y) {
  return fmaxf(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))),
               fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
}
// A column's power of two from its largest magnitude: 2^-e (2^e and 2^-e both normal
// numbers), and the scores' factor with 2^e in it, held to f32's largest.
__device__ __forceinline__ float column_unit(float scale, float am, float& down) {
  const int e = min(max((int)(__float_as_uint(am) >> 23) - 127, -126), 126);
  down = __uint_as_float((uint32_t)(127 - e) << 23);
  return fminf(scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + e) << 23), 0x1.fffffep127f);
}
// Eight scaled queries in decode8_mixed's order as f16 high parts and remainders.
__device__ __forceinline__ void pack_queries(const float4& x, const float4& y, float down, h16x8& hi, h16x8& lo) {
  const float q[8] = {x.x * down, y.x * down, x.y * down, y.y * down, x.z * down, y.z * down, x.w * down, y.w * down};
  split8(q, hi, lo);
}

// A lane's parts of its column, eight dims each `stride` apart from element `at` on (the four
// lanes of a column have it all).  Returns the scores' factor.
template <int D, bool SPLIT>
__device__ __forceinline__ float column(const TreeArgs& a, uint64_t at, int stride, h16x8 (&hi)[D / 32], h16x8 (&lo)[D / 32]) {
  float4 x[D / 32], y[D / 32];
  float am = 0.0f, down;
#pragma unroll
  for (int c = 0; c < D / 32; ++c) queries8<SPLIT>(a, at + stride * c, x[c], y[c]);
#pragma unroll
  for (int c = 0; c < D / 32; ++c) am = fmaxf(am, largest8(x[c], y[c]));
  am = fmaxf(am, xor16_f(am));
  am = fmaxf(am, xor32_f(am));
  const float s2 = column_unit(a.scale, am, down);
#pragma unroll
  for (int c = 0; c < D / 32; ++c) {
    h16x8 rest;
    pack_queries(x[c], y[c], down, hi[c], rest);
    if constexpr (SPLIT) lo[c] = rest;
  }
  return s2;
}

// An accumulator of 16 dims x 16 columns over rows in decode8_mixed's order: a lane of an
// even kq (its 16 lanes of the wave) has dims 0 4 1 5 of eight, those of kq + 1 have 2 6 3 7;
// 0 1 2 3 and 4 5 6 7 by exchanges of 16 lanes with the next 16.
__device__ __forceinline__ float4 in_order(const f32x4& v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[0]), __float_as_uint(v[1]), false, false);
  const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[2]), __float_as_uint(v[3]), false, false);
  return make_float4(__uint_as_float(x[0]), __uint_as_float(y[0]), __uint_as_float(x[1]), __uint_as_float(y[1]));
}

}  // namespace tree
}  // namespace knj
