// kanjoos_amd/csrc/knj_pages.h -- groups of a 4-bit page as the f16 values they stand for.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "knj_common.h"

namespace knj {
namespace dev {

typedef _Float16 hx2 __attribute__((ext_vector_type(2)));

// Bytes of a page's kv head: key codes, value codes, key words, value words.
template <int D>
struct PageHead {
  static constexpr int kCode = D / 2, kMeta = D / 8, kSlot = 2 * (kCode + kMeta);  // bytes a slot
  // start of the four blocks in a page of 1 << shift slots
  static __host__ __device__ __forceinline__ uint32_t codes(int v, int shift) { return (uint32_t)(v * kCode) << shift; }
  static __host__ __device__ __forceinline__ uint32_t meta(int v, int shift) {
    return (uint32_t)(2 * kCode + v * kMeta) << shift;
  }
};

// A group's word that makes each of its values a NaN: step 0, low NaN.
constexpr uint32_t kNanGroup = 0x7E000000u;

// A group's step and low, each in both halves.
__device__ __forceinline__ void group_word(uint32_t m, hx2& step, hx2& low) {
  const hx2 w = __builtin_bit_cast(hx2, m);
  step = hx2{w[0], w[0]};
  low = hx2{w[1], w[1]};
}

// Eight codes as f16(low + step * code), one rounding each, in order of the dims: of rows that
// are loaded, and of k_tree, whose operands take any cache's rows in that order.  A
// code's bits become the low bits of 1024's significand, or, four bits up, of 64's
// (steps of 1 and of 1/16: 64 + code), from which the offset is taken off exactly.
// The two exponents are kept in vector registers, so that one instruction masks and joins
// (of two constants it takes one from a scalar register; as literals they are two
// instructions, a fifth of the whole decoding).
struct Decoder {
  uint32_t e10, e6;
  __device__ __forceinline__ Decoder() : e10(0x64006400u), e6(0x54005400u) { asm("" : "+v"(e10), "+v"(e6)); }
  __device__ __forceinline__ uint4 eight(uint32_t w, hx2 step, hx2 low) const {
    const hx2 o10 = {(_Float16)1024.0f, (_Float16)1024.0f}, o6 = {(_Float16)64.0f, (_Float16)64.0f};
    const uint32_t u = w >> 8;
    const hx2 a = __builtin_bit_cast(hx2, (w & 0x000F000Fu) | e10) - o10;
    const hx2 b = __builtin_bit_cast(hx2, (w & 0x00F000F0u) | e6) - o6;
    const hx2 c = __builtin_bit_cast(hx2, (u & 0x000F000Fu) | e10) - o10;
    const hx2 d = __builtin_bit_cast(hx2, (u & 0x00F000F0u) | e6) - o6;
    auto value = [&](hx2 x) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, step, low)); };
    return make_uint4(value(a), value(b), value(c), value(d));
  }
};

// The same in the order 0 4 1 5 2 6 3 7 of the dims, for kernels that pack their queries and
// put their results in order to suit (pack_queries, in_order): a code as a byte is the e4m3
// number code * 2^-9 (subnormal or not), which the conversion of two takes back to the whole
// number.
__device__ __forceinline__ uint4 decode8_mixed(uint32_t w, hx2 step, hx2 low) {
  const uint32_t a = w & 0x0F0F0F0Fu, b = (w >> 4) & 0x0F0F0F0Fu;
  auto value = [&](hx2 x) { return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(x, step, low)); };
  return make_uint4(value(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 512.0f, false)),
                    value(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)a, 512.0f, true)),
                    value(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 512.0f, false)),
                    value(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)b, 512.0f, true)));
}

}  // namespace dev
}  // namespace knj
