// kanjoos_amd/csrc/knj_mfma.h -- f16 matrix-core steps and transposed LDS reads of the attention kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace knj {
namespace dev {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));

// One 16x16x32 f16 matrix-core step: acc[i] += sum_k A[4*(l/16)+i][k] B[k][l%16]
// where lane l supplies A[l%16][8*(l/16) + j] and B[8*(l/16) + j][l%16], j < 8.
__device__ __forceinline__ f32x4 mfma16(h16x8 a, h16x8 b, f32x4 acc) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
}

// f32 values as f16 high parts and f16 remainders (x = hi + lo to ~22 bits):
// against f16 cache values the two products are exact and summed in f32.
__device__ __forceinline__ void split_h8(const float4& p, const float4& q, h16x8& hi, h16x8& lo) {
  const float v[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    hi[j] = (_Float16)v[j];
    lo[j] = (_Float16)(v[j] - (float)hi[j]);
  }
}

typedef __attribute__((address_space(3))) void lds_void;
typedef __attribute__((address_space(1))) void glb_void;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// Four f16 of a transposed LDS read (ds_read_b64_tr_b16).  Within each group
// of 16 lanes, lane 4q + e receives element e of the 8-byte pieces addressed
// by lanes q, 4 + q, 8 + q and 12 + q, in that order: a 4 x 16 block of a
// row-major matrix read one piece per lane arrives as its columns.  Issued as
// asm: the compiler's wait placement treats the builtin as aliasing every
// LDS DMA in flight and would wait for the next chunk's DMA before it; the
// caller waits for the reads itself (lds_wait8) before using the values.
template <int OFF>
__device__ __forceinline__ u32x2 lds_tr16(uint32_t addr) {
  u32x2 v;
  asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(v) : "v"(addr), "i"(OFF));
  return v;
}
// every LDS access of this wave complete; the eight values are tied to the
// wait so that no use moves above it
__device__ __forceinline__ void lds_wait8(u32x2* v) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(v[4]), "+v"(v[5]), "+v"(v[6]), "+v"(v[7]));
}
__device__ __forceinline__ void lds_tie8(u32x2* v) {
  asm volatile("" : "+v"(v[0]), "+v"(v[1]), "+v"(v[2]), "+v"(v[3]), "+v"(v[4]), "+v"(v[5]), "+v"(v[6]), "+v"(v[7]));
}

}  // namespace dev
}  // namespace knj
