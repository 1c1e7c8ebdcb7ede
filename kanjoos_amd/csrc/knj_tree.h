// kanjoos_amd/csrc/knj_tree.h -- attention of drafted tokens over a cache of one format.
//
// o_t = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s_j = scale log2(e) q_t.k_j, over
// the slots j that draft t sees: those of the prefix, and the drafts in its mask
// row.  One pass over the cache with a running maximum and sum per column; a
// column is one (draft, query head) pair of a kv head, so that the cache is read
// once for all drafts and heads of a tile.
#pragma once

#include "knj_common.h"
#include "knj_dev.h"
#include "knj_mfma.h"

namespace knj {

struct TreePlan {
  int cps;       // chunks per split of the slots
  int n_split;   // splits of the longest sequence
  int n_tiles;   // column tiles of a full set of drafts
  int units;     // n_seq * n_split * n_head_kv
};

namespace tree {

using namespace dev;

// Sixteen codes as f16 (exact): e4m3 by the conversion, int8 by setting the
// offset code under the exponent of 1024 and subtracting 1024 + 128.
template <int FORMAT>
__device__ __forceinline__ uint2 codes4_h(uint32_t w) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  if constexpr (FORMAT == KNJ_KV_F8) {
    const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false);
    const h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true);
    return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
  } else {
    const uint32_t u = w ^ 0x80808080u;
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    const h2 a = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
    const h2 b = __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
    return make_uint2(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b));
  }
}

// The f16 of a word that are infinite or NaN replaced by zero; true if any was.
__device__ __forceinline__ bool drop_nonfinite(uint32_t& w) {
  const bool lo = (w & 0x7C00u) == 0x7C00u, hi = (w & 0x7C000000u) == 0x7C000000u;
  if (lo) w &= 0xFFFF0000u;
  if (hi) w &= 0x0000FFFFu;
  return lo || hi;
}

// Four transposed f16 (see lds_tr16) by the builtin: its waits are the compiler's.
__device__ __forceinline__ u32x2 lds_tr16_at(const uint8_t* p) {
  typedef short s4 __attribute__((__vector_size__(8)));
  typedef __attribute__((address_space(3))) s4 lds_s4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p));
}

// Weights (and their sum) are held times 2^14: the largest stay below f16's
// 65,504 and f16 keeps all of a weight's bits down to 2^-28 of the largest.
constexpr float kLift = 14.0f;

template <int TYPE>
__device__ __forceinline__ void store4(void* p, uint64_t i, float4 v) {
  if constexpr (TYPE == KNJ_TYPE_F32) *reinterpret_cast<float4*>((float*)p + i) = v;
  else *reinterpret_cast<uint2*>((uint16_t*)p + i) = make_uint2(pack_act<TYPE>(v.x, v.y), pack_act<TYPE>(v.z, v.w));
}
__device__ __forceinline__ void store4(int type, void* p, uint64_t i, float4 v) {
  if (type == KNJ_TYPE_F32) store4<KNJ_TYPE_F32>(p, i, v);
  else if (type == KNJ_TYPE_F16) store4<KNJ_TYPE_F16>(p, i, v);
  else store4<KNJ_TYPE_BF16>(p, i, v);
}

// Eight activations as f32.
__device__ __forceinline__ void load8(int type, const void* p, uint64_t i, float4& a, float4& b) {
  if (type == KNJ_TYPE_F32) {
    a = *reinterpret_cast<const float4*>((const float*)p + i);
    b = *reinterpret_cast<const float4*>((const float*)p + i + 4);
    return;
  }
  const uint4 u = *reinterpret_cast<const uint4*>((const uint16_t*)p + i);
  if (type == KNJ_TYPE_F16) {
    a = make_float4(h2f(u.x), h2f(u.x >> 16), h2f(u.y), h2f(u.y >> 16));
    b = make_float4(h2f(u.z), h2f(u.z >> 16), h2f(u.w), h2f(u.w >> 16));
  } else {
    a = make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                    __uint_as_float(u.y & 0xFFFF0000u));
    b = make_float4(__uint_as_float(u.z << 16), __uint_as_float(u.z & 0xFFFF0000u), __uint_as_float(u.w << 16),
                    __uint_as_float(u.w & 0xFFFF0000u));
  }
}

// Prefix and drafts of a sequence, held to what the host checked.
__device__ __forceinline__ void seq_lengths(const TreeArgs& a, int s, int& P, int& N) {
  P = min(max(a.prefix[s], 0), a.max_prefix);
  N = a.counts ? min(max(a.counts[s], 0), a.n_rows) : a.n_rows;
}

// Which of the 64 slots from P + rel on draft t sees (rel > -64): the prefix
// slots, then the bits of its mask row below N.
__device__ __forceinline__ uint64_t seen64(const uint64_t* row, int words, int t, int N, int rel) {
  auto below = [](int n) -> uint64_t { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; };
  auto word = [&](int i) -> uint64_t {
    if (i < 0) return ~0ull;
    if (i >= words) return 0ull;
    return (row ? row[i] : below(t + 1 - 64 * i)) & below(N - 64 * i);
  };
  const int i = rel >> 6, sh = rel & 63;
  uint64_t v = word(i) >> sh;
  if (sh) v |= word(i + 1) << (64 - sh);
  return v;
}

// A column's result or split record, four dims at a time: the maximum in base-2
// units, the sum and the weighted values.
template <int D>
__device__ __forceinline__ void emit(const TreeArgs& a, const TreePlan& p, int s, int kvh, int split, int n_cols, int G,
                                     int N, int col, int d, float M, float L, float4 o) {
  if (col >= N * G) return;
  if (p.n_split > 1) {
    float* rec = a.partial + ((((uint64_t)s * a.c.n_head_kv + kvh) * p.n_split + split) * n_cols + col) * (D + 4);
    if (d == 0) {
      rec[0] = M;
      rec[1] = L;
    }
    *reinterpret_cast<float4*>(rec + 4 + d) = o;
    return;
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // nothing seen: zeros
  const int t = col / G;
  store4(a.type, a.out, ((uint64_t)s * a.n_rows + t) * a.out_stride + (uint64_t)(kvh * G + col - t * G) * D + d,
         make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

// Workgroup = (sequence, split of the slots, kv head, tile of WC * NT * 16 columns).
// Wave (wc, ws) holds NT tiles of 16 columns -- queries as the B operand in
// registers -- against SW of the chunk's WS * SW slots:
//   scores  S[slot][col] = K (16 slots x 32 dims) x Q (32 dims x 16 columns); lane
//           (r = l % 16, kq = l / 16) ends with column r's slots 16 st + 4 kq + i;
//   values  O^T[d][col] = V^T (16 dims x 32 slots) x E (32 slots x 16 columns), the
//           weights as the lane holds them, V^T by transposed LDS reads.
// With few columns the waves share the slots instead (WS > 1, each with running
// statistics of its own, joined at the end).  Chunks go through registers to
// LDS as f16, the next one's loads in flight while one is computed; 8-bit codes
// are exact in f16 and their scales stay out of the products: a score is
// multiplied by its slot's, a weight by its slot's over the running largest of
// the scales its column has seen (a power of two; a weight then stays in f16's
// range whatever the cache's units).  Queries are scaled by a power of two per
// row, so that f16 holds any of them.  SPLIT keeps queries and weights as f16
// high parts and remainders (22 bits), for f32 activations.
template <int D, int FORMAT, bool SPLIT, int NT, int WC, int SW>
__global__ __launch_bounds__(kBlock, 2) void k_tree(TreeArgs a, TreePlan p) {
  constexpr int WS = 4 / WC, C = WS * SW, COLS = WC * NT * 16, ST = SW / 16;
  constexpr int RB = 2 * D, RPB = 256 / RB, NSLOT = RB / 16, NPAIR = RB / 32, CB = C * RB;
  constexpr bool Q8 = FORMAT != KNJ_KV_F16;
  constexpr int NP = C * D / (Q8 ? 16 : 8) / kBlock;  // 16-byte loads per thread and matrix
  static_assert(NP >= 1 && C * D % (16 * kBlock) == 0, "whole loads");
  constexpr int JOIN = WS > 1 ? WS * COLS * (D + 4) * 4 : 0;
  constexpr int LDS = 2 * CB > JOIN ? 2 * CB : JOIN;
  auto kslot = [](int q, int sl) { return sl ^ ((q / RPB) & (NSLOT - 1)); };
  auto vslot = [](int q, int sl) { return sl ^ (((q / RPB) & (NPAIR - 1)) << 1); };
  __shared__ __align__(16) uint8_t lds[LDS];
  __shared__ __align__(16) float ksc[Q8 ? C : 4], vsc[Q8 ? C : 4];
  __shared__ uint32_t poison[C / 32];
  __shared__ float jm[WS > 1 ? WS * COLS : 1], jl[WS > 1 ? WS * COLS : 1];
  uint8_t *ks = lds, *vs = lds + CB;

  // tiles of one unit run on one XCD, whose L2 then serves their shared slots
  const int tile = (blockIdx.x >> 3) % p.n_tiles;
  const int unit = ((blockIdx.x >> 3) / p.n_tiles) * 8 + (blockIdx.x & 7);
  if (unit >= p.units) return;
  const int nk = a.c.n_head_kv, G = a.n_head / nk;
  const int kvh = unit % nk, split = (unit / nk) % p.n_split, s = unit / (nk * p.n_split);
  int P, N;
  seq_lengths(a, s, P, N);
  const int valid = P + N;
  const int c0 = split * p.cps, c1 = min((valid + C - 1) / C, c0 + p.cps);
  if (tile * COLS >= N * G || c0 >= c1) return;
  const int n_cols = p.n_tiles * COLS;

  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wc = wave % WC, ws = wave / WC, r = lane & 15, kq = lane >> 4;
  const uint64_t seq_at = (uint64_t)s * a.c.seq_stride + (uint64_t)kvh * a.c.n_ctx * D;
  constexpr int EB = Q8 ? 1 : 2;
  const uint8_t* kc = (const uint8_t*)a.c.k + seq_at * EB;
  const uint8_t* vc = (const uint8_t*)a.c.v + seq_at * EB;
  const float *kscale = nullptr, *vscale = nullptr;
  if constexpr (Q8) {
    kscale = a.c.k_scale + seq_at / D;
    vscale = a.c.v_scale + seq_at / D;
  }

  // ---- a chunk's bytes into registers (zeros past the sequence's slots)
  uint4 kr[NP], vr[NP];
  float ksr = 0.0f, vsr = 0.0f;
  constexpr int PR = Q8 ? D / 16 : D / 8;  // 16-byte loads per row
  auto fetch = [&](int p0) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int at = tid + kBlock * i, q = at / PR, sl = at % PR;
      const bool in = p0 + q < valid;
      const uint64_t off = (uint64_t)(in ? p0 + q : valid - 1) * (D * EB) + 16 * sl;
      kr[i] = *reinterpret_cast<const uint4*>(kc + off);
      vr[i] = *reinterpret_cast<const uint4*>(vc + off);
      if (!in) kr[i] = vr[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    if constexpr (Q8) {
      if (tid < C) {
        const bool in = p0 + tid < valid;
        ksr = in ? kscale[p0 + tid] : 0.0f;
        vsr = in ? vscale[p0 + tid] : 0.0f;
      }
    }
  };
  fetch(c0 * C);

  // ---- this lane's query columns
  h16x8 qh[NT][D / 32], ql[SPLIT ? NT : 1][D / 32];
  float s2[NT];
  int tcol[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = min(tile * COLS + (wc * NT + nt) * 16 + r, N * G - 1);  // (past the drafts: not stored)
    const int t = col / G;
    tcol[nt] = t;
    const uint64_t at = ((uint64_t)s * a.n_rows + t) * a.q_stride + (uint64_t)(kvh * G + col - t * G) * D + 8 * kq;
    float4 x[D / 32], y[D / 32];
    float am = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      load8(SPLIT ? KNJ_TYPE_F32 : a.type, a.q, at + 32 * c, x[c], y[c]);
      am = fmaxf(am, fmaxf(fmaxf(fabsf(x[c].x), fabsf(x[c].y)), fmaxf(fabsf(x[c].z), fabsf(x[c].w))));
      am = fmaxf(am, fmaxf(fmaxf(fabsf(y[c].x), fabsf(y[c].y)), fmaxf(fabsf(y[c].z), fabsf(y[c].w))));
    }
    am = fmaxf(am, xor16_f(am));
    am = fmaxf(am, xor32_f(am));
    const int e = min(max((int)(__float_as_uint(am) >> 23) - 127, -100), 100);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
    s2[nt] = a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      const float4 u = make_float4(x[c].x * down, x[c].y * down, x[c].z * down, x[c].w * down);
      const float4 v = make_float4(y[c].x * down, y[c].y * down, y[c].z * down, y[c].w * down);
      h16x8 hi, lo;
      split_h8(u, v, hi, lo);
      qh[nt][c] = hi;
      if constexpr (SPLIT) ql[nt][c] = lo;
    }
  }

  // (maxima in units of the stored scores, before s2)
  float m[NT], l[NT], vref[NT];
  bool spoilt[NT];
  f32x4 acc[NT][D / 16];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -INFINITY;
    l[nt] = 0.0f;
    vref[nt] = 0.0f;
    spoilt[nt] = false;
#pragma unroll
    for (int dt = 0; dt < D / 16; ++dt) acc[nt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int words = (a.n_rows + 63) / 64;
  const uint64_t* mask = a.mask ? a.mask + (a.mask_shared ? 0 : (uint64_t)s * a.n_rows * words) : nullptr;

  for (int j = c0; j < c1; ++j) {
    const int p0 = j * C;
    const bool drafts = p0 + C > P;  // the chunk reaches the drafts (or the end)
    __syncthreads();                 // every wave is done with the chunk before
    if (drafts) {
      if (tid < C / 32) poison[tid] = 0u;
      __syncthreads();
    }
    // ---- registers to LDS, as f16
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const int at = tid + kBlock * i, q = at / PR, sl = at % PR;
      uint4 kw[Q8 ? 2 : 1], vw[Q8 ? 2 : 1];
      if constexpr (Q8) {
        const uint2 k0 = codes4_h<FORMAT>(kr[i].x), k1 = codes4_h<FORMAT>(kr[i].y);
        const uint2 k2 = codes4_h<FORMAT>(kr[i].z), k3 = codes4_h<FORMAT>(kr[i].w);
        const uint2 v0 = codes4_h<FORMAT>(vr[i].x), v1 = codes4_h<FORMAT>(vr[i].y);
        const uint2 v2 = codes4_h<FORMAT>(vr[i].z), v3 = codes4_h<FORMAT>(vr[i].w);
        kw[0] = make_uint4(k0.x, k0.y, k1.x, k1.y);
        kw[1] = make_uint4(k2.x, k2.y, k3.x, k3.y);
        vw[0] = make_uint4(v0.x, v0.y, v1.x, v1.y);
        vw[1] = make_uint4(v2.x, v2.y, v3.x, v3.y);
      } else {
        kw[0] = kr[i];
        vw[0] = vr[i];
      }
      // a draft's value row may be unseen by some columns of the tile: what is
      // not finite in it would reach them as 0 x inf, and is kept out
      if (FORMAT != KNJ_KV_I8 && drafts && p0 + q >= P) {
        bool any = false;
#pragma unroll
        for (int h = 0; h < (Q8 ? 2 : 1); ++h) {
          any |= drop_nonfinite(vw[h].x);
          any |= drop_nonfinite(vw[h].y);
          any |= drop_nonfinite(vw[h].z);
          any |= drop_nonfinite(vw[h].w);
        }
        if (any) atomicOr(&poison[q >> 5], 1u << (q & 31));
      }
#pragma unroll
      for (int h = 0; h < (Q8 ? 2 : 1); ++h) {
        const int slot = Q8 ? 2 * sl + h : sl;
        *reinterpret_cast<uint4*>(ks + q * RB + 16 * kslot(q, slot)) = kw[h];
        *reinterpret_cast<uint4*>(vs + q * RB + 16 * vslot(q, slot)) = vw[h];
      }
    }
    if constexpr (Q8) {
      if (tid < C) {
        ksc[tid] = ksr;
        vsc[tid] = vsr;
      }
    }
    __syncthreads();
    if (j + 1 < c1) fetch(p0 + C);

    // ---- scores
    f32x4 sc[NT][ST];
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      const int q = ws * SW + 16 * st + r;
      const uint8_t* krow = ks + q * RB;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const h16x8 ka = __builtin_bit_cast(h16x8, *reinterpret_cast<const uint4*>(krow + 16 * kslot(q, 4 * c + kq)));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[nt][st] = mfma16(ka, qh[nt][c], sc[nt][st]);
          if constexpr (SPLIT) sc[nt][st] = mfma16(ka, ql[nt][c], sc[nt][st]);
        }
      }
    }
    float4 vq[Q8 ? ST : 1];  // value scales of this lane's slots
    if constexpr (Q8) {
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const float4 kv = *reinterpret_cast<const float4*>(ksc + ws * SW + 16 * st + 4 * kq);
        vq[st] = *reinterpret_cast<const float4*>(vsc + ws * SW + 16 * st + 4 * kq);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[nt][st][0] *= kv.x;
          sc[nt][st][1] *= kv.y;
          sc[nt][st][2] *= kv.z;
          sc[nt][st][3] *= kv.w;
        }
      }
    }
    // ---- the slots a column does not see, where the chunk reaches the drafts
    uint32_t nib[NT][ST];  // four bits per lane and slot tile
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int st = 0; st < ST; ++st) nib[nt][st] = 15u;
    if (drafts) {
      uint64_t bad = 0;
      if constexpr (FORMAT != KNJ_KV_I8) {
        bad = poison[ws * (SW / 32)];
        if constexpr (SW == 64) bad |= (uint64_t)poison[ws * (SW / 32) + 1] << 32;
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint64_t seen =
            seen64(mask ? mask + (uint64_t)tcol[nt] * words : nullptr, words, tcol[nt], N, p0 + ws * SW - P);
        spoilt[nt] |= (seen & bad) != 0;
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const uint32_t b = (uint32_t)(seen >> (16 * st + 4 * kq)) & 15u;
          nib[nt][st] = b;
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[nt][st][i] = (b >> i) & 1u ? sc[nt][st][i] : -INFINITY;
        }
      }
    }
    // ---- running softmax per column, and the weights as the values' operand
    h16x8 eh[NT][ST / 2], el[SPLIT ? NT : 1][ST / 2];
    float alpha[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float mx = -INFINITY;
#pragma unroll
      for (int st = 0; st < ST; ++st)
        mx = fmaxf(mx, fmaxf(fmaxf(sc[nt][st][0], sc[nt][st][1]), fmaxf(sc[nt][st][2], sc[nt][st][3])));
      mx = fmaxf(mx, xor16_f(mx));
      mx = fmaxf(mx, xor32_f(mx));
      const float mn = fmaxf(m[nt], mx);
      // (-inf while the column has seen nothing: exponents then from 0)
      const float mr = mn == -INFINITY ? 0.0f : mn * s2[nt];
      alpha[nt] = __builtin_amdgcn_exp2f(fmaf(m[nt], s2[nt], -mr));
      m[nt] = mn;
      float es = 0.0f;
      float w[4 * ST];
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = __builtin_amdgcn_exp2f(fmaf(sc[nt][st][i], s2[nt], kLift - mr));
          es += e;
          w[4 * st + i] = e;
        }
      l[nt] = l[nt] * alpha[nt] + es;
      if constexpr (Q8) {
        float vm = 0.0f;  // the largest finite scale that the column sees here
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const float v[4] = {vq[st].x, vq[st].y, vq[st].z, vq[st].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) vm = fmaxf(vm, (!drafts || (nib[nt][st] >> i) & 1u) && v[i] < INFINITY ? v[i] : 0.0f);
        }
        vm = fmaxf(vm, xor16_f(vm));
        vm = fmaxf(vm, xor32_f(vm));
        const float ref = fmaxf(vref[nt], __uint_as_float(__float_as_uint(vm) & 0x7F800000u));
        const float inv = ref > 0.0f ? __uint_as_float((254u << 23) - __float_as_uint(ref)) : 0.0f;
        alpha[nt] *= vref[nt] * inv;
        vref[nt] = ref;
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const float v[4] = {vq[st].x, vq[st].y, vq[st].z, vq[st].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float x = w[4 * st + i] * (v[i] * inv);
            w[4 * st + i] = !drafts || (nib[nt][st] >> i) & 1u ? x : 0.0f;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < ST / 2; ++c) {
        h16x8 hi, lo;
        split_h8(make_float4(w[8 * c], w[8 * c + 1], w[8 * c + 2], w[8 * c + 3]),
                 make_float4(w[8 * c + 4], w[8 * c + 5], w[8 * c + 6], w[8 * c + 7]), hi, lo);
        eh[nt][c] = hi;
        if constexpr (SPLIT) el[nt][c] = lo;
      }
      if (__ballot(alpha[nt] != 1.0f) != 0) {
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][dt][i] *= alpha[nt];
      }
    }
    // ---- values: step c covers slots 32c + 4kq + i and 32c + 16 + 4kq + i; lane r's
    // transposed read takes row 32c (+ 16) + 4kq + r/4, dims 16dt + 4(r%4) .. + 3,
    // and receives dim 16dt + r of the four rows
    const int pa = 4 * kq + (r >> 2), sub = 8 * (r & 3);
#pragma unroll
    for (int c = 0; c < ST / 2; ++c) {
      const uint8_t* vrow = vs + (ws * SW + 32 * c + pa) * RB + (sub & 15);
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt) {
        // (rows pa + 16 k share the swizzle of row pa)
        const uint8_t* at = vrow + 16 * vslot(pa, (32 * dt + sub) >> 4);
        const u32x2 v0 = lds_tr16_at(at), v1 = lds_tr16_at(at + 16 * RB);
        const h16x8 vv = __builtin_bit_cast(h16x8, make_uint4(v0.x, v0.y, v1.x, v1.y));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          acc[nt][dt] = mfma16(vv, eh[nt][c], acc[nt][dt]);
          if constexpr (SPLIT) acc[nt][dt] = mfma16(vv, el[nt][c], acc[nt][dt]);
        }
      }
    }
  }

  // ---- columns out: sums over the four lanes of a column, scales back in
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] += xor16_f(l[nt]);
    l[nt] += xor32_f(l[nt]);
    if (spoilt[nt]) l[nt] = NAN;
    m[nt] = m[nt] == -INFINITY ? -INFINITY : m[nt] * s2[nt];
    if constexpr (Q8) {
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[nt][dt][i] *= vref[nt];
    }
  }
  if constexpr (WS == 1) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = tile * COLS + (wc * NT + nt) * 16 + r;
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
        emit<D>(a, p, s, kvh, split, n_cols, G, N, col, 16 * dt + 4 * kq, m[nt], l[nt],
                make_float4(acc[nt][dt][0], acc[nt][dt][1], acc[nt][dt][2], acc[nt][dt][3]));
    }
  } else {
    // the waves that shared the slots join their columns through LDS
    float* ja = reinterpret_cast<float*>(lds);
    __syncthreads();
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int col = (wc * NT + nt) * 16 + r;
      if (kq == 0) {
        jm[ws * COLS + col] = m[nt];
        jl[ws * COLS + col] = l[nt];
      }
#pragma unroll
      for (int dt = 0; dt < D / 16; ++dt)
        *reinterpret_cast<float4*>(ja + (ws * COLS + col) * (D + 4) + 16 * dt + 4 * kq) =
            make_float4(acc[nt][dt][0], acc[nt][dt][1], acc[nt][dt][2], acc[nt][dt][3]);
    }
    __syncthreads();
    for (int i = tid; i < COLS * (D / 4); i += kBlock) {
      const int col = i / (D / 4), d = 4 * (i % (D / 4));
      float M = -INFINITY, L = 0.0f;
#pragma unroll
      for (int k = 0; k < WS; ++k) M = fmaxf(M, jm[k * COLS + col]);
      const float mr = M == -INFINITY ? 0.0f : M;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < WS; ++k) {
        const float f = exp2f(jm[k * COLS + col] - mr);
        const float4 v = *reinterpret_cast<const float4*>(ja + (k * COLS + col) * (D + 4) + d);
        L += jl[k * COLS + col] * f;
        o.x += v.x * f;
        o.y += v.y * f;
        o.z += v.z * f;
        o.w += v.w * f;
      }
      emit<D>(a, p, s, kvh, split, n_cols, G, N, tile * COLS + col, d, M, L, o);
    }
  }
}

// One launch of a format's kernel: D, split and the column tile's shape at run
// time (columns per kv head up to 16, 32, 64 or more).
template <int FORMAT>
hipError_t launch_format(const TreeArgs& a, const TreePlan& p, int cols, hipStream_t s);

#define KNJ_TREE_FORMAT(FORMAT)                                                                          \
  template <>                                                                                            \
  hipError_t launch_format<FORMAT>(const TreeArgs& a, const TreePlan& p, int cols, hipStream_t s) {      \
    const dim3 grid((unsigned)((p.units + 7) / 8 * 8 * p.n_tiles));                                      \
    const bool split = a.type == KNJ_TYPE_F32;                                                           \
    if (a.c.head_dim == 128) {                                                                           \
      if (split) KNJ_TREE_COLS(128, FORMAT, true);                                                       \
      else KNJ_TREE_COLS(128, FORMAT, false);                                                            \
    } else {                                                                                             \
      if (split) KNJ_TREE_COLS(64, FORMAT, true);                                                        \
      else KNJ_TREE_COLS(64, FORMAT, false);                                                             \
    }                                                                                                    \
    return hipGetLastError();                                                                            \
  }
#define KNJ_TREE_COLS(DD, FORMAT, SPLIT)                                                                 \
  do {                                                                                                   \
    if (cols == 16) KNJ_LAUNCH((k_tree<DD, FORMAT, SPLIT, 1, 1, 32>), grid, dim3(kBlock), 0, s, a, p);   \
    else if (cols == 32) KNJ_LAUNCH((k_tree<DD, FORMAT, SPLIT, 2, 1, 32>), grid, dim3(kBlock), 0, s, a, p); \
    else if (cols == 64) KNJ_LAUNCH((k_tree<DD, FORMAT, SPLIT, 2, 2, 64>), grid, dim3(kBlock), 0, s, a, p); \
    else KNJ_LAUNCH((k_tree<DD, FORMAT, SPLIT, 2, 4, 64>), grid, dim3(kBlock), 0, s, a, p);              \
  } while (0)

}  // namespace tree
}  // namespace knj
