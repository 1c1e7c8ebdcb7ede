// kanjoos_amd/csrc/knj_tree.h -- attention of drafted tokens over a cache of one format.
//
// o_t = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m), s_j = scale log2(e) q_t.k_j, over
// the slots j that draft t sees: those of the prefix, and the drafts in its mask
// row.  One pass over the cache with a running maximum and sum per column; a
// column is one (draft, query head) pair of a kv head, so that the cache is read
// once for all drafts and heads of a tile.
#pragma once

#include <type_traits>

#include "knj_common.h"
#include "knj_dev.h"
#include "knj_mfma.h"
#include "knj_pages.h"

namespace knj {

// n / d for n < 2^31 by one multiplication: with L = ceil(log2 d) and m = ceil(2^(31 +
// L) / d), which 32 bits hold, n m 2^-(31 + L) is above n / d by less than 1 / d.
struct FastDiv {
  uint32_t d, m, sh;  // m 0 for d = 1
  FastDiv() = default;
  explicit FastDiv(uint32_t v) : d(v), m(0), sh(0) {
    if (v == 1) return;
    while ((1ull << (sh + 1)) < v) ++sh;  // L - 1
    m = (uint32_t)(((1ull << (32 + sh)) + v - 1) / v);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const { return m ? __umulhi(n, m) >> sh : n; }
};

// Attention over 4-bit pages for few columns a kv head: workgroups of kStepWaves waves
// that take tiles of kStepTile slots in turn.
constexpr int kStepTile = 32, kStepWaves = 4;
// For many: column tiles of 16 a wave over steps of kWideStep slots.
constexpr int kWideStep = 64, kWideWaves = 8;

struct TreePlan {
  int cps;       // chunks per split of the slots
  int n_split;   // splits of the longest sequence
  int n_tiles;   // column tiles of a full set of drafts
  int units;     // n_seq * n_split * n_head_kv
  FastDiv by_nk, by_split, by_group;  // n_head_kv, n_split, query heads per kv head
  FastDiv by_head, by_rows, by_cps;   // n_head, n_rows, cps
  bool even;     // of launch_pages_step: a sequence's own tiles are split evenly
  // Tiles per split of a sequence: a multiple of the waves that take them in turn, and as
  // many as it has splits for, so that a batch's shorter sequences keep as many workgroups
  // busy as its longest.
  __device__ __forceinline__ int even_cps(int tiles) const {
    return max(((int)by_split.div(tiles + n_split - 1) + kStepWaves - 1) & -kStepWaves, kStepWaves);
  }
};

namespace tree {

using namespace dev;

// Four codes as f16 (exact): e4m3 by the conversion, int8 by setting the
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

// Of four codes (slot 0 dims 0, 1, slot 1 dims 0, 1 in one word, slots 2, 3 in the
// other) the even and the odd dim's four slots as f16.
template <int FORMAT>
__device__ __forceinline__ void pairs_h(u32x2 w, uint2& even, uint2& odd) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  if constexpr (FORMAT == KNJ_KV_F8) {
    const uint32_t x = __builtin_amdgcn_perm(0u, w.x, 0x03010200u), y = __builtin_amdgcn_perm(0u, w.y, 0x03010200u);
    const uint2 a = codes4_h<FORMAT>(x), b = codes4_h<FORMAT>(y);
    even = make_uint2(a.x, b.x);
    odd = make_uint2(a.y, b.y);
  } else {
    const uint32_t x = w.x ^ 0x80808080u, y = w.y ^ 0x80808080u;
    const h2 off = {(_Float16)1152.0f, (_Float16)1152.0f};
    auto half = [&](uint32_t u, uint32_t sel) {
      return __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, __builtin_amdgcn_perm(0x64646464u, u, sel)) - off);
    };
    even = make_uint2(half(x, 0x04020400u), half(y, 0x04020400u));
    odd = make_uint2(half(x, 0x04030401u), half(y, 0x04030401u));
  }
}

// The elements of a word that are infinite or NaN replaced by zero; true if any was.
template <int FORMAT>
__device__ __forceinline__ bool drop_nonfinite(uint32_t& w) {
  if constexpr (FORMAT == KNJ_KV_F8) {  // codes 0x7F and 0xFF
    const uint32_t m = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    w &= ~(m | (m - (m >> 7)));
    return m != 0;
  } else {
    const bool lo = (w & 0x7C00u) == 0x7C00u, hi = (w & 0x7C000000u) == 0x7C000000u;
    if (lo) w &= 0xFFFF0000u;
    if (hi) w &= 0x0000FFFFu;
    return lo || hi;
  }
}

// Four transposed f16 (see lds_tr16) by the builtin: its waits are the compiler's.
__device__ __forceinline__ u32x2 lds_tr16_at(uint32_t p) {
  typedef short s4 __attribute__((__vector_size__(8)));
  typedef __attribute__((address_space(3))) s4 lds_s4;
  return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(uintptr_t)p));
}

// A weight is 2^(s - r), its column's reference r 6 below the running maximum when it
// was set and moved only when that has passed it by 13 (the accumulators are rescaled
// then, which after a column's first slots is rare): at most 2^13, or 2^15 with a value
// scale's factor, below f16's 65,504, and f16 keeps all of a weight's bits down to
// 2^-20 of the maximum.  r is kept as the f32 that the exponents subtract, so that
// a rescale by 2^(old - new) fits the weights on both sides, and is 1 where r stays.
constexpr float kLift = 6.0f, kLag = 13.0f;

// With 8-bit values the slot of a column's largest scale may have next to no weight, and
// the weights that the column lives on then meet small factors: r is set further
// below the maximum, by up to 2^80, wherever the largest product of a weight and its
// factor would stay below 1.  (The sum of weights, in f32, has the room; the products
// are what f16 has to hold, and are held to 65,504 from then on.)
constexpr float kMostLift = 80.0f;

// Maximum that carries a NaN (a NaN score makes its column NaN); the instruction
// takes three, without the quieting of its inputs that fmaxf asks for.
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// 16 bytes at an LDS address.
__device__ __forceinline__ uint4 lds_b128(uint32_t p) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) const u32x4 lds_v4;
  return __builtin_bit_cast(uint4, *(lds_v4*)(uintptr_t)p);
}

__device__ __forceinline__ void lds_put_b128(uint32_t p, uint4 v) {
  typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) u32x4 lds_v4;
  *(lds_v4*)(uintptr_t)p = __builtin_bit_cast(u32x4, v);
}

// Four results as activations.
__device__ __forceinline__ uint2 pack4(int type, float4 v) {
  if (type == KNJ_TYPE_F16) return make_uint2(pack_act<KNJ_TYPE_F16>(v.x, v.y), pack_act<KNJ_TYPE_F16>(v.z, v.w));
  return make_uint2(pack_act<KNJ_TYPE_BF16>(v.x, v.y), pack_act<KNJ_TYPE_BF16>(v.z, v.w));
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

// LDS DMA of 16 bytes per lane, as dma16, from a wave-uniform address and each lane's offset.
__device__ __forceinline__ void dma16_at(const void* g, uint32_t off, uint32_t base) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(off), "s"(g), "s"(base) : "memory");
}

// LDS DMA of 4 bytes per lane, as dma16.
__device__ __forceinline__ void dma4(const void* g, uint32_t base) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" : : "v"(g), "s"(base) : "memory");
}

typedef _Float16 h16x4 __attribute__((ext_vector_type(4)));

// Workgroup = (sequence, split of the slots, kv head, tile of WC * NT * 16 columns)
// of WC * WS waves.  Wave (wc, ws) holds NT tiles of 16 columns -- queries as the B
// operand in registers -- against SW of the chunk's C = WS * SW slots:
//   scores  S[slot][col] = K (16 slots x 32 dims) x Q (32 dims x 16 columns); lane
//           (r = l % 16, kq = l / 16) ends with column r's slots 16 st + 4 kq + i;
//   values  O^T[d][col] = V^T (16 dims x 32 slots) x E (32 slots x 16 columns), the
//           weights as the lane holds them, V^T by transposed LDS reads.
// Waves that share the columns (WS > 1) keep running statistics of their own and
// join them at the end, through LDS, in pairs.
//
// Chunks reach LDS by DMA, as the cache holds them, the next one while one is
// computed, one barrier a chunk; 16-byte pieces (K) and 32-byte pairs (V) of a row
// are permuted by an XOR of the row index, so that the operand reads fall on
// distinct banks.
// 8-bit codes become f16 (exactly) as operands.  Their scales stay out of the
// products: a score is multiplied by its slot's, a weight by its slot's over the
// running largest of the scales its column has seen (a power of two, so a weight
// stays in f16's range whatever the cache's units; kMostLift has the other end).
// Queries are scaled by a power of two per row, so that f16 holds any of them.  Weights
// are f16 high parts and remainders (22 bits) whatever the activations: 11 bits of a
// weight leave errors of the size of an f16 output's own rounding.  SPLIT keeps f32
// queries so too.
//
// The loads that need no sequence length (a chunk's rows, the queries) come
// first; rows of a chunk past the sequence's slots hold whatever the cache does
// there, and the chunks that reach the drafts are cleaned before use (below).
//
// What bounds it (f16, 64 drafts x 32 heads over 32,764 slots of 4 kv heads, 34 GFLOP:
// 69.6 us a call, 0.49 PFLOP/s; profiled, 73 us here, 65 at least, and 9 in the merge):
// of a wave's life the matrix cores are busy for 49 % (96 products a wave and chunk,
// a third of them the weights' remainders, without which the call took 57.7 us), vector
// instructions issue for 29 % (two waves share a SIMD, so 57 % of it); the two waves
// that the accumulators leave room for do not cover one another's waits.  Calls of few
// drafts are one wave's path through a chunk, 1.7 us of conversions, reductions and
// waits, and two launches: 9.5 us for 4 drafts over 1000 f16 slots.
// Tried before the remainders and no faster: eight waves to a tile (of 128 columns
// within 3 %, of 32 slower), a raised wave priority around the products, 768 or 1024
// workgroups, chunks of 128 slots, chunks through registers instead of DMA, the next
// chunk's DMA behind this one's reads (1 to 5 % slower).
template <int D, int FORMAT, bool SPLIT, int NT, int WC, int WS, int SW>
__global__ __launch_bounds__(64 * WC * WS, 2) void k_tree(TreeArgs a, TreePlan p) {
  constexpr bool PAGES = FORMAT == kFormatPages, Q8 = FORMAT == KNJ_KV_F8 || FORMAT == KNJ_KV_I8;
  constexpr int NW = WC * WS, NTH = 64 * NW, C = WS * SW, COLS = WC * NT * 16, ST = SW / 16;
  constexpr int RB = Q8 ? D : 2 * D;                     // bytes of a chunk's row in LDS
  constexpr int RPB = 256 / RB, NSLOT = RB / 16, NPAIR = RB / 32, CB = C * RB;
  constexpr int NI = CB / 1024 / NW;                     // 1 KB DMA instructions per wave and matrix
  constexpr int SB = 2 * CB + (Q8 ? 8 * C : 0);          // bytes of a stage: K, V, scales of both
  constexpr int DT = D / 16;                             // accumulator tiles per column tile
  constexpr int JOIN = WS > 1 ? WS / 2 * WC * NT * (DT * 1024 + 512) : 0;
  constexpr int LDS = 2 * SB > JOIN ? 2 * SB : JOIN;
  static_assert(CB % (1024 * NW) == 0, "whole DMA instructions");
  static_assert(C % 32 == 0 && NW % (C / 32) == 0, "whole DMA instructions of scales");
  static_assert(SB % 256 == 0, "stages on whole rows");
  static_assert(SW == 16 || SW % 32 == 0, "16 slots, or steps of 32");
  __shared__ __align__(1024) uint8_t lds[LDS];
  __shared__ uint32_t poison[C / 32];

  // tiles of one unit run on one XCD, whose L2 then serves their shared slots
  // (workgroups go to the eight XCDs in turn; gridDim.x is a multiple of eight)
  const int tile = blockIdx.x >> 3, unit = (blockIdx.z * gridDim.y + blockIdx.y) * 8 + (blockIdx.x & 7);
  if (unit >= p.units) return;
  const int nk = a.c.n_head_kv, G = p.by_group.d, n_ctx = a.c.n_ctx;
  const int rest = p.by_nk.div(unit), kvh = unit - rest * nk;
  const int s = p.by_split.div(rest), split = rest - s * p.n_split;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wc = wave % WC, ws = wave / WC, r = lane & 15, kq = lane >> 4;
  const uint64_t seq_at = (uint64_t)s * a.c.seq_stride + (uint64_t)kvh * n_ctx * D;
  constexpr int EB = Q8 ? 1 : 2;
  const uint8_t* kc = (const uint8_t*)a.c.k + seq_at * EB;
  const uint8_t* vc = (const uint8_t*)a.c.v + seq_at * EB;

  // ---- chunk j's bytes into stage `st`: wave w's instruction i fills KB i NW + w
  // of the chunk's K and of its V, whose rows share row 1024 w / RB + lane RB/16's
  // permutation (rows past the cache are its last row); with 8 bits, 64 of the scales
  const int dq = (wave * 1024 + 16 * lane) / RB, dsl = lane % NSLOT;
  const uint32_t koff = 16 * (dsl ^ ((dq / RPB) & (NSLOT - 1)));
  const uint32_t voff = 16 * (dsl ^ (((dq / RPB) & (NPAIR - 1)) << 1));
  auto dma = [&](int j, int st) {
    const int p0 = j * C;
    const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr(lds + st * SB + wave * 1024));
    if (__builtin_expect(p0 + C <= n_ctx, 1)) {  // uniform
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const uint64_t at = (uint64_t)p0 * RB + i * NW * 1024;
        dma16_at(kc + at, dq * RB + koff, to + i * NW * 1024);
        dma16_at(vc + at, dq * RB + voff, to + CB + i * NW * 1024);
      }
    } else {
#pragma unroll
      for (int i = 0; i < NI; ++i) {
        const uint64_t row = (uint64_t)min(p0 + i * (NW * 1024 / RB) + dq, n_ctx - 1) * RB;
        dma16(kc + row + koff, to + i * NW * 1024);
        dma16(vc + row + voff, to + CB + i * NW * 1024);
      }
    }
    if constexpr (Q8) {
      // (waves beyond the scales' 2 C floats repeat: the same bytes)
      const int x = wave % (2 * C / 64) * 64 + lane;
      const float* sc = (x < C ? a.c.k_scale : a.c.v_scale) + seq_at / D;
      dma4(sc + min(p0 + x % C, n_ctx - 1),
           __builtin_amdgcn_readfirstlane(lds_addr(lds + st * SB + 2 * CB + wave % (2 * C / 64) * 256)));
    }
  };
  // ---- chunk j of 4-bit pages: fetched into registers as it is, group by group, and put
  // into a stage as f16 rows, permuted as above.  A thread has NG groups, of one slot:
  // its key's and its value's, or with D 64, where there are half as many, one of them.
  // The slot's page is looked up a chunk ahead of its fetch.  (25 drafts x 8 heads over 4000
  // slots of pages 21 us a call, 8 of 32 sequences over up to 2000 34; what bounds it is the
  // decoding, which each workgroup does for its own columns.)
  constexpr int GROUPS = C * D / 32, NG = 2 * GROUPS / NTH;  // groups of a matrix, and of a thread
  static_assert(!PAGES || NG == 2 || NG == 1, "a thread's groups are of one slot");
  using H = PageHead<D>;
  const int pg = tid % GROUPS, prow = pg / (D / 32), pgroup = pg % (D / 32), pmat = NG == 1 ? tid / GROUPS : 0;
  const int last_entry = a.n_table - 1;
  int page = 0;  // of the next chunk to fetch
  uint4 pcode[NG];
  uint32_t pword[NG];
  const Decoder decode;
  bool pin = false;  // (a slot without a page holds NaN)
  auto look_up = [&](int j) {
    const int e = min((j * C + prow) >> a.page_shift, last_entry);
    page = a.table[(uint64_t)s * a.n_table + e];
  };
  auto fetch = [&](int j) {
    pin = page >= 0 && page < a.n_page;
    const uint32_t head = H::kSlot << a.page_shift;
    const uint8_t* at = a.pages + ((uint64_t)(pin ? page : 0) * nk + kvh) * head;
    const uint32_t row = (j * C + prow) & ((1 << a.page_shift) - 1);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int v = NG == 1 ? pmat : i;
      pcode[i] = *reinterpret_cast<const uint4*>(at + H::codes(v, a.page_shift) + row * H::kCode + 16 * pgroup);
      pword[i] = *reinterpret_cast<const uint32_t*>(at + H::meta(v, a.page_shift) + row * H::kMeta + 4 * pgroup);
    }
  };
  auto put = [&](int st) {
    const uint32_t to = lds_addr(lds + st * SB) + prow * RB;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      const int v = NG == 1 ? pmat : i;
      hx2 step, low;
      group_word(pin ? pword[i] : kNanGroup, step, low);
      const uint32_t perm = v ? ((prow / RPB) & (NPAIR - 1)) << 1 : (prow / RPB) & (NSLOT - 1);
      const uint32_t c[4] = {pcode[i].x, pcode[i].y, pcode[i].z, pcode[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        lds_put_b128(to + (v ? CB : 0) + 16 * ((4 * pgroup + k) ^ perm), decode.eight(c[k], step, low));
    }
  };
  const int c0 = split * p.cps;
  if constexpr (PAGES) {
    look_up(c0);
    fetch(c0);
    look_up(c0 + 1);
  } else {
    dma(c0, 0);
  }

  // ---- this lane's query columns.  Step c's dims 8 kq .. + 7 of 32; with 8 bits,
  // where a 16-byte piece of a K row is two steps', dims 64 (c/2) + 16 kq + 8 (c%2)
  h16x8 qh[NT][D / 32], ql[SPLIT ? NT : 1][D / 32];
  float s2[NT];
  int tcol[NT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = min(tile * COLS + (wc * NT + nt) * 16 + r, a.n_rows * G - 1);  // (past the drafts: not stored)
    const int t = p.by_group.div(col);
    tcol[nt] = t;
    const uint64_t at = ((uint64_t)s * a.n_rows + t) * a.q_stride + (uint64_t)(kvh * G + col - t * G) * D;
    float4 x[D / 32], y[D / 32];
    if constexpr (SPLIT) {
#pragma unroll
      for (int c = 0; c < D / 32; ++c) {
        const float* q = (const float*)a.q + at + (Q8 ? 64 * (c >> 1) + 16 * kq + 8 * (c & 1) : 32 * c + 8 * kq);
        x[c] = *reinterpret_cast<const float4*>(q);
        y[c] = *reinterpret_cast<const float4*>(q + 4);
      }
    } else {
      uint4 u[D / 32];
#pragma unroll
      for (int c = 0; c < D / 32; ++c)
        u[c] = *reinterpret_cast<const uint4*>((const uint16_t*)a.q + at +
                                               (Q8 ? 64 * (c >> 1) + 16 * kq + 8 * (c & 1) : 32 * c + 8 * kq));
      if (a.type == KNJ_TYPE_F16) {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          x[c] = make_float4(h2f(u[c].x), h2f(u[c].x >> 16), h2f(u[c].y), h2f(u[c].y >> 16));
          y[c] = make_float4(h2f(u[c].z), h2f(u[c].z >> 16), h2f(u[c].w), h2f(u[c].w >> 16));
        }
      } else {
#pragma unroll
        for (int c = 0; c < D / 32; ++c) {
          x[c] = make_float4(__uint_as_float(u[c].x << 16), __uint_as_float(u[c].x & 0xFFFF0000u),
                             __uint_as_float(u[c].y << 16), __uint_as_float(u[c].y & 0xFFFF0000u));
          y[c] = make_float4(__uint_as_float(u[c].z << 16), __uint_as_float(u[c].z & 0xFFFF0000u),
                             __uint_as_float(u[c].w << 16), __uint_as_float(u[c].w & 0xFFFF0000u));
        }
      }
    }
    float am = 0.0f;
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
      am = fmaxf(am, fmaxf(fmaxf(fabsf(x[c].x), fabsf(x[c].y)), fmaxf(fabsf(x[c].z), fabsf(x[c].w))));
      am = fmaxf(am, fmaxf(fmaxf(fabsf(y[c].x), fabsf(y[c].y)), fmaxf(fabsf(y[c].z), fabsf(y[c].w))));
    }
    am = fmaxf(am, xor16_f(am));
    am = fmaxf(am, xor32_f(am));
    // (2^e and 2^-e both normal numbers; a factor beyond f32 is held to its largest)
    const int e = min(max((int)(__float_as_uint(am) >> 23) - 127, -126), 126);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
    s2[nt] = fminf(a.scale * 1.4426950408889634f * __uint_as_float((uint32_t)(127 + e) << 23), 0x1.fffffep127f);
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
  int P, N;
  seq_lengths(a, s, P, N);
  const int valid = P + N, n_cols = p.n_tiles * COLS;
  const int c1 = min((valid + C - 1) / C, c0 + p.cps);
  if (tile * COLS >= N * G || c0 >= c1) {
    __builtin_amdgcn_s_waitcnt(0);  // the fetch lands before the workgroup ends
    return;
  }

  // (m: the references)
  float m[NT], l[NT], vref[NT];
  float lag[Q8 ? NT : 1], top[Q8 ? NT : 1];  // kLag and the lift; a product that the column has had
  bool lifted = false;                       // any column of the wave (uniform)
  bool spoilt[NT];
  f32x4 acc[NT][DT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -INFINITY;
    l[nt] = 0.0f;
    vref[nt] = 0.0f;
    if constexpr (Q8) {
      lag[nt] = kLag;
      top[nt] = 0.0f;
    }
    spoilt[nt] = false;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[nt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int words = (a.n_rows + 63) / 64;
  const uint64_t* mask = a.mask ? a.mask + (a.mask_shared ? 0 : (uint64_t)s * a.n_rows * words) : nullptr;

  // Operand addresses within a stage.  K rows 16 st + r share row r's permutation, V
  // rows 16 k + pa row pa's; a row starts on a multiple of its size, so piece c's
  // (pair b's) permuted place is an XOR of the address with the first one's.
  const uint32_t kat = (ws * SW + r) * RB + 16 * (kq ^ ((r / RPB) & (NSLOT - 1)));
  const int pa = 4 * kq + (r >> 2);
  const uint32_t vat = CB + (ws * SW + pa) * RB + 32 * ((pa / RPB) & (NPAIR - 1)) + 8 * (r & 3);
  const uint32_t lds0 = lds_addr(lds);

  // ---- a chunk's scores, in units of 1 / s2, and this lane's value scales
  constexpr int NE = SW == 16 ? 1 : ST / 2;  // value steps
  auto scores = [&](uint32_t at, f32x4 (&sc)[NT][ST], float (&vq)[Q8 ? 4 * ST : 1]) {
    const uint32_t k0 = at + kat;
    constexpr int NK = Q8 ? D / 64 : D / 32;  // 16-byte reads of a K row per lane
    uint4 w[NK][ST];
#pragma unroll
    for (int c = 0; c < NK; ++c)
#pragma unroll
      for (int st = 0; st < ST; ++st) w[c][st] = lds_b128((k0 ^ (64 * c)) + 16 * st * RB);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int st = 0; st < ST; ++st)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < D / 32; ++c) {
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        h16x8 ka;
        if constexpr (Q8) {
          const uint4 u = w[c >> 1][st];
          const uint2 x = codes4_h<FORMAT>((c & 1) ? u.z : u.x), y = codes4_h<FORMAT>((c & 1) ? u.w : u.y);
          ka = __builtin_bit_cast(h16x8, make_uint4(x.x, x.y, y.x, y.y));
        } else {
          ka = __builtin_bit_cast(h16x8, w[c][st]);
        }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[nt][st] = mfma16(ka, qh[nt][c], sc[nt][st]);
          if constexpr (SPLIT) sc[nt][st] = mfma16(ka, ql[nt][c], sc[nt][st]);
        }
      }
    }
    if constexpr (Q8) {
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const uint32_t q = at + 2 * CB + 4 * (ws * SW + 16 * st + 4 * kq);
        const float4 kv = __builtin_bit_cast(float4, lds_b128(q)), vv = __builtin_bit_cast(float4, lds_b128(q + 4 * C));
        vq[4 * st] = vv.x;
        vq[4 * st + 1] = vv.y;
        vq[4 * st + 2] = vv.z;
        vq[4 * st + 3] = vv.w;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[nt][st][0] *= kv.x;
          sc[nt][st][1] *= kv.y;
          sc[nt][st][2] *= kv.z;
          sc[nt][st][3] *= kv.w;
        }
      }
    }
  };
  // the largest of a column's scores
  auto largest = [&](const f32x4 (&sc)[ST]) {
    float mx = -INFINITY;
#pragma unroll
    for (int st = 0; st < ST; ++st)
      mx = max_nan(max_nan(max_nan(mx, sc[st][0]), max_nan(sc[st][1], sc[st][2])), sc[st][3]);
    const float2 m16 = pair16_f(mx);
    mx = max_nan(m16.x, m16.y);
    const float2 m32 = pair32_f(mx);
    return max_nan(m32.x, m32.y);
  };
  // Weights of a column's scores against its reference; with 8 bits times w8, the slots'
  // value scales over the column's.  Returns their sum (without those).
  auto weights = [&](const f32x4 (&sc)[ST], float s2c, float mref, const float (&w8)[Q8 ? 4 * ST : 1], float (&w)[4 * ST]) {
    // (the reference is -inf while the column has seen nothing: exponents then from 0)
    const float mr = mref == -INFINITY ? 0.0f : mref;
    float es = 0.0f;
#pragma unroll
    for (int i = 0; i < 4 * ST; ++i) {
      w[i] = __builtin_amdgcn_exp2f(fmaf(sc[i >> 2][i & 3], s2c, -mr));
      es += w[i];
      if constexpr (Q8) {
        w[i] *= w8[i];
        // (the weight itself, rounded to f32, is what is split in `operand`: formed
        // anew inside the conversion to f16, the product could round the other way
        // there than in the remainder, an f16 step off)
        asm("" : "+v"(w[i]));
      }
    }
    return es;
  };
  // the same as the values' operand
  auto operand = [&](const float (&w)[4 * ST], h16x8 (&eh)[NE], h16x8 (&el)[NE]) {
#pragma unroll
    for (int c = 0; c < NE; ++c)
      split_h8(make_float4(w[8 * c], w[8 * c + 1], w[8 * c + 2], w[8 * c + 3]),
               SW == 16 ? make_float4(0.f, 0.f, 0.f, 0.f)
                        : make_float4(w[(8 * c + 4) % (4 * ST)], w[(8 * c + 5) % (4 * ST)], w[(8 * c + 6) % (4 * ST)],
                                      w[(8 * c + 7) % (4 * ST)]),
               eh[c], el[c]);
  };
  // Values: step c covers slots 32c + 4kq + i and 32c + 16 + 4kq + i (SW 16: the
  // first).  Lane r's transposed read takes bytes 8 (r%4) .. + 7 of 32-byte pair b
  // of row 4kq + r/4 and receives 16-bit element r of the pair, of four rows:
  // dim 16b + r, or with 8 bits dims 32b + 2r (tile 2b) and 32b + 2r + 1 (2b + 1).
  struct VPair {
    u32x2 x, y;
  };
  auto vread = [&](uint32_t at, int c, int b) {
    const uint32_t q = ((at + vat) ^ (32 * b)) + 32 * c * RB;
    VPair v;
    v.x = lds_tr16_at(q);
    v.y = v.x;
    if constexpr (SW != 16) v.y = lds_tr16_at(q + 16 * RB);
    return v;
  };
  auto product = [&](int dt, uint2 v0, uint2 v1, int c, const h16x8 (&eh)[NT][NE], const h16x8 (&el)[NT][NE]) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      if constexpr (SW == 16) {
        const h16x4 vv = __builtin_bit_cast(h16x4, v0);
        const h16x4 hi = __builtin_shufflevector(eh[nt][0], eh[nt][0], 0, 1, 2, 3);
        acc[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x16f16(vv, hi, acc[nt][dt], 0, 0, 0);
        const h16x4 lo = __builtin_shufflevector(el[nt][0], el[nt][0], 0, 1, 2, 3);
        acc[nt][dt] = __builtin_amdgcn_mfma_f32_16x16x16f16(vv, lo, acc[nt][dt], 0, 0, 0);
      } else {
        const h16x8 vv = __builtin_bit_cast(h16x8, make_uint4(v0.x, v0.y, v1.x, v1.y));
        acc[nt][dt] = mfma16(vv, eh[nt][c], acc[nt][dt]);
        acc[nt][dt] = mfma16(vv, el[nt][c], acc[nt][dt]);
      }
    }
  };
  // the products of a chunk, its first step's reads given; each step's operands are
  // read while the step before is multiplied
  auto values = [&](uint32_t at, VPair (&v)[NPAIR], const h16x8 (&eh)[NT][NE], const h16x8 (&el)[NT][NE]) {
#pragma unroll
    for (int c = 0; c < NE; ++c) {
#pragma unroll
      for (int b = 0; b < NPAIR; ++b) {
        if constexpr (Q8) {
          uint2 e0, o0, e1, o1;
          pairs_h<FORMAT>(v[b].x, e0, o0);
          if constexpr (SW != 16) pairs_h<FORMAT>(v[b].y, e1, o1);
          else e1 = e0, o1 = o0;
          if (c + 1 < NE) v[b] = vread(at, c + 1, b);
          product(2 * b, e0, e1, c, eh, el);
          product(2 * b + 1, o0, o1, c, eh, el);
        } else {
          product(b, make_uint2(v[b].x.x, v[b].x.y), make_uint2(v[b].y.x, v[b].y.y), c, eh, el);
          if (c + 1 < NE) v[b] = vread(at, c + 1, b);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // a value scale's reference: the power of two above the largest, which a later
  // scale may pass fourfold before it moves (weights stay up to 2^15); 2^-126 above
  // subnormal scales, and at most 2^126, so that its inverse is a normal number too
  auto vref_of = [](float vm) {
    const uint32_t e = __float_as_uint(vm) & 0x7F800000u;
    return __uint_as_float(vm > 0.0f ? min(e + 0x00800000u, 0x7E800000u) : 0u);
  };
  auto inverse = [](float ref) { return ref > 0.0f ? __uint_as_float((254u << 23) - __float_as_uint(ref)) : 0.0f; };
  // column nt's reference moved if the largest score has passed it; the factor of what
  // was summed before
  auto lag_of = [&](int nt) {
    if constexpr (Q8) return lag[nt];
    else return kLag;
  };
  auto moved = [&](int nt, float mx) {
    const float old = m[nt];
    if (!(fmaf(mx, s2[nt], -old) <= lag_of(nt))) m[nt] = max_nan(old, fmaf(mx, s2[nt], kLag - kLift - lag_of(nt)));
    return __builtin_amdgcn_exp2f(old - (m[nt] == -INFINITY ? 0.0f : m[nt]));
  };
  // Largest of a column's products, and whether one is beyond f16.  (A NaN is its
  // column's result, whatever the references.)
  auto largest_product = [&](const float (&w)[4 * ST]) {
    float pm = 0.0f;
#pragma unroll
    for (int i = 0; i < 4 * ST; i += 2) pm = max_nan(max_nan(pm, w[i]), w[i + 1]);
    const float2 m16 = pair16_f(pm);
    pm = max_nan(m16.x, m16.y);
    const float2 m32 = pair32_f(pm);
    return max_nan(m32.x, m32.y);
  };
  auto beyond = [](float pm) { return pm >= 65520.0f; };
  // Whether a column's references have to move for its products: t, the largest of them
  // as far as known (`top` before this chunk's, which are asked where that is below 1),
  // is below 1 since they last moved, or one of this chunk's is beyond f16.
  auto low_or_beyond = [&](float top, float pm, bool fresh, float& t) {
    t = (fresh && !(top >= 1.0f)) || beyond(pm) ? max_nan(top, pm) : top;
    return (fresh && t > 0.0f && t < 1.0f) || beyond(pm);
  };
  // Column nt's lift: the factor of what was and is summed that brings t, a product that
  // the column has had, to between 2^6 and 2^7.
  auto lift = [&](int nt, float t) {
    const float e = (float)((int)(__float_as_uint(t) >> 23) - 127);
    const float d = t < INFINITY ? fminf(fmaxf(kLift - e, kLag - lag[nt]), kMostLift + kLag - lag[nt]) : 0.0f;
    const float old = m[nt];
    m[nt] -= d;
    lag[nt] += d;
    return d == 0.0f ? 1.0f : __builtin_amdgcn_exp2f(old - m[nt]);
  };
  auto rescale = [&](int nt, float alpha) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[nt][dt][i] *= alpha;
  };

  // chunk j's stage ready: this wave's DMA of it has landed; the barrier hands every
  // wave's part over and ends the reads of chunk j - 1, whose stage the next chunk
  // then refills (past the range: fetched and not used).  A third stage, a chunk more
  // ahead, was 4 % slower (one draft over 32K int8 slots).
  int j = c0, stage = 0;
  // With 4-bit pages chunk j + 1, fetched while j - 1 was computed, is put there now and
  // j + 2 is fetched.
  auto ready = [&]() {
    if constexpr (PAGES) {
      KNJ_BARRIER_AFTER(kLdsOnly);
      put(stage ^ 1);
      fetch(j + 2);
      look_up(j + 3);
    } else {
      KNJ_BARRIER_AFTER(vm_lds_imm(0));
      dma(j + 1, stage ^ 1);
    }
  };
  auto next = [&]() {
    ++j;
    stage ^= 1;
    if (j < c1) ready();
  };
  const int j_prefix = min(c1, P / C);  // chunks below lie in the prefix
  if constexpr (PAGES) {
    put(0);
    fetch(c0 + 1);
    look_up(c0 + 2);
  }
  ready();
  while (j < c1) {
    // ---- the first chunk, those that reach the drafts or the end, and those of the
    // prefix that move a reference
    const int p0 = j * C;
    const uint32_t at = lds0 + stage * SB;
    const bool drafts = p0 + C > P;
    // A draft's value row may be unseen by some columns of the tile, and rows past
    // the drafts are seen by none: what is not finite in them would reach a column
    // as 0 x inf, and is replaced by zeros.  Columns that see such a draft are
    // marked and come out as NaN.  (int8 codes are finite; their scales are
    // selected away.)
    uint64_t bad = 0;
    if (FORMAT != KNJ_KV_I8 && drafts) {
      if (tid < C / 32) poison[tid] = 0u;
      KNJ_BARRIER_AFTER(kLdsOnly);
      for (int o = 16 * tid; o < CB; o += 16 * NTH) {
        const int q = o / RB;
        if (p0 + q < P) continue;
        uint4* w = reinterpret_cast<uint4*>(lds + stage * SB + CB + o);
        uint4 v = *w;
        bool any = false;
        any |= drop_nonfinite<FORMAT>(v.x);
        any |= drop_nonfinite<FORMAT>(v.y);
        any |= drop_nonfinite<FORMAT>(v.z);
        any |= drop_nonfinite<FORMAT>(v.w);
        if (!any) continue;
        *w = v;
        if (p0 + q < valid) atomicOr(&poison[q >> 5], 1u << (q & 31));
      }
      KNJ_BARRIER_AFTER(kLdsOnly);
      bad = poison[(ws * SW) >> 5];
      if constexpr (SW == 64) bad |= (uint64_t)poison[((ws * SW) >> 5) + 1] << 32;
      if constexpr (SW == 16) bad = (bad >> ((ws * SW) & 31)) & 0xFFFFu;
    }
    f32x4 sc[NT][ST];
    float vq[Q8 ? 4 * ST : 1];
    scores(at, sc, vq);
    h16x8 eh[NT][NE], el[NT][NE];
    float w[NT][4 * ST], es[NT], alpha[NT], t[Q8 ? NT : 1];
    bool out[Q8 ? NT : 1];
    auto add = [&](int nt) {
      l[nt] += es[nt];
      operand(w[nt], eh[nt], el[nt]);
      rescale(nt, alpha[nt]);
    };
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      // the slots that the column sees: four bits per lane and slot tile
      uint64_t seen = ~0ull;
      if (drafts) seen = seen64(mask ? mask + (uint64_t)tcol[nt] * words : nullptr, words, tcol[nt], N, p0 + ws * SW - P);
      spoilt[nt] |= (seen & bad) != 0;
      seen >>= 4 * kq;
      float vm = 0.0f, vin[Q8 ? 4 * ST : 1];  // value scales of the slots seen, and the largest finite one
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const uint32_t four = (uint32_t)(seen >> (16 * st));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = (four & (1u << i)) != 0;
          sc[nt][st][i] = in ? sc[nt][st][i] : -INFINITY;
          if constexpr (Q8) {
            vin[4 * st + i] = in ? vq[4 * st + i] : 0.0f;
            vm = fmaxf(vm, vin[4 * st + i] < INFINITY ? vin[4 * st + i] : 0.0f);
          }
        }
      }
      const float before = m[nt];
      alpha[nt] = moved(nt, largest(sc[nt]));
      l[nt] *= alpha[nt];
      bool same = true;
      float w8[Q8 ? 4 * ST : 1];
      if constexpr (Q8) {
        vm = fmaxf(vm, xor16_f(vm));
        vm = fmaxf(vm, xor32_f(vm));
        const float ref = vm > 4.0f * vref[nt] ? vref_of(vm) : vref[nt];
        const float inv = inverse(ref);
        same = m[nt] == before && ref == vref[nt];
        alpha[nt] *= vref[nt] * inv;
        vref[nt] = ref;
#pragma unroll
        for (int i = 0; i < 4 * ST; ++i) w8[i] = vin[i] * inv;
      }
      es[nt] = weights(sc[nt], s2[nt], m[nt], w8, w[nt]);
      if constexpr (Q8) out[nt] = low_or_beyond(top[nt] * alpha[nt], largest_product(w[nt]), !same, t[nt]);
      else add(nt);
    }
    if constexpr (Q8) {
      bool any = false, any_lift = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) any |= out[nt];
      if (__builtin_expect(__ballot(any) != 0, 0)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float f = out[nt] ? lift(nt, t[nt]) : 1.0f;
#pragma unroll
          for (int i = 0; i < 4 * ST; ++i) w[nt][i] *= f;
          es[nt] *= f;
          l[nt] *= f;
          alpha[nt] *= f;
          t[nt] *= f;
        }
      }
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        top[nt] = t[nt];
        any_lift |= lag[nt] > kLag;
      }
      lifted = __ballot(any_lift) != 0;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) add(nt);
    }
    VPair v[NPAIR];
#pragma unroll
    for (int b = 0; b < NPAIR; ++b) v[b] = vread(at, 0, b);
    values(at, v, eh, el);
    next();
    // ---- the chunks of the prefix: every column sees every slot.  A chunk whose
    // scores or value scales have left the columns' references behind is with 8 bits
    // done above, as is every chunk while a column is lifted and its products have to
    // be watched; over f16 it is begun again after a rescale.  Either leaves the columns
    // that it does not move as they were.  (A column that a NaN or +inf has reached
    // asks for none of it: its queries may be those of rows past the drafts, which
    // hold anything.)
    int settled = -1;
    while (j < j_prefix && !lifted) {
      float mx[NT];
      for (;;) {
        const uint32_t at = lds0 + stage * SB;
        f32x4 sc[NT][ST];
        float vq[Q8 ? 4 * ST : 1];
        scores(at, sc, vq);
        bool over = false;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mx[nt] = largest(sc[nt]);
          over |= !(fmaf(mx[nt], s2[nt], -m[nt]) <= kLag) && m[nt] < INFINITY;
        }
        if constexpr (Q8) {
          float vm = 0.0f;  // the largest finite scale
#pragma unroll
          for (int i = 0; i < 4 * ST; ++i) vm = fmaxf(vm, vq[i] < INFINITY ? vq[i] : 0.0f);
          vm = fmaxf(vm, xor16_f(vm));
          vm = fmaxf(vm, xor32_f(vm));
          over |= vm > 4.0f * vref[0];
        }
        if ((Q8 || j != settled) && __ballot(over) != 0) break;
        VPair v[NPAIR];
#pragma unroll
        for (int b = 0; b < NPAIR; ++b) v[b] = vread(at, 0, b);
        float w8[Q8 ? 4 * ST : 1];
        if constexpr (Q8) {
          const float inv = inverse(vref[0]);  // (alike in every column)
#pragma unroll
          for (int i = 0; i < 4 * ST; ++i) w8[i] = vq[i] * inv;
        }
        __builtin_amdgcn_sched_barrier(0);
        h16x8 eh[NT][NE], el[NT][NE];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float w[4 * ST];
          l[nt] += weights(sc[nt], s2[nt], m[nt], w8, w);
          operand(w, eh[nt], el[nt]);
        }
        __builtin_amdgcn_sched_barrier(0);
        values(at, v, eh, el);
        next();
        if (j >= j_prefix) break;
      }
      if (Q8 || j >= j_prefix) break;
      settled = j;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float alpha = moved(nt, mx[nt]);
        l[nt] *= alpha;
        rescale(nt, alpha);
      }
    }
  }

  // ---- columns out: sums over the four lanes of a column, scales back in
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    l[nt] += xor16_f(l[nt]);
    l[nt] += xor32_f(l[nt]);
    if (spoilt[nt]) l[nt] = NAN;
    if constexpr (Q8) {
      // (a scale above 1 goes into the sum's unit, 2^-k of it against a reference k
      // higher: times the values it could pass f32; what the sum r + k is rounded by
      // goes into the factors)
      const float up = fmaxf(vref[nt], 1.0f), k = (float)((int)(__float_as_uint(up) >> 23) - 127);
      const float old = m[nt];
      m[nt] += k;
      const float part = m[nt] - old;
      const float f = fabsf(old) < INFINITY ? __builtin_amdgcn_exp2f((old - (m[nt] - part)) + (k - part)) : 1.0f;
      l[nt] *= inverse(up) * f;
      rescale(nt, fminf(vref[nt], 1.0f) * f);
    }
  }
  __builtin_amdgcn_s_waitcnt(0);  // the fetches past the range land before LDS is reused or given back
  if constexpr (WS > 1) {
    // the waves that shared the columns, in pairs: the upper half leaves its
    // registers in LDS, the lower half takes them in
    constexpr int WV = WC * NT;  // column tiles of one ws
    float4* ja = reinterpret_cast<float4*>(lds);
    float2* jm = reinterpret_cast<float2*>(lds + WS / 2 * WV * DT * 1024);
#pragma unroll
    for (int h = WS / 2; h >= 1; h >>= 1) {
      __syncthreads();
      if (ws >= h && ws < 2 * h) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int u = (ws - h) * WV + wc * NT + nt;
          jm[u * 64 + lane] = make_float2(m[nt], l[nt]);
#pragma unroll
          for (int dt = 0; dt < DT; ++dt)
            ja[(u * DT + dt) * 64 + lane] = make_float4(acc[nt][dt][0], acc[nt][dt][1], acc[nt][dt][2], acc[nt][dt][3]);
        }
      }
      __syncthreads();
      if (ws < h) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const int u = ws * WV + wc * NT + nt;
          const float2 ml = jm[u * 64 + lane];
          const float M = fmaxf(m[nt], ml.x), mr = M == -INFINITY ? 0.0f : M;
          const float fa = exp2f(m[nt] - mr), fb = exp2f(ml.x - mr);
          m[nt] = M;
          l[nt] = l[nt] * fa + ml.y * fb;
#pragma unroll
          for (int dt = 0; dt < DT; ++dt) {
            const float4 v = ja[(u * DT + dt) * 64 + lane];
            acc[nt][dt][0] = acc[nt][dt][0] * fa + v.x * fb;
            acc[nt][dt][1] = acc[nt][dt][1] * fa + v.y * fb;
            acc[nt][dt][2] = acc[nt][dt][2] * fa + v.z * fb;
            acc[nt][dt][3] = acc[nt][dt][3] * fa + v.w * fb;
          }
        }
      }
    }
    if (ws != 0) return;
  }
  // the results of a column, or its split record: the reference, the
  // sum and the weighted values.  A lane has dims 16 dt + 4 kq + i, or with 8 bits
  // 32 b + 8 kq + 2 i of tile 2b and the dims after those of tile 2b + 1.
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int col = tile * COLS + (wc * NT + nt) * 16 + r;
    if (col >= N * G) continue;
    float4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      if constexpr (Q8) {
        const f32x4 e = acc[nt][dt & ~1], f = acc[nt][dt | 1];
        o[dt] = (dt & 1) ? make_float4(e[2], f[2], e[3], f[3]) : make_float4(e[0], f[0], e[1], f[1]);
      } else {
        o[dt] = make_float4(acc[nt][dt][0], acc[nt][dt][1], acc[nt][dt][2], acc[nt][dt][3]);
      }
    }
    constexpr auto dim = [](int dt) { return Q8 ? 32 * (dt >> 1) + 4 * (dt & 1) : 16 * dt; };
    const int d0 = (Q8 ? 8 : 4) * kq;
    if (p.n_split > 1) {
      float* rec = a.partial + ((((uint64_t)s * nk + kvh) * p.n_split + split) * n_cols + col) * (D + 4);
      if (kq == 0) *reinterpret_cast<float2*>(rec) = make_float2(m[nt], l[nt]);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4*>(rec + 4 + d0 + dim(dt)) = o[dt];
      continue;
    }
    const float inv = l[nt] == 0.0f ? 0.0f : 1.0f / l[nt];  // nothing seen: zeros
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = make_float4(o[dt].x * inv, o[dt].y * inv, o[dt].z * inv, o[dt].w * inv);
    const int t = tcol[nt];  // (col is below N G: t is its own)
    const uint64_t to = ((uint64_t)s * a.n_rows + t) * a.out_stride + (uint64_t)(kvh * G + col - t * G) * D + d0;
    if constexpr (SPLIT) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4*>((float*)a.out + to + dim(dt)) = o[dt];
    } else if (a.type == KNJ_TYPE_F16) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<uint2*>((uint16_t*)a.out + to + dim(dt)) = pack4(KNJ_TYPE_F16, o[dt]);
    } else {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
        *reinterpret_cast<uint2*>((uint16_t*)a.out + to + dim(dt)) = pack4(KNJ_TYPE_BF16, o[dt]);
    }
  }
}

hipError_t launch_pages_step(const TreeArgs& a, const TreePlan& p, int cols, hipStream_t s);
hipError_t launch_pages_wide(const TreeArgs& a, const TreePlan& p, hipStream_t s);

// One launch of a format's kernel: D, split and the column tile's shape at run
// time (columns per kv head up to 16, 32, 64 or more).
template <int FORMAT>
hipError_t launch_format(const TreeArgs& a, const TreePlan& p, int cols, hipStream_t s);

#define KNJ_TREE_FORMAT(FORMAT)                                                                          \
  template <>                                                                                            \
  hipError_t launch_format<FORMAT>(const TreeArgs& a, const TreePlan& p, int cols, hipStream_t s) {      \
    const unsigned eights = (p.units + 7) / 8, y = eights < 32768u ? eights : 32768u;                    \
    const dim3 grid(8 * p.n_tiles, y, (eights + y - 1) / y);                                             \
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
// (Shapes of pages that are not built are those of launch_pages_step and launch_pages_wide; `plan`
// asserts that it gives none of them to this.)
#define KNJ_TREE_COLS(DD, FORMAT, SPLIT)                                                             \
  do {                                                                                               \
    if (cols == 16) {                                                                                \
      if constexpr (FORMAT != kFormatPages) KNJ_TREE_LAUNCH(DD, FORMAT, SPLIT, 1, 1, 4, 16);         \
      else return hipErrorInvalidValue;                                                              \
    } else if (cols == 32) {                                                                         \
      KNJ_TREE_LAUNCH(DD, FORMAT, SPLIT, 1, 2, 2, 32);                                               \
    } else if (SPLIT || cols == 64) {                                                                \
      KNJ_TREE_LAUNCH(DD, FORMAT, SPLIT, 2, 2, 2, 32);                                               \
    } else {                                                                                         \
      if constexpr (FORMAT != kFormatPages || DD == 64) KNJ_TREE_LAUNCH(DD, FORMAT, false, 2, 4, 1, 64); \
      else return hipErrorInvalidValue;                                                              \
    }                                                                                                \
  } while (0)
#define KNJ_TREE_LAUNCH(DD, FORMAT, SPLIT, NT, WC, WS, SW) \
  KNJ_LAUNCH((k_tree<DD, FORMAT, SPLIT, NT, WC, WS, SW>), grid, dim3(64 * WC * WS), 0, s, a, p)

}  // namespace tree
}  // namespace knj
