// kanjoos_amd/csrc/knj_pages_wide.hip -- attention over 4-bit pages for many columns a kv head
// (a column is a row and a query head): trees of drafts over long caches, pieces of prompts.
#include "knj_pages_attn.h"

namespace knj {
namespace tree {
namespace {

// Heads of 128.  Workgroup = (sequence, split of the slots, kv head, tile of up to 128 columns) of
// eight waves of 16 columns each, over steps of 64 slots:
//   scores  S[slot][col] = K (16 slots x 32 dims) x Q (32 dims x 16 columns);
//   values  O^T[d][col] = V^T (16 dims x 32 slots) x E (32 slots x 16 columns),
// E the weights as f16 high parts and remainders.  Their reference, the splits and the records
// are k_tree's.
//
// All threads decode a step's rows into LDS, one group of 32 dims each, while the step before
// is computed: one barrier a step, the codes fetched two steps ahead, their pages looked up
// three (a wave's 16 rows are of one page: scalar).  Rows are padded by 32 bytes.
//
// What bounds it (500 rows x 32 heads over 8000 slots of 4 kv heads, 68 GFLOP and half
// as many for the remainders: 120 us a call, 8 of them the merge, 0.56 PFLOP/s): a SIMD's
// products take 43 % of its cycles and its other vector instructions 43 %, one after the
// other (a loop of a step's 48 products and 180 other instructions alone, four waves a SIMD:
// 344 and 311 ns a wave apart, 560 together).  Of a wave's vector instructions a
// step (180) 48 form the weights, 32 split them and 44 decode its share of the rows.  Hence
// many columns to a workgroup: k_tree with as many in four waves, which decode twice as much
// each, takes 135.  Nothing gained: codes by DMA, decoded behind the products or between
// them (138 to 151), four reads ahead of the products (121).
template <bool SPLIT>
__global__ __launch_bounds__(64 * kWideWaves, 4) void k_pages_wide(TreeArgs a, TreePlan p) {
  using H = PageHead<128>;
  constexpr int D = 128, S = kWideStep, DT = D / 16, NC = D / 32, ST = S / 16;
  constexpr int RS = 2 * D + 32, SB = S * RS;      // bytes of a row in LDS, of a matrix's step
  static_assert(2 * S * NC == 64 * kWideWaves && S == 64, "a group a thread");
  __shared__ __align__(16) uint8_t lds[4 * SB];    // keys and values of even steps, of odd steps
  __shared__ uint32_t poison[2][S / 16];           // rows of values of a step with what is not finite, 16 a word

  // (tiles of one unit on one XCD, as in k_tree)
  const int tile = blockIdx.x >> 3, unit = (blockIdx.z * gridDim.y + blockIdx.y) * 8 + (blockIdx.x & 7);
  if (unit >= p.units) return;
  const int nk = a.c.n_head_kv, G = p.by_group.d;
  const int rest = p.by_nk.div(unit), kvh = unit - rest * nk;
  const int s = p.by_split.div(rest), split = rest - s * p.n_split;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, kq = lane >> 4;
  int P, N;
  seq_lengths(a, s, P, N);
  const int valid = P + N, n_cols = p.n_tiles * 16 * kWideWaves;
  const int c0 = split * p.cps, steps = (valid + S - 1) / S;
  // the columns, 16 a wave, spread evenly over the tiles: a wave without any only decodes (25
  // drafts x 8 heads, 7 and 6 waves with some, over 32,700 slots 41.6 us a call; with 8 and 5, or
  // 8 and the last 3 computing what is not stored, 42.5 and 43.6)
  const int each = ((a.n_rows * G + 15) / 16 + p.n_tiles - 1) / p.n_tiles, col0 = 16 * (tile * each + wave);
  const bool mine = wave < each && col0 < N * G;
  if (16 * tile * each >= N * G || c0 >= steps) return;
  // slots before `all` are seen by every row of the tile; a chain's tile goes no further than
  // its last row (a split that begins behind it has an empty record)
  const int row_0 = p.by_group.div(16 * tile * each), row_1 = p.by_group.div(min(16 * (tile + 1) * each, N * G) - 1);
  const int all = a.mask ? P : P + row_0 + 1;
  const int c1 = min(min(a.mask ? steps : (P + row_1) / S + 1, steps), c0 + p.cps);

  // ---- this thread's group of a step: of keys (waves 0 to 3) or values, 16 rows a wave
  const int last = a.n_table - 1, shift = a.page_shift;
  typedef __attribute__((address_space(4))) const int32_t* Const;
  const Const table = (Const)(uintptr_t)(a.table + (uint64_t)s * a.n_table);
  const uint32_t head = (uint32_t)H::kSlot << shift;
  const int matrix = wave >> 2, row0 = 16 * (wave & 3), row = row0 + (lane >> 2), group = lane & 3;
  uint4 code;
  uint32_t word;
  bool in;
  int page;
  auto look_up = [&](int x) __attribute__((always_inline)) { page = table[min((x * S + row0) >> shift, last)]; };
  auto fetch = [&](int x) __attribute__((always_inline)) {
    in = (uint32_t)page < (uint32_t)a.n_page;
    const uint8_t* base = a.pages + (uint64_t)(uint32_t)((in ? page : 0) * nk + kvh) * head;
    const uint32_t slot = ((x * S + row0) & ((1 << shift) - 1)) + (lane >> 2);
    code = *reinterpret_cast<const uint4*>(base + H::codes(matrix, shift) + slot * H::kCode + 16 * group);
    word = *reinterpret_cast<const uint32_t*>(base + H::meta(matrix, shift) + slot * H::kMeta + 4 * group);
  };
  // Step x's group, decoded, into its buffer.  Of values behind the prefix what is not finite
  // is dropped and the rows that held it noted; slots past the rows are zeros.  (A prefix slot
  // is seen by every column and keeps its group's NaN.)
  const uint32_t put_at = lds_addr(lds) + matrix * SB + row * RS + 64 * group;
  auto put = [&](int x) __attribute__((always_inline)) {
    const bool drafts = matrix == 1 && (x + 1) * S > P;
    hx2 st, low;
    const uint32_t w = in ? word : kNanGroup;
    group_word((drafts & (x * S + row >= valid)) ? 0u : w, st, low);
    uint4 v[4] = {decode8_mixed(code.x, st, low), decode8_mixed(code.y, st, low),
                  decode8_mixed(code.z, st, low), decode8_mixed(code.w, st, low)};
    if (drafts) {
      uint32_t any = 0;
      const uint32_t signs = x * S + row >= P ? 0x80008000u : 0u;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        any |= clear_nonfinite(v[k].x, signs) | clear_nonfinite(v[k].y, signs) | clear_nonfinite(v[k].z, signs) |
               clear_nonfinite(v[k].w, signs);
      uint64_t b = __ballot(any != 0);  // four bits a row: into one
      b |= b >> 1;
      b |= b >> 2;
      uint32_t rows = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) rows |= (uint32_t)((b >> (4 * k)) & 1) << k;
      if (lane == 0) poison[x & 1][row0 / 16] = rows;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) lds_put_b128(put_at + 2 * (x & 1) * SB + 16 * k, v[k]);
  };
  look_up(c0);
  fetch(c0);
  look_up(c0 + 1);

  // ---- this lane's query column: step c's dims 32 c + 8 kq .. + 7, in decode8_mixed's order
  const int col = col0 + r, ccol = min(col, a.n_rows * G - 1);  // (past the rows: not stored)
  const int trow = p.by_group.div(ccol);
  h16x8 qh[NC], ql[NC];
  const float s2 = column<D, SPLIT>(
      a, ((uint64_t)s * a.n_rows + trow) * a.q_stride + (uint64_t)(kvh * G + ccol - trow * G) * D + 8 * kq, 32, qh, ql);

  float m = -INFINITY, l = 0.0f;
  f32x4 acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  const int words = (a.n_rows + 63) / 64;
  const uint64_t* mask = a.mask ? a.mask + (a.mask_shared ? 0 : (uint64_t)s * a.n_rows) * words : nullptr;
  const uint32_t kat = lds_addr(lds) + r * RS + 16 * kq;
  const uint32_t vat = lds_addr(lds) + SB + (4 * kq + (r >> 2)) * RS + 8 * (r & 3);

  put(c0);
  fetch(c0 + 1);
  look_up(c0 + 2);
  for (int h = c0; h < c1; ++h) {
    KNJ_BARRIER_AFTER(kLdsOnly);
    if (mine) {
      const uint32_t stage = 2 * (h & 1) * SB;
      f32x4 sc[ST];
#pragma unroll
      for (int st = 0; st < ST; ++st) sc[st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int st = 0; st < ST; ++st) {
          const h16x8 ka = lds_h8(kat + stage + 16 * st * RS + 64 * c);
          sc[st] = mfma16(ka, qh[c], sc[st]);
          if constexpr (SPLIT) sc[st] = mfma16(ka, ql[c], sc[st]);
        }
      if (__builtin_expect((h + 1) * S > P, 0)) {
        uint64_t seen = ~0ull, bad = 0;
#pragma unroll
        for (int st = 0; st < ST; ++st) bad |= (uint64_t)poison[h & 1][st] << (16 * st);
        if ((h + 1) * S > all) {
          seen = seen64(mask ? mask + (uint64_t)trow * words : nullptr, words, trow, N, h * S - P);
#pragma unroll
          for (int st = 0; st < ST; ++st)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (!((seen >> (16 * st + 4 * kq + i)) & 1)) sc[st][i] = -INFINITY;
        }
        if ((seen & bad) != 0) l = NAN;  // (and stays so)
      }
      // a weight beyond 2^kLag shows in the sum (and a column that has seen nothing yet in its
      // reference, -inf): the reference is moved and the weights formed again
      float w[4 * ST], sum;
      auto weights = [&]() __attribute__((always_inline)) {
        const float mr = m == -INFINITY ? 0.0f : m;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * ST; ++i) {
          w[i] = __builtin_amdgcn_exp2f(fmaf(sc[i >> 2][i & 3], s2, -mr));
          sum += w[i];
        }
      };
      weights();
      if (__builtin_expect(__ballot((!(sum <= 0x1p13f) | (m == -INFINITY)) & (m < INFINITY)) != 0, 0)) {
        float mx = -INFINITY;
#pragma unroll
        for (int st = 0; st < ST; ++st)
          mx = max_nan(max_nan(max_nan(mx, sc[st][0]), max_nan(sc[st][1], sc[st][2])), sc[st][3]);
        const float2 m16 = pair16_f(mx);
        const float2 m32 = pair32_f(max_nan(m16.x, m16.y));
        mx = max_nan(m32.x, m32.y);
        const float old = m;
        if (!(fmaf(mx, s2, -old) <= kLag)) m = max_nan(old, fmaf(mx, s2, -kLift));
        const float alpha = __builtin_amdgcn_exp2f(old - (m == -INFINITY ? 0.0f : m));
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[dt][i] *= alpha;
        weights();
      }
      l += sum;
      h16x8 eh[ST / 2], el[ST / 2];
#pragma unroll
      for (int e = 0; e < ST / 2; ++e) {
        const float x[8] = {w[8 * e], w[8 * e + 1], w[8 * e + 2], w[8 * e + 3], w[8 * e + 4], w[8 * e + 5], w[8 * e + 6], w[8 * e + 7]};
        split8(x, eh[e], el[e]);
      }
#pragma unroll
      for (int e = 0; e < ST / 2; ++e)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
          const uint32_t at = vat + stage + 32 * e * RS + 32 * dt;
          const u32x2 v0 = lds_tr16_at(at), v1 = lds_tr16_at(at + 16 * RS);
          const h16x8 v = __builtin_bit_cast(h16x8, make_uint4(v0.x, v0.y, v1.x, v1.y));
          acc[dt] = mfma16(v, eh[e], acc[dt]);
          acc[dt] = mfma16(v, el[e], acc[dt]);
        }
    }
    put(h + 1);
    fetch(h + 2);
    look_up(h + 3);
  }

  // ---- results, or a split's record
  l += xor16_f(l);
  l += xor32_f(l);
  float4 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = in_order(acc[dt]);
  if (!mine || col >= N * G) return;
  if (p.n_split > 1) {
    float* rec = a.partial + ((((uint64_t)s * nk + kvh) * p.n_split + split) * n_cols + col) * (D + 4);
    if (kq == 0) *reinterpret_cast<float2*>(rec) = make_float2(m, l);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<float4*>(rec + 4 + 16 * dt + 4 * kq) = o[dt];
    return;
  }
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // nothing seen: zeros
  const uint64_t to = ((uint64_t)s * a.n_rows + trow) * a.out_stride + (uint64_t)(kvh * G + col - trow * G) * D + 4 * kq;
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) {
    const float4 v = make_float4(o[dt].x * inv, o[dt].y * inv, o[dt].z * inv, o[dt].w * inv);
    if constexpr (SPLIT) *reinterpret_cast<float4*>((float*)a.out + to + 16 * dt) = v;
    else *reinterpret_cast<uint2*>((uint16_t*)a.out + to + 16 * dt) = pack4(a.type, v);
  }
}

}  // namespace

hipError_t launch_pages_wide(const TreeArgs& a, const TreePlan& p, hipStream_t s) {
  const unsigned eights = (p.units + 7) / 8, y = eights < 32768u ? eights : 32768u;
  const dim3 grid(8 * p.n_tiles, y, (eights + y - 1) / y);
  if (a.type == KNJ_TYPE_F32) KNJ_LAUNCH((k_pages_wide<true>), grid, dim3(64 * kWideWaves), 0, s, a, p);
  else KNJ_LAUNCH((k_pages_wide<false>), grid, dim3(64 * kWideWaves), 0, s, a, p);
  return hipGetLastError();
}

}  // namespace tree
}  // namespace knj
