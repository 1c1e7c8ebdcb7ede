// kanjoos_amd/csrc/knj_pages_step.hip -- attention over 4-bit pages for up to 32 columns a kv
// head (a column is a row and a query head): decode steps and short chains of drafts.
#include "knj_pages_attn.h"

namespace knj {
namespace tree {
namespace {

// Workgroup = (sequence, split of the slots, kv head) of four waves that take its tiles of
// 32 slots in turn, each by itself: no barrier until the end.  A lane (r = l % 16, kq =
// l / 16) loads the part kq of rows r and 16 + r, decodes it, and, for NT times 16 columns,
//   scores  S[slot][col] = K (16 slots x 32 dims) x Q, keys from registers (a step's dims
//           are D/4 kq + 8 c ..: whichever order, as long as the queries have the same);
//   values  O^T[d][col] = V^T (16 dims x 32 slots) x E, the decoded rows through 9 KB of
//           LDS of the wave's own, read back transposed.
// The weights' reference, split and the records are k_tree's.  Registers are those of three
// waves a SIMD (held to four it spills: 32 sequences over 8000 slots 40.4 us a call against
// 39.1, over 500 10.2 against 9.9), with 17 to 32 columns of two.
//
// What bounds it (32 sequences of up to 8000 slots, 32 heads over 4 kv heads, 144 MB: 39 us a
// call, 3.7 TB/s; the loads alone, nothing decoded or multiplied, 34): 250 tiles a unit over
// two workgroups a CU, each wave some 280 vector instructions a tile of which 190 decode, in
// waves that the memory keeps waiting; 4 of the 39 are the merge.  A step over 1000 slots,
// 9.2 us, is one tile a wave (1.0 us), the prologue's chain of loads (lengths, table, rows)
// and two launches.  Four drafts instead of one cost 7 us more (46; k_tree, which shares a
// chunk's rows between waves behind barriers, 57); over 8000 slots in each sequence, 164 MB,
// four take 59.
template <int D, bool SPLIT, int NT>
__global__ __launch_bounds__(64 * kStepWaves, NT == 2 ? 2 : 3) void k_pages_step(TreeArgs a, TreePlan p) {
  using H = PageHead<D>;
  constexpr int NW = kStepWaves;
  constexpr int DT = D / 16, NC = D / 32;
  constexpr int RS = 2 * D + 32;       // from a row in LDS to the next: 8 rows' 32 bytes on banks of their own
  constexpr int LW = kStepTile * RS;   // bytes of a wave's LDS
  using Codes = std::conditional_t<D == 128, uint4, uint2>;
  __shared__ __align__(1024) uint8_t lds[NW * LW];
  __shared__ float2 stats[NW][16 * NT];

  const int nk = a.c.n_head_kv, G = p.by_group.d;
  const int unit = blockIdx.y * gridDim.x + blockIdx.x;
  if (unit >= p.units) return;
  const int rest = p.by_nk.div(unit), kvh = unit - rest * nk;
  const int s = p.by_split.div(rest), split = rest - s * p.n_split;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, kq = lane >> 4;

  // ---- a tile's rows as they are: of one matrix, fetched again as soon as the tile before
  // has been decoded.  The next tile's pages are looked up a tile ahead.
  // (what is constant while the kernel runs, by scalar loads, whatever asm lies between)
  typedef __attribute__((address_space(4))) const int32_t* Const;
  const Const table = (Const)(uintptr_t)(a.table + (uint64_t)s * a.n_table);
  const int given = ((Const)(uintptr_t)a.prefix)[s], count = a.counts ? ((Const)(uintptr_t)a.counts)[s] : a.n_rows;
  const int shift = a.page_shift, last = a.n_table - 1;
  const uint32_t head = (uint32_t)H::kSlot << shift;
  const uint32_t codes_at = r * H::kCode + (D / 8) * kq, words_at = r * H::kMeta + (D == 128 ? 4 * kq : 4 * (kq >> 1));
  struct Rows {
    Codes c[2];
    uint32_t w[2];
    bool in[2];  // (of the whole wave: a slot without a page holds NaN)
  };
  int page[2];             // of the next tile, and what follows from them:
  const uint8_t* base[2];  // its pages, and their first rows
  uint32_t row[2];
  bool in[2];
  auto look_up = [&](int j) {
#pragma unroll
    for (int st = 0; st < 2; ++st) page[st] = table[min((j * kStepTile + 16 * st) >> shift, last)];
  };
  auto place = [&](int j) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      in[st] = (uint32_t)page[st] < (uint32_t)a.n_page;
      base[st] = a.pages + (uint64_t)(uint32_t)((in[st] ? page[st] : 0) * nk + kvh) * head;
      row[st] = (j * kStepTile + 16 * st) & ((1 << shift) - 1);
    }
  };
  auto load = [&](int v, Rows& t) {
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      t.in[st] = in[st];
      const uint8_t* codes = base[st] + (H::codes(v, shift) + row[st] * H::kCode);
      const uint8_t* words = base[st] + (H::meta(v, shift) + row[st] * H::kMeta);
      // (scalar base and 32-bit offset: hoisted, the widened offset would take a register more)
      uint32_t c = codes_at, w = words_at;
      asm volatile("" : "+v"(c), "+v"(w));
      t.c[st] = *reinterpret_cast<const Codes*>(codes + c);
      t.w[st] = *reinterpret_cast<const uint32_t*>(words + w);
    }
  };
  Rows K, V;
  const int P = min(max(given, 0), a.max_prefix), N = min(max(count, 0), a.n_rows);
  const int valid = P + N, n_cols = 16 * NT;
  const int tiles = (valid + kStepTile - 1) / kStepTile, cps = p.even_cps(tiles);
  const int c0 = split * cps, c1 = min(tiles, c0 + cps);
  if (N == 0 || c0 >= c1) return;  // (all waves)
  int j = c0 + wave;
  look_up(j);
  place(j);
  load(1, V);
  load(0, K);
  look_up(j + NW < c1 ? j + NW : j);

  // ---- the queries, read row by row (a lane's own parts of its column lie in 64 lines) and
  // handed round in LDS.  Scaled by a power of two per column, as in k_tree.
  constexpr int QS = 2 * D + 16, QP = D / 8;  // from a column to the next in LDS; pieces of eight of a column
  static_assert((SPLIT ? 2 : 1) * 16 * NT * QS <= NW * LW, "the queries fit");
  __shared__ float scales[16 * NT];
  if (threadIdx.x < 16 * QP) {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int qc = 16 * nt + threadIdx.x / QP, piece = threadIdx.x % QP, c = min(qc, a.n_rows * G - 1), t = p.by_group.div(c);
      const uint64_t at = ((uint64_t)s * a.n_rows + t) * a.q_stride + (uint64_t)(kvh * G + c - t * G) * D + 8 * piece;
      float4 x, y;
      queries8<SPLIT>(a, at, x, y);
      float down;
      const float unit = column_unit(a.scale, group_max<QP>(largest8(x, y)), down);
      if (piece == 0) scales[qc] = unit;
      h16x8 hi, lo;
      pack_queries(x, y, down, hi, lo);
      lds_put_b128(lds_addr(lds) + qc * QS + 16 * piece, __builtin_bit_cast(uint4, hi));
      if constexpr (SPLIT) lds_put_b128(lds_addr(lds) + 16 * NT * QS + qc * QS + 16 * piece, __builtin_bit_cast(uint4, lo));
    }
  }
  KNJ_BARRIER_AFTER(kLdsOnly);
  int trow[NT];
  float s2[NT];
  h16x8 qh[NT][NC], ql[NT][SPLIT ? NC : 1];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    trow[nt] = p.by_group.div(min(16 * nt + r, a.n_rows * G - 1));
    s2[nt] = scales[16 * nt + r];
    const uint32_t from = lds_addr(lds) + (16 * nt + r) * QS + 16 * NC * kq;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      qh[nt][c] = lds_h8(from + 16 * c);
      if constexpr (SPLIT) ql[nt][c] = lds_h8(from + 16 * NT * QS + 16 * c);
    }
  }
  KNJ_BARRIER_AFTER(kLdsOnly);
  float m[NT], l[NT];
  f32x4 acc[NT][DT];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    m[nt] = -INFINITY;
    l[nt] = 0.0f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[nt][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const int words = (a.n_rows + 63) / 64;
  const uint64_t* mask = a.mask ? a.mask + (a.mask_shared ? 0 : (uint64_t)s * a.n_rows) * words : nullptr;

  const uint32_t mine = lds_addr(lds + wave * LW);
  const uint32_t put = mine + r * RS + (D / 2) * kq, get = mine + (4 * kq + (r >> 2)) * RS + 8 * (r & 3);

  auto words_of = [](const Codes& c, int i) {
    if constexpr (D == 128) return i == 0 ? c.x : i == 1 ? c.y : i == 2 ? c.z : c.w;
    else return i == 0 ? c.x : c.y;
  };
  for (; j < c1; j += NW) {
    // (after the last tile it is fetched once more: loads on every path are waited for by
    // their count, those on some only all at once)
    const int next = j + NW < c1 ? j + NW : j;
    const int p0 = j * kStepTile;
    const bool drafts = p0 + kStepTile > P;
    // the values' rows to LDS; of slots beyond the prefix what is not finite there is dropped,
    // and the rows that held it noted (slots past the rows are zeros; a prefix slot is seen
    // by every column and keeps its group's NaN)
    uint32_t bad = 0;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      hx2 step, low;
      const int slot = p0 + 16 * st + r;
      group_word(drafts && slot >= valid ? 0u : V.in[st] ? V.w[st] : kNanGroup, step, low);
      uint4 x[NC];
#pragma unroll
      for (int i = 0; i < NC; ++i) x[i] = decode8_mixed(words_of(V.c[st], i), step, low);
      if (drafts) {
        uint32_t any = 0;
        const uint32_t signs = slot >= P ? 0x80008000u : 0u;
#pragma unroll
        for (int i = 0; i < NC; ++i)
          any |= clear_nonfinite(x[i].x, signs) | clear_nonfinite(x[i].y, signs) | clear_nonfinite(x[i].z, signs) |
                 clear_nonfinite(x[i].w, signs);
        const uint64_t b = __ballot(any != 0);
        bad |= (uint32_t)((b | b >> 16 | b >> 32 | b >> 48) & 0xFFFF) << (16 * st);
      }
#pragma unroll
      for (int i = 0; i < NC; ++i) lds_put_b128(put + 16 * st * RS + 16 * i, x[i]);
    }
    place(next);
    load(1, V);
    __builtin_amdgcn_sched_barrier(0);
    // scores, in units of 1 / s2
    f32x4 sc[NT][2];
#pragma unroll
    for (int st = 0; st < 2; ++st) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) sc[nt][st] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      hx2 step, low;
      group_word(K.in[st] ? K.w[st] : kNanGroup, step, low);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const h16x8 ka = __builtin_bit_cast(h16x8, decode8_mixed(words_of(K.c[st], c), step, low));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          sc[nt][st] = mfma16(ka, qh[nt][c], sc[nt][st]);
          if constexpr (SPLIT) sc[nt][st] = mfma16(ka, ql[nt][c], sc[nt][st]);
        }
      }
    }
    load(0, K);
    look_up(j + 2 * NW < c1 ? j + 2 * NW : j + NW);
    __builtin_amdgcn_sched_barrier(0);
    if (drafts) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const uint64_t seen = seen64(mask ? mask + trow[nt] * words : nullptr, words, trow[nt], N, p0 - P);
        if (((uint32_t)seen & bad) != 0) l[nt] = NAN;  // (and stays so)
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (!((seen >> (16 * st + 4 * kq + i)) & 1)) sc[nt][st][i] = -INFINITY;
      }
    }
    // the reference moves where a score has passed it by kLag (a NaN or +inf carries)
    float mx[NT];
    bool over = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mx[nt] = max_nan(max_nan(max_nan(sc[nt][0][0], sc[nt][0][1]), max_nan(sc[nt][0][2], sc[nt][0][3])),
                       max_nan(max_nan(sc[nt][1][0], sc[nt][1][1]), max_nan(sc[nt][1][2], sc[nt][1][3])));
      over |= !(fmaf(mx[nt], s2[nt], -m[nt]) <= kLag) && m[nt] < INFINITY;
    }
    if (__ballot(over) != 0) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float2 m16 = pair16_f(mx[nt]);
        const float2 m32 = pair32_f(max_nan(m16.x, m16.y));
        const float most = max_nan(m32.x, m32.y), old = m[nt];
        if (!(fmaf(most, s2[nt], -old) <= kLag)) m[nt] = max_nan(old, fmaf(most, s2[nt], -kLift));
        const float alpha = __builtin_amdgcn_exp2f(old - (m[nt] == -INFINITY ? 0.0f : m[nt]));
        l[nt] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[nt][dt][i] *= alpha;
      }
    }
    // (the reference is -inf while the column has seen nothing: exponents then from 0)
    h16x8 eh[NT], el[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float mr = m[nt] == -INFINITY ? 0.0f : m[nt];
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = __builtin_amdgcn_exp2f(fmaf(sc[nt][i >> 2][i & 3], s2[nt], -mr));
        l[nt] += w[i];
      }
      split8(w, eh[nt], el[nt]);
    }
    // four tiles of dims at a time, read before they are multiplied
#pragma unroll
    for (int b0 = 0; b0 < DT; b0 += 4) {
      u32x2 v[4][2];
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        v[b][0] = lds_tr16_at(get + 32 * (b0 + b));
        v[b][1] = lds_tr16_at(get + 32 * (b0 + b) + 16 * RS);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const h16x8 vv = __builtin_bit_cast(h16x8, make_uint4(v[b][0].x, v[b][0].y, v[b][1].x, v[b][1].y));
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          acc[nt][b0 + b] = mfma16(vv, eh[nt], acc[nt][b0 + b]);
          acc[nt][b0 + b] = mfma16(vv, el[nt], acc[nt][b0 + b]);
        }
      }
    }
  }

  // ---- the waves joined, 16 columns at a time: each leaves them in its own LDS, each takes
  // dims of all
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    float sum = l[nt];
    sum += xor16_f(sum);
    sum += xor32_f(sum);
    if (kq == 0) stats[wave][16 * nt + r] = make_float2(m[nt], sum);
  }
  float4* mine4 = reinterpret_cast<float4*>(lds + wave * LW);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (nt) __syncthreads();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) mine4[64 * dt + lane] = in_order(acc[nt][dt]);
    __syncthreads();
    float M = -INFINITY, L = 0.0f, f[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) M = fmaxf(M, stats[w][16 * nt + r].x);
    const float mr = M == -INFINITY ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float2 ml = stats[w][16 * nt + r];
      f[w] = __builtin_amdgcn_exp2f(ml.x - mr);
      L += ml.y * f[w];
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // nothing seen: zeros
    const int ocol = 16 * nt + r;
    for (int dt = wave; dt < DT; dt += NW) {
      if (ocol >= N * G) continue;
      float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float4 x = reinterpret_cast<const float4*>(lds + w * LW)[64 * dt + lane];
        o = make_float4(o.x + x.x * f[w], o.y + x.y * f[w], o.z + x.z * f[w], o.w + x.w * f[w]);
      }
      const int d = 16 * dt + 4 * kq;
      if (p.n_split > 1) {
        float* rec = a.partial + ((((uint64_t)s * nk + kvh) * p.n_split + split) * n_cols + ocol) * (D + 4);
        if (dt == 0 && kq == 0) *reinterpret_cast<float2*>(rec) = make_float2(M, L);
        *reinterpret_cast<float4*>(rec + 4 + d) = o;
        continue;
      }
      o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
      const uint64_t to = ((uint64_t)s * a.n_rows + trow[nt]) * a.out_stride + (uint64_t)(kvh * G + ocol - trow[nt] * G) * D + d;
      if constexpr (SPLIT) *reinterpret_cast<float4*>((float*)a.out + to) = o;
      else *reinterpret_cast<uint2*>((uint16_t*)a.out + to) = pack4(a.type, o);
    }
  }
}

}  // namespace

hipError_t launch_pages_step(const TreeArgs& a, const TreePlan& p, int cols, hipStream_t s) {
  const unsigned y = (p.units + 65534u) / 65535u, x = (p.units + y - 1) / y;
#define KNJ_STEP(DD, SPLIT)                                                                                         \
  do {                                                                                                              \
    if (cols == 16) KNJ_LAUNCH((k_pages_step<DD, SPLIT, 1>), dim3(x, y), dim3(64 * kStepWaves), 0, s, a, p);        \
    else KNJ_LAUNCH((k_pages_step<DD, SPLIT, 2>), dim3(x, y), dim3(64 * kStepWaves), 0, s, a, p);                   \
  } while (0)
  const bool split = a.type == KNJ_TYPE_F32;
  if (a.c.head_dim == 128) {
    if (split) KNJ_STEP(128, true);
    else KNJ_STEP(128, false);
  } else {
    if (split) KNJ_STEP(64, true);
    else KNJ_STEP(64, false);
  }
#undef KNJ_STEP
  return hipGetLastError();
}

}  // namespace tree
}  // namespace knj
