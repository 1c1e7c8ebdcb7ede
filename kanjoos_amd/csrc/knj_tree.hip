// kanjoos_amd/csrc/knj_tree.hip -- plan, merge and launch of the drafts' attention.
#include <algorithm>
#include <string>

#include "knj_tree.h"

namespace knj {
namespace tree {

template <>
hipError_t launch_format<KNJ_KV_F16>(const TreeArgs&, const TreePlan&, int, hipStream_t);
template <>
hipError_t launch_format<KNJ_KV_F8>(const TreeArgs&, const TreePlan&, int, hipStream_t);
template <>
hipError_t launch_format<KNJ_KV_I8>(const TreeArgs&, const TreePlan&, int, hipStream_t);
template <>
hipError_t launch_format<kFormatPages>(const TreeArgs&, const TreePlan&, int, hipStream_t);

// Merge of a (draft, head)'s split records: M = max m, out = sum acc 2^(m - M) /
// sum l 2^(m - M).  Thread = four dims of every NP-th split, eight splits' loads at
// once, the parts added in order through LDS (NP 1: no parts, and a workgroup
// holds several outputs).  The loads do not wait for the sequence's length: every
// split has its place, and those that the sequence does not reach, which hold no
// record, are dropped afterwards.
// Bound by the records: 64 drafts x 32 heads of 32 splits (35 MB, written just before)
// 9.2 us, 3.8 TB/s; 4 drafts 3.3 us, a launch and one batch of loads.
template <int D, int NP>
__global__ __launch_bounds__(kBlock) void k_tree_merge(TreeArgs a, TreePlan p, int chunk, int n_cols, uint32_t n_out) {
  constexpr int ND = D / 4, B = 8, PER = kBlock / (ND * NP);
  __shared__ float pm[PER][NP], pl[PER][NP];
  __shared__ float4 pa[NP > 1 ? PER : 1][NP][ND];
  const int nk = a.c.n_head_kv, G = p.by_group.d;
  const int slot = threadIdx.x / (ND * NP), part = threadIdx.x / ND % NP, d = threadIdx.x % ND;
  const uint32_t at = blockIdx.x * PER + slot, out = min(at, n_out - 1);
  const uint32_t row = p.by_head.div(out), h = out - row * a.n_head;
  const uint32_t s = p.by_rows.div(row), t = row - s * a.n_rows, kvh = p.by_group.div(h);
  const float* rec = a.partial + (((uint64_t)s * nk + kvh) * p.n_split * n_cols + t * G + (h - kvh * G)) * (D + 4);
  const uint64_t stride = (uint64_t)n_cols * (D + 4);
  float2 ml[B];
  float4 v[B];
  auto fetch = [&](int i0) {
#pragma unroll
    for (int k = 0; k < B; ++k) {
      const int i = i0 + part + k * NP;
      ml[k] = make_float2(-INFINITY, 0.0f);
      if (i >= p.n_split) continue;
      ml[k] = *reinterpret_cast<const float2*>(rec + i * stride);
      v[k] = *reinterpret_cast<const float4*>(rec + i * stride + 4 + 4 * d);
    }
  };
  fetch(0);
  int P, N;
  seq_lengths(a, s, P, N);
  const int chunks = (P + N + chunk - 1) / chunk;
  int used;
  if (p.even) {
    const int cps = p.even_cps(chunks);
    used = (chunks + cps - 1) / cps;
  } else {
    used = p.by_cps.div(chunks + p.cps - 1);
  }
  float M = -INFINITY, L = 0.0f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < used; i0 += B * NP) {
    if (i0) fetch(i0);
    float Mn = M;
#pragma unroll
    for (int k = 0; k < B; ++k) {
      if (i0 + part + k * NP >= used) ml[k] = make_float2(-INFINITY, 0.0f);
      Mn = fmaxf(Mn, ml[k].x);
    }
    const float ref = Mn == -INFINITY ? 0.0f : Mn, fo = __builtin_amdgcn_exp2f(M - ref);
    L *= fo;
    o = make_float4(o.x * fo, o.y * fo, o.z * fo, o.w * fo);
#pragma unroll
    for (int k = 0; k < B; ++k) {
      if (i0 + part + k * NP >= used) continue;
      const float f = __builtin_amdgcn_exp2f(ml[k].x - ref);
      L += ml[k].y * f;
      o = make_float4(o.x + v[k].x * f, o.y + v[k].y * f, o.z + v[k].z * f, o.w + v[k].w * f);
    }
    M = Mn;
  }
  if constexpr (NP > 1) {
    if (d == 0) {
      pm[slot][part] = M;
      pl[slot][part] = L;
    }
    pa[slot][part][d] = o;
    __syncthreads();
    if (part != 0) return;
    M = pm[slot][0];
#pragma unroll
    for (int i = 1; i < NP; ++i) M = fmaxf(M, pm[slot][i]);
    const float ref = M == -INFINITY ? 0.0f : M;
    L = 0.0f;
    o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      const float f = __builtin_amdgcn_exp2f(pm[slot][i] - ref);
      const float4 x = pa[slot][i][d];
      L += pl[slot][i] * f;
      o = make_float4(o.x + x.x * f, o.y + x.y * f, o.z + x.z * f, o.w + x.w * f);
    }
  }
  if (at >= n_out || (int)t >= N) return;
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // nothing seen: zeros
  o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  const uint64_t to = (uint64_t)row * a.out_stride + (uint64_t)h * D + 4 * d;
  if (a.type == KNJ_TYPE_F32) *reinterpret_cast<float4*>((float*)a.out + to) = o;
  else *reinterpret_cast<uint2*>((uint16_t*)a.out + to) = pack4(a.type, o);
}

namespace {

constexpr int kTreeChunk = 64;  // slots of a chunk in every shape

struct Planned {
  TreePlan p;
  int cols;   // columns of a tile
  int chunk;  // slots of a split's chunks
  bool wide;  // launch_pages_wide's
};

// Tiles of 32 columns (16 where there are no more) finish a chunk soonest; wider ones
// read and decode the cache for more columns at once and win when there is work enough
// for every wave, counted in chunks of 32-column tiles.  Wide against narrow over e4m3,
// 16-bit queries: 64 drafts x 8 heads a kv head at 8,064, 12,096 and 16,064 chunks 40.0,
// 46.9 and 54.8 against 36.4, 48.8 and 59.5 us, 32 sequences of 8 drafts at 8,448 and
// 12,032 40.3 and 48.0 against 39.0 and 49.4 (int8 with f32 queries crosses there too);
// over f16, where nothing is decoded, 64 drafts at 12,096 and 16,064 38.8 and 44.4
// against 37.4 and 45.1, 25 at 14,028 and 28,028 43.5 and 69.0 against 40.9 and 72.3
// (with f32 queries between 12,000, for many sequences, and 30,000, for one); over 4-bit
// pages, where decoding costs most, 8 drafts x 8 heads of 32 sequences at 8,192, 12,288 and
// 16,384 35.9, 43.9 and 54.7 against 37.9, 48.3 and 60.1, heads of 64 at 8,192 and 33,250 25.0
// and 53.6 against 26.9 and 122 (at 4,032 18.3 against 19.4, with f32 queries 22.0 against 20.3).
// Two workgroups a CU where each then has several chunks, else one, with fewer records
// to merge: two against one for 16 drafts x 8 heads over 8,000, 12,000 and 16,000 f16
// slots (2,016, 3,008 and 4,016 chunks of tiles) 16.0, 18.3 and 20.6 against 15.6, 19.1
// and 22.2 us, over int8 with f32 queries 21.8, 25.4 and 29.5 against 22.5, 28.2 and 34.0;
// 4 drafts over 8,000 f16 slots (504) 16.8 against 12.5.
constexpr int64_t kWideWork = 10000, kWideWorkF16 = 16000, kWideWorkPages = 8000;  // chunks of 32-column tiles
constexpr int64_t kTwoWork = 2500;  // chunks of tiles

// Of launch_pages_step.  A wave's tile takes 1.0 us and a merge 3: one workgroup a unit up to
// four tiles a wave (32 sequences of 500 slots 10.2 us against 12.3 in four splits, 8 of
// 200 7.4 against 9.6 in two; 32 of 2000, 16 tiles a wave, 22.9 against 17.1).  Else two
// workgroups a CU (32 of 8000: 39.8 us; with one, three and four 44.6, 39.8 and 40.8) in up
// to 64 splits, one batch of the merge's loads (one sequence of 32,700: 13.9; in 128 splits
// 16.9, in 256 23.6).
// Columns 17 to 32 go there where that is work enough, or without a merge, and else, sooner
// done, to k_tree (below): 4 drafts x 8 heads a kv head, 16 and 32 sequences of 2000 slots
// (4,096 and 8,192 tiles) 18.8 and 23.5 us against 19.3 and 25.5, 16 of 1000 (2,048) 16.4
// against 14.3; without a merge 16 and 32 of 200 and 450 9.8 and 13.3 against 10.8 and 14.9,
// 8 of 300 11.1 against 9.6.
constexpr int kStepMerges = 16, kStepUnits = 64;
constexpr int64_t kStepWork = 4000;  // tiles
Planned plan_step(const knj_kv_cache& c, int n_head, int n_rows, int max_prefix) {
  const int tiles = (max_prefix + n_rows + kStepTile - 1) / kStepTile;
  const int64_t units = (int64_t)c.n_seq * c.n_head_kv;
  const int n_split = tiles <= kStepMerges ? 1 : (int)std::min<int64_t>({std::max<int64_t>(512 / units, 1), 64, tiles / kStepWaves});
  const FastDiv none(1);
  return {TreePlan{0, n_split, 1, (int)(units * n_split), FastDiv(c.n_head_kv), FastDiv(n_split),
                   FastDiv(n_head / c.n_head_kv), FastDiv(n_head), FastDiv(n_rows), none, true},
          n_rows * (n_head / c.n_head_kv) <= 16 ? 16 : 32, kStepTile, false};
}

// Of launch_pages_wide, for heads of 128 and more than 64 columns: two workgroups a CU (one and
// three: 141 and 129 us for 500 rows x 32 heads over 8000 slots, 121 with two).  It against
// k_tree, bf16, rows x query heads a kv head, in us:
// - where there is work enough, in chunks of 32-column tiles: at 5,400, 7,028, 8,064 and 9,216 of
//   them (25 drafts) 39.1, 32.1, 34.7 and 40.1 against 35.1, 33.7, 37.0 and 41.4 (f32 queries
//   cross at 8,000);
// - with more than 2,048 columns, 64 of k_tree's tiles, whatever the work: those of one split
//   and kv head share an XCD, whose 32 CUs hold two each.  At 2,080 (260 x 8 of 4 kv heads,
//   nothing before) 22.1 against 28.1, 2,240 (70 x 32 of one, 1,500 before) 30.5 and 30.9, 2,400
//   (300 x 8 of 4, 800 before) 30.0 and 56.7; at 1,920 (60 x 32 of one, 1,500 before) 27.4 and
//   19.6, 2,000 (250 x 8 of 4, 250 before; 500 x 4 of 8, 200 before) 25.9 and 34.5 against 22.4
//   and 30.2;
// - where it has no splits to merge, from 600 chunks on: 20 sequences of 32 x 8 of 4 behind 20
//   slots (640), 64 of 16 behind 16 (1,024) and 32 of 64 behind 64 (4,096) 10.6, 10.8 and 19.8
//   against 12.1, 14.4 and 31.5; 16 of 32 behind 30 (512) 10.3 against 8.5.  (In splits 4 of 100
//   behind 100, 1,600, take 25.0 against 14.7, 8 of 25 behind 900, 3,360, 25.3 against 21.5.)
// With a mask, which leaves no upper triangle out, they cross at the same places (2,000 and 2,080
// columns 26.8 and 23.6 against 22.7 and 28.9).
constexpr int64_t kPagesWork = 7000, kPagesUnsplit = 600;
constexpr int kPagesCols = 2048;
static_assert(kPagesWork <= kWideWorkPages && kPagesUnsplit <= kPagesWork,
              "over pages of heads of 128 k_tree has no tile of 128 columns: launch_pages_wide takes them first");
Planned plan_wide(const knj_kv_cache& c, int n_head, int n_rows, int max_prefix) {
  const int n_cols = n_rows * (n_head / c.n_head_kv), steps = (max_prefix + n_rows + kWideStep - 1) / kWideStep;
  const int cols = 16 * kWideWaves, tiles = (n_cols + cols - 1) / cols;
  const int64_t units = (int64_t)c.n_seq * c.n_head_kv, want = std::max<int64_t>(1, 512 / (units * tiles));
  const int cps = (int)std::max<int64_t>(1, (steps + want - 1) / want), n_split = (steps + cps - 1) / cps;
  return {TreePlan{cps, n_split, tiles, (int)(units * n_split), FastDiv(c.n_head_kv), FastDiv(n_split),
                   FastDiv(n_head / c.n_head_kv), FastDiv(n_head), FastDiv(n_rows), FastDiv(cps), false},
          cols, kWideStep, true};
}

Planned plan(const knj_kv_cache& c, int type, int n_head, int n_rows, int max_prefix) {
  const int group = n_head / c.n_head_kv, n_cols = n_rows * group;
  const int chunks = (max_prefix + n_rows + kTreeChunk - 1) / kTreeChunk;
  const int64_t units = (int64_t)c.n_seq * c.n_head_kv;
  const int64_t tiles32 = (max_prefix + n_rows + kStepTile - 1) / kStepTile;
  if (c.format == kFormatPages &&
      (n_cols <= 16 || (n_cols <= 32 && (units * tiles32 >= kStepWork || (tiles32 <= kStepMerges && units >= kStepUnits)))))
    return plan_step(c, n_head, n_rows, max_prefix);
  const int64_t work = units * ((n_cols + 31) / 32) * chunks;
  if (c.format == kFormatPages && c.head_dim == 128 && n_cols > 64) {
    const Planned q = plan_wide(c, n_head, n_rows, max_prefix);
    if (n_cols > kPagesCols || work >= (q.p.n_split == 1 ? kPagesUnsplit : kPagesWork)) return q;
  }
  int cols = n_cols <= 16 ? 16 : 32;
  const int64_t wide = c.format == KNJ_KV_F16 ? kWideWorkF16 : c.format == kFormatPages ? kWideWorkPages : kWideWork;
  if (n_cols > 32 && work >= wide)
    cols = n_cols <= 64 || type == KNJ_TYPE_F32 ? 64 : 128;
  const int tiles = (n_cols + cols - 1) / cols;
  const int64_t wgs = units * tiles * chunks >= kTwoWork ? 512 : 256;
  const int64_t want = std::max<int64_t>(1, wgs / (units * tiles));
  const int cps = (int)std::max<int64_t>(1, (chunks + want - 1) / want);
  const int n_split = (chunks + cps - 1) / cps;
  return {TreePlan{cps, n_split, tiles, (int)(units * n_split), FastDiv(c.n_head_kv), FastDiv(n_split), FastDiv(group),
                   FastDiv(n_head), FastDiv(n_rows), FastDiv(cps), false},
          cols, kTreeChunk, false};
}

}  // namespace
}  // namespace tree

uint64_t tree_partial_bytes(const knj_kv_cache& c, int type, int n_head, int n_rows, int max_prefix) {
  const tree::Planned q = tree::plan(c, type, n_head, n_rows, max_prefix);
  if (q.p.n_split == 1) return 0;
  return (uint64_t)q.p.units * q.p.n_tiles * q.cols * (c.head_dim + 4) * sizeof(float);
}

uint64_t tree_workspace(const knj_kv_cache& c, int n_head, int n_rows, int max_prefix) {
  if (n_head <= 0 || n_head > 1024 || n_head % c.n_head_kv || n_rows <= 0 || n_rows > 1024 || max_prefix < 0 ||
      (int64_t)max_prefix + n_rows > std::min<int64_t>(c.n_ctx, kMaxSlots))
    return 0;
  return std::max(tree_partial_bytes(c, KNJ_TYPE_F32, n_head, n_rows, max_prefix),
                  tree_partial_bytes(c, KNJ_TYPE_F16, n_head, n_rows, max_prefix));
}

int check_tree(const TreeArgs& a, uint64_t workspace_bytes, const char* what) {
  const int eb = act_bytes(a.type);
  KNJ_CHECK_ARG(eb, "activations must be F32, F16 or BF16");
  KNJ_CHECK_ARG(a.q && a.out && a.prefix, "null pointer");
  KNJ_CHECK_ARG(words_aligned(a.prefix, a.counts) && ((uintptr_t)a.mask & 7) == 0,
                "prefix, counts and mask must be aligned to their types");
  KNJ_CHECK_ARG(a.n_rows >= 0 && a.n_rows <= 1024, "n_rows must be in [0, 1024]");
  KNJ_CHECK_ARG(a.n_head > 0 && a.n_head <= 1024 && a.n_head % a.c.n_head_kv == 0,
                "n_head must be a positive multiple of n_head_kv, at most 1024");
  KNJ_CHECK_ARG(a.max_prefix >= 0 && (int64_t)a.max_prefix + a.n_rows <= a.c.n_ctx,
                "max_prefix and the drafts must fit into n_ctx");
  KNJ_CHECK_ARG((int64_t)a.max_prefix + a.n_rows <= kMaxSlots, "max_prefix and the drafts must stay below 2^31 - 256");
  KNJ_CHECK_ARG(a.scale >= 1e-6f && a.scale <= 1e6f, "the scale must be in [1e-6, 1e6]");
  KNJ_CHECK_ARG((uint64_t)a.c.n_seq * a.n_rows * a.n_head < (1ull << 31), "too many rows for one call");
  const uint64_t width = (uint64_t)a.n_head * a.c.head_dim;
  KNJ_CHECK_ARG(a.q_stride >= width && a.out_stride >= width, "a row stride is below the row's width");
  KNJ_CHECK_ARG(rows_aligned(a.q, a.q_stride, eb) && rows_aligned(a.out, a.out_stride, eb),
                "rows must start on 16-byte boundaries");
  KNJ_CHECK_ARG(a.q != a.out || a.q_stride == a.out_stride || (uint64_t)a.c.n_seq * a.n_rows <= 1,
                "an output in place takes its input's stride");
  const uint64_t need = a.n_rows ? tree_partial_bytes(a.c, a.type, a.n_head, a.n_rows, a.max_prefix) : 0;
  if (need && (!a.partial || workspace_bytes < need || ((uintptr_t)a.partial & 15))) {
    set_error(std::string(what) + ": these sizes need a 16-byte aligned workspace of " + std::to_string(need) + " bytes");
    return KNJ_E_ARG;
  }
  return KNJ_OK;
}

hipError_t launch_attention_tree(const TreeArgs& a, hipStream_t s) {
  const tree::Planned q = tree::plan(a.c, a.type, a.n_head, a.n_rows, a.max_prefix);
  hipError_t e;
  if (q.p.even) e = tree::launch_pages_step(a, q.p, q.cols, s);
  else if (q.wide) e = tree::launch_pages_wide(a, q.p, s);
  else if (a.c.format == KNJ_KV_F16) e = tree::launch_format<KNJ_KV_F16>(a, q.p, q.cols, s);
  else if (a.c.format == KNJ_KV_F8) e = tree::launch_format<KNJ_KV_F8>(a, q.p, q.cols, s);
  else if (a.c.format == KNJ_KV_I8) e = tree::launch_format<KNJ_KV_I8>(a, q.p, q.cols, s);
  else e = tree::launch_format<kFormatPages>(a, q.p, q.cols, s);
  if (e != hipSuccess || q.p.n_split == 1) return e;
  // Few outputs or many splits: the splits over a workgroup's parts, for latency (one
  // draft over 4000 f16 slots 10.4 us a call, 16.8 with one part; 8 over 32K int8 28.9
  // and 34.8).  Many outputs of up to eight splits, one batch of loads: one part (32 x 8
  // drafts at 2K 37.1 us, 46.6 with eight).
  const uint32_t n_out = (uint32_t)a.c.n_seq * a.n_rows * a.n_head;
  const int n_cols = q.p.n_tiles * q.cols;
  const bool wide = n_out <= 512 || q.p.n_split > 8;
#define KNJ_TREE_MERGE(DD, NP)                                                                                  \
  KNJ_LAUNCH((tree::k_tree_merge<DD, NP>), dim3((n_out + 1024 / (DD) / (NP) - 1) / (1024 / (DD) / (NP))),        \
             dim3(dev::kBlock), 0, s, a, q.p, q.chunk, n_cols, n_out)
  if (a.c.head_dim == 128) {
    if (wide) KNJ_TREE_MERGE(128, 8);
    else KNJ_TREE_MERGE(128, 1);
  } else {
    if (wide) KNJ_TREE_MERGE(64, 16);
    else KNJ_TREE_MERGE(64, 1);
  }
#undef KNJ_TREE_MERGE
  return hipGetLastError();
}

}  // namespace knj
