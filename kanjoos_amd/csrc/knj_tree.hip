// kanjoos_amd/csrc/knj_tree.hip -- plan, merge and launch of the drafts' attention.
#include <algorithm>

#include "knj_tree.h"

namespace knj {
namespace tree {

template <>
hipError_t launch_format<KNJ_KV_F16>(const TreeArgs&, const TreePlan&, int, hipStream_t);
template <>
hipError_t launch_format<KNJ_KV_F8>(const TreeArgs&, const TreePlan&, int, hipStream_t);
template <>
hipError_t launch_format<KNJ_KV_I8>(const TreeArgs&, const TreePlan&, int, hipStream_t);

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
  const int chunks = (P + N + chunk - 1) / chunk, used = p.by_cps.div(chunks + p.cps - 1);
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
  int cols;  // columns of a tile
};

// Tiles of 32 columns (16 where there are no more) finish a chunk soonest; wider ones
// read and decode the cache for more columns at once and win when there is work enough
// for every wave, counted in chunks of 32-column tiles.  Wide against narrow over e4m3,
// 16-bit queries: 64 drafts x 8 heads a kv head at 8,064, 12,096 and 16,064 chunks 40.0,
// 46.9 and 54.8 against 36.4, 48.8 and 59.5 us, 32 sequences of 8 drafts at 8,448 and
// 12,032 40.3 and 48.0 against 39.0 and 49.4 (int8 with f32 queries crosses there too);
// over f16, where nothing is decoded, 64 drafts at 12,096 and 16,064 38.8 and 44.4
// against 37.4 and 45.1, 25 at 14,028 and 28,028 43.5 and 69.0 against 40.9 and 72.3
// (with f32 queries between 12,000, for many sequences, and 30,000, for one).
// Two workgroups a CU where each then has several chunks, else one, with fewer records
// to merge: two against one for 16 drafts x 8 heads over 8,000, 12,000 and 16,000 f16
// slots (2,016, 3,008 and 4,016 chunks of tiles) 16.0, 18.3 and 20.6 against 15.6, 19.1
// and 22.2 us, over int8 with f32 queries 21.8, 25.4 and 29.5 against 22.5, 28.2 and 34.0;
// 4 drafts over 8,000 f16 slots (504) 16.8 against 12.5.
constexpr int64_t kWideWork = 10000, kWideWorkF16 = 16000, kTwoWork = 2500;  // chunks of 32-column tiles, chunks of tiles

Planned plan(const knj_kv_cache& c, int type, int n_head, int n_rows, int max_prefix) {
  const int group = n_head / c.n_head_kv, n_cols = n_rows * group;
  const int chunks = (max_prefix + n_rows + kTreeChunk - 1) / kTreeChunk;
  const int64_t units = (int64_t)c.n_seq * c.n_head_kv;
  int cols = n_cols <= 16 ? 16 : 32;
  if (n_cols > 32 && units * ((n_cols + 31) / 32) * chunks >= (c.format == KNJ_KV_F16 ? kWideWorkF16 : kWideWork))
    cols = n_cols <= 64 || type == KNJ_TYPE_F32 ? 64 : 128;
  const int tiles = (n_cols + cols - 1) / cols;
  const int64_t wgs = units * tiles * chunks >= kTwoWork ? 512 : 256;
  const int64_t want = std::max<int64_t>(1, wgs / (units * tiles));
  const int cps = (int)std::max<int64_t>(1, (chunks + want - 1) / want);
  const int n_split = (chunks + cps - 1) / cps;
  return {TreePlan{cps, n_split, tiles, (int)(units * n_split), FastDiv(c.n_head_kv), FastDiv(n_split), FastDiv(group),
                   FastDiv(n_head), FastDiv(n_rows), FastDiv(cps)},
          cols};
}

}  // namespace
}  // namespace tree

uint64_t tree_partial_bytes(const knj_kv_cache& c, int type, int n_head, int n_rows, int max_prefix) {
  const tree::Planned q = tree::plan(c, type, n_head, n_rows, max_prefix);
  if (q.p.n_split == 1) return 0;
  return (uint64_t)q.p.units * q.p.n_tiles * q.cols * (c.head_dim + 4) * sizeof(float);
}

hipError_t launch_attention_tree(const TreeArgs& a, hipStream_t s) {
  const tree::Planned q = tree::plan(a.c, a.type, a.n_head, a.n_rows, a.max_prefix);
  hipError_t e;
  if (a.c.format == KNJ_KV_F16) e = tree::launch_format<KNJ_KV_F16>(a, q.p, q.cols, s);
  else if (a.c.format == KNJ_KV_F8) e = tree::launch_format<KNJ_KV_F8>(a, q.p, q.cols, s);
  else e = tree::launch_format<KNJ_KV_I8>(a, q.p, q.cols, s);
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
             dim3(dev::kBlock), 0, s, a, q.p, tree::kTreeChunk, n_cols, n_out)
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
