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
// sum l 2^(m - M).  Thread = four dims of every NP-th split, the parts added in
// order through LDS.  Only the splits that the sequence reaches hold a record.
template <int D>
__global__ __launch_bounds__(kBlock) void k_tree_merge(TreeArgs a, TreePlan p, int chunk, int n_cols) {
  constexpr int ND = D / 4, NP = kBlock / ND;
  __shared__ float pm[NP], pl[NP];
  __shared__ float4 pa[NP][ND];
  const int h = blockIdx.x % a.n_head;
  const uint32_t row = blockIdx.x / a.n_head;
  const int s = row / a.n_rows, t = row - s * a.n_rows;
  int P, N;
  seq_lengths(a, s, P, N);
  if (t >= N) return;
  const int chunks = (P + N + chunk - 1) / chunk, used = (chunks + p.cps - 1) / p.cps;
  const int nk = a.c.n_head_kv, G = a.n_head / nk, kvh = h / G;
  const float* rec = a.partial + (((uint64_t)s * nk + kvh) * p.n_split * n_cols + t * G + h % G) * (D + 4);
  const uint64_t stride = (uint64_t)n_cols * (D + 4);
  const int part = threadIdx.x / ND, d = threadIdx.x % ND;
  float M = -INFINITY, L = 0.0f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = part; i < used; i += NP) {
    const float2 ml = *reinterpret_cast<const float2*>(rec + i * stride);
    const float4 v = *reinterpret_cast<const float4*>(rec + i * stride + 4 + 4 * d);
    const float Mn = fmaxf(M, ml.x), ref = Mn == -INFINITY ? 0.0f : Mn;
    const float fo = exp2f(M - ref), fn = exp2f(ml.x - ref);
    L = L * fo + ml.y * fn;
    o = make_float4(o.x * fo + v.x * fn, o.y * fo + v.y * fn, o.z * fo + v.z * fn, o.w * fo + v.w * fn);
    M = Mn;
  }
  if (d == 0) {
    pm[part] = M;
    pl[part] = L;
  }
  pa[part][d] = o;
  __syncthreads();
  if (part != 0) return;
  M = pm[0];
#pragma unroll
  for (int i = 1; i < NP; ++i) M = fmaxf(M, pm[i]);
  const float ref = M == -INFINITY ? 0.0f : M;
  L = 0.0f;
  o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const float f = exp2f(pm[i] - ref);
    const float4 v = pa[i][d];
    L += pl[i] * f;
    o = make_float4(o.x + v.x * f, o.y + v.y * f, o.z + v.z * f, o.w + v.w * f);
  }
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;  // nothing seen: zeros
  o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
  const uint64_t to = (uint64_t)row * a.out_stride + (uint64_t)h * D + 4 * d;
  if (a.type == KNJ_TYPE_F32) *reinterpret_cast<float4*>((float*)a.out + to) = o;
  else *reinterpret_cast<uint2*>((uint16_t*)a.out + to) = pack4(a.type, o);
}

namespace {

// Columns of a tile and slots of a chunk, by the columns a kv head has in all.
struct Shape {
  int cols, chunk, waves;
};
Shape shape_of(int cols, bool split) {
  if (cols <= 16) return {16, 64, 4};
  if (cols <= 32) return {32, 64, 4};
  if (cols <= 64 || split) return {64, 64, 4};
  return {128, 64, 4};
}

// waves that the slots are split for: two per SIMD, what the registers admit
constexpr int kTreeWaves = 2048;

struct Planned {
  TreePlan p;
  Shape sh;
};
Planned plan(const knj_kv_cache& c, int type, int n_head, int n_rows, int max_prefix) {
  const int cols = n_rows * (n_head / c.n_head_kv);
  const Shape sh = shape_of(cols, type == KNJ_TYPE_F32);
  const int tiles = (cols + sh.cols - 1) / sh.cols;
  const int chunks = (max_prefix + n_rows + sh.chunk - 1) / sh.chunk;
  const int64_t base = (int64_t)c.n_seq * c.n_head_kv * tiles;
  const int64_t want = std::max<int64_t>(1, kTreeWaves / sh.waves / base);
  const int cps = (int)std::max<int64_t>(1, (chunks + want - 1) / want);
  const int n_split = (chunks + cps - 1) / cps;
  return {TreePlan{cps, n_split, tiles, (int)(c.n_seq * (int64_t)c.n_head_kv * n_split), FastDiv(c.n_head_kv),
                   FastDiv(n_split), FastDiv(n_head / c.n_head_kv)},
          sh};
}

}  // namespace
}  // namespace tree

uint64_t tree_partial_bytes(const knj_kv_cache& c, int type, int n_head, int n_rows, int max_prefix) {
  const tree::Planned q = tree::plan(c, type, n_head, n_rows, max_prefix);
  if (q.p.n_split == 1) return 0;
  return (uint64_t)q.p.units * q.p.n_tiles * q.sh.cols * (c.head_dim + 4) * sizeof(float);
}

hipError_t launch_attention_tree(const TreeArgs& a, hipStream_t s) {
  const tree::Planned q = tree::plan(a.c, a.type, a.n_head, a.n_rows, a.max_prefix);
  hipError_t e;
  if (a.c.format == KNJ_KV_F16) e = tree::launch_format<KNJ_KV_F16>(a, q.p, q.sh.cols, s);
  else if (a.c.format == KNJ_KV_F8) e = tree::launch_format<KNJ_KV_F8>(a, q.p, q.sh.cols, s);
  else e = tree::launch_format<KNJ_KV_I8>(a, q.p, q.sh.cols, s);
  if (e != hipSuccess || q.p.n_split == 1) return e;
  const dim3 grid((unsigned)((uint64_t)a.c.n_seq * a.n_rows * a.n_head));
  const int n_cols = q.p.n_tiles * q.sh.cols;
  if (a.c.head_dim == 128)
    KNJ_LAUNCH(tree::k_tree_merge<128>, grid, dim3(dev::kBlock), 0, s, a, q.p, q.sh.chunk, n_cols);
  else
    KNJ_LAUNCH(tree::k_tree_merge<64>, grid, dim3(dev::kBlock), 0, s, a, q.p, q.sh.chunk, n_cols);
  return hipGetLastError();
}

}  // namespace knj
