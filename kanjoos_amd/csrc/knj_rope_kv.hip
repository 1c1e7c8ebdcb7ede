// kanjoos_amd/csrc/knj_rope_kv.hip -- rotary positions of query and key rows, and cache rows
// written in f16 or 8 bits and read back.
//
// Both are streams over rows of heads: a group of D/8 lanes holds one head's row (of
// a cache its key and its value), eight elements a lane, so a head's reductions (the
// norm's sum, the largest magnitude) stay inside the group's DPP moves and every
// element is read and written once.
#include <algorithm>
#include <cmath>
#include <string>

#include "knj_common.h"
#include "knj_dev.h"

namespace knj {
namespace {

using namespace dev;

// Eight consecutive activations as f32 (16-byte aligned rows; 4 at a time for
// the halves of a rotation).
template <int TYPE>
__device__ __forceinline__ float4 ld4(const void* p, uint64_t i) {
  if constexpr (TYPE == KNJ_TYPE_F32) {
    return *reinterpret_cast<const float4*>((const float*)p + i);
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>((const uint16_t*)p + i);
    if constexpr (TYPE == KNJ_TYPE_F16)
      return make_float4(h2f(u.x), h2f(u.x >> 16), h2f(u.y), h2f(u.y >> 16));
    else
      return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                         __uint_as_float(u.y & 0xFFFF0000u));
  }
}

template <int TYPE>
__device__ __forceinline__ void st4(void* p, uint64_t i, float4 v) {
  if constexpr (TYPE == KNJ_TYPE_F32)
    *reinterpret_cast<float4*>((float*)p + i) = v;
  else
    *reinterpret_cast<uint2*>((uint16_t*)p + i) = make_uint2(pack_act<TYPE>(v.x, v.y), pack_act<TYPE>(v.z, v.w));
}

// ---------------------------------------------------------------- rotary positions
// y = R(pos) (x / sqrt(mean x^2 + eps) * w).  A lane holds both elements of its
// four pairs: elements 4c.. of the rotated part's two halves (HALF) or eight
// consecutive ones; lanes past the rotated part hold eight that pass.  The cos
// and sin of the row's angles are formed once per workgroup: the product
// pos * f and its reduction to [-pi, pi] in f64 (an f32 product is off by
// pos * 2^-24 radians, 0.06 at a million), the functions in f32 on the reduced
// angle's f32 part a, with its remainder d (up to 2^-23, which alone would cost an
// angle near pi a bit) by cos(a + d) = cos a - d sin a, sin(a + d) = sin a + d cos a.
//
// Bound by memory: 4000 rows of 36 f32 heads of 128 (147 MB in and out) 30.8 us a call,
// 4.8 TB/s, where a large copy reaches 5.1; of bf16 (74 MB) 18.1, 4.1 TB/s: a row's three
// workgroups form the same angles.  One row is a launch: 2.3 us on the chip.
template <int TYPE, int LAYOUT, int D>
__global__ __launch_bounds__(kBlock) void k_rope(RopeArgs a) {
  constexpr int T = D / 8, HPB = kBlock / T;
  __shared__ float cs[D / 2], sn[D / 2];
  const int row = blockIdx.x;
  const int nh = a.n_head + a.n_head_kv, half = a.n_rot / 2;
  const int hh = blockIdx.y * HPB + threadIdx.x / T, c = threadIdx.x % T;
  const int hc = min(hh, nh - 1);  // every lane computes; lanes past the heads store nothing
  const bool is_q = hc < a.n_head;
  const int h = is_q ? hc : hc - a.n_head;
  const bool rot = 8 * c < a.n_rot;
  // elements e0..e0+3 and e1..e1+3 of the head
  const int e0 = (LAYOUT == KNJ_ROPE_HALF && rot) ? 4 * c : 8 * c;
  const int e1 = (LAYOUT == KNJ_ROPE_HALF && rot) ? half + 4 * c : 8 * c + 4;
  const void* src = is_q ? a.q : a.k;
  const uint64_t at = (uint64_t)row * (is_q ? a.q_stride : a.k_stride) + (uint64_t)h * D;
  float4 x = ld4<TYPE>(src, at + e0), y = ld4<TYPE>(src, at + e1);
  const float* nw = is_q ? a.q_norm : a.k_norm;
  float4 wx = make_float4(1.f, 1.f, 1.f, 1.f), wy = wx;
  if (nw) {
    wx = *reinterpret_cast<const float4*>(nw + e0);
    wy = *reinterpret_cast<const float4*>(nw + e1);
  }
  if ((int)threadIdx.x < half) {
    const double t = (double)a.pos[row] * a.inv_freq[threadIdx.x];
    const double n = rint(t * 0.15915494309189535);            // turns
    double r = fma(-n, 6.283185307179586, t);                   // 2 pi in two parts
    r = fma(-n, 2.4492935982947064e-16, r);
    const float near = (float)r, d = (float)(r - (double)near);
    float s, co;
    sincosf(near, &s, &co);
    cs[threadIdx.x] = fmaf(-d, s, co) * a.mscale;
    sn[threadIdx.x] = fmaf(d, co, s) * a.mscale;
  }
  float ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
  ss = group_sum<T>(ss);
  if (nw) {
    float g = 1.0f / sqrtf(ss / (float)D + a.eps);
    // (squares beyond f32, or lost below it: again with the head's largest near 1)
    const bool far = !(ss <= 0x1p100f) || ss < 0x1p-60f;
    if (__builtin_expect(__ballot(far) != 0, 0)) {
      float am = fmaxf(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))),
                       fmaxf(fmaxf(fabsf(y.x), fabsf(y.y)), fmaxf(fabsf(y.z), fabsf(y.w))));
      am = group_max<T>(am);
      const int e = far ? min(max((int)(__float_as_uint(am) >> 23) - 127, -126), 126) : 0;
      const float down = __uint_as_float((uint32_t)(127 - e) << 23);
      x = make_float4(x.x * down, x.y * down, x.z * down, x.w * down);
      y = make_float4(y.x * down, y.y * down, y.z * down, y.w * down);
      ss = x.x * x.x + x.y * x.y + x.z * x.z + x.w * x.w + y.x * y.x + y.y * y.y + y.z * y.z + y.w * y.w;
      ss = group_sum<T>(ss);
      if (far) g = (float)(1.0 / sqrt((double)ss / D + ldexp((double)a.eps, -2 * e)));
    }
    x = make_float4(x.x * g * wx.x, x.y * g * wx.y, x.z * g * wx.z, x.w * g * wx.w);
    y = make_float4(y.x * g * wy.x, y.y * g * wy.y, y.z * g * wy.z, y.w * g * wy.w);
  }
  __syncthreads();
  if (rot) {
    const float4 co = *reinterpret_cast<const float4*>(cs + 4 * c), si = *reinterpret_cast<const float4*>(sn + 4 * c);
    const float4 u = x, v = y;
    if constexpr (LAYOUT == KNJ_ROPE_HALF) {
      x = make_float4(u.x * co.x - v.x * si.x, u.y * co.y - v.y * si.y, u.z * co.z - v.z * si.z, u.w * co.w - v.w * si.w);
      y = make_float4(u.x * si.x + v.x * co.x, u.y * si.y + v.y * co.y, u.z * si.z + v.z * co.z, u.w * si.w + v.w * co.w);
    } else {
      x = make_float4(u.x * co.x - u.y * si.x, u.x * si.x + u.y * co.x, u.z * co.y - u.w * si.y, u.z * si.y + u.w * co.y);
      y = make_float4(v.x * co.z - v.y * si.z, v.x * si.z + v.y * co.z, v.z * co.w - v.w * si.w, v.z * si.w + v.w * co.w);
    }
  }
  if (hh >= nh) return;
  void* dst = is_q ? a.q_out : a.k_out;
  const uint64_t to = (uint64_t)row * (is_q ? a.q_out_stride : a.k_out_stride) + (uint64_t)h * D;
  st4<TYPE>(dst, to + e0, x);
  st4<TYPE>(dst, to + e1, y);
}

// ---------------------------------------------------------------- cache rows
// rint(x * top / amax * rstep) of the exact quotient, ties to even (rstep a power
// of two, the result at most 127); `inv` is top / amax.  The f32 product with it is
// off by 2^-23 of itself, 1.6e-5, which decides a rounding only next to a tie:
// there the quotient is divided out in f64 (x * top * rstep is exact, and a division
// that is correctly rounded gives the tie itself for a quotient that is one).
__device__ __forceinline__ float quotient_code(float x, float inv, double top, float amax, float rstep) {
  const float z = x * inv * rstep;
  float t = rintf(z);
  if (fabsf(fabsf(z - t) - 0.5f) < 1e-4f) t = (float)rint((double)x * top * (double)rstep / (double)amax);
  return t;
}

// Where unit u of a sequence's rows (a row's kv head: its key and its value) lies:
// T lanes hold eight elements of each.
template <int T>
struct Unit {
  uint32_t t;  // row
  int h, lane;
  bool in;     // a unit there is (the lanes past the last repeat it and store nothing)
  __device__ __forceinline__ Unit(const KvRowsArgs& a) {
    const uint32_t nk = a.c.n_head_kv, total = (uint32_t)a.n_rows * nk;
    const uint32_t u = blockIdx.x * (kBlock / T) + threadIdx.x / T;
    in = u < total;
    const uint32_t v = in ? u : total - 1;
    t = v / nk;
    h = (int)(v - t * nk);
    lane = threadIdx.x % T;
  }
};

// Eight values of a head's row as codes, and the row's scale, by its T lanes.
template <int FORMAT, int T>
__device__ __forceinline__ uint2 quantise8(const float (&x)[8], float& scale) {
  constexpr double kTop = FORMAT == KNJ_KV_I8 ? 127.0 : 448.0;
  float amax = 0.0f;
  bool bad = false;  // an infinity or a NaN
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    amax = fmaxf(amax, fabsf(x[i]));
    bad |= !(fabsf(x[i]) < INFINITY);
  }
  amax = group_max<T>(amax);
  bad = group_max<T>(bad ? 1.0f : 0.0f) != 0.0f;
  const bool live = !bad && amax >= 0x1p-119f;
  const float inv = live ? (float)kTop / amax : 0.0f;
  scale = bad ? NAN : live ? amax / (float)kTop : 0.0f;
  uint2 o;
  if constexpr (FORMAT == KNJ_KV_I8) {
    int w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = (int)quotient_code(live ? x[i] : 0.0f, inv, kTop, amax, 1.0f);
    o.x = (w[0] & 255) | ((w[1] & 255) << 8) | ((w[2] & 255) << 16) | ((uint32_t)w[3] << 24);
    o.y = (w[4] & 255) | ((w[5] & 255) << 8) | ((w[6] & 255) << 16) | ((uint32_t)w[7] << 24);
  } else {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // e4m3: three bits after the leading one, steps of 2^-9 below 2^-6
      const float xi = live ? x[i] : 0.0f;
      const int e = max((int)((__float_as_uint(xi * inv) >> 23) & 0xFF) - 127, -6);
      const float step = __uint_as_float((uint32_t)(127 + e - 3) << 23);
      const float rstep = __uint_as_float((uint32_t)(127 - e + 3) << 23);
      f[i] = quotient_code(xi, inv, kTop, amax, rstep) * step;  // a value of e4m3
    }
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(f[0], f[1], 0, false);
    const int hi = __builtin_amdgcn_cvt_pk_fp8_f32(f[4], f[5], 0, false);
    o.x = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[2], f[3], lo, true);
    o.y = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(f[6], f[7], hi, true);
  }
  return o;
}

// Rows of `FORMAT` from rows of activations; blockIdx.y is the sequence.  The same
// lanes take a head's key and its value, so that the two reductions and divisions
// run side by side (a group for each matrix was 9 % slower): 4096 rows of 4 f32 heads
// of 128 as e4m3 7.0 us.  That is 21 MB, 4.1 us at a copy's rate: the rest is one
// pass of latency (loads, two maxima over 16 lanes, a division, stores) of 1024
// workgroups that are all resident at once; 32 sequences' one row 3.3 us.
template <int TYPE, int FORMAT, int D>
__global__ __launch_bounds__(kBlock) void k_kv_store(KvRowsArgs a) {
  const knj_kv_cache& c = a.c;
  const Unit<D / 8> u(a);
  const uint32_t s = blockIdx.y;
  const uint64_t at = ((uint64_t)s * a.n_rows + u.t) * a.row_stride + (uint64_t)u.h * D + 8 * u.lane;
  const float4 k0 = ld4<TYPE>(a.k, at), k1 = ld4<TYPE>(a.k, at + 4);
  const float4 v0 = ld4<TYPE>(a.v, at), v1 = ld4<TYPE>(a.v, at + 4);
  const int64_t slot = (int64_t)a.index[s] + u.t;
  const bool keep = u.in && slot >= 0 && slot < c.n_ctx && (!a.counts || (int64_t)u.t < a.counts[s]);
  const uint64_t row = (uint64_t)u.h * c.n_ctx + slot;
  const uint64_t to = (uint64_t)s * c.seq_stride + row * D + 8 * u.lane;
  const float k[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
  const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
  if constexpr (FORMAT == KNJ_KV_F16) {
    if (!keep) return;
    auto pack = [](const float (&x)[8]) {
      return make_uint4(pack_act<KNJ_TYPE_F16>(x[0], x[1]), pack_act<KNJ_TYPE_F16>(x[2], x[3]),
                        pack_act<KNJ_TYPE_F16>(x[4], x[5]), pack_act<KNJ_TYPE_F16>(x[6], x[7]));
    };
    *reinterpret_cast<uint4*>((uint16_t*)c.k + to) = pack(k);
    *reinterpret_cast<uint4*>((uint16_t*)c.v + to) = pack(v);
  } else {
    float ks, vs;
    const uint2 kw = quantise8<FORMAT, D / 8>(k, ks), vw = quantise8<FORMAT, D / 8>(v, vs);
    if (!keep) return;
    *reinterpret_cast<uint2*>((uint8_t*)c.k + to) = kw;
    *reinterpret_cast<uint2*>((uint8_t*)c.v + to) = vw;
    if (u.lane == 0) {
      const uint64_t sc = (uint64_t)s * (c.seq_stride / D) + row;
      c.k_scale[sc] = ks;
      c.v_scale[sc] = vs;
    }
  }
}

// Eight codes times their scale.
template <int FORMAT>
__device__ __forceinline__ void values8(uint2 w, float scale, float4& a, float4& b) {
  if constexpr (FORMAT == KNJ_KV_I8) {
    auto at = [](uint32_t x, int j) { return (float)(int8_t)(x >> (8 * j)); };
    a = make_float4(at(w.x, 0) * scale, at(w.x, 1) * scale, at(w.x, 2) * scale, at(w.x, 3) * scale);
    b = make_float4(at(w.y, 0) * scale, at(w.y, 1) * scale, at(w.y, 2) * scale, at(w.y, 3) * scale);
  } else {
    const auto p = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.x, true);
    const auto r = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, false), t = __builtin_amdgcn_cvt_pk_f32_fp8((int)w.y, true);
    a = make_float4(p[0] * scale, p[1] * scale, q[0] * scale, q[1] * scale);
    b = make_float4(r[0] * scale, r[1] * scale, t[0] * scale, t[1] * scale);
  }
}

// The reverse: rows of activations from cache slots.  Bound by memory: 32,000 rows of
// 4 int8 heads of 128 to f16 (99 MB) 21.8 us, 4.5 TB/s, with keys and values by the
// same lanes (28 with a group for each); gathered rows of 32 sequences 2.7 us.
template <int TYPE, int FORMAT, int D>
__global__ __launch_bounds__(kBlock) void k_kv_load(KvRowsArgs a) {
  const knj_kv_cache& c = a.c;
  const Unit<D / 8> u(a);
  const uint32_t s = blockIdx.y;
  const uint64_t out = (uint64_t)s * a.n_rows + u.t;
  const int slot = a.index ? a.index[out] : (int)u.t;
  if (!u.in || slot < 0 || slot >= c.n_ctx) return;
  const uint64_t row = (uint64_t)u.h * c.n_ctx + slot;
  const uint64_t from = (uint64_t)s * c.seq_stride + row * D + 8 * u.lane;
  float4 k0, k1, v0, v1;
  if constexpr (FORMAT == KNJ_KV_F16) {
    k0 = ld4<KNJ_TYPE_F16>(c.k, from);
    k1 = ld4<KNJ_TYPE_F16>(c.k, from + 4);
    v0 = ld4<KNJ_TYPE_F16>(c.v, from);
    v1 = ld4<KNJ_TYPE_F16>(c.v, from + 4);
  } else {
    const uint2 kw = *reinterpret_cast<const uint2*>((const uint8_t*)c.k + from);
    const uint2 vw = *reinterpret_cast<const uint2*>((const uint8_t*)c.v + from);
    const uint64_t sc = (uint64_t)s * (c.seq_stride / D) + row;
    values8<FORMAT>(kw, c.k_scale[sc], k0, k1);
    values8<FORMAT>(vw, c.v_scale[sc], v0, v1);
  }
  const uint64_t to = out * a.row_stride + (uint64_t)u.h * D + 8 * u.lane;
  st4<TYPE>(a.k, to, k0);
  st4<TYPE>(a.k, to + 4, k1);
  st4<TYPE>(a.v, to, v0);
  st4<TYPE>(a.v, to + 4, v1);
}

// KERNEL<TYPE, second argument, D> for a run-time type, format and head_dim.
#define KNJ_BY_TYPE_FORM(KERNEL, type, form, D, ...)                              \
  do {                                                                            \
    if (type == KNJ_TYPE_F32) KNJ_BY_FORM(KERNEL, KNJ_TYPE_F32, form, D, __VA_ARGS__);       \
    else if (type == KNJ_TYPE_F16) KNJ_BY_FORM(KERNEL, KNJ_TYPE_F16, form, D, __VA_ARGS__);  \
    else KNJ_BY_FORM(KERNEL, KNJ_TYPE_BF16, form, D, __VA_ARGS__);                \
  } while (0)
#define KNJ_BY_FORM(KERNEL, TYPE, form, D, ...)                                   \
  do {                                                                            \
    if (form == KNJ_KV_F16) KNJ_BY_DIM(KERNEL, TYPE, KNJ_KV_F16, D, __VA_ARGS__); \
    else if (form == KNJ_KV_F8) KNJ_BY_DIM(KERNEL, TYPE, KNJ_KV_F8, D, __VA_ARGS__); \
    else KNJ_BY_DIM(KERNEL, TYPE, KNJ_KV_I8, D, __VA_ARGS__);                     \
  } while (0)
#define KNJ_BY_DIM(KERNEL, TYPE, FORM, D, ...)                                    \
  do {                                                                            \
    if (D == 128) KNJ_LAUNCH((KERNEL<TYPE, FORM, 128>), __VA_ARGS__);             \
    else KNJ_LAUNCH((KERNEL<TYPE, FORM, 64>), __VA_ARGS__);                       \
  } while (0)

dim3 kv_rows_grid(const KvRowsArgs& a) {
  const uint32_t units = (uint32_t)a.n_rows * a.c.n_head_kv, per = kBlock / (a.c.head_dim / 8);
  return dim3((units + per - 1) / per, a.c.n_seq);
}

}  // namespace

hipError_t launch_rope(int type, int layout, int head_dim, const RopeArgs& a, hipStream_t s) {
  const int hpb = kBlock / (head_dim / 8);
  const dim3 grid(a.n_rows, (a.n_head + a.n_head_kv + hpb - 1) / hpb);
#define KNJ_ROPE(TYPE)                                                                                     \
  do {                                                                                                     \
    if (layout == KNJ_ROPE_HALF) KNJ_BY_DIM(k_rope, TYPE, KNJ_ROPE_HALF, head_dim, grid, dim3(kBlock), 0, s, a); \
    else KNJ_BY_DIM(k_rope, TYPE, KNJ_ROPE_INTERLEAVED, head_dim, grid, dim3(kBlock), 0, s, a);            \
  } while (0)
  if (type == KNJ_TYPE_F32) KNJ_ROPE(KNJ_TYPE_F32);
  else if (type == KNJ_TYPE_F16) KNJ_ROPE(KNJ_TYPE_F16);
  else KNJ_ROPE(KNJ_TYPE_BF16);
#undef KNJ_ROPE
  return hipGetLastError();
}

hipError_t launch_kv_store(int type, const KvRowsArgs& a, hipStream_t s) {
  KNJ_BY_TYPE_FORM(k_kv_store, type, a.c.format, a.c.head_dim, kv_rows_grid(a), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

hipError_t launch_kv_load(int type, const KvRowsArgs& a, hipStream_t s) {
  KNJ_BY_TYPE_FORM(k_kv_load, type, a.c.format, a.c.head_dim, kv_rows_grid(a), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

int check_kv_cache(const knj_kv_cache* c) {
  KNJ_CHECK_ARG(c && c->k && c->v, "null cache pointer");
  KNJ_CHECK_ARG(c->format == KNJ_KV_F16 || c->format == KNJ_KV_F8 || c->format == KNJ_KV_I8,
                "cache format must be KNJ_KV_F16, KNJ_KV_F8 or KNJ_KV_I8");
  KNJ_CHECK_ARG(c->format == KNJ_KV_F16 || (c->k_scale && c->v_scale), "an 8-bit cache needs k_scale and v_scale");
  KNJ_CHECK_ARG(c->head_dim == 64 || c->head_dim == 128, "head_dim must be 64 or 128");
  KNJ_CHECK_ARG(c->n_seq > 0 && c->n_seq <= 65535, "n_seq must be in [1, 65535]");
  KNJ_CHECK_ARG(c->n_head_kv > 0 && c->n_head_kv <= 64, "n_head_kv must be in [1, 64]");
  KNJ_CHECK_ARG(c->n_ctx > 0, "n_ctx must be positive");
  const uint64_t seq = (uint64_t)c->n_head_kv * c->n_ctx * c->head_dim;
  KNJ_CHECK_ARG(c->seq_stride == 0 || (c->seq_stride >= seq && c->seq_stride % c->head_dim == 0),
                "seq_stride must be 0 or a multiple of head_dim that a sequence's cache fits into");
  KNJ_CHECK_ARG((((uintptr_t)c->k | (uintptr_t)c->v) & 15) == 0, "cache pointers must be 16-byte aligned");
  KNJ_CHECK_ARG((((uintptr_t)c->k_scale | (uintptr_t)c->v_scale) & 3) == 0, "scale pointers must be 4-byte aligned");
  return KNJ_OK;
}

}  // namespace knj

using namespace knj;

static knj_kv_cache with_stride(const knj_kv_cache& c) {
  knj_kv_cache r = c;
  if (!r.seq_stride) r.seq_stride = (uint64_t)c.n_head_kv * c.n_ctx * c.head_dim;
  return r;
}

extern "C" {

int knj_rope_freqs(int n_rot, double base, int scaling, double factor, int orig_ctx, double p0,
                   double p1, double* inv_freq, float* mscale) {
  KNJ_CHECK_ARG(inv_freq && mscale, "null pointer");
  KNJ_CHECK_ARG(n_rot > 0 && n_rot % 8 == 0 && n_rot <= 128, "n_rot must be a multiple of 8, at most 128");
  KNJ_CHECK_ARG(base > 1.0 && std::isfinite(base), "the base must be finite and above 1");
  KNJ_CHECK_ARG(scaling >= KNJ_ROPE_NONE && scaling <= KNJ_ROPE_LLAMA3, "unknown rope scaling");
  KNJ_CHECK_ARG(scaling == KNJ_ROPE_NONE || (factor >= 1.0 && std::isfinite(factor)),
                "the scaling factor must be finite and at least 1");
  const double pi2 = 6.283185307179586;
  if (scaling == KNJ_ROPE_YARN)
    KNJ_CHECK_ARG(orig_ctx > 0 && p0 > p1 && p1 > 0.0, "yarn takes orig_ctx > 0 and p0 (fast) > p1 (slow) > 0 turns");
  if (scaling == KNJ_ROPE_LLAMA3)
    KNJ_CHECK_ARG(orig_ctx > 0 && p1 > p0 && p0 > 0.0, "llama3 takes orig_ctx > 0 and p1 (high) > p0 (low) > 0");
  const int half = n_rot / 2;
  if (scaling == KNJ_ROPE_NTK) base *= std::pow(factor, (double)n_rot / (n_rot - 2.0));
  *mscale = scaling == KNJ_ROPE_YARN ? (float)(0.1 * std::log(factor) + 1.0) : 1.0f;
  double lo = 0.0, hi = 0.0;
  if (scaling == KNJ_ROPE_YARN) {
    // the dim whose frequency makes `turns` turns in orig_ctx
    auto dim = [&](double turns) { return n_rot * std::log(orig_ctx / (turns * pi2)) / (2.0 * std::log(base)); };
    lo = std::fmax(std::floor(dim(p0)), 0.0);
    hi = std::fmin(std::ceil(dim(p1)), n_rot - 1.0);
    if (hi <= lo) hi = lo + 0.001;
  }
  for (int i = 0; i < half; ++i) {
    const double f = std::pow(base, -2.0 * i / n_rot);
    double keep = 1.0;  // of f, the rest of f / factor
    if (scaling == KNJ_ROPE_LINEAR) keep = 0.0;
    else if (scaling == KNJ_ROPE_YARN) keep = 1.0 - std::fmin(std::fmax((i - lo) / (hi - lo), 0.0), 1.0);
    else if (scaling == KNJ_ROPE_LLAMA3)
      keep = std::fmin(std::fmax((orig_ctx * f / pi2 - p0) / (p1 - p0), 0.0), 1.0);
    inv_freq[i] = keep == 1.0 ? f : f / factor * (1.0 - keep) + f * keep;
  }
  return KNJ_OK;
}

int knj_rope(int type, int layout, int n_rot, const double* inv_freq, float mscale,
             const int32_t* pos, int n_rows, int head_dim, const void* q, int n_head,
             uint64_t q_stride, const float* q_norm, void* q_out, uint64_t q_out_stride,
             const void* k, int n_head_kv, uint64_t k_stride, const float* k_norm, void* k_out,
             uint64_t k_out_stride, float eps, void* stream) {
  const int eb = act_bytes(type);
  KNJ_CHECK_ARG(eb, "activations must be F32, F16 or BF16");
  KNJ_CHECK_ARG(layout == KNJ_ROPE_HALF || layout == KNJ_ROPE_INTERLEAVED, "unknown rope layout");
  KNJ_CHECK_ARG(head_dim == 64 || head_dim == 128, "head_dim must be 64 or 128");
  KNJ_CHECK_ARG(n_rot > 0 && n_rot % 8 == 0 && n_rot <= head_dim, "n_rot must be a multiple of 8, at most head_dim");
  KNJ_CHECK_ARG(inv_freq && pos && q && q_out, "null pointer");
  KNJ_CHECK_ARG(((uintptr_t)inv_freq & 7) == 0 && (((uintptr_t)q_norm | (uintptr_t)k_norm) & 15) == 0,
                "inv_freq must be 8-byte and the norm weights 16-byte aligned");
  KNJ_CHECK_ARG(words_aligned(pos), "pos must be aligned to its type");
  KNJ_CHECK_ARG(n_rows >= 0, "negative row count");
  KNJ_CHECK_ARG(n_rows < (1 << 24), "too many rows for one call");  // (a grid holds 2^32 threads a dim)
  KNJ_CHECK_ARG(n_head > 0 && n_head <= 4096 && n_head_kv >= 0 && n_head_kv <= 4096,
                "n_head must be in [1, 4096], n_head_kv in [0, 4096]");
  KNJ_CHECK_ARG(n_head_kv == 0 || (k && k_out), "null key pointer");
  KNJ_CHECK_ARG(q_stride >= (uint64_t)n_head * head_dim && q_out_stride >= (uint64_t)n_head * head_dim &&
                    (n_head_kv == 0 || (k_stride >= (uint64_t)n_head_kv * head_dim &&
                                        k_out_stride >= (uint64_t)n_head_kv * head_dim)),
                "a row stride is below the row's width");
  KNJ_CHECK_ARG(rows_aligned(q, q_stride, eb) && rows_aligned(q_out, q_out_stride, eb) &&
                    (n_head_kv == 0 || (rows_aligned(k, k_stride, eb) && rows_aligned(k_out, k_out_stride, eb))),
                "rows must start on 16-byte boundaries");
  KNJ_CHECK_ARG(n_rows <= 1 || ((q != q_out || q_stride == q_out_stride) &&
                                (n_head_kv == 0 || k != k_out || k_stride == k_out_stride)),
                "an output in place takes its input's stride");
  KNJ_CHECK_ARG(mscale > 0.0f && std::isfinite(mscale), "mscale must be finite and positive");
  KNJ_CHECK_ARG((!q_norm && !k_norm) || (eps >= 0.0f && std::isfinite(eps)), "eps must be finite and not negative");
  const int rc = require_device();
  if (rc || n_rows == 0) return rc;
  RopeArgs a{q, k, q_out, k_out, q_stride, k_stride, q_out_stride, k_out_stride, q_norm, k_norm,
             eps, inv_freq, mscale, pos, n_rows, n_head, n_head_kv, n_rot};
  KNJ_HIP(launch_rope(type, layout, head_dim, a, (hipStream_t)stream));
  return KNJ_OK;
}

static int check_kv_rows(const knj_kv_cache* cache, int type, const void* k, const void* v, uint64_t row_stride,
                         int n_rows) {
  const int rc = check_kv_cache(cache);
  if (rc) return rc;
  const int eb = act_bytes(type);
  KNJ_CHECK_ARG(eb, "activations must be F32, F16 or BF16");
  KNJ_CHECK_ARG(k && v, "null pointer");
  KNJ_CHECK_ARG(n_rows >= 0, "negative row count");
  KNJ_CHECK_ARG(row_stride >= (uint64_t)cache->n_head_kv * cache->head_dim, "the row stride is below the row's width");
  KNJ_CHECK_ARG(rows_aligned(k, row_stride, eb) && rows_aligned(v, row_stride, eb),
                "rows must start on 16-byte boundaries");
  KNJ_CHECK_ARG((uint64_t)n_rows * cache->n_head_kv < (1ull << 27), "too many rows for one call");
  return KNJ_OK;
}

int knj_kv_store(const knj_kv_cache* cache, int type, const void* k, const void* v,
                 uint64_t row_stride, const int32_t* start, const int32_t* counts, int n_rows,
                 void* stream) {
  int rc = check_kv_rows(cache, type, k, v, row_stride, n_rows);
  if (rc) return rc;
  KNJ_CHECK_ARG(start, "null start");
  KNJ_CHECK_ARG(words_aligned(start, counts), "start and counts must be aligned to their type");
  rc = require_device();
  if (rc || n_rows == 0) return rc;
  KvRowsArgs a{with_stride(*cache), const_cast<void*>(k), const_cast<void*>(v), row_stride, start, counts, n_rows};
  KNJ_HIP(launch_kv_store(type, a, (hipStream_t)stream));
  return KNJ_OK;
}

int knj_kv_load(const knj_kv_cache* cache, int type, const int32_t* slots, int n_rows, void* k,
                void* v, uint64_t row_stride, void* stream) {
  int rc = check_kv_rows(cache, type, k, v, row_stride, n_rows);
  if (rc) return rc;
  KNJ_CHECK_ARG(words_aligned(slots), "slots must be aligned to their type");
  rc = require_device();
  if (rc || n_rows == 0) return rc;
  KvRowsArgs a{with_stride(*cache), k, v, row_stride, slots, nullptr, n_rows};
  KNJ_HIP(launch_kv_load(type, a, (hipStream_t)stream));
  return KNJ_OK;
}

// Slots of a sequence that the attention numbers in 32 bits, with the chunk that is
// fetched past the last one.
static constexpr int64_t kMaxSlots = 0x7FFFFFFF - 256;

int knj_attention_tree(const knj_kv_cache* cache, int type, const void* q, uint64_t q_stride,
                       int n_head, int n_rows, const int32_t* prefix, int max_prefix,
                       const int32_t* counts, const uint64_t* mask, int mask_shared, float scale,
                       void* out, uint64_t out_stride, void* workspace, uint64_t workspace_bytes,
                       void* stream) {
  int rc = check_kv_cache(cache);
  if (rc) return rc;
  const int eb = act_bytes(type);
  KNJ_CHECK_ARG(eb, "activations must be F32, F16 or BF16");
  KNJ_CHECK_ARG(q && out && prefix, "null pointer");
  KNJ_CHECK_ARG(words_aligned(prefix, counts) && ((uintptr_t)mask & 7) == 0,
                "prefix, counts and mask must be aligned to their types");
  KNJ_CHECK_ARG(n_rows >= 0 && n_rows <= 1024, "n_rows must be in [0, 1024]");
  KNJ_CHECK_ARG(n_head > 0 && n_head <= 1024 && n_head % cache->n_head_kv == 0,
                "n_head must be a positive multiple of n_head_kv, at most 1024");
  KNJ_CHECK_ARG(max_prefix >= 0 && (int64_t)max_prefix + n_rows <= cache->n_ctx,
                "max_prefix and the drafts must fit into n_ctx");
  KNJ_CHECK_ARG((int64_t)max_prefix + n_rows <= kMaxSlots, "max_prefix and the drafts must stay below 2^31 - 256");
  KNJ_CHECK_ARG(scale >= 1e-6f && scale <= 1e6f, "the scale must be in [1e-6, 1e6]");
  KNJ_CHECK_ARG((uint64_t)cache->n_seq * n_rows * n_head < (1ull << 31), "too many rows for one call");
  const uint64_t width = (uint64_t)n_head * cache->head_dim;
  KNJ_CHECK_ARG(q_stride >= width && out_stride >= width, "a row stride is below the row's width");
  KNJ_CHECK_ARG(rows_aligned(q, q_stride, eb) && rows_aligned(out, out_stride, eb),
                "rows must start on 16-byte boundaries");
  KNJ_CHECK_ARG(q != out || q_stride == out_stride || (uint64_t)cache->n_seq * n_rows <= 1,
                "an output in place takes its input's stride");
  const uint64_t need = n_rows ? tree_partial_bytes(*cache, type, n_head, n_rows, max_prefix) : 0;
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) {
    set_error("knj_attention_tree: these sizes need a 16-byte aligned workspace of " + std::to_string(need) + " bytes");
    return KNJ_E_ARG;
  }
  rc = require_device();
  if (rc || n_rows == 0) return rc;
  TreeArgs a{with_stride(*cache), q, out, q_stride, out_stride, prefix, counts, mask, (float*)workspace, scale,
             n_head, n_rows, max_prefix, mask_shared, type};
  KNJ_HIP(launch_attention_tree(a, (hipStream_t)stream));
  return KNJ_OK;
}

uint64_t knj_attention_tree_workspace(const knj_kv_cache* cache, int n_head, int n_rows, int max_prefix) {
  if (check_kv_cache(cache) || n_head <= 0 || n_head > 1024 || n_head % cache->n_head_kv || n_rows <= 0 ||
      n_rows > 1024 || max_prefix < 0 || (int64_t)max_prefix + n_rows > std::min<int64_t>(cache->n_ctx, kMaxSlots))
    return 0;
  // (enough for every type)
  return std::max(tree_partial_bytes(*cache, KNJ_TYPE_F32, n_head, n_rows, max_prefix),
                  tree_partial_bytes(*cache, KNJ_TYPE_F16, n_head, n_rows, max_prefix));
}

}  // extern "C"
