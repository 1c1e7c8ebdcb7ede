// kanjoos_amd/csrc/knj_logprobs.hip -- log probabilities of given tokens over rows of logits, with
// the rows' entropy and their largest entries.
//
// Two launches.  The first reads every logit once: a wave takes 2048 of a row
// into registers and leaves a record of them -- the largest (value and index),
// the sum of the others' exponentials relative to it, and the entropy's sum.
// The second, a workgroup per row, joins a row's records in f64 and finds the
// n largest logits: only the n pieces with the largest maxima can hold any, so
// those n are read again.
#include <string>

#include "knj_common.h"
#include "knj_dev.h"

namespace knj {
namespace {

using namespace dev;

constexpr int kPiece = 2048;   // logits of one wave
constexpr int kPer = kPiece / 64;
constexpr int kMaxTop = 32;
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxPieces = kMaxVocab / kPiece;  // 512
constexpr int kCand = kMaxTop * (kMaxTop + 1) / 2;  // candidates of the largest: sum of n - q over the n pieces
// Waves of a row's joining workgroup: sixteen hold the pieces of the n largest at
// once, for the latency of a row; with more rows than CUs, four a row keep more rows
// going.  Calls over rows of 151,936 f32 with the 5 and the 20 largest, sixteen
// against four: 1 row 9.9 and 11.5 against 11.6 and 16.2 us, 256 rows 37.9 and 42.2
// against 38.5 and 44.4, 400 rows 57.4 and 63.0 against 53.3 and 59.2 (eight were
// between the two at every count).  With fewer pieces than n, which only sixteen hold
// all of for a threshold, sixteen: 1 and 500 rows of 32,000 f32 with the 20 largest 11.7
// and 35.6 us, where taking them out of the pieces one by one was 39.4 and 108.
constexpr int kJoinRows = 256;

struct Record {
  uint32_t key;   // order_key of the piece's largest logit
  uint32_t idx;   // its index in the row
  float rest;     // sum over the piece's other logits of 2^((x - max) c); NaN: the piece holds a NaN or +inf
  float ent;      // sum over them of 2^((x - max) c) (x - max) c
};

// Unsigned keys in the order of the floats (+0 and -0 alike); at least
// 0x007FFFFF (-inf), so 0 is below every logit.
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// Where lane l's value i of a piece stands in the row.
template <int TYPE>
__device__ __forceinline__ int piece_index(int piece, int lane, int i) {
  constexpr int V = TYPE == KNJ_TYPE_F32 ? 4 : 8;  // values per 16 bytes
  return piece * kPiece + ((i / V) * 64 + lane) * V + i % V;
}

// A piece of a row, kPer values per lane, -inf past the row's end; 16-byte loads
// at the alignment of the type (the device runs with unaligned access on).
template <int TYPE>
__device__ __forceinline__ void load_piece(const void* logits, uint64_t row_at, int piece, int n_vocab, int lane,
                                           float (&v)[kPer]) {
  constexpr int V = TYPE == KNJ_TYPE_F32 ? 4 : 8, EB = 16 / V;
  const char* base = (const char*)logits + row_at * EB;
#pragma unroll
  for (int j = 0; j < kPer / V; ++j) {
    const int at = piece_index<TYPE>(piece, lane, j * V);
    uint4 w = make_uint4(0u, 0u, 0u, 0u);
    if (at + V <= n_vocab) {
      __builtin_memcpy(&w, base + (uint64_t)at * EB, 16);
    } else if (at < n_vocab) {
      uint32_t t[4] = {0u, 0u, 0u, 0u};
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (at + i < n_vocab) {
          if constexpr (EB == 4) t[i] = ((const uint32_t*)base)[at + i];
          else t[i / 2] |= (uint32_t)((const uint16_t*)base)[at + i] << (16 * (i & 1));
        }
      }
      w = make_uint4(t[0], t[1], t[2], t[3]);
    }
    const uint32_t t[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float x;
      if constexpr (TYPE == KNJ_TYPE_F32) x = __uint_as_float(t[i]);
      else if constexpr (TYPE == KNJ_TYPE_F16) x = h2f(t[i / 2] >> (16 * (i & 1)));
      else x = __uint_as_float((i & 1) ? (t[i / 2] & 0xFFFF0000u) : (t[i / 2] << 16));
      v[j * V + i] = at + i < n_vocab ? x : -INFINITY;
    }
  }
}

// A logit's place in the order of the largest: by value, ties to the lowest
// index; a NaN as -inf, 0 past the row's end.
__device__ __forceinline__ unsigned long long piece_key(float v, uint32_t idx, int n_vocab) {
  if (idx >= (uint32_t)n_vocab) return 0ull;
  return ((unsigned long long)order_key(v == v ? v : -INFINITY) << 32) | (0xFFFFFFFFu - idx);
}

// Record of one piece per wave.  With the largest logit m of the piece and
// d = (x - m) log2(e) / T <= 0: rest = sum 2^d, ent = sum 2^d d over all but the
// largest itself, so that a row with one likely token keeps log(1 + rest) to the
// rest's own precision.  log2(e)/T comes as two floats (its rounding would be a
// common error of every term).
//
// Bound by the read of the logits: 32 values a lane are eight (f32) or four loads in
// flight a wave, then kept in registers, so that the largest is known before the
// exponentials and no running rescale is needed.  500 rows of 151,936 f32 (304 MB):
// 55.2 us, 5.5 TB/s (a copy reads and writes 5.1); of f16 50.0, the exponentials and
// the entropy's products of 76 million logits then count; one row 4.2 us, the latency of a
// launch, one load and the two reductions.
template <int TYPE>
__global__ __launch_bounds__(kBlock) void k_logprob_pieces(LogprobArgs a, int n_pieces, float c_hi, float c_lo) {
  const int lane = threadIdx.x & 63;
  const uint32_t w = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6);
  const uint32_t row = w / (uint32_t)n_pieces, piece = w - row * (uint32_t)n_pieces;
  if (row >= (uint32_t)a.n_rows) return;
  float v[kPer];
  load_piece<TYPE>(a.logits, (uint64_t)row * a.row_stride, piece, a.n_vocab, lane, v);
  bool bad = false;
  float best = -INFINITY;
  int bi = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    bad |= v[i] != v[i] || v[i] == INFINITY;
    v[i] = v[i] == v[i] ? v[i] : -INFINITY;
    if (v[i] > best) {
      best = v[i];
      bi = i;
    }
  }
  const uint32_t idx = piece_index<TYPE>(piece, lane, bi);
  const unsigned long long top =
      wave_max_u64(((unsigned long long)order_key(best) << 32) | (0xFFFFFFFFu - idx));
  const uint32_t top_idx = 0xFFFFFFFFu - (uint32_t)top;
  const float m = order_value((uint32_t)(top >> 32));
  const int skip = idx == top_idx ? bi : -1;
  float rest = 0.0f, ent = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const float t = v[i] - m;
    // (-inf, and -inf - -inf, weigh nothing: held where 2^d is 0 and d finite)
    const float d = fmaxf(fmaf(t, c_hi, t * c_lo), -16384.0f);
    const float e = i == skip ? 0.0f : __builtin_amdgcn_exp2f(d);
    rest += e;
    ent = fmaf(e, d, ent);
  }
  rest = group_sum<64>(rest);
  ent = group_sum<64>(ent);
  bad = __ballot(bad) != 0;
  if (lane == 0)
    ((Record*)a.records)[w] = Record{(uint32_t)(top >> 32), top_idx, bad ? NAN : rest, ent};
}

// 2^d in f64 to f32's precision, d <= 0.
__device__ __forceinline__ double exp2_neg(double d) {
  const double n = rint(fmax(d, -2000.0));
  return ldexp((double)__builtin_amdgcn_exp2f((float)(fmax(d, -2000.0) - n)), (int)n);
}

// Ranks of keys[0 .. n) among themselves (how many are above), by all threads: eight
// lanes a key, each against every eighth.  found(i, rank) on one of the eight.
template <int NT, class F>
__device__ __forceinline__ void rank_keys(const unsigned long long* keys, int n, F found) {
  const int sub = threadIdx.x & 7;
  for (int i0 = 0; i0 < n; i0 += NT / 8) {  // (uniform: the lanes' sums need all eight)
    const int i = i0 + (threadIdx.x >> 3);
    const unsigned long long key = keys[min(i, n - 1)];
    int above = 0;
#pragma unroll 4
    for (int j = sub; j < n; j += 8) above += keys[j] > key;
    const int rank = (int)group_sum<8>((float)above);
    if (sub == 0 && i < n) found(i, rank);
  }
}

// A row's records joined.  With M the row's largest logit, f = 2^((m - M) c) of
// each piece: rest = sum over the pieces of f (1 + rest_p), without the 1 of the
// piece that holds M, and ent = sum of f (ent_p + (1 + rest_p) (m - M) c); then
// log sum e^(x - M) = log1p(rest), the entropy log1p(rest) - ln 2 ent / (1 + rest).
// The pieces that can hold one of the n largest are ranked and fetched first, so
// that the sums are formed while they are on their way.  W waves a row.
//
// Bound by its own chain of steps (records, maximum, ranks, pieces, candidates, ranks
// again): 7.1 us for one row and its 20 largest, of which 3.7 are the top's (the f32
// kernel of sixteen waves leaves three of its registers in scratch, at its limit of
// 128); 11.8 us for 500 rows and 5.  Sums over few records cost nothing in f64, and
// ranks counted by comparison need no passes over the keys: eight lanes a key took 2 us
// off a lane a key.
template <int TYPE, int W>
__global__ __launch_bounds__(64 * W) void k_logprob_join(LogprobArgs a, int n_pieces, double c) {
  constexpr int NT = 64 * W, R = kMaxPieces > NT ? kMaxPieces / NT : 1;  // records a thread
  constexpr bool kHoldAll = 2 * W >= kMaxTop;  // pieces, where there are fewer than n
  __shared__ __align__(16) unsigned long long keys[kMaxPieces];
  __shared__ __align__(16) unsigned long long cand[kCand];
  __shared__ unsigned long long red_key[W];
  __shared__ double red_rest[W], red_ent[W];
  __shared__ int red_bad[W], chosen[kMaxTop];
  __shared__ int n_cand;
  const int row = blockIdx.y * gridDim.x + blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (row >= a.n_rows) return;
  const Record* rec = (const Record*)a.records + (uint64_t)row * n_pieces;
  const uint64_t row_at = (uint64_t)row * a.row_stride;
  const int n = a.n_top, n_sel = min(n, n_pieces);
  Record r[R];
  unsigned long long key[R], wk = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int p = tid + i * NT;
    r[i] = Record{0u, 0u, 0.0f, 0.0f};
    key[i] = 0;
    if (p < n_pieces) {
      r[i] = rec[p];
      key[i] = ((unsigned long long)r[i].key << 32) | (0xFFFFFFFFu - r[i].idx);
    }
    if (p < kMaxPieces) keys[p] = key[i];
    wk = key[i] > wk ? key[i] : wk;
  }
  if (tid == 0) n_cand = 0;
  wk = wave_max_u64(wk);
  if (lane == 0) red_key[wave] = wk;
  __syncthreads();
  unsigned long long top = red_key[0];
#pragma unroll
  for (int i = 1; i < W; ++i) top = red_key[i] > top ? red_key[i] : top;
  const float M = order_value((uint32_t)(top >> 32));
  // the n pieces with the largest keys, by rank (keys differ: their indexes do)
  if (n)
    rank_keys<NT>(keys, n_pieces, [&](int i, int rank) {
      if (rank < n) chosen[rank] = i;
    });
  float x_tok = 0.0f;  // the given token's logit
  const int tok = tid == 0 && a.logprob ? a.tokens[row] : -1;
  if (tok >= 0 && tok < a.n_vocab) {
    if constexpr (TYPE == KNJ_TYPE_F32) x_tok = ((const float*)a.logits)[row_at + tok];
    else if constexpr (TYPE == KNJ_TYPE_F16) x_tok = h2f(((const uint16_t*)a.logits)[row_at + tok]);
    else x_tok = __uint_as_float((uint32_t)((const uint16_t*)a.logits)[row_at + tok] << 16);
  }
  double rest = 0.0, ent = 0.0;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (tid + i * NT >= n_pieces) break;
    const bool b = r[i].rest != r[i].rest;
    bad |= b;
    const float m = order_value(r[i].key);
    if (m > -INFINITY && M < INFINITY && !b) {
      const double d = ((double)m - (double)M) * c;
      const double f = exp2_neg(d);
      rest += f * ((double)r[i].rest + (key[i] == top ? 0.0 : 1.0));
      ent += f * ((double)r[i].ent + (1.0 + (double)r[i].rest) * d);
    }
  }
  const int waves = min(W, (n_pieces + 63) >> 6);  // that hold records
  if (wave < waves) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      rest += __shfl_xor(rest, o);
      ent += __shfl_xor(ent, o);
    }
    bad = __ballot(bad) != 0;
    if (lane == 0) {
      red_rest[wave] = rest;
      red_ent[wave] = ent;
      red_bad[wave] = bad;
    }
  }
  __syncthreads();
  float v[2][kPer];  // the chosen pieces of ranks `wave` and W + wave
  auto fetch = [&](int q0) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (q0 + h * W + wave < n_sel)
        load_piece<TYPE>(a.logits, row_at, chosen[q0 + h * W + wave], a.n_vocab, lane, v[h]);
  };
  fetch(0);
  rest = ent = 0.0;
  bad = false;
  for (int i = 0; i < waves; ++i) {
    rest += red_rest[i];
    ent += red_ent[i];
    bad |= red_bad[i] != 0;
  }
  const bool none = M == -INFINITY;  // nothing left in the row
  const double lse = log1p(rest);    // above M / T
  // log probability of a logit x of this row
  auto logp = [&](float x) -> float {
    if (bad) return NAN;
    if (none || x == -INFINITY) return -INFINITY;
    return (float)(((double)x - (double)M) * a.inv_temp - lse);
  };
  if (tid == 0) {
    if (a.entropy) a.entropy[row] = bad ? NAN : none ? 0.0f : (float)(lse - 0.6931471805599453 * ent / (1.0 + rest));
    if (a.logprob) a.logprob[row] = tok < 0 ? 0.0f : tok >= a.n_vocab ? NAN : logp(x_tok);
  }
  if (n == 0) return;
  // Every one of the n largest logits is at least the n-th piece's largest, or with
  // fewer pieces than n the n-th largest of the maxima of groups of lanes, 2 n to 4 n of
  // them (the waves then hold all pieces): the logits that are (few more than n, as a
  // rule) become candidates, in any order.
  unsigned long long least;
  if constexpr (kHoldAll) {
    if (n_pieces < n) {
      int g = 64;  // lanes of a group
      while (g > 1 && n_pieces * (64 / g) < 2 * n) g >>= 1;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int q = h * W + wave;
        if (q >= n_sel) break;
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPer; ++i) m = fmaxf(m, v[h][i]);
        for (int o = 1; o < g; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        const int at = (q * 64 + lane) / g;
        if (lane % g == 0) keys[at] = ((unsigned long long)order_key(m) << 32) | (0xFFFFFFFFu - (uint32_t)at);
      }
      __syncthreads();
      rank_keys<NT>(keys, n_pieces * (64 / g), [&](int i, int rank) {
        if (rank == n - 1) red_key[0] = keys[i] >> 32 << 32;
      });
      __syncthreads();
      least = red_key[0];
    } else {
      least = keys[chosen[n - 1]];
    }
  } else {
    least = keys[chosen[n - 1]];
  }
  const float least_value = order_value((uint32_t)(least >> 32));
  for (int q0 = 0; q0 < n_sel; q0 += 2 * W) {
    if (q0) fetch(q0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (q0 + h * W + wave >= n_sel) break;
      const int piece = chosen[q0 + h * W + wave];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const bool may = !(v[h][i] < least_value);  // (a NaN may, where -inf does)
        if (__builtin_expect(__ballot(may) == 0, 1)) continue;
        const unsigned long long mine = piece_key(v[h][i], piece_index<TYPE>(piece, lane, i), a.n_vocab);
        if (!may || mine < least) continue;
        const int at = atomicAdd(&n_cand, 1);
        if (at < kCand) cand[at] = mine;
      }
    }
  }
  __syncthreads();
  int nc = n_cand;
  if (nc > kCand) {
    // Rows whose largest logits crowd into few pieces (sorted ones, equal ones; a row of
    // 151,936 and its 20 largest then take 44 us, of 32,000 33 to 40): the
    // chosen piece of rank q holds at most n - q of the n largest, taken out one
    // after the other.
    __syncthreads();
    if (tid == 0) n_cand = 0;
    __syncthreads();
    for (int q = wave; q < n_sel; q += W) {
      const int piece = chosen[q];
      load_piece<TYPE>(a.logits, row_at, piece, a.n_vocab, lane, v[0]);
      unsigned long long last = ~0ull;  // the key taken out before
      for (int t = 0; t < n - q; ++t) {
        unsigned long long mine = 0;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const unsigned long long k = piece_key(v[0][i], piece_index<TYPE>(piece, lane, i), a.n_vocab);
          mine = k < last && k > mine ? k : mine;
        }
        last = wave_max_u64(mine);
        if (last < least) break;  // (uniform; also when the piece is used up)
        if (lane == 0) cand[atomicAdd(&n_cand, 1)] = last;
      }
    }
    __syncthreads();
    nc = n_cand;
  }
  rank_keys<NT>(cand, nc, [&](int i, int rank) {
    if (rank >= n) return;
    const unsigned long long k = cand[i];
    a.top_idx[(uint64_t)row * n + rank] = (int32_t)(0xFFFFFFFFu - (uint32_t)k);
    a.top_logprob[(uint64_t)row * n + rank] = logp(order_value((uint32_t)(k >> 32)));
  });
}

int pieces_of(int n_vocab) { return (n_vocab + kPiece - 1) / kPiece; }

}  // namespace

uint64_t logprob_record_bytes(int n_rows, int n_vocab) {
  return (uint64_t)n_rows * pieces_of(n_vocab) * sizeof(Record);
}

hipError_t launch_token_logprobs(int type, const LogprobArgs& a, hipStream_t s) {
  const int n_pieces = pieces_of(a.n_vocab);
  const uint64_t waves = (uint64_t)a.n_rows * n_pieces;
  const dim3 grid((unsigned)((waves + kBlock / 64 - 1) / (kBlock / 64)));
  // (a grid holds 2^32 threads a dim: 2^21 workgroups of 1024 are half of it)
  const unsigned across = a.n_rows < (1 << 21) ? a.n_rows : 1u << 21;
  const dim3 join(across, (a.n_rows + across - 1) / across);
  const double c = 1.4426950408889634 * a.inv_temp;
  const float c_hi = (float)c, c_lo = (float)(c - (double)c_hi);
#define KNJ_LOGPROBS(TYPE)                                                                            \
  do {                                                                                                \
    KNJ_LAUNCH(k_logprob_pieces<TYPE>, grid, dim3(kBlock), 0, s, a, n_pieces, c_hi, c_lo);            \
    if (a.n_rows <= kJoinRows || n_pieces < a.n_top)                                                  \
      KNJ_LAUNCH((k_logprob_join<TYPE, 16>), join, dim3(1024), 0, s, a, n_pieces, c);                 \
    else                                                                                              \
      KNJ_LAUNCH((k_logprob_join<TYPE, 4>), join, dim3(256), 0, s, a, n_pieces, c);                   \
  } while (0)
  if (type == KNJ_TYPE_F32) KNJ_LOGPROBS(KNJ_TYPE_F32);
  else if (type == KNJ_TYPE_F16) KNJ_LOGPROBS(KNJ_TYPE_F16);
  else KNJ_LOGPROBS(KNJ_TYPE_BF16);
#undef KNJ_LOGPROBS
  return hipGetLastError();
}

}  // namespace knj

using namespace knj;

extern "C" {

int knj_token_logprobs(int type, const void* logits, uint64_t row_stride, int n_rows, int n_vocab,
                       float temperature, const int32_t* tokens, float* logprob, float* entropy,
                       int n_top, int32_t* top_idx, float* top_logprob, void* workspace,
                       uint64_t workspace_bytes, void* stream) {
  const int eb = act_bytes(type);
  KNJ_CHECK_ARG(eb, "logits must be F32, F16 or BF16");
  KNJ_CHECK_ARG(logits, "null pointer");
  KNJ_CHECK_ARG(((uintptr_t)logits & (eb - 1)) == 0, "the logits must be aligned to their type");
  KNJ_CHECK_ARG(n_rows >= 0, "negative row count");
  KNJ_CHECK_ARG(n_vocab > 0 && n_vocab <= kMaxVocab, "n_vocab must be in [1, 2^20]");
  KNJ_CHECK_ARG(row_stride >= (uint64_t)n_vocab, "the row stride is below the row's width");
  KNJ_CHECK_ARG(n_rows < (1 << 24) && (uint64_t)n_rows * pieces_of(n_vocab) < (1ull << 26),
                "too many rows for one call");  // (a grid holds 2^32 threads a dim)
  KNJ_CHECK_ARG(temperature >= 1e-4f && temperature <= 1e4f, "the temperature must be in [1e-4, 1e4]");
  KNJ_CHECK_ARG(!tokens == !logprob, "tokens and logprob go together");
  KNJ_CHECK_ARG(n_top >= 0 && n_top <= kMaxTop && n_top <= n_vocab, "n_top must be in [0, min(32, n_vocab)]");
  KNJ_CHECK_ARG(n_top == 0 || (top_idx && top_logprob), "null top_idx or top_logprob");
  KNJ_CHECK_ARG(words_aligned(tokens, logprob, entropy, top_idx, top_logprob),
                "tokens and outputs must be aligned to their types");
  const uint64_t need = logprob_record_bytes(n_rows, n_vocab);
  if (n_rows && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) {
    set_error("knj_token_logprobs: these sizes need a 16-byte aligned workspace of " + std::to_string(need) + " bytes");
    return KNJ_E_ARG;
  }
  const int rc = require_device();
  if (rc || n_rows == 0) return rc;
  LogprobArgs a{logits, row_stride, n_rows, n_vocab, n_top, 1.0 / (double)temperature, tokens, logprob, entropy,
                top_idx, top_logprob, workspace};
  KNJ_HIP(launch_token_logprobs(type, a, (hipStream_t)stream));
  return KNJ_OK;
}

uint64_t knj_token_logprobs_workspace(int n_rows, int n_vocab) {
  if (n_rows <= 0 || n_vocab <= 0 || n_vocab > kMaxVocab) return 0;
  return logprob_record_bytes(n_rows, n_vocab);
}

}  // extern "C"
