// kanjoos_amd/csrc/knj_pages.hip -- a 4-bit cache in pages: rows stored and read back, pages
// reserved, shared, given back, moved together and copied.
#include "knj_pages.h"

#include <algorithm>
#include <string>

#include "knj_common.h"
#include "knj_dev.h"

namespace knj {
namespace {

using namespace dev;

// Pieces of D/8 bytes: of a row four of codes a matrix and one of words.  (Vectors of the
// compiler's own: arrays of its structs, loaded under a condition, end up in LDS.)
typedef uint32_t u32v4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32v2 __attribute__((ext_vector_type(2)));
template <int D>
using Piece = std::conditional_t<D == 128, u32v4, u32v2>;

// ---------------------------------------------------------------- rows
// A row's kv head is D/8 lanes of eight dims, four lanes a group of 32; the same lanes
// take its key and its value.  blockIdx.y is the sequence.  Each element is read once and
// written once: 4096 f32 rows of 4 kv heads, 19.4 MB either way, 7.1 us a call (2.7 TB/s, half
// of it the launch's own latency; one row of 32 sequences takes 3.5 and 2.4; 65,536 rows, 310 MB,
// stored 56 and loaded 63, 5.6 and 4.9 TB/s).
template <int D>
struct PageUnit {
  static constexpr int T = D / 8;
  uint32_t t;  // row
  int h, lane;
  bool in;  // (the lanes past the last unit repeat it and store nothing)
  __device__ __forceinline__ PageUnit(const PageRowsArgs& a) {
    const uint32_t nk = a.g.n_head_kv, total = (uint32_t)a.n_rows * nk;
    const uint32_t u = blockIdx.x * (kBlock / T) + threadIdx.x / T;
    in = u < total;
    const uint32_t v = in ? u : total - 1;
    t = v / nk;
    h = (int)(v - t * nk);
    lane = threadIdx.x % T;
  }
};

// Page of a sequence's slot, -1 if it has none.
__device__ __forceinline__ int page_of(const PageGeom& g, uint32_t s, int64_t slot) {
  if (slot < 0 || slot >= ((int64_t)g.n_table << g.shift)) return -1;
  const int p = g.table[(uint64_t)s * g.n_table + (slot >> g.shift)];
  return p >= 0 && p < g.n_page ? p : -1;
}

// Eight dims of a group held by four lanes as codes, and the group's word.
// The f32 quotient is off by at most 16 * 2^-22 (x - low is rounded only where the two
// are far apart, and then to 2^-24 of itself), which decides a rounding only next to a
// tie: there it is formed in f64.
__device__ __forceinline__ uint32_t quantise4(const float (&x)[8], uint32_t& word) {
  float mn = x[0], mx = x[0];
  bool bad = false;  // (of a NaN or what f16 does not hold)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    mn = fminf(mn, x[i]);
    mx = fmaxf(mx, x[i]);
    bad |= !(fabsf(x[i]) <= 65504.0f);
  }
  mn = -group_max<4>(-mn);
  mx = group_max<4>(mx);
  bad = group_max<4>(bad ? 1.0f : 0.0f) != 0.0f;
  const uint32_t low16 = f2h(mn + 0.0f);
  const float low = h2f(low16);
  // the quotient towards zero: to f32, then to f16
  const double room = fmax(((double)mx - (double)low) / 15.0, 0.0);
  float r = (float)room;
  if ((double)r > room) r = __uint_as_float(__float_as_uint(r) - 1);
  const uint32_t step16 = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(r, 0.0f)) & 0xFFFFu;
  const float step = h2f(step16);
  const bool live = !bad && step > 0.0f;
  const float inv = live ? 1.0f / step : 0.0f;
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float y = live ? (x[i] - low) * inv : 0.0f;
    float t = rintf(y);
    if (fabsf(fabsf(y - t) - 0.5f) < 1e-4f) t = (float)rint(((double)x[i] - (double)low) / (double)step);
    w |= (uint32_t)fminf(fmaxf(t, 0.0f), 15.0f) << (4 * (i >> 1) + 16 * (i & 1));
  }
  word = bad ? kNanGroup : (low16 << 16) | step16;
  return w;
}

template <int TYPE, int D>
__global__ __launch_bounds__(kBlock) void k_pages_store(PageRowsArgs a) {
  const PageGeom& g = a.g;
  const PageUnit<D> u(a);
  const uint32_t s = blockIdx.y;
  const int64_t slot = (int64_t)a.index[s] + u.t;
  const uint64_t at = ((uint64_t)s * a.n_rows + u.t) * a.row_stride + (uint64_t)u.h * D + 8 * u.lane;
  const float4 k0 = ld4<TYPE>(a.k, at), k1 = ld4<TYPE>(a.k, at + 4);
  const float4 v0 = ld4<TYPE>(a.v, at), v1 = ld4<TYPE>(a.v, at + 4);
  const int page = u.in && (!a.counts || (int64_t)u.t < a.counts[s]) ? page_of(g, s, slot) : -1;
  const float k[8] = {k0.x, k0.y, k0.z, k0.w, k1.x, k1.y, k1.z, k1.w};
  const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
  uint32_t km, vm;
  const uint32_t kw = quantise4(k, km), vw = quantise4(v, vm);
  if (page < 0) return;
  using H = PageHead<D>;
  uint8_t* to = g.data + a.layer + (uint64_t)page * g.page_bytes() + (uint64_t)u.h * g.head_bytes();
  const uint32_t r = (uint32_t)slot & (g.size() - 1), c = r * H::kCode + 4 * u.lane, m = r * H::kMeta + u.lane;
  *reinterpret_cast<uint32_t*>(to + H::codes(0, g.shift) + c) = kw;
  *reinterpret_cast<uint32_t*>(to + H::codes(1, g.shift) + c) = vw;
  if ((u.lane & 3) == 0) {
    *reinterpret_cast<uint32_t*>(to + H::meta(0, g.shift) + m) = km;
    *reinterpret_cast<uint32_t*>(to + H::meta(1, g.shift) + m) = vm;
  }
}

template <int TYPE, int D>
__global__ __launch_bounds__(kBlock) void k_pages_load(PageRowsArgs a) {
  const PageGeom& g = a.g;
  const PageUnit<D> u(a);
  const uint32_t s = blockIdx.y;
  const uint64_t out = (uint64_t)s * a.n_rows + u.t;
  const int slot = a.index ? a.index[out] : (int)u.t;
  const int page = u.in ? page_of(g, s, slot) : -1;
  if (page < 0) return;
  using H = PageHead<D>;
  const uint8_t* from = g.data + a.layer + (uint64_t)page * g.page_bytes() + (uint64_t)u.h * g.head_bytes();
  const uint32_t r = (uint32_t)slot & (g.size() - 1), c = r * H::kCode + 4 * u.lane, m = r * H::kMeta + (u.lane & ~3);
  const uint64_t to = out * a.row_stride + (uint64_t)u.h * D + 8 * u.lane;
  uint32_t w[2], meta[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    w[i] = *reinterpret_cast<const uint32_t*>(from + H::codes(i, g.shift) + c);
    meta[i] = *reinterpret_cast<const uint32_t*>(from + H::meta(i, g.shift) + m);
  }
  const Decoder decode;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    hx2 step, low;
    group_word(meta[i], step, low);
    const uint4 x = decode.eight(w[i], step, low);
    st4<TYPE>(i ? a.v : a.k, to, make_float4(h2f(x.x), h2f(x.x >> 16), h2f(x.y), h2f(x.y >> 16)));
    st4<TYPE>(i ? a.v : a.k, to + 4, make_float4(h2f(x.z), h2f(x.z >> 16), h2f(x.w), h2f(x.w >> 16)));
  }
}

// ---------------------------------------------------------------- the table
// Entries that slots below `slots` need.
__device__ __forceinline__ int entries_of(const PageGeom& g, int slots) {
  return (int)(((int64_t)max(slots, 0) + g.size() - 1) >> g.shift);
}

// Entry (s, e) of the forked table into the workspace, its holder counted (where another page
// comes: beams share most of theirs with their parents already).
__global__ __launch_bounds__(kBlock) void k_pages_fork_read(PageGeom g, const int32_t* parent, const int32_t* keep,
                                                            int32_t* ws) {
  const uint32_t s = blockIdx.y, e = blockIdx.x * kBlock + threadIdx.x;
  if (e >= (uint32_t)g.n_table) return;
  const int p = parent[s];
  int page = -1;
  if (p >= 0 && p < g.n_seq && (!keep || (int)e < entries_of(g, keep[s]))) page = g.table[(uint64_t)p * g.n_table + e];
  if (page < 0 || page >= g.n_page) page = -1;
  ws[(uint64_t)s * g.n_table + e] = page;
  if (page >= 0 && page != g.table[(uint64_t)s * g.n_table + e]) atomicAdd(&g.refs[page], 1);
}

__global__ __launch_bounds__(kBlock) void k_pages_fork_write(PageGeom g, const int32_t* ws) {
  const uint32_t s = blockIdx.y, e = blockIdx.x * kBlock + threadIdx.x;
  if (e >= (uint32_t)g.n_table) return;
  const uint64_t i = (uint64_t)s * g.n_table + e;
  const int old = g.table[i], page = ws[i];
  if (old == page) return;
  if (old >= 0 && old < g.n_page) atomicSub(&g.refs[old], 1);
  g.table[i] = page;
}

// Both by one workgroup, of tables up to kForkOne entries.
constexpr int kForkEach = 8, kForkOne = 1024 * kForkEach;
__global__ __launch_bounds__(1024) void k_pages_fork(PageGeom g, const int32_t* parent, const int32_t* keep) {
  const uint32_t total = (uint32_t)g.n_seq * g.n_table;
  int old[kForkEach], page[kForkEach];
#pragma unroll
  for (int k = 0; k < kForkEach; ++k) {
    const uint32_t i = threadIdx.x + 1024 * k, j = min(i, total - 1), s = j / g.n_table, e = j - s * g.n_table;
    old[k] = g.table[j];
    const int p = parent[s];
    int v = -1;
    if (p >= 0 && p < g.n_seq && (!keep || (int)e < entries_of(g, keep[s]))) v = g.table[(uint32_t)p * g.n_table + e];
    page[k] = v >= 0 && v < g.n_page ? v : -1;
  }
  __builtin_amdgcn_s_waitcnt(0);  // every entry has been read
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kForkEach; ++k) {
    const uint32_t i = threadIdx.x + 1024 * k;
    if (i >= total || old[k] == page[k]) continue;
    if (old[k] >= 0 && old[k] < g.n_page) atomicSub(&g.refs[old[k]], 1);
    if (page[k] >= 0) atomicAdd(&g.refs[page[k]], 1);
    g.table[i] = page[k];
  }
}

__global__ __launch_bounds__(kBlock) void k_pages_free(PageGeom g, const int32_t* keep) {
  const uint32_t s = blockIdx.y, e = blockIdx.x * kBlock + threadIdx.x;
  const int n = keep[s];
  if (e >= (uint32_t)g.n_table || n < 0 || (int)e < entries_of(g, n)) return;
  const uint64_t i = (uint64_t)s * g.n_table + e;
  const int old = g.table[i];
  if (old >= 0 && old < g.n_page) atomicSub(&g.refs[old], 1);
  g.table[i] = -1;
}

// Workspace of a reservation, in words: the copies' count and their (source,
// destination, rows); of each page how many entries ask to replace it and the last of
// them; the entries that get a free page, and the free pages, in order.
struct ReserveWs {
  int32_t *count, *copies, *asked, *last, *fresh, *unused;
  __host__ __device__ ReserveWs(int32_t* p, int n_page)
      : count(p), copies(p + 4), asked(copies + 3 * (uint64_t)n_page), last(asked + n_page), fresh(last + n_page),
        unused(fresh + n_page) {}
};

constexpr int kMaxSeq = 4096, kPlan = 1024, kPlanWaves = kPlan / 64, kPlanFew = 64;

// How many of the workgroup's flags are set before this thread's, and in all.
__device__ __forceinline__ int flags_before(bool f, int* waves, int& total) {
  const uint64_t b = __ballot(f);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  __syncthreads();
  if (lane == 0) waves[wave] = __popcll(b);
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < kPlanWaves; ++i) {
    if (i < wave) before += waves[i];
    total += waves[i];
  }
  return before + __popcll(b & ((1ull << lane) - 1));
}

__device__ __forceinline__ int ld_agent(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Which entries get which page, by one workgroup: the answer hangs on an order over all
// sequences (lowest page first, all or none), and the entries of a step are few.  The
// asked entries of all sequences are numbered through, and each thread takes every
// 1024th.  Nothing but latency: 5 to 6 us for 4 to 32 sequences, a chain of lengths, table,
// holders and stores with ten barriers between them, while enough free pages lie among the
// first 4096, whose counts are fetched ahead.  Each 4096 further are a round trip more: with the
// free pages last, a call over 4,000, 60,000, 250,000 and 1,000,000 pages takes 6, 24, 86 and
// 326 us.  So do entries past the first 1024, which each pass looks up anew: 1,024, 4,032 and
// 32,256 of them 7, 15 and 119 us.
__global__ __launch_bounds__(kPlan) void k_pages_plan(PageReserveArgs a) {
  const PageGeom& g = a.g;
  const ReserveWs ws(a.ws, g.n_page);
  __shared__ int first[kMaxSeq + 1];  // asked entries of the sequences before
  __shared__ int lowest[kMaxSeq];     // a sequence's first asked entry
  __shared__ int waves[kPlanWaves], counts[64], n_copies;
  __shared__ int pages[kPlanFew], free_pages[kPlan];  // shared pages asked for (few entries); the first free ones
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // (of the first 4096 pages which are free, fetched before anything waits)
  auto free_of = [&](int p0, int i) {
    const int p = p0 + wave * 256 + 64 * i + lane;
    return p < g.n_page && g.refs[p] <= 0;
  };
  bool free0[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) free0[i] = free_of(0, i);

  int n_asked = 0;
  for (int s0 = 0; s0 < g.n_seq; s0 += kPlan) {
    const int s = s0 + tid;
    int lo = 0, n = 0;
    if (s < g.n_seq) {
      const int want = a.want[s], from = max((a.start ? a.start : a.length)[s], 0);
      lo = from >> g.shift;
      n = want > from ? max(min(entries_of(g, want), g.n_table) - lo, 0) : 0;
      lowest[s] = lo;
    }
    int sum = n;  // up to this lane
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = sum;
    __syncthreads();
    int before = n_asked;
#pragma unroll
    for (int i = 0; i < kPlanWaves; ++i) {
      if (i < wave) before += waves[i];
      n_asked += waves[i];
    }
    if (s < g.n_seq) first[s] = before + sum - n;
  }
  if (tid == 0) {
    first[g.n_seq] = n_asked;
    n_copies = 0;
  }
  __syncthreads();

  // entry number f: its place in the table, the page that it holds (-1: none), that page's
  // holders and its sequence's length.  A thread's first one is kept: a step's entries are
  // rarely more.
  struct Entry {
    int at, e, length, page, holders;
  };
  auto find = [&](int f) {
    Entry x;
    int lo = 0, hi = g.n_seq;  // first[lo] <= f < first[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (first[mid] <= f) lo = mid;
      else hi = mid;
    }
    x.length = a.length[lo];
    x.e = lowest[lo] + (f - first[lo]);
    x.at = lo * g.n_table + x.e;
    x.page = g.table[x.at];
    if (x.page < 0 || x.page >= g.n_page) x.page = -1;
    x.holders = x.page < 0 ? 0 : g.refs[x.page];
    return x;
  };
  Entry mine{0, 0, 0, -1, 0};
  if (tid < n_asked) mine = find(tid);
  auto entry = [&](int f) { return f == tid ? mine : find(f); };
  auto each_shared = [&](auto&& fn) {
    for (int f = tid; f < n_asked; f += kPlan) {
      const Entry x = entry(f);
      if (x.holders > 1) fn(x);
    }
    __builtin_amdgcn_s_waitcnt(0);  // (stores, then atomics, of one page by several waves)
    __syncthreads();
  };
  // How many entries ask to replace a page, and the last of them: with few entries each
  // counts for itself (32 entries 9.2 us a call against 10.2, 64 10.9 against 12.0; of 128 1.0
  // more), else by atomics (where any page has other holders).
  const bool few = n_asked <= kPlanFew;
  int asked = 0, last = -1;
  if (few) {
    if (tid < n_asked) pages[tid] = mine.holders > 1 ? mine.page : -1;
    __syncthreads();
    if (mine.holders > 1)
      for (int i = 0; i < n_asked; ++i)
        if (pages[i] == mine.page) {
          ++asked;
          last = i;  // (entries are numbered in the table's order)
        }
  } else {
    bool shared = mine.holders > 1;
    for (int f = tid + kPlan; f < n_asked; f += kPlan) shared |= find(f).holders > 1;
    if (__syncthreads_or(shared)) {
      each_shared([&](const Entry& x) {
        ws.asked[x.page] = 0;
        ws.last[x.page] = -1;
      });
      each_shared([&](const Entry& x) {
        atomicAdd(&ws.asked[x.page], 1);
        atomicMax(&ws.last[x.page], x.at);
      });
    }
  }
  int n_fresh = 0, n_first = 0, rank = -1;  // of the first 1024 entries: how many, and this thread's number
  for (int f0 = 0; f0 < n_asked; f0 += kPlan) {
    const int f = f0 + tid;
    bool fresh = false;
    if (f < n_asked) {
      const Entry x = entry(f);
      fresh = x.page < 0;
      if (x.holders > 1)
        fresh = few ? asked != x.holders || last != f
                    : ld_agent(&ws.asked[x.page]) != x.holders || ld_agent(&ws.last[x.page]) != x.at;
    }
    int n;
    const int i = n_fresh + flags_before(fresh, waves, n);
    n_fresh += n;
    if (f0 == 0) {
      n_first = n_fresh;
      if (fresh) rank = i;
    } else if (fresh && i < g.n_page) {
      ws.fresh[i] = f;
    }
  }
  // the free pages, in order, until there are enough: four in a row of 64 lanes at a time
  int found = 0;
  for (int p0 = 0; p0 < g.n_page && found < n_fresh; p0 += 4 * kPlan) {
    uint64_t b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      b[i] = __ballot(p0 == 0 ? free0[i] : free_of(p0, i));
    }
    __syncthreads();
    if (lane < 4) counts[4 * wave + lane] = __popcll(lane == 0 ? b[0] : lane == 1 ? b[1] : lane == 2 ? b[2] : b[3]);
    __syncthreads();
    int sum = counts[lane];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(sum, d);
      if (lane >= d) sum += v;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = found + __shfl(sum, 4 * wave + i) - __popcll(b[i]) + __popcll(b[i] & ((1ull << lane) - 1));
      const int p = p0 + wave * 256 + 64 * i + lane;
      if (!((b[i] >> lane) & 1)) continue;
      if (at < kPlan) free_pages[at] = p;
      else ws.unused[at] = p;
    }
    found += __shfl(sum, 63);
  }
  __syncthreads();
  if (found < n_fresh) {
    if (tid == 0) {
      *a.missing = n_fresh - found;
      *ws.count = 0;
    }
    return;
  }
  auto give = [&](const Entry& x, int page) {
    g.table[x.at] = page;
    g.refs[page] = 1;
    if (x.page < 0) return;
    atomicSub(&g.refs[x.page], 1);
    const int64_t rows = min((int64_t)x.length - ((int64_t)x.e << g.shift), (int64_t)g.size());
    if (rows <= 0) return;
    int32_t* c = ws.copies + 3 * (uint64_t)atomicAdd(&n_copies, 1);
    c[0] = x.page;
    c[1] = page;
    c[2] = (int)rows;
  };
  if (rank >= 0) give(mine, free_pages[rank]);
  for (int i = n_first + tid; i < n_fresh; i += kPlan) give(find(ws.fresh[i]), i < kPlan ? free_pages[i] : ws.unused[i]);
  __syncthreads();
  if (tid == 0) {
    *a.missing = 0;
    *ws.count = n_copies;
  }
}

// The first rows of pages copied, a layer per blockIdx.y, kBlock units of a page a
// workgroup: units of D/8 bytes, of a row four of key codes, four of value codes and one
// of either's words.  (Where nothing or one page a sequence is copied, 1.6 to 4 us, a launch.
// One load a thread is in flight, behind the count, the copy's entry and its rows: a reservation
// that copies 250 pages of 41 KB in 48 layers takes 262 us, 3.7 TB/s, where k_pages_copy, with
// four, moves them in 182.)
template <int D>
__global__ __launch_bounds__(kBlock) void k_pages_cow(PageGeom g, int32_t* words, uint32_t pieces) {
  using P = Piece<D>;
  const ReserveWs ws(words, g.n_page);
  const uint64_t n = (uint64_t)*ws.count * pieces;
  uint8_t* layer = g.data + (uint64_t)blockIdx.y * g.n_page * g.page_bytes();
  for (uint64_t w = blockIdx.x; w < n; w += gridDim.x) {
    const uint32_t i = (uint32_t)(w / pieces);
    const uint32_t rows = ws.copies[3 * (uint64_t)i + 2], units = 10 * rows;
    const uint32_t u = (uint32_t)(w - (uint64_t)i * pieces) * kBlock + threadIdx.x;
    if (u >= units * g.n_head_kv) continue;
    const P* from = reinterpret_cast<const P*>(layer + (uint64_t)ws.copies[3 * (uint64_t)i] * g.page_bytes());
    P* to = reinterpret_cast<P*>(layer + (uint64_t)ws.copies[3 * (uint64_t)i + 1] * g.page_bytes());
    const uint32_t h = u / units, r = u - h * units;
    const uint32_t at = r < 4 * rows   ? r
                        : r < 8 * rows ? (4u << g.shift) + r - 4 * rows
                        : r < 9 * rows ? (8u << g.shift) + r - 8 * rows
                                       : (9u << g.shift) + r - 9 * rows;
    const uint32_t o = h * (10u << g.shift) + at;
    to[o] = from[o];
  }
}

// Rows moved together in place.  A workgroup has `width` of the 10 n_head_kv pieces of a
// layer's rows of a sequence (of a head: four of key codes and one of its words, the same of
// values) and takes the rows in order, `batch` at a time, which are all read before one is
// written: a row's new slot is at or below its old one, so none is overwritten before it has
// been read, and the next batch is fetched while this one is written.
// What bounds it: memory.  8000 of 16,000 slots, at random, in 48 layers of 4 kv heads are
// 246 MB of rows, but lie in three quarters of the codes' lines of 128 bytes and in all of the
// words': by the counters 3.07 million lines, 393 MB, read and 246 MB written, 132 us a call,
// 4.8 TB/s (4858 and 6984 kept 86 and 118).
struct MoveArgs {
  PageGeom g;
  const int32_t *start, *rows, *counts;
  int n_rows, width, batch;
  uint32_t by_width;  // 2^32 / width rounded up: i / width for i below 2^16
};
constexpr int kMoveBatch = 2 * kBlock;  // at most
constexpr int kMoveFew = 256;
template <int D, int PIECES>
__global__ __launch_bounds__(kBlock) void k_pages_compact(MoveArgs a) {
  using P = Piece<D>;
  const PageGeom& g = a.g;
  const uint32_t s = blockIdx.z, q0 = blockIdx.x * a.width;
  const int tid = threadIdx.x;
  const int64_t to0 = a.start[s];
  // (unsigned: the first row past the last batch may lie beyond 2^31)
  const uint32_t n = a.counts ? min(max(a.counts[s], 0), a.n_rows) : a.n_rows;
  if (n == 0) return;
  P* layer = reinterpret_cast<P*>(g.data + (uint64_t)blockIdx.y * g.n_page * g.page_bytes());
  const uint32_t head = 10u << g.shift, size = g.size();
  // a batch's rows: pages and rows in them of the old slot and the new, page -1 if it stays
  // (three buffers: a wave may look up the next batch while another writes the one before)
  __shared__ int src[3][kMoveBatch], dst[3][kMoveBatch], src_row[3][kMoveBatch];
  auto look_up = [&](uint32_t i0, int buf) {
#pragma unroll
    for (int r = tid; r < kMoveBatch; r += kBlock) {
      if (r >= a.batch) break;
      const uint32_t i = i0 + r;
      int p = -1, q = -1, from = 0;
      if (i < n) {
        from = a.rows[(uint64_t)s * a.n_rows + i];
        q = page_of(g, s, to0 + i);
        p = from == to0 + i || q < 0 ? -1 : page_of(g, s, from);
      }
      src[buf][r] = p;
      dst[buf][r] = q;
      src_row[buf][r] = from & (size - 1);
    }
  };
  // this thread's pieces: rows of a batch, and their places in a page (without the row)
  int row[PIECES];
  uint32_t at[PIECES], step[PIECES];
#pragma unroll
  for (int k = 0; k < PIECES; ++k) {
    const uint32_t i = tid + kBlock * k;
    row[k] = (int)__umulhi(i, a.by_width);
    const uint32_t q = q0 + i - row[k] * a.width, h = q / 10, r = q - 10 * h;
    const bool in = row[k] < a.batch && q < 10u * g.n_head_kv;
    if (!in) row[k] = -1;
    const uint32_t v = r >= 5, part = r - 5 * v;  // of which matrix, which
    step[k] = part < 4 ? 4 : 1;
    at[k] = in ? h * head + (part < 4 ? (4 * v << g.shift) + part : (8 + v) << g.shift) : 0;
  }
  P x[2][PIECES];
  // (a piece that stays is read all the same, from page 0)
  auto fetch = [&](int buf, P (&x)[PIECES]) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      const int r = max(row[k], 0), p = max(src[buf][r], 0);
      x[k] = layer[(uint64_t)p * g.n_head_kv * head + at[k] + step[k] * src_row[buf][r]];
    }
  };
  auto put = [&](uint32_t i0, int buf, const P (&x)[PIECES]) {
#pragma unroll
    for (int k = 0; k < PIECES; ++k) {
      if (row[k] < 0 || src[buf][row[k]] < 0) continue;
      const uint32_t r = (uint32_t)(to0 + i0 + row[k]) & (size - 1);
      layer[(uint64_t)dst[buf][row[k]] * g.n_head_kv * head + at[k] + step[k] * r] = x[k];
    }
  };
  look_up(0, 0);
  __syncthreads();
  fetch(0, x[0]);
  int buf = 0;
  for (uint32_t i0 = 0; i0 < n; i0 += 2 * a.batch) {
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const uint32_t i = i0 + b * a.batch;
      const int next = buf == 2 ? 0 : buf + 1;
      if (i >= n) break;
      const bool more = i + a.batch < n;
      if (more) look_up(i + a.batch, next);
      __builtin_amdgcn_s_waitcnt(0);  // every piece of this batch has been read
      __syncthreads();
      if (more) fetch(next, x[b ^ 1]);
      put(i, buf, x[b]);
      buf = next;
    }
  }
}

// Whole pages, a layer per blockIdx.y: 16 KB a workgroup, four 16-byte loads a thread (400
// pages of 41 KB in 48 layers, 1.57 GB both ways: 298 us, 5.3 TB/s, as fast as a plain copy).
constexpr int kCopyPiece = 4 * kBlock;  // of 16 bytes
__global__ __launch_bounds__(kBlock) void k_pages_copy(PageGeom to, PageGeom from, const int32_t* dst, const int32_t* src,
                                                       uint32_t pieces, uint64_t n) {
  const uint32_t units = to.page_bytes() / 16;
  for (uint64_t w = blockIdx.x; w < n; w += gridDim.x) {
    const uint32_t i = (uint32_t)(w / pieces);
    const int p = src[i], q = dst[i];
    if (p < 0 || p >= from.n_page || q < 0 || q >= to.n_page) continue;
    const u32v4* f = reinterpret_cast<const u32v4*>(from.data + ((uint64_t)blockIdx.y * from.n_page + p) * from.page_bytes());
    u32v4* t = reinterpret_cast<u32v4*>(to.data + ((uint64_t)blockIdx.y * to.n_page + q) * to.page_bytes());
    const uint32_t u0 = (uint32_t)(w - (uint64_t)i * pieces) * kCopyPiece + threadIdx.x;
    u32v4 x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) x[k] = f[min(u0 + k * kBlock, units - 1)];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (u0 + k * kBlock < units) t[u0 + k * kBlock] = x[k];
  }
}

dim3 page_rows_grid(const PageRowsArgs& a) {
  const uint32_t units = (uint32_t)a.n_rows * a.g.n_head_kv, per = kBlock / (a.g.head_dim / 8);
  return dim3((units + per - 1) / per, a.g.n_seq);
}
dim3 table_grid(const PageGeom& g) { return dim3((g.n_table + kBlock - 1) / kBlock, g.n_seq); }

}  // namespace

#define KNJ_PAGE_ROWS(KERNEL)                                                                       \
  do {                                                                                              \
    const dim3 grid = page_rows_grid(a);                                                            \
    if (type == KNJ_TYPE_F32) KNJ_PAGE_DIM(KERNEL, KNJ_TYPE_F32);                                   \
    else if (type == KNJ_TYPE_F16) KNJ_PAGE_DIM(KERNEL, KNJ_TYPE_F16);                              \
    else KNJ_PAGE_DIM(KERNEL, KNJ_TYPE_BF16);                                                       \
    return hipGetLastError();                                                                       \
  } while (0)
#define KNJ_PAGE_DIM(KERNEL, TYPE)                                                                  \
  do {                                                                                              \
    if (a.g.head_dim == 128) KNJ_LAUNCH((KERNEL<TYPE, 128>), grid, dim3(kBlock), 0, s, a);          \
    else KNJ_LAUNCH((KERNEL<TYPE, 64>), grid, dim3(kBlock), 0, s, a);                               \
  } while (0)

hipError_t launch_pages_store(int type, const PageRowsArgs& a, hipStream_t s) { KNJ_PAGE_ROWS(k_pages_store); }
hipError_t launch_pages_load(int type, const PageRowsArgs& a, hipStream_t s) { KNJ_PAGE_ROWS(k_pages_load); }

uint64_t page_workspace_ints(const PageGeom& g) {
  return std::max<uint64_t>(4 + 7 * (uint64_t)g.n_page, (uint64_t)g.n_seq * g.n_table);
}

hipError_t launch_pages_reserve(const PageReserveArgs& a, hipStream_t s) {
  KNJ_LAUNCH(k_pages_plan, dim3(1), dim3(kPlan), 0, s, a);
  // (how many pages are copied is known on the device only: as many workgroups as a page
  // of each sequence needs, to eight a CU)
  const uint32_t pieces = (a.g.page_bytes() / (a.g.head_dim / 8) + kBlock - 1) / kBlock;
  const uint64_t want = std::min<uint64_t>((uint64_t)pieces * a.g.n_seq, 2048 / a.g.n_layer);
  const dim3 grid((uint32_t)std::max<uint64_t>(want, 1), a.g.n_layer);
  if (a.g.head_dim == 128) KNJ_LAUNCH(k_pages_cow<128>, grid, dim3(kBlock), 0, s, a.g, a.ws, pieces);
  else KNJ_LAUNCH(k_pages_cow<64>, grid, dim3(kBlock), 0, s, a.g, a.ws, pieces);
  return hipGetLastError();
}

hipError_t launch_pages_fork(const PageGeom& g, const int32_t* parent, const int32_t* keep, int32_t* ws, hipStream_t s) {
  // (one launch: 4 beams of 17 pages 4.2 us against 6.5 in two, 32 of 126 4.3 against 6.0, 32 of
  // 256 5.4 against 6.0)
  if ((int64_t)g.n_seq * g.n_table <= kForkOne) {
    KNJ_LAUNCH(k_pages_fork, dim3(1), dim3(1024), 0, s, g, parent, keep);
    return hipGetLastError();
  }
  KNJ_LAUNCH(k_pages_fork_read, table_grid(g), dim3(kBlock), 0, s, g, parent, keep, ws);
  KNJ_LAUNCH(k_pages_fork_write, table_grid(g), dim3(kBlock), 0, s, g, ws);
  return hipGetLastError();
}

hipError_t launch_pages_free(const PageGeom& g, const int32_t* keep, hipStream_t s) {
  KNJ_LAUNCH(k_pages_free, table_grid(g), dim3(kBlock), 0, s, g, keep);
  return hipGetLastError();
}

hipError_t launch_pages_compact(const PageGeom& g, const int32_t* start, const int32_t* rows, const int32_t* counts,
                                int n_rows, hipStream_t s) {
  // A head's rows to a workgroup.  Few rows: two pieces a thread (48 layers x 4 kv heads, 8, 12
  // and 32 sequences of 60, 100 and 200 rows 7.4, 15.0 and 83 us against 11.4, 18.6 and 87 with
  // ten; one of 500 10.4 against 8.7, of 8000 182 against 128), and so few that those of all
  // heads fit at once, all of a layer's (32 of 8 rows 5.2 us against 9.9; 4 of 8 in 24 layers
  // 5.0 and 4.8).  Many rows in few layers: a matrix's (one of 8000 in 24 layers 55 us against
  // 70; in 48 layers 128 and 127).
  const int all = 10 * std::min(g.n_head_kv, 16), pieces = n_rows <= kMoveFew ? 2 : 10;
  const int64_t heads = (int64_t)g.n_layer * g.n_seq * g.n_head_kv;
  const int width = (int64_t)n_rows * all <= 2 * dev::kBlock ? all : pieces == 10 && heads < 128 ? 5 : 10;
  const int parts = (10 * g.n_head_kv + width - 1) / width;
  const int batch = std::min(pieces * dev::kBlock / width, kMoveBatch);
  const MoveArgs a{g, start, rows, counts, n_rows, width, batch, (uint32_t)((0x100000000ull + width - 1) / width)};
  const dim3 grid(parts, g.n_layer, g.n_seq);
#define KNJ_PAGE_COMPACT(D)                                                                    \
  do {                                                                                         \
    if (pieces == 2) KNJ_LAUNCH((k_pages_compact<D, 2>), grid, dim3(kBlock), 0, s, a);         \
    else KNJ_LAUNCH((k_pages_compact<D, 10>), grid, dim3(kBlock), 0, s, a);                    \
  } while (0)
  if (g.head_dim == 128) KNJ_PAGE_COMPACT(128);
  else KNJ_PAGE_COMPACT(64);
#undef KNJ_PAGE_COMPACT
  return hipGetLastError();
}

hipError_t launch_pages_copy(const PageGeom& to, const PageGeom& from, const int32_t* dst, const int32_t* src, int n,
                             hipStream_t s) {
  const uint32_t pieces = (to.page_bytes() / 16 + kCopyPiece - 1) / kCopyPiece;
  const uint64_t work = (uint64_t)pieces * n;
  KNJ_LAUNCH(k_pages_copy, dim3((uint32_t)std::min<uint64_t>(work, 1 << 20), to.n_layer), dim3(kBlock), 0, s, to, from,
             dst, src, pieces, work);
  return hipGetLastError();
}

}  // namespace knj

using namespace knj;

// The cache that the attention's sizes are taken from.
static knj_kv_cache page_cache(const PageGeom& g) {
  return {nullptr, nullptr, nullptr, nullptr, 0, kFormatPages, g.n_seq, g.n_head_kv, g.n_table << g.shift, g.head_dim};
}

// KNJ_E_ARG, with the reason, for sizes that are not a pool's; pointers are not looked at.
static int check_page_sizes(const knj_kv_pages* p) {
  KNJ_CHECK_ARG(p, "null pages");
  KNJ_CHECK_ARG(p->head_dim == 64 || p->head_dim == 128, "head_dim must be 64 or 128");
  KNJ_CHECK_ARG(p->page_size >= 16 && p->page_size <= 256 && (p->page_size & (p->page_size - 1)) == 0,
                "page_size must be a power of two from 16 to 256");
  KNJ_CHECK_ARG(p->n_head_kv > 0 && p->n_head_kv <= 64, "n_head_kv must be in [1, 64]");
  KNJ_CHECK_ARG(p->n_layer > 0 && p->n_layer <= 1024, "n_layer must be in [1, 1024]");
  KNJ_CHECK_ARG(p->n_page > 0 && p->n_page < (1 << 26), "n_page must be in [1, 2^26)");
  KNJ_CHECK_ARG(p->n_seq > 0 && p->n_seq <= kMaxSeq, "n_seq must be in [1, 4096]");
  KNJ_CHECK_ARG(p->n_table > 0 && (int64_t)p->n_table * p->page_size < kMaxSlots,
                "n_table must be positive and its slots fewer than 2^31 - 256");
  // (k_pages_plan's threads count entries in 32 bits, kPlan further than the last)
  KNJ_CHECK_ARG((int64_t)p->n_seq * p->n_table < (1ll << 31) - kPlan, "the table must have fewer than 2^31 - 1024 entries");
  return KNJ_OK;
}

static int check_pages(const knj_kv_pages* p, bool table, bool refs) {
  const int rc = check_page_sizes(p);
  if (rc) return rc;
  KNJ_CHECK_ARG(p->data && (!table || p->table) && (!refs || p->refs), "null pointer in the pages");
  KNJ_CHECK_ARG(((uintptr_t)p->data & 15) == 0, "page data must be 16-byte aligned");
  KNJ_CHECK_ARG(words_aligned(p->table, p->refs), "table and refs must be aligned to their type");
  return KNJ_OK;
}

static PageGeom geom(const knj_kv_pages& p) {
  int shift = 4;
  while ((1 << shift) < p.page_size) ++shift;
  return {(uint8_t*)p.data, p.table, p.refs, p.n_layer, p.n_page, shift, p.n_head_kv, p.head_dim, p.n_seq, p.n_table};
}

static uint64_t layer_at(const PageGeom& g, int layer) { return (uint64_t)layer * g.n_page * g.page_bytes(); }

static int check_page_rows(const knj_kv_pages* pages, int layer, int type, const void* k, const void* v,
                           uint64_t row_stride, int n_rows) {
  const int rc = check_pages(pages, true, false);
  if (rc) return rc;
  const int eb = act_bytes(type);
  KNJ_CHECK_ARG(layer >= 0 && layer < pages->n_layer, "the layer must be in [0, n_layer)");
  KNJ_CHECK_ARG(eb, "activations must be F32, F16 or BF16");
  KNJ_CHECK_ARG(k && v, "null pointer");
  KNJ_CHECK_ARG(n_rows >= 0, "negative row count");
  KNJ_CHECK_ARG(row_stride >= (uint64_t)pages->n_head_kv * pages->head_dim, "the row stride is below the row's width");
  KNJ_CHECK_ARG(rows_aligned(k, row_stride, eb) && rows_aligned(v, row_stride, eb),
                "rows must start on 16-byte boundaries");
  KNJ_CHECK_ARG((uint64_t)n_rows * pages->n_head_kv < (1ull << 27), "too many rows for one call");
  return KNJ_OK;
}

static int check_page_workspace(const knj_kv_pages* pages, const void* workspace, uint64_t bytes, const char* what) {
  const uint64_t need = page_workspace_ints(geom(*pages)) * sizeof(int32_t);
  if (workspace && bytes >= need && words_aligned((const char*)workspace)) return KNJ_OK;
  set_error(std::string(what) + ": these sizes need a 4-byte aligned workspace of " + std::to_string(need) + " bytes");
  return KNJ_E_ARG;
}

extern "C" {

uint64_t knj_pages_bytes(const knj_kv_pages* pages) {
  if (check_page_sizes(pages)) return 0;
  const PageGeom g = geom(*pages);
  return layer_at(g, g.n_layer);
}

uint64_t knj_pages_workspace(const knj_kv_pages* pages) {
  return check_page_sizes(pages) ? 0 : page_workspace_ints(geom(*pages)) * sizeof(int32_t);
}

int knj_pages_store(const knj_kv_pages* pages, int layer, int type, const void* k, const void* v,
                    uint64_t row_stride, const int32_t* start, const int32_t* counts, int n_rows,
                    void* stream) {
  int rc = check_page_rows(pages, layer, type, k, v, row_stride, n_rows);
  if (rc) return rc;
  KNJ_CHECK_ARG(start, "null start");
  KNJ_CHECK_ARG(words_aligned(start, counts), "start and counts must be aligned to their type");
  rc = require_device();
  if (rc || n_rows == 0) return rc;
  const PageGeom g = geom(*pages);
  KNJ_HIP(launch_pages_store(type, {g, layer_at(g, layer), const_cast<void*>(k), const_cast<void*>(v), row_stride, start,
                                    counts, n_rows}, (hipStream_t)stream));
  return KNJ_OK;
}

int knj_pages_load(const knj_kv_pages* pages, int layer, int type, const int32_t* slots,
                   int n_rows, void* k, void* v, uint64_t row_stride, void* stream) {
  int rc = check_page_rows(pages, layer, type, k, v, row_stride, n_rows);
  if (rc) return rc;
  KNJ_CHECK_ARG(words_aligned(slots), "slots must be aligned to their type");
  rc = require_device();
  if (rc || n_rows == 0) return rc;
  const PageGeom g = geom(*pages);
  KNJ_HIP(launch_pages_load(type, {g, layer_at(g, layer), k, v, row_stride, slots, nullptr, n_rows},
                            (hipStream_t)stream));
  return KNJ_OK;
}

int knj_pages_reserve(const knj_kv_pages* pages, const int32_t* start, const int32_t* length,
                      const int32_t* want, int32_t* missing, void* workspace,
                      uint64_t workspace_bytes, void* stream) {
  int rc = check_pages(pages, true, true);
  if (rc) return rc;
  KNJ_CHECK_ARG(length && want && missing, "null pointer");
  KNJ_CHECK_ARG(words_aligned(start, length, want, missing), "start, length, want and missing must be aligned to their type");
  rc = check_page_workspace(pages, workspace, workspace_bytes, "knj_pages_reserve");
  if (rc) return rc;
  rc = require_device();
  if (rc) return rc;
  KNJ_HIP(launch_pages_reserve({geom(*pages), start, length, want, missing, (int32_t*)workspace}, (hipStream_t)stream));
  return KNJ_OK;
}

int knj_pages_fork(const knj_kv_pages* pages, const int32_t* parent, const int32_t* keep,
                   void* workspace, uint64_t workspace_bytes, void* stream) {
  int rc = check_pages(pages, true, true);
  if (rc) return rc;
  KNJ_CHECK_ARG(parent, "null pointer");
  KNJ_CHECK_ARG(words_aligned(parent, keep), "parent and keep must be aligned to their type");
  rc = check_page_workspace(pages, workspace, workspace_bytes, "knj_pages_fork");
  if (rc) return rc;
  rc = require_device();
  if (rc) return rc;
  KNJ_HIP(launch_pages_fork(geom(*pages), parent, keep, (int32_t*)workspace, (hipStream_t)stream));
  return KNJ_OK;
}

int knj_pages_free(const knj_kv_pages* pages, const int32_t* keep, void* stream) {
  int rc = check_pages(pages, true, true);
  if (rc) return rc;
  KNJ_CHECK_ARG(keep, "null pointer");
  KNJ_CHECK_ARG(words_aligned(keep), "keep must be aligned to its type");
  rc = require_device();
  if (rc) return rc;
  KNJ_HIP(launch_pages_free(geom(*pages), keep, (hipStream_t)stream));
  return KNJ_OK;
}

int knj_pages_compact(const knj_kv_pages* pages, const int32_t* start, const int32_t* rows,
                      const int32_t* counts, int n_rows, void* stream) {
  int rc = check_pages(pages, true, false);
  if (rc) return rc;
  KNJ_CHECK_ARG(start && rows, "null pointer");
  KNJ_CHECK_ARG(words_aligned(start, rows, counts), "start, rows and counts must be aligned to their type");
  KNJ_CHECK_ARG(n_rows >= 0 && n_rows < kMaxSlots, "n_rows must be in [0, 2^31 - 256)");
  rc = require_device();
  if (rc || n_rows == 0) return rc;
  KNJ_HIP(launch_pages_compact(geom(*pages), start, rows, counts, n_rows, (hipStream_t)stream));
  return KNJ_OK;
}

int knj_pages_copy(const knj_kv_pages* to, const knj_kv_pages* from, const int32_t* dst,
                   const int32_t* src, int n, void* stream) {
  int rc = check_pages(to, false, false);
  if (!rc) rc = check_pages(from, false, false);
  if (rc) return rc;
  KNJ_CHECK_ARG(to->n_layer == from->n_layer && to->page_size == from->page_size && to->n_head_kv == from->n_head_kv &&
                    to->head_dim == from->head_dim,
                "the pools must have the same n_layer, page_size, n_head_kv and head_dim");
  KNJ_CHECK_ARG(dst && src, "null pointer");
  KNJ_CHECK_ARG(words_aligned(dst, src), "dst and src must be aligned to their type");
  KNJ_CHECK_ARG(n >= 0 && n < (1 << 24), "n must be in [0, 2^24)");
  rc = require_device();
  if (rc || n == 0) return rc;
  KNJ_HIP(launch_pages_copy(geom(*to), geom(*from), dst, src, n, (hipStream_t)stream));
  return KNJ_OK;
}

int knj_attention_pages(const knj_kv_pages* pages, int layer, int type, const void* q,
                        uint64_t q_stride, int n_head, int n_rows, const int32_t* prefix,
                        int max_prefix, const int32_t* counts, const uint64_t* mask,
                        int mask_shared, float scale, void* out, uint64_t out_stride,
                        void* workspace, uint64_t workspace_bytes, void* stream) {
  int rc = check_pages(pages, true, false);
  if (rc) return rc;
  KNJ_CHECK_ARG(layer >= 0 && layer < pages->n_layer, "the layer must be in [0, n_layer)");
  const PageGeom g = geom(*pages);
  TreeArgs a{page_cache(g), q, out, q_stride, out_stride, prefix, counts, mask, (float*)workspace, scale,
             n_head, n_rows, max_prefix, mask_shared, type, g.data + layer_at(g, layer), g.table, g.n_page, g.n_table,
             g.shift};
  rc = check_tree(a, workspace_bytes, "knj_attention_pages");
  if (rc) return rc;
  rc = require_device();
  if (rc || n_rows == 0) return rc;
  KNJ_HIP(launch_attention_tree(a, (hipStream_t)stream));
  return KNJ_OK;
}

uint64_t knj_attention_pages_workspace(const knj_kv_pages* pages, int n_head, int n_rows, int max_prefix) {
  return check_page_sizes(pages) ? 0 : tree_workspace(page_cache(geom(*pages)), n_head, n_rows, max_prefix);
}

}  // extern "C"
