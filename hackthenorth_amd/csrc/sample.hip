// Token sampling for gfx950: temperature, top-k, top-p, min-p and one uniform
// number per row, without sorting the vocabulary.
//
// The order of a row is falling logit, the lower id first among equals. Every
// truncation keeps a leading part of it, so a row's answer is a place in that
// order: the first token whose cumulative weight exp((x - max) / T) passes u times
// the weight kept. Weights are summed as integers, which do not depend on the
// order in which blocks and atomics take them: within a bin of 1/32 nat, 2^33 exp
// of the token's distance to the bin's edge (half a unit, 2^-34 of the weight, is
// lost a token), and a bin's sum times 2^11 exp of the edge, rounded, over the
// bins. Borders between tokens so fall where 64-bit sums put them but for some
// 2^-34 of a token's weight, and for the tokens 32 nats and more below the largest,
// which weigh nothing: e^-32 of the largest weight each, 524160 of them 2^-27. A
// draw of 24 bits never falls among them.
//
//   1. every chunk of a row: its largest logit;
//   2. every chunk: the count and weight of its tokens in 1024 bins below the
//      row's largest;
//   3. one block a row: from the running sums over the bins, those in which each
//      border can lie (top-k's is certain; the weight kept, and with it the later
//      borders, only within its bin's);
//   4. every chunk: its tokens in these bins as lists;
//   5. one block a row: each border in turn, its bin and then its tokens, by 1024
//      finer bins and by rank. Lists of more than 2048 tokens stay in memory; where
//      a chunk's own passes that, the bin's tokens are read again from the row. More
//      than 1024 in a finer bin (many equal logits) are narrowed by eight bits of
//      (logit, id) at a time.
//
// One row of 151936 bf16 logits takes 23.7 us: five launches of 3, 5, 6, 4.5 and
// 7 us, each a chain of loads, scans and barriers. 64 such rows in fp32 (39 MB) take
// 51: 6, 15, 9, 11 and 10.5 us, the second bound by its arithmetic (vector instructions
// issue in 83% of the cycles; two or four copies of the bins change nothing). A row of equal logits takes 165. Before the
// steps were as short, steps 2 + 3 and 4 + 5 in one launch each, by the row's last
// block, gained one row 0.8 us and cost 64 rows 12; steps 3 + 4, each block planning
// for itself, gained 1.6 and cost 2.
#include "common.h"

namespace htn {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 1024;        // one a thread
constexpr int kListed = 2048;      // tokens listed for a border, of a chunk
constexpr int kBorders = 3;        // top-k's, top-p's and the draw's
constexpr int kMaxChunks = 16;
constexpr long kChunk = 32760;     // tokens of a chunk at most
constexpr int kCountBit = 49;      // a chunk's bin: its count above, its weight (little over 2^48 at most) below
constexpr double kOne = 17592186044416.0;  // 2^44, the largest token's weight

// Bins [lo, hi] in which a border can lie, and the tokens in them.
struct Range {
  int lo, hi;
  uint32_t tokens;
};

struct RowPlan {
  Range range[kBorders];  // of borders that are not sought, none
  uint64_t all;      // weight of the row
  uint64_t floor_p;  // and of what min-p keeps
  int by_count, by_weight;
};

struct SampleArgs {
  const void* logits; long row_st;
  long vocab; int rows, chunks; long chunk;
  const float* uniform;
  const float* temperature; const int64_t* top_k; const float* top_p; const float* min_p;  // or null:
  float temperature_all; int64_t top_k_all; float top_p_all, min_p_all;                    // for all rows
  int64_t* out;
  float* maxima;        // [rows, chunks]
  uint64_t* bins;       // [rows, chunks, kBins]: count and weight
  uint64_t* edges;      // [rows, chunks, 3]: weight that min-p keeps in the bins around its border
  RowPlan* plans;       // [rows]
  uint32_t* counts;     // [rows, kBins]: running sums of the row
  uint64_t* weights;    // [rows, kBins]
  uint32_t* listed;     // [rows, chunks, kBorders]: tokens in the lists
  uint64_t* lists;      // [rows, chunks, kBorders, kListed]: order keys
};

__device__ __forceinline__ float logit_of(bf16_t v) { return bf2f(v); }
__device__ __forceinline__ float logit_of(float v) { return v; }

// f(x, id) for the elements [first, last) of a row, spread over the block: whole
// 16-byte vectors where the row's own alignment lets them, U at a time.
template <typename L, int U, typename F>
__device__ __forceinline__ void each_logit(const L* row, long first, long last, F&& f) {
  constexpr int E = 16 / sizeof(L);
  const int tid = threadIdx.x;
  const long off = static_cast<long>((reinterpret_cast<uintptr_t>(row + first) & 15) / sizeof(L));
  long body = off ? first + E - off : first;
  if (body > last) body = last;
  const long vecs = (last - body) / E, tail = body + vecs * E;
  if (first + tid < body) f(logit_of(row[first + tid]), first + tid);
  for (long v0 = 0; v0 < vecs; v0 += kThreads * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long v = v0 + u * kThreads + tid;
      w[u] = *reinterpret_cast<const uint4*>(row + body + (v < vecs ? v : 0) * E);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const long v = v0 + u * kThreads + tid;
      if (v >= vecs) continue;
      const long id = body + v * E;
      if constexpr (sizeof(L) == 2) {
        float x[8];
        unpack8(w[u], x);
#pragma unroll
        for (int i = 0; i < 8; ++i) f(x[i], id + i);
      } else {
        f(__uint_as_float(w[u].x), id);
        f(__uint_as_float(w[u].y), id + 1);
        f(__uint_as_float(w[u].z), id + 2);
        f(__uint_as_float(w[u].w), id + 3);
      }
    }
  }
  if (tail + tid < last) f(logit_of(row[tail + tid]), tail + tid);
}

__device__ __forceinline__ long chunk_end(const SampleArgs& a, long first) {
  return first + a.chunk < a.vocab ? first + a.chunk : a.vocab;
}

// The largest logit of a chunk; NaN counts as masked.
template <typename L>
__global__ __launch_bounds__(kThreads) void sample_max(SampleArgs a) {
  __shared__ float red[kWaves];
  const int r = blockIdx.y, c = blockIdx.x;
  const L* row = static_cast<const L*>(a.logits) + r * a.row_st;
  const long first = c * a.chunk;
  float m = -INFINITY;
  each_logit<L, 4>(row, first, chunk_end(a, first), [&](float x, long) { m = fmaxf(m, x); });
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, red[w]);
    a.maxima[r * a.chunks + c] = m;
  }
}

struct Row {
  float top;      // its largest logit (0 in place of +inf)
  bool none;      // every logit is masked
  bool infinite;  // +inf tokens share the row: they count as 0, the others as masked
  float heat;     // bins per unit of logit, for the bin
  double fine;    // the same for the weight
  bool greedy;
  double edge;    // bins below the largest to which min-p keeps tokens
  int edge_bin;
  bool cut;       // whether min-p cuts
};

__device__ __forceinline__ Row row_of(const SampleArgs& a, int r) {
  const int lane = threadIdx.x & 63;
  Row w;
  w.top = wave_max(lane < a.chunks ? a.maxima[r * a.chunks + lane] : -INFINITY);
  w.none = w.top == -INFINITY;
  w.infinite = w.top == INFINITY;
  w.top = w.infinite ? 0.f : w.top;
  const float t = a.temperature ? a.temperature[r] : a.temperature_all;
  const float min_p = a.min_p ? a.min_p[r] : a.min_p_all;
  w.greedy = !(t > 0.f);
  // Below 1e-36 the bins per unit would pass fp32's range; no logits but those
  // that differ by less than 1e-34 tell such temperatures apart.
  w.fine = w.greedy ? kBins / 32.0 : kBins / 32.0 / (t > 1e-36f ? static_cast<double>(t) : 1e-36);
  w.heat = static_cast<float>(w.fine);
  w.cut = !w.greedy && min_p > 0.f;
  w.edge = w.cut ? -log(static_cast<double>(min_p)) * (kBins / 32.0) : 0.0;
  // Past the bins either way: nothing or everything cut but the first token.
  w.edge_bin = w.edge < 2 * kBins ? (w.edge > -8.0 ? static_cast<int>(floor(w.edge)) : -8) : 2 * kBins;
  return w;
}

__device__ __forceinline__ float seen_logit(const Row& w, float x) {
  return w.infinite ? (x == INFINITY ? 0.f : -INFINITY) : x;
}

// The token's bin, rising as the logit falls (every step is monotone); kBins for
// one that weighs nothing: past the bins, or masked (-inf and NaN give an infinity
// or a NaN). In fp32: any split of the order that all passes agree on will do.
__device__ __forceinline__ int bin_of(const Row& w, float x) {
  const float y = (w.top - x) * w.heat;
  return y < kBins ? static_cast<int>(y) : kBins;
}

// Bins that the token lies past the near edge of bin b, exactly: in about [0, 1)
// for its own (bin_of is off by up to 1e-3).
__device__ __forceinline__ double past_edge(const Row& w, float x, int b) {
  return fma(static_cast<double>(w.top) - static_cast<double>(x), w.fine, -static_cast<double>(b));
}

// 2^33 exp(-y / 32) of a token y past its bin's edge: five terms of the Taylor sum
// (the next is 1.3e-12), as an integer by the shift of adding 2^52.
__device__ __forceinline__ uint64_t weight_in_bin(double y) {
  constexpr double h = -1.0 / 32.0;
  double s = fma(y, h * h * h * h * h / 120, h * h * h * h / 24);
  s = fma(y, s, h * h * h / 6);
  s = fma(y, s, h * h / 2);
  s = fma(y, s, h);
  s = fma(y, s, 1.0);
  return __double_as_longlong(fma(s, 8589934592.0, 4503599627370496.0)) - (0x433ULL << 52);
}

// What a unit of weight within bin b weighs in units of 2^-44 of the largest token.
__device__ __forceinline__ double unit_of(int b) { return 2048.0 * exp(b * (-1.0 / 32.0)); }

__device__ __forceinline__ uint64_t outside(uint64_t sum, double unit) {
  return static_cast<uint64_t>(static_cast<double>(sum) * unit + 0.5);
}

// Order of a row as one key: falling logit, rising id. -0 counts as 0.
__device__ __forceinline__ uint64_t order_key(float x, long id) {
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
  return (static_cast<uint64_t>(k) << 32) | (0xffffffffu - static_cast<uint32_t>(id));
}

__device__ __forceinline__ float key_logit(uint64_t key) {
  const uint32_t k = static_cast<uint32_t>(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

template <typename L>
__global__ __launch_bounds__(kThreads) void sample_histogram(SampleArgs a) {
  __shared__ unsigned long long bins[kBins], edges[3];
  const int tid = threadIdx.x, r = blockIdx.y, c = blockIdx.x;
  bins[tid] = 0;
  if (tid < 3) edges[tid] = 0;
  const Row w = row_of(a, r);
  __syncthreads();
  const L* row = static_cast<const L*>(a.logits) + r * a.row_st;
  const long first = c * a.chunk;
  each_logit<L, 2>(row, first, chunk_end(a, first), [&](float x, long) {
    x = seen_logit(w, x);
    const int b = bin_of(w, x);
    if (b >= kBins) return;
    const double y = past_edge(w, x, b);
    const uint64_t v = weight_in_bin(y);
    atomicAdd(&bins[b], static_cast<unsigned long long>(v + (1ULL << kCountBit)));
    // Bins before these are kept whole, those behind cut whole.
    if (w.cut && static_cast<uint32_t>(b - w.edge_bin + 1) <= 2u && b + y <= w.edge)
      atomicAdd(&edges[b - w.edge_bin + 1], static_cast<unsigned long long>(v));
  });
  __syncthreads();
  const long at = static_cast<long>(r) * a.chunks + c;
  a.bins[at * kBins + tid] = bins[tid];
  if (tid < 3) a.edges[at * 3 + tid] = edges[tid];
}

// Where a border lies: by count (the first `target` tokens), by weight before the
// token (below `goal`), or by weight up to it (past `goal`).
enum Kind { kCount, kBefore, kPast };

struct Border {
  Kind kind;
  uint64_t target;
  double goal;
};

// Whether `c` tokens that weigh `w` reach it.
__device__ __forceinline__ bool reached(const Border& b, uint32_t c, uint64_t w) {
  if (b.kind == kCount) return c >= b.target;
  if (b.kind == kBefore) return static_cast<double>(w) >= b.goal;
  return static_cast<double>(w) > b.goal;
}

struct Ranks {
  uint32_t wave_count[kWaves];
  uint64_t wave_weight[kWaves];
  int at;
  uint32_t count_before, here;
  uint64_t weight_before, weight_with;
};

// Running sums over the block's threads.
__device__ __forceinline__ void scan(Ranks& s, uint32_t& count, uint64_t& weight) {
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  count = wave_scan(count);
  weight = wave_scan(weight);
  __syncthreads();
  if (lane == 63) {
    s.wave_count[wave] = count;
    s.wave_weight[wave] = weight;
  }
  __syncthreads();
  // The sums of the waves before, scanned by each wave for itself.
  const uint32_t cs = row_scan(s.wave_count[lane & 15]);
  const uint64_t ws = row_scan(s.wave_weight[lane & 15]);
  if (wave > 0) {
    count += __builtin_amdgcn_readlane(cs, wave - 1);
    weight += static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(ws >> 32), wave - 1)) << 32 |
              static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(ws), wave - 1));
  }
}

// The first of the threads' entries that reaches the border, or holds the last of
// `end` tokens: sums c0, w0 before it and c1, w1 with it. Sums only grow, and those
// before the first are short of the border.
__device__ __forceinline__ void find_border(Ranks& s, const Border& b, uint32_t c0, uint64_t w0, uint32_t c1,
                                            uint64_t w1, uint32_t end) {
  __syncthreads();
  if (c0 < c1 && !reached(b, c0, w0) && (reached(b, c1, w1) || c1 == end)) {
    s.at = threadIdx.x;
    s.count_before = c0;
    s.weight_before = w0;
    s.weight_with = w1;
    s.here = c1 - c0;
  }
  __syncthreads();
}

struct Settings {
  int64_t top_k;
  float top_p, u;
};

__device__ __forceinline__ Settings settings_of(const SampleArgs& a, const Row& w, int r) {
  Settings s;
  s.top_k = w.greedy ? 1 : (a.top_k ? a.top_k[r] : a.top_k_all);
  s.top_p = w.greedy ? 1.f : (a.top_p ? a.top_p[r] : a.top_p_all);
  const float u = a.uniform[r];
  s.u = u > 0.f ? (u < 0.99999994f ? u : 0.99999994f) : 0.f;  // [0, 1 - 2^-24]
  return s;
}

// Top-p's border and the draw's, in terms of the weight kept up to then. The first
// token is always kept.
__device__ __forceinline__ Border border_p(const Settings& s, uint64_t kept) {
  const double g = static_cast<double>(s.top_p) * static_cast<double>(kept);
  return Border{kBefore, 0, g > 0.5 ? g : 0.5};
}
__device__ __forceinline__ Border border_u(const Settings& s, uint64_t kept) {
  return Border{kPast, 0, static_cast<double>(s.u) * static_cast<double>(kept)};
}
// Of p x kept >= kept (p of 1 and more) nothing is cut.
__device__ __forceinline__ bool cuts(const Settings& s, uint64_t kept) {
  return static_cast<double>(s.top_p) * static_cast<double>(kept) < static_cast<double>(kept);
}
__device__ __forceinline__ uint64_t least(uint64_t x, uint64_t y) { return x < y ? x : y; }

__global__ __launch_bounds__(kThreads) void sample_plan(SampleArgs a) {
  __shared__ Ranks ranks;
  __shared__ uint64_t whole;
  const int tid = threadIdx.x, lane = tid & 63, r = blockIdx.x;
  const long row_at = static_cast<long>(r) * a.chunks;
  // The row's bins (a thread's own one), and what min-p keeps at its edge: all loads
  // in flight at once.
  uint64_t v[kMaxChunks], edge[3];
#pragma unroll
  for (int i = 0; i < kMaxChunks; ++i) v[i] = i < a.chunks ? a.bins[(row_at + i) * kBins + tid] : 0;
#pragma unroll
  for (int i = 0; i < 3; ++i) edge[i] = lane < a.chunks ? a.edges[(row_at + lane) * 3 + i] : 0;
  const Row w = row_of(a, r);
  const Settings set = settings_of(a, w, r);
  if (w.none) return;
  uint32_t count = 0;
  uint64_t sum = 0;
#pragma unroll
  for (int i = 0; i < kMaxChunks; ++i) {
    count += static_cast<uint32_t>(v[i] >> kCountBit);
    sum += v[i] & ((1ULL << kCountBit) - 1);
  }
  if (tid == 0) whole = 0;
  uint32_t c1 = count;
  uint64_t w1 = outside(sum, unit_of(tid));
  const uint64_t weight = w1;
  scan(ranks, c1, w1);
  const uint32_t c0 = c1 - count;
  const uint64_t w0 = w1 - weight;
  if (tid == w.edge_bin - 2) whole = w1;
  __syncthreads();
  uint32_t all_c = 0;
  uint64_t all = 0;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    all_c += ranks.wave_count[v];
    all += ranks.wave_weight[v];
  }
  const uint64_t first = static_cast<uint64_t>(kOne);
  RowPlan p;
  p.all = all;
  p.floor_p = all;
  if (w.cut && w.edge_bin <= kBins + 1) {
    p.floor_p = whole;
#pragma unroll
    for (int i = 0; i < 3; ++i) {
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) edge[i] += __shfl_xor(edge[i], m, kWave);
      const int b = w.edge_bin - 1 + i;
      if (b >= 0 && b < kBins) p.floor_p += outside(edge[i], unit_of(b));
    }
    p.floor_p = p.floor_p > first ? p.floor_p : first;
  }
  // The bins that reach a border for the least and the most that its goal can be;
  // the weight before the first of them, and with the last (left in `ranks`).
  auto range_of = [&](Range& g, const Border& from, const Border& to) {
    find_border(ranks, from, c0, w0, c1, w1, all_c);
    g.lo = g.hi = ranks.at;
    g.tokens = ranks.here;
    const uint64_t before = ranks.weight_before;
    if (to.goal != from.goal) {
      const uint32_t behind = ranks.count_before;
      find_border(ranks, to, c0, w0, c1, w1, all_c);
      g.hi = ranks.at;
      g.tokens = ranks.count_before + ranks.here - behind;
    }
    return before > first ? before : first;
  };
  // Least and most that can be kept after each truncation.
  uint64_t kept_lo = all, kept_hi = all;
  p.range[0] = p.range[1] = Range{1, 0, 0};
  p.by_count = set.top_k > 0 && static_cast<uint64_t>(set.top_k) < all_c;
  if (p.by_count) {
    const Border k{kCount, static_cast<uint64_t>(set.top_k), 0.0};
    kept_lo = range_of(p.range[0], k, k);
    kept_hi = ranks.weight_with;
  }
  p.by_weight = cuts(set, kept_hi);
  if (p.by_weight) {
    kept_lo = least(kept_lo, range_of(p.range[1], border_p(set, kept_lo), border_p(set, kept_hi)));
    kept_hi = least(kept_hi, ranks.weight_with);
  }
  range_of(p.range[2], border_u(set, least(kept_lo, p.floor_p)), border_u(set, least(kept_hi, p.floor_p)));
  a.counts[static_cast<long>(r) * kBins + tid] = c1;
  a.weights[static_cast<long>(r) * kBins + tid] = w1;
  if (tid == 0) a.plans[r] = p;
}

template <typename L>
__global__ __launch_bounds__(kThreads) void sample_collect(SampleArgs a) {
  __shared__ uint32_t taken[kBorders];
  const int tid = threadIdx.x, r = blockIdx.y, c = blockIdx.x;
  if (tid < kBorders) taken[tid] = 0;
  const RowPlan& plan = a.plans[r];
  int lo[kBorders], any_lo = kBins, any_hi = -1;
  uint32_t span[kBorders];
#pragma unroll
  for (int i = 0; i < kBorders; ++i) {
    const Range g = plan.range[i];
    const bool on = g.hi >= g.lo && g.tokens <= static_cast<uint32_t>(a.chunks) * kListed;
    lo[i] = on ? g.lo : 2 * kBins;  // no bin is in it
    span[i] = on ? g.hi - g.lo : 0;
    any_lo = on && g.lo < any_lo ? g.lo : any_lo;
    any_hi = on && g.hi > any_hi ? g.hi : any_hi;
  }
  const Row w = row_of(a, r);
  if (w.none) return;  // no plan was made
  __syncthreads();
  const long at = static_cast<long>(r) * a.chunks + c;
  uint64_t* lists = a.lists + at * kBorders * kListed;
  const long from = c * a.chunk;
  if (any_hi >= any_lo)
    each_logit<L, 2>(static_cast<const L*>(a.logits) + r * a.row_st, from, chunk_end(a, from),
                     [&](float x, long id) {
                       x = seen_logit(w, x);
                       const int bin = bin_of(w, x);
                       if (bin < any_lo || bin > any_hi) return;
#pragma unroll
                       for (int i = 0; i < kBorders; ++i)
                         if (static_cast<uint32_t>(bin - lo[i]) <= span[i]) {
                           const uint32_t n = atomicAdd(&taken[i], 1u);
                           if (n < kListed) lists[i * kListed + n] = order_key(x, id);
                         }
                     });
  __syncthreads();
  if (tid < kBorders) a.listed[at * kBorders + tid] = taken[tid];
}

struct Found {
  uint64_t weight;  // of the tokens up to and with the one at the border
  uint32_t id;      // that token
};

struct Shared {
  Ranks ranks;
  Found found;
  uint64_t keys[kBorders][kListed], near[kThreads];
  uint32_t fine_count[kThreads];
  unsigned long long fine_weight[kThreads];
  uint32_t ends[kBorders][kMaxChunks];  // running sums of the chunks' lists
  uint32_t taken;
};

// The first n of the keys in falling order. Keys differ: up to 256 are ranked
// against each other, more go through a bitonic network.
__device__ __forceinline__ void sort_keys(uint64_t* keys, int n) {
  const int tid = threadIdx.x;
  __syncthreads();
  if (n <= 256) {
    const uint64_t key = tid < n ? keys[tid] : 0;
    int rank = 0;
    if (tid < n) {
#pragma unroll 8
      for (int i = 0; i < n; ++i) rank += keys[i] > key;
    }
    __syncthreads();
    if (tid < n) keys[rank] = key;
    __syncthreads();
    return;
  }
  if (tid >= n) keys[tid] = 0;  // below every key
  for (int k = 2; k <= kThreads; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      const int o = tid ^ j;
      if (o > tid) {
        const uint64_t x = keys[tid], y = keys[o];
        if ((x < y) == ((tid & k) == 0)) {
          keys[tid] = y;
          keys[o] = x;
        }
      }
    }
  __syncthreads();
}

// A place in the order: the tokens of `bin` there, behind `count` others of the
// row, `weight` before the bin and `sum` before them in it.
struct Place {
  int bin;
  uint32_t here, count;
  uint64_t weight, sum;
};

// The entry (tokens and weight within the bin, in thread order) of a place in
// which the border lies.
__device__ __forceinline__ void narrow(Ranks& s, Place& p, const Border& b, uint32_t count, uint64_t sum) {
  uint32_t c1 = count;
  uint64_t s1 = sum;
  scan(s, c1, s1);
  const uint64_t s0 = p.sum + s1 - sum;
  s1 += p.sum;
  const double unit = unit_of(p.bin);
  find_border(s, b, p.count + c1 - count, p.weight + outside(s0, unit), p.count + c1,
              p.weight + outside(s1, unit), p.count + p.here);
  if (threadIdx.x == s.at) s.weight_before = s0;
  __syncthreads();
  p.count = s.count_before;
  p.here = s.here;
  p.sum = s.weight_before;
}


__device__ __forceinline__ uint64_t key_weight(const Row& w, uint64_t key, int bin) {
  return weight_in_bin(past_edge(w, key_logit(key), bin));
}

// The border among the p.here <= 1024 keys of a place.
__device__ __forceinline__ Found among(Shared& s, const Row& w, uint64_t* keys, Place p, const Border& b) {
  const int tid = threadIdx.x, n = p.here;
  sort_keys(keys, n);
  narrow(s.ranks, p, b, tid < n ? 1u : 0u, tid < n ? key_weight(w, keys[tid], p.bin) : 0);
  return Found{s.ranks.weight_with, 0xffffffffu - static_cast<uint32_t>(keys[s.ranks.at] & 0xffffffffu)};
}

// The same among p.here <= 64 keys, by the first wave alone: the others wait at one
// barrier instead of taking their turns at scans and at eight.
__device__ __forceinline__ Found among_few(Shared& s, const Row& w, uint64_t* keys, const Place& p, const Border& b) {
  const int lane = threadIdx.x & 63, n = p.here;
  __syncthreads();
  if (threadIdx.x < kWave) {
    uint64_t key = lane < n ? keys[lane] : 0;
    int rank = 0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) rank += keys[i] > key;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < n) keys[rank] = key;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    key = lane < n ? keys[lane] : 0;
    const uint64_t own = lane < n ? key_weight(w, key, p.bin) : 0, s1 = p.sum + wave_scan(own);
    const double unit = unit_of(p.bin);
    const uint64_t w0 = p.weight + outside(s1 - own, unit), w1 = p.weight + outside(s1, unit);
    const uint32_t c0 = p.count + lane;
    if (lane < n && !reached(b, c0, w0) && (reached(b, c0 + 1, w1) || lane == n - 1))
      s.found = Found{w1, 0xffffffffu - static_cast<uint32_t>(key & 0xffffffffu)};
  }
  __syncthreads();
  return s.found;
}

// Narrows a place to 1024 tokens at most, by eight bits of the key at a time from
// the first in which they differ, and leaves their keys in `near`. each(f) calls
// f(key) for the tokens of the place's bin.
template <typename E>
__device__ __forceinline__ void by_digits(Shared& s, const Row& w, Place& p, const Border& b, E&& each) {
  const int tid = threadIdx.x;
  enum { kCommon, kDigits, kGather } step = kCommon;
  uint64_t all = ~0ULL, prefix = 0;
  int bits = 64, digit = 0;  // keys sought agree with the prefix above `bits`
#pragma unroll 1
  for (;;) {
    __syncthreads();
    if (step == kDigits) {
      s.fine_count[tid] = 0;
      s.fine_weight[tid] = 0;
    } else if (tid == 0) {
      s.taken = 0;
      s.near[0] = ~0ULL;
      s.near[1] = 0;
    }
    __syncthreads();
    each([&](uint64_t key) {
      if (step == kCommon) {
        all &= key;
        prefix |= key;
        return;
      }
      if (bits < 64 && (key ^ prefix) >> bits) return;
      if (step == kDigits) {
        // Larger keys first; four sums a digit, as neighbours tend to share it.
        const int d = 4 * (255 - static_cast<int>((key >> (bits - digit)) & ((1 << digit) - 1))) + (tid & 3);
        atomicAdd(&s.fine_count[d], 1u);
        atomicAdd(&s.fine_weight[d], static_cast<unsigned long long>(key_weight(w, key, p.bin)));
      } else {
        const uint32_t i = atomicAdd(&s.taken, 1u);
        if (i < kThreads) s.near[i] = key;
      }
    });
    if (step == kGather) return;
    if (step == kCommon) {
      atomicAnd(reinterpret_cast<unsigned long long*>(&s.near[0]), static_cast<unsigned long long>(all));
      atomicOr(reinterpret_cast<unsigned long long*>(&s.near[1]), static_cast<unsigned long long>(prefix));
      __syncthreads();
      prefix = s.near[1];
      const uint64_t differ = prefix & ~s.near[0];
      bits = differ ? 64 - __builtin_clzll(differ) : 0;
      prefix = bits < 64 ? prefix >> bits << bits : 0;
    } else {
      __syncthreads();
      uint32_t count = 0;
      uint64_t sum = 0;
      if (tid < 256) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          count += s.fine_count[4 * tid + i];
          sum += s.fine_weight[4 * tid + i];
        }
      }
      narrow(s.ranks, p, b, count, sum);
      bits -= digit;
      prefix |= static_cast<uint64_t>(255 - s.ranks.at) << bits;
    }
    step = p.here > kThreads && bits > 0 ? kDigits : kGather;
    digit = bits < 8 ? bits : 8;
  }
}

template <typename L>
__global__ __launch_bounds__(kThreads) void sample_pick(SampleArgs a) {
  __shared__ Shared s;
  const int tid = threadIdx.x, lane = tid & 63, r = blockIdx.x;
  const long row_at = static_cast<long>(r) * a.chunks;
  const uint32_t* counts = a.counts + static_cast<long>(r) * kBins;
  const uint64_t* weights = a.weights + static_cast<long>(r) * kBins;
  const uint32_t c1 = counts[tid], c0 = tid ? counts[tid - 1] : 0, all_c = counts[kBins - 1];
  const uint64_t w1 = weights[tid], w0 = tid ? weights[tid - 1] : 0;
  const RowPlan& plan = a.plans[r];
  if (tid < kBorders * kWave) {
    const int i = tid >> 6;
    uint32_t n = lane < a.chunks ? a.listed[(row_at + lane) * kBorders + i] : 0;
    if (__any(n > kListed)) n = 0;  // a list that did not hold them all is none
#pragma unroll
    for (int m = 1; m < kMaxChunks; m <<= 1) {
      const uint32_t o = __shfl_up(n, m, kWave);
      if (lane >= m) n += o;
    }
    if (lane < kMaxChunks) s.ends[i][lane] = n;
  }
  const Row w = row_of(a, r);
  if (w.none) {  // nothing to choose
    if (tid == 0) a.out[r] = -1;
    return;
  }
  const Settings set = settings_of(a, w, r);
  __syncthreads();
  // Key `at` of border i's lists, the chunks' one after the other.
  auto key_at = [&](int i, uint32_t at) {
    int c = 0;
#pragma unroll
    for (int m = kMaxChunks / 2; m >= 1; m >>= 1)
      if (s.ends[i][c + m - 1] <= at) c += m;
    const uint32_t before = c ? s.ends[i][c - 1] : 0;
    return a.lists[((row_at + c) * kBorders + i) * kListed + at - before];
  };
  // All borders' lists that fit the block's memory at once.
  constexpr int kEach = kListed / kThreads;
  uint64_t key[kBorders][kEach];
  auto kept_here = [&](int i) { return s.ends[i][kMaxChunks - 1] <= kListed ? s.ends[i][kMaxChunks - 1] : 0; };
#pragma unroll
  for (int i = 0; i < kBorders; ++i)
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (tid + j * kThreads < kept_here(i)) key[i][j] = key_at(i, tid + j * kThreads);
#pragma unroll
  for (int i = 0; i < kBorders; ++i)
#pragma unroll
    for (int j = 0; j < kEach; ++j)
      if (tid + j * kThreads < kept_here(i)) s.keys[i][tid + j * kThreads] = key[i][j];
  uint64_t kept = plan.all;
  Found f{};
#pragma unroll 1
  for (int i = 0; i < kBorders; ++i) {
    if (i == 0 && !plan.by_count) continue;
    if (i == 1 && !(plan.by_weight && cuts(set, kept))) continue;
    const Border b = i == 0 ? Border{kCount, static_cast<uint64_t>(set.top_k), 0.0}
                            : (i == 1 ? border_p(set, kept) : border_u(set, least(kept, plan.floor_p)));
    find_border(s.ranks, b, c0, w0, c1, w1, all_c);
    Place p{s.ranks.at, s.ranks.here, s.ranks.count_before, s.ranks.weight_before, 0};
    const uint32_t listed = s.ends[i][kMaxChunks - 1];
    // g(key, logit) for the listed tokens of the border's bin.
    auto each_listed = [&](auto&& g) {
      auto one = [&](uint64_t k) {
        const float x = key_logit(k);
        if (bin_of(w, x) == p.bin) g(k, x);
      };
      if (listed <= kListed) {
#pragma unroll 1
        for (int j = 0; j < kEach; ++j)
          if (tid + j * kThreads < listed) one(s.keys[i][tid + j * kThreads]);
        return;
      }
      for (uint32_t at = tid; at < listed; at += 2 * kThreads) {
        uint64_t k[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) k[u] = key_at(i, at + u * kThreads < listed ? at + u * kThreads : at);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          if (at + u * kThreads < listed) one(k[u]);
      }
    };
    // The token's place among 1024 finer bins of the bin.
    auto fine_of = [&](float x) {
      const double g = past_edge(w, x, p.bin) * kThreads;
      return g > 0.0 ? (g < kThreads - 1 ? static_cast<int>(g) : kThreads - 1) : 0;
    };
    bool whole = listed > 0;
    int only = -1;
    if (whole && p.here > kWave) {
      s.fine_count[tid] = 0;
      s.fine_weight[tid] = 0;
      __syncthreads();
      each_listed([&](uint64_t k, float x) {
        const int d = fine_of(x);
        atomicAdd(&s.fine_count[d], 1u);
        atomicAdd(&s.fine_weight[d], static_cast<unsigned long long>(key_weight(w, k, p.bin)));
      });
      __syncthreads();
      Place q = p;
      narrow(s.ranks, q, b, s.fine_count[tid], s.fine_weight[tid]);
      only = s.ranks.at;
      whole = q.here <= kThreads;
      if (whole) p = q;
    }
    if (whole) {
      if (tid == 0) s.taken = 0;
      __syncthreads();
      each_listed([&](uint64_t k, float x) {
        if (only < 0 || fine_of(x) == only) s.near[atomicAdd(&s.taken, 1u)] = k;
      });
    } else {
      by_digits(s, w, p, b, [&](auto&& g) {
        if (listed) {
          each_listed([&](uint64_t k, float) { g(k); });
          return;
        }
        each_logit<L, 1>(static_cast<const L*>(a.logits) + r * a.row_st, 0, a.vocab, [&](float x, long id) {
          x = seen_logit(w, x);
          if (bin_of(w, x) == p.bin) g(order_key(x, id));
        });
      });
    }
    f = p.here <= kWave ? among_few(s, w, s.near, p, b) : among(s, w, s.near, p, b);
    kept = i < 2 ? least(kept, f.weight) : kept;
  }
  if (tid == 0) a.out[r] = f.id;
}

struct Layout {
  int chunks;
  long chunk, bins, edges, plans, counts, weights, listed, lists, bytes;
};

Layout layout_of(long rows, long vocab) {
  Layout l;
  // Two blocks a CU where the chunks stay at 2048 tokens or more, 16 a row at most
  // (8: one row 28.8 us instead of 27.2).
  long c = 512 / rows;
  const long most = (vocab + 2047) / 2048, fewest = (vocab + kChunk - 1) / kChunk;
  c = c < most ? c : most;
  c = c < kMaxChunks ? c : kMaxChunks;
  c = c > fewest ? c : fewest;
  l.chunk = (vocab + c - 1) / c;
  l.chunks = static_cast<int>((vocab + l.chunk - 1) / l.chunk);
  const long n = rows * l.chunks;
  l.bytes = 0;
  auto place = [&](long bytes) {
    const long at = l.bytes;
    l.bytes += (bytes + 255) / 256 * 256;
    return at;
  };
  place(n * 4);  // maxima
  l.bins = place(n * kBins * 8);
  l.edges = place(n * 3 * 8);
  l.plans = place(rows * static_cast<long>(sizeof(RowPlan)));
  l.counts = place(rows * kBins * 4);
  l.weights = place(rows * kBins * 8);
  l.listed = place(n * kBorders * 4);
  l.lists = place(n * kBorders * kListed * 8);
  return l;
}

template <typename L>
int sample(const SampleArgs& a, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.rows));
  hipLaunchKernelGGL(sample_max<L>, grid, dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(sample_histogram<L>, grid, dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(sample_plan, dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(sample_collect<L>, grid, dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(sample_pick<L>, dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0, st, a);
  return launch_status();
}

constexpr long kMaxRows = 65535, kMaxVocab = kMaxChunks * kChunk;  // weights sum to less than 2^64

}  // namespace
}  // namespace htn

using namespace htn;

extern "C" int64_t htn_sample_scratch_bytes(int64_t rows, int64_t vocab) {
  if (rows <= 0 || vocab <= 0 || rows > kMaxRows || vocab > kMaxVocab) return 0;
  return layout_of(rows, vocab).bytes;
}

extern "C" int htn_sample(const void* logits, int64_t row_st, int fp32, int64_t rows, int64_t vocab,
                          const float* uniform, const float* temperature, float temperature_all,
                          const int64_t* top_k, int64_t top_k_all, const float* top_p, float top_p_all,
                          const float* min_p, float min_p_all, int64_t* out, void* scratch,
                          int64_t scratch_bytes, htn_stream_t stream) {
  if (!logits || !uniform || !out || !scratch || rows <= 0 || vocab <= 0 || (rows > 1 && row_st < vocab))
    return HTN_EINVAL;
  if (rows > kMaxRows || vocab > kMaxVocab || (reinterpret_cast<uintptr_t>(logits) & (fp32 ? 3u : 1u)) ||
      !aligned16(scratch))
    return HTN_EUNSUPPORTED;
  const Layout l = layout_of(rows, vocab);
  if (scratch_bytes < l.bytes) return HTN_EINVAL;
  char* p = static_cast<char*>(scratch);
  SampleArgs a{};
  a.logits = logits; a.row_st = row_st; a.vocab = vocab;
  a.rows = static_cast<int>(rows); a.chunks = l.chunks; a.chunk = l.chunk;
  a.uniform = uniform;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p;
  a.temperature_all = temperature_all; a.top_k_all = top_k_all; a.top_p_all = top_p_all; a.min_p_all = min_p_all;
  a.out = out;
  a.maxima = reinterpret_cast<float*>(p);
  a.bins = reinterpret_cast<uint64_t*>(p + l.bins);
  a.edges = reinterpret_cast<uint64_t*>(p + l.edges);
  a.plans = reinterpret_cast<RowPlan*>(p + l.plans);
  a.counts = reinterpret_cast<uint32_t*>(p + l.counts);
  a.weights = reinterpret_cast<uint64_t*>(p + l.weights);
  a.listed = reinterpret_cast<uint32_t*>(p + l.listed);
  a.lists = reinterpret_cast<uint64_t*>(p + l.lists);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return fp32 ? sample<float>(a, st) : sample<bf16_t>(a, st);
}
