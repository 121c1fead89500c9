// Token sampling for gfx950: temperature, top-k, top-p, min-p and one uniform
// number per row, without sorting the vocabulary.
//
// The order of a row is falling logit, the lower id first among equals. Every
// truncation keeps a leading part of it, so a row's answer is a place in that
// order: the first token whose cumulative weight passes u times the weight kept.
// A token's weight is exp((x - max) / T), held in 64-bit fixed point (2^44 for the
// largest token): sums of integers are exact, so they do not depend on the order
// in which blocks and atomics take them, and a border between two tokens falls
// where 64-bit sums put it. Tokens 32 nats and more below the largest weigh
// nothing (below half a unit).
//
//   1. every chunk of a row: its largest logit;
//   2. every chunk: a histogram over 1024 bins of 1/32 nat below the row's
//      largest, with the tokens' count and weight in each bin;
//   3. one block a row: the bins' running sums give the bin in which a border
//      lies; the bin's tokens, read again from the chunks that have any, are
//      ranked and the border found among them. Bins of more than 1024 tokens
//      are first narrowed by eight bits of (logit, id) at a time.
#include "common.h"

namespace htn {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 1024;
constexpr int kRanked = 1024;  // tokens ranked at once
constexpr int kMaxChunks = 16;
constexpr double kOne = 17592186044416.0;  // 2^44

struct SampleArgs {
  const void* logits; long row_st;
  long vocab; int rows, chunks; long chunk;
  const float* uniform;
  const float* temperature; const int64_t* top_k; const float* top_p; const float* min_p;  // or null:
  float temperature_all; int64_t top_k_all; float top_p_all, min_p_all;                    // for all rows
  int64_t* out;
  float* maxima;         // [rows, chunks]
  uint32_t* counts;      // [rows, chunks, kBins]
  uint64_t* weights;     // [rows, chunks, kBins]
  uint64_t* above_min;   // [rows, chunks]: weight of the tokens that min-p keeps
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

// The largest logit of a chunk; NaN counts as masked.
template <typename L>
__global__ __launch_bounds__(kThreads) void sample_max(SampleArgs a) {
  __shared__ float red[kWaves];
  const int r = blockIdx.y, c = blockIdx.x;
  const L* row = static_cast<const L*>(a.logits) + r * a.row_st;
  const long first = c * a.chunk, last = first + a.chunk < a.vocab ? first + a.chunk : a.vocab;
  float m = -INFINITY;
  each_logit<L, 4>(row, first, last, [&](float x, long) { m = fmaxf(m, x); });
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, red[w]);
    a.maxima[r * a.chunks + c] = m;
  }
}

struct Row {
  float top;     // its largest logit
  double heat;   // 1 / T
  bool greedy;
};

__device__ __forceinline__ Row row_of(const SampleArgs& a, int r) {
  Row w;
  w.top = -INFINITY;
  for (int c = 0; c < a.chunks; ++c) w.top = fmaxf(w.top, a.maxima[r * a.chunks + c]);
  const float t = a.temperature ? a.temperature[r] : a.temperature_all;
  w.greedy = !(t > 0.f);
  w.heat = w.greedy ? 1.0 : 1.0 / static_cast<double>(t);
  return w;
}

// Nats below the largest, in bins; kBins and more: the token weighs nothing. A
// masked logit (-inf, NaN) gives a NaN or an infinity.
__device__ __forceinline__ double bins_below(const Row& w, float x) {
  if (x == w.top) return 0.0;
  return (static_cast<double>(w.top) - static_cast<double>(x)) * w.heat * (kBins / 32.0);
}

// 2^44 exp(-y / 32) for y bins: the table's 2^44 exp(-b / 32) of its whole part
// times the Taylor sum of the rest (below 1/32: the eighth term is 2e-17), as an
// integer by the shift of adding 2^52.
__device__ __forceinline__ uint64_t weight_of(const double* table, double y, int b) {
  const double f = (b - y) * (1.0 / 32.0);
  double s = fma(f, 1.0 / 5040, 1.0 / 720);
  s = fma(f, s, 1.0 / 120);
  s = fma(f, s, 1.0 / 24);
  s = fma(f, s, 1.0 / 6);
  s = fma(f, s, 0.5);
  s = fma(f, s, 1.0);
  s = fma(f, s, 1.0);
  return __double_as_longlong(fma(table[b], s, 4503599627370496.0)) & 0xfffffffffffffULL;
}

__device__ __forceinline__ void fill_table(double* table) {
  table[threadIdx.x] = kOne * exp(-static_cast<double>(threadIdx.x) / 32.0);
}

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, kWave);
  return v;
}

template <typename L>
__global__ __launch_bounds__(kThreads) void sample_histogram(SampleArgs a) {
  __shared__ double table[kBins];
  __shared__ uint32_t counts[kBins];
  __shared__ unsigned long long weights[kBins];
  __shared__ uint64_t red[kWaves];
  const int tid = threadIdx.x, r = blockIdx.y, c = blockIdx.x;
  const Row w = row_of(a, r);
  counts[tid] = 0;
  weights[tid] = 0;
  fill_table(table);
  __syncthreads();
  const L* row = static_cast<const L*>(a.logits) + r * a.row_st;
  const long first = c * a.chunk, last = first + a.chunk < a.vocab ? first + a.chunk : a.vocab;
  const float min_p = a.min_p ? a.min_p[r] : a.min_p_all;
  const double least = static_cast<double>(min_p) * kOne;
  uint64_t above = 0;
  each_logit<L, 2>(row, first, last, [&](float x, long) {
    const double y = bins_below(w, x);
    if (!(y < kBins)) return;
    const int b = static_cast<int>(y);
    const uint64_t v = weight_of(table, y, b);
    atomicAdd(&counts[b], 1u);
    atomicAdd(&weights[b], static_cast<unsigned long long>(v));
    above += static_cast<double>(v) >= least ? v : 0;
  });
  above = wave_sum_u64(above);
  if ((tid & 63) == 0) red[tid >> 6] = above;
  __syncthreads();
  const long at = static_cast<long>(r) * a.chunks + c;
  a.counts[at * kBins + tid] = counts[tid];
  a.weights[at * kBins + tid] = weights[tid];
  if (tid == 0) {
    for (int v = 1; v < kWaves; ++v) above += red[v];
    a.above_min[at] = above;
  }
}

// Where a border lies: by count (the first `target` tokens), by weight before the
// token (below `goal`), or by weight up to it (past `goal`).
enum Border { kCount, kBefore, kPast };

struct Ranks {
  uint32_t wave_count[kWaves];
  uint64_t wave_weight[kWaves];
  int at;
  uint32_t count_before, here;
  uint64_t weight_before;
};

// The first of the block's 1024 entries (in thread order, each with the count and
// weight it holds) that reaches the border: `at`, with the sums before it.
__device__ __forceinline__ void find_border(Ranks& s, uint32_t count, uint64_t weight, uint32_t count_base,
                                            uint64_t weight_base, Border kind, uint64_t target, double goal) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  uint32_t cs = count;
  uint64_t ws = weight;
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const uint32_t co = __shfl_up(cs, m, kWave);
    const uint64_t wo = __shfl_up(ws, m, kWave);
    if (lane >= m) {
      cs += co;
      ws += wo;
    }
  }
  __syncthreads();
  if (lane == 63) {
    s.wave_count[wave] = cs;
    s.wave_weight[wave] = ws;
  }
  __syncthreads();
  uint32_t cb = count_base;
  uint64_t wb = weight_base;
  for (int v = 0; v < wave; ++v) {
    cb += s.wave_count[v];
    wb += s.wave_weight[v];
  }
  const uint32_t c1 = cb + cs, c0 = c1 - count;
  const uint64_t w1 = wb + ws, w0 = w1 - weight;
  auto reached = [&](uint32_t c, uint64_t w) {
    if (kind == kCount) return static_cast<uint64_t>(c) >= target;
    if (kind == kBefore) return static_cast<double>(w) >= goal;
    return static_cast<double>(w) > goal;
  };
  // Sums only grow, and the sums before the first entry are short of the border:
  // one entry at most is the first to reach it.
  if (!reached(c0, w0) && reached(c1, w1)) {
    s.at = tid;
    s.count_before = c0;
    s.weight_before = w0;
    s.here = count;
  }
  __syncthreads();
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

struct Shared {
  double table[kBins];
  Ranks ranks;
  uint64_t keys[kRanked], sorted[kRanked];
  uint32_t digit_count[256];
  unsigned long long digit_weight[256];
  uint32_t chunk_has[kMaxChunks];
  uint32_t taken;
};

struct Found {
  uint64_t weight;  // of the tokens up to the border
  uint32_t id;      // kPast: the token there
};

// The border among a row's tokens; its bins' counts and weights are this
// thread's `count` and `weight`. The weight returned is that of the tokens that
// lie before the border.
template <typename L>
__device__ Found resolve(const SampleArgs& a, Shared& s, const Row& w, int r, uint32_t count, uint64_t weight,
                         Border kind, uint64_t target, double goal) {
  const int tid = threadIdx.x;
  const L* row = static_cast<const L*>(a.logits) + r * a.row_st;
  find_border(s.ranks, count, weight, 0, 0, kind, target, goal);
  const int bin = s.ranks.at;
  uint32_t count_before = s.ranks.count_before, here = s.ranks.here;
  uint64_t weight_before = s.ranks.weight_before;
  if (tid < a.chunks) s.chunk_has[tid] = a.counts[(static_cast<long>(r) * a.chunks + tid) * kBins + bin];
  __syncthreads();
  // f(key, weight) for the bin's tokens whose key agrees with `prefix` above `bits`.
  auto each_token = [&](uint64_t prefix, int bits, auto&& f) {
    for (int c = 0; c < a.chunks; ++c) {
      if (!s.chunk_has[c]) continue;
      const long first = c * a.chunk, last = first + a.chunk < a.vocab ? first + a.chunk : a.vocab;
      each_logit<L, 2>(row, first, last, [&](float x, long id) {
        const double y = bins_below(w, x);
        if (!(y < kBins) || static_cast<int>(y) != bin) return;
        const uint64_t key = order_key(x, id);
        if (bits < 64 && (key ^ prefix) >> bits) return;
        f(key, weight_of(s.table, y, bin));
      });
    }
  };
  uint64_t prefix = 0;
  int bits = 64;
  while (here > kRanked) {  // keys differ, so eight digits at most
    if (tid < 256) {
      s.digit_count[tid] = 0;
      s.digit_weight[tid] = 0;
    }
    __syncthreads();
    each_token(prefix, bits, [&](uint64_t key, uint64_t v) {
      const int d = 255 - static_cast<int>((key >> (bits - 8)) & 255);  // larger keys first
      atomicAdd(&s.digit_count[d], 1u);
      atomicAdd(&s.digit_weight[d], static_cast<unsigned long long>(v));
    });
    __syncthreads();
    find_border(s.ranks, tid < 256 ? s.digit_count[tid] : 0, tid < 256 ? s.digit_weight[tid] : 0, count_before,
                weight_before, kind, target, goal);
    bits -= 8;
    prefix = (prefix & (bits < 56 ? ~0ULL << (bits + 8) : 0ULL)) |
             (static_cast<uint64_t>(255 - s.ranks.at) << bits);
    count_before = s.ranks.count_before;
    weight_before = s.ranks.weight_before;
    here = s.ranks.here;
  }
  if (tid == 0) s.taken = 0;
  __syncthreads();
  each_token(prefix, bits, [&](uint64_t key, uint64_t) {
    const uint32_t i = atomicAdd(&s.taken, 1u);
    if (i < kRanked) s.keys[i] = key;
  });
  __syncthreads();
  if (tid < static_cast<int>(here)) {
    const uint64_t key = s.keys[tid];
    uint32_t rank = 0;
    for (uint32_t i = 0; i < here; ++i) rank += s.keys[i] > key;
    s.sorted[rank] = key;
  }
  __syncthreads();
  uint64_t mine = 0;
  if (tid < static_cast<int>(here)) {
    const double y = bins_below(w, key_logit(s.sorted[tid]));
    mine = weight_of(s.table, y, bin);
  }
  find_border(s.ranks, tid < static_cast<int>(here) ? 1u : 0u, mine, count_before, weight_before, kind, target,
              goal);
  Found f;
  // By count or by weight before: the token that reaches the border is the last kept.
  const int at = s.ranks.at;
  const uint64_t last = s.sorted[at];
  f.id = 0xffffffffu - static_cast<uint32_t>(last & 0xffffffffu);
  f.weight = s.ranks.weight_before + weight_of(s.table, bins_below(w, key_logit(last)), bin);
  __syncthreads();
  return f;
}

template <typename L>
__global__ __launch_bounds__(kThreads) void sample_pick(SampleArgs a) {
  __shared__ Shared s;
  const int tid = threadIdx.x, r = blockIdx.x;
  const Row w = row_of(a, r);
  if (w.top == -INFINITY) {  // nothing to choose
    if (tid == 0) a.out[r] = -1;
    return;
  }
  fill_table(s.table);
  uint32_t count = 0;
  uint64_t weight = 0, above = 0;
  for (int c = 0; c < a.chunks; ++c) {
    const long at = static_cast<long>(r) * a.chunks + c;
    count += a.counts[at * kBins + tid];
    weight += a.weights[at * kBins + tid];
    above += a.above_min[at];
  }
  // The row's totals, the same in every thread.
  uint64_t all_w = wave_sum_u64(weight), all_c = wave_sum_u64(count);
  if ((tid & 63) == 0) {
    s.keys[tid >> 6] = all_w;
    s.keys[kWaves + (tid >> 6)] = all_c;
  }
  __syncthreads();
  all_w = all_c = 0;
  for (int v = 0; v < kWaves; ++v) {
    all_w += s.keys[v];
    all_c += s.keys[kWaves + v];
  }
  __syncthreads();
  double goal = 0.0;
  if (!w.greedy) {
    const int64_t top_k = a.top_k ? a.top_k[r] : a.top_k_all;
    const float top_p = a.top_p ? a.top_p[r] : a.top_p_all, min_p = a.min_p ? a.min_p[r] : a.min_p_all;
    uint64_t kept = all_w;
    if (top_k > 0 && static_cast<uint64_t>(top_k) < all_c)
      kept = resolve<L>(a, s, w, r, count, weight, kCount, top_k, 0.0).weight;
    const double part = static_cast<double>(top_p) * static_cast<double>(kept);
    if (part < static_cast<double>(kept)) {
      const uint64_t p = resolve<L>(a, s, w, r, count, weight, kBefore, 0, part > 0.0 ? part : 0.5).weight;
      kept = p < kept ? p : kept;
    }
    if (min_p > 0.f) {
      const uint64_t first = static_cast<uint64_t>(kOne);
      const uint64_t m = above > first ? above : first;
      kept = m < kept ? m : kept;
    }
    const float u = a.uniform[r];
    goal = u > 0.f ? static_cast<double>(u < 0.99999994f ? u : 0.99999994f) * static_cast<double>(kept) : 0.0;
  }
  const Found f = resolve<L>(a, s, w, r, count, weight, w.greedy ? kCount : kPast, 1, goal);
  if (tid == 0) a.out[r] = f.id;
}

struct Layout {
  int chunks;
  long chunk, counts, weights, above, bytes;
};

Layout layout_of(long rows, long vocab) {
  Layout l;
  long c = 512 / rows;
  const long most = (vocab + 2047) / 2048;
  c = c < most ? c : most;
  c = c < 1 ? 1 : (c > kMaxChunks ? kMaxChunks : c);
  l.chunk = (vocab + c - 1) / c;
  l.chunks = static_cast<int>((vocab + l.chunk - 1) / l.chunk);
  const long n = rows * l.chunks;
  l.weights = (n * 4 + 255) / 256 * 256;
  l.above = l.weights + n * kBins * 8;
  l.counts = l.above + n * 8;
  l.bytes = l.counts + n * kBins * 4;
  return l;
}

template <typename L>
int sample(const SampleArgs& a, hipStream_t st) {
  const dim3 grid(static_cast<unsigned>(a.chunks), static_cast<unsigned>(a.rows));
  hipLaunchKernelGGL(sample_max<L>, grid, dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(sample_histogram<L>, grid, dim3(kThreads), 0, st, a);
  hipLaunchKernelGGL(sample_pick<L>, dim3(static_cast<unsigned>(a.rows)), dim3(kThreads), 0, st, a);
  return launch_status();
}

constexpr long kMaxRows = 65535, kMaxVocab = 1L << 19;  // weights sum to at most 2^63

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
  a.weights = reinterpret_cast<uint64_t*>(p + l.weights);
  a.above_min = reinterpret_cast<uint64_t*>(p + l.above);
  a.counts = reinterpret_cast<uint32_t*>(p + l.counts);
  hipStream_t st = static_cast<hipStream_t>(stream);
  return fp32 ? sample<float>(a, st) : sample<bf16_t>(a, st);
}
