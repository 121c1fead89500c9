// Paged K/V cache for gfx950 (head_dim 128): the append of new keys and
// values, and the attention of a ragged batch over the pages.
//
//   pools   keys, values [pages, Hkv, page, 128] bf16; slot s of sequence b is
//           row s % page of page table[b, s / page]
//   batch   sequence b's new tokens are rows starts[b] .. starts[b + 1] - 1 of
//           the packed inputs, its last one at position lengths[b] - 1
//
// starts, lengths, tables and the prefix length are read on the device, so a
// captured call replays with other sequences; nothing they hold can make a
// kernel leave its buffers: starts that fall or leave the batch give no work at
// all, a sequence whose length does not fit its table sees nothing, and a page
// id outside the pool reads as zeros and is not written.
#include "attention.h"

namespace htn {

namespace {

typedef const __attribute__((address_space(4))) int32_t* const_i32_t;

// Wave-uniform read of an array that earlier launches wrote: a scalar load, which
// does not count among the vector loads that the tile loops wait for.
__device__ __forceinline__ int32_t scalar_i32(const int32_t* p, long i) {
  return ((const_i32_t)(uintptr_t)p)[i];
}
// Rows t0 .. t0 + n - 1 of a sequence, the first at position p0. A length that
// does not fit the table puts every row before slot 0.
struct Span {
  int t0, n, p0;
};

__device__ __forceinline__ Span make_span(int64_t s0, int64_t s1, int64_t length, long tokens,
                                          long cap) {
  Span s;
  const bool ok = s0 >= 0 && s1 >= s0 && s1 <= tokens;
  s.t0 = ok ? static_cast<int>(s0) : 0;
  s.n = ok ? static_cast<int>(s1 - s0) : 0;
  s.p0 = length >= 0 && length <= cap ? static_cast<int>(length) - s.n : -s.n;
  return s;
}

// The sequence of row t: the first whose end lies past it. All lanes of the
// wave call it with one t. `batch` if there is none.
__device__ __forceinline__ int sequence_of(const int64_t* starts, int batch, long t, int lane) {
  int before = 0;
  for (int j0 = 0; j0 < batch; j0 += kWave) {
    const int j = j0 + lane;
    before += __popcll(__ballot(j < batch && starts[j < batch ? j + 1 : 0] <= t));
  }
  return before;
}

// ------------------------------------------------------------------ append

struct AppendArgs {
  const bf16_t* q; const bf16_t* k; const bf16_t* v; long q_st, k_st, v_st;
  const bf16_t* qg; const bf16_t* kg; float q_eps, k_eps;
  const void* cos; const void* sin; long rope_st, rope_rows;
  bf16_t* keys; bf16_t* values; long pages; int page_shift;
  const int32_t* table; long table_st; long table_pages;
  const int64_t* starts; const int64_t* lengths;
  bf16_t* out_q;
  int B, T, Hq, Hkv;
};

// x of the lane 8 further round the 16-lane row: the other half of the head.
__device__ __forceinline__ float half_partner(float x) { return dpp<0x128>(x); }

template <typename R>
__device__ __forceinline__ void load_rope8(const R* p, float* o) {
  if constexpr (sizeof(R) == 2) {
    unpack8(*reinterpret_cast<const uint4*>(p), o);
  } else {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    o[0] = a.x; o[1] = a.y; o[2] = a.z; o[3] = a.w;
    o[4] = b.x; o[5] = b.y; o[6] = b.z; o[7] = b.w;
  }
}

// One new token's heads, q then k then v, 16 lanes each (lane e holds elements
// 8 e .. 8 e + 7, its rotation partners sit 8 lanes further):
//   n = x g / sqrt(mean(x^2) + eps),  out = n cos + rot(n) sin,
// in fp32 throughout and rounded once, where norm_rope_cache rounds after each
// of the reference's steps. Everything is read and written once, 16 bytes a lane:
// with 32 + 8 heads, 3133 tokens of seven prompts (80 MB) take 18.2 us, 4.4 TB/s
// where a large copy reaches 4.9; 16 single tokens 3.0 us, a launch's time.
template <typename R>
__global__ __launch_bounds__(kBlock) void norm_rope_paged_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63, e = lane & 15;
  const int t = blockIdx.x;
  const int j = sequence_of(a.starts, a.B, t, lane);
  if (j >= a.B) return;
  const Span s = make_span(a.starts[j], a.starts[j + 1], a.lengths[j], a.T, a.table_pages << a.page_shift);
  const int i = t - s.t0;
  if (i < 0 || i >= s.n) return;
  const int pos = s.p0 + i;
  const bool placed = pos >= 0;
  int id = placed ? a.table[j * a.table_st + (pos >> a.page_shift)] : -1;
  const bool stored = id >= 0 && id < a.pages;
  const bool turned = placed && pos < a.rope_rows;  // a row past the tables turns to zeros
  float c[8], sn[8];
  const long rr = turned ? pos : 0;
  load_rope8(static_cast<const R*>(a.cos) + rr * a.rope_st + 8 * e, c);
  load_rope8(static_cast<const R*>(a.sin) + rr * a.rope_st + 8 * e, sn);
#pragma unroll
  for (int d = 0; d < 8; ++d) {
    c[d] = turned ? c[d] : 0.f;
    // rot(n) is -n of the second half in the first, n of the first in the second.
    sn[d] = turned ? (e < 8 ? -sn[d] : sn[d]) : 0.f;
  }
  const int heads = a.Hq + 2 * a.Hkv;
  const long slot = (static_cast<long>(stored ? id : 0) * a.Hkv << a.page_shift) +
                    (pos & ((1 << a.page_shift) - 1));
  // Whole 16-lane rows pass the loop, so the cross-lane steps are whole too.
  for (int h = blockIdx.y * 16 + (threadIdx.x >> 4); h < heads; h += gridDim.y * 16) {
    const bool is_q = h < a.Hq, is_v = h >= a.Hq + a.Hkv;
    const int hk = is_q ? 0 : (is_v ? h - a.Hq - a.Hkv : h - a.Hq);
    const bf16_t* src = is_q ? a.q + t * a.q_st + static_cast<long>(h) * D
                             : (is_v ? a.v + t * a.v_st : a.k + t * a.k_st) + static_cast<long>(hk) * D;
    const uint4 xv = *reinterpret_cast<const uint4*>(src + 8 * e);
    bf16_t* dst = is_q ? a.out_q + (static_cast<long>(t) * a.Hq + h) * D
                       : (is_v ? a.values : a.keys) + (slot + (static_cast<long>(hk) << a.page_shift)) * D;
    uint4 ov = xv;
    if (!is_v) {
      float x[8];
      unpack8(xv, x);
      const bf16_t* g = is_q ? a.qg : a.kg;
      if (g) {
        float ss = 0.f, gain[8];
#pragma unroll
        for (int d = 0; d < 8; ++d) ss = fmaf(x[d], x[d], ss);
        ss = row16_sum(ss);
        const float inv = 1.0f / sqrtf(ss / static_cast<float>(D) + (is_q ? a.q_eps : a.k_eps));
        unpack8(*reinterpret_cast<const uint4*>(g + 8 * e), gain);
#pragma unroll
        for (int d = 0; d < 8; ++d) x[d] *= inv * gain[d];
      }
      float o[8];
#pragma unroll
      for (int d = 0; d < 8; ++d) o[d] = fmaf(half_partner(x[d]), sn[d], x[d] * c[d]);
      ov = make_uint4(pack_bf2(o[0], o[1]), pack_bf2(o[2], o[3]), pack_bf2(o[4], o[5]), pack_bf2(o[6], o[7]));
    }
    if (is_q || stored) *reinterpret_cast<uint4*>(dst + 8 * e) = ov;
  }
}

// ------------------------------------------------------------------ attention

constexpr int kFewRows = 32;               // query rows of a block whose waves split the slots, at most
constexpr int kManyRows = 128;             // and of one whose waves split the rows
constexpr int kGroupBytes = 16 * D * 2;    // K or V of 16 slots
constexpr int kTileBytes = 2 * kSplit * D * 2;
constexpr int kRing = 2;                   // staged 64-slot tiles

struct PlanEntry {
  int part;     // first row of the sequence's partials
  int chunks;   // parts that each row's slots are split in; 0: its blocks finish their rows
  int stride;   // rows that a block's partials take
  int split;    // (first entry) whether any sequence is split
};

struct PagedArgs {
  const bf16_t* q; long q_st, q_sh;
  const bf16_t* keys; const bf16_t* values; long pages; int page_shift;
  const int32_t* table; long table_st; long table_pages;
  const int64_t* starts; const int64_t* lengths;
  const int32_t* prefix_pages; long prefix_count; const int64_t* prefix_length;  // shared prefix, or null
  bf16_t* out; long o_st, o_sh;
  PlanEntry* plan; float2* ml; float* part;
  int B, T, Hq, Hkv, G;
  int window, sinks;  // window 0: none
  float scale2;       // log2(e) / sqrt(128)
};

// Slots of a block's rows: tiles [0, sink_tiles) and from first_tile on,
// `tiles` in all, slots from lo0 and below hi.
struct Slots {
  int lo0, hi, sink_tiles, first_tile, tiles;
};

__device__ __forceinline__ Slots slots_of(int p_first, int p_last, int lo0, int window, int sinks) {
  Slots s;
  s.lo0 = lo0;
  s.hi = p_last + 1;
  s.sink_tiles = 0;
  s.first_tile = lo0 / kSplit;
  if (window) {
    const int start = p_first + 1 - window;
    const int ns = ((sinks < s.hi ? sinks : s.hi) + kSplit - 1) / kSplit;
    if (start > 0 && start / kSplit > ns) {
      s.sink_tiles = ns;
      s.first_tile = start / kSplit;
    }
  }
  const int last_tile = (s.hi + kSplit - 1) / kSplit;
  s.tiles = s.hi > lo0 ? s.sink_tiles + (last_tile > s.first_tile ? last_tile - s.first_tile : 0) : 0;
  return s;
}

struct SeqWork {
  Span span;
  int rows, tile_rows, row_tiles, max_tiles;
};

// The slots of the shared prefix: of its whole pages. A page that the prefix ends in
// holds each sequence's own slots behind it, so it is a page of the sequence's, as
// its table has it.
__device__ __forceinline__ int prefix_slots(const PagedArgs& a) {
  if (!a.prefix_length) return 0;
  const int64_t p = a.prefix_length[0], cap = a.prefix_count << a.page_shift;
  const int within = static_cast<int>(p < 0 ? 0 : (p > cap ? cap : p));
  return within >> a.page_shift << a.page_shift;
}

// Sequence s of the plan: with a shared prefix, 0 is the prefix under all rows
// and sequence j is s = j + 1. `bad` if the starts around it fall or leave the
// batch.
__device__ __forceinline__ SeqWork seq_work(const PagedArgs& a, int s, int prefix, bool& bad) {
  SeqWork w;
  const bool shared = a.prefix_length != nullptr;
  const int j = shared ? s - 1 : s;
  Slots all;
  if (j < 0) {
    const int64_t end = a.starts[a.B];
    bad |= end < 0 || end > a.T;
    w.span = Span{0, bad ? 0 : static_cast<int>(end), 0};
    all = slots_of(0, prefix - 1, 0, 0, 0);
  } else {
    const int64_t s0 = a.starts[j], s1 = a.starts[j + 1];
    bad |= s0 < 0 || s1 < s0 || s1 > a.T;
    w.span = make_span(s0, s1, a.lengths[j], a.T, a.table_pages << a.page_shift);
    all = slots_of(0, w.span.p0 + w.span.n - 1, prefix, 0, 0);
  }
  w.rows = w.span.n * a.G;
  w.tile_rows = w.rows <= kFewRows ? kFewRows : kManyRows;
  w.row_tiles = (w.rows + w.tile_rows - 1) / w.tile_rows;
  w.max_tiles = all.tiles;
  if (a.window) {
    // At most: the sinks, the window of the tile's first row, its further rows.
    const int most = (a.sinks + kSplit - 1) / kSplit +
                     (a.window + w.tile_rows / a.G + 2) / kSplit + 2;
    w.max_tiles = most < w.max_tiles ? most : w.max_tiles;
  }
  return w;
}

// Blocks wanted: two per CU, all at once. With 768, 16 sequences (24 K slots) took
// 28.5 us instead of 25.9, and a 1000-token chunk beside 15 sequences 145 instead
// of 124.
constexpr int kTargetBlocks = 512;

// Tiles that a block takes at least, where a row's slots are split: a split
// writes and merges a partial of its rows (520 bytes each) for K and V of 32 KB
// a tile. With 1 and with 4, 540 slots under 16 heads take 9.9 and 11.3 us (2:
// 10.5), 30 verify rows behind a prefix of 2048 both 19.5 (2: 17.0).
constexpr int kMinTiles = 2;

__device__ __forceinline__ int chunks_of(const SeqWork& w, uint32_t per_block) {
  const uint32_t n = (w.max_tiles + per_block - 1) / per_block;
  return n < 1 ? 1 : static_cast<int>(n);
}

__device__ __forceinline__ int part_stride(const SeqWork& w) {
  return w.rows < kManyRows ? (w.rows + 15) / 16 * 16 : kManyRows;
}

// One block's work.
struct Item {
  int seq;             // sequence, or -1 for the shared prefix
  int t0, n, p0;       // its tokens
  int tile, rows;      // row tile, and the rows in it
  int kvh, chunk, chunks;
  int part;            // first row of the block's partials, or -1: the block finishes its rows
};

// Which rows, K/V head and slots this block takes; false if none. Every wave
// derives the same plan from starts and lengths, a sequence a lane: the tiles of
// all rows over kTargetBlocks give the tiles per block, each sequence's rows are
// cut in equal chunks of at most that many, and blocks are numbered sequence by
// sequence, in each by row tile (the last, longest, first), chunk and K/V head.
//
// A sequence's chunks number below twice its tiles over the tiles per block where
// they are two or more, so all split blocks number below 2 kTargetBlocks, and all
// blocks at most kTargetBlocks plus one per (row tile, K/V head). With 64 sequences or
// fewer the tiles per block are raised until all blocks fit it (they run at once).
__device__ __forceinline__ bool make_plan(const PagedArgs& a, int prefix, Item& it) {
  const int lane = threadIdx.x & 63;
  const bool shared = a.prefix_length != nullptr;
  const int n = a.B + (shared ? 1 : 0);
  uint64_t total = 0;
  int items = 0;
  SeqWork w{};
  bool bad = false;
  for (int s = lane; s < n; s += kWave) {
    w = seq_work(a, s, prefix, bad);
    total += static_cast<uint64_t>(w.row_tiles) * w.max_tiles * a.Hkv;
    items += w.row_tiles * a.Hkv;
  }
  // Starts must rise: the bounds of the blocks and partials count every row once.
  if (__any(bad)) {
    if (blockIdx.x == 0)
      for (int s = threadIdx.x; s < n; s += kBlock) a.plan[s] = PlanEntry{0, 0, 0, 0};
    return false;
  }
  total = wave_last(wave_scan(total));
  items = wave_last(wave_scan(static_cast<uint32_t>(items)));
  uint32_t per_block = static_cast<uint32_t>((total + kTargetBlocks - 1) / kTargetBlocks);
  per_block = per_block > kMinTiles ? per_block : kMinTiles;
  if (n <= kWave && items <= kTargetBlocks)
    for (;; per_block += 1 + per_block / 16) {
      const uint32_t mine = lane < n ? w.row_tiles * chunks_of(w, per_block) * a.Hkv : 0;
      if (wave_last(wave_scan(mine)) <= static_cast<uint32_t>(kTargetBlocks)) break;
    }
  // Blocks (low half) and rows of partials (high half) before each sequence.
  uint64_t base = 0;
  bool found = false;
  for (int s0 = 0; s0 < n; s0 += kWave) {
    const int s = s0 + lane;
    if (n > kWave) w = seq_work(a, s < n ? s : n - 1, prefix, bad);
    const int chunks = s < n ? chunks_of(w, per_block) : 0;
    const int blocks = w.row_tiles * chunks * a.Hkv;
    const bool split = blocks && (shared || chunks > 1);
    const int stride = part_stride(w);
    const uint64_t mine = static_cast<uint64_t>(blocks) |
                          (split ? static_cast<uint64_t>(blocks) * stride << 32 : 0);
    const uint64_t sum = wave_scan(mine);
    const uint64_t first = base + sum - mine;
    base += wave_last(sum);
    const int at = static_cast<int>(blockIdx.x) - static_cast<int>(first & 0xffffffffu);
    const int part = static_cast<int>(first >> 32);
    if (blockIdx.x == 0 && threadIdx.x < kWave && s < n) a.plan[s] = PlanEntry{part, split ? chunks : 0, stride, 0};
    const uint64_t mask = __ballot(at >= 0 && at < blocks);
    if (!mask) continue;
    found = true;
    const int src = __builtin_ctzll(mask);
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, src); };
    it.seq = s0 + src - (shared ? 1 : 0);
    it.t0 = of(w.span.t0);
    it.n = of(w.span.n);
    it.p0 = of(w.span.p0);
    it.chunks = of(chunks);
    const int place = of(at), tile_rows = of(w.tile_rows);
    it.kvh = place % a.Hkv;
    const int rest = place / a.Hkv;
    it.chunk = rest % it.chunks;
    it.tile = of(w.row_tiles) - 1 - rest / it.chunks;
    const int left = of(w.rows) - it.tile * tile_rows;
    it.rows = left < tile_rows ? left : tile_rows;
    it.part = of(split) ? of(part) + ((it.tile * it.chunks + it.chunk) * a.Hkv + it.kvh) * of(stride) : -1;
    if (blockIdx.x) break;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.plan[0].split = base >> 32 ? 1 : 0;
  return found;
}

// The page of the 16-slot group at `slot`, -1 where none of slots lo0 .. hi - 1 is in it.
__device__ __forceinline__ int page_of(const PagedArgs& a, const int32_t* table, int slot, int lo0, int hi) {
  return slot < hi && slot + 16 > lo0 ? scalar_i32(table, slot >> a.page_shift) : -1;
}

// Where a group's K or V rows lie in a pool: an element offset, and the rows that may
// be read (the rest of the group reads as zeros).
struct Group {
  long offset;
  uint32_t bytes;
};

__device__ __forceinline__ Group group_of(const PagedArgs& a, int page, int kvh, int slot, int hi) {
  const bool in_pool = page >= 0 && page < a.pages;
  const int left = hi - slot;
  Group g;
  g.offset = in_pool ? ((((static_cast<long>(page) * a.Hkv + kvh) << a.page_shift) +
                         (slot & ((1 << a.page_shift) - 1))) * D) : 0;
  g.bytes = in_pool ? static_cast<uint32_t>(left < 16 ? left : 16) * (D * 2) : 0u;
  return g;
}

// A staged row's sixteen 16-byte chunks are rotated by two a slot, chunk c of slot
// s at (c + 2 s) % 16, through the loads' source offsets, so that the operand reads
// (one chunk of 16 slots, or four chunks' parts of four) spread over the banks. The
// offsets of slots 8 further are 2048 bytes on.
__device__ __forceinline__ void stage_offsets(int lane, uint32_t (&off)[2]) {
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    const int s = 4 * u + (lane >> 4);
    off[u] = static_cast<uint32_t>(s * 256 + (((lane & 15) - 2 * s) & 15) * 16);
  }
}

// Quarter u of a group's K or V rows, a 1 KB LDS-direct load (whose own offset moves
// both ends).
__device__ __forceinline__ void stage_quarter(__amdgpu_buffer_rsrc_t rows, unsigned char* lds, int u,
                                              const uint32_t (&off)[2]) {
  lds_void_t* to = (lds_void_t*)(lds + (u & 1) * 1024);
  if (u & 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, to, 16, off[u & 1], 0, 2048, 0);
  else __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, to, 16, off[u & 1], 0, 0, 0);
}

// Addresses of the operand reads in a tile whose K rows start at LDS byte k and V
// rows at v (multiples of 256): K chunk 4 ks + quad of slot col, and for the V^T
// transpose reads, of slot r = 4 quad + col / 4, dims 16 j + 4 (col % 4) .. + 3: 8
// bytes of chunk 2 j + (col % 4) / 2. Steps ks + 2 and j + 4 are 8 chunks on: bit
// 7 of the address turned.
struct ReadAddrs {
  uint32_t k[2], v[4];
};

__device__ __forceinline__ ReadAddrs read_addrs(uint32_t k, uint32_t v, int col, int quad) {
  ReadAddrs r;
#pragma unroll
  for (int ks = 0; ks < 2; ++ks)
    r.k[ks] = k + static_cast<uint32_t>(col * 256 + ((4 * ks + quad + 2 * col) & 15) * 16);
  const int s = 4 * quad + (col >> 2);
#pragma unroll
  for (int j = 0; j < 4; ++j)
    r.v[j] = v + static_cast<uint32_t>(s * 256 + ((2 * j + ((col & 3) >> 1) + 2 * s) & 15) * 16 + (col & 1) * 8);
  return r;
}
__device__ __forceinline__ uint32_t k_addr(const ReadAddrs& r, int ks, uint32_t tile) {
  return (r.k[ks & 1] ^ (ks & 2 ? 128u : 0u)) + tile;
}
__device__ __forceinline__ uint32_t v_addr(const ReadAddrs& r, int j, uint32_t tile) {
  return (r.v[j & 3] ^ (j & 4 ? 128u : 0u)) + tile;
}

// What a query row sees: slots vlo .. vhi and those below `sinks`.
struct Sight {
  int vlo, vhi;
};

__device__ __forceinline__ Sight sight_of(int pos, const Slots& s, int window) {
  Sight v;
  v.vhi = pos < s.hi ? pos : s.hi - 1;
  v.vlo = s.lo0;
  if (window && pos + 1 - window > v.vlo) v.vlo = pos + 1 - window;
  return v;
}

__device__ __forceinline__ int min16(int v) {
#pragma unroll
  for (int m = 1; m < 16; m <<= 1) {
    const int o = __shfl_xor(v, m, kWave);
    v = o < v ? o : v;
  }
  return __builtin_amdgcn_readfirstlane(v);
}

// The bf16 pair with an infinity or a NaN as zero, and whether there was one.
__device__ __forceinline__ uint32_t finite_pair(uint32_t w, bool& odd) {
  const bool lo = (w & 0x7f80u) == 0x7f80u, hi = (w & 0x7f800000u) == 0x7f800000u;
  odd |= lo || hi;
  return w & ((lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u));
}

// The infinities and NaN of `slots` rows of V from slot s0 on (staged at `v`, 16
// slots a kGroupBytes), which the products took as zeros, for the rows that see
// their slot, and for no other: a visible slot's weight is positive, so the
// output is infinite or NaN there whatever it weighs.
__device__ __forceinline__ void add_nonfinite(const unsigned char* v, int slots, int s0, const Sight& sight,
                                              int sinks, int quad, f32x4_t (&acc)[8]) {
#pragma unroll 1
  for (int s = 0; s < slots; ++s) {
    const uint32_t seen = s0 + s <= sight.vhi && (s0 + s >= sight.vlo || s0 + s < sinks) ? ~0u : 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int chunk = (2 * j + (quad >> 1) + 2 * (s & 7)) & 15;
      u32x2_t w;
      asm volatile("ds_read_b64 %0, %1\n\ts_waitcnt lgkmcnt(0)"
                   : "=&v"(w)
                   : "v"(static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_t*)v)) +
                         static_cast<uint32_t>(s * 256 + chunk * 16 + (quad & 1) * 8))
                   : "memory");
      bool odd = false;
      w.x = (w.x ^ finite_pair(w.x, odd)) & seen;
      w.y = (w.y ^ finite_pair(w.y, odd)) & seen;
      acc[j] += f32x4_t{bf_lo(w.x), bf_hi(w.x), bf_lo(w.y), bf_hi(w.y)};
    }
  }
}

__device__ __forceinline__ f32x4_t mfma(u32x4 x, u32x4 y, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, x),
                                                 __builtin_bit_cast(bf16x8_t, y), c, 0, 0, 0);
}

// Until at most N of the wave's LDS reads are left, after which these are there.
template <int N>
__device__ __forceinline__ void wait_k4(u32x4 (&k)[4]) {
  asm volatile("s_waitcnt lgkmcnt(%4)" : "+v"(k[0]), "+v"(k[1]), "+v"(k[2]), "+v"(k[3]) : "n"(N) : "memory");
}

// The largest of three; fmaxf first quiets each operand, an instruction of its own.
// The compiler does not see the instruction: scores pass `settle` before.
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}

// quad_max of a value that max3 made.
__device__ __forceinline__ float quad_max3(float v) {
  auto pair = [](auto w) {
    float r;
    asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(__uint_as_float(w[0])), "v"(__uint_as_float(w[1])));
    return r;
  };
  v = pair(__builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
  return pair(__builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
}

// The wait states that a vector instruction must keep from the matrix instruction
// whose result it reads (19 at most), which the compiler does not insert ahead of
// inline asm.
__device__ __forceinline__ void settle(f32x4_t (&s)[2][4]) {
  asm volatile("s_nop 15\n\ts_nop 7"
               : "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[0][2]), "+v"(s[0][3]), "+v"(s[1][0]), "+v"(s[1][1]),
                 "+v"(s[1][2]), "+v"(s[1][3]));
}

// The first of `tiles` tiles that chunk c of n takes: all take the same, some one more.
__device__ __forceinline__ int chunk_start(int tiles, int c, int n) {
  const int each = static_cast<uint32_t>(tiles) / static_cast<uint32_t>(n), more = tiles - each * n;
  return c * each + (c < more ? c : more);
}

// Token and head of row r of an item's row tile.
__device__ __forceinline__ void row_of(int group, const Item& it, int tile_rows, int r, int& t, int& h) {
  const int rr = it.tile * tile_rows + r;
  t = it.t0 + rr / group;
  h = it.kvh * group + rr % group;
}

// The kernel's arguments read anew: what only the end of a block needs would
// otherwise stay in scalar registers, or spill from them, through its tile loop.
typedef const __attribute__((address_space(4))) PagedArgs* late_args_t;
__device__ __forceinline__ late_args_t late_args() {
  uintptr_t p = (uintptr_t)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return (late_args_t)p;
}

// What earlier sums weigh against later ones, 2^x. Not 0, so that an infinity or a NaN
// in them stays one, but the least that fp32 holds: sums of any finite V then come to
// less than 5e-7 where they should not count.
__device__ __forceinline__ float share(float x) { return fmaxf(__builtin_amdgcn_exp2f(x), 0x1p-149f); }

// The reference that a finished state without a finite score is said to have: then it
// sums to nothing (no slot seen, or scores of -inf alone) or to NaN (a NaN score), and
// the sums go into those of other states like any. Whether a row sees a slot is told
// by its position: from 0 on it sees its own. So a row of NaN scores, or of -inf ones
// alone (0 / 0), gives NaN, and only a row that sees nothing gives zeros.
constexpr float kNoScore = -3.402823466e38f;

// The reference that weights are taken against moves only when a row's maximum has
// outgrown it by 2^kSlack: the sums have room for that, and most tiles then leave
// the accumulators alone (5000-token prompt 250 -> 240 us).
constexpr float kSlack = 8.f;

// Up to 32 query rows (one token of a sequence, or a few): the four waves split
// the slots, 16 of each tile, and each runs a softmax of its own over them; the
// states meet in LDS at the end. Slots are the M index of S^T = K Q^T and query
// rows the N index (NT tiles of 16); the scores' layout is the P^T operand's of
// O^T += V^T P^T, whose K = 32 holds the 16 slots twice, with the upper and with
// the lower bf16 half of their weights (about 16 bits; the product waits for
// memory anyway). An infinite V in a slot that every row sees gives NaN (the lower
// half is 0).
//
// Bound by the K/V stream: each wave stages its own 16 slots through LDS, two tiles
// ahead, and waits for nobody. 16 sequences of 32 + 8 heads, 24 K slots in all
// (98 MB): 21 us, 4.7 TB/s; three of 30 K slots (306 MB): 50 us, 6.1 TB/s.
// Against the waves splitting the rows (attend_many), 8 sequences of up to 5 rows, 20 a
// head, at up to 4096 slots (101 MB) take 30.1 us to 29.8, 32 of them (382 MB) 93.7 to
// 100; with 32 rows a head the two are within 8% either way, and this one keeps 16 bits
// of a weight.
template <int NT>
__device__ __forceinline__ void attend_few(const PagedArgs& a, const Item& it, const Slots& sl,
                                           const int32_t* table, const int* rowpos,
                                           unsigned char* ring, float (&wm)[4][16], float (&wl)[4][16]) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int i0 = chunk_start(sl.tiles, it.chunk, it.chunks), i1 = chunk_start(sl.tiles, it.chunk + 1, it.chunks);
  const int sinks = a.window ? a.sinks : 0;
  u32x4 qf[NT][4];
  Sight sight[NT];
  int all_hi = 0x7fffffff, all_lo = -0x7fffffff;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int r = 16 * n + col;
    int t, h;
    row_of(a.G, it, kFewRows, r < it.rows ? r : 0, t, h);  // padding columns repeat row 0
    const bf16_t* qrow = a.q + t * a.q_st + h * a.q_sh + 8 * quad;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) qf[n][ks] = *reinterpret_cast<const u32x4*>(qrow + 32 * ks);
    sight[n] = sight_of(it.seq < 0 ? rowpos[t] : it.p0 + (t - it.t0), sl, a.window);
    const int lo = min16(sight[n].vhi), hi = -min16(-sight[n].vlo);
    all_hi = lo < all_hi ? lo : all_hi;
    all_lo = hi > all_lo ? hi : all_lo;
  }
  uint32_t off[2];
  stage_offsets(lane, off);
  unsigned char* lds = ring + wave * 2 * kGroupBytes;
  auto slot_of = [&](int i) {
    return (i < sl.sink_tiles ? i : i - sl.sink_tiles + sl.first_tile) * kSplit + wave * 16;
  };
  // Every turn stages a group, past the last one an empty one, so that the
  // count of loads in flight stays the same.
  auto stage = [&](int i) {
    Group g{0, 0};
    if (i < i1) g = group_of(a, page_of(a, table, slot_of(i), sl.lo0, sl.hi), it.kvh, slot_of(i), sl.hi);
    const __amdgpu_buffer_rsrc_t k_rows = uniform_rsrc(a.keys + g.offset, g.bytes);
    const __amdgpu_buffer_rsrc_t v_rows = uniform_rsrc(a.values + g.offset, g.bytes);
    unsigned char* b = lds + ((i - i0) % kRing) * kTileBytes;
#pragma unroll
    for (int u = 0; u < 4; ++u) stage_quarter(k_rows, b, u, off);
#pragma unroll
    for (int u = 0; u < 4; ++u) stage_quarter(v_rows, b + kGroupBytes, u, off);
  };
  __builtin_amdgcn_sched_barrier(0);
  if (i0 < i1) {
#pragma unroll
    for (int i = 0; i < kRing; ++i) stage(i0 + i);
  }
  const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_t*)lds));
  const ReadAddrs from = read_addrs(base, base + kGroupBytes, col, quad);
  f32x4_t acc[NT][8];
  float m[NT], l[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[n][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  for (int i = i0; i < i1; ++i) {
    const uint32_t ro = static_cast<uint32_t>((i - i0) % kRing) * kTileBytes;
    u32x4 k[4];
    asm volatile(
        "s_waitcnt vmcnt(%4)\n\t"
        "ds_read_b128 %0, %5\n\t"
        "ds_read_b128 %1, %6\n\t"
        "ds_read_b128 %2, %7\n\t"
        "ds_read_b128 %3, %8"
        : "=&v"(k[0]), "=&v"(k[1]), "=&v"(k[2]), "=&v"(k[3])
        : "n"(8 * (kRing - 1)), "v"(k_addr(from, 0, ro)), "v"(k_addr(from, 1, ro)), "v"(k_addr(from, 2, ro)),
          "v"(k_addr(from, 3, ro))
        : "memory");
    uint32_t va[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) va[j] = v_addr(from, j, ro);
    u32x2_t v[8];
    issue_vt_tr<0>(va, v);
    asm volatile("s_waitcnt lgkmcnt(0)"
                 : "+v"(k[0]), "+v"(k[1]), "+v"(k[2]), "+v"(k[3]), "+v"(v[0]), "+v"(v[1]), "+v"(v[2]),
                   "+v"(v[3]), "+v"(v[4]), "+v"(v[5]), "+v"(v[6]), "+v"(v[7])
                 :
                 : "memory");
    const int s0 = slot_of(i), slot = s0 + 4 * quad;
    const bool whole = s0 + 15 <= all_hi && (s0 >= all_lo || s0 + 15 < sinks) && s0 >= sl.lo0;
    bool odd = false;
    if (!whole) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = u32x2_t{finite_pair(v[j].x, odd), finite_pair(v[j].y, odd)};
    }
    // The group's reads are done, so the next one goes into its buffer, unless
    // its V is to be read once more.
    const bool late = __any(odd);
    if (!late) stage(i + kRing);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      f32x4_t st = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) st = mfma(k[ks], qf[n][ks], st);
      float sc[4];
      if (whole) {
#pragma unroll
        for (int r = 0; r < 4; ++r) sc[r] = st[r] * a.scale2;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int s = slot + r;
          sc[r] = s <= sight[n].vhi && (s >= sight[n].vlo || s < sinks) ? st[r] * a.scale2 : -INFINITY;
        }
      }
      const float tmax = quad_max(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])));
      const bool moves = tmax > m[n] + kSlack;  // see kSlack
      if (__any(moves)) {
        const float m_new = moves ? tmax : m[n];
        const float alpha = share(m[n] - (m_new == -INFINITY ? 0.f : m_new));
        l[n] *= alpha;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[n][j] *= alpha;
        m[n] = m_new;
      }
      const float ms = m[n] == -INFINITY ? 0.f : m[n];  // nothing visible yet: weights of 0
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(sc[r] - ms);
      l[n] += (p[0] + p[1]) + (p[2] + p[3]);
      const uint32_t h0 = pack_bf2(p[0], p[1]), h1 = pack_bf2(p[2], p[3]);
      const u32x4 ph = {h0, h1, pack_bf2(p[0] - bf_lo(h0), p[1] - bf_hi(h0)),
                        pack_bf2(p[2] - bf_lo(h1), p[3] - bf_hi(h1))};
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[n][j] = mfma(u32x4{v[j].x, v[j].y, v[j].x, v[j].y}, ph, acc[n][j]);
      if (late) add_nonfinite(lds + ro + kGroupBytes, 16, s0, sight[n], sinks, quad, acc[n]);
    }
    if (late) stage(i + kRing);
  }
  // The waves' states, in LDS rows of 132 floats (the 16 rows in other banks).
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const late_args_t la = late_args();
  float* wacc = reinterpret_cast<float*>(ring);
  constexpr int kRowFloats = D + 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    l[n] = quad_sum(l[n]);
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<f32x4_t*>(wacc + (wave * 16 + col) * kRowFloats + 16 * j + 4 * quad) = acc[n][j];
    if (quad == 0) {
      wm[wave][col] = m[n];
      wl[wave][col] = l[n];
    }
    __syncthreads();
    for (int c = wave; c < 16 && 16 * n + c < it.rows; c += 4) {
      const float M = fmaxf(fmaxf(fmaxf(wm[0][c], wm[1][c]), fmaxf(wm[2][c], wm[3][c])), kNoScore);
      float L = 0.f, x = 0.f, y = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = share(wm[w][c] - M);
        const float2 o = *reinterpret_cast<const float2*>(wacc + (w * 16 + c) * kRowFloats + 2 * lane);
        L = fmaf(f, wl[w][c], L);
        x = fmaf(f, o.x, x);
        y = fmaf(f, o.y, y);
      }
      if (it.part >= 0) {
        const long row = it.part + 16 * n + c;
        *reinterpret_cast<float2*>(la->part + row * D + 2 * lane) = make_float2(x, y);
        if (lane == 0) la->ml[row] = make_float2(M, L);
      } else {
        int tr, hr;
        row_of(la->G, it, kFewRows, 16 * n + c, tr, hr);
        const float inv = it.p0 + (tr - it.t0) < 0 ? 0.f : 1.0f / L;
        *reinterpret_cast<uint32_t*>(la->out + tr * la->o_st + hr * la->o_sh + 2 * lane) = pack_bf2(x * inv, y * inv);
      }
    }
  }
}

// Up to 128 query rows: the waves split the rows, 32 each in two 16-row N
// tiles, and share each staged 64-slot tile of K and V, whose operand reads
// feed two products. Weights are rounded once to bf16 for the product, and the
// sum is taken over the rounded ones (as one more product, by ones), so that a
// row's weights add up to 1.
//
// Bound by the matrix and vector instructions, which share a SIMD's issue: a
// 5000-token prompt of 32 + 8 heads takes 228-235 us, 0.87-0.9 PFLOP/s of the causal
// products (an 8192^3 product 1.35), with the matrix cores at work in 44% of the
// cycles and vector instructions issued in 33%; LDS reads take a quarter. Neither
// 32x32 products, nor one half's products under the other half's softmax, nor fewer
// vector instructions (weights cut instead of rounded) changed that by more than 2%.
// A 1000-token chunk beside 15 single tokens, where a block has half a CU's issue to
// itself, takes 109-114 us, 0.53 PFLOP/s; staging loads all at the start of a tile,
// waiting for all of K, and accumulators copied around the rescaling made that 121.
__device__ __forceinline__ void attend_many(const PagedArgs& a, const Item& it, const Slots& sl,
                                            const int32_t* table, const int* rowpos,
                                            unsigned char* ring, int2* bounds, int* odd_tile) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int col = lane & 15, quad = lane >> 4;
  const int i0 = chunk_start(sl.tiles, it.chunk, it.chunks), i1 = chunk_start(sl.tiles, it.chunk + 1, it.chunks);
  const bool active = 32 * wave < it.rows;  // wave-uniform
  const int sinks = a.window ? a.sinks : 0;
  u32x4 qf[2][4];
  Sight sight[2];
  int all_hi = 0x7fffffff, all_lo = -0x7fffffff;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int r = 32 * wave + 16 * n + col;
    int t, h;
    row_of(a.G, it, kManyRows, r < it.rows ? r : it.rows - 1, t, h);
    const bf16_t* qrow = a.q + t * a.q_st + h * a.q_sh + 8 * quad;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) qf[n][ks] = *reinterpret_cast<const u32x4*>(qrow + 32 * ks);
    const int first = it.t0 + it.tile * kManyRows / a.G;
    sight[n] = sight_of(it.seq < 0 ? rowpos[t - first] : it.p0 + (t - it.t0), sl, a.window);
    const int lo = min16(sight[n].vhi), hi = -min16(-sight[n].vlo);
    all_hi = lo < all_hi ? lo : all_hi;
    all_lo = hi > all_lo ? hi : all_lo;
  }
  uint32_t off[2];
  stage_offsets(lane, off);
  auto tile_of = [&](int i) {
    return (i < sl.sink_tiles ? i : i - sl.sink_tiles + sl.first_tile) * kSplit;
  };
  // A tile is staged during the work on the one before, 16 slots a wave, a load after
  // every four products (all eight at once hold the wave), from descriptors made a
  // tile and a page looked up two tiles ahead. Past the last tile they load zeros.
  auto page_at = [&](int i) {
    return i < i1 ? page_of(a, table, tile_of(i) + wave * 16, sl.lo0, sl.hi) : -1;
  };
  int page = page_at(i0);
  __amdgpu_buffer_rsrc_t k_rows, v_rows;
  auto prepare = [&](int i) {
    const Group g = group_of(a, page, it.kvh, tile_of(i) + wave * 16, sl.hi);
    k_rows = uniform_rsrc(a.keys + g.offset, g.bytes);
    v_rows = uniform_rsrc(a.values + g.offset, g.bytes);
    page = page_at(i + 1);
  };
  auto load = [&](int i, int u) {
    unsigned char* b = ring + ((i - i0) & 1) * kTileBytes + wave * kGroupBytes;
    if (u < 4) stage_quarter(k_rows, b, u, off);
    else stage_quarter(v_rows, b + kSplit * D * 2, u - 4, off);
  };
  __builtin_amdgcn_sched_barrier(0);
  if (i0 < i1) {
    prepare(i0);
#pragma unroll
    for (int u = 0; u < 8; ++u) load(i0, u);
    prepare(i0 + 1);
  }
  const uint32_t ring_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_void_t*)ring));
  const ReadAddrs from = read_addrs(ring_base, ring_base + kSplit * D * 2, col, quad);
  const u32x4 ones = {0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  f32x4_t acc[2][8], sum[2];
  float m[2] = {-INFINITY, -INFINITY}, base[2] = {0.f, 0.f};  // of the unscaled scores, and scaled
  const float slack = kSlack / a.scale2;
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    sum[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[n][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  auto tile = [&](int i, int s0, uint32_t tb, bool whole) {
    f32x4_t st[2][4];
    u32x4 kf[4][4];
    issue_k_pf<0>(k_addr(from, 0, tb), kf[0]);
    issue_k_pf<0>(k_addr(from, 1, tb), kf[1]);
    issue_k_pf<0>(k_addr(from, 2, tb), kf[2]);
    issue_k_pf<0>(k_addr(from, 3, tb), kf[3]);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        if (n == 0 && ks == 0) wait_k4<12>(kf[0]);  // K as it arrives
        if (n == 0 && ks == 1) wait_k4<8>(kf[1]);
        if (n == 0 && ks == 2) wait_k4<4>(kf[2]);
        if (n == 0 && ks == 3) wait_k4<0>(kf[3]);
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
          st[n][mt] = mfma(kf[ks][mt], qf[n][ks], ks ? st[n][mt] : f32x4_t{0.f, 0.f, 0.f, 0.f});
        load(i + 1, 4 * n + ks);
        __builtin_amdgcn_sched_barrier(0);
      }
    // The V^T operands of half the tile in flight during the softmax.
    uint32_t va[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) va[j] = v_addr(from, j, tb);
    u32x2_t vw[2][8];
    issue_vt_tr<0>(va, vw[0]);
    issue_vt_tr<4096>(va, vw[1]);
    settle(st);
    uint2 pb[2][4];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      if (!whole) {
        asm volatile("");  // a branch, not 16 selects on every tile
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int s = s0 + 16 * mt + 4 * quad + r;
            st[n][mt][r] = s <= sight[n].vhi && (s >= sight[n].vlo || s < sinks) ? st[n][mt][r] : -INFINITY;
          }
      }
      float tmax = max3(st[n][0][0], st[n][0][1], st[n][0][2]);
#pragma unroll
      for (int i = 3; i < 15; i += 2)
        tmax = max3(tmax, st[n][i / 4][i % 4], st[n][(i + 1) / 4][(i + 1) % 4]);
      tmax = quad_max3(max3(tmax, st[n][3][3], st[n][3][3]));
      const bool moves = tmax > m[n] + slack;  // see kSlack
      if (__builtin_expect(__any(moves), 0)) {
        const float m_new = moves ? tmax : m[n];  // of that row alone: no row's sums depend on another's scores
        const float ms = m_new == -INFINITY ? 0.f : m_new * a.scale2;  // nothing visible yet: weights of 0
        const float alpha = moves ? share(fmaf(m[n], a.scale2, -ms)) : 1.f;
        sum[n] *= alpha;
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[n][j] *= alpha;
        m[n] = m_new;
        base[n] = ms;
      }
      // The branch not taken would copy the accumulators into the products' registers:
      // they pass into another block first.
#pragma unroll
      for (int j = 0; j < 8; ++j) asm volatile("" : "+v"(acc[n][j]));
      int never = 0;
      asm volatile("" : "+s"(never));
      if (__builtin_expect(never, 0)) asm volatile("s_nop 0");
#pragma unroll
      for (int mt = 0; mt < 4; ++mt) {
        float p[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) p[r] = __builtin_amdgcn_exp2f(fmaf(st[n][mt][r], a.scale2, -base[n]));
        pb[n][mt] = make_uint2(pack_bf2(p[0], p[1]), pack_bf2(p[2], p[3]));
      }
    }
    auto weigh = [&](const u32x2_t (&v)[2][8], int mt) {
      u32x4 p[2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        p[n] = u32x4{pb[n][mt].x, pb[n][mt].y, pb[n][mt + 1].x, pb[n][mt + 1].y};
        sum[n] = mfma(ones, p[n], sum[n]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const u32x4 x = {v[0][j].x, v[0][j].y, v[1][j].x, v[1][j].y};
#pragma unroll
        for (int n = 0; n < 2; ++n) acc[n][j] = mfma(x, p[n], acc[n][j]);
      }
    };
    wait_v16(vw);
    u32x2_t vx[2][8];
    issue_vt_tr<8192>(va, vx[0]);
    issue_vt_tr<12288>(va, vx[1]);
    __builtin_amdgcn_sched_barrier(0);
    weigh(vw, 0);
    __builtin_amdgcn_sched_barrier(0);
    wait_v16(vx);
    weigh(vx, 2);
  };
  // The slots that all rows of the block see.
  if (lane == 0) bounds[wave] = make_int2(all_hi, all_lo);
  if (tid == 0) *odd_tile = 0;
  lds_barrier();
  int block_hi = bounds[0].x, block_lo = bounds[0].y;
#pragma unroll
  for (int w = 1; w < 4; ++w) {
    block_hi = bounds[w].x < block_hi ? bounds[w].x : block_hi;
    block_lo = bounds[w].y > block_lo ? bounds[w].y : block_lo;
  }
  block_hi = __builtin_amdgcn_readfirstlane(block_hi);
  block_lo = __builtin_amdgcn_readfirstlane(block_lo);
  auto seen_by_all = [&](int s0, int hi, int lo) {
    return s0 + kSplit - 1 <= hi && s0 >= sl.lo0 && (s0 >= lo || s0 + kSplit - 1 < sinks);
  };
  for (int i = i0; i < i1; ++i) {
    // This wave's part of tile i has landed; after the barrier everyone's has,
    // and every wave is done with tile i - 1, whose buffer tile i + 1 now takes.
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    lds_barrier();
    const uint32_t tb = static_cast<uint32_t>(((i - i0) & 1) * kTileBytes);
    const int s0 = tile_of(i);
    if (__builtin_expect(!seen_by_all(s0, block_hi, block_lo), 0)) {
      // Zero times an infinite or NaN V is NaN: where a tile has any, the rows that
      // see its slot get it by addition, and the products take it as zero.
      unsigned char* v = ring + tb + kSplit * D * 2;
      uint4* own = reinterpret_cast<uint4*>(v + wave * kGroupBytes) + lane;
      bool odd = false;
#pragma unroll 1
      for (int u = 0; u < 4; ++u) {
        const uint4 x = own[u * 64];
        finite_pair(x.x, odd);
        finite_pair(x.y, odd);
        finite_pair(x.z, odd);
        finite_pair(x.w, odd);
      }
      if (odd) *odd_tile = 1;
      __syncthreads();
      if (*odd_tile) {
        if (active) {
#pragma unroll
          for (int n = 0; n < 2; ++n) add_nonfinite(v, kSplit, s0, sight[n], sinks, quad, acc[n]);
        }
        __syncthreads();
        if (tid == 0) *odd_tile = 0;
#pragma unroll 1
        for (int u = 0; u < 4; ++u) {
          const uint4 x = own[u * 64];
          own[u * 64] = make_uint4(finite_pair(x.x, odd), finite_pair(x.y, odd), finite_pair(x.z, odd),
                                   finite_pair(x.w, odd));
        }
        __syncthreads();
      }
    }
    tile(i, s0, tb, seen_by_all(s0, all_hi, all_lo));
    prepare(i + 2);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  const late_args_t la = late_args();
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int r = 32 * wave + 16 * n + col;
    if (r >= it.rows) continue;
    if (it.part >= 0) {
      const long row = it.part + r;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<f32x4_t*>(la->part + row * D + 16 * j + 4 * quad) = acc[n][j];
      if (quad == 0) la->ml[row] = make_float2(fmaxf(m[n] * la->scale2, kNoScore), sum[n][0]);
    } else {
      int t, h;
      row_of(la->G, it, kManyRows, r, t, h);
      const float inv = it.p0 + (t - it.t0) < 0 ? 0.f : 1.0f / sum[n][0];
      bf16_t* dst = la->out + t * la->o_st + h * la->o_sh + 4 * quad;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        *reinterpret_cast<uint2*>(dst + 16 * j) = make_uint2(pack_bf2(acc[n][j][0] * inv, acc[n][j][1] * inv),
                                                             pack_bf2(acc[n][j][2] * inv, acc[n][j][3] * inv));
    }
  }
}

__global__ __launch_bounds__(kBlock, 2) void paged_attention_kernel(PagedArgs a) {
  extern __shared__ __align__(256) unsigned char ring[];  // two staged tiles
  __shared__ int rowpos[kManyRows];
  __shared__ float wm[4][16], wl[4][16];
  __shared__ int2 bounds[4];
  __shared__ int odd_tile;
  const int prefix = __builtin_amdgcn_readfirstlane(prefix_slots(a));
  Item it{};
  if (!make_plan(a, prefix, it)) return;
  const bool few = it.n * a.G <= kFewRows;
  const int tile_rows = few ? kFewRows : kManyRows;
  // The tile's first and last token, and the slots that its rows see.
  const int first = it.tile * tile_rows / a.G, last = (it.tile * tile_rows + it.rows - 1) / a.G;
  Slots sl;
  const int32_t* table;
  if (it.seq < 0) {
    sl = slots_of(0, prefix - 1, 0, 0, 0);
    table = a.prefix_pages;
    // Positions of the tile's tokens, from the sequences that they belong to.
    if (threadIdx.x < kManyRows) rowpos[threadIdx.x] = -1;
    __syncthreads();
    for (int j = threadIdx.x; j < a.B; j += kBlock) {
      const Span s = make_span(a.starts[j], a.starts[j + 1], a.lengths[j], a.T, a.table_pages << a.page_shift);
      const int from = s.t0 > first ? s.t0 : first, to = s.t0 + s.n - 1 < last ? s.t0 + s.n - 1 : last;
      for (int t = from; t <= to; ++t) rowpos[t - first] = s.p0 + (t - s.t0);
    }
    __syncthreads();
  } else {
    sl = slots_of(it.p0 + first, it.p0 + last, prefix, a.window, a.sinks);
    table = a.table + it.seq * a.table_st;
  }
  if (it.rows <= 16 && few) attend_few<1>(a, it, sl, table, rowpos, ring, wm, wl);
  else if (few) attend_few<2>(a, it, sl, table, rowpos, ring, wm, wl);
  else attend_many(a, it, sl, table, rowpos, ring, bounds, &odd_tile);
}

// The rows whose slots were split, one wave each:
//   out = sum_c 2^(m_c - M) acc_c / sum_c 2^(m_c - M) l_c,  M = max_c m_c
// over the chunks of the row's own slots and, where one is shared, of the prefix.
// A lane first holds a chunk's (m, l); then each half of the wave takes every
// other chunk's row, four dims a lane, eight chunks' loads in flight. A launch of
// 4-6 us, 2048 blocks at most, and 4.0-4.6 where the prompt's 160000 rows are not split:
// its waves end at their first row, once they have the plan.
__global__ __launch_bounds__(kBlock) void paged_merge_kernel(PagedArgs a) {
  const int lane = threadIdx.x & 63, half = lane >> 5, dim = 4 * (lane & 31);
  const int split = a.plan[0].split;
  const bool shared = a.prefix_length != nullptr;
  const long rows = static_cast<long>(a.T) * a.Hq;
  for (long orow = static_cast<long>(blockIdx.x) * 4 + (threadIdx.x >> 6); orow < rows;
       orow += static_cast<long>(gridDim.x) * 4) {
    const int t = static_cast<int>(orow / a.Hq), h = static_cast<int>(orow % a.Hq);
    const int j = sequence_of(a.starts, a.B, t, lane);
    if (!split) return;
    if (j >= a.B) continue;
    const PlanEntry own = a.plan[j + (shared ? 1 : 0)];
    const int64_t from = a.starts[j], to = a.starts[j + 1], end = a.starts[a.B], length = a.lengths[j];
    if (!own.chunks || t < from || t >= to) continue;  // with chunks, starts rise
    const int kvh = h / a.G;
    float M = kNoScore, L = 0.f;
    f32x4_t o = {0.f, 0.f, 0.f, 0.f};
    auto fold = [&](const PlanEntry& p, int token, int tokens) {
      const int r = token * a.G + h % a.G;
      const int tile_rows = tokens * a.G <= kFewRows ? kFewRows : kManyRows;
      const long row = p.part + (static_cast<long>(r / tile_rows) * p.chunks * a.Hkv + kvh) * p.stride + r % tile_rows;
      const long step = static_cast<long>(a.Hkv) * p.stride;
      for (int c0 = 0; c0 < p.chunks; c0 += kWave) {
        const int n = p.chunks - c0 < kWave ? p.chunks - c0 : kWave;
        const float2 ml = lane < n ? a.ml[row + (c0 + lane) * step] : make_float2(kNoScore, 0.f);
        constexpr int U = 8;
        f32x4_t x[U];
        auto fetch = [&](int c) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int at = c + 2 * u + half;
            x[u] = *reinterpret_cast<const f32x4_t*>(a.part + (row + (c0 + (at < n ? at : 0)) * step) * D + dim);
          }
        };
        fetch(0);
        const float mb = fmaxf(M, wave_max(ml.x));
        const float f0 = share(M - mb), f = share(ml.x - mb);
        M = mb;
        L = fmaf(L, f0, wave_sum(f * ml.y));
        o *= f0;
        for (int c = 0;;) {
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int at = c + 2 * u + half;
            const float g = __shfl(f, at < n ? at : 0, kWave);
            if (at < n) o += x[u] * g;
          }
          c += 2 * U;
          if (c >= n) break;
          fetch(c);
        }
      }
    };
    fold(own, t - static_cast<int>(from), static_cast<int>(to - from));
    if (shared) fold(a.plan[0], t, static_cast<int>(end));
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] += __shfl_xor(o[i], 32, kWave);
    const Span s = make_span(from, to, length, a.T, a.table_pages << a.page_shift);
    const float inv = s.p0 + (t - s.t0) < 0 ? 0.f : 1.0f / L;
    if (half == 0)
      *reinterpret_cast<uint2*>(a.out + t * a.o_st + h * a.o_sh + dim) =
          make_uint2(pack_bf2(o[0] * inv, o[1] * inv), pack_bf2(o[2] * inv, o[3] * inv));
  }
}

// ------------------------------------------------------------------ host

constexpr long kMergeBlocks = 2048;
constexpr long kMaxSlots = 1L << 29;

int page_shift_of(int64_t page) {
  for (int s = 4; s <= 10; ++s)
    if (page == (1L << s)) return s;
  return -1;
}

struct Sizes {
  long plan, rows;  // bytes of the plan, rows of partials
  long blocks;
};

// Upper bounds of what the plan needs (see make_plan), from the sizes alone.
Sizes sizes_of(long tokens, long batch, long q_heads, long kv_heads, bool shared) {
  Sizes s;
  const long rows = tokens * (q_heads / kv_heads), with = batch < tokens ? batch : tokens;
  const long top = rows < kManyRows ? (rows + 15) / 16 * 16 : kManyRows;
  s.plan = ((batch + 1) * static_cast<long>(sizeof(PlanEntry)) + 255) / 256 * 256;
  s.rows = 2L * kTargetBlocks * top;
  long tiles = rows / kManyRows + with;
  if (shared) {
    s.rows += kv_heads * (2 * rows + (with + 1) * (top - 1));
    tiles += rows / kManyRows + 1;
  }
  s.blocks = kTargetBlocks + kv_heads * tiles;
  return s;
}

bool bad_batch(long tokens, long batch, long q_heads, long kv_heads, long pages, long table_pages, int shift) {
  return tokens <= 0 || batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || pages <= 0 ||
         table_pages <= 0 || shift < 0;
}

int attend(PagedArgs& a, void* scratch, int64_t scratch_bytes, hipStream_t st) {
  const bool shared = a.prefix_length != nullptr;
  const Sizes s = sizes_of(a.T, a.B, a.Hq, a.Hkv, shared);
  if (s.blocks >= (1L << 31) || s.rows >= (1L << 31)) return HTN_EUNSUPPORTED;
  if (scratch_bytes < s.plan + s.rows * (D * 4 + 8)) return HTN_EINVAL;
  char* p = static_cast<char*>(scratch);
  a.plan = reinterpret_cast<PlanEntry*>(p);
  a.part = reinterpret_cast<float*>(p + s.plan);
  a.ml = reinterpret_cast<float2*>(p + s.plan + s.rows * D * 4);
  a.scale2 = 1.4426950408889634f / sqrtf(static_cast<float>(D));
  constexpr int lds = kRing * kTileBytes;
  const long merge = (static_cast<long>(a.T) * a.Hq + 3) / 4;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&paged_attention_kernel),
                                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  (void)attr;  // a refused size surfaces as a launch error
  hipLaunchKernelGGL(paged_attention_kernel, dim3(static_cast<unsigned>(s.blocks)), dim3(kBlock), lds, st, a);
  if (launch_status() != HTN_OK) return HTN_ELAUNCH;
  hipLaunchKernelGGL(paged_merge_kernel, dim3(static_cast<unsigned>(merge < kMergeBlocks ? merge : kMergeBlocks)), dim3(kBlock), 0, st, a);
  return launch_status();
}

}  // namespace
}  // namespace htn

using namespace htn;

extern "C" int htn_norm_rope_paged(const void* q, int64_t q_st, const void* k, int64_t k_st, const void* v,
                                   int64_t v_st, const void* q_gain, const void* k_gain, float q_eps,
                                   float k_eps, const void* cos, const void* sin, int64_t rope_st,
                                   int64_t rope_rows, int rope_fp32, void* keys, void* values, int64_t pages,
                                   int64_t page_size, const int32_t* page_table, int64_t table_st,
                                   int64_t table_pages, const int64_t* starts, const int64_t* lengths,
                                   int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads, void* out_q,
                                   htn_stream_t stream) {
  const int shift = page_shift_of(page_size);
  if (!q || !k || !v || !cos || !sin || !keys || !values || !page_table || !starts || !lengths || !out_q ||
      rope_rows <= 0 || bad_batch(tokens, batch, q_heads, kv_heads, pages, table_pages, shift))
    return HTN_EINVAL;
  if ((q_st | k_st | v_st | rope_st) & 7) return HTN_EUNSUPPORTED;
  for (const void* p : {q, k, v, q_gain, k_gain, cos, sin, static_cast<const void*>(keys),
                        static_cast<const void*>(values), static_cast<const void*>(out_q)})
    if (!aligned16(p)) return HTN_EUNSUPPORTED;
  if (tokens > (1L << 30) || batch > (1L << 24) || q_heads + 2 * kv_heads > (1L << 16) ||
      (table_pages << shift) > kMaxSlots)
    return HTN_EUNSUPPORTED;
  AppendArgs a{};
  a.q = static_cast<const bf16_t*>(q); a.k = static_cast<const bf16_t*>(k); a.v = static_cast<const bf16_t*>(v);
  a.q_st = q_st; a.k_st = k_st; a.v_st = v_st;
  a.qg = static_cast<const bf16_t*>(q_gain); a.kg = static_cast<const bf16_t*>(k_gain);
  a.q_eps = q_eps; a.k_eps = k_eps;
  a.cos = cos; a.sin = sin; a.rope_st = rope_st; a.rope_rows = rope_rows;
  a.keys = static_cast<bf16_t*>(keys); a.values = static_cast<bf16_t*>(values);
  a.pages = pages; a.page_shift = shift;
  a.table = page_table; a.table_st = table_st; a.table_pages = table_pages;
  a.starts = starts; a.lengths = lengths;
  a.out_q = static_cast<bf16_t*>(out_q);
  a.B = static_cast<int>(batch); a.T = static_cast<int>(tokens);
  a.Hq = static_cast<int>(q_heads); a.Hkv = static_cast<int>(kv_heads);
  const dim3 grid(static_cast<unsigned>(tokens), static_cast<unsigned>((q_heads + 2 * kv_heads + 15) / 16));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rope_fp32) hipLaunchKernelGGL(norm_rope_paged_kernel<float>, grid, dim3(kBlock), 0, st, a);
  else hipLaunchKernelGGL(norm_rope_paged_kernel<bf16_t>, grid, dim3(kBlock), 0, st, a);
  return launch_status();
}

extern "C" int64_t htn_paged_attention_scratch_bytes(int64_t tokens, int64_t batch, int64_t q_heads,
                                                     int64_t kv_heads, int shared_prefix) {
  if (tokens <= 0 || batch <= 0 || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads ||
      tokens > (1L << 30) || batch > (1L << 24) || q_heads > (1L << 16))
    return 0;
  const Sizes s = sizes_of(tokens, batch, q_heads, kv_heads, shared_prefix != 0);
  return s.plan + s.rows * (D * 4 + 8);
}

namespace {

int fill_args(PagedArgs& a, const void* q, int64_t q_st, int64_t q_sh, const void* keys, const void* values,
              int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_st,
              int64_t table_pages, const int64_t* starts, const int64_t* lengths, void* out, int64_t o_st,
              int64_t o_sh, int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads,
              const void* scratch) {
  const int shift = page_shift_of(page_size);
  if (!q || !keys || !values || !page_table || !starts || !lengths || !out || !scratch ||
      bad_batch(tokens, batch, q_heads, kv_heads, pages, table_pages, shift))
    return HTN_EINVAL;
  if (((q_st | q_sh) & 7) || ((o_st | o_sh) & 3) || !aligned16(q) || !aligned16(keys) || !aligned16(values) ||
      !aligned8(out) || !aligned16(scratch))
    return HTN_EUNSUPPORTED;
  // Row numbers (tokens x group) and slots are 32-bit in the kernels; offsets
  // into the pools, q and out are 64-bit.
  if (tokens > (1L << 30) || batch > (1L << 24) || q_heads > (1L << 16) ||
      tokens * (q_heads / kv_heads) > (1L << 30) || (table_pages << shift) > kMaxSlots)
    return HTN_EUNSUPPORTED;
  a.q = static_cast<const bf16_t*>(q); a.q_st = q_st; a.q_sh = q_sh;
  a.keys = static_cast<const bf16_t*>(keys); a.values = static_cast<const bf16_t*>(values);
  a.pages = pages; a.page_shift = shift;
  a.table = page_table; a.table_st = table_st; a.table_pages = table_pages;
  a.starts = starts; a.lengths = lengths;
  a.out = static_cast<bf16_t*>(out); a.o_st = o_st; a.o_sh = o_sh;
  a.B = static_cast<int>(batch); a.T = static_cast<int>(tokens);
  a.Hq = static_cast<int>(q_heads); a.Hkv = static_cast<int>(kv_heads);
  a.G = static_cast<int>(q_heads / kv_heads);
  return HTN_OK;
}

}  // namespace

extern "C" int htn_paged_attention(const void* q, int64_t q_st, int64_t q_sh, const void* keys,
                                   const void* values, int64_t pages, int64_t page_size,
                                   const int32_t* page_table, int64_t table_st, int64_t table_pages,
                                   const int64_t* starts, const int64_t* lengths, int64_t window, int64_t sinks,
                                   void* out, int64_t o_st, int64_t o_sh, int64_t batch, int64_t tokens,
                                   int64_t q_heads, int64_t kv_heads, void* scratch, int64_t scratch_bytes,
                                   htn_stream_t stream) {
  PagedArgs a{};
  const int rc = fill_args(a, q, q_st, q_sh, keys, values, pages, page_size, page_table, table_st, table_pages,
                           starts, lengths, out, o_st, o_sh, batch, tokens, q_heads, kv_heads, scratch);
  if (rc != HTN_OK) return rc;
  if (window < 0 || sinks < 0) return HTN_EINVAL;
  // A window past the table's slots hides nothing, and no more sinks than slots exist.
  const int64_t slots = table_pages * page_size;
  a.window = static_cast<int>(window >= slots ? 0 : window);
  a.sinks = static_cast<int>(sinks < slots ? sinks : slots);
  return attend(a, scratch, scratch_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int htn_shared_prefix_attention(const void* q, int64_t q_st, int64_t q_sh, const void* keys,
                                           const void* values, int64_t pages, int64_t page_size,
                                           const int32_t* prefix_pages, int64_t prefix_count,
                                           const int64_t* prefix_length, const int32_t* page_table,
                                           int64_t table_st, int64_t table_pages, const int64_t* starts,
                                           const int64_t* lengths, void* out, int64_t o_st, int64_t o_sh,
                                           int64_t batch, int64_t tokens, int64_t q_heads, int64_t kv_heads,
                                           void* scratch, int64_t scratch_bytes, htn_stream_t stream) {
  PagedArgs a{};
  const int rc = fill_args(a, q, q_st, q_sh, keys, values, pages, page_size, page_table, table_st, table_pages,
                           starts, lengths, out, o_st, o_sh, batch, tokens, q_heads, kv_heads, scratch);
  if (rc != HTN_OK) return rc;
  if (!prefix_pages || !prefix_length || prefix_count <= 0) return HTN_EINVAL;
  if ((prefix_count << a.page_shift) > kMaxSlots) return HTN_EUNSUPPORTED;
  a.prefix_pages = prefix_pages;
  a.prefix_count = prefix_count;
  a.prefix_length = prefix_length;
  return attend(a, scratch, scratch_bytes, static_cast<hipStream_t>(stream));
}
