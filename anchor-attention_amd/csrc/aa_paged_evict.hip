// Giving up the keys of a cache in pages that have had the least attention, on gfx950: which ones stay, and their move to the front of the sequence's pages.
//
// Choosing: a work-group for each (sequence, KV head) finds what the wanted number of weights reaches by histograms of 256 equal ranges of the weights' order, each inside the range
// of the last one that holds it, as pages are chosen for sparse steps, and lists the places in order by sums over the work-group.  Integers only: the order in which counts are added
// does not matter.  Weights stay in registers between the rounds, or are read again where there are more than these hold.  (In LDS: 33000 keys 28 us; with one copy of the bins no
// more.)
//
// Moving is bound by reading and writing the rows once.  It is in place, and rows go to lower places in their order, so a work-group that takes them in turn, each chunk read by all before
// any of it is written, needs no room beside: no later row lies where an earlier one goes.  A work-group has 32 channels of keys or values; where that makes too few
// work-groups, the rows of a (sequence, KV head) are cut into groups, and those that come from another group's places are copied to scratch by a launch of its own first.
//
// Measured: 8 sequences of 3000 to 33000 keys down to 4096, 8 KV heads of 128, 92 us a step: choosing 25.4, as long as one work-group takes for the longest, moving 53.7, 4.4
// TB/s; one of 4160 keys, 8 of 64, 21 us: choosing 8.4, saving 3.5, moving 9.0, chains of loads all three.  (Slices of 64 channels: moving 60.)
#include <algorithm>

#include "aa_kernels.h"
#include "aa_paged.h"

namespace aa {

constexpr int kKeepThreads = 1024, kKeepWaves = kKeepThreads / 64, kKeepStep = 4 * kKeepThreads;
constexpr int kKeepItems = 9, kKeepHeld = kKeepItems * kKeepStep;  // fours of weights that a thread holds
constexpr int kMostKeys = 1 << 20;

// HELD: no sequence has more keys than a work-group holds
template <bool HELD>
__global__ void __launch_bounds__(kKeepThreads) paged_keep_kernel(const PagedEvictArgs p) {
  constexpr int kCopies = 8;  // of the first round's bins, for every eighth lane: most weights are of few bins, which lanes would wait for
  __shared__ __attribute__((aligned(16))) uint32_t bins[3 + kCopies][256];  // (the first round's last)
  __shared__ uint32_t ranges[2][kKeepWaves];
  __shared__ uint64_t counts[(HELD ? kKeepItems : kMostKeys / kKeepStep) * kKeepWaves];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / p.n_kv_heads, kvh = blockIdx.x - b * p.n_kv_heads;
  const int n = clamped_length(p.lengths, b, p.max_pages, p.page_log);
  int32_t* kept = p.kept + (int64_t)blockIdx.x * p.n_keys;
  if (kvh == 0 && tid == 0) p.new_lengths[b] = n > p.above ? p.n_keys : n;
  if (n <= p.above) {
    for (int i = tid; i < p.n_keys; i += kKeepThreads) kept[i] = -1;
    return;
  }
  const bool held = HELD || n <= kKeepHeld;
  const int first = p.n_first, end = n - p.n_last;  // the candidates
  for (int i = tid; i < (3 + kCopies) * 256; i += kKeepThreads) bins[0][i] = 0u;
  // weights as numbers of the same order; 0 for what is no candidate
  auto load = [&](const int i, uint32_t (&x)[4]) {
    const int64_t page = clamped_page(p.table[b * p.t_sb + (i >> p.page_log)], p.n_pages);
    const floatx4 w = *reinterpret_cast<const floatx4*>(p.weights + ((page * p.n_kv_heads + kvh) << p.page_log) + (i & ((1 << p.page_log) - 1)));
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = i + e >= first && i + e < end ? ordered(w[e]) : 0u;
  };
  const int items = (n + kKeepStep - 1) / kKeepStep;
  uint32_t mine[kKeepItems][4] = {};
  if (held) {
#pragma unroll
    for (int j = 0; j < kKeepItems; ++j)
      if (kKeepStep * j + 4 * tid < n) load(kKeepStep * j + 4 * tid, mine[j]);
  }
  auto each = [&](auto&& f) {  // f(j, numbers): item j of a thread is four keys
    if (held) {
#pragma unroll
      for (int j = 0; j < kKeepItems; ++j) {
        if (j > 0 && j >= items) break;
        f(j, mine[j]);
      }
    } else {
#pragma nounroll
      for (int j = 0; j < items; ++j) {
        const int i = kKeepStep * j + 4 * tid;
        uint32_t x[4] = {0u, 0u, 0u, 0u};
        if (i < n) load(i, x);
        f(j, x);
      }
    }
  };
  uint32_t lo = 0xffffffffu, hi = 0u;
  auto extend = [&](const uint32_t (&x)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      lo = min(lo, x[e] - 1u);  // (0 becomes the largest; no number is)
      hi = max(hi, x[e]);
    }
  };
  each([&](const int, const uint32_t (&x)[4]) { extend(x); });
  lo = up_to(lo, 0xffffffffu, [](const uint32_t a, const uint32_t b) { return min(a, b); });
  hi = up_to(hi, 0u, [](const uint32_t a, const uint32_t b) { return max(a, b); });
  if (lane == 63) {
    ranges[0][wave] = lo;
    ranges[1][wave] = hi;
  }
  __syncthreads();  // (the bins are 0 too)
#pragma unroll
  for (int w = 0; w < kKeepWaves; ++w) {
    lo = w == 0 ? ranges[0][0] : min(lo, ranges[0][w]);
    hi = w == 0 ? ranges[1][0] : max(hi, ranges[1][w]);
  }
  lo = __builtin_amdgcn_readfirstlane(lo) + 1u;
  hi = __builtin_amdgcn_readfirstlane(hi);
  // The wanted-th largest weight lies from lo to hi; all of those above are taken.  A range is 2^32 long at most and the next one a 256th, so four do.
  int wanted = p.n_keys - p.n_first - p.n_last;
  if (wanted == 0) lo = hi = 0xffffffffu;  // (none)
#pragma nounroll
  for (int round = 0; wanted > 0 && lo < hi; ++round) {
    const uint32_t span = hi - lo;
    const int shift = span < 256u ? 0 : 24 - __builtin_clz(span);  // span >> shift < 256
    uint32_t* own_bins = bins[round == 0 ? 3 + (lane & (kCopies - 1)) : round - 1];
    uint32_t least_ones = 0;  // (not one by one: weights that nothing has been added to are alike)
    each([&](const int, const uint32_t (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t d = x[e] - lo;
        if (d == 0u) ++least_ones;
        else if (d <= span) atomicAdd(&own_bins[d >> shift], 1u);
      }
    });
    least_ones = (uint32_t)sums_up_to((int)least_ones);
    if (lane == 63 && least_ones > 0) atomicAdd(&own_bins[0], least_ones);
    __syncthreads();
    int m[4] = {0, 0, 0, 0};
    for (int c = round == 0 ? 3 : round - 1; c < (round == 0 ? 3 + kCopies : round); ++c) {
      const uint4 bin4 = *reinterpret_cast<const uint4*>(&bins[c][4 * lane]);
      m[0] += bin4.x, m[1] += bin4.y, m[2] += bin4.z, m[3] += bin4.w;
    }
    const int own = m[0] + m[1] + m[2] + m[3], sums = sums_up_to(own), all = __builtin_amdgcn_readlane(sums, 63);
    // the last lane that has `wanted` weights in its bins or behind them, and the last of its bins that has
    const int at = 63 - __builtin_clzll(__ballot(all - sums + own >= wanted));
    int above = __builtin_amdgcn_readlane(all - sums, at), in_bin = 0, bin = 4 * at;
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      in_bin = __builtin_amdgcn_readlane(m[j], at);
      if (above + in_bin >= wanted) {
        bin += j;
        break;
      }
      above += in_bin;
    }
    wanted -= above;  // of this bin
    lo += (uint32_t)bin << shift;
    hi = lo + min(hi - lo, (1u << shift) - 1u);
    if (shift == 0 || wanted == in_bin) break;  // (one number is left, or all of the bin are taken)
  }

  // Weights above hi are taken, and of those from lo to hi the first `wanted`: counted by item and wave, which is the keys' order.
  auto counts_of = [&](const uint32_t (&x)[4]) {  // of an item, in the upper and the lower half
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) packed += (x[e] - lo <= hi - lo ? 0x10000u : 0u) + (x[e] > hi ? 1u : 0u);
    return packed;
  };
  each([&](const int j, const uint32_t (&x)[4]) {
    const uint32_t all = (uint32_t)sums_up_to((int)counts_of(x));
    if (lane == 63) counts[kKeepWaves * j + wave] = (uint64_t)(all >> 16) << 32 | (all & 0xffffu);
  });
  __syncthreads();
  if (wave == 0) {  // (sums of all before each)
    uint32_t so_far_equal = 0, so_far_sure = 0;
#pragma nounroll
    for (int i = 0; i < items * kKeepWaves; i += 64) {
      const uint64_t x = i + lane < items * kKeepWaves ? counts[i + lane] : 0u;
      const uint32_t equal = (uint32_t)(x >> 32), sure = (uint32_t)x;
      const uint32_t equals = (uint32_t)sums_up_to((int)equal), sures = (uint32_t)sums_up_to((int)sure);
      if (i + lane < items * kKeepWaves) counts[i + lane] = (uint64_t)(so_far_equal + equals - equal) << 32 | (so_far_sure + sures - sure);
      so_far_equal += __builtin_amdgcn_readlane(equals, 63);
      so_far_sure += __builtin_amdgcn_readlane(sures, 63);
    }
  }
  __syncthreads();
  each([&](const int j, const uint32_t (&x)[4]) {
    const uint64_t before = counts[kKeepWaves * j + wave];
    const uint32_t own = counts_of(x), in_wave = (uint32_t)sums_up_to((int)own) - own;
    int equal_before = (int)(before >> 32) + (int)(in_wave >> 16), sure_before = (int)(uint32_t)before + (int)(in_wave & 0xffffu);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const bool equal = x[e] - lo <= hi - lo, sure = x[e] > hi;
      if (sure || (equal && equal_before < wanted)) kept[first + sure_before + min(equal_before, wanted)] = kKeepStep * j + 4 * tid + e;
      equal_before += equal;
      sure_before += sure;
    }
  });
  for (int i = tid; i < first; i += kKeepThreads) kept[i] = i;
  for (int i = tid; i < p.n_last; i += kKeepThreads) kept[p.n_keys - p.n_last + i] = end + i;
}

// A slice: so many channels of a row, 8 by a lane.
constexpr int kSlice = 32, kPieces = kSlice / 8, kWaveRows = 64 / kPieces;
// f over the lanes of a wave that have the same piece (lane % kPieces)
template <typename F>
__device__ __forceinline__ uint32_t over_rows(uint32_t x, F f) {
  if (kPieces == 4) x = f(x, dpp<kDppRor4>(x));
  x = f(x, dpp<kDppRor8>(x));
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = f(r[0], r[1]);
  const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return f(s[0], s[1]);
}

constexpr int kMoveThreads = 512, kMoveRows = kMoveThreads / kPieces;  // side by side
constexpr int kMoveEach = 256 / kMoveRows, kMoveChunk = kMoveEach * kMoveRows;   // where there are several groups, whose rows are a multiple of it

// A (sequence, KV head) and what of its rows this work-group has: a slice of keys or of values.
struct MoveSlice {
  int b, kvh;
  int64_t unit;      // its first entry of p.kept
  bool values;
  int channel;
  __device__ __forceinline__ int64_t row(const PagedEvictArgs& p, const int64_t page, const int slot) const {
    return (values ? page * p.vp_sp + kvh * p.vp_sh + slot * p.vp_sn : page * p.kp_sp + kvh * p.kp_sh + slot * p.kp_sn) + channel;
  }
};
template <int D>
__device__ __forceinline__ MoveSlice slice_of(const PagedEvictArgs& p) {
  constexpr int kSlices = D / kSlice;
  MoveSlice s;
  s.b = blockIdx.x / p.n_kv_heads;
  s.kvh = blockIdx.x - s.b * p.n_kv_heads;
  s.unit = (int64_t)blockIdx.x * p.n_keys;
  s.values = blockIdx.y >= kSlices;
  s.channel = kSlice * (blockIdx.y % kSlices) + 8 * (threadIdx.x % kPieces);
  return s;
}

// Rows that come from other groups' places, to scratch: [unit][row][keys, values][channel], and their weights.
template <int D>
__global__ void __launch_bounds__(kMoveThreads) paged_save_kernel(const PagedEvictArgs p) {
  const MoveSlice s = slice_of<D>(p);
  const uint16_t* pool = s.values ? p.values : p.keys;
  const int begin = blockIdx.z * kMoveChunk, end = min(begin + kMoveChunk, p.n_keys);
  if (p.kept[s.unit + end - 1] <= end - 1) return;  // (none moves, or nothing does)
  const int group_end = (begin / p.group_rows + 1) * p.group_rows;
#pragma unroll
  for (int j = 0; j < kMoveEach; ++j) {
    const int i = begin + kMoveRows * j + (int)(threadIdx.x / kPieces);
    if (i >= end) break;
    const int from = p.kept[s.unit + i];
    if (from < group_end || from >= p.n_keys) continue;
    const int64_t page = clamped_page(p.table[s.b * p.t_sb + (from >> p.page_log)], p.n_pages);
    const int slot = from & ((1 << p.page_log) - 1);
    *reinterpret_cast<uint4*>(p.rows + ((s.unit + i) * 2 + s.values) * D + s.channel) = *reinterpret_cast<const uint4*>(pool + s.row(p, page, slot));
    if (s.values && s.channel == 0) p.row_weights[s.unit + i] = p.weights[((page * p.n_kv_heads + s.kvh) << p.page_log) + slot];
  }
}

// The weights of a group's rows, by a work-group of its own.
__device__ __forceinline__ void move_weights(const PagedEvictArgs& p, const MoveSlice& s, const int end) {
  constexpr int kEach = 8;
  const int32_t* table = p.table + s.b * p.t_sb;
  for (int begin = blockIdx.z * p.group_rows; begin < end; begin += kEach * kMoveThreads) {
    int from[kEach], page[kEach], to[kEach];
    float w[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) from[j] = p.kept[s.unit + min(begin + kMoveThreads * j + (int)threadIdx.x, end - 1)];
    if (from[0] < 0) return;
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      page[j] = table[from[j] >> p.page_log];
      to[j] = table[min(begin + kMoveThreads * j + (int)threadIdx.x, end - 1) >> p.page_log];
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = min(begin + kMoveThreads * j + (int)threadIdx.x, end - 1);
      const float* row = p.weights + (((int64_t)clamped_page(page[j], p.n_pages) * p.n_kv_heads + s.kvh) << p.page_log) + (from[j] & ((1 << p.page_log) - 1));
      w[j] = *(from[j] >= end && from[j] < p.n_keys ? p.row_weights + s.unit + i : row);
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j) asm volatile("" : "+v"(w[j]));
    lds_barrier();
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
      const int i = begin + kMoveThreads * j + threadIdx.x;
      if (i < end && from[j] != i && (uint32_t)to[j] < (uint32_t)p.n_pages)
        p.weights[(((int64_t)to[j] * p.n_kv_heads + s.kvh) << p.page_log) + (i & ((1 << p.page_log) - 1))] = w[j];
    }
  }
}

// EACH: rows of a thread in a chunk
template <typename T, int D, int EACH>
__global__ void __launch_bounds__(kMoveThreads) paged_move_kernel(const PagedEvictArgs p) {
  constexpr int kWaves = kMoveThreads / 64, kChunk = EACH * kMoveRows;
  static_assert(kChunk % 256 == 0, "a page's rows lie in a chunk");
  constexpr int kStaged = 4096;                    // rows whose places are in LDS, a multiple of a chunk
  __shared__ uint4 red[EACH * kWaves][kPieces][2];  // bounds of kWaveRows rows each, in their order
  __shared__ int2 source[kStaged];                 // the place that a row comes from, and its page
  __shared__ int target[kStaged / 16];             // the pages that rows go to
  const MoveSlice s = slice_of<D>(p);
  uint16_t* pool = s.values ? p.values : p.keys;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, page_size = 1 << p.page_log;
  const int end = min((int)(blockIdx.z + 1) * p.group_rows, p.n_keys);
  if (blockIdx.y == 2 * D / kSlice) return move_weights(p, s, end);
  const int32_t* table = p.table + s.b * p.t_sb;
  int begin = blockIdx.z * p.group_rows;
  // what keeps its place is left alone: the chunks whose last row does, and is the last of its page
  for (; begin < end; begin += kChunk) {
    const int last = min(begin + kChunk, end) - 1, from = p.kept[s.unit + last];
    if (from < 0) return;
    if (from > last || (last + 1) % page_size != 0) break;
  }
  const int64_t row_page = s.values ? p.vp_sp : p.kp_sp, row_slot = s.values ? p.vp_sn : p.kp_sn, row_head = s.row(p, 0, 0);
  struct Chunk {
    u32x4 x[EACH];
  };
  for (; begin < end; begin += kStaged) {
    const int staged_end = min(begin + kStaged, end);
    __syncthreads();  // (the last ones have been used)
#pragma unroll
    for (int j = 0; j < kStaged / kMoveThreads; ++j) {
      const int from = p.kept[s.unit + min(begin + kMoveThreads * j + tid, end - 1)];
      source[kMoveThreads * j + tid] = int2{from, clamped_page(table[from >> p.page_log], p.n_pages)};
    }
    if (tid < kStaged / 16) target[tid] = table[min((begin >> p.page_log) + tid, (end - 1) >> p.page_log)];
    __syncthreads();
    auto load = [&](Chunk& c, const int at) __attribute__((always_inline)) {  // (behind the last row, that one)
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int i = min(at + kMoveRows * j + tid / kPieces, staged_end - 1);
        const uint64_t both = *reinterpret_cast<const uint64_t*>(&source[i - begin]);
        const int from = (int)(uint32_t)both, page = (int)(uint32_t)(both >> 32);
        const int64_t row = page * row_page + (from & (page_size - 1)) * row_slot + row_head, scratch_row = ((s.unit + i) * 2 + s.values) * D + s.channel;
        const bool saved = from >= end && from < p.n_keys;  // (from another group's places)
        c.x[j] = *reinterpret_cast<const u32x4*>((saved ? p.rows : pool) + (saved ? scratch_row : row));
      }
    };
    auto store = [&](Chunk& c, const int at) __attribute__((always_inline)) {
      // all rows of the chunk have been read when one is written
#pragma unroll
      for (int j = 0; j < EACH; ++j) asm volatile("" ::"v"(c.x[j]));
      lds_barrier();
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int i = at + kMoveRows * j + tid / kPieces;
        if (i >= staged_end) continue;
        const int page = target[(i - begin) >> p.page_log];
        if (source[i - begin].x != i && (uint32_t)page < (uint32_t)p.n_pages) *reinterpret_cast<u32x4*>(pool + page * row_page + (i & (page_size - 1)) * row_slot + row_head) = c.x[j];
      }
      if (s.values || p.bounds == nullptr) return;
#pragma unroll
      for (int j = 0; j < EACH; ++j) {
        const int i = at + kMoveRows * j + tid / kPieces;
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lo[e] = i < staged_end ? in_order(c.x[j][e]) : 0x7fff7fffu;
          hi[e] = i < staged_end ? in_order(c.x[j][e]) : 0x80008000u;
          lo[e] = over_rows(lo[e], least);
          hi[e] = over_rows(hi[e], most);
        }
        if (lane < kPieces) {
          red[kWaves * j + wave][lane][0] = uint4{lo[0], lo[1], lo[2], lo[3]};
          red[kWaves * j + wave][lane][1] = uint4{hi[0], hi[1], hi[2], hi[3]};
        }
      }
      lds_barrier();
      // kPieces lanes a page of the chunk
      const int mine = at + tid / kPieces * page_size, last = min(mine + page_size, staged_end) - 1;
      if (mine >= min(at + kChunk, staged_end) || (source[last - begin].x == last && last + 1 == mine + page_size)) return;
      const int page = target[(mine - begin) >> p.page_log], r0 = (mine - at) / kWaveRows;
      uint32_t lo[4] = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu}, hi[4] = {0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
      for (int r = r0; r < r0 + page_size / kWaveRows; ++r) {
        const uint4 l = red[r][tid % kPieces][0], h = red[r][tid % kPieces][1];
        const uint32_t ls[4] = {l.x, l.y, l.z, l.w}, hs[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          lo[e] = least(lo[e], ls[e]);
          hi[e] = most(hi[e], hs[e]);
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) bounds_back<T>(lo[e], hi[e]);
      if ((uint32_t)page >= (uint32_t)p.n_pages) return;
      uint16_t* out = p.bounds + ((int64_t)page * p.n_kv_heads + s.kvh) * 2 * D + s.channel;
      *reinterpret_cast<uint4*>(out) = uint4{lo[0], lo[1], lo[2], lo[3]};
      *reinterpret_cast<uint4*>(out + D) = uint4{hi[0], hi[1], hi[2], hi[3]};
    };
    // a chunk is requested before the last one is stored: its rows lie behind that one's places
    Chunk a, c;
    load(a, begin);
    for (int at = begin;;) {
      load(c, at + kChunk);
      store(a, at);
      if ((at += kChunk) >= staged_end) break;
      load(a, at + kChunk);
      store(c, at);
      if ((at += kChunk) >= staged_end) break;
    }
  }
}

// Rows of a group: all of them where that makes work-groups enough, one for each compute unit, or as few as make four times that (256 rows at least).  A step that gives up 64 keys of 4160, in turn
// and in groups: 1 sequence with 8 KV heads of 128 (64 slices) 39.5 and 25.4 us, 2 (128) 41.4 and 31.1 (36.7 with groups for 256), 4 (256) 44.0 and 45.9, 8 (512) 49.4 and 62.2; of
// heads of 64: 1 39.1 and 21.2, 4 (128) 41.5 and 33.5, 8 (256) 43.6 and 44.9.  232 keys of 33000: 1 with 8 of 128 256 and 99, 2 273 and 174, 4 338 and 314, 8 439 and 540.
constexpr int kMoveEnough = 256, kMoveSpread = 1024;
int paged_evict_group_rows(int batch, int n_kv_heads, int head_dim, int n_keys) {
  const int64_t slices = (int64_t)batch * n_kv_heads * 2 * (head_dim / kSlice);
  const int chunks = (n_keys + kMoveChunk - 1) / kMoveChunk;
  if (slices >= kMoveEnough) return chunks * kMoveChunk;
  const int64_t groups = std::min<int64_t>((kMoveSpread + slices - 1) / slices, chunks);
  return (int)((chunks + groups - 1) / groups) * kMoveChunk;
}

template <typename T, int D>
static hipError_t launch_paged_evict_for(PagedEvictArgs a, hipStream_t stream) {
  const int64_t most = (int64_t)a.max_pages << a.page_log;
  const dim3 units(a.batch * a.n_kv_heads);
  if (most <= kKeepHeld) hipLaunchKernelGGL(paged_keep_kernel<true>, units, dim3(kKeepThreads), 0, stream, a);
  else hipLaunchKernelGGL(paged_keep_kernel<false>, units, dim3(kKeepThreads), 0, stream, a);
  if (most <= a.above) return hipGetLastError();  // (no sequence is longer than its table)
  a.group_rows = paged_evict_group_rows(a.batch, a.n_kv_heads, D, a.n_keys);
  const int groups = (a.n_keys + a.group_rows - 1) / a.group_rows;
  if (groups > 1) hipLaunchKernelGGL((paged_save_kernel<D>), dim3(units.x, 2 * D / kSlice, (a.n_keys + kMoveChunk - 1) / kMoveChunk), dim3(kMoveThreads), 0, stream, a);
  const dim3 grid(units.x, 2 * D / kSlice + 1, groups);
  if (groups > 1) hipLaunchKernelGGL((paged_move_kernel<T, D, kMoveEach>), grid, dim3(kMoveThreads), 0, stream, a);
  else hipLaunchKernelGGL((paged_move_kernel<T, D, 2 * kMoveEach>), grid, dim3(kMoveThreads), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_paged_evict(const PagedEvictArgs& a, hipStream_t stream) {
  if (a.head_dim == 128) return a.dtype == 0 ? launch_paged_evict_for<Bf16, 128>(a, stream) : launch_paged_evict_for<F16, 128>(a, stream);
  return a.dtype == 0 ? launch_paged_evict_for<Bf16, 64>(a, stream) : launch_paged_evict_for<F16, 64>(a, stream);
}

}  // namespace aa
