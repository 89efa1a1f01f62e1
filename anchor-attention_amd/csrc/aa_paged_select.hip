// Which pages of a cache a sparse decode step reads, on gfx950: the scores of the pages' bounds and the largest of them.
//
// A score is defined by a float64 sum, so that the chosen pages do not depend on its order: products of two 16-bit numbers are exact (in float32 those of fp16 and nearly all of
// bf16), their sum is formed in float64 and rounded once.  A lane has 8 channels of 4 pages, so a page is 8 or 16 lanes'; their sums are exchanged inside rows of
// lanes so that each lane ends with one page's.  With many pages conversions and additions in float64 bound it: 16 sequences of 6000 to 60000 keys in pages of 16,
// 32/8 heads of 64, fp16 17.5 us for 49 MB of bounds, which take 9.4 to read; one sequence of 131072 keys in pages of 64, 32/8 of 128 5.8 us, 8 MB.  (Choosing the head that
// counts by sums in float32 and summing only that one's in float64 where no other is near was slower, 23 and 6.4 us against 18.5 and 5.7: twice the exchanges between lanes, and a
// wave nearly always has a page where two heads are near.  So were bounds kept in float64, two products with the positive and the negative part of a query, 21: 200
// registers leave two waves to a SIMD.)
//
// Choosing is latency (6.0 us for 2048 pages of one sequence, 7.5 for 8192, 18 for 25000; 8.5 with the scores, for 132 pages): a work-group per (sequence, KV head)
// finds what the wanted number of scores reaches by histograms of 256 equal ranges of the numbers' order, each inside the range of the last one that holds it; the
// first spans the smallest to the largest score, so that two or three do, whatever the scores' exponents (at most four).  Every wave reads the bins for itself,
// which leaves one barrier for each histogram.  Integer work: the order in which counts are added does not matter.  The code is kept short, since most of it runs
// once and its first instructions come from memory.
#include "aa_kernels.h"
#include "aa_paged.h"

namespace aa {

// Pages of a lane: several share a head's queries and their sums' exchange, one leaves a wave soonest.
// (1 in the scores' launch: the 16 sequences above 46.2 us a step instead of 43.1.)
constexpr int kAbreast = 4, kAbreastFused = 1;
constexpr int kChooseThreads = 1024, kChooseWaves = kChooseThreads / 64;
constexpr int kFused = 1024;       // a table of at most that many pages is scored and chosen from by one launch
// ... if one work-group does that sooner than a launch of its own starts.  It takes pages * D * (heads of the group + kPerPage): a page's bounds cost as much to
// fetch and convert as the products of twelve heads.  Steps of one sequence, bf16, pages of 16, by one launch and by two: 32/8 heads of 128, 96 pages 17.8 and 19.3 us, 128
// 19.5 and 19.3; 28/4 of 128, 96 pages 19.0 and 19.5, 128 21.8 and 20.3; 32/8 of 64, 192 pages 16.6 and 18.4, 256 17.9 and 18.2; 14/2 of 64, 192 pages 17.6 and 18.6,
// 256 20.1 and 18.9.  16 sequences, and fp16, the same within 5 %.  Where the units fill the CUs, scores by themselves are no more side by side than with the choosing: 64
// sequences, 32/8 of 128, 192 pages 44.3 and 45.3, 256 48.5 and 48.4; 28/4 of 128, 192 pages 32.2 and 32.4, 256 36.0 and 35.1; 32/8 of 64, 384 pages 34.5 and 36.0.
constexpr int kPerPage = 12, kFusedWork = 256 * 1024, kFusedWorkMany = 460 * 1024, kManyUnits = 256;
constexpr int kInLds = 32768;      // the scores of at most that many pages are kept in LDS
// Pages that a thread of the choosing work-group looks at together, side by side: 4, and 1 in tables of at most kOnes pages, where the other threads would have
// nothing to do.  (Steps of one sequence, 32/8 heads of 128: 8192 pages one 34.6 us, four 29.8; 1875 pages the same, 469 20.5 and 21.5.)
constexpr int kItem = 4, kOnes = 2048;
// ITEM numbers from p on
template <int ITEM, typename X>
__device__ __forceinline__ void load_item(const X* p, X (&x)[ITEM]) {
  typedef X four __attribute__((ext_vector_type(4)));
  if constexpr (ITEM == 4) {
    const four y = *reinterpret_cast<const four*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = y[e];
  } else {
    x[0] = *p;
  }
}
constexpr int kMostPages = 1 << 16;
constexpr int kListed = 1024;      // the chosen pages up to that many pass through LDS
constexpr int kQueryWords = 4096;  // of LDS for a group's queries; those of more heads are read from memory

// Scores are compared as ordered() numbers them, from 1 to below kEnd - 1.
constexpr uint32_t kEnd = 0xffffffffu;  // what stands for pages that are taken in any case; 0 stands for no page

// Bounds of 8 channels of N pages, and sums of their products with queries in float64.
//
// WIDE: products in float64 too.  bf16 has the exponents of float32, in which a product may overflow, or lose bits below 2^-126; those of fp16 do not.  bf16 products are
// formed in float32 all the same, which is sooner (32/8 heads of 64, 256 pages scored and chosen from in one launch 17.5 us a step instead of 18.1), and once more
// in float64 where the sum shows that this may have counted: one that overflowed leaves an infinity or NaN, and 128 that lost 2^-150 each are off by
// 2^-143, less than a float64 sum's own rounding of what is 2^-80 or larger.
template <typename T, int N, bool WIDE = false>
struct Products {
  static constexpr bool kMayLeave = !WIDE;  // float32
  float bounds[N][2][8];
  static __device__ __forceinline__ u32x4 query(const u32x4 q) { return q; }  // as it is staged
  __device__ __forceinline__ explicit Products(const u32x4 (&raw)[N][2]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int w = 0; w < 2; ++w) unpack8<T>(*reinterpret_cast<const uint4*>(&raw[i][w]), bounds[i][w]);
  }
  __device__ __forceinline__ void add(double (&sum)[N], const u32x4 raw) const {
    float q[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(&raw), q);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool larger = q[j] >= 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float x = larger ? bounds[i][1][j] : bounds[i][0][j];
        if constexpr (WIDE) sum[i] = __builtin_fma((double)q[j], (double)x, sum[i]);
        else sum[i] += (double)(q[j] * x);
      }
    }
  }
};
// A product of two fp16 numbers is exact in float32; an instruction multiplies two of them into one, and two bounds are chosen at once by their queries' signs, for which -0 becomes 0
// (16 sequences of 6000 to 60000 keys in pages of 16: 43.0 us a step, with conversions as in bf16 44.7).
template <int N>
struct Products<F16, N, false> {
  static constexpr bool kMayLeave = false;
  u32x4 bounds[N][2];
  static __device__ __forceinline__ u32x4 query(u32x4 q) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((q[i] & 0xffffu) == 0x8000u) q[i] &= 0xffff0000u;
      if (q[i] >> 16 == 0x8000u) q[i] &= 0xffffu;
    }
    return q;
  }
  __device__ __forceinline__ explicit Products(const u32x4 (&raw)[N][2]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int w = 0; w < 2; ++w) bounds[i][w] = raw[i][w];
  }
  __device__ __forceinline__ void add(double (&sum)[N], const u32x4 raw) const {
    typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
    typedef _Float16 pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t both = raw[j];
      const i16x2 signs = *reinterpret_cast<const i16x2*>(&both) >> 15;
      const uint32_t smaller = *reinterpret_cast<const uint32_t*>(&signs);
      const pair q = *reinterpret_cast<const pair*>(&both);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t chosen = (bounds[i][0][j] & smaller) | (bounds[i][1][j] & ~smaller);
        const pair x = *reinterpret_cast<const pair*>(&chosen);
        sum[i] += (double)__builtin_fmaf((float)q[0], (float)x[0], 0.f);
        sum[i] += (double)__builtin_fmaf((float)q[1], (float)x[1], 0.f);
      }
    }
  }
};

// The scores of kPages consecutive pages of a sequence by one wave, N by each lane.
template <typename T, int D, int N>
struct Scores {
  static constexpr int kLanes = D / 8, kSide = 64 / kLanes, kPages = kSide * N;
  static_assert(N == 4 || N == 1, "what the exchange is written for");
  struct Pages {  // of the pool
    int at[N];
  };
  static __device__ __forceinline__ Pages find(const PagedSelectArgs& p, const int b, const int first) {
    const int32_t* table = p.table + b * p.t_sb;
    Pages x;
#pragma unroll
    for (int i = 0; i < N; ++i) x.at[i] = table[min(first + kSide * i + (int)(threadIdx.x & 63) / kLanes, p.max_pages - 1)];
    return x;
  }
  struct Bounds {
    u32x4 raw[N][2];
  };
  static __device__ __forceinline__ Bounds load(const PagedSelectArgs& p, const int kvh, const Pages& x) {
    Bounds y;
#pragma unroll
    for (int i = 0; i < N; ++i) {  // (behind the last page the table holds anything)
      const uint16_t* lo = p.bounds + ((int64_t)clamped_page(x.at[i], p.n_pages) * p.n_kv_heads + kvh) * 2 * D + 8 * (threadIdx.x % kLanes);
      y.raw[i][0] = *reinterpret_cast<const u32x4*>(lo);
      y.raw[i][1] = *reinterpret_cast<const u32x4*>(lo + D);
    }
    return y;
  }
  // `staged`: the group's queries one after the other (as many as stage() has room for); `count`: of the pages there are; store(k, score) is called by one lane for each page,
  // 0 <= k < kPages
  template <typename Store>
  static __device__ __forceinline__ void form(const PagedSelectArgs& p, const int b, const int kvh, const Bounds& y, const uint32_t* staged, const int room, const int count,
                                              Store store) {
    const int lane = threadIdx.x & 63, c = lane % kLanes, group = p.n_q_heads / p.n_kv_heads;
    const uint16_t* qp = p.q + b * p.q_sb + (int64_t)kvh * group * p.q_sh + 8 * c;
    auto query = [&](const int h) {
      if (h < room) return *reinterpret_cast<const u32x4*>(staged + h * (D / 2) + 4 * c);
      return Products<T, N>::query(__builtin_nontemporal_load(reinterpret_cast<const u32x4*>(qp + h * p.q_sh)));
    };
    // bits of a lane that say which of its pages it ends with: the same in the lane that is mirrored in 8
    const bool odd = (kLanes == 8 ? lane ^ lane >> 2 : lane) & 1, odd2 = (kLanes == 8 ? lane ^ lane >> 1 : lane) & 2;
    const int mine = kSide * (N == 4 ? (odd ? 2 : 0) + (odd2 ? 1 : 0) : 0) + lane / kLanes;
    float best;
    bool nan, unsure;
    auto over_heads = [&](const auto products) __attribute__((always_inline)) {
      best = -INFINITY;
      nan = unsure = false;
      u32x4 next = query(0);
#pragma nounroll
      for (int h = 1; h <= group; ++h) {
        const u32x4 q = next;
        next = query(min(h, group - 1));
        double sum[N] = {};
        products.add(sum, q);
        double s;
        if constexpr (N == 4) {  // twice a lane keeps the half of what it has that a bit of it names, and gives the other away
          const double a = (odd ? sum[2] : sum[0]) + dpp<kDppXor1>(odd ? sum[0] : sum[2]);
          const double b = (odd ? sum[3] : sum[1]) + dpp<kDppXor1>(odd ? sum[1] : sum[3]);
          s = (odd2 ? b : a) + dpp<kDppXor2>(odd2 ? a : b);
        } else {
          s = sum[0] + dpp<kDppXor1>(sum[0]);
          s += dpp<kDppXor2>(s);
        }
        if (kLanes == 8) {
          s += dpp<kDppHalfMirror>(s);
        } else {
          s += dpp<kDppRor8>(s);
          s += dpp<kDppRor4>(s);
        }
        nan = nan || s != s;
        best = fmaxf(best, (float)s);
        if constexpr (products.kMayLeave) {  // (by its exponent: below -80, or that of infinities and NaN)
          const uint32_t exponent = (uint32_t)__double2hiint(s) >> 20 & 0x7ffu;
          unsure = unsure || exponent - (1023u - 80u) >= 2047u - (1023u - 80u);
        }
      }
    };
    over_heads(Products<T, N>(y.raw));
    if constexpr (Products<T, N>::kMayLeave)
      if (__builtin_expect(__any(unsure && mine < count), 0)) over_heads(Products<T, N, true>(y.raw));
    if (c < (N == 4 ? 4 : 1)) store(mine, nan ? INFINITY : best);
  }
};

// A group's queries to LDS by some threads, so that no head waits for memory; for how many heads there is room.
template <typename T, int D>
__device__ __forceinline__ int stage_queries(const PagedSelectArgs& p, const int b, const int kvh, uint32_t* staged, const int words, const int thread, const int threads) {
  const int group = p.n_q_heads / p.n_kv_heads, room = min(group, words / (D / 2));
  for (int i = thread; i < room * (D / 8); i += threads)
    reinterpret_cast<u32x4*>(staged)[i] =
        Products<T, 1>::query(*reinterpret_cast<const u32x4*>(p.q + b * p.q_sb + (int64_t)(kvh * group + i / (D / 8)) * p.q_sh + 8 * (i % (D / 8))));
  return room;
}

// A work-group's waves have neighbouring KV heads, whose bounds lie side by side, of the same pages of a sequence.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_scores_kernel(const PagedSelectArgs p) {
  typedef Scores<T, D, kAbreast> S;
  __shared__ __attribute__((aligned(16))) uint32_t staged[4][kQueryWords / 4];
  const int b = blockIdx.z, step = gridDim.x * S::kPages, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kvh = min((int)(4 * blockIdx.y) + wave, p.n_kv_heads - 1);  // (a wave without one does the last one's once more)
  int first = blockIdx.x * S::kPages;
  typename S::Pages at = S::find(p, b, first);
  const int there = pages_of(clamped_length(p.lengths, b, p.max_pages, p.page_log), p.page_log);
  if (there <= p.n_chosen || first >= there) return;
  typename S::Bounds y = S::load(p, kvh, at);
  const int room = stage_queries<T, D>(p, b, kvh, staged[wave], kQueryWords / 4, threadIdx.x & 63, 64);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (read by the same wave only)
  __builtin_amdgcn_wave_barrier();
  at = S::find(p, b, first + step);
  float* scores = p.scores + ((int64_t)b * p.n_kv_heads + kvh) * paged_score_pitch(p.max_pages);
  for (;;) {
    S::form(p, b, kvh, y, staged[wave], room, there - first, [&](const int k, const float x) {
      if (first + k < there) scores[first + k] = x;
    });
    first += step;
    if (first >= there) return;
    y = S::load(p, kvh, at);
    at = S::find(p, b, first + step);
  }
}

// FROM: 0 the scores are formed here, 1 they are read once, 2 as often as they are needed (more than LDS is to hold).  ITEM: pages of a thread, side by side
template <typename T, int D, int FROM, int ITEM>
__global__ void __launch_bounds__(kChooseThreads) paged_choose_kernel(const PagedSelectArgs p) {
  typedef Scores<T, D, kAbreastFused> S;
  constexpr int kMostItems = (FROM == 0 ? kFused : FROM == 2 ? kMostPages : ITEM == 1 ? kOnes : kInLds) / (ITEM * kChooseThreads);
  extern __shared__ __attribute__((aligned(16))) uint32_t kept[];  // (not where they stay in memory)
  __shared__ uint32_t bins[4][256], ranges[2][kChooseWaves], counts[kMostItems * kChooseWaves], before[kMostItems * kChooseWaves];
  const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t unit = (int64_t)b * p.n_kv_heads + kvh;
  const float* scores = p.scores + unit * paged_score_pitch(p.max_pages);
  int32_t* pages = p.pages + unit * p.n_chosen;
  int32_t* chosen = p.chosen + unit * p.n_chosen;
  const int32_t* table = p.table + b * p.t_sb;
  __shared__ __attribute__((aligned(16))) uint32_t staged[FROM == 0 ? kQueryWords : 1];
  __shared__ int list[kListed];
  // (what does not depend on the length is requested before it is known)
  float early[2][ITEM] = {};
  typename S::Pages at;
  int room = 0;
  if (FROM == 0) {
    at = S::find(p, b, wave * S::kPages);
    room = stage_queries<T, D>(p, b, kvh, staged, kQueryWords, tid, kChooseThreads);
  } else {
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (ITEM * (kChooseThreads * j + tid) < p.max_pages) load_item(scores + ITEM * (kChooseThreads * j + tid), early[j]);
  }
  const int there = pages_of(clamped_length(p.lengths, b, p.max_pages, p.page_log), p.page_log);
  if (there <= p.n_chosen) {
    for (int i = tid; i < p.n_chosen; i += kChooseThreads) {
      pages[i] = i < there ? i : -1;
      chosen[i] = i < there ? table[i] : 0;
    }
    return;
  }
  const int first = p.n_first, last = there - p.n_last;  // the pages to choose from
  auto number = [&](const int i, const float score) { return i >= there ? 0u : i < first || i >= last ? kEnd : ordered(score); };
  if (FROM == 0) {
    typename S::Bounds y = S::load(p, kvh, at);
    __syncthreads();
#pragma nounroll
    for (int i = wave * S::kPages; i < there;) {
      S::form(p, b, kvh, y, staged, room, there - i, [&](const int k, const float x) {
        if (i + k < there) kept[i + k] = number(i + k, x);
      });
      i += kChooseWaves * S::kPages;
      if (i < there) y = S::load(p, kvh, S::find(p, b, i));
    }
  }
  // item j of a thread is ITEM pages from place(j) on
  const int items = (there + ITEM * kChooseThreads - 1) / (ITEM * kChooseThreads);
  auto place = [&](const int j) { return ITEM * (kChooseThreads * j + tid); };
  if (FROM == 1) {
    for (int j = 0; j < items; ++j) {
      const int i = place(j);
      if (i >= there) break;
      float x[ITEM];
      if (j > 1) load_item(scores + i, x);
#pragma unroll
      for (int e = 0; e < ITEM; ++e) kept[i + e] = number(i + e, j == 0 ? early[0][e] : j == 1 ? early[1][e] : x[e]);
    }
  }
#pragma unroll
  for (int i = 0; i < 4 * 256; i += kChooseThreads) bins[0][i + tid] = 0u;
  if (FROM == 0) __syncthreads();

  auto each = [&](auto&& f) {  // f(j, numbers)
#pragma nounroll
    for (int j = 0; j < items; ++j) {
      const int i = place(j);
      uint32_t x[ITEM] = {};
      if (i < there) {
        if constexpr (FROM < 2) {
          load_item(kept + i, x);
        } else {
          float y[ITEM];
          load_item(scores + i, y);
#pragma unroll
          for (int e = 0; e < ITEM; ++e) x[e] = number(i + e, y[e]);
        }
      }
      f(j, x);
    }
  };

  uint32_t lo = kEnd - 1u, hi = kEnd - 1u;  // (no score has them)
  int wanted = p.n_chosen - p.n_first - p.n_last;
  if (wanted > 0) {
    lo = kEnd;
    hi = 0u;
    each([&](const int, const uint32_t (&x)[ITEM]) {
#pragma unroll
      for (int e = 0; e < ITEM; ++e) {
        lo = min(lo, x[e] - 1u);  // (0 becomes the largest, kEnd the one below)
        hi = max(hi, x[e] + 1u);  // (kEnd becomes 0)
      }
    });
    lo = up_to(lo, 0xffffffffu, [](const uint32_t a, const uint32_t b) { return min(a, b); });
    hi = up_to(hi, 0u, [](const uint32_t a, const uint32_t b) { return max(a, b); });
    if (lane == 63) {
      ranges[0][wave] = lo;
      ranges[1][wave] = hi;
    }
    __syncthreads();  // (the bins are 0 too)
    lo = ranges[0][0];
    hi = ranges[1][0];
#pragma unroll
    for (int w = 1; w < kChooseWaves; ++w) {
      lo = min(lo, ranges[0][w]);
      hi = max(hi, ranges[1][w]);
    }
    lo = __builtin_amdgcn_readfirstlane(lo) + 1u;
    hi = __builtin_amdgcn_readfirstlane(hi) - 1u;
    // The wanted-th largest score lies from lo to hi; all of those above are taken.  A range is 2^32 long at most and the next one a 256th, so four do.
#pragma nounroll
    for (int round = 0;; ++round) {
      const uint32_t span = hi - lo;
      const int shift = span < 256u ? 0 : 24 - __builtin_clz(span);  // span >> shift < 256
      each([&](const int, const uint32_t (&x)[ITEM]) {
#pragma unroll
        for (int e = 0; e < ITEM; ++e)
          if (x[e] - lo <= span) atomicAdd(&bins[round][(x[e] - lo) >> shift], 1u);
      });
      __syncthreads();
      const uint4 bin4 = *reinterpret_cast<const uint4*>(&bins[round][4 * lane]);
      const int n[4] = {(int)bin4.x, (int)bin4.y, (int)bin4.z, (int)bin4.w};
      const int own = n[0] + n[1] + n[2] + n[3], sums = sums_up_to(own), all = __builtin_amdgcn_readlane(sums, 63);
      // the last lane that has `wanted` scores in its bins or behind them, and the last of its bins that has
      const int at = 63 - __builtin_clzll(__ballot(all - sums + own >= wanted));
      int above = __builtin_amdgcn_readlane(all - sums, at), in_bin = 0, bin = 4 * at;
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        in_bin = __builtin_amdgcn_readlane(n[j], at);
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
  }

  // Scores above hi are taken, and of those from lo to hi the first `wanted`: counted by item and wave, which is the pages' order.
  auto counts_of = [&](const uint32_t (&x)[ITEM]) {  // of an item, in the upper and the lower half
    uint32_t packed = 0;
#pragma unroll
    for (int e = 0; e < ITEM; ++e) packed += (x[e] - lo <= hi - lo ? 0x10000u : 0u) + (x[e] > hi ? 1u : 0u);
    return packed;
  };
  each([&](const int j, const uint32_t (&x)[ITEM]) {
    const uint32_t all = sums_up_to(counts_of(x));
    if (lane == 63) counts[kChooseWaves * j + wave] = all;
  });
  __syncthreads();
  uint32_t so_far_equal = 0, so_far_sure = 0;
#pragma nounroll
  for (int i = 0; i < items * kChooseWaves; i += 64) {  // (each wave for itself, all with the same result)
    const uint32_t x = i + lane < items * kChooseWaves ? counts[i + lane] : 0u, equal = x >> 16, sure = x & 0xffffu;
    const uint32_t equals = sums_up_to(equal), sures = sums_up_to(sure);
    if (i + lane < items * kChooseWaves) before[i + lane] = (so_far_equal + equals - equal) << 16 | (so_far_sure + sures - sure);
    so_far_equal += __builtin_amdgcn_readlane(equals, 63);
    so_far_sure += __builtin_amdgcn_readlane(sures, 63);
  }
  each([&](const int j, const uint32_t (&x)[ITEM]) {
    const uint32_t packed = before[kChooseWaves * j + wave], own = counts_of(x), in_wave = sums_up_to(own) - own;
    int equal_before = (packed >> 16) + (in_wave >> 16), sure_before = (packed & 0xffffu) + (in_wave & 0xffffu);
#pragma unroll
    for (int e = 0; e < ITEM; ++e) {
      const bool equal = x[e] - lo <= hi - lo, sure = x[e] > hi;
      if (sure || (equal && equal_before < wanted)) {
        const int to = sure_before + min(equal_before, wanted);
        if (to < kListed) list[to] = place(j) + e;
        else pages[to] = place(j) + e;
      }
      equal_before += equal;
      sure_before += sure;
    }
  });
  __syncthreads();  // (the list is complete: its pages of the pool are read side by side)
  for (int i = tid; i < p.n_chosen; i += kChooseThreads) {
    const int page = i < kListed ? list[i] : pages[i];
    if (i < kListed) pages[i] = page;
    chosen[i] = table[page];
  }
}

template <typename T, int D>
static void launch_paged_select_for(const PagedSelectArgs& a, hipStream_t stream) {
  const dim3 units(a.n_kv_heads, a.batch);
  const int64_t work = (int64_t)a.max_pages * D * (a.n_q_heads / a.n_kv_heads + kPerPage);
  if (a.max_pages <= kFused && work <= ((int64_t)a.batch * a.n_kv_heads < kManyUnits ? kFusedWork : kFusedWorkMany)) {
    hipLaunchKernelGGL((paged_choose_kernel<T, D, 0, 1>), units, dim3(kChooseThreads), 4 * paged_score_pitch(a.max_pages), stream, a);
    return;
  }
  // (some four thousand work-groups, however long the table is and however short the sequences: the step above 43.1 us, with 2560 43.6, with 1024 46.5)
  const int chunks = (a.max_pages + Scores<T, D, kAbreast>::kPages - 1) / Scores<T, D, kAbreast>::kPages, fours = (a.n_kv_heads + 3) / 4;
  const int64_t n = (int64_t)fours * a.batch;
  const int side = (int)((4096 + n - 1) / n);
  hipLaunchKernelGGL((paged_scores_kernel<T, D>), dim3(chunks < side ? chunks : side, fours, a.batch), dim3(256), 0, stream, a);
  const size_t lds = 4 * paged_score_pitch(a.max_pages);
  if (a.max_pages <= kOnes) hipLaunchKernelGGL((paged_choose_kernel<T, D, 1, 1>), units, dim3(kChooseThreads), lds, stream, a);
  else if (a.max_pages <= kInLds) hipLaunchKernelGGL((paged_choose_kernel<T, D, 1, kItem>), units, dim3(kChooseThreads), lds, stream, a);
  else hipLaunchKernelGGL((paged_choose_kernel<T, D, 2, kItem>), units, dim3(kChooseThreads), 0, stream, a);
}

hipError_t launch_paged_select(const PagedSelectArgs& a, hipStream_t stream) {
  if (a.head_dim == 128) {
    if (a.dtype == 0) launch_paged_select_for<Bf16, 128>(a, stream);
    else launch_paged_select_for<F16, 128>(a, stream);
  } else {
    if (a.dtype == 0) launch_paged_select_for<Bf16, 64>(a, stream);
    else launch_paged_select_for<F16, 64>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace aa
