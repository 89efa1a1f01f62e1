// Which pages of a cache a sparse decode step reads, on gfx950: the scores of the pages' bounds and the largest of them.
//
// The scores are bound by reading the bounds once.  Products of two 16-bit numbers are exact in float32; their sum is
// formed in float64 and rounded once, so that the chosen pages do not depend on its order.  A lane has 8 channels of 4 pages, so a page is 8 or 16
// lanes'; their sums are exchanged inside rows of lanes so that each lane ends with one page's.
//
// Choosing is latency: a work-group per (sequence, KV head) finds the wanted-th largest score by histograms of 256 equal ranges of the numbers' order, each
// inside the range of the last one that holds it; the first spans the smallest to the largest score, so that two or three do, whatever the
// scores' exponents (at most five).  A thread's scores stay in its registers, and every wave reads the bins for itself, which leaves one barrier for
// each histogram.  Integer work: the order in which counts are added does not matter.
#include "aa_kernels.h"
#include "aa_paged.h"

namespace aa {

constexpr int kAbreast = 4;        // pages of a lane
constexpr int kChooseThreads = 512;
constexpr int kChooseWaves = kChooseThreads / 64;
constexpr int kFused = 1024;       // a table of at most that many pages is scored and chosen from by one launch
constexpr int kInRegisters = 8192; // the scores of at most that many pages are kept in registers
constexpr int kMostPages = 1 << 16;

// A score as an unsigned number of the same order, from 1 on; NaN as infinity, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
  x = x != x ? INFINITY : x + 0.f;
  const uint32_t u = __float_as_uint(x);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// The scores of kPages consecutive pages of a sequence by one wave.
template <typename T, int D>
struct Scores {
  static constexpr int kLanes = D / 8, kSide = 64 / kLanes, kPages = kSide * kAbreast;
  struct Pages {  // of the pool
    int at[kAbreast];
  };
  struct Bounds {
    uint4 raw[kAbreast][2];
  };
  static __device__ __forceinline__ Pages find(const PagedSelectArgs& p, const int b, const int first) {
    const int32_t* table = p.table + b * p.t_sb;
    Pages x;
#pragma unroll
    for (int i = 0; i < kAbreast; ++i) x.at[i] = table[min(first + kSide * i + (int)(threadIdx.x & 63) / kLanes, p.max_pages - 1)];
    return x;
  }
  static __device__ __forceinline__ Bounds load(const PagedSelectArgs& p, const int kvh, const Pages& x) {
    Bounds y;
#pragma unroll
    for (int i = 0; i < kAbreast; ++i) {  // (behind the last page the table holds anything)
      const uint16_t* lo = p.bounds + ((int64_t)clamped_page(x.at[i], p.n_pages) * p.n_kv_heads + kvh) * 2 * D + 8 * (threadIdx.x % kLanes);
      y.raw[i][0] = *reinterpret_cast<const uint4*>(lo);
      y.raw[i][1] = *reinterpret_cast<const uint4*>(lo + D);
    }
    return y;
  }
  // store(place, score) is called by one lane for each page, 0 <= place < kPages
  template <typename Store>
  static __device__ __forceinline__ void form(const PagedSelectArgs& p, const int b, const int kvh, const Bounds& y, Store store) {
    const int lane = threadIdx.x & 63, c = lane % kLanes, side = lane / kLanes, group = p.n_q_heads / p.n_kv_heads;
    const uint16_t* qp = p.q + b * p.q_sb + (int64_t)kvh * group * p.q_sh + 8 * c;
    uint4 q_raw = *reinterpret_cast<const uint4*>(qp);
    float bounds[kAbreast][2][8];
#pragma unroll
    for (int i = 0; i < kAbreast; ++i)
#pragma unroll
      for (int w = 0; w < 2; ++w) unpack8<T>(y.raw[i][w], bounds[i][w]);
    const bool odd = lane & 1, odd2 = lane & 2;
    float best = -INFINITY;
    bool nan = false;
    for (int h = 0; h < group; ++h) {
      float q[8];
      unpack8<T>(q_raw, q);
      if (h + 1 < group) q_raw = *reinterpret_cast<const uint4*>(qp + (h + 1) * p.q_sh);
      double sum[kAbreast];
#pragma unroll
      for (int i = 0; i < kAbreast; ++i) sum[i] = 0.0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool larger = q[j] >= 0.f;
#pragma unroll
        for (int i = 0; i < kAbreast; ++i) sum[i] += (double)(q[j] * (larger ? bounds[i][1][j] : bounds[i][0][j]));
      }
      if (kLanes == 8) {  // (a lane and the one mirrored in their 8 then hold the same, and 4 neighbours all parts)
#pragma unroll
        for (int i = 0; i < kAbreast; ++i) sum[i] += dpp<kDppHalfMirror>(sum[i]);
      }
      // a lane keeps the half of the sums that its bit names and gives the other half away
      double a = odd ? sum[2] : sum[0], a2 = odd ? sum[3] : sum[1];
      a += dpp<kDppXor1>(odd ? sum[0] : sum[2]);
      a2 += dpp<kDppXor1>(odd ? sum[1] : sum[3]);
      double s = odd2 ? a2 : a;
      s += dpp<kDppXor2>(odd2 ? a : a2);
      if (kLanes == 16) {
        s += dpp<kDppRor8>(s);
        s += dpp<kDppRor4>(s);
      }
      nan = nan || s != s;
      best = fmaxf(best, (float)s);
    }
    if (c < 4) store(kSide * ((odd ? 2 : 0) + (odd2 ? 1 : 0)) + side, nan ? INFINITY : best);
  }
};

// A work-group's waves take every so many pages of a (KV head, sequence); the next pages' bounds are on the way meanwhile.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_scores_kernel(const PagedSelectArgs p) {
  typedef Scores<T, D> S;
  const int kvh = blockIdx.y, b = blockIdx.z, step = 4 * gridDim.x * S::kPages;
  int first = (4 * blockIdx.x + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * S::kPages;
  typename S::Pages at = S::find(p, b, first);
  const int there = pages_of(clamped_length(p.lengths, b, p.max_pages, p.page_log), p.page_log);
  if (there <= p.n_chosen || first >= there) return;
  typename S::Bounds y = S::load(p, kvh, at);
  at = S::find(p, b, first + step);
  float* scores = p.scores + ((int64_t)b * p.n_kv_heads + kvh) * p.max_pages;
  for (; first < there; first += step) {
    const typename S::Bounds now = y;
    if (first + step < there) {
      y = S::load(p, kvh, at);
      at = S::find(p, b, first + 2 * step);
    }
    S::form(p, b, kvh, now, [&](const int place, const float x) {
      if (first + place < there) scores[first + place] = x;
    });
  }
}

// FUSED: the scores are formed here.  ITEMS: of a thread, kept in registers; 0: read from memory as often as they are needed.
template <typename T, int D, bool FUSED, int ITEMS>
__global__ void __launch_bounds__(kChooseThreads) paged_choose_kernel(const PagedSelectArgs p) {
  constexpr int kMostItems = ITEMS ? ITEMS : kMostPages / kChooseThreads;
  __shared__ float formed[FUSED ? kFused : 1];
  __shared__ uint32_t bins[5][256], ranges[2][kChooseWaves], counts[kMostItems * kChooseWaves], before[kMostItems * kChooseWaves];
  const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t unit = (int64_t)b * p.n_kv_heads + kvh;
  const float* scores = p.scores + unit * p.max_pages;
  int32_t* pages = p.pages + unit * p.n_chosen;
  int32_t* chosen = p.chosen + unit * p.n_chosen;
  const int32_t* table = p.table + b * p.t_sb;
  const int there = pages_of(clamped_length(p.lengths, b, p.max_pages, p.page_log), p.page_log);
  if (there <= p.n_chosen) {
    for (int i = tid; i < p.n_chosen; i += kChooseThreads) {
      pages[i] = i < there ? i : -1;
      chosen[i] = i < there ? table[i] : 0;
    }
    return;
  }
  if (FUSED) {
    typedef Scores<T, D> S;
    for (int i = wave * S::kPages; i < there; i += kChooseWaves * S::kPages)
      S::form(p, b, kvh, S::load(p, kvh, S::find(p, b, i)), [&](const int place, const float x) {
        if (i + place < kFused) formed[i + place] = x;
      });
  }
  for (int i = tid; i < 5 * 256; i += kChooseThreads) bins[0][i] = 0u;
  if (FUSED) __syncthreads();
  // item j of a thread is page 512 j + tid; of those to choose from a number from 1 on, else 0
  const int first = p.n_first, last = there - p.n_last, items = (there + kChooseThreads - 1) / kChooseThreads;
  auto read = [&](const int j) {
    const int i = kChooseThreads * j + tid;
    return i >= first && i < last ? ordered(FUSED ? formed[i] : scores[i]) : 0u;
  };
  uint32_t item[ITEMS ? ITEMS : 1];
  if (ITEMS) {
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) item[j] = j < items ? read(j) : 0u;
  }
  auto each = [&](auto&& f) {  // f(j, item)
    if (ITEMS) {
#pragma unroll
      for (int j = 0; j < ITEMS; ++j)
        if (j < items) f(j, item[j]);
    } else {
      for (int j = 0; j < items; ++j) f(j, read(j));
    }
  };

  int wanted = p.n_chosen - p.n_first - p.n_last;
  uint32_t lo = 0xffffffffu, hi = 0u;
  each([&](const int j, const uint32_t x) {
    lo = x ? min(lo, x) : lo;
    hi = max(hi, x);
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
  lo = __builtin_amdgcn_readfirstlane(lo);
  hi = __builtin_amdgcn_readfirstlane(hi);
  if (wanted == 0) lo = hi = 0xffffffffu;  // (no score reaches them)
  // The wanted-th largest score lies from lo to hi; all of those above are taken.  A range is 2^32 long at most and the next one a 256th, so five do.
  for (int round = 0; wanted > 0; ++round) {
    const uint32_t span = hi - lo;
    const int shift = span < 256u ? 0 : 24 - __builtin_clz(span);  // span >> shift < 256
    each([&](const int j, const uint32_t x) {
      if (x >= lo && x <= hi) atomicAdd(&bins[round][(x - lo) >> shift], 1u);
    });
    __syncthreads();
    const uint4 bin4 = *reinterpret_cast<const uint4*>(&bins[round][4 * lane]);
    const int n[4] = {(int)bin4.x, (int)bin4.y, (int)bin4.z, (int)bin4.w};
    const int sums = sums_up_to(n[0] + n[1] + n[2] + n[3]), all = __builtin_amdgcn_readlane(sums, 63);
    // the last lane that has `wanted` scores in its bins or behind them, and the last of its bins that has
    const int behind = all - sums;
    const int at = 63 - __builtin_clzll(__ballot(all - sums + n[0] + n[1] + n[2] + n[3] >= wanted));
    int above = __builtin_amdgcn_readlane(behind, at), in_bin = 0, bin = 4 * at;
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

  // Scores above hi are taken, and of those from lo to hi the first `wanted`: counted by item and wave, which is the pages' order.
  auto is_end = [&](const int j) {
    const int i = kChooseThreads * j + tid;
    return i < there && (i < first || i >= last);
  };
  each([&](const int j, const uint32_t x) {
    const uint32_t equal = __popcll(__ballot(x >= lo && x <= hi)), sure = __popcll(__ballot(x > hi || is_end(j)));
    if (lane == 0) counts[kChooseWaves * j + wave] = equal << 16 | sure;
  });
  __syncthreads();
  uint32_t so_far_equal = 0, so_far_sure = 0;
  for (int i = 0; i < items * kChooseWaves; i += 64) {  // (each wave for itself, all with the same result)
    const uint32_t x = i + lane < items * kChooseWaves ? counts[i + lane] : 0u, equal = x >> 16, sure = x & 0xffffu;
    const uint32_t equals = sums_up_to(equal), sures = sums_up_to(sure);
    if (i + lane < items * kChooseWaves) before[i + lane] = (so_far_equal + equals - equal) << 16 | (so_far_sure + sures - sure);
    so_far_equal += __builtin_amdgcn_readlane(equals, 63);
    so_far_sure += __builtin_amdgcn_readlane(sures, 63);
  }
  each([&](const int j, const uint32_t x) {
    const uint32_t packed = before[kChooseWaves * j + wave];
    const int equal_before = packed >> 16, out = (packed & 0xffffu) + min(equal_before, wanted);
    const uint64_t equals = __ballot(x >= lo && x <= hi), below = (1ull << lane) - 1;
    const bool mine = x > hi || is_end(j) || (x >= lo && equal_before + __popcll(equals & below) < wanted);
    const uint64_t takes = __ballot(mine);
    if (mine) {
      const int to = out + __popcll(takes & below), i = kChooseThreads * j + tid;
      pages[to] = i;
      chosen[to] = table[i];
    }
  });
}

template <typename T, int D>
static void launch_paged_select_for(const PagedSelectArgs& a, hipStream_t stream) {
  const dim3 units(a.n_kv_heads, a.batch);
  if (a.max_pages <= kFused) {
    hipLaunchKernelGGL((paged_choose_kernel<T, D, true, kFused / kChooseThreads>), units, dim3(kChooseThreads), 0, stream, a);
    return;
  }
  // (some two thousand work-groups, however long the table is and however short the sequences)
  const int chunks = (a.max_pages + 4 * Scores<T, D>::kPages - 1) / (4 * Scores<T, D>::kPages);
  const int64_t n_units = (int64_t)a.n_kv_heads * a.batch;
  const int side = (int)((2048 + n_units - 1) / n_units);
  hipLaunchKernelGGL((paged_scores_kernel<T, D>), dim3(chunks < side ? chunks : side, a.n_kv_heads, a.batch), dim3(256), 0, stream, a);
  if (a.max_pages <= kInRegisters) hipLaunchKernelGGL((paged_choose_kernel<T, D, false, kInRegisters / kChooseThreads>), units, dim3(kChooseThreads), 0, stream, a);
  else hipLaunchKernelGGL((paged_choose_kernel<T, D, false, 0>), units, dim3(kChooseThreads), 0, stream, a);
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
