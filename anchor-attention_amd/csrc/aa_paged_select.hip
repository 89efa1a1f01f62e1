// Which pages of a cache a sparse decode step reads, on gfx950: the scores of the pages' bounds and the largest of them.
//
// The scores are bound by reading the bounds once.  Products of two 16-bit numbers are exact in float32; their sum is
// formed in float64 and rounded once, so that the chosen pages do not depend on its order.  A lane has 8 channels of 4 pages, so a page is 8 or 16
// lanes'; their sums are exchanged so that each lane ends with a part of them (two halvings, then additions): 5 exchanges
// for 4 pages instead of 16.
//
// Choosing is latency: a work-group per (sequence, KV head) finds what the wanted number of scores reaches by histograms of 256 equal ranges of the
// numbers' order, each inside the range of the last one that holds it; the first spans the smallest to the largest score, so that two or three do, whatever
// the scores' exponents (at most five).  Integer work: the order in which counts are added does not matter.
#include "aa_kernels.h"
#include "aa_paged.h"

namespace aa {

constexpr int kAbreast = 4;        // pages of a lane
constexpr int kChooseThreads = 512;
constexpr int kChooseWaves = kChooseThreads / 64;
constexpr int kFused = 1024;       // a table of at most that many pages is scored and chosen from by one launch
constexpr int kInLds = 8192;       // the scores of at most that many pages are kept in LDS

// A score as an unsigned number of the same order, from 1 on; NaN as infinity, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
  x = x != x ? INFINITY : x + 0.f;
  const uint32_t u = __float_as_uint(x);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// The scores of pages first .. first + kPages - 1 of a sequence by one wave; store(page, score) is called by one lane for each.
template <typename T, int D>
struct Scores {
  static constexpr int kLanes = D / 8, kSide = 64 / kLanes, kPages = kSide * kAbreast;
  template <typename Store>
  static __device__ __forceinline__ void form(const PagedSelectArgs& p, const int b, const int kvh, const int there, const int first, Store store) {
    const int lane = threadIdx.x & 63, c = lane % kLanes, side = lane / kLanes, group = p.n_q_heads / p.n_kv_heads;
    const int32_t* table = p.table + b * p.t_sb;
    uint4 raw[kAbreast][2];
#pragma unroll
    for (int i = 0; i < kAbreast; ++i) {
      const int page = clamped_page(table[min(first + kSide * i + side, there - 1)], p.n_pages);
      const uint16_t* lo = p.bounds + ((int64_t)page * p.n_kv_heads + kvh) * 2 * D + 8 * c;
      raw[i][0] = *reinterpret_cast<const uint4*>(lo);
      raw[i][1] = *reinterpret_cast<const uint4*>(lo + D);
    }
    const uint16_t* qp = p.q + b * p.q_sb + (int64_t)kvh * group * p.q_sh + 8 * c;
    uint4 q_raw = *reinterpret_cast<const uint4*>(qp);
    float bounds[kAbreast][2][8];
#pragma unroll
    for (int i = 0; i < kAbreast; ++i)
#pragma unroll
      for (int w = 0; w < 2; ++w) unpack8<T>(raw[i][w], bounds[i][w]);
    const bool upper8 = (lane & (kLanes / 2)) != 0, upper4 = (lane & (kLanes / 4)) != 0;
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
      // (a lane keeps the half of the sums that its bit names and gives the other half away)
      double a = upper8 ? sum[2] : sum[0], a2 = upper8 ? sum[3] : sum[1];
      a += __shfl_xor(upper8 ? sum[0] : sum[2], kLanes / 2, 64);
      a2 += __shfl_xor(upper8 ? sum[1] : sum[3], kLanes / 2, 64);
      double s = upper4 ? a2 : a;
      s += __shfl_xor(upper4 ? a : a2, kLanes / 4, 64);
#pragma unroll
      for (int d = kLanes / 8; d > 0; d >>= 1) s += __shfl_xor(s, d, 64);
      nan = nan || s != s;
      best = fmaxf(best, (float)s);
    }
    const int page = first + kSide * ((upper8 ? 2 : 0) + (upper4 ? 1 : 0)) + side;
    if ((lane & (kLanes / 4 - 1)) == 0 && page < there) store(page, nan ? INFINITY : best);
  }
};

template <typename T, int D>
__global__ void __launch_bounds__(256) paged_scores_kernel(const PagedSelectArgs p) {
  const int kvh = blockIdx.y, b = blockIdx.z;
  const int there = pages_of(clamped_length(p.lengths, b, p.max_pages, p.page_log), p.page_log);
  if (there <= p.n_chosen) return;
  float* scores = p.scores + ((int64_t)b * p.n_kv_heads + kvh) * p.max_pages;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  for (int first = (4 * blockIdx.x + wave) * Scores<T, D>::kPages; first < there; first += 4 * gridDim.x * Scores<T, D>::kPages)
    Scores<T, D>::form(p, b, kvh, there, first, [&](const int page, const float x) { scores[page] = x; });
}

// FROM: 0 the scores are formed here, 1 read once, 2 read from memory as often as they are needed (more than fit)
template <typename T, int D, int FROM>
__global__ void __launch_bounds__(kChooseThreads) paged_choose_kernel(const PagedSelectArgs p) {
  __shared__ uint32_t kept[FROM == 0 ? kFused : FROM == 1 ? kInLds : 1];
  __shared__ uint32_t bins[256], range[2];
  __shared__ int found[2], counts[2][kChooseWaves];
  const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int there = pages_of(clamped_length(p.lengths, b, p.max_pages, p.page_log), p.page_log);
  const int64_t unit = (int64_t)b * p.n_kv_heads + kvh;
  const float* scores = p.scores + unit * p.max_pages;
  int32_t* pages = p.pages + unit * p.n_chosen;
  int32_t* chosen = p.chosen + unit * p.n_chosen;
  const int32_t* table = p.table + b * p.t_sb;
  if (there <= p.n_chosen) {
    for (int i = tid; i < p.n_chosen; i += kChooseThreads) {
      pages[i] = i < there ? i : -1;
      chosen[i] = i < there ? table[i] : 0;
    }
    return;
  }
  const int first = p.n_first, last = there - p.n_last;  // the pages to choose from
  int wanted = p.n_chosen - p.n_first - p.n_last;
  uint32_t lo = 0xffffffffu, hi = 0xffffffffu;  // (no score reaches them)
  if (tid == 0) {
    range[0] = 0xffffffffu;
    range[1] = 0u;
  }
  if (FROM == 0) {
    for (int i = wave * Scores<T, D>::kPages; i < there; i += kChooseWaves * Scores<T, D>::kPages)
      Scores<T, D>::form(p, b, kvh, there, i, [&](const int page, const float x) { kept[page] = ordered(x); });
  }
  if (FROM == 1) {
    for (int i = tid; i < there; i += kChooseThreads) kept[i] = ordered(scores[i]);
  }
  __syncthreads();
  auto get = [&](const int i) { return FROM == 2 ? ordered(scores[i]) : kept[i]; };
  if (wanted > 0) {
    hi = 0u;
    for (int i = first + tid; i < last; i += kChooseThreads) {
      const uint32_t x = get(i);
      lo = min(lo, x);
      hi = max(hi, x);
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
      lo = min(lo, (uint32_t)__shfl_xor((int)lo, d, 64));
      hi = max(hi, (uint32_t)__shfl_xor((int)hi, d, 64));
    }
    if (lane == 0) {
      atomicMin(&range[0], lo);
      atomicMax(&range[1], hi);
    }
    if (tid < 256) bins[tid] = 0u;
    __syncthreads();
    lo = range[0];
    hi = range[1];
    // the wanted-th largest score lies in [lo, hi]; all of those above hi are taken
    for (;;) {
      const uint32_t span = hi - lo;
      const int shift = span < 256u ? 0 : 24 - __builtin_clz(span);  // span >> shift < 256
      for (int i = first + tid; i < last; i += kChooseThreads) {
        const uint32_t x = get(i);
        if (x >= lo && x <= hi) atomicAdd(&bins[(x - lo) >> shift], 1u);
      }
      __syncthreads();
      if (wave == 0) {  // the last bin that has `wanted` scores in it or behind it
        int n[4], sum = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) sum += n[j] = (int)bins[4 * lane + j];
        int behind = sum;  // of this lane's bins and the next lanes'
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int y = __shfl_down(behind, d, 64);
          if (lane + d < 64) behind += y;
        }
        int above = behind - sum;
        if (above < wanted && behind >= wanted) {
#pragma unroll
          for (int j = 3; j >= 0; --j) {
            if (above < wanted && above + n[j] >= wanted) {
              found[0] = 4 * lane + j;
              found[1] = wanted - above;
            }
            above += n[j];
          }
        }
      }
      __syncthreads();
      const int bin = found[0], in_bin = (int)bins[bin];
      wanted = found[1];  // of this bin
      lo += (uint32_t)bin << shift;
      hi = lo + min(hi - lo, (1u << shift) - 1u);
      if (shift == 0 || wanted == in_bin) break;  // (one number is left, or all of the bin are taken)
      __syncthreads();
      if (tid < 256) bins[tid] = 0u;
      __syncthreads();
    }
  }
  // Scores above hi are taken, and of those from lo to hi the first `wanted`.
  const int per_wave = ((there + kChooseWaves - 1) / kChooseWaves + 63) / 64 * 64, begin = min(wave * per_wave, there), stop = min(begin + per_wave, there);
  int equal = 0, above = 0;
  for (int base = begin; base < stop; base += 64) {
    const int i = base + lane;
    const bool middle = i < stop && i >= first && i < last;
    const uint32_t x = middle ? get(i) : 0u;
    const bool end = i < stop && !middle;
    equal += __popcll(__ballot(middle && x >= lo && x <= hi));
    above += __popcll(__ballot(end || (middle && x > hi)));
  }
  if (lane == 0) {
    counts[0][wave] = equal;
    counts[1][wave] = above;
  }
  __syncthreads();
  int equal_before = 0, out = 0;
  for (int w = 0; w < wave; ++w) {
    const int e = counts[0][w];
    out += counts[1][w] + min(e, max(0, wanted - equal_before));
    equal_before += e;
  }
  for (int base = begin; base < stop; base += 64) {
    const int i = base + lane;
    const bool middle = i < stop && i >= first && i < last;
    const uint32_t x = middle ? get(i) : 0u;
    const bool end = i < stop && !middle;
    const uint64_t equals = __ballot(middle && x >= lo && x <= hi), below = (1ull << lane) - 1;
    const bool mine = end || (middle && (x > hi || (x >= lo && equal_before + __popcll(equals & below) < wanted)));
    const uint64_t takes = __ballot(mine);
    if (mine) {
      const int to = out + __popcll(takes & below);
      pages[to] = i;
      chosen[to] = table[i];
    }
    out += __popcll(takes);
    equal_before += __popcll(equals);
  }
}

template <typename T, int D>
static void launch_paged_select_for(const PagedSelectArgs& a, hipStream_t stream) {
  const dim3 units(a.n_kv_heads, a.batch);
  if (a.max_pages <= kFused) {
    hipLaunchKernelGGL((paged_choose_kernel<T, D, 0>), units, dim3(kChooseThreads), 0, stream, a);
    return;
  }
  // (about a thousand work-groups, however long the table is and however short the sequences)
  const int chunks = (a.max_pages + 4 * Scores<T, D>::kPages - 1) / (4 * Scores<T, D>::kPages);
  const int64_t n_units = (int64_t)a.n_kv_heads * a.batch;
  const int side = (int)((2048 + n_units - 1) / n_units);
  hipLaunchKernelGGL((paged_scores_kernel<T, D>), dim3(chunks < side ? chunks : side, a.n_kv_heads, a.batch), dim3(256), 0, stream, a);
  if (a.max_pages <= kInLds) hipLaunchKernelGGL((paged_choose_kernel<T, D, 1>), units, dim3(kChooseThreads), 0, stream, a);
  else hipLaunchKernelGGL((paged_choose_kernel<T, D, 2>), units, dim3(kChooseThreads), 0, stream, a);
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
