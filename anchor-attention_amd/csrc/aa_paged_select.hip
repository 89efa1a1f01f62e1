// Which pages of a cache a sparse decode step reads, on gfx950: the scores of the pages' bounds and the largest of them.
//
// The scores are bound by reading the bounds once.  Products of two 16-bit numbers are exact in float32; their sum is
// formed in float64 and rounded once, so that the chosen pages do not depend on its order.
#include "aa_kernels.h"
#include "aa_paged.h"

namespace aa {

// A score as an unsigned number of the same order; NaN as infinity, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
  x = x != x ? INFINITY : x + 0.f;
  const uint32_t u = __float_as_uint(x);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// One work-group per (KV head, sequence): a thread a page.
template <typename T>
__global__ void __launch_bounds__(256) paged_scores_kernel(const PagedSelectArgs p) {
  const int kvh = blockIdx.x, b = blockIdx.y, D = p.head_dim, group = p.n_q_heads / p.n_kv_heads;
  const int there = pages_of(clamped_length(p.lengths, b, p.max_pages, p.page_log), p.page_log);
  float* scores = p.scores + ((int64_t)b * p.n_kv_heads + kvh) * p.max_pages;
  if (there <= p.n_chosen) return;
  for (int i = threadIdx.x; i < there; i += 256) {
    const uint16_t* lo = p.bounds + ((int64_t)clamped_page(p.table[b * p.t_sb + i], p.n_pages) * p.n_kv_heads + kvh) * 2 * D;
    float best = -INFINITY;
    bool nan = false;
    for (int h = 0; h < group; ++h) {
      const uint16_t* q = p.q + b * p.q_sb + (kvh * group + h) * p.q_sh;
      double sum = 0.0;
      for (int d = 0; d < D; ++d) {
        const float x = T::from16(q[d]);
        sum += (double)(x * T::from16(lo[x >= 0.f ? D + d : d]));
      }
      nan = nan || sum != sum;
      best = fmaxf(best, (float)sum);
    }
    scores[i] = nan ? INFINITY : best;
  }
}

// One work-group per (KV head, sequence): the n-th largest score bit by bit, then the pages above it and the first of those at it.
__global__ void __launch_bounds__(256) paged_choose_kernel(const PagedSelectArgs p) {
  __shared__ int count[4];
  const int kvh = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int there = pages_of(clamped_length(p.lengths, b, p.max_pages, p.page_log), p.page_log);
  const int64_t unit = (int64_t)b * p.n_kv_heads + kvh;
  const float* scores = p.scores + unit * p.max_pages;
  int32_t* pages = p.pages + unit * p.n_chosen;
  int32_t* chosen = p.chosen + unit * p.n_chosen;
  const int32_t* table = p.table + b * p.t_sb;
  if (there <= p.n_chosen) {
    for (int i = tid; i < p.n_chosen; i += 256) {
      pages[i] = i < there ? i : -1;
      chosen[i] = i < there ? table[i] : 0;
    }
    return;
  }
  const int first = p.n_first, last = there - p.n_last, wanted = p.n_chosen - p.n_first - p.n_last;
  uint32_t bar = 0;
  for (int bit = 31; bit >= 0 && wanted > 0; --bit) {
    const uint32_t higher = bar | 1u << bit;
    int n = 0;
    for (int i = first + tid; i < last; i += 256) n += ordered(scores[i]) >= higher;
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d, 64);
    if (lane == 0) count[wave] = n;
    __syncthreads();
    if (count[0] + count[1] + count[2] + count[3] >= wanted) bar = higher;
    __syncthreads();
  }
  int n = 0;
  for (int i = first + tid; i < last; i += 256) n += ordered(scores[i]) > bar;
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) n += __shfl_xor(n, d, 64);
  if (lane == 0) count[wave] = n;
  __syncthreads();
  const int at_bar = wanted - (count[0] + count[1] + count[2] + count[3]);
  if (wave != 0) return;
  int out = 0, equal = 0;  // (by one wave: in order)
  for (int base = 0; base < there; base += 64) {
    const int i = base + lane;
    const bool end = i < there && (i < first || i >= last), middle = i >= first && i < last && wanted > 0;
    const uint32_t x = middle ? ordered(scores[i]) : 0u;
    const uint64_t equals = __ballot(middle && x == bar), below = (1ull << lane) - 1;
    const bool mine = end || (middle && (x > bar || (x == bar && equal + __popcll(equals & below) < at_bar)));
    const uint64_t takes = __ballot(mine);
    if (mine) {
      const int to = out + __popcll(takes & below);
      pages[to] = i;
      chosen[to] = table[i];
    }
    out += __popcll(takes);
    equal += __popcll(equals);
  }
}

hipError_t launch_paged_select(const PagedSelectArgs& a, hipStream_t stream) {
  const dim3 grid(a.n_kv_heads, a.batch), block(256);
  if (a.dtype == 0) hipLaunchKernelGGL((paged_scores_kernel<Bf16>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((paged_scores_kernel<F16>), grid, block, 0, stream, a);
  hipLaunchKernelGGL(paged_choose_kernel, grid, block, 0, stream, a);
  return hipGetLastError();
}

}  // namespace aa
