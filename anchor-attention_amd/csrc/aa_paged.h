// What the kernels over a cache in pages share: how they read tables and lengths, which come from device memory and are not trusted.
#pragma once
#include "aa_common.h"

namespace aa {

// Tables and lengths that no kernel that reads them writes: scalar loads where the index is wave-uniform.
typedef __attribute__((address_space(4))) const int32_t const_i32;

__device__ __forceinline__ int clamped_length(const int32_t* lengths, const int b, const int max_pages, const int page_log) {
  return min(max(lengths[b], 0), max_pages << page_log);
}
// pages of a sequence
__device__ __forceinline__ int pages_of(const int length, const int page_log) { return (length + (1 << page_log) - 1) >> page_log; }
// the nearest page there is
__device__ __forceinline__ int clamped_page(const int page, const int n_pages) { return min(max(page, 0), n_pages - 1); }

// The smaller (larger) of two numbers; NaN where one is NaN (the hardware's minimum drops it).
__device__ __forceinline__ float min_or_nan(const float a, const float b) { return b < a || b != b ? b : a; }
__device__ __forceinline__ float max_or_nan(const float a, const float b) { return b > a || b != b ? b : a; }

template <typename T>
__device__ __forceinline__ void unpack8(const uint4 raw, float (&x)[8]) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = T::lo(w[j]);
    x[2 * j + 1] = T::hi(w[j]);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  return uint4{T::pack(x[0], x[1]), T::pack(x[2], x[3]), T::pack(x[4], x[5]), T::pack(x[6], x[7])};
}

}  // namespace aa
