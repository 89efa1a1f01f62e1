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

// One instruction's exchange inside rows of 16 lanes (the lanes are all active); those that receive nothing get `none`.
constexpr int kDppXor1 = 0xb1, kDppXor2 = 0x4e, kDppHalfMirror = 0x141, kDppRor4 = 0x124, kDppRor8 = 0x128;
template <int CONTROL, int ROWS = 0xf>
__device__ __forceinline__ uint32_t dpp(const uint32_t x, const uint32_t none = 0) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, CONTROL, ROWS, 0xf, false);
}
template <int CONTROL>
__device__ __forceinline__ double dpp(const double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  return __longlong_as_double((long long)((uint64_t)dpp<CONTROL>((uint32_t)(u >> 32)) << 32 | dpp<CONTROL>((uint32_t)u)));
}
// f of all lanes up to each, f being associative with the neutral element `none`
template <typename F>
__device__ __forceinline__ uint32_t up_to(uint32_t x, const uint32_t none, F f) {
  x = f(x, dpp<0x111>(x, none));        // 1, 2, 4 and 8 lanes before, inside a row
  x = f(x, dpp<0x112>(x, none));
  x = f(x, dpp<0x114>(x, none));
  x = f(x, dpp<0x118>(x, none));
  x = f(x, dpp<0x142, 0xa>(x, none));   // the last of the row before, to rows 1 and 3
  return f(x, dpp<0x143, 0xc>(x, none));  // lane 31, to rows 2 and 3
}
__device__ __forceinline__ int sums_up_to(const int x) {
  return (int)up_to((uint32_t)x, 0u, [](const uint32_t a, const uint32_t b) { return a + b; });
}

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
