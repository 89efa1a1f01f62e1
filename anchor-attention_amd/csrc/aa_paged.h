// What the kernels over a cache in pages share: how they read tables and lengths, which come from device memory and are not trusted, and what attention over tiles of
// keys is made of.
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

// A score or weight as an unsigned number of the same order; NaN as infinity, -0 as 0.
__device__ __forceinline__ uint32_t ordered(float x) {
  x = x != x ? INFINITY : x + 0.f;
  const uint32_t u = __float_as_uint(x);
  return (u >> 31) ? ~u : u | 0x80000000u;
}

// Bounds are kept as pairs of 16-bit whole numbers of the same order (-0 below 0, NaN of either sign beyond the infinities), two to an
// instruction.  There and back:
__device__ __forceinline__ uint32_t in_order(const uint32_t x) {
  typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
  const i16x2 signs = *reinterpret_cast<const i16x2*>(&x) >> 15;
  return x ^ (*reinterpret_cast<const uint32_t*>(&signs) & 0x7fff7fffu);
}
__device__ __forceinline__ uint32_t least(const uint32_t a, const uint32_t b) {
  typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
  const i16x2 m = __builtin_elementwise_min(*reinterpret_cast<const i16x2*>(&a), *reinterpret_cast<const i16x2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
__device__ __forceinline__ uint32_t most(const uint32_t a, const uint32_t b) {
  typedef int16_t i16x2 __attribute__((ext_vector_type(2)));
  const i16x2 m = __builtin_elementwise_max(*reinterpret_cast<const i16x2*>(&a), *reinterpret_cast<const i16x2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&m);
}
// Back, where both bounds of a channel become NaN if a key was.
template <typename T>
__device__ __forceinline__ void bounds_back(uint32_t& lo, uint32_t& hi) {
  lo = in_order(lo);
  hi = in_order(hi);
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint32_t mask = 0x7fffu << (16 * half), most_finite = (uint32_t)T::kExponent << (16 * half);
    if ((lo & mask) > most_finite || (hi & mask) > most_finite) {
      lo |= mask;
      hi |= mask;
    }
  }
}

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

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

template <typename T> __device__ __forceinline__ floatx4 mfma16(u32x4 a, u32x4 b, floatx4 c);
template <> __device__ __forceinline__ floatx4 mfma16<Bf16>(u32x4 a, u32x4 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const bf16x8*>(&a), *reinterpret_cast<const bf16x8*>(&b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ floatx4 mfma16<F16>(u32x4 a, u32x4 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const f16x8*>(&a), *reinterpret_cast<const f16x8*>(&b), c, 0, 0, 0);
}

// max and sum over the lanes 16, 32 and 48 away, which hold the other keys of a column
__device__ __forceinline__ float max_over_quarters(float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return max_with_other_half(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ __forceinline__ float sum_over_quarters(const float v) {
  const uint32_t u = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t w = __float_as_uint(__uint_as_float(r[0]) + __uint_as_float(r[1]));
  const auto s = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}
// f over all lanes of a wave
template <typename F>
__device__ __forceinline__ float over_wave(const float x, const float none, F f) {
  const uint32_t all = up_to(__float_as_uint(x), __float_as_uint(none),
                             [&](const uint32_t a, const uint32_t b) { return __float_as_uint(f(__uint_as_float(a), __uint_as_float(b))); });
  return __uint_as_float(__builtin_amdgcn_readlane(all, 63));
}

// Rows of a page behind a wave-uniform address: a lane's loads then have an offset of 32 bits, and the address is scalar arithmetic.  Rows behind the last key are out
// of range, so that nothing is fetched for them (1000 sequences of 1 to 200 keys, 32/8 heads of 128, 56.7 -> 47.2 us).
typedef __amdgpu_buffer_rsrc_t Rows;
__device__ __forceinline__ Rows rows_at(const uint16_t* base, const int bytes) {
  const uint64_t u = (uint64_t)base;
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u), hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return __builtin_amdgcn_make_buffer_rsrc((void*)((uint64_t)hi << 32 | lo), 0, __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

}  // namespace aa
