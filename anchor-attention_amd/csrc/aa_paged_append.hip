// New tokens of a paged key/value cache on gfx950: the rotary embedding of queries and keys, keys and values into their pages, and the bounds
// of the pages' keys.
//
// Bound by reading and writing each element once.  A work-group has one token and KV head: it rotates the queries of the group and copies
// the value; the first of a page's new tokens has the keys of all of them, so that a page's bounds are one work-group's and need
// no atomics.
#include "aa_kernels.h"
#include "aa_paged.h"

namespace aa {

// 8 channels of each half of a row, 16 bytes each, turned by their angles (float32, one rounding)
template <typename T>
__device__ __forceinline__ void rotate8(float (&first)[8], float (&second)[8], const float* __restrict__ cos, const float* __restrict__ sin) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float c = cos[j], s = sin[j], x = first[j], y = second[j];
    first[j] = __builtin_fmaf(x, c, -(y * s));
    second[j] = __builtin_fmaf(y, c, x * s);
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedAppendArgs p) {
  constexpr int kPieces = D / 16;        // 8 channels of each half are a thread's
  constexpr int kRows = 256 / kPieces;   // rows side by side
  __shared__ float red[2][4][D];
  const int tid = threadIdx.x, c = tid % kPieces, row = tid / kPieces;
  const int t = blockIdx.x, kvh = blockIdx.y;
  const int page_size = 1 << p.page_log;
  int b = t, begin = t, end = t + 1;
  if (p.starts != nullptr) {
    b = 0;
    while (b < p.batch && p.starts[b + 1] <= t) ++b;
    if (b >= p.batch) return;
    begin = p.starts[b];
    end = p.starts[b + 1];
  }
  const int64_t position = (int64_t)p.lengths[b] - end + t;
  if (t < begin || position < 0 || position >> p.page_log >= p.max_pages) return;
  const int at = p.table[b * p.t_sb + (position >> p.page_log)], slot = (int)(position & (page_size - 1));
  if ((uint32_t)at >= (uint32_t)p.n_pages || (p.cos != nullptr && position >= p.n_positions)) return;

  const int group = p.n_q_heads / p.n_kv_heads;
  const float* cos = p.cos + position * p.cs_sn + 8 * c;
  const float* sin = p.sin + position * p.cs_sn + 8 * c;
  for (int h = row; h < group; h += kRows) {
    const uint16_t* src = p.q + t * p.q_st + (int64_t)(kvh * group + h) * p.q_sh + 8 * c;
    uint16_t* dst = p.q_out + t * p.qo_st + (int64_t)(kvh * group + h) * p.qo_sh + 8 * c;
    float x[8], y[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(src), x);
    unpack8<T>(*reinterpret_cast<const uint4*>(src + D / 2), y);
    rotate8<T>(x, y, cos, sin);
    *reinterpret_cast<uint4*>(dst) = pack8<T>(x);
    *reinterpret_cast<uint4*>(dst + D / 2) = pack8<T>(y);
  }
  if (tid < D / 8)
    *reinterpret_cast<uint4*>(p.values + at * p.vp_sp + kvh * p.vp_sh + slot * p.vp_sn + 8 * tid) =
        *reinterpret_cast<const uint4*>(p.v + t * p.v_st + kvh * p.v_sh + 8 * tid);

  // the first of the page's tokens that have a place
  if (t != begin && slot != 0) return;
  int n = min(min(end, p.n_tokens) - t, page_size - slot);
  if (p.cos != nullptr) n = (int)min((int64_t)n, p.n_positions - position);
  float lo[16], hi[16];
  bool none = true;
  for (int i = row; i < n; i += kRows) {
    const uint16_t* src = p.k + (int64_t)(t + i) * p.k_st + kvh * p.k_sh + 8 * c;
    uint16_t* dst = p.keys + at * p.kp_sp + kvh * p.kp_sh + (int64_t)(slot + i) * p.kp_sn + 8 * c;
    float x[8], y[8];
    unpack8<T>(*reinterpret_cast<const uint4*>(src), x);
    unpack8<T>(*reinterpret_cast<const uint4*>(src + D / 2), y);
    if (p.cos != nullptr) rotate8<T>(x, y, cos + i * p.cs_sn, sin + i * p.cs_sn);
    const uint4 px = pack8<T>(x), py = pack8<T>(y);
    *reinterpret_cast<uint4*>(dst) = px;
    *reinterpret_cast<uint4*>(dst + D / 2) = py;
    unpack8<T>(px, x);  // (the bounds are those of the keys as stored)
    unpack8<T>(py, y);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float z = j < 8 ? x[j & 7] : y[j & 7];
      lo[j] = none ? z : min_or_nan(lo[j], z);
      hi[j] = none ? z : max_or_nan(hi[j], z);
    }
    none = false;
  }
  if (p.bounds == nullptr) return;
  // over the rows of a wave that hold keys, then over the waves
#pragma unroll
  for (int d = kPieces; d < 64; d <<= 1) {
    const bool other_none = __shfl_xor((int)none, d, 64) != 0;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float l = __shfl_xor(lo[j], d, 64), h = __shfl_xor(hi[j], d, 64);
      if (!other_none) {
        lo[j] = none ? l : min_or_nan(lo[j], l);
        hi[j] = none ? h : max_or_nan(hi[j], h);
      }
    }
    none = none && other_none;
  }
  const int wave = tid >> 6, lane = tid & 63;
  if (lane < kPieces) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      red[0][wave][(j >> 3) * (D / 2) + 8 * c + (j & 7)] = lo[j];
      red[1][wave][(j >> 3) * (D / 2) + 8 * c + (j & 7)] = hi[j];
    }
  }
  __syncthreads();
  const int waves = min(4, (n + 64 / kPieces - 1) / (64 / kPieces));  // (those that hold a key)
  for (int i = tid; i < 2 * D; i += 256) {
    const int which = i / D, d = i % D;
    float x = red[which][0][d];
    for (int w = 1; w < waves; ++w) x = which == 0 ? min_or_nan(x, red[0][w][d]) : max_or_nan(x, red[1][w][d]);
    uint16_t* dst = p.bounds + ((int64_t)at * p.n_kv_heads + kvh) * 2 * D + i;
    if (slot != 0) x = which == 0 ? min_or_nan(x, T::from16(*dst)) : max_or_nan(x, T::from16(*dst));
    *dst = (uint16_t)T::pack(x, 0.f);
  }
}

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t stream) {
  const dim3 grid(a.n_tokens, a.n_kv_heads), block(256);
  if (a.head_dim == 128) {
    if (a.dtype == 0) hipLaunchKernelGGL((paged_append_kernel<Bf16, 128>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((paged_append_kernel<F16, 128>), grid, block, 0, stream, a);
  } else {
    if (a.dtype == 0) hipLaunchKernelGGL((paged_append_kernel<Bf16, 64>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((paged_append_kernel<F16, 64>), grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace aa
