// New tokens of a paged key/value cache on gfx950: the rotary embedding of queries and keys, keys and values into their pages, and the bounds
// of the pages' keys.
//
// Bound by reading and writing each element once.  A run is what a page receives: the tokens of one sequence that go to one page.  A work-group
// has the runs that begin among its few tokens, for one KV head and its group of queries, so that a page's bounds are one work-group's and need
// no atomics.  A lane takes 8 channels of each half of all rows of a token (D / 16 lanes a token), whose cosines and sines it loads once.
// A step of one token each is latency: what does not depend on the token's place is requested before that is known.
#include "aa_kernels.h"
#include "aa_paged.h"

namespace aa {

struct Rows8 {  // 8 channels of each half
  uint4 first, second;
};
__device__ __forceinline__ Rows8 load8(const uint16_t* p, const int half) {
  return {*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(p + half)};
}
__device__ __forceinline__ void store8(uint16_t* p, const int half, const Rows8& x) {
  *reinterpret_cast<uint4*>(p) = x.first;
  *reinterpret_cast<uint4*>(p + half) = x.second;
}
struct Angles {
  float4 cos[2], sin[2];
};
// turned by their angles: float32, one rounding
template <typename T>
__device__ __forceinline__ Rows8 rotated(const Rows8& raw, const Angles& a) {
  float x[8], y[8];
  unpack8<T>(raw.first, x);
  unpack8<T>(raw.second, y);
  const float c[8] = {a.cos[0].x, a.cos[0].y, a.cos[0].z, a.cos[0].w, a.cos[1].x, a.cos[1].y, a.cos[1].z, a.cos[1].w};
  const float s[8] = {a.sin[0].x, a.sin[0].y, a.sin[0].z, a.sin[0].w, a.sin[1].x, a.sin[1].y, a.sin[1].z, a.sin[1].w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float u = x[j], v = y[j];
    x[j] = __builtin_fmaf(u, c[j], -(v * s[j]));
    y[j] = __builtin_fmaf(v, c[j], u * s[j]);
  }
  return {pack8<T>(x), pack8<T>(y)};
}

template <typename T, int D, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) paged_append_kernel(const PagedAppendArgs p) {
  constexpr int kPieces = D / 16;                  // lanes of a token
  constexpr int kInWave = 64 / kPieces;            // tokens of a wave
  constexpr int kTokens = WAVES * kInWave;         // ... and of the work-group, side by side
  __shared__ float red[WAVES > 1 ? WAVES - 1 : 1][kPieces][32];
  const int tid = threadIdx.x, lane = tid & 63, c = tid % kPieces, row = tid / kPieces;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kvh = blockIdx.x % p.n_kv_heads, group = p.n_q_heads / p.n_kv_heads, page_size = 1 << p.page_log;
  const int first = blockIdx.x / p.n_kv_heads * p.chunk;
  const const_i32 *lengths = (const_i32*)p.lengths, *starts = (const_i32*)p.starts;

  for (int t = first; t < min(first + p.chunk, p.n_tokens);) {
    int b = t, begin = t, end = t + 1;
    if (p.starts != nullptr) {
      b = 0;
      for (int i = 0; i < p.batch; i += 64) {  // the sequences that end at or before t
        const int n = __popcll(__ballot(i + lane < p.batch && p.starts[min(i + lane, p.batch - 1) + 1] <= t));
        b += n;
        if (n < 64) break;
      }
      if (b >= p.batch) return;  // (behind the last sequence)
      begin = starts[b];
      end = starts[b + 1];
    }
    const int64_t position = (int64_t)lengths[b] - end + t;
    if (t < begin || t >= end || position < 0 || position >> p.page_log >= p.max_pages) {
      ++t;
      continue;
    }
    const int at = ((const_i32*)(p.table + b * p.t_sb))[position >> p.page_log], slot = (int)position & (page_size - 1);
    int n = min(min(end, p.n_tokens) - t, page_size - slot);
    const int t0 = t;
    t += n;
    if (t0 != begin && slot != 0) continue;  // (the rest of a run that began among the tokens before)
    if (p.cos != nullptr) n = (int)min((int64_t)n, p.n_positions - position);
    if ((uint32_t)at >= (uint32_t)p.n_pages || n <= 0) continue;

    uint16_t* bounds = p.bounds + ((int64_t)at * p.n_kv_heads + kvh) * 2 * D + 8 * c;
    Rows8 old[2];
    const bool writes = p.bounds != nullptr && row == 0;  // the bounds, at the end
    if (writes && slot != 0) {
      old[0] = load8(bounds, D / 2);
      old[1] = load8(bounds + D, D / 2);
    }
    float lo[16], hi[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      lo[j] = INFINITY;
      hi[j] = -INFINITY;
    }
    for (int i = row; i < n; i += kTokens) {
      const int64_t tok = t0 + i;
      Rows8 k = load8(p.k + tok * p.k_st + kvh * p.k_sh + 8 * c, D / 2);
      const Rows8 v = load8(p.v + tok * p.v_st + kvh * p.v_sh + 8 * c, D / 2);
      Angles a;
      if (p.cos != nullptr) {
        const float *cos = p.cos + (position + i) * p.cs_sn + 8 * c, *sin = p.sin + (position + i) * p.cs_sn + 8 * c;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          a.cos[j] = reinterpret_cast<const float4*>(cos)[j];
          a.sin[j] = reinterpret_cast<const float4*>(sin)[j];
        }
        for (int h = 0; h < group; h += 4) {
          Rows8 q[4];
          const uint16_t* src = p.q + tok * p.q_st + (int64_t)(kvh * group + h) * p.q_sh + 8 * c;
          uint16_t* dst = p.q_out + tok * p.qo_st + (int64_t)(kvh * group + h) * p.qo_sh + 8 * c;
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (h + j < group) q[j] = load8(src + j * p.q_sh, D / 2);
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (h + j < group) store8(dst + j * p.qo_sh, D / 2, rotated<T>(q[j], a));
        }
        k = rotated<T>(k, a);
      }
      store8(p.keys + at * p.kp_sp + kvh * p.kp_sh + (slot + i) * p.kp_sn + 8 * c, D / 2, k);
      store8(p.values + at * p.vp_sp + kvh * p.vp_sh + (slot + i) * p.vp_sn + 8 * c, D / 2, v);
      if (p.bounds != nullptr) {  // (those of the keys as stored)
        float x[2][8];
        unpack8<T>(k.first, x[0]);
        unpack8<T>(k.second, x[1]);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          lo[j] = min_or_nan(lo[j], x[j >> 3][j & 7]);
          hi[j] = max_or_nan(hi[j], x[j >> 3][j & 7]);
        }
      }
    }
    if (p.bounds == nullptr) continue;
#pragma unroll
    for (int d = kPieces; d < 64; d <<= 1) {  // over the tokens of a wave
      if (n * kPieces > d) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          lo[j] = min_or_nan(lo[j], __shfl_xor(lo[j], d, 64));
          hi[j] = max_or_nan(hi[j], __shfl_xor(hi[j], d, 64));
        }
      }
    }
    if (WAVES > 1 && n > kInWave) {  // over the waves
      if (wave > 0 && lane < kPieces) {
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          red[wave - 1][c][j] = lo[j];
          red[wave - 1][c][16 + j] = hi[j];
        }
      }
      __syncthreads();
      if (row == 0)
#pragma unroll
        for (int w = 0; w < WAVES - 1; ++w)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            lo[j] = min_or_nan(lo[j], red[w][c][j]);
            hi[j] = max_or_nan(hi[j], red[w][c][16 + j]);
          }
      __syncthreads();
    }
    if (writes) {
      if (slot != 0) {
        float x[4][8];
        unpack8<T>(old[0].first, x[0]);
        unpack8<T>(old[0].second, x[1]);
        unpack8<T>(old[1].first, x[2]);
        unpack8<T>(old[1].second, x[3]);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          lo[j] = min_or_nan(lo[j], x[j >> 3][j & 7]);
          hi[j] = max_or_nan(hi[j], x[2 + (j >> 3)][j & 7]);
        }
      }
      float y[4][8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        y[0][j] = lo[j];
        y[1][j] = lo[8 + j];
        y[2][j] = hi[j];
        y[3][j] = hi[8 + j];
      }
      store8(bounds, D / 2, {pack8<T>(y[0]), pack8<T>(y[1])});
      store8(bounds + D, D / 2, {pack8<T>(y[2]), pack8<T>(y[3])});
    }
  }
}

template <typename T, int D>
static void launch_paged_append_for(PagedAppendArgs a, hipStream_t stream) {
  // Tokens of a work-group: few, so that short runs do not queue up in one, but no fewer than make some thousand work-groups
  const int64_t most = (int64_t)a.n_tokens * a.n_kv_heads / 4096, page_size = 1 << a.page_log;
  a.chunk = a.starts == nullptr || most < 1 ? 1 : (int)(most < page_size ? most : page_size);
  const dim3 grid((uint32_t)((a.n_tokens + a.chunk - 1) / a.chunk) * (uint32_t)a.n_kv_heads);
  const int waves = a.starts == nullptr ? 1 : (int)(page_size * (D / 16) / 64);
  if (waves <= 1) hipLaunchKernelGGL((paged_append_kernel<T, D, 1>), grid, dim3(64), 0, stream, a);
  else if (waves == 2) hipLaunchKernelGGL((paged_append_kernel<T, D, 2>), grid, dim3(128), 0, stream, a);
  else hipLaunchKernelGGL((paged_append_kernel<T, D, 4>), grid, dim3(256), 0, stream, a);
}

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t stream) {
  if (a.head_dim == 128) {
    if (a.dtype == 0) launch_paged_append_for<Bf16, 128>(a, stream);
    else launch_paged_append_for<F16, 128>(a, stream);
  } else {
    if (a.dtype == 0) launch_paged_append_for<Bf16, 64>(a, stream);
    else launch_paged_append_for<F16, 64>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace aa
