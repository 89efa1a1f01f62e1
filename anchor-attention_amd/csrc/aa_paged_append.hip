// New tokens of a paged key/value cache on gfx950: the rotary embedding of queries and keys, keys and values into their pages, and the bounds
// of the pages' keys.
//
// Bound by reading and writing each element once.  A lane takes 8 channels of each half of rows (D / 16 lanes a row).  Two kinds of work-groups
// share the launch.  One has a few tokens and a KV head: queries of its group and the value, any token apart from the others, with the token's cosines and
// sines in registers.  The other has the keys that pages receive: a run is the tokens of one sequence that go to one page, and a work-group takes the runs
// that begin among its few tokens, so that a page's bounds are one work-group's and need no atomics.  (With queries and values in the runs, too, prompts
// of few KV heads or large pages had too few work-groups: 6001 tokens, 14/2 heads of 64, pages of 64 48 us, of 256 47; 21 and 18 so.)
//
// Measured: a token of each of 96 sequences, 28/4 heads of 128, bf16 4.5 us, the launch and a chain of three loads; a prompt of 6001, 32/8 of 64, fp16 16.0 us, 4.8
// TB/s; six prompts of 700 to 21000 tokens, 32/8 of 128, bf16 205 us, 5.1 TB/s, where a copy reaches 5.2.  With norms (MORE), which need a head's squares summed over its lanes before its
// first product and its weights beside its angles: the same prompt 18.6 us a step, six prompts of 28/4 of 128 169 us, 4.9 TB/s, a token 4.7 us.  Norms in a launch of their own would read and
// write queries and keys once more.
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
// A norm: x * w / sqrt(mean of the head's x^2 + eps), float32.  A head is D / 16 neighbouring lanes', all of them active.  Its weights stay as they lie in memory: unpacked, they would
// leave three waves to a SIMD instead of four.
template <typename T, int PIECES>
__device__ __forceinline__ void normalise(float (&x)[8], float (&y)[8], const Rows8& weight, const float eps) {
  float sum = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) sum += x[j] * x[j] + y[j] * y[j];
  sum += __uint_as_float(dpp<kDppXor1>(__float_as_uint(sum)));
  sum += __uint_as_float(dpp<kDppXor2>(__float_as_uint(sum)));
  if (PIECES == 8) sum += __uint_as_float(dpp<kDppHalfMirror>(__float_as_uint(sum)));  // (the four lanes of either half have the same sum)
  const float scale = rsqrtf(sum * (1.f / (16 * PIECES)) + eps);
  float w[8];
  unpack8<T>(weight.first, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] *= scale * w[j];
  unpack8<T>(weight.second, w);
#pragma unroll
  for (int j = 0; j < 8; ++j) y[j] *= scale * w[j];
}

// turned by their angles, after a norm if there is one: float32, one rounding
template <typename T, int PIECES>
__device__ __forceinline__ Rows8 rotated(const Rows8& raw, const Angles& a, const Rows8* norm = nullptr, const float eps = 0.f) {
  float x[8], y[8];
  unpack8<T>(raw.first, x);
  unpack8<T>(raw.second, y);
  if (norm != nullptr) normalise<T, PIECES>(x, y, *norm, eps);
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

struct Bounds8 {  // of 8 channels of each half
  uint32_t lo[8], hi[8];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = 0x7fff7fffu;
      hi[j] = 0x80008000u;
    }
  }
  __device__ __forceinline__ void widen(const uint32_t (&low)[8], const uint32_t (&high)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = least(lo[j], low[j]);
      hi[j] = most(hi[j], high[j]);
    }
  }
};
__device__ __forceinline__ void words(const Rows8& x, uint32_t (&w)[8]) {
  const uint32_t raw[8] = {x.first.x, x.first.y, x.first.z, x.first.w, x.second.x, x.second.y, x.second.z, x.second.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = in_order(raw[j]);
}
template <typename T>
__device__ __forceinline__ void bounds_of(const Bounds8& b, Rows8& lo, Rows8& hi) {
  uint32_t l[8], h[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    l[j] = b.lo[j];
    h[j] = b.hi[j];
    bounds_back<T>(l[j], h[j]);
  }
  lo = {uint4{l[0], l[1], l[2], l[3]}, uint4{l[4], l[5], l[6], l[7]}};
  hi = {uint4{h[0], h[1], h[2], h[3]}, uint4{h[4], h[5], h[6], h[7]}};
}
// f over the lanes of a wave that have the same piece (lane % PIECES), one instruction or two each
template <int PIECES, typename F>
__device__ __forceinline__ uint32_t over_tokens(uint32_t x, F f) {
  if (PIECES == 4) x = f(x, dpp<kDppRor4>(x));
  x = f(x, dpp<kDppRor8>(x));
  const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = f(r[0], r[1]);
  const auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return f(s[0], s[1]);
}

// Where a token goes: its place in the sequence, what its position is more than that, the page of the pool and the row in it; not ok: nowhere.
struct Place {
  int64_t position;
  int64_t shift;
  int at, slot;
  bool ok;
};
// token t of sequence b, whose tokens are those from begin to end; TABLE, a pointer to tables and lengths
template <bool MORE, typename Words>
__device__ __forceinline__ Place place_of(const PagedAppendArgs& p, const Words* lengths, const Words* table, const int b, const int begin, const int end, const int t) {
  Place x = {(int64_t)lengths[b] - end + t, 0, 0, 0, false};
  if (MORE && p.positions != nullptr) x.shift = (int64_t)((const Words*)p.positions)[b] - lengths[b];
  if (t < begin || t >= end || x.position < 0 || x.shift < 0 || x.position >> p.page_log >= p.max_pages ||
      (p.cos != nullptr && x.position + x.shift >= p.n_positions))
    return x;
  x.at = table[b * p.t_sb + (x.position >> p.page_log)];
  x.slot = (int)x.position & ((1 << p.page_log) - 1);
  x.ok = (uint32_t)x.at < (uint32_t)p.n_pages;
  return x;
}
// The sequences that end at or before t (wave-uniform), which is the one that t belongs to: every lane asks for the end of a 64th of those left, so that
// a load does for 64 sequences, two for 4096 and three for all.
__device__ __forceinline__ int sequence_of(const PagedAppendArgs& p, const int t) {
  const int lane = threadIdx.x & 63;
  int from = 0, left = p.batch;  // (those before `from` end at or before t, those from from + left on do not)
  for (;;) {
    const int step = (left + 63) >> 6, at = from + (lane + 1) * step - 1;
    const int n = __popcll(__ballot(at < from + left && p.starts[min(at, p.batch - 1) + 1] <= t));
    from += n * step;
    left = min(left - n * step, step - 1);
    if (left <= 0) return from;
  }
}
__device__ __forceinline__ Angles angles_of(const PagedAppendArgs& p, const int64_t position, const int c) {
  Angles a;
  const float *cos = p.cos + position * p.cs_sn + 8 * c, *sin = p.sin + position * p.cs_sn + 8 * c;
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    a.cos[j] = reinterpret_cast<const float4*>(cos)[j];
    a.sin[j] = reinterpret_cast<const float4*>(sin)[j];
  }
  return a;
}

// Queries and values of the tokens from `first` on, one of each kPieces lanes.
template <typename T, int D, bool MORE>
__device__ __forceinline__ void queries_and_values(const PagedAppendArgs& p, const int first, const int kvh) {
  constexpr int kPieces = D / 16, kInWave = 64 / kPieces;
  const int c = threadIdx.x % kPieces, group = p.n_q_heads / p.n_kv_heads;
  const int t0 = first + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * kInWave, t = t0 + (threadIdx.x & 63) / kPieces;
  if (t0 >= p.n_tokens) return;
  int b = t, begin = t, end = t + 1;
  if (p.starts != nullptr) {
    b = sequence_of(p, t0);
    if (b >= p.batch) return;
    if (((const_i32*)p.starts)[b + 1] < t0 + kInWave) {  // several sequences' tokens: the next 64 are looked through for each
      const int lane = threadIdx.x & 63, b0 = b, ends = p.starts[min(b0 + lane, p.batch - 1) + 1];
#pragma nounroll
      for (int j = 0; j < kInWave; ++j) {
        int n = __popcll(__ballot(b0 + lane < p.batch && ends <= t0 + j));
        if (n == 64) n = sequence_of(p, t0 + j) - b0;
        b = lane / kPieces == j ? b0 + n : b;
      }
      if (b >= p.batch) return;
    }
    begin = p.starts[b];
    end = p.starts[b + 1];
  }
  if (t >= p.n_tokens) return;
  const Place x = place_of<MORE>(p, p.lengths, p.table, b, begin, end, t);
  if (!x.ok) return;
  const Rows8 v = load8(p.v + t * p.v_st + kvh * p.v_sh + 8 * c, D / 2);
  if (group > 0) {
    const Angles a = angles_of(p, x.position + x.shift, c);
    const bool normed = MORE && p.q_norm != nullptr;
    Rows8 norm;
    if (normed) norm = load8(p.q_norm + 8 * c, D / 2);
    for (int h = 0; h < group; h += 4) {
      Rows8 q[4];
      const uint16_t* src = p.q + t * p.q_st + (int64_t)(kvh * group + h) * p.q_sh + 8 * c;
      uint16_t* dst = p.q_out + t * p.qo_st + (int64_t)(kvh * group + h) * p.qo_sh + 8 * c;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (h + j < group) q[j] = load8(src + j * p.q_sh, D / 2);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (h + j < group) store8(dst + j * p.qo_sh, D / 2, normed ? rotated<T, kPieces>(q[j], a, &norm, p.norm_eps) : rotated<T, kPieces>(q[j], a));
    }
  }
  store8(p.values + x.at * p.vp_sp + kvh * p.vp_sh + x.slot * p.vp_sn + 8 * c, D / 2, v);
}

// Keys of the runs that begin among the `chunk` tokens from `first` on, and their pages' bounds.
template <typename T, int D, int WAVES, bool MORE>
__device__ __forceinline__ void keys_and_bounds(const PagedAppendArgs& p, const int first, const int kvh, uint32_t (*red)[D / 16][16]) {
  constexpr int kPieces = D / 16;                  // lanes of a token
  constexpr int kInWave = 64 / kPieces;            // tokens of a wave
  constexpr int kTokens = WAVES * kInWave;         // ... and of the work-group, side by side
  const int tid = threadIdx.x, lane = tid & 63, c = tid % kPieces, row = tid / kPieces;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), page_size = 1 << p.page_log;
  const const_i32 *lengths = (const_i32*)p.lengths, *starts = (const_i32*)p.starts, *table = (const_i32*)p.table;
  const bool normed = MORE && p.k_norm != nullptr;
  Rows8 norm;
  if (normed) norm = load8(p.k_norm + 8 * c, D / 2);

  for (int t = first; t < min(first + p.chunk, p.n_tokens);) {
    int b = t, begin = t, end = t + 1;
    if (p.starts != nullptr) {
      b = sequence_of(p, t);
      if (b >= p.batch) return;  // (behind the last sequence)
      begin = starts[b];
      end = starts[b + 1];
    }
    const Place x = place_of<MORE>(p, lengths, table, b, begin, end, t);
    // the rest of the run; of tokens before the first position as many as there are
    int n = 1;
    if (t >= begin && t < end) n = x.position < 0 ? (int)min(-x.position, (int64_t)(end - t)) : min(min(end, p.n_tokens) - t, page_size - ((int)x.position & (page_size - 1)));
    const int t0 = t;
    t += n;
    // (nowhere; the rest of a run that began among the tokens before, of which there are none before token 0, wherever the sequence begins)
    if (!x.ok || (t0 != max(begin, 0) && x.slot != 0)) continue;
    if (p.cos != nullptr) n = (int)min((int64_t)n, p.n_positions - x.position - x.shift);

    uint16_t* bounds = p.bounds + ((int64_t)x.at * p.n_kv_heads + kvh) * 2 * D + 8 * c;
    Rows8 old[2];
    const bool writes = p.bounds != nullptr && row == 0;  // the bounds, at the end
    if (!MORE && writes && x.slot != 0) {  // (with a norm they would take the registers of a fourth wave)
      old[0] = load8(bounds, D / 2);
      old[1] = load8(bounds + D, D / 2);
    }
    Bounds8 own;
    own.clear();
    for (int i = row; i < n; i += kTokens) {
      Rows8 k = load8(p.k + (int64_t)(t0 + i) * p.k_st + kvh * p.k_sh + 8 * c, D / 2);
      if (p.cos != nullptr) {
        const Angles a = angles_of(p, x.position + x.shift + i, c);
        k = normed ? rotated<T, kPieces>(k, a, &norm, p.norm_eps) : rotated<T, kPieces>(k, a);
      }
      if (MORE && p.k_out != nullptr) store8(p.k_out + (int64_t)(t0 + i) * p.ko_st + kvh * p.ko_sh + 8 * c, D / 2, k);
      if (MORE && p.weights != nullptr && c == 0) p.weights[(((int64_t)x.at * p.n_kv_heads + kvh) << p.page_log) + x.slot + i] = 0.f;
      store8(p.keys + x.at * p.kp_sp + kvh * p.kp_sh + (x.slot + i) * p.kp_sn + 8 * c, D / 2, k);
      uint32_t w[8];  // (of the keys as stored)
      words(k, w);
      own.widen(w, w);
    }
    if (p.bounds == nullptr) continue;
    if (n > 1) {  // over the tokens of a wave
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        own.lo[j] = over_tokens<kPieces>(own.lo[j], least);
        own.hi[j] = over_tokens<kPieces>(own.hi[j], most);
      }
    }
    if (WAVES > 1 && n > kInWave) {  // over the waves
      if (wave > 0 && lane < kPieces) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          red[wave - 1][c][j] = own.lo[j];
          red[wave - 1][c][8 + j] = own.hi[j];
        }
      }
      __syncthreads();
      if (row == 0) {
#pragma unroll
        for (int w = 0; w < WAVES - 1; ++w) {
          uint32_t low[8], high[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            low[j] = red[w][c][j];
            high[j] = red[w][c][8 + j];
          }
          own.widen(low, high);
        }
      }
      __syncthreads();
    }
    if (writes) {
      if (x.slot != 0) {
        if (MORE) {
          old[0] = load8(bounds, D / 2);
          old[1] = load8(bounds + D, D / 2);
        }
        uint32_t low[8], high[8];
        words(old[0], low);
        words(old[1], high);
        own.widen(low, high);
      }
      Rows8 lo, hi;
      bounds_of<T>(own, lo, hi);
      store8(bounds, D / 2, lo);
      store8(bounds + D, D / 2, hi);
    }
  }
}

// Work-groups of the same tokens are one XCD's, one after the other, so that its L2 reads their cosines and sines once (a prompt of
// 6001 tokens, 32/8 heads of 128 32.3 -> 29.7 us).  Turns are dealt out by a hash, since runs may begin every so many work-groups: 64 tokens of a sequence each and a
// prompt of 2000 took 20.3 us in plain order, 15.8 so, 18.3 with the KV heads' work-groups spread over the XCDs.
constexpr uint32_t kXcds = 8;
template <typename T, int D, int WAVES, bool MORE>
__global__ void __launch_bounds__(64 * WAVES, MORE ? 4 : 1) paged_append_kernel(const PagedAppendArgs p) {
  __shared__ uint32_t red[WAVES > 1 ? WAVES - 1 : 1][D / 16][16];
  const uint32_t xcd = blockIdx.x % kXcds, of_xcd = blockIdx.x / kXcds, turn = of_xcd / p.n_kv_heads;
  const int kvh = of_xcd - turn * p.n_kv_heads, at = turn * kXcds + (xcd + (turn * 0x9e3779b1u >> 29)) % kXcds;
  if (at < p.key_chunks) keys_and_bounds<T, D, WAVES, MORE>(p, at * p.chunk, kvh, red);
  else queries_and_values<T, D, MORE>(p, (at - p.key_chunks) * (WAVES * 1024 / D), kvh);
}

template <typename T, int D, bool MORE>
static void launch_paged_append_for(PagedAppendArgs a, hipStream_t stream) {
  // Tokens of a work-group of keys: few, so that short runs do not queue up in one, but no fewer than make some thousand work-groups (prompts of 700 to 21000 tokens,
  // 32/8 heads of 128: 205 us, with 1 everywhere some 600; 200 sequences of a token, padded to 256: 14, with a page everywhere 109; 64 of a token and a prompt of 2000: 18, 122)
  const int64_t most = (int64_t)a.n_tokens * a.n_kv_heads / 4096, page_size = 1 << a.page_log;
  a.chunk = a.starts == nullptr || most < 1 ? 1 : (int)(most < page_size ? most : page_size);
  a.key_chunks = (a.n_tokens + a.chunk - 1) / a.chunk;
  // waves of a work-group: as many as the tokens of a page fill
  const int waves = a.starts == nullptr ? 1 : (int)(page_size * (D / 16) / 64), w = waves <= 1 ? 1 : waves == 2 ? 2 : 4;
  const uint32_t chunks = a.key_chunks + (a.n_tokens + w * 1024 / D - 1) / (w * 1024 / D);
  const dim3 grid((chunks + kXcds - 1) / kXcds * kXcds * a.n_kv_heads);
  if (w == 1) hipLaunchKernelGGL((paged_append_kernel<T, D, 1, MORE>), grid, dim3(64), 0, stream, a);
  else if (w == 2) hipLaunchKernelGGL((paged_append_kernel<T, D, 2, MORE>), grid, dim3(128), 0, stream, a);
  else hipLaunchKernelGGL((paged_append_kernel<T, D, 4, MORE>), grid, dim3(256), 0, stream, a);
}

template <typename T, int D>
static void launch_paged_append_of(const PagedAppendArgs& a, hipStream_t stream) {
  if (a.q_norm != nullptr || a.k_norm != nullptr || a.k_out != nullptr || a.positions != nullptr || a.weights != nullptr) launch_paged_append_for<T, D, true>(a, stream);
  else launch_paged_append_for<T, D, false>(a, stream);
}

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t stream) {
  if (a.head_dim == 128) {
    if (a.dtype == 0) launch_paged_append_of<Bf16, 128>(a, stream);
    else launch_paged_append_of<F16, 128>(a, stream);
  } else {
    if (a.dtype == 0) launch_paged_append_of<Bf16, 64>(a, stream);
    else launch_paged_append_of<F16, 64>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace aa
