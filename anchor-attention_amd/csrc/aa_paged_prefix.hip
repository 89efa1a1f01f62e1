// Attention of one new token per sequence over the first pages of its group's sequences, which all of them share, on gfx950: the state (maximum, sum,
// accumulator) of each head over the prefix, which the decode kernel joins with the sequence's own keys.
//
// The heads of a KV head's queries, of all sequences of the group, are rows of one product, so that keys and values are read once for 16 * BLOCKS of them.  A unit is a
// (group, KV head, 16 * BLOCKS rows); its keys come in tiles of 32.  The tiles of all units, one after the other, are cut into equal shares, one for each of a
// fixed number of work-groups; inside a share a unit's tiles are its four waves', each with accumulators of its own, joined through LDS.  A unit that several shares
// have is joined by paged_prefix_join_kernel in order, so that results do not depend on timing.
//
// Inside a wave, as in the decode kernel: S^T = K Q^T straight from memory, P^T in S^T's registers, V turned by v_perm once for all rows, P as two 16-bit numbers.
#include "aa_kernels.h"
#include "aa_nonfinite.h"
#include "aa_paged.h"

namespace aa {

constexpr int kPrefixTile = 32, kPrefixWaves = 4, kPrefixShares = 256, kPrefixSharesLog = 8;
constexpr int kPrefixLeast = 8;  // tiles of a share at least

// A group's sequences and prefix; nothing that memory says is trusted.
struct PagedGroup {
  int first, sequences, pages;
};
__device__ __forceinline__ PagedGroup group_at(const PagedPrefixArgs& p, const int g) {
  PagedGroup x;
  if (p.groups == nullptr) return {0, p.step.batch, min(max(p.shared_pages[0], 0), p.step.max_pages)};
  x.first = min(max(p.groups[g], 0), p.step.batch);
  x.sequences = max(min(max(p.groups[g + 1], 0), p.step.batch) - x.first, 0);
  x.pages = min(max(p.shared_pages[g], 0), p.step.max_pages);
  return x;
}

template <typename T, int D, int BLOCKS>
__global__ void __launch_bounds__(64 * kPrefixWaves, 1) paged_prefix_kernel(const PagedPrefixArgs all) {
  constexpr int kKS = D / 32;  // MFMAs of a score
  constexpr int kDV = D / 16;  // channels of V that a lane loads
  constexpr int kVW = kDV / 2;
  constexpr int kRows = 16 * BLOCKS, kPitch = D + 4;
  extern __shared__ __attribute__((aligned(16))) float states[];  // [wave][row][kPitch]: the accumulator, maximum and sum
  const PagedDecodeArgs& p = all.step;
  const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = p.n_q_heads / p.n_kv_heads, page_size = 1 << p.page_log;

  // ---- whose prefixes count: sequences that are as long -----------------------------------------------
  for (int b = blockIdx.x * 256 + tid; b < p.batch; b += kPrefixShares * 256) {
    int from = 0, to = all.groups == nullptr ? 0 : all.n_groups;  // groups that end at or before b
    while (from < to) {
      const int mid = (from + to) >> 1;
      if (all.groups[mid + 1] <= b) from = mid + 1;
      else to = mid;
    }
    int skip = 0;
    if (from < all.n_groups) {
      const PagedGroup x = group_at(all, from);
      if (b >= x.first && b < x.first + x.sequences && clamped_length(p.lengths, b, p.max_pages, p.page_log) >= x.pages << p.page_log) skip = x.pages;
    }
    p.skips[b] = skip;
  }

  // ---- this work-group's share ---------------------------------------------------------------------
  auto tiles_of = [&](const PagedGroup& x) { return ((x.pages << p.page_log) + kPrefixTile - 1) / kPrefixTile; };
  auto blocks_of = [&](const PagedGroup& x) { return (x.sequences * heads + kRows - 1) / kRows; };
  auto extent_of = [&](const int i) {  // of group i's units
    if (i >= all.n_groups) return (int64_t)0;
    const PagedGroup x = group_at(all, i);
    return (int64_t)tiles_of(x) * blocks_of(x) * p.n_kv_heads;
  };
  auto up_to_lane = [&](int64_t x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int64_t y = __shfl_up((long long)x, d, 64);
      x += lane >= d ? y : 0;
    }
    return x;
  };
  int64_t total = 0;
  for (int i = 0; i < all.n_groups; i += 64) total += __shfl((long long)up_to_lane(extent_of(i + lane)), 63, 64);
  const int64_t share = max((total + (kPrefixShares - 1)) >> kPrefixSharesLog, (int64_t)kPrefixLeast);
  int64_t at = min(share * blockIdx.x, total);
  const int64_t end = min(at + share, total);
  int group = 0;
  int64_t start = 0;  // of the group
  if (at < end) {
    for (int i = 0; i < all.n_groups; i += 64) {
      const int64_t sum = up_to_lane(extent_of(i + lane));
      const int in = __popcll(__ballot(start + sum <= at));
      if (in < 64) {
        group = i + in;
        if (in > 0) start += __shfl((long long)sum, in - 1, 64);
        break;
      }
      start += __shfl((long long)sum, 63, 64);
    }
  }
  int4* header = reinterpret_cast<int4*>(all.headers) + blockIdx.x;
  if (tid == 0) header->x = 0;

  const float scale = p.sm_scale * kLog2e;
  const uint32_t k_lane = (2u * (c16 * (uint32_t)p.kp_sn + 8 * g)) & 0xfffffu, v_lane = (2u * (4 * g * (uint32_t)p.vp_sn + kDV * c16)) & 0xfffffu;
  struct Tile {
    u32x4 k[2][kKS];
    uint32_t v[8][kVW];
  };
  while (at < end && group < all.n_groups) {
    PagedGroup x = group_at(all, group);
    x.first = __builtin_amdgcn_readfirstlane(x.first);
    x.sequences = __builtin_amdgcn_readfirstlane(x.sequences);
    x.pages = __builtin_amdgcn_readfirstlane(x.pages);
    const int tiles = tiles_of(x), blocks = blocks_of(x), length = x.pages << p.page_log, rows = x.sequences * heads;
    if (at - start >= (int64_t)tiles * blocks * p.n_kv_heads) {  // (the next group, perhaps of nothing)
      start += (int64_t)tiles * blocks * p.n_kv_heads;
      ++group;
      continue;
    }
    const uint32_t unit = (uint32_t)((at - start) / tiles), block = unit % (uint32_t)blocks, kvh = unit / (uint32_t)blocks;
    const int t0 = (int)(at - start - (int64_t)unit * tiles), t1 = (int)min((int64_t)tiles, t0 + (end - at));
    const int row0 = block * kRows, n_blocks = min(BLOCKS, (rows - row0 + 15) / 16);
    const int from = t0 + (t1 - t0) * wave / kPrefixWaves, to = t0 + (t1 - t0) * (wave + 1) / kPrefixWaves;

    u32x4 q[BLOCKS][kKS];
#pragma unroll
    for (int c = 0; c < BLOCKS; ++c) {
      const int row = min(row0 + 16 * c + c16, rows - 1), s = row / heads;
      const uint16_t* qp = p.q + (int64_t)(x.first + s) * p.q_sb + (int64_t)((int)kvh * heads + row - s * heads) * p.q_sh + 8 * g;
#pragma unroll
      for (int s = 0; s < kKS; ++s) q[c][s] = *reinterpret_cast<const u32x4*>(qp + 32 * s);
    }
    const const_i32* table = (const_i32*)(p.table + x.first * p.t_sb);
    struct Spot {
      int64_t k[2], v[2];
      int rows[2];
    };
    auto spot = [&](const int t) __attribute__((always_inline)) {
      Spot o;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int key = kPrefixTile * t + 16 * half, row = key & (page_size - 1);
        const int64_t page = clamped_page(table[min(key >> p.page_log, x.pages - 1)], p.n_pages);
        o.k[half] = page * p.kp_sp + row * p.kp_sn + kvh * p.kp_sh;
        o.v[half] = page * p.vp_sp + row * p.vp_sn + kvh * p.vp_sh;
        o.rows[half] = key < length ? 16 : 0;
      }
      return o;
    };
    auto load_k = [&](Tile& y, const Spot& o) __attribute__((always_inline)) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const Rows kr = rows_at(p.keys + o.k[half], o.rows[half] * (2 * (int)p.kp_sn));
#pragma unroll
        for (int s = 0; s < kKS; ++s) y.k[half][s] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_lane + 64 * s, 0, 0);
      }
    };
    auto load_v = [&](Tile& y, const Spot& o) __attribute__((always_inline)) {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const Rows vr = rows_at(p.values + o.v[half], o.rows[half] * (2 * (int)p.vp_sn));
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if constexpr (kVW == 4) *reinterpret_cast<u32x4*>(y.v[4 * half + r]) = __builtin_amdgcn_raw_buffer_load_b128(vr, v_lane, 2 * r * (uint32_t)p.vp_sn, 0);
          else *reinterpret_cast<u32x2*>(y.v[4 * half + r]) = __builtin_amdgcn_raw_buffer_load_b64(vr, v_lane, 2 * r * (uint32_t)p.vp_sn, 0);
        }
      }
    };
    float m_run[BLOCKS], l_run[BLOCKS];
    floatx4 acc[BLOCKS][kDV];
    auto clear = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < BLOCKS; ++c) {
        l_run[c] = 0.f;
#pragma unroll
        for (int j = 0; j < kDV; ++j) acc[c][j] = floatx4{0.f, 0.f, 0.f, 0.f};
      }
    };
    clear();
#pragma unroll
    for (int c = 0; c < BLOCKS; ++c) m_run[c] = -INFINITY;

    // (the last tile of a prefix of 16 * odd keys has no second half)
    auto seen = [&](const int t, const int i) __attribute__((always_inline)) { return kPrefixTile * t + 16 * (i >> 2) < length; };
    auto scores = [&](const Tile& y, floatx4 (&s)[BLOCKS][2]) __attribute__((always_inline)) {
#pragma unroll
      for (int c = 0; c < BLOCKS; ++c) {
        if (c > 0 && c >= n_blocks) break;
        s[c][0] = s[c][1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kKS; ++i)
#pragma unroll
          for (int half = 0; half < 2; ++half) s[c][half] = mfma16<T>(y.k[half][i], q[c][i], s[c][half]);
      }
    };
    auto probabilities = [&](floatx4 (&s)[2], const int t, const int c, u32x4& prob, u32x4& rest, const bool exact) __attribute__((always_inline)) {
      if (kPrefixTile * (t + 1) > length) {
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = seen(t, i) ? s[i >> 2][i & 3] : -INFINITY;
      }
      float mx = s[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
      const float m_new = fmaxf(m_run[c], max_over_quarters(mx));
      const float m_base = m_new == -INFINITY ? 0.f : m_new;
      if (__any(m_new > m_run[c])) {
        const float alpha = fast_exp2((m_run[c] - m_base) * scale);
        l_run[c] *= alpha;
#pragma unroll
        for (int j = 0; j < kDV; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[c][j][r] *= alpha;
        m_run[c] = m_new;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e0 = prob_exp2<T>(s[i >> 1][2 * (i & 1)] - m_base, scale), e1 = prob_exp2<T>(s[i >> 1][2 * (i & 1) + 1] - m_base, scale);
        l_run[c] += e0 + e1;
        uint32_t w = T::pack(e0, e1);
        if (exact) {
          if (e0 > 0.f && (w & 0xffffu) == 0u) w |= 1u;
          if (e1 > 0.f && (w >> 16) == 0u) w |= 0x10000u;
        }
        prob[i] = w;
        rest[i] = T::pack_rest(e0, e1, w);
      }
    };
    auto add_values = [&](Tile& y, const int t, const u32x4 (&prob)[BLOCKS], const u32x4 (&rest)[BLOCKS], const bool exact) __attribute__((always_inline)) {
#pragma unroll
      for (int w = 0; w < kVW; ++w)
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          u32x4 v, finite;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = finite[i] = __builtin_amdgcn_perm(y.v[2 * i + 1][w], y.v[2 * i][w], odd ? 0x07060302u : 0x05040100u);
          if (exact) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if ((v[i] & T::kExponent) == T::kExponent) finite[i] &= 0xffff0000u;
              if (((v[i] >> 16) & T::kExponent) == T::kExponent) finite[i] &= 0xffffu;
            }
          }
#pragma unroll
          for (int c = 0; c < BLOCKS; ++c) {
            if (c > 0 && c >= n_blocks) break;
            acc[c][2 * w + odd] = mfma16<T>(v, prob[c], acc[c][2 * w + odd]);
            acc[c][2 * w + odd] = mfma16<T>(finite, rest[c], acc[c][2 * w + odd]);
          }
        }
    };

    Tile y;
    if (from < to) {
      const Spot o = spot(from);
      load_k(y, o);
      __builtin_amdgcn_sched_barrier(0);
      load_v(y, o);
    }
    for (int t = from; t < to; ++t) {
      const Spot o = spot(min(t + 1, to - 1));
      floatx4 s[BLOCKS][2];
      scores(y, s);
      __builtin_amdgcn_sched_barrier(0);
      load_k(y, o);
      __builtin_amdgcn_sched_barrier(0);
      u32x4 prob[BLOCKS], rest[BLOCKS];
#pragma unroll
      for (int c = 0; c < BLOCKS; ++c) {
        if (c > 0 && c >= n_blocks) break;
        probabilities(s[c], t, c, prob[c], rest[c], false);
      }
      add_values(y, t, prob, rest, false);
      __builtin_amdgcn_sched_barrier(0);
      load_v(y, o);
    }
    bool again = false;
#pragma unroll
    for (int c = 0; c < BLOCKS; ++c) {
      l_run[c] = sum_over_quarters(l_run[c]);
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < kDV; ++j) sum += (acc[c][j][0] + acc[c][j][1]) + (acc[c][j][2] + acc[c][j][3]);
      again |= is_nan(sum) && !is_nan(l_run[c]);
    }
    if (__builtin_expect(__any(again), 0)) {
      // Infinite values: with two products per key they give NaN.  Once more, relative to the maximum: the rest meets the finite values only and a positive
      // probability does not round to 0.
      clear();
      for (int t = from; t < to; ++t) {
        Tile z;
        const Spot o = spot(t);
        load_k(z, o);
        load_v(z, o);
        floatx4 s[BLOCKS][2];
        scores(z, s);
        u32x4 prob[BLOCKS], rest[BLOCKS];
#pragma unroll
        for (int c = 0; c < BLOCKS; ++c) {
          if (c > 0 && c >= n_blocks) break;
          probabilities(s[c], t, c, prob[c], rest[c], true);
        }
        add_values(z, t, prob, rest, true);
      }
#pragma unroll
      for (int c = 0; c < BLOCKS; ++c) l_run[c] = sum_over_quarters(l_run[c]);
    }

    // ---- the waves' states -> the unit's, or a part of it -----------------------------------------------
#pragma unroll
    for (int c = 0; c < BLOCKS; ++c) {
      if (c > 0 && c >= n_blocks) break;
      float* to_lds = states + (wave * kRows + 16 * c + c16) * kPitch;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < kDV; j += 4)
          *reinterpret_cast<floatx4*>(to_lds + kDV * (4 * g + r) + j) = floatx4{acc[c][j][r], acc[c][j + 1][r], acc[c][j + 2][r], acc[c][j + 3][r]};
      if (g == 0) *reinterpret_cast<floatx2*>(to_lds + D) = floatx2{m_run[c], l_run[c]};
    }
    __syncthreads();
    const bool begins = t0 == 0, ends = t1 == tiles;
    for (int i = tid; i < 16 * n_blocks * (D / 4); i += 64 * kPrefixWaves) {
      const int r = i / (D / 4), d = 4 * (i % (D / 4)), row = row0 + r;
      if (row >= rows) break;  // (rows ascend)
      float m = -INFINITY, l = 0.f, ms[kPrefixWaves];
      floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kPrefixWaves; ++w) {
        ms[w] = states[(w * kRows + r) * kPitch + D];
        m = fmaxf(m, ms[w]);
      }
#pragma unroll
      for (int w = 0; w < kPrefixWaves; ++w) {
        const float weight = ms[w] == -INFINITY ? 0.f : fast_exp2((ms[w] - m) * scale);
        const floatx4 part = *reinterpret_cast<const floatx4*>(states + (w * kRows + r) * kPitch + d);
        l += weight * states[(w * kRows + r) * kPitch + D + 1];
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += weight * part[e];
      }
      int64_t to_row;
      float *sums, *stats;
      if (begins && ends) {
        const int s = row / heads;
        to_row = (int64_t)(x.first + s) * p.n_q_heads + (int)kvh * heads + row - s * heads;
        sums = p.prefix;
        stats = p.prefix_stats;
      } else {
        to_row = (int64_t)(2 * blockIdx.x + (begins ? 1 : 0)) * kRows + r;
        sums = all.parts;
        stats = all.part_stats;
      }
      *reinterpret_cast<floatx4*>(sums + to_row * D + d) = sum;
      if (d == 0) *reinterpret_cast<floatx2*>(stats + 2 * to_row) = floatx2{m, l};
    }
    if (begins && !ends && tid == 0) {  // its other parts are the next work-groups'
      const int64_t last = start + (int64_t)(unit + 1) * tiles - 1;
      *header = int4{(int)(last / share) - (int)blockIdx.x + 1, group, (int)kvh, (int)block};
    }
    __syncthreads();
    at += t1 - t0;
  }
}

// Joins the parts of a unit that begins in share blockIdx.x and ends in another, a row by a wave.
template <int D, int BLOCKS>
__global__ void __launch_bounds__(256) paged_prefix_join_kernel(const PagedPrefixArgs all) {
  constexpr int kRows = 16 * BLOCKS, kEach = D / 64;
  typedef float floats __attribute__((ext_vector_type(kEach)));
  const PagedDecodeArgs& p = all.step;
  const int lane = threadIdx.x & 63, r = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int4 header = *reinterpret_cast<const int4*>(all.headers + 4 * blockIdx.x);
  const int parts = header.x, heads = p.n_q_heads / p.n_kv_heads;
  if (parts == 0) return;
  const PagedGroup x = group_at(all, header.y);
  const int row = header.w * kRows + r;
  if (row >= x.sequences * heads) return;
  const float scale = p.sm_scale * kLog2e;
  // the first part is the second of its share, the others the first of theirs
  auto part = [&](const int i) { return ((int64_t)2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * kRows + r; };
  float m = -INFINITY;
  for (int i = lane; i < parts; i += 64) m = fmaxf(m, all.part_stats[2 * part(i)]);
  m = over_wave(m, -INFINITY, [](const float a, const float b) { return fmaxf(a, b); });
  float l = 0.f;
  floats sum = {};
  for (int i = 0; i < parts; ++i) {
    const float mi = all.part_stats[2 * part(i)], w = mi == -INFINITY ? 0.f : fast_exp2((mi - m) * scale);
    l += w * all.part_stats[2 * part(i) + 1];
    const floats y = *reinterpret_cast<const floats*>(all.parts + part(i) * D + kEach * lane);
#pragma unroll
    for (int e = 0; e < kEach; ++e) sum[e] += w * y[e];
  }
  const int s = row / heads;
  const int64_t to = (int64_t)(x.first + s) * p.n_q_heads + header.z * heads + row - s * heads;
  *reinterpret_cast<floats*>(p.prefix + to * D + kEach * lane) = sum;
  if (lane == 0) *reinterpret_cast<floatx2*>(p.prefix_stats + 2 * to) = floatx2{m, l};
}

// Rows of a unit, in blocks of 16: as many as a KV head's queries of the batch fill, and their accumulators leave registers for.
static int prefix_blocks(int batch, int n_q_heads, int n_kv_heads, int head_dim) {
  const int64_t rows = (int64_t)batch * (n_q_heads / n_kv_heads);
  return rows <= 16 ? 1 : rows <= 32 || head_dim == 128 ? 2 : 4;
}

PagedScratch paged_prefix_scratch(int batch, int n_q_heads, int n_kv_heads, int head_dim) {
  const size_t rows = (size_t)kPrefixShares * 2 * 16 * prefix_blocks(batch, n_q_heads, n_kv_heads, head_dim);
  PagedScratch s = {0, 0, 0, 0};
  s.stats = (size_t)kPrefixShares * 16;
  s.parts = s.stats + rows * 8;
  s.total = s.parts + rows * head_dim * 4;
  return s;
}

template <typename T, int D, int BLOCKS>
static hipError_t launch_paged_prefix_for(const PagedPrefixArgs& a, hipStream_t stream) {
  constexpr size_t lds = (size_t)kPrefixWaves * 16 * BLOCKS * (D + 4) * 4;
  hipLaunchKernelGGL((paged_prefix_kernel<T, D, BLOCKS>), dim3(kPrefixShares), dim3(64 * kPrefixWaves), lds, stream, a);
  hipLaunchKernelGGL((paged_prefix_join_kernel<D, BLOCKS>), dim3(kPrefixShares, 4 * BLOCKS), dim3(256), 0, stream, a);
  return hipGetLastError();
}
template <typename T, int D>
static hipError_t launch_paged_prefix_of(const PagedPrefixArgs& a, hipStream_t stream) {
  const int blocks = prefix_blocks(a.step.batch, a.step.n_q_heads, a.step.n_kv_heads, D);
  if (blocks == 1) return launch_paged_prefix_for<T, D, 1>(a, stream);
  if (blocks == 2) return launch_paged_prefix_for<T, D, 2>(a, stream);
  return launch_paged_prefix_for<T, D, D == 128 ? 2 : 4>(a, stream);
}
hipError_t launch_paged_prefix(const PagedPrefixArgs& a, hipStream_t stream) {
  if (a.step.head_dim == 128) return a.step.dtype == 0 ? launch_paged_prefix_of<Bf16, 128>(a, stream) : launch_paged_prefix_of<F16, 128>(a, stream);
  return a.step.dtype == 0 ? launch_paged_prefix_of<Bf16, 64>(a, stream) : launch_paged_prefix_of<F16, 64>(a, stream);
}

}  // namespace aa
