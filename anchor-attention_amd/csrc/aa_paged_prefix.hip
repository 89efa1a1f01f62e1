// Attention of one new token per sequence over the first pages of its group's sequences, which all of them share, on gfx950: of each head over the prefix the largest score m, the sum l of
// 2^((score - m) * scale) and the accumulator of these times the values.  The decode kernel has the same of the sequence's own keys, and paged_finish_kernel joins them:
//   o = (w a + w' a') / (w l + w' l'),  w = 2^((m - max(m, m')) * scale).
//
// The heads of a KV head's queries, of all sequences of the group, are rows of one product, so that keys and values are read once for 16 or 128 of them (takes_many).  A unit is a
// (group, KV head, rows); its keys come in tiles of 32 or 64.  The tiles of all units, one after the other, are cut into equal shares, one for each of a fixed number of
// work-groups.  A unit that several shares have is joined in their order, so that results do not depend on timing.
//
// Of 16 rows a share's tiles are its eight waves', each with accumulators of its own, joined through LDS: inside a wave, as in the decode kernel, S^T = K Q^T straight from memory, P^T in
// S^T's registers, V turned by v_perm, P as two 16-bit numbers.  It is bound by memory: 4 sequences behind 32768 keys, 32/8 heads of 128 (134 MB), in 26.8 us, near the rate of a copy;
// behind 8192 in 13.0.
// Of 128 rows: below.
#include <type_traits>

#include "aa_kernels.h"
#include "aa_nonfinite.h"
#include "aa_paged.h"

namespace aa {

constexpr int kPrefixShares = 256, kPrefixSharesLog = 8, kPrefixWaves = 8, kPrefixThreads = 64 * kPrefixWaves;
// How the work is cut: keys of a tile and rows of a unit; tiles of a share at least; what a unit costs beside its tiles, in tiles
struct PrefixForm {
  int tile, rows, least, over;
};
constexpr PrefixForm kFew = {32, 16, 8, 4}, kMany = {64, 128, 4, 10};

// A group's sequences and prefix; nothing that memory says is trusted.
struct PagedGroup {
  int first, sequences, pages;
};
template <typename Words>
__device__ __forceinline__ PagedGroup group_of(const PagedPrefixArgs& p, const Words* groups, const Words* shared_pages, const int g) {
  PagedGroup x = {0, p.step.batch, 0};
  if (p.groups != nullptr) {
    x.first = min(max(groups[g], 0), p.step.batch);
    x.sequences = max(min(max(groups[g + 1], 0), p.step.batch) - x.first, 0);
  }
  x.pages = x.sequences > 1 ? min(max(shared_pages[g], 0), p.step.max_pages) : 0;  // (one alone shares nothing)
  return x;
}
// of a lane's group, and of one that all lanes have (by scalar loads, which are there sooner)
__device__ __forceinline__ PagedGroup group_at(const PagedPrefixArgs& p, const int g) { return group_of(p, p.groups, p.shared_pages, g); }
__device__ __forceinline__ PagedGroup common_group_at(const PagedPrefixArgs& p, const int g) {
  return group_of(p, (const_i32*)p.groups, (const_i32*)p.shared_pages, __builtin_amdgcn_readfirstlane(g));
}

// How many of a sequence's first pages its group's state stands for: those that are shared, if it is as long, or none; and the group's first sequence.
__device__ __forceinline__ void find_skips(const PagedPrefixArgs& all, const int tid, const int threads) {
  const PagedDecodeArgs& p = all.step;
  for (int b = blockIdx.x * threads + tid; b < p.batch; b += kPrefixShares * threads) {
    int from = 0, to = all.groups == nullptr ? 0 : all.n_groups;  // groups that end at or before b
    while (from < to) {
      const int mid = (from + to) >> 1;
      if (all.groups[mid + 1] <= b) from = mid + 1;
      else to = mid;
    }
    int skip = 0, first = 0;
    if (from < all.n_groups) {
      const PagedGroup x = group_at(all, from);
      if (b >= x.first && b < x.first + x.sequences && clamped_length(p.lengths, b, p.max_pages, p.page_log) >= x.pages << p.page_log) skip = x.pages;
      first = x.first;
    }
    p.skips[b] = skip;
    p.firsts[b] = first;
  }
}

// Where the states of a unit's rows are, by its first row: the share that it begins in and how many have parts of it (0: it is whole)
template <int ROWS>
__device__ __forceinline__ void note_unit(const PagedDecodeArgs& p, const int first, const int kvh, const int block, const int heads, const int share, const int parts) {
  const int row0 = ROWS * block, s = row0 / heads;
  *reinterpret_cast<int2*>(p.entries + 2 * ((int64_t)(first + s) * p.n_q_heads + kvh * heads + row0 - s * heads)) = int2{share, parts};
}

// a number that all lanes have, in scalar registers
__device__ __forceinline__ int64_t uniform(const int64_t x) {
  return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)x >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x));
}

__device__ __forceinline__ int tiles_of(const PagedDecodeArgs& p, const PrefixForm& form, const PagedGroup& x) {
  return ((x.pages << p.page_log) + form.tile - 1) / form.tile;
}
__device__ __forceinline__ int blocks_of(const PrefixForm& form, const PagedGroup& x, const int heads) {
  return (x.sequences * heads + form.rows - 1) / form.rows;
}
// A unit's extent: its tiles, and before them what its beginning and end cost, in tiles (0 where there are none)
__device__ __forceinline__ int extent_of(const PrefixForm& form, const int tiles) { return tiles > 0 ? tiles + form.over : 0; }
// ... of all of a group's units
__device__ __forceinline__ int64_t extents_in(const PagedDecodeArgs& p, const PrefixForm& form, const PagedGroup& x) {
  return (int64_t)extent_of(form, tiles_of(p, form, x)) * blocks_of(form, x, p.n_q_heads / p.n_kv_heads) * p.n_kv_heads;
}
// the group of the lane's number from i on, one of nothing where there is none
__device__ __forceinline__ PagedGroup lane_group_at(const PagedPrefixArgs& all, const int i) {
  const int g = i + (int)(threadIdx.x & 63);
  return g < all.n_groups ? group_at(all, g) : PagedGroup{0, 0, 0};
}
__device__ __forceinline__ int64_t up_to_lane(int64_t x) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t y = __shfl_up((long long)x, d, 64);
    x += lane >= d ? y : 0;
  }
  return x;
}
// All units' extents in either form, found by every wave for itself; `mine`, the group of the lane's number.
struct PrefixTotals {
  int64_t few, many;
};
__device__ __forceinline__ PrefixTotals totals_of(const PagedPrefixArgs& all, const PagedGroup& mine) {
  PrefixTotals t = {0, 0};
  if (all.n_groups == 1) {
    const PagedGroup x = common_group_at(all, 0);
    return {extents_in(all.step, kFew, x), extents_in(all.step, kMany, x)};
  }
  for (int i = 0; i < all.n_groups; i += 64) {
    const PagedGroup x = i == 0 ? mine : lane_group_at(all, i);
    t.few += __shfl((long long)up_to_lane(extents_in(all.step, kFew, x)), 63, 64);
    t.many += __shfl((long long)up_to_lane(extents_in(all.step, kMany, x)), 63, 64);
  }
  return {uniform(t.few), uniform(t.many)};
}
__device__ __forceinline__ int64_t length_of_share(const PrefixForm& form, const int64_t total) {
  return max((total + (kPrefixShares - 1)) >> kPrefixSharesLog, (int64_t)form.least);
}
// The share-th of kPrefixShares equal parts of all units' extents, and the group that it begins in.
struct PrefixShare {
  int64_t at, end, share, start;  // from, to; how long a share is; where the group begins
  int group;
};
__device__ __forceinline__ PrefixShare share_of(const PagedPrefixArgs& all, const PrefixForm& form, const int64_t total, const PagedGroup& mine, const int share) {
  PrefixShare r = {0, 0, length_of_share(form, total), 0, 0};
  r.at = min(r.share * share, total);
  r.end = min(r.at + r.share, total);
  if (r.at < r.end && all.n_groups > 1) {
    for (int i = 0; i < all.n_groups; i += 64) {
      const int64_t sum = up_to_lane(extents_in(all.step, form, i == 0 ? mine : lane_group_at(all, i)));
      const int in = __popcll(__ballot(r.start + sum <= r.at));
      if (in < 64) {
        r.group = i + in;
        if (in > 0) r.start += __shfl((long long)sum, in - 1, 64);
        break;
      }
      r.start += __shfl((long long)sum, 63, 64);
    }
  }
  return {uniform(r.at), uniform(r.end), uniform(r.share), uniform(r.start), (int)__builtin_amdgcn_readfirstlane(r.group)};
}

// `states`: [wave][row][kPitch] floats of LDS, the accumulator, maximum and sum
template <typename T, int D>
__device__ __forceinline__ void few_rows(const PagedPrefixArgs& all, const int64_t total, const PagedGroup& lanes, float* states) {
  constexpr int kKS = D / 32;  // MFMAs of a score
  constexpr int kDV = D / 16;  // channels of V that a lane loads
  constexpr int kVW = kDV / 2;
  constexpr int kRows = kFew.rows, kTile = kFew.tile, kPitch = D + 4;
  const PagedDecodeArgs& p = all.step;
  const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int heads = p.n_q_heads / p.n_kv_heads, page_size = 1 << p.page_log;

  // ---- this work-group's share ---------------------------------------------------------------------
  const PrefixShare mine = share_of(all, kFew, total, lanes, blockIdx.x);
  int64_t at = mine.at, start = mine.start;
  const int64_t end = mine.end, share = mine.share;
  int group = mine.group;

  const float scale = p.sm_scale * kLog2e;
  const uint32_t k_lane = (2u * (c16 * (uint32_t)p.kp_sn + 8 * g)) & 0xfffffu, v_lane = (2u * (4 * g * (uint32_t)p.vp_sn + kDV * c16)) & 0xfffffu;
  struct Tile {
    u32x4 k[2][kKS];
    uint32_t v[8][kVW];
  };
  while (at < end && group < all.n_groups) {
    at = uniform(at), start = uniform(start), group = __builtin_amdgcn_readfirstlane(group);  // (which the compiler does not see of what a loop carries)
    const PagedGroup x = common_group_at(all, group);
    const int tiles = tiles_of(p, kFew, x), blocks = blocks_of(kFew, x, heads), length = x.pages << p.page_log, rows = x.sequences * heads;
    const int extent = extent_of(kFew, tiles);
    if (at - start >= (int64_t)extent * blocks * p.n_kv_heads) {  // (the next group, perhaps of nothing)
      start += (int64_t)extent * blocks * p.n_kv_heads;
      ++group;
      continue;
    }
    const uint32_t unit = (uint32_t)((at - start) / extent), block = unit % (uint32_t)blocks, kvh = unit / (uint32_t)blocks;
    const int64_t unit_end = start + (int64_t)(unit + 1) * extent, until = min(end, unit_end);
    const int t0 = max(tiles - (int)(unit_end - at), 0), t1 = max(tiles - (int)(unit_end - until), 0);
    if (t1 == 0) break;  // (nothing of it is in this share, which ends)
    const int row0 = block * kRows;
    const int from = t0 + (t1 - t0) * wave / kPrefixWaves, to = t0 + (t1 - t0) * (wave + 1) / kPrefixWaves;

    u32x4 q[kKS];
    {
      const int row = min(row0 + c16, rows - 1), s = row / heads;
      const uint16_t* qp = p.q + (int64_t)(x.first + s) * p.q_sb + (int64_t)((int)kvh * heads + row - s * heads) * p.q_sh + 8 * g;
#pragma unroll
      for (int s = 0; s < kKS; ++s) q[s] = *reinterpret_cast<const u32x4*>(qp + 32 * s);
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
        const int key = kTile * t + 16 * half, row = key & (page_size - 1);
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
    float m_run = -INFINITY, l_run;
    floatx4 acc[kDV];
    auto clear = [&]() __attribute__((always_inline)) {
      l_run = 0.f;
#pragma unroll
      for (int j = 0; j < kDV; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
    };
    clear();

    // (the last tile of a prefix of 16 * odd keys has no second half)
    auto seen = [&](const int t, const int i) __attribute__((always_inline)) { return kTile * t + 16 * (i >> 2) < length; };
    auto scores = [&](const Tile& y, floatx4 (&s)[2]) __attribute__((always_inline)) {
      s[0] = s[1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kKS; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) s[half] = mfma16<T>(y.k[half][i], q[i], s[half]);
    };
    auto probabilities = [&](floatx4 (&s)[2], const int t, u32x4& prob, u32x4& rest, const bool exact) __attribute__((always_inline)) {
      if (kTile * (t + 1) > length) {
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = seen(t, i) ? s[i >> 2][i & 3] : -INFINITY;
      }
      float mx = s[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
      const float m_new = fmaxf(m_run, max_over_quarters(mx));
      const float m_base = m_new == -INFINITY ? 0.f : m_new;
      if (__any(m_new > m_run)) {
        const float alpha = fast_exp2((m_run - m_base) * scale);
        l_run *= alpha;
#pragma unroll
        for (int j = 0; j < kDV; ++j)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[j][r] *= alpha;
        m_run = m_new;
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e0 = prob_exp2<T>(s[i >> 1][2 * (i & 1)] - m_base, scale), e1 = prob_exp2<T>(s[i >> 1][2 * (i & 1) + 1] - m_base, scale);
        l_run += e0 + e1;
        uint32_t w = T::pack(e0, e1);
        if (exact) {
          if (e0 > 0.f && (w & 0xffffu) == 0u) w |= 1u;
          if (e1 > 0.f && (w >> 16) == 0u) w |= 0x10000u;
        }
        prob[i] = w;
        rest[i] = T::pack_rest(e0, e1, w);
      }
    };
    auto add_values = [&](Tile& y, const int t, const u32x4& prob, const u32x4& rest, const bool exact) __attribute__((always_inline)) {
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
          acc[2 * w + odd] = mfma16<T>(v, prob, acc[2 * w + odd]);
          acc[2 * w + odd] = mfma16<T>(finite, rest, acc[2 * w + odd]);
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
      floatx4 s[2];
      scores(y, s);
      __builtin_amdgcn_sched_barrier(0);
      load_k(y, o);
      __builtin_amdgcn_sched_barrier(0);
      u32x4 prob, rest;
      probabilities(s, t, prob, rest, false);
      add_values(y, t, prob, rest, false);
      __builtin_amdgcn_sched_barrier(0);
      load_v(y, o);
    }
    l_run = sum_over_quarters(l_run);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kDV; ++j) sum += (acc[j][0] + acc[j][1]) + (acc[j][2] + acc[j][3]);
    if (__builtin_expect(__any(is_nan(sum) && !is_nan(l_run)), 0)) {
      // Infinite values: with two products per key they give NaN.  Once more, relative to the maximum: the rest meets the finite values only and a positive
      // probability does not round to 0.
      clear();
      for (int t = from; t < to; ++t) {
        Tile z;
        const Spot o = spot(t);
        load_k(z, o);
        load_v(z, o);
        floatx4 s[2];
        u32x4 prob, rest;
        scores(z, s);
        probabilities(s, t, prob, rest, true);
        add_values(z, t, prob, rest, true);
      }
      l_run = sum_over_quarters(l_run);
    }

    // ---- the waves' states -> the unit's, or a part of it -----------------------------------------------
    {
      float* to_lds = states + (wave * kRows + c16) * kPitch;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < kDV; j += 4)
          *reinterpret_cast<floatx4*>(to_lds + kDV * (4 * g + r) + j) = floatx4{acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]};
      if (g == 0) *reinterpret_cast<floatx2*>(to_lds + D) = floatx2{m_run, l_run};
    }
    __syncthreads();
    const bool begins = t0 == 0, ends = t1 == tiles;
    for (int i = tid; i < kRows * (D / 4); i += kPrefixThreads) {
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
        sums = p.prefix_parts;
        stats = p.prefix_part_stats;
      }
      *reinterpret_cast<floatx4*>(sums + to_row * D + d) = sum;
      if (d == 0) *reinterpret_cast<floatx2*>(stats + 2 * to_row) = floatx2{m, l};
    }
    if (begins && tid == 0) note_unit<kRows>(p, x.first, (int)kvh, (int)block, heads, blockIdx.x, ends ? 0 : (int)((unit_end - 1) / share) - (int)blockIdx.x + 1);
    __syncthreads();
    at = until;
  }
}

// ---- many rows ------------------------------------------------------------------------------------
// 128 rows by a work-group, 32 by a wave, as in the flash kernel: 32 x 32 x 16 MFMAs, S^T = K Q^T with keys from LDS, P^T in S^T's registers, V^T by transposing reads, tiles of 64 keys
// that the memory system fills, chunks swizzled.  Eight waves are two teams that take the tiles in turn and are never in the same half of a tile: while one multiplies (the last tile's
// probabilities with its values, the next one's keys with the queries), the other forms probabilities, a barrier between the halves, so that the matrix pipe has one team's work at a time and
// the vector ALU the other's.  Tiles are requested one tile ahead.
//
// Measured: 32 sequences behind 32768 keys, 32/8 heads of 128, bf16 37.5 us, 134 MB at 3.6 TB/s; 128 behind 8000, 28/4 of 128, fp16 31.5 us, 467 TFLOP/s with each product counted once; 200 in
// groups of 2 to 76 behind 600 to 24000, 32/8 of 64, bf16 40.8.  A tile's products are 1536 cycles of a wave's; the matrix pipe is busy in 39 % of the cycles of the second (a share has 14 tiles, and begins
// and ends as long as ten take).
// A probability enters as two 16-bit numbers, its rounding and the rest, as in the decode kernel, so that a step has the same precision however many sequences share its pages.  It costs
// half as many products again: these three take 58.0, 50.1 and 66.8 us a step, 53.1, 46.6 and 60.3 with the rounding alone.  (Sums by products with ones, a product more for each of
// the two: 59.6, 51.0, 68.5.  Exponents as the decode kernel has them, (score - m) * scale, at all scores: 58.7, 50.6 and 68.3.  kMany.over, what a unit counts beside its tiles, 0, 5, 16 and 24 instead of
// 10: 58.9, 59.4, 59.3 and 59.2 instead of 59.3, 56.9, 53.8, 52.8 and 53.0 instead of 51.5, 75.1, 65.6, 67.4 and 69.9 instead of 67.2.)

template <int D>
__device__ __forceinline__ int wide_k_swizzle(const int r) { return D == 128 ? r & 15 : (r & 7) ^ ((r >> 3) & 1); }
template <int D>
__device__ __forceinline__ int wide_v_swizzle(const int r) { return D == 128 ? (r & 3) << 2 : (r & 3) << 1; }

// load16_to_lds for an address that vector instructions may have formed: one of memory must not read a scalar register within five wait states of their write, which the
// compiler, which does not look inside, would not see to
__device__ __forceinline__ void load16_to_lds_from_any(const char* base, const uint32_t byte_off, const uint32_t lds_dst) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" : : "{m0}"(lds_dst), "v"(byte_off), "s"(base) : "memory");
}

// a barrier that waits for nothing of its own
__device__ __forceinline__ void wave_barrier() { asm volatile("s_barrier" ::: "memory"); }

// `tiles`: kManyLds<D> bytes of LDS, on a 1024-byte boundary: [team][keys 0, 1, values 0, 1]; at the end the second team's states
template <int D> constexpr int kManyLds = 2 * 4 * kMany.tile * 2 * D;
template <typename T, int D>
__device__ __forceinline__ void many_rows(const PagedPrefixArgs& all, const int64_t total, const PagedGroup& lanes, char* tiles) {
  constexpr int kKS = D / 16, kDB = D / 32;        // MFMAs of a score, blocks of 32 channels
  constexpr int kRowBytes = 2 * D, kTileBytes = kMany.tile * kRowBytes;
  constexpr int kRowsALoad = 1024 / kRowBytes, kLoads = 16 / kRowsALoad;  // rows of a load instruction; loads of a wave's 16 rows
  constexpr int kFours = 4 * kDB;                  // accumulators of a lane, in fours
  typedef __attribute__((address_space(3))) const typename T::vec8 lds_vec8;
  typedef short shortx4 __attribute__((ext_vector_type(4)));
  typedef short shortx8 __attribute__((ext_vector_type(8)));
  typedef __attribute__((address_space(3))) shortx4 lds_shortx4;
  static_assert(kManyLds<D> >= 4 * 64 * (4 * kFours + 4) * 4, "a team's states take less room");
  const PagedDecodeArgs& p = all.step;
  const int tid = threadIdx.x, lane = tid & 63, c32 = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane((tid >> 6) & 3), team = __builtin_amdgcn_readfirstlane(tid >> 8);
  const int heads = p.n_q_heads / p.n_kv_heads, page_mask = (1 << p.page_log) - 1;
  // neighbouring shares, which have neighbouring rows of one KV head, are one XCD's
  const int share_at = (blockIdx.x % 8) * (kPrefixShares / 8) + blockIdx.x / 8;
  const PrefixShare mine = share_of(all, kMany, total, lanes, share_at);
  int64_t at = mine.at, start = mine.start;
  const int64_t end = mine.end, share = mine.share;
  int group = mine.group;

  const float scale = p.sm_scale * kLog2e;
  // where a lane's pieces of 16 rows come from (its chunk, which belongs in its slot), and what it reads of a tile
  uint32_t k_from[kLoads], v_from[kLoads];
#pragma unroll
  for (int j = 0; j < kLoads; ++j) {
    const int r = kRowsALoad * j + lane / (D / 8), slot = lane % (D / 8);
    k_from[j] = 2u * (uint32_t)p.kp_sn * r + 16u * (slot ^ wide_k_swizzle<D>(r));
    v_from[j] = 2u * (uint32_t)p.vp_sn * r + 16u * (slot ^ wide_v_swizzle<D>(r));
  }
  const uint32_t my_tiles = lds_addr(tiles) + team * 4 * kTileBytes;
  // (chunk 2 ks + half of a row: the bits of ks are their own; so are those of the block of channels)
  const uint32_t k_rd = my_tiles + c32 * kRowBytes + ((half ^ wide_k_swizzle<D>(c32)) << 4);
  const int r0 = 4 * half + ((lane & 15) >> 2), y0 = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
  const uint32_t v_rd = my_tiles + 2 * kTileBytes + r0 * kRowBytes + ((y0 ^ wide_v_swizzle<D>(r0)) << 4) + 8 * (lane & 1);

  while (at < end && group < all.n_groups) {
    at = uniform(at), start = uniform(start), group = __builtin_amdgcn_readfirstlane(group);  // (which the compiler does not see of what a loop carries)
    const PagedGroup x = common_group_at(all, group);
    const int n_tiles = tiles_of(p, kMany, x), blocks = blocks_of(kMany, x, heads), length = x.pages << p.page_log, rows = x.sequences * heads;
    const int extent = extent_of(kMany, n_tiles);
    if (at - start >= (int64_t)extent * blocks * p.n_kv_heads) {  // (the next group, perhaps of nothing)
      start += (int64_t)extent * blocks * p.n_kv_heads;
      ++group;
      continue;
    }
    // a KV head's blocks one after the other
    const uint32_t unit = (uint32_t)((at - start) / extent), block = unit % (uint32_t)blocks, kvh = unit / (uint32_t)blocks;
    const int64_t unit_end = start + (int64_t)(unit + 1) * extent, until = min(end, unit_end);
    const int t0 = max(n_tiles - (int)(unit_end - at), 0), t1 = max(n_tiles - (int)(unit_end - until), 0);
    if (t1 == 0) break;  // (nothing of it is in this share, which ends)
    const int my_row = min((int)(block * kMany.rows) + 32 * wave + c32, rows - 1), sequence = my_row / heads;
    const int64_t my_head = (int64_t)(x.first + sequence) * p.n_q_heads + (int)kvh * heads + my_row - sequence * heads;
    typename T::vec8 q[kKS];
    {
      const uint16_t* qp = p.q + (int64_t)(x.first + sequence) * p.q_sb + (int64_t)((int)kvh * heads + my_row - sequence * heads) * p.q_sh + 8 * half;
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) q[ks] = *reinterpret_cast<const typename T::vec8*>(qp + 16 * ks);
    }
    const const_i32* table = (const_i32*)(p.table + x.first * p.t_sb);
    const int rounds = (t1 - t0 + 1) / 2, own = (t1 - t0 + 1 - team) / 2;  // tiles t0 + team, t0 + team + 2, ...
    auto tile_at = [&](const int i) { return t0 + team + 2 * i; };
    // 16 of a tile's rows are a wave's to request, which lie in one page; rows behind the prefix are zeros
    auto key_of = [&](const int i) { return kMany.tile * tile_at(i) + 16 * wave; };
    auto page_of = [&](const int i) { return table[min(key_of(min(i, max(own - 1, 0))) >> p.page_log, x.pages - 1)]; };
    auto request = [&](const int i, const int page_there, const bool values) __attribute__((always_inline)) {
      const int key = key_of(i);
      const uint32_t to = my_tiles + ((values ? 2 : 0) + (i & 1)) * kTileBytes + 16 * wave * kRowBytes;
      if (key < length) {
        const int64_t page = clamped_page(page_there, p.n_pages);
        const int slot = key & page_mask;
        const char* base = (const char*)(values ? p.values + page * p.vp_sp + kvh * p.vp_sh + slot * p.vp_sn : p.keys + page * p.kp_sp + kvh * p.kp_sh + slot * p.kp_sn);
#pragma unroll
        for (int j = 0; j < kLoads; ++j) load16_to_lds_from_any(base, values ? v_from[j] : k_from[j], to + j * 1024);
      } else {
#pragma unroll
        for (int j = 0; j < kLoads; ++j) *(__attribute__((address_space(3))) u32x4*)(uintptr_t)(to + j * 1024 + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      }
    };
    float m_run = -INFINITY, l_run;  // (until the end a lane's sum is of its half of the keys)
    floatx16 acc[kDB], s[2];
    u32x4 prob[4], rest[4];
    // What a team multiplies of a round: operand f is of values or, from kValues on, of the next tile's keys.  Operands are read from LDS
    // kAhead ahead of the products that take them, in this order, which the compiler would not keep; the first ones before the barrier.
    constexpr int kAhead = 4, kValues = 4 * kDB, kKeys = 2 * kKS;
    u32x4 operand[kAhead];
    auto read = [&](const int i, const int f) __attribute__((always_inline)) {  // of values of tile i, keys of tile i + 1
      if (f < kValues) {
        const uint32_t at = ((v_rd + (i & 1) * kTileBytes) ^ ((f % kDB) << 6)) + 16 * (f / kDB) * kRowBytes;
        const shortx4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(uintptr_t)at);
        const shortx4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_shortx4*)(uintptr_t)(at + 8 * kRowBytes));
        const shortx8 both = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
        operand[f % kAhead] = *reinterpret_cast<const u32x4*>(&both);
      } else {
        const int g = f - kValues;
        operand[f % kAhead] = *(const __attribute__((address_space(3))) u32x4*)(uintptr_t)(((k_rd + ((i + 1) & 1) * kTileBytes) ^ ((g % kKS) << 5)) + 32 * (g / kKS) * kRowBytes);
      }
    };
    auto multiply_values = [&](const int f, auto exact) __attribute__((always_inline)) {
      u32x4 finite = operand[f % kAhead];
      if constexpr (decltype(exact)::value) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if ((finite[i] & T::kExponent) == T::kExponent) finite[i] &= 0xffff0000u;
          if (((finite[i] >> 16) & T::kExponent) == T::kExponent) finite[i] &= 0xffffu;
        }
      }
      const auto p1 = *reinterpret_cast<const typename T::vec8*>(&prob[f / kDB]), p2 = *reinterpret_cast<const typename T::vec8*>(&rest[f / kDB]);
      acc[f % kDB] = T::mfma(*reinterpret_cast<const typename T::vec8*>(&operand[f % kAhead]), p1, acc[f % kDB]);
      acc[f % kDB] = T::mfma(*reinterpret_cast<const typename T::vec8*>(&finite), p2, acc[f % kDB]);
    };
    auto multiply_keys = [&](const int g) __attribute__((always_inline)) {
      floatx16 none;
#pragma unroll
      for (int r = 0; r < 16; ++r) none[r] = 0.f;
      s[g / kKS] = T::mfma(*reinterpret_cast<const typename T::vec8*>(&operand[(kValues + g) % kAhead]), q[g % kKS], g % kKS == 0 ? none : s[g / kKS]);
    };
    auto probabilities = [&](const int i, auto exact) __attribute__((always_inline)) {
      const int key0 = kMany.tile * tile_at(i);
      if (key0 + kMany.tile > length) {
#pragma unroll
        for (int r = 0; r < 32; ++r)
          if (key0 + 32 * (r >> 4) + 16 * ((r & 15) >> 3) >= length) s[r >> 4][r & 15] = -INFINITY;
      }
      float mx[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
      for (int r = 4; r < 32; ++r) mx[r & 3] = fmaxf(mx[r & 3], s[r >> 4][r & 15]);
      const float m_new = fmaxf(m_run, max_with_other_half(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]))));
      const float m_base = m_new == -INFINITY ? 0.f : m_new;  // (no key of this row's so far)
      if (__any(m_new > m_run)) {
        const float alpha = fast_exp2((m_run - m_base) * scale);
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < kDB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[db][r] *= alpha;
        m_run = m_new;
      }
      auto form = [&](auto near) __attribute__((always_inline)) {
        const float bias = T::kProbLog2 - m_base * scale;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 16; ++w) {
          const float s0 = s[w >> 3][2 * (w & 7)], s1 = s[w >> 3][2 * (w & 7) + 1];
          const float e0 = decltype(near)::value ? fast_exp2(__builtin_fmaf(s0, scale, bias)) : prob_exp2<T>(s0 - m_base, scale);
          const float e1 = decltype(near)::value ? fast_exp2(__builtin_fmaf(s1, scale, bias)) : prob_exp2<T>(s1 - m_base, scale);
          uint32_t both = T::pack(e0, e1);
          if constexpr (decltype(exact)::value) {
            if (e0 > 0.f && (both & 0xffffu) == 0u) both |= 1u;
            if (e1 > 0.f && (both >> 16) == 0u) both |= 0x10000u;
          }
          prob[w >> 2][w & 3] = both;
          rest[w >> 2][w & 3] = T::pack_rest(e0, e1, both);
          sum[0] += e0;
          sum[1] += e1;
        }
        l_run += sum[0] + sum[1];
      };
      // One fused operation a key, where the rounding of m * scale, which is in every probability as long as m is the maximum, is 2^-17 at most; elsewhere it would reach whole powers of two
      if (__builtin_expect(__any(!(fabsf(m_base * scale) < 256.f)), 0)) form(std::false_type{});
      else form(std::true_type{});
    };
    auto run = [&](auto exact) __attribute__((always_inline)) {
      l_run = 0.f;
#pragma unroll
      for (int db = 0; db < kDB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[db][r] = 0.f;
      int page1 = page_of(1), page2 = page_of(2);  // of the next tile and the one behind it
      if (own > 0) {
        const int page0 = page_of(0);
        request(0, page0, false);
        request(0, page0, true);
        if (own > 1) request(1, page1, false);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int ks = 0; ks < kKS; ++ks) asm volatile("" ::"v"(q[ks]));  // (so that the compiler does not wait for them, and all that was requested since, inside the loop)
      lds_barrier();
      if (team == 1) wave_barrier();
      if (own > 0) {
#pragma unroll
        for (int f = 0; f < kAhead; ++f) read(-1, kValues + f);
      }
      for (int i = 0; i < own; ++i) {
        if (i > 0) {
#pragma unroll
          for (int f = 0; f < kValues; ++f) {
            multiply_values(f, exact);
            read(i - 1, f + kAhead);
            __builtin_amdgcn_sched_barrier(0);
          }
        }
#pragma unroll
        for (int g = 0; g < kKeys; ++g) {
          multiply_keys(g);
          if (g + kAhead < kKeys) read(i - 1, kValues + g + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
        // (keys i and values i - 1 have been read; keys i + 1 and values i, requested a round ago, are there)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        wave_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (i + 1 < own) request(i + 1, page1, true);
        if (i + 2 < own) request(i + 2, page2, false);
        page1 = page2;
        page2 = page_of(i + 3);
        probabilities(i, exact);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int f = 0; f < kAhead; ++f) read(i, f);
        __builtin_amdgcn_sched_barrier(0);
        wave_barrier();
        __builtin_amdgcn_sched_barrier(0);
      }
      if (own > 0) {
#pragma unroll
        for (int f = 0; f < kValues; ++f) {
          multiply_values(f, exact);
          if (f + kAhead < kValues) read(own - 1, f + kAhead);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      for (int i = own; i < rounds; ++i) {  // (the second team has one tile less where there is an odd number)
        wave_barrier();
        wave_barrier();
      }
      lds_barrier();
      if (team == 0) lds_barrier();
      l_run += xor32(l_run);
    };
    run(std::false_type{});
    float sum = 0.f;
#pragma unroll
    for (int db = 0; db < kDB; ++db)
#pragma unroll
      for (int r = 0; r < 16; ++r) sum += acc[db][r];
    // Infinite values: with two products per key they give NaN.  Once more, relative to the last maximum: the rest meets the finite values only and a positive probability does not round to 0.
    if (__builtin_expect(__syncthreads_or(is_nan(sum) && !is_nan(l_run)), 0)) run(std::true_type{});

    // ---- the teams' states -> the unit's, or a part of it: fours of accumulators, lane by lane, half of them by each team ----
    floatx4* states = reinterpret_cast<floatx4*>(tiles) + wave * kFours * 64;
    floatx2* stats = reinterpret_cast<floatx2*>(reinterpret_cast<floatx4*>(tiles) + 4 * kFours * 64) + wave * 128;
    auto four = [&](const int f) { return floatx4{acc[f >> 2][4 * (f & 3)], acc[f >> 2][4 * (f & 3) + 1], acc[f >> 2][4 * (f & 3) + 2], acc[f >> 2][4 * (f & 3) + 3]}; };
    const int64_t part = (2 * share_at + (t0 == 0 ? 1 : 0)) * 4 + wave;
    const bool whole = t0 == 0 && t1 == n_tiles, there = (int)(block * kMany.rows) + 32 * wave + c32 < rows;
    auto hand_over = [&](auto first) __attribute__((always_inline)) {
#pragma unroll
      for (int f = 0; f < kFours / 2; ++f) states[(decltype(first)::value + f) * 64 + lane] = four(decltype(first)::value + f);
      stats[team * 64 + lane] = floatx2{m_run, l_run};
    };
    auto finish = [&](auto first) __attribute__((always_inline)) {
      const floatx2 other = stats[(1 - team) * 64 + lane];
      const float m = fmaxf(m_run, other[0]), w = m_run == -INFINITY ? 0.f : fast_exp2((m_run - m) * scale);
      const float w2 = other[0] == -INFINITY ? 0.f : fast_exp2((other[0] - m) * scale);
      const float l = w * l_run + w2 * other[1];
#pragma unroll
      for (int g = 0; g < kFours / 2; ++g) {
        const int f = decltype(first)::value + g;
        const floatx4 a = four(f), b = states[f * 64 + lane];
        const floatx4 y = {w * a[0] + w2 * b[0], w * a[1] + w2 * b[1], w * a[2] + w2 * b[2], w * a[3] + w2 * b[3]};
        if (!whole) *reinterpret_cast<floatx4*>(p.prefix_parts + ((part * kFours + f) * 64 + lane) * 4) = y;
        else if (there) *reinterpret_cast<floatx4*>(p.prefix + my_head * D + 8 * f + 4 * half) = y;
      }
      if (decltype(first)::value != 0) return;
      if (!whole) *reinterpret_cast<floatx2*>(p.prefix_part_stats + (part * 64 + lane) * 2) = floatx2{m, l};
      else if (there && half == 0) *reinterpret_cast<floatx2*>(p.prefix_stats + 2 * my_head) = floatx2{m, l};
    };
    std::integral_constant<int, 0> lower;
    std::integral_constant<int, kFours / 2> upper;
    if (team == 0) hand_over(upper);
    else hand_over(lower);
    __syncthreads();
    if (team == 0) finish(lower);
    else finish(upper);
    if (t0 == 0 && tid == 0) note_unit<kMany.rows>(p, x.first, (int)kvh, (int)block, heads, share_at, whole ? 0 : (int)((unit_end - 1) / share) - share_at + 1);
    __syncthreads();
    at = until;
  }
}

// Which form the launch takes, by all units' extents in either: an extent of few rows takes about 0.6 us of its work-group, one of many 1.5, and many rows' parts some 8 us more to begin, join
// and read again.  The groups are looked at as they are; their number and the batch, all that the host knows, say little of groups of which many are empty, as where a captured step has room for more, or one
// is large and the others are small: 128 sequences, 28/4 heads of 128, behind 8000 keys in one group of 64 that could be take 112 us a step with few rows to a unit and 49 with many, 32, 32/8 of 128,
// behind 32768 in one of 200 100 and 56.  A step of one group, bf16, 100 keys of their own, few and many rows, behind 8192 keys and behind 32768 (* where the rule takes the slower one):
//   32/8 heads of 128: 4 sequences (16 rows) 27.6 and 33.6 us, 42.3 and 48.2; 8 (32 rows) 31.8 and 33.6, 58.5 and 48.1; 12 (48 rows) 37.2 and 33.9, 77.4 and 49.2
//   28/4 of 128: 3 (21 rows) 30.6 and 36.1, 44.5 and 46.2; 6 (42 rows) 29.7 and 36.3, 53.2 and 47.0; 16 (112 rows) 40.8 and 38.0, 87.9 and 47.8
//   32/8 of 64: 4 (16 rows) 22.6 and 25.7, 30.8 and 35.8; 8 (32 rows) 25.1 and 25.5, 38.8 and 35.9; 16 (64 rows) 28.6 and 26.0, 55.5 and 36.0
//   14/2 of 64: 4 (28 rows) 23.2 and 27.0, 29.4 and 34.6; 16 (112 rows) 25.9 and 27.2, 34.5 and 36.5 *; 32 (224 rows) 28.9 and 27.9, 52.5 and 35.5
//   128 sequences behind 1024 keys: 32/8 of 128 36.3 and 38.5 *, 28/4 of 128 38.6 and 33.2, 32/8 of 64 27.3 and 27.8 *
__device__ __forceinline__ bool takes_many(const PrefixTotals& t) {
  const int64_t few = max(t.few, (int64_t)kFew.least * kPrefixShares), many = max(t.many, (int64_t)kMany.least * kPrefixShares);
  return 2 * few > 5 * many + 26 * kPrefixShares;
}

template <typename T, int D>
__global__ void __launch_bounds__(kPrefixThreads) paged_prefix_kernel(const PagedPrefixArgs all) {
  constexpr int kFewLds = kPrefixWaves * kFew.rows * (D + 4) * 4;
  __shared__ __attribute__((aligned(1024))) char lds[kManyLds<D> > kFewLds ? kManyLds<D> : kFewLds];
  find_skips(all, threadIdx.x, kPrefixThreads);
  const PagedGroup lanes = all.n_groups == 1 ? PagedGroup{0, 0, 0} : lane_group_at(all, 0);
  const PrefixTotals totals = totals_of(all, lanes);
  const bool many = takes_many(totals);
  if (blockIdx.x == 0 && threadIdx.x == 0) *all.step.prefix_rows = many ? kMany.rows : kFew.rows;
  if (many) many_rows<T, D>(all, totals.many, lanes, lds);
  else few_rows<T, D>(all, totals.few, lanes, reinterpret_cast<float*>(lds));
}

// Where the keys and values of all sequences fit the caches, as much as the table has room for, what sequences share is there after the first one's read, and the steps of the others cost less than
// two kernels more.  One group, 100 keys of their own, all bytes as if none were shared, time by this path and with every sequence by itself:
//   32/8 heads of 64: 64 sequences behind 1024 keys (151 MB) 23.0 and 19.3 us, 12 behind 8192 (204 MB) 25.6 and 25.8, 32 behind 4096 (277 MB) 25.5 and 29.2, 16 behind 8192 (273 MB) 26.0 and 31.2
//   14/2 of 64: 32 behind 8192 (136 MB) 27.9 and 20.4, 64 behind 8192 (273 MB) 29.5 and 31.2, 32 behind 16384 (271 MB) 32.3 and 30.5 *, 16 behind 32768 (269 MB) 36.5 and 30.2 *, 64 behind 16384 (541 MB) 32.8 and 52.1
//   32/8 of 128: 16 behind 4096 (277 MB) 30.2 and 28.0, 8 behind 8192 (273 MB) 31.8 and 28.0, 2 behind 32768 (269 MB) 41.8 and 44.7 *, 64 behind 1024 (302 MB) 29.6 and 28.9, 12 behind 8192 (409 MB)
//     33.9 and 36.6, 6 behind 16384 (406 MB) 39.4 and 63.0
//   28/4 of 128: 16 behind 8192 (273 MB) 38.0 and 28.3, 128 behind 1024 (302 MB) 33.2 and 30.0, 12 behind 16384 (406 MB) 41.9 and 63.3, 16 behind 16384 (541 MB) 42.0 and 45.5
// (* where the rule takes the slower one.)  The lengths are the device's to know: in a table with room for more, few keys take this path too.
bool paged_prefix_pays(int batch, int n_kv_heads, int head_dim, int page_size, int max_pages) {
  return batch > 1 && (double)batch * max_pages * page_size * n_kv_heads * head_dim * 4 > (head_dim == 64 ? 256e6 : 340e6);
}

PagedScratch paged_prefix_scratch(int head_dim) {
  constexpr size_t kRows = (size_t)kPrefixShares * 2 * kMany.rows;
  PagedScratch s = {0, 0, 0, 0};
  s.parts = s.stats + kRows * 16;  // (a row's statistics are there twice, once for each of its lanes)
  s.total = s.parts + kRows * head_dim * 4;
  return s;
}

template <typename T, int D>
static hipError_t launch_paged_prefix_of(const PagedPrefixArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((paged_prefix_kernel<T, D>), dim3(kPrefixShares), dim3(kPrefixThreads), 0, stream, a);
  return hipGetLastError();
}
hipError_t launch_paged_prefix(const PagedPrefixArgs& a, hipStream_t stream) {
  if (a.step.head_dim == 128) return a.step.dtype == 0 ? launch_paged_prefix_of<Bf16, 128>(a, stream) : launch_paged_prefix_of<F16, 128>(a, stream);
  return a.step.dtype == 0 ? launch_paged_prefix_of<Bf16, 64>(a, stream) : launch_paged_prefix_of<F16, 64>(a, stream);
}

}  // namespace aa
