// Attention of one new token per sequence over a key/value cache in pages, on gfx950.
//
// Bound by reading keys and values once.  A unit is a (sequence, KV head) with up to 16 heads of its group as the columns of 16 x 16 x 32 MFMAs; its
// keys come in tiles of 32.  Lengths are known on the device only and may differ a lot, so the tiles of all units, one after the other, are cut into equal
// shares, one for each of a fixed number of work-groups, and each share into equal parts of its four waves: every wave sums the lengths and finds its part
// by itself.  A wave walks its part alone, from unit to unit, and nothing passes through LDS until the end, where the states (maximum, sum, accumulator) of units
// that several waves have are joined.  A share that begins or ends inside a unit leaves that unit's state in the workspace, two states at most, and
// paged_combine_kernel (paged_finish_kernel behind a shared prefix, paged_weigh_kernel where attention is counted) joins them in order, so that results do not depend on timing.  Where the table has room for few tiles only, no unit is cut between
// work-groups, and there is no second launch.
//
// Inside a wave:
//   S^T = K Q^T: a lane holds 8 channels of one key, the MFMA's own layout, straight from memory;
//   O^T = V^T P^T: the order of keys inside a product is free, so P^T is S^T's registers as they lie (lane 16 g + c has keys 4 g + r and
//   16 + 4 g + r of column c), and V^T wants 8 keys of one channel in a lane: a lane loads D / 16 channels of its 8 keys, whole rows
//   by 16 lanes, and v_perm turns the block, one instruction per two elements.
// P enters as two 16-bit numbers, its rounding and the rest, as in the other decode kernel: the MFMAs are idle most of the time, and one rounding of P
// costs as much as that of the output.  There is one set of registers for a tile; its keys are requested anew as soon as the scores have read them, its values after
// the last product, so that loads are always in flight.
//
// Measured (bf16 unless said): 32 sequences of 500 to 16000 keys, 32/8 heads of 128 108 us, of which 4.8 the join: 5.7 TB/s while it reads, where a copy of that
// size reaches 5.2 to 5.4; 2 of 131071, 28/4 heads of 128, fp16 99 us, 5.6 TB/s; one of 33001, 32/8 of 128 31.2 us, of which about 4 pass before the first
// tile has come (lengths, table, rows, one after the other), 1 at the end and 4 in the join; one of 300, 14/2 of 64 7.4 us, nothing but such chains.  What is
// executed before the first load counts there: a place is looked for only where it is not in the unit of the one before.
#include "aa_kernels.h"
#include "aa_nonfinite.h"
#include "aa_paged.h"

namespace aa {

constexpr int kCols = 16;       // columns of a unit: heads of the group
constexpr int kTile = 32;       // keys of a tile
// What a unit costs beside its tiles, in tiles.  (128 sequences of 20 to 1200 keys, 32/8 heads of 64: 0 28.5 us, 3 21.7, 6 23.1; 32 of 500 to 16000, 32/8 of 128:
// 111, 107.7, 110.)
constexpr int kOver = 3;
// Where the table has room for that many tiles of a sequence at most, units are not cut between work-groups and nothing is joined.  (By the table's room, since the host knows
// no lengths: the same 300 keys cost a step with a join in a table for more.  One sequence, cut and joined or not: 300 keys, 14/2 heads of 64, 14.0 and 10.1 us, 1500 keys 14.4
// and 12.8, 1780 14.6 and 14.1; 760 keys, 32/8 of 128, 14.4 and 11.9, 890 14.5 and 12.7, 1200 14.2 and 15.8; 32 of 200 to 890 17.5 and 15.9.)  Many units keep all
// work-groups busy for longer than a join takes, and uncut ones of different lengths do so less evenly: 128 sequences of 1 to 1500 keys, 32/8 of 64, 19.2 and 20.8, of 1 to
// 890, 32/8 of 128, 20.8 and 22.2.
template <int D> constexpr int kWhole = 28;
template <> constexpr int kWhole<64> = 48;
constexpr int kMany = 768, kWholeMany = 20;  // units, and what holds for more
// Work-groups, one to a CU.  (128: 32 sequences of 500 to 16000 keys, 32/8 heads of 128 124 us instead of 108, 128 of 20 to 1200, 32/8 of 64 27.9 instead of 21.7; 512, when these
// were 110 and 22.9, 112 and 23.8.)
constexpr int kShares = 256;
constexpr int kSharesLog = 8;
// Sequences that a lane counts where there are more than 64, so that 256 are one scan.  (1: 256 of 1 to 800 keys, 14/2 heads of 64, 14.6 us instead of 12.2; 1000 of 1 to 200, 32/8 of 64, 49.4
// instead of 39.8; 128 of 20 to 1200 23.0 instead of 21.7.)
constexpr int kPerLane = 4, kPerLaneLog = 2;
// Tiles of a share at least: fewer work-groups leave fewer parts to join, and each has longer to go.  (64 pages of 64 of one sequence, 32/8 heads of 128, chosen and
// read: 4 22.2 us, 8 22.2, 16 24.4.)
constexpr int kLeast = 8;

// Place: an integer that counts the tiles of all units
template <typename Place>
struct PagedPlace {       // of a tile, among all
  int b, unit, tile;      // sequence, unit of it, tile of the unit
  int n_tiles, length;    // of the sequence
  Place start;            // the unit's beginning
};

// kWeigh: the scores and each head's maximum and sum are kept for paged_weigh_kernel; kShared: the first pages of a sequence have been read for its group, whose states paged_finish_kernel joins with those of the own keys
enum DecodeMode { kPlain, kWeigh, kShared };

// keys that are read of sequence b
template <DecodeMode MODE>
__device__ __forceinline__ int keys_of(const PagedDecodeArgs& p, const int b, const int length) {
  const int n = min(max(length, 0), p.max_pages << p.page_log);
  if (MODE == kShared) return n - (((const_i32*)p.skips)[b] << p.page_log);
  return p.n_chosen ? n - (max(0, pages_of(n, p.page_log) - p.n_chosen) << p.page_log) : n;
}
__device__ __forceinline__ int tiles_of(const int keys) { return max(1, (keys + kTile - 1) / kTile); }  // (a sequence of none has to be written too)

// n / d where the quotient is below 2^16
__device__ __forceinline__ uint32_t small_quotient(const uint32_t n, const uint32_t d) {
  uint32_t q = (uint32_t)((float)n * __builtin_amdgcn_rcpf((float)d));
  q = __builtin_amdgcn_readfirstlane(q);
  // (off by one at most: three roundings of 2^-23 of a quotient below 2^16)
  if (q * d > n) --q;
  else if (n - q * d >= d) ++q;
  return q;
}

// What some heads of a group (from head0 on in all of the batch's) give four keys from i on: the sum of 2^((score - maximum) * scale) / sum; total(h): a head's maximum and 1 / sum.
template <typename T, typename F>
__device__ __forceinline__ void add_probabilities(const PagedDecodeArgs& p, const int64_t head0, const int heads, const int i, const float scale, floatx4& sum, F total) {
  const int64_t room = p.max_pages << p.page_log;
  const float* from = p.scores + head0 * room + i;
#pragma unroll 4
  for (int h = 0; h < heads; ++h) {
    const floatx4 s = *reinterpret_cast<const floatx4*>(from + h * room);
    const floatx2 t = total(h);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += prob_exp2<T>(s[e] - t[0], scale) * t[1];
  }
}
// ... and into the weights of the first n keys
__device__ __forceinline__ void add_to_weights(const PagedDecodeArgs& p, const int b, const int kvh, const int i, const int n, const floatx4 sum) {
  const int page = p.table[b * p.t_sb + (i >> p.page_log)];
  if ((uint32_t)page >= (uint32_t)p.n_pages) return;  // (what is read in its place is another sequence's)
  float* w = p.weights + (((int64_t)page * p.n_kv_heads + kvh) << p.page_log) + (i & ((1 << p.page_log) - 1));
  const floatx4 old = *reinterpret_cast<const floatx4*>(w);
  if (i >= p.n_first && i + 3 < n) {
    *reinterpret_cast<floatx4*>(w) = floatx4{old[0] + sum[0], old[1] + sum[1], old[2] + sum[2], old[3] + sum[3]};
    return;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)  // (what is not this sequence's to count is not written, not even as it was)
    if (i + e < n && i + e >= p.n_first) w[e] = old[e] + sum[e];
}
// the first four keys of n that has any to count
__device__ __forceinline__ int first_counted(const PagedDecodeArgs& p, const int n) { return min(p.n_first, n) & ~3; }

template <typename T, int D, int WAVES, typename Place, DecodeMode MODE>
__global__ void __launch_bounds__(64 * WAVES, 2) paged_decode_kernel(const PagedDecodeArgs p) {
  constexpr int kKS = D / 32;      // MFMAs of a score
  constexpr int kDV = D / 16;      // channels of V that a lane loads
  constexpr int kVW = kDV / 2;     // ... in words
  constexpr int kPitch = D + 4;
  // States of units that a wave has a part of only: [wave][0: the first of its units, which began before; 1: its last, which goes on][column]
  extern __shared__ __attribute__((aligned(16))) float states[];
  __shared__ float stats[WAVES][2][2][kCols];
  __shared__ floatx2 unit_totals[MODE == kWeigh ? kCols : 1], wave_totals[MODE == kWeigh ? WAVES : 1][kCols];
  __shared__ int4 parts_of[WAVES][2];  // 0 if there is none, 2 if the unit ends in it; sequence; first head, and columns in the upper half; parts of work-groups

  const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = p.n_q_heads / p.n_kv_heads, col_blocks = (group + kCols - 1) / kCols, units = p.n_kv_heads * col_blocks;
  const int most_cols = min(group, kCols);
  // whether a unit's keys get their weights here: where it is one work-group's, and all of its KV head's
  const bool weighs = MODE == kWeigh && p.headers == nullptr && col_blocks == 1;

  // ---- this wave's share -------------------------------------------------------------------------
  // All units one after the other, each as long as its tiles and kOver.  A lane has kPerLane sequences in a row, a scan 64 lanes' (whose numbers stay if
  // there are no more)
  const int per_log = p.batch <= 64 ? 0 : kPerLaneLog;
  int keys0[kPerLane] = {}, sum0 = 0;
  auto scan = [&](const int i, int (&keys)[kPerLane], int& sum) __attribute__((always_inline)) {  // of the sequences from i on: their keys, and the sums up to each lane's last
    int own = 0;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
      if (j > 0 && per_log == 0) break;
      const int b = i + (lane << per_log) + j;
      keys[j] = b < p.batch ? keys_of<MODE>(p, b, p.lengths[b]) : 0;
      own += b < p.batch ? tiles_of(keys[j]) + kOver : 0;
    }
    sum = sums_up_to(own);
  };
  auto keys_at = [&](const int (&keys)[kPerLane], const int at) {  // of the at-th sequence of a scan
    int x = __builtin_amdgcn_readlane(keys[0], at >> per_log);
#pragma unroll
    for (int j = 1; j < kPerLane; ++j) {
      if (per_log == 0) break;
      const int y = __builtin_amdgcn_readlane(keys[j], at >> per_log);
      x = at % kPerLane == j ? y : x;
    }
    return x;
  };
  constexpr int kScan = 64 * kPerLane;
  Place total = 0;
  for (int i = 0; i < p.batch; i += kScan) {
    scan(i, keys0, sum0);
    total += __builtin_amdgcn_readlane(sum0, 63);
  }
  total *= units;
  // x becomes the beginning of its unit if that is near, or if units are not cut and `whole`
  auto settle = [&](PagedPlace<Place>& f, Place& x, const bool whole) __attribute__((always_inline)) {
    f.tile = (int)(x - f.start) - kOver;
    if (f.tile <= 0 || (whole && p.headers == nullptr)) {
      f.tile = 0;
      x = f.start;
    }
  };
  // the place x < total
  auto find = [&](Place& x, const bool whole) {
    PagedPlace<Place> f = {};
    Place before = 0;
    for (int i = 0;; i += kScan) {
      int keys[kPerLane], sum = sum0;
#pragma unroll
      for (int j = 0; j < kPerLane; ++j) keys[j] = keys0[j];
      if (p.batch > kScan) scan(i, keys, sum);
      const int in = __popcll(__ballot((before + sum) * units <= x));  // lanes whose sequences end at or before x
      if (in < 64 || i + kScan >= p.batch) {
        f.start = in > 0 ? (before + __builtin_amdgcn_readlane(sum, in - 1)) * units : before * units;
        uint32_t extent = 1;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) {  // (its last sequence that begins at or before x)
          if (j > 0 && per_log == 0) break;
          const int length = __builtin_amdgcn_readlane(keys[j], in), tiles = tiles_of(length);
          const Place next = f.start + (Place)extent * units;
          if (j == 0 || (next <= x && i + (in << per_log) + j < p.batch)) {
            if (j > 0) f.start = next;
            f.b = i + (in << per_log) + j;
            f.length = length;
            f.n_tiles = tiles;
            extent = tiles + kOver;
          }
        }
        f.unit = small_quotient((uint32_t)(x - f.start), extent);
        f.start += (Place)f.unit * (Place)extent;
        settle(f, x, whole);
        return f;
      }
      before += __builtin_amdgcn_readlane(sum, 63);
    }
  };
  // the same for a place that is not before f's
  auto find_from = [&](const PagedPlace<Place>& f, Place& x, const bool whole) {
    if (x >= f.start + f.n_tiles + kOver) return find(x, whole);
    PagedPlace<Place> r = f;
    settle(r, x, whole);
    return r;
  };
  const Place share = max((total + (kShares - 1)) >> kSharesLog, (Place)kLeast), raw = share * (Place)blockIdx.x;
  Place at = min(raw, total), end = min(raw + share, total);
  PagedPlace<Place> f = {};
  if (at < end) {
    f = find(at, true);
    if (end < total) find_from(f, end, true);
    // the waves' parts of it
    const Place all = end - at, to = at + all * (wave + 1) / WAVES;
    at += all * wave / WAVES;
    if (at < end) {
      f = find_from(f, at, false);
      if (wave + 1 < WAVES) {
        end = to;
        if (end < total) find_from(f, end, false);
      }
    }
  }
  if (lane < 2) parts_of[wave][lane] = int4{0, 0, 0, 0};

  const float scale = p.sm_scale * kLog2e;
  const uint32_t k_lane = (2u * (c16 * (uint32_t)p.kp_sn + 8 * g)) & 0xfffffu, v_lane = (2u * (4 * g * (uint32_t)p.vp_sn + kDV * c16)) & 0xfffffu;
  // what finds the tiles of a unit
  struct Unit {
    const_i32* table;
    int64_t k_head, v_head;
    int length, last_page, kvh, head0, n_cols;
  };
  auto unit_of = [&](const PagedPlace<Place>& f) __attribute__((always_inline)) {
    Unit u;
    u.kvh = col_blocks == 1 ? f.unit : f.unit / col_blocks;
    u.head0 = u.kvh * group + (f.unit - u.kvh * col_blocks) * kCols;
    u.n_cols = min(kCols, (u.kvh + 1) * group - u.head0);
    u.length = f.length;
    u.last_page = max(0, (u.length - 1) >> p.page_log);
    u.table = (const_i32*)(p.table + f.b * p.t_sb + u.kvh * p.t_sh);
    if (MODE == kShared) u.table += min(((const_i32*)p.skips)[f.b], p.max_pages - 1);  // (of a sequence without keys of its own no page is read)
    u.k_head = u.kvh * p.kp_sh;
    u.v_head = u.kvh * p.vp_sh;
    return u;
  };
  struct Tile {
    u32x4 k[2][kKS];
    uint32_t v[8][kVW];
  };
  // Where a tile lies: the first rows of its two halves, and how many rows are read.  (16 keys lie in one page; of a tile that is not there, nothing)
  struct Spot {
    int64_t k[2], v[2];
    int rows[2];
  };
  auto spot = [&](const Unit& u, const int t, const bool there) __attribute__((always_inline)) {
    Spot o;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int key = kTile * t + 16 * half, row = key & ((1 << p.page_log) - 1);
      const int64_t page = clamped_page(u.table[min(key >> p.page_log, u.last_page)], p.n_pages);
      o.k[half] = page * p.kp_sp + row * p.kp_sn + u.k_head;
      o.v[half] = page * p.vp_sp + row * p.vp_sn + u.v_head;
      o.rows[half] = there ? min(max(u.length - key, 0), 16) : 0;
    }
    return o;
  };
  auto load_k = [&](Tile& x, const Spot& o) __attribute__((always_inline)) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const Rows kr = rows_at(p.keys + o.k[half], o.rows[half] * (2 * (int)p.kp_sn));
#pragma unroll
      for (int s = 0; s < kKS; ++s) x.k[half][s] = __builtin_amdgcn_raw_buffer_load_b128(kr, k_lane + 64 * s, 0, 0);
    }
  };
  auto load_v = [&](Tile& x, const Spot& o) __attribute__((always_inline)) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const Rows vr = rows_at(p.values + o.v[half], o.rows[half] * (2 * (int)p.vp_sn));
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        if constexpr (kVW == 4) *reinterpret_cast<u32x4*>(x.v[4 * half + r]) = __builtin_amdgcn_raw_buffer_load_b128(vr, v_lane, 2 * r * (uint32_t)p.vp_sn, 0);
        else *reinterpret_cast<u32x2*>(x.v[4 * half + r]) = __builtin_amdgcn_raw_buffer_load_b64(vr, v_lane, 2 * r * (uint32_t)p.vp_sn, 0);
      }
    }
  };
  u32x4 q[kKS], q2[kKS];
  auto load_q = [&](u32x4 (&q)[kKS], const PagedPlace<Place>& f, const Unit& u) __attribute__((always_inline)) {
    const uint16_t* qp = p.q + f.b * p.q_sb + (int64_t)(u.head0 + min(c16, u.n_cols - 1)) * p.q_sh + 8 * g;
#pragma unroll
    for (int s = 0; s < kKS; ++s) q[s] = *reinterpret_cast<const u32x4*>(qp + 32 * s);
  };

  Tile x;
  Unit u = {};
  if (at < end) {
    u = unit_of(f);
    load_q(q2, f, u);
    __builtin_amdgcn_sched_barrier(0);
    const Spot o = spot(u, f.tile, true);
    load_k(x, o);
    __builtin_amdgcn_sched_barrier(0);
    load_v(x, o);
  }
  while (at < end) {
    // ---- a unit's tiles [f.tile, last), and what comes after it -------------------------------------
    const Place unit_end = f.start + f.n_tiles + kOver;
    const int last = (int)min((Place)f.n_tiles, end - f.start - kOver);
    const Place at2 = min(unit_end, end);
    PagedPlace<Place> f2 = f;
    Unit u2 = u;
    const bool more = at2 < end;
    if (more) {
      f2.tile = 0;
      f2.start = unit_end;
      if (++f2.unit == units) {
        f2.unit = 0;
        ++f2.b;
        f2.length = p.batch <= kScan ? keys_at(keys0, f2.b) : keys_of<MODE>(p, f2.b, ((const_i32*)p.lengths)[f2.b]);
        f2.n_tiles = tiles_of(f2.length);
      }
      u2 = unit_of(f2);
    }
#pragma unroll
    for (int s = 0; s < kKS; ++s) q[s] = q2[s];
    load_q(q2, f2, u2);  // (the last unit's once more)
    __builtin_amdgcn_sched_barrier(0);
    const int length = u.length, head0 = u.head0, n_cols = u.n_cols;
    float m_run = -INFINITY, l_run = 0.f;
    floatx4 acc[kDV];
#pragma unroll
    for (int j = 0; j < kDV; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};

    auto scores = [&](const Tile& x, floatx4 (&s)[2]) __attribute__((always_inline)) {
      s[0] = s[1] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kKS; ++i)
#pragma unroll
        for (int half = 0; half < 2; ++half) s[half] = mfma16<T>(x.k[half][i], q[i], s[half]);
    };
    // rows behind the last key hold anything: their scores and values go
    auto seen = [&](const int t, const int i) __attribute__((always_inline)) { return kTile * t + 16 * (i >> 2) + 4 * g + (i & 3) < length; };
    auto probabilities = [&](floatx4 (&s)[2], const int t, u32x4& prob, u32x4& rest, const bool exact) __attribute__((always_inline)) {
      if (kTile * (t + 1) > length) {
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = seen(t, i) ? s[i >> 2][i & 3] : -INFINITY;
      }
      float mx = s[0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i >> 2][i & 3]);
      const float m_new = fmaxf(m_run, max_over_quarters(mx));
      const float m_base = m_new == -INFINITY ? 0.f : m_new;  // (no key of this column's so far)
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
    auto add_values = [&](Tile& x, const int t, const u32x4 prob, const u32x4 rest, const bool exact) __attribute__((always_inline)) {
      if (kTile * (t + 1) > length) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int w = 0; w < kVW; ++w) x.v[i][w] = seen(t, i) ? x.v[i][w] : 0u;
      }
#pragma unroll
      for (int w = 0; w < kVW; ++w)
#pragma unroll
        for (int odd = 0; odd < 2; ++odd) {
          u32x4 v;
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_perm(x.v[2 * i + 1][w], x.v[2 * i][w], odd ? 0x07060302u : 0x05040100u);
          acc[2 * w + odd] = mfma16<T>(v, prob, acc[2 * w + odd]);
          if (exact) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if ((v[i] & T::kExponent) == T::kExponent) v[i] &= 0xffff0000u;
              if (((v[i] >> 16) & T::kExponent) == T::kExponent) v[i] &= 0xffffu;
            }
          }
          acc[2 * w + odd] = mfma16<T>(v, rest, acc[2 * w + odd]);
        }
    };

    // A tile's keys are read before its soft-max and its values after it, and each at once gives its registers to the next tile's, which is the
    // next unit's first where this one has no more.
    for (int t = f.tile; t < last; ++t) {
      const bool here = t + 1 < last;
      Unit n;
      n.table = here ? u.table : u2.table;
      n.last_page = here ? u.last_page : u2.last_page;
      n.length = here ? u.length : u2.length;
      n.k_head = here ? u.k_head : u2.k_head;
      n.v_head = here ? u.v_head : u2.v_head;
      const Spot o = spot(n, here ? t + 1 : 0, here || more);
      floatx4 s[2];
      scores(x, s);
      __builtin_amdgcn_sched_barrier(0);
      load_k(x, o);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (MODE == kWeigh) {
        const int room = p.max_pages << p.page_log;
        float* to = p.scores + ((int64_t)f.b * p.n_q_heads + head0 + c16) * room + kTile * t + 4 * g;
        if (c16 < n_cols && kTile * (t + 1) > p.n_first) {
          *reinterpret_cast<floatx4*>(to) = s[0];
          if (kTile * t + 16 < room) *reinterpret_cast<floatx4*>(to + 16) = s[1];
        }
      }
      u32x4 prob, rest;
      probabilities(s, t, prob, rest, false);
      add_values(x, t, prob, rest, false);
      __builtin_amdgcn_sched_barrier(0);
      load_v(x, o);
    }
    l_run = sum_over_quarters(l_run);
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < kDV; ++j) sum += (acc[j][0] + acc[j][1]) + (acc[j][2] + acc[j][3]);
    if (__builtin_expect(__any(is_nan(sum) && !is_nan(l_run)), 0)) {
      // Infinite values: with two products per key they give NaN.  The wave's sums once more, relative to the maximum: the rest meets the
      // finite values only and a positive probability does not round to 0.
      l_run = 0.f;
#pragma unroll
      for (int j = 0; j < kDV; ++j) acc[j] = floatx4{0.f, 0.f, 0.f, 0.f};
      for (int t = f.tile; t < last; ++t) {
        Tile y;
        const Spot o = spot(u, t, true);
        load_k(y, o);
        load_v(y, o);
        floatx4 s[2];
        u32x4 prob, rest;
        scores(y, s);
        probabilities(s, t, prob, rest, true);
        add_values(y, t, prob, rest, true);
      }
      l_run = sum_over_quarters(l_run);
    }

    const bool from_start = f.tile == 0, to_end = last == f.n_tiles;
    if (from_start && to_end) {
      if (MODE == kWeigh && !weighs) {
        if (g == 0 && c16 < n_cols) *reinterpret_cast<floatx2*>(p.totals + 2 * ((int64_t)f.b * p.n_q_heads + head0 + c16)) = floatx2{m_run, l_run};
        if (lane == 0) *reinterpret_cast<int2*>(p.cuts + 2 * ((int64_t)f.b * units + f.unit)) = int2{0, 0};
      }
      bool joins = false;  // (with the state of the prefix, by paged_finish_kernel)
      if constexpr (MODE == kShared) {
        joins = ((const_i32*)p.skips)[f.b] > 0;
        if (lane == 0) *reinterpret_cast<int2*>(p.cuts + 2 * ((int64_t)f.b * units + f.unit)) = int2{0, 0};
        if (joins && c16 < n_cols) {
          const int64_t row = (int64_t)f.b * p.n_q_heads + head0 + c16;
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < kDV; j += 4)
              *reinterpret_cast<floatx4*>(p.own + row * D + kDV * (4 * g + r) + j) = floatx4{acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]};
          if (g == 0) *reinterpret_cast<floatx2*>(p.own_stats + 2 * row) = floatx2{m_run, l_run};
        }
      }
      const float inv = length == 0 ? 0.f : 1.f / l_run;  // (no keys: 0; keys whose scores are all minus infinity: 0 / 0, as a soft-max has it)
      if (MODE == kWeigh && weighs) {  // (this wave's own scores, which it has stored)
        if (g == 0) wave_totals[wave][c16] = floatx2{m_run, 1.f / l_run};
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        for (int i = first_counted(p, length) + 4 * lane; i < length; i += 256) {
          floatx4 sum = {0.f, 0.f, 0.f, 0.f};
          add_probabilities<T>(p, (int64_t)f.b * p.n_q_heads + head0, n_cols, i, scale, sum, [&](const int h) { return wave_totals[wave][h]; });
          add_to_weights(p, f.b, u.kvh, i, length, sum);
        }
      }
      if (c16 < n_cols && !joins) {
        uint16_t* op = p.out + f.b * p.o_sb + (int64_t)(head0 + c16) * p.o_sh + kDV * 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < kDV; j += 4)
            *reinterpret_cast<u32x2*>(op + kDV * r + j) = u32x2{T::pack(acc[j][r] * inv, acc[j + 1][r] * inv), T::pack(acc[j + 2][r] * inv, acc[j + 3][r] * inv)};
      }
    } else {
      const int which = from_start ? 1 : 0;
      if (g == 0) {
        stats[wave][which][0][c16] = m_run;
        stats[wave][which][1][c16] = l_run;
      }
      if (c16 < n_cols) {
        float* to = states + ((2 * wave + which) * most_cols + c16) * kPitch + kDV * 4 * g;
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < kDV; j += 4) *reinterpret_cast<floatx4*>(to + kDV * r + j) = floatx4{acc[j][r], acc[j + 1][r], acc[j + 2][r], acc[j + 3][r]};
      }
      // (how many shares its places from this one's beginning on are)
      if (lane == 0) {
        const uint32_t left = (uint32_t)(unit_end - 1 - raw);
        parts_of[wave][which] = int4{1 + (int)to_end, f.b, n_cols << 16 | head0, share > (Place)left ? 1 : 1 + (int)(left / (uint32_t)share)};
      }
    }
    at = at2;
    f = f2;
    u = u2;
  }

  // ---- the waves' parts of a unit -> one ------------------------------------------------------------
  __syncthreads();
  int4* header = reinterpret_cast<int4*>(p.headers) + blockIdx.x;
  bool goes_on = false;
  // the unit that began before this work-group, then those that begin in a wave and do not end there.  (Entry 2 w + which of parts_of is a lane's; waves without
  // a share have none)
  const int4 mine = parts_of[min(lane, 2 * WAVES - 1) >> 1][lane & 1];
  uint32_t left = (uint32_t)__ballot(lane < 2 * WAVES && mine.x != 0);
  const uint32_t last_ones = (uint32_t)__ballot(lane < 2 * WAVES && mine.x == 2);
  while (left != 0) {
    const int first = __builtin_ctz(left);
    const bool begins = first & 1;
    uint32_t entries = 1u << first;  // of this unit
    left &= left - 1;
    bool ends = last_ones & entries;
    while (!ends && left != 0 && !(__builtin_ctz(left) & 1)) {
      const uint32_t next = left & -left;
      entries |= next;
      ends = last_ones & next;
      left &= left - 1;
    }
    const int4 info = {0, __builtin_amdgcn_readlane(mine.y, first), __builtin_amdgcn_readlane(mine.z, first), __builtin_amdgcn_readlane(mine.w, first)};
    const int head0 = info.z & 0xffff, n_cols = info.z >> 16;
    for (int i = tid; i < n_cols * (D / 4); i += 64 * WAVES) {
      const int col = i / (D / 4), d = 4 * (i % (D / 4));
      float m = -INFINITY, l = 0.f, ms[WAVES], ls[WAVES];
      floatx4 x = {0.f, 0.f, 0.f, 0.f}, xs[WAVES];
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {  // (one entry a wave: the second of the one that the unit begins in, the first of others; all are read at once)
        const int k = 2 * w + 1 == first;
        ms[w] = stats[w][k][0][col];
        ls[w] = stats[w][k][1][col];
        xs[w] = *reinterpret_cast<const floatx4*>(states + ((2 * w + k) * most_cols + col) * kPitch + d);
      }
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        ms[w] = entries >> (2 * w) & 3u ? ms[w] : -INFINITY;
        m = fmaxf(m, ms[w]);
      }
#pragma unroll
      for (int w = 0; w < WAVES; ++w) {
        if (!(entries >> (2 * w) & 3u)) continue;
        const float weight = ms[w] == -INFINITY ? 0.f : fast_exp2((ms[w] - m) * scale);
        l += weight * ls[w];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] += weight * xs[w][e];
      }
      if (begins && ends) {
        if constexpr (MODE == kShared) {
          if (((const_i32*)p.skips)[info.y] > 0) {
            const int64_t row = (int64_t)info.y * p.n_q_heads + head0 + col;
            *reinterpret_cast<floatx4*>(p.own + row * D + d) = x;
            if (d == 0) *reinterpret_cast<floatx2*>(p.own_stats + 2 * row) = floatx2{m, l};
            continue;
          }
        }
        if (MODE == kWeigh && d == 0) {
          if (weighs) unit_totals[col] = floatx2{m, 1.f / l};
          else *reinterpret_cast<floatx2*>(p.totals + 2 * ((int64_t)info.y * p.n_q_heads + head0 + col)) = floatx2{m, l};
        }
        const float inv = 1.f / l;  // (a unit that is cut has keys)
        uint16_t* op = p.out + info.y * p.o_sb + (int64_t)(head0 + col) * p.o_sh + d;
        *reinterpret_cast<u32x2*>(op) = u32x2{T::pack(x[0] * inv, x[1] * inv), T::pack(x[2] * inv, x[3] * inv)};
      } else {
        const int64_t to = (int64_t)(2 * blockIdx.x + (begins ? 1 : 0)) * kCols + col;
        *reinterpret_cast<floatx4*>(p.parts + to * D + d) = x;
        if (d == 0) {
          p.part_stats[2 * to] = m;
          p.part_stats[2 * to + 1] = l;
        }
      }
    }
    if (MODE == kWeigh && weighs) {
      __syncthreads();  // (all waves have stored their scores before the parts were joined)
      const int n = keys_of<MODE>(p, info.y, ((const_i32*)p.lengths)[info.y]);
      for (int i = first_counted(p, n) + 4 * tid; i < n; i += 256 * WAVES) {
        floatx4 sum = {0.f, 0.f, 0.f, 0.f};
        add_probabilities<T>(p, (int64_t)info.y * p.n_q_heads + head0, n_cols, i, scale, sum, [&](const int h) { return unit_totals[h]; });
        add_to_weights(p, info.y, head0 / group, i, n, sum);
      }
      __syncthreads();  // (before the next unit's totals)
    } else if (MODE != kPlain && begins && tid == 0) {
      const int kvh = head0 / group, unit = kvh * col_blocks + (head0 - kvh * group) / kCols;
      *reinterpret_cast<int2*>(p.cuts + 2 * ((int64_t)info.y * units + unit)) = ends ? int2{0, 0} : int2{(int)blockIdx.x, info.w};
    }
    if (begins && !ends) {  // the unit's other parts are the next work-groups'
      goes_on = true;
      if (MODE != kShared && tid == 0) *header = int4{info.w, info.y, head0, n_cols};
    }
  }
  if (MODE != kShared && !goes_on && tid == 0 && p.headers != nullptr) header->x = 0;
}

// Joins the parts of a column whose unit begins in share blockIdx.y and ends in another (units begin every so many shares: shares as blockIdx.x would be one XCD's): the
// weights first, then groups of D / 4 lanes add up
// every so many parts.  Few bytes; the launch and three loads one after the other take 3 to 5 us, which a step pays whether or not a unit was cut, since the
// host does not know the lengths.
template <typename T, int D>
__device__ __forceinline__ void combine(const PagedDecodeArgs& p, const int col, const int share) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ float weight[256], red[2][4];
  __shared__ floatx4 sums[kGroups][kLanes];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int4 header = *reinterpret_cast<const int4*>(p.headers + 4 * share);
  const int parts = header.x;
  if (parts == 0 || col >= header.w) return;
  const float scale = p.sm_scale * kLog2e;
  // the first part is the second of its share, the others the first of theirs
  auto part = [&](const int i) { return ((int64_t)2 * (share + i) + (i == 0 ? 1 : 0)) * kCols + col; };
  static_assert(kShares <= 256, "a thread has a part's maximum and sum");
  const int gr = tid / kLanes, d4 = tid % kLanes;
  floatx4 early[4];  // (requested with the maxima)
#pragma unroll
  for (int j = 0; j < 4; ++j) early[j] = *reinterpret_cast<const floatx4*>(p.parts + part(min(gr + j * kGroups, parts - 1)) * D + 4 * d4);
  const float mine = tid < parts ? p.part_stats[2 * part(tid)] : -INFINITY;
  float l = tid < parts ? p.part_stats[2 * part(tid) + 1] : 0.f;
  float m = over_wave(mine, -INFINITY, [](const float a, const float b) { return fmaxf(a, b); });
  if (lane == 0) red[0][wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  const float w = mine == -INFINITY ? 0.f : fast_exp2((mine - m) * scale);
  weight[tid] = w;
  l = over_wave(l * w, 0.f, [](const float a, const float b) { return a + b; });
  if (lane == 0) red[1][wave] = l;
  __syncthreads();
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (gr + j * kGroups < parts) {
      const float w = weight[gr + j * kGroups];
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += w * early[j][e];
    }
#pragma unroll 4
  for (int i = gr + 4 * kGroups; i < parts; i += kGroups) {
    const floatx4 x = *reinterpret_cast<const floatx4*>(p.parts + part(i) * D + 4 * d4);
    const float w = weight[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += w * x[e];
  }
  sums[gr][d4] = sum;
  __syncthreads();
  if (tid < kLanes) {
#pragma unroll
    for (int i = 1; i < kGroups; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += sums[i][tid][e];
    l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const float inv = 1.f / l;
    uint16_t* op = p.out + header.y * p.o_sb + (int64_t)(header.z + col) * p.o_sh + 4 * tid;
    *reinterpret_cast<u32x2*>(op) = u32x2{T::pack(sum[0] * inv, sum[1] * inv), T::pack(sum[2] * inv, sum[3] * inv)};
  }
}
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_combine_kernel(const PagedDecodeArgs p) {
  combine<T, D>(p, blockIdx.x, blockIdx.y);
}

// Joins what is known of a unit's heads over the shared prefix and over the sequence's own keys, each whole or in parts.  256 threads have four channels of a head each; of few heads, every
// so many of its parts.  Heads lie beside one another in a wave as they do in the parts of many rows, and fours of channels as in the others.  Bound by the latency of what it
// reads, each thing known by the one before (cut, unit, parts): 32 sequences behind 32768 keys, 32/8 heads of 128 (256 work-groups of 32 parts) 9.0 us, of the step's 65.  (The prefix joined
// by a launch of its own, before the decode kernel, which read its state: 61.3 a step.  A head's channels side by side in a wave: 9.7 us.)
// A line of many rows' parts has heads of two sequences, which should be one XCD's: neighbours are where an XCD's share is consecutive, or, of 8 units a sequence, where each has its own
// (128 sequences, 28/4 heads of 128, in plain order 51.8 us a step, so 50.0).
constexpr int kXcds = 8;
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_finish_kernel(const PagedDecodeArgs p) {
  constexpr int kLanes = D / 4, kHeads = 256 / kLanes, kFours = D / 8;
  __shared__ floatx4 sums[256];
  __shared__ floatx2 stats[256];
  const int group = p.n_q_heads / p.n_kv_heads, col_blocks = (group + kCols - 1) / kCols, units = p.n_kv_heads * col_blocks, tid = threadIdx.x;
  const int at = units % kXcds == 0 ? blockIdx.x : blockIdx.x % kXcds * (gridDim.x / kXcds) + blockIdx.x / kXcds;
  const int b = at / units, unit = at - b * units, kvh = col_blocks == 1 ? unit : unit / col_blocks;
  if (b >= p.batch) return;
  const int head0 = kvh * group + (unit - kvh * col_blocks) * kCols, n_cols = min(kCols, (kvh + 1) * group - head0);
  const const_i32* cut = (const_i32*)p.cuts + 2 * ((int64_t)b * units + unit);
  const int skip = ((const_i32*)p.skips)[b], of_group = ((const_i32*)p.firsts)[b], first = cut[0], parts = cut[1], prefix_rows = *(const_i32*)p.prefix_rows;
  if (skip == 0 && parts == 0) return;  // (the decode kernel's own)
  int heads_log = 0;
  while (1 << heads_log < min(n_cols, kHeads)) ++heads_log;
  const int heads = 1 << heads_log, side = kHeads >> heads_log, d = 4 * ((tid >> heads_log) % kLanes), sub = (tid >> heads_log) / kLanes;
  const float scale = p.sm_scale * kLog2e;
  for (int col0 = 0; col0 < n_cols; col0 += heads) {
    const int col = col0 + (tid & (heads - 1)), head = head0 + min(col, n_cols - 1);
    const int64_t row = (int64_t)b * p.n_q_heads + head;
    // (read where they are not there too: sooner than what says so)
    const floatx2 own_stats = *reinterpret_cast<const floatx2*>(p.own_stats + 2 * row);
    const floatx4 own = *reinterpret_cast<const floatx4*>(p.own + row * D + d);
    const bool has = parts == 0 && sub == 0;
    float m = has ? own_stats[0] : -INFINITY, l = has ? own_stats[1] : 0.f;
    floatx4 x = {has ? own[0] : 0.f, has ? own[1] : 0.f, has ? own[2] : 0.f, has ? own[3] : 0.f};
    auto add = [&](const floatx2 s, const floatx4 y) __attribute__((always_inline)) {
      const float m_new = fmaxf(m, s[0]), w = m == -INFINITY ? 0.f : fast_exp2((m - m_new) * scale), w2 = s[0] == -INFINITY ? 0.f : fast_exp2((s[0] - m_new) * scale);
      m = m_new;
      l = w * l + w2 * s[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = w * x[e] + w2 * y[e];
    };
    auto add_all = [&](const int n, auto stats_at, auto part_at) __attribute__((always_inline)) {  // a part's statistics and accumulators
      constexpr int kSide = 8;  // that are read side by side
      for (int i = sub; i < n; i += side * kSide) {
        floatx2 s[kSide];
        floatx4 y[kSide];
#pragma unroll
        for (int j = 0; j < kSide; ++j) {
          const int at = min(i + side * j, n - 1);
          s[j] = *reinterpret_cast<const floatx2*>(stats_at(at));
          y[j] = *reinterpret_cast<const floatx4*>(part_at(at));
        }
#pragma unroll
        for (int j = 0; j < kSide; ++j)
          if (i + side * j < n) add(s[j], y[j]);
      }
    };
    // (the first part of several is the second of its share, the others the first of theirs)
    if (skip > 0) {
      const int in_group = (b - of_group) * group + head - kvh * group, row0 = in_group & -prefix_rows, s0 = row0 / group, r = in_group - row0;
      const int2 entry = *reinterpret_cast<const int2*>(p.entries + 2 * ((int64_t)(of_group + s0) * p.n_q_heads + kvh * group + row0 - s0 * group));
      if (entry.y == 0) {
        if (sub == 0) add(*reinterpret_cast<const floatx2*>(p.prefix_stats + 2 * row), *reinterpret_cast<const floatx4*>(p.prefix + row * D + d));
      } else if (prefix_rows != 16) {  // four waves' 32 rows, fours of channels lane by lane
        const int lane = (r & 31) + 32 * (d >> 2 & 1), f = d >> 3;
        auto at = [&](const int i) { return ((int64_t)2 * (entry.x + i) + (i == 0 ? 1 : 0)) * 4 + (r >> 5); };
        add_all(entry.y, [&](const int i) { return p.prefix_part_stats + (at(i) * 64 + lane) * 2; }, [&](const int i) { return p.prefix_parts + ((at(i) * kFours + f) * 64 + lane) * 4; });
      } else {
        auto at = [&](const int i) { return ((int64_t)2 * (entry.x + i) + (i == 0 ? 1 : 0)) * 16 + r; };
        add_all(entry.y, [&](const int i) { return p.prefix_part_stats + 2 * at(i); }, [&](const int i) { return p.prefix_parts + at(i) * D + d; });
      }
    }
    if (parts > 0) {
      auto at = [&](const int i) { return ((int64_t)2 * (first + i) + (i == 0 ? 1 : 0)) * kCols + (head - head0); };
      add_all(parts, [&](const int i) { return p.part_stats + 2 * at(i); }, [&](const int i) { return p.parts + at(i) * D + d; });
    }
    if (side > 1) {
      sums[tid] = x;
      stats[tid] = floatx2{m, l};
      __syncthreads();
      if (sub == 0)
        for (int i = 1; i < side; ++i) add(stats[tid + i * heads * kLanes], sums[tid + i * heads * kLanes]);
    }
    if (sub == 0 && col < n_cols) {
      const float inv = 1.f / l;
      *reinterpret_cast<u32x2*>(p.out + b * p.o_sb + (int64_t)head * p.o_sh + d) = u32x2{T::pack(x[0] * inv, x[1] * inv), T::pack(x[2] * inv, x[3] * inv)};
    }
    if (side > 1) __syncthreads();
  }
}

// Scratch of a step: a header, and two parts of 16 columns, for each share.  None where no unit is cut.
PagedScratch paged_decode_scratch(int batch, int n_q_heads, int n_kv_heads, int head_dim, int page_log, int max_pages) {
  PagedScratch s = {0, 0, 0, 0};
  const int64_t units = (int64_t)batch * n_kv_heads * ((n_q_heads / n_kv_heads + kCols - 1) / kCols);
  const int whole = units > kMany ? kWholeMany : head_dim == 64 ? kWhole<64> : kWhole<128>;
  if (max_pages << page_log <= whole * kTile) return s;
  s.stats = (size_t)kShares * 16;
  s.parts = s.stats + (size_t)kShares * 2 * kCols * 8;
  s.total = s.parts + (size_t)kShares * 2 * kCols * head_dim * 4;
  return s;
}

// Adds to each key's weight what its KV head's queries have given it: the sum over the heads of the group of 2^((score - maximum) * scale) / sum, from the scores that the
// decode kernel has left.  Bound by reading these once.  A thread has four keys, a work-group 1024, and as many more as it takes for all of a sequence's.  The work-groups before these
// join the parts of cut units, whose maxima and sums are therefore joined here once more, 16 heads at a time, instead of waiting for them: one sequence of 131071 keys, 28/4
// heads of 128, 7.9 us beside the decode kernel's 44.5, 69.3 a step (71.8 with the join and this one after the other); 16 of 500 to 16000, 32/8 of 128, 10.0 beside 59.8, 79 a step, where a copy of what is
// read and written takes 61.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_weigh_kernel(const PagedDecodeArgs p, const int combiners, const int cols, const int side) {
  __shared__ floatx2 parts_of[16][kCols], totals[kCols];
  if ((int)blockIdx.x < combiners) {
    const int share = blockIdx.x / cols;
    return combine<T, D>(p, blockIdx.x - share * cols, share);
  }
  const int tid = threadIdx.x, at = blockIdx.x - combiners, u = at / side, b = u / p.n_kv_heads, kvh = u - b * p.n_kv_heads;
  const int group = p.n_q_heads / p.n_kv_heads, col_blocks = (group + kCols - 1) / kCols, n = keys_of<kWeigh>(p, b, p.lengths[b]);
  const int64_t head0 = (int64_t)b * p.n_q_heads + (int64_t)kvh * group;
  const float scale = p.sm_scale * kLog2e;
  const int first = first_counted(p, n) + (at - u * side) * 1024;
  if (first >= n) return;
  auto find_totals = [&](const int block) {  // of its heads: maxima, and what probabilities are multiplied by
    const int2 cut = *reinterpret_cast<const int2*>(p.cuts + 2 * ((int64_t)u * col_blocks + block));
    const int col = tid & 15, slice = tid >> 4;
    float m = -INFINITY, l = 0.f;
    if (cut.y == 0) {
      if (slice == 0 && kCols * block + col < group) {
        const floatx2 x = *reinterpret_cast<const floatx2*>(p.totals + 2 * (head0 + kCols * block + col));
        m = x[0];
        l = x[1];
      }
    } else {
      for (int i = slice; i < cut.y; i += 16) {
        const floatx2 x = *reinterpret_cast<const floatx2*>(p.part_stats + 2 * (((int64_t)2 * (cut.x + i) + (i == 0 ? 1 : 0)) * kCols + col));
        const float m_new = fmaxf(m, x[0]), w = m == -INFINITY ? 0.f : fast_exp2((m - m_new) * scale), w2 = x[0] == -INFINITY ? 0.f : fast_exp2((x[0] - m_new) * scale);
        l = w * l + w2 * x[1];
        m = m_new;
      }
    }
    parts_of[slice][col] = floatx2{m, l};
    __syncthreads();
    if (tid < kCols) {
      m = -INFINITY;
      l = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) m = fmaxf(m, parts_of[i][tid][0]);
#pragma unroll
      for (int i = 0; i < 16; ++i) {  // (the sum of a part whose scores are all NaN, which has no maximum, is NaN and stays so)
        const floatx2 x = parts_of[i][tid];
        l += (x[0] == -INFINITY ? 0.f : fast_exp2((x[0] - m) * scale)) * x[1];
      }
      totals[tid] = floatx2{m, 1.f / l};  // (of none, and of scores that are all minus infinity, infinity times 0)
    }
    __syncthreads();
  };
  if (col_blocks == 1) find_totals(0);
  for (int i0 = first; i0 < n; i0 += side * 1024) {
    const int i = i0 + 4 * tid;
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
    for (int block = 0; block < col_blocks; ++block) {
      if (col_blocks > 1) find_totals(block);
      if (i >= n) continue;
      add_probabilities<T>(p, head0 + kCols * block, min(kCols, group - kCols * block), i, scale, sum, [&](const int h) { return totals[h]; });
    }
    if (i < n) add_to_weights(p, b, kvh, i, n, sum);
  }
}

template <typename T, int D, DecodeMode MODE>
static void launch_paged_decode_as(const PagedDecodeArgs& a, hipStream_t stream) {
  const int group = a.n_q_heads / a.n_kv_heads, cols = group < kCols ? group : kCols, units = a.n_kv_heads * ((group + kCols - 1) / kCols);
  const size_t lds = (size_t)8 * cols * (D + 4) * 4;
  // (places fit 32 bits unless thousands of sequences have tables for a million keys)
  const int64_t most = (int64_t)a.batch * units * (((int64_t)a.max_pages << a.page_log) / kTile + 1 + kOver);
  if (most < 1ll << 30) hipLaunchKernelGGL((paged_decode_kernel<T, D, 4, int, MODE>), dim3(kShares), dim3(256), lds, stream, a);
  else hipLaunchKernelGGL((paged_decode_kernel<T, D, 4, int64_t, MODE>), dim3(kShares), dim3(256), lds, stream, a);
  if constexpr (MODE == kWeigh) {
    if (a.headers == nullptr && group <= kCols) return;  // (the decode kernel has done it: 600 keys, 14/2 heads of 64, 14.5 -> 12 us)
    // work-groups of a (sequence, KV head): as many as its table has room for, or fewer where there are thousands in all
    const int64_t all = (int64_t)a.batch * a.n_kv_heads, room = (((int64_t)a.max_pages << a.page_log) + 1023) / 1024, each = all < 8192 ? 8192 / all : 1;
    const int side = (int)(room < each ? room : each), combiners = a.headers != nullptr ? kShares * cols : 0;
    hipLaunchKernelGGL((paged_weigh_kernel<T, D>), dim3((uint32_t)(combiners + side * all)), dim3(256), 0, stream, a, combiners, cols, side);
  } else if constexpr (MODE == kShared) {
    hipLaunchKernelGGL((paged_finish_kernel<T, D>), dim3(((uint32_t)((int64_t)a.batch * units) + kXcds - 1) / kXcds * kXcds), dim3(256), 0, stream, a);
  } else {
    if (a.headers != nullptr) hipLaunchKernelGGL((paged_combine_kernel<T, D>), dim3(cols, kShares), dim3(256), 0, stream, a);
  }
}

template <typename T, int D>
static void launch_paged_decode_for(const PagedDecodeArgs& a, hipStream_t stream) {
  if (a.scores != nullptr) launch_paged_decode_as<T, D, kWeigh>(a, stream);
  else if (a.skips != nullptr) launch_paged_decode_as<T, D, kShared>(a, stream);
  else launch_paged_decode_as<T, D, kPlain>(a, stream);
}

hipError_t launch_paged_decode(const PagedDecodeArgs& a, hipStream_t stream) {
  if (a.head_dim == 128) {
    if (a.dtype == 0) launch_paged_decode_for<Bf16, 128>(a, stream);
    else launch_paged_decode_for<F16, 128>(a, stream);
  } else {
    if (a.dtype == 0) launch_paged_decode_for<Bf16, 64>(a, stream);
    else launch_paged_decode_for<F16, 64>(a, stream);
  }
  return hipGetLastError();
}

}  // namespace aa
