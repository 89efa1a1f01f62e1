// Attention of one new token per sequence over a key/value cache in pages, on gfx950.
//
// Bound by reading keys and values once.  A unit is a (sequence, KV head) with up to 16 heads of its group as the columns of 16 x 16 x 32 MFMAs; its
// keys come in tiles of 32.  Lengths are known on the device only and may differ a lot, so the tiles of all units, one after the other, are cut into equal
// shares, one for each of a fixed number of work-groups, and each share into equal parts of its four waves: every wave sums the lengths and finds its part
// by itself.  A wave walks its part alone, from unit to unit, and nothing passes through LDS until the end, where the states (maximum, sum, accumulator) of units
// that several waves have are joined.  A share that begins or ends inside a unit leaves that unit's state in the workspace, two states at most, and
// paged_combine_kernel joins them in order, so that results do not depend on timing.  Where the table has room for few tiles only, no unit is cut between
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

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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

// Place: an integer that counts the tiles of all units
template <typename Place>
struct PagedPlace {       // of a tile, among all
  int b, unit, tile;      // sequence, unit of it, tile of the unit
  int n_tiles, length;    // of the sequence
  Place start;            // the unit's beginning
};

// keys that are read of a sequence
__device__ __forceinline__ int keys_of(const PagedDecodeArgs& p, const int length) {
  const int n = min(max(length, 0), p.max_pages << p.page_log);
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

template <typename T, int D, int WAVES, typename Place>
__global__ void __launch_bounds__(64 * WAVES, 2) paged_decode_kernel(const PagedDecodeArgs p) {
  constexpr int kKS = D / 32;      // MFMAs of a score
  constexpr int kDV = D / 16;      // channels of V that a lane loads
  constexpr int kVW = kDV / 2;     // ... in words
  constexpr int kPitch = D + 4;
  // States of units that a wave has a part of only: [wave][0: the first of its units, which began before; 1: its last, which goes on][column]
  extern __shared__ __attribute__((aligned(16))) float states[];
  __shared__ float stats[WAVES][2][2][kCols];
  __shared__ int4 parts_of[WAVES][2];  // 0 if there is none, 2 if the unit ends in it; sequence; first head, and columns in the upper half; parts of work-groups

  const int tid = threadIdx.x, lane = tid & 63, c16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = p.n_q_heads / p.n_kv_heads, col_blocks = (group + kCols - 1) / kCols, units = p.n_kv_heads * col_blocks;
  const int most_cols = min(group, kCols);

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
      keys[j] = b < p.batch ? keys_of(p, p.lengths[b]) : 0;
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
        f2.length = p.batch <= kScan ? keys_at(keys0, f2.b) : keys_of(p, ((const_i32*)p.lengths)[f2.b]);
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
      const float inv = length == 0 ? 0.f : 1.f / l_run;  // (no keys: 0; keys whose scores are all minus infinity: 0 / 0, as a soft-max has it)
      if (c16 < n_cols) {
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
    if (begins && !ends) {  // the unit's other parts are the next work-groups'
      goes_on = true;
      if (tid == 0) *header = int4{info.w, info.y, head0, n_cols};
    }
  }
  if (!goes_on && tid == 0 && p.headers != nullptr) header->x = 0;
}

// Joins the parts of a column whose unit begins in share blockIdx.x and ends in another: the weights first, then groups of D / 4 lanes add up
// every so many parts.  Few bytes; the launch and three loads one after the other take 3 to 5 us, which a step pays whether or not a unit was cut, since the
// host does not know the lengths.
template <typename T, int D>
__global__ void __launch_bounds__(256) paged_combine_kernel(const PagedDecodeArgs p) {
  constexpr int kLanes = D / 4, kGroups = 256 / kLanes;
  __shared__ float weight[256], red[2][4];
  __shared__ floatx4 sums[kGroups][kLanes];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, col = blockIdx.y;
  const int4 header = *reinterpret_cast<const int4*>(p.headers + 4 * blockIdx.x);
  const int parts = header.x;
  if (parts == 0 || col >= header.w) return;
  const float scale = p.sm_scale * kLog2e;
  // the first part is the second of its share, the others the first of theirs
  auto part = [&](const int i) { return ((int64_t)2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * kCols + col; };
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

template <typename T, int D>
static void launch_paged_decode_for(const PagedDecodeArgs& a, hipStream_t stream) {
  const int group = a.n_q_heads / a.n_kv_heads, cols = group < kCols ? group : kCols, units = a.n_kv_heads * ((group + kCols - 1) / kCols);
  const size_t lds = (size_t)8 * cols * (D + 4) * 4;
  // (places fit 32 bits unless thousands of sequences have tables for a million keys)
  const int64_t most = (int64_t)a.batch * units * (((int64_t)a.max_pages << a.page_log) / kTile + 1 + kOver);
  if (most < 1ll << 30) hipLaunchKernelGGL((paged_decode_kernel<T, D, 4, int>), dim3(kShares), dim3(256), lds, stream, a);
  else hipLaunchKernelGGL((paged_decode_kernel<T, D, 4, int64_t>), dim3(kShares), dim3(256), lds, stream, a);
  if (a.headers != nullptr) hipLaunchKernelGGL((paged_combine_kernel<T, D>), dim3(kShares, cols), dim3(256), 0, stream, a);
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
