// Giving up the keys of a cache in pages that have had the least attention, on gfx950: which ones stay, and their move to the front of the sequence's pages.
//
// Choosing: a work-group for each (sequence, KV head) finds the weight that the wanted number of candidates reaches, by histograms of 8 bits of the weights' order at a time,
// and then lists the places in order, chunk by chunk, with sums over the work-group.  Integers only: the order in which counts are added does not matter.
// Moving is bound by reading and writing the rows once.  It is in place, and a row goes to a lower place: rows that lie where others will go (below the n_keys-th) are copied to
// scratch by a launch of its own first, the others are read where they are, which nothing writes.  A work-group has a page of a KV head, whose bounds it forms.
#include "aa_kernels.h"
#include "aa_paged.h"

namespace aa {

constexpr int kEvictThreads = 1024, kEvictWaves = kEvictThreads / 64;

__global__ void __launch_bounds__(kEvictThreads) paged_keep_kernel(const PagedEvictArgs p) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t counts[kEvictWaves][2], found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x / p.n_kv_heads, kvh = blockIdx.x % p.n_kv_heads;
  const int n = clamped_length(p.lengths, b, p.max_pages, p.page_log);
  int32_t* kept = p.kept + (int64_t)blockIdx.x * p.n_keys;
  if (kvh == 0 && tid == 0) p.new_lengths[b] = n > p.above ? p.n_keys : n;
  if (n <= p.above) {
    for (int i = tid; i < p.n_keys; i += kEvictThreads) kept[i] = -1;
    return;
  }
  const int first = p.n_first, end = n - p.n_last;  // the candidates
  auto key_at = [&](const int i) {
    const int64_t page = clamped_page(p.table[b * p.t_sb + (i >> p.page_log)], p.n_pages);
    return ordered(p.weights[((page * p.n_kv_heads + kvh) << p.page_log) + (i & ((1 << p.page_log) - 1))]);
  };
  uint32_t want = p.n_keys - p.n_first - p.n_last, prefix = 0;  // of them, those of this prefix and not above it
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = first + tid; i < end; i += kEvictThreads) {
      const uint32_t x = key_at(i);
      if (shift == 24 || x >> (shift + 8) == prefix) atomicAdd(&hist[x >> shift & 255u], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t left = want, bin = 255;
      while (bin > 0 && hist[bin] < left) left -= hist[bin--];
      found[0] = bin;
      found[1] = left;
    }
    __syncthreads();
    prefix = prefix << 8 | found[0];
    want = found[1];
  }
  // larger ones all, `want` of the equal ones
  for (int i = tid; i < first; i += kEvictThreads) kept[i] = i;
  for (int i = tid; i < p.n_last; i += kEvictThreads) kept[p.n_keys - p.n_last + i] = end + i;
  uint32_t above = 0, equal = 0;  // before this chunk
  for (int i0 = first; i0 < end; i0 += kEvictThreads) {
    const int i = i0 + tid;
    const uint32_t x = i < end ? key_at(i) : 0u;
    const bool gt = i < end && x > prefix, eq = i < end && x == prefix;
    const uint64_t gts = __ballot(gt), eqs = __ballot(eq);
    if (lane == 0) {
      counts[wave][0] = __popcll(gts);
      counts[wave][1] = __popcll(eqs);
    }
    __syncthreads();
    uint32_t a = above, e = equal;
    for (int w = 0; w < kEvictWaves; ++w) {
      if (w == wave) {
        const uint64_t before = (1ull << lane) - 1;
        a += __popcll(gts & before);
        e += __popcll(eqs & before);
        if (gt || (eq && e < want)) kept[first + a + min(e, want)] = i;
      }
      above += counts[w][0];
      equal += counts[w][1];
      if (w < wave) {
        a = above;
        e = equal;
      }
    }
    __syncthreads();
  }
}

// Where row i of a (sequence, KV head) is.
struct EvictRow {
  int64_t k, v, w;
  bool ok;
};
__device__ __forceinline__ EvictRow row_at(const PagedEvictArgs& p, const int b, const int kvh, const int i) {
  const int page = p.table[b * p.t_sb + (i >> p.page_log)], slot = i & ((1 << p.page_log) - 1);
  const int64_t at = clamped_page(page, p.n_pages);
  return {at * p.kp_sp + kvh * p.kp_sh + slot * p.kp_sn, at * p.vp_sp + kvh * p.vp_sh + slot * p.vp_sn, ((at * p.n_kv_heads + kvh) << p.page_log) + slot, at == page};
}

// Rows that move from where others go, to scratch.
template <int D>
__global__ void __launch_bounds__(256) paged_save_kernel(const PagedEvictArgs p) {
  constexpr int kPieces = D / 8, kSide = 256 / kPieces;
  const int c = threadIdx.x % kPieces, kvh = blockIdx.y, b = blockIdx.z;
  const int64_t unit = ((int64_t)b * p.n_kv_heads + kvh) * p.n_keys;
  const int begin = blockIdx.x << p.page_log, end = min(begin + (1 << p.page_log), p.n_keys);
  for (int i = begin + threadIdx.x / kPieces; i < end; i += kSide) {
    const int from = p.kept[unit + i];
    if (from < 0 || from == i || from >= p.n_keys) continue;
    const EvictRow x = row_at(p, b, kvh, from);
    uint16_t* to = p.rows + (unit + i) * 2 * D + 8 * c;
    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(p.keys + x.k + 8 * c);
    *reinterpret_cast<uint4*>(to + D) = *reinterpret_cast<const uint4*>(p.values + x.v + 8 * c);
    if (c == 0) p.row_weights[unit + i] = p.weights[x.w];
  }
}

template <typename T, int D>
__global__ void __launch_bounds__(256) paged_move_kernel(const PagedEvictArgs p) {
  constexpr int kPieces = D / 8, kSide = 256 / kPieces;
  __shared__ uint32_t red[4][kPieces][8];
  const int tid = threadIdx.x, lane = tid & 63, c = tid % kPieces, kvh = blockIdx.y, b = blockIdx.z;
  const int64_t unit = ((int64_t)b * p.n_kv_heads + kvh) * p.n_keys;
  const int begin = blockIdx.x << p.page_log, end = min(begin + (1 << p.page_log), p.n_keys);
  // (a page stays as it is if its last row does and none is taken from behind that)
  const int last = p.kept[unit + end - 1];
  if (last < 0 || (last == end - 1 && end - begin == 1 << p.page_log)) return;
  uint32_t lo[4] = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu}, hi[4] = {0x80008000u, 0x80008000u, 0x80008000u, 0x80008000u};
  for (int i = begin + tid / kPieces; i < end; i += kSide) {
    const int from = p.kept[unit + i];
    const EvictRow to = row_at(p, b, kvh, i), x = row_at(p, b, kvh, from);
    const bool saved = from != i && from < p.n_keys;
    const uint16_t* rows = p.rows + (unit + i) * 2 * D;
    const uint4 k = *reinterpret_cast<const uint4*>((saved ? rows : p.keys + x.k) + 8 * c);
    if (from != i && to.ok) {
      const uint4 v = *reinterpret_cast<const uint4*>((saved ? rows + D : p.values + x.v) + 8 * c);
      const float w = saved ? p.row_weights[unit + i] : p.weights[x.w];
      *reinterpret_cast<uint4*>(p.keys + to.k + 8 * c) = k;
      *reinterpret_cast<uint4*>(p.values + to.v + 8 * c) = v;
      if (c == 0) p.weights[to.w] = w;
    }
    const uint32_t words[4] = {k.x, k.y, k.z, k.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      lo[j] = least(lo[j], in_order(words[j]));
      hi[j] = most(hi[j], in_order(words[j]));
    }
  }
  if (p.bounds == nullptr) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int d = 32; d >= kPieces; d >>= 1) {
      lo[j] = least(lo[j], __shfl_xor(lo[j], d, 64));
      hi[j] = most(hi[j], __shfl_xor(hi[j], d, 64));
    }
  if (lane < kPieces) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      red[tid >> 6][c][j] = lo[j];
      red[tid >> 6][c][4 + j] = hi[j];
    }
  }
  __syncthreads();
  const int page = p.table[b * p.t_sb + blockIdx.x];
  if (tid < kPieces && (uint32_t)page < (uint32_t)p.n_pages) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int w = 1; w < 4; ++w) {
        lo[j] = least(lo[j], red[w][c][j]);
        hi[j] = most(hi[j], red[w][c][4 + j]);
      }
      bounds_back<T>(lo[j], hi[j]);
    }
    uint16_t* to = p.bounds + ((int64_t)page * p.n_kv_heads + kvh) * 2 * D + 8 * c;
    *reinterpret_cast<uint4*>(to) = uint4{lo[0], lo[1], lo[2], lo[3]};
    *reinterpret_cast<uint4*>(to + D) = uint4{hi[0], hi[1], hi[2], hi[3]};
  }
}

template <typename T, int D>
static hipError_t launch_paged_evict_for(const PagedEvictArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(paged_keep_kernel, dim3(a.batch * a.n_kv_heads), dim3(kEvictThreads), 0, stream, a);
  if ((int64_t)a.max_pages << a.page_log > a.above) {  // (no sequence is longer than its table)
    const dim3 grid((a.n_keys + (1 << a.page_log) - 1) >> a.page_log, a.n_kv_heads, a.batch);
    hipLaunchKernelGGL((paged_save_kernel<D>), grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL((paged_move_kernel<T, D>), grid, dim3(256), 0, stream, a);
  }
  return hipGetLastError();
}

hipError_t launch_paged_evict(const PagedEvictArgs& a, hipStream_t stream) {
  if (a.head_dim == 128) return a.dtype == 0 ? launch_paged_evict_for<Bf16, 128>(a, stream) : launch_paged_evict_for<F16, 128>(a, stream);
  return a.dtype == 0 ? launch_paged_evict_for<Bf16, 64>(a, stream) : launch_paged_evict_for<F16, 64>(a, stream);
}

}  // namespace aa
