// Attention of one new token per sequence over a key/value cache in pages, on gfx950.
//
// Bound by reading keys and values once.  A work-group has one (sequence, query head) and takes 256 keys at a time: a thread's score each, then
// a channel of the output each.
#include "aa_kernels.h"
#include "aa_paged.h"

namespace aa {

template <typename T, int D>
__global__ void __launch_bounds__(256) paged_decode_kernel(const PagedDecodeArgs p) {
  constexpr int kParts = 256 / D;
  __shared__ float q[D], prob[256], red[2][4], part[kParts][D];
  const int tid = threadIdx.x, h = blockIdx.x, b = blockIdx.y;
  const int kvh = h / (p.n_q_heads / p.n_kv_heads);
  int length = clamped_length(p.lengths, b, p.max_pages, p.page_log);
  const int left_out = p.n_chosen ? max(0, pages_of(length, p.page_log) - p.n_chosen) : 0;
  length -= left_out << p.page_log;
  const int32_t* table = p.table + b * p.t_sb + kvh * p.t_sh;
  if (tid < D) q[tid] = T::from16(p.q[b * p.q_sb + h * p.q_sh + tid]);
  __syncthreads();
  const float scale = p.sm_scale * kLog2e;
  float m = -INFINITY, l = 0.f, acc = 0.f;
  const int d = tid % D, g = tid / D;
  for (int base = 0; base < length; base += 256) {
    const int key = base + tid;
    float s = -INFINITY;
    if (key < length) {
      const uint16_t* k = p.keys + clamped_page(table[key >> p.page_log], p.n_pages) * p.kp_sp + kvh * p.kp_sh + (key & ((1 << p.page_log) - 1)) * p.kp_sn;
      s = 0.f;
      for (int i = 0; i < D; i += 8) {
        float x[8];
        unpack8<T>(*reinterpret_cast<const uint4*>(k + i), x);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = __builtin_fmaf(q[i + j], x[j], s);
      }
    }
    float mx = s;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) mx = fmaxf(mx, __shfl_xor(mx, x, 64));
    if ((tid & 63) == 0) red[0][tid >> 6] = mx;
    __syncthreads();
    const float m_new = fmaxf(m, fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3])));
    const float m_base = m_new == -INFINITY ? 0.f : m_new;
    const float e = key < length ? fast_exp2((s - m_base) * scale) : 0.f;
    prob[tid] = e;
    float sum = e;
#pragma unroll
    for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
    if ((tid & 63) == 0) red[1][tid >> 6] = sum;
    __syncthreads();
    const float alpha = fast_exp2((m - m_base) * scale);
    l = l * alpha + ((red[1][0] + red[1][1]) + (red[1][2] + red[1][3]));
    acc *= alpha;
    m = m_new;
    for (int i = g; i < min(256, length - base); i += kParts) {
      const int k = base + i;
      const uint16_t* v = p.values + clamped_page(table[k >> p.page_log], p.n_pages) * p.vp_sp + kvh * p.vp_sh + (k & ((1 << p.page_log) - 1)) * p.vp_sn;
      acc = __builtin_fmaf(prob[i], T::from16(v[d]), acc);
    }
    __syncthreads();
  }
  part[g][d] = acc;
  __syncthreads();
  if (tid < D) {
    for (int i = 1; i < kParts; ++i) acc += part[i][d];
    p.out[b * p.o_sb + h * p.o_sh + d] = (uint16_t)T::pack(l == 0.f ? 0.f : acc / l, 0.f);
  }
}

hipError_t launch_paged_decode(const PagedDecodeArgs& a, hipStream_t stream) {
  const dim3 grid(a.n_q_heads, a.batch), block(256);
  if (a.head_dim == 128) {
    if (a.dtype == 0) hipLaunchKernelGGL((paged_decode_kernel<Bf16, 128>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((paged_decode_kernel<F16, 128>), grid, block, 0, stream, a);
  } else {
    if (a.dtype == 0) hipLaunchKernelGGL((paged_decode_kernel<Bf16, 64>), grid, block, 0, stream, a);
    else hipLaunchKernelGGL((paged_decode_kernel<F16, 64>), grid, block, 0, stream, a);
  }
  return hipGetLastError();
}

}  // namespace aa
