// K15: attention of ragged chunks of new tokens over the paged K/V cache.
//
// Replaces the FlexAttention call of FlexDecodeSession.forward
// (src/mouse_core/models/backbone/flex_decode.py:226-229) for a step whose
// rows append different numbers of tokens: the queries are a packed stream
// [T, Hq, HD], row b's n_b = cu_q[b + 1] - cu_q[b] tokens being the last n_b of
// its kv_len[b] cached ones. Token i of the row sits at position
//   p = kv_len[b] - n_b + i   and   out = sum_{j <= p} softmax_j(scale q . k_j) v_j
// over the row's cached slots; a token with p < 0 sees nothing and gets 0.
//
// One warp per (token, q-head) walks the keys with an online softmax: every
// lane holds HD / 32 elements of q and of the output.
#include "common.cuh"
#include "kernels.h"

namespace mb {

// Row of token t: the last b with cu_q[b] <= t, or -1 behind the last row.
__device__ __forceinline__ int chunk_row(const int32_t* cu_q, int batch, int t) {
  if (batch <= 0 || t >= cu_q[batch] || t < cu_q[0]) return -1;
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu_q[mid] <= t)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

template <int HD>
__global__ void __launch_bounds__(128) chunk_attention_kernel(const ChunkParams p) {
  constexpr int E = HD / 32;
  const int lane = threadIdx.x & 31;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (item >= (long long)p.tokens * p.Hq) return;
  const int t = (int)(item / p.Hq), h = (int)(item % p.Hq), kvh = h / p.G;
  const int b = chunk_row(p.cu_q, p.batch, t);
  if (b < 0) return;
  const int len = p.kv_len[b];
  const int see = min(len - (p.cu_q[b + 1] - t), len - 1) + 1;  // keys 0 .. see - 1
  float q[E], o[E], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    q[e] = __bfloat162float(p.q[(size_t)t * p.q_stride + (size_t)h * HD + lane * E + e]) * p.scale_log2;
    o[e] = 0.f;
  }
  for (int j = 0; j < see; ++j) {
    const int col = j / p.page_size;
    const int page = col < p.max_pages ? p.block_table[(size_t)b * p.max_pages + col] : -1;
    float k[E], v[E];
    if (page >= 0 && page < p.num_pages) {
      const size_t at = (((size_t)page * p.Hkv + kvh) * p.page_size + j % p.page_size) * HD + lane * E;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        k[e] = __bfloat162float(p.k_pool[at + e]);
        v[e] = __bfloat162float(p.v_pool[at + e]);
      }
    } else {
      report(kDevBadPage);
#pragma unroll
      for (int e = 0; e < E; ++e) k[e] = v[e] = 0.f;
    }
    float s = 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) s += q[e] * k[e];
    s = warp_sum(s);
    const float m_new = fmaxf(m, s);
    const float a = exp2f(m - m_new), w = exp2f(s - m_new);
    m = m_new;
    l = l * a + w;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = o[e] * a + w * v[e];
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    p.out[((size_t)t * p.Hq + h) * HD + lane * E + e] = __float2bfloat16_rn(l > 0.f ? o[e] / l : 0.f);
}

cudaError_t launch_chunk_attention(const ChunkParams& p, cudaStream_t stream) {
  const long long items = (long long)p.tokens * p.Hq;
  const unsigned grid = (unsigned)((items + 3) / 4);
  if (p.head_dim == 128)
    chunk_attention_kernel<128><<<grid, 128, 0, stream>>>(p);
  else
    chunk_attention_kernel<64><<<grid, 128, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace mb
