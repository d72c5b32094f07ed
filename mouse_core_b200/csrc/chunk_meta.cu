// K14: block table, positions and slot map of a ragged step, on the device.
//
// Replaces the position and slot bookkeeping of FlexDecodeSession.forward
// (src/mouse_core/models/backbone/flex_decode.py:180-196) for a step in which
// row b appends n_b tokens (any number, zero included), the new tokens of all
// rows lying one after the other in a packed stream. With c_b the row's cached
// length, P the page size and f the ids of free pages in the order they are
// handed out:
//   cu_q[b + 1]     = n_0 + ... + n_b
//   cu_pages[b + 1] = o_0 + ... + o_b,  o_b = ceil((c_b + n_b) / P) - ceil(c_b / P)
//   table[b, ceil(c_b / P) + j] = f[cu_pages[b] + j]            j < o_b
//   token cu_q[b] + i: position c_b + i, slot = table[b, (c_b + i) / P] * P + (c_b + i) % P
//   new_len[b]      = c_b + n_b
//
// Bound: launch latency below some hundred thousand tokens (8 bytes written per
// token, 20 per row). Every block walks the rows in groups of one per thread
// and scans (tokens, pages) itself, so one launch without a grid barrier does
// the whole step; the tokens and opened pages of a group are spread over the
// blocks, each token finding its row by bisection in shared memory.
#include "common.cuh"
#include "kernels.h"

namespace mb {

constexpr int kChunkMetaThreads = 1024;

// Pages that hold n tokens.
__device__ __forceinline__ int pages_of(int n, int page_size) { return n / page_size + (n % page_size > 0); }

// Sum of two counts in [0, INT_MAX], capped there (associative, so a scan in
// any order gives the same prefix): an absurd count cannot wrap an index.
__device__ __forceinline__ int add_capped(int a, int b) {
  return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu);
}

__global__ void __launch_bounds__(kChunkMetaThreads) chunk_meta_kernel(const ChunkMetaParams p) {
  __shared__ int cu[kChunkMetaThreads + 1], cup[kChunkMetaThreads + 1], old_len[kChunkMetaThreads];
  __shared__ int warp_n[32], warp_o[32];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int first = blockIdx.x * kChunkMetaThreads + tid, stride = gridDim.x * kChunkMetaThreads;
  const int P = p.page_size;
  int base_n = 0, base_o = 0;  // tokens and pages of the groups before this one
  for (int r0 = 0, group = 0; r0 < p.batch; r0 += kChunkMetaThreads, ++group) {
    const int rows = min(kChunkMetaThreads, p.batch - r0);
    int n = 0, c = 0, o = 0;
    if (tid < rows) {
      n = max(p.lengths[r0 + tid], 0);
      c = max(p.kv_len[r0 + tid], 0);
      o = pages_of(add_capped(c, n), P) - pages_of(c, P);
    }
    int sn = n, so = o;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int an = __shfl_up_sync(0xffffffffu, sn, d), ao = __shfl_up_sync(0xffffffffu, so, d);
      if (lane >= d) {
        sn = add_capped(sn, an);
        so = add_capped(so, ao);
      }
    }
    if (lane == 31) {
      warp_n[w] = sn;
      warp_o[w] = so;
    }
    __syncthreads();  // (also: every thread has left the previous group's arrays)
    if (w == 0) {
      int tn = warp_n[lane], to = warp_o[lane];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int an = __shfl_up_sync(0xffffffffu, tn, d), ao = __shfl_up_sync(0xffffffffu, to, d);
        if (lane >= d) {
          tn = add_capped(tn, an);
          to = add_capped(to, ao);
        }
      }
      warp_n[lane] = tn;
      warp_o[lane] = to;
    }
    __syncthreads();
    sn = add_capped(base_n, add_capped(sn, w > 0 ? warp_n[w - 1] : 0));
    so = add_capped(base_o, add_capped(so, w > 0 ? warp_o[w - 1] : 0));
    cu[tid + 1] = sn;
    cup[tid + 1] = so;
    old_len[tid] = c;
    if (tid == 0) {
      cu[0] = base_n;
      cup[0] = base_o;
    }
    if (group % gridDim.x == blockIdx.x && tid < rows) {
      p.cu_q[r0 + tid + 1] = sn;
      p.cu_pages[r0 + tid + 1] = so;
      p.new_len[r0 + tid] = add_capped(c, n);
      if (r0 + tid == 0) {
        p.cu_q[0] = 0;
        p.cu_pages[0] = 0;
      }
      // More tokens or pages than the caller gave room for: what fits is done.
      if (sn > p.tokens) report(kDevBadIndex);
      if (so > p.n_free || (o > 0 && pages_of(c, P) + o > p.max_pages)) report(kDevBadPage);
    }
    __syncthreads();
    // Row of the group that element x lies in: the last one whose prefix is <= x.
    auto row_of = [&](const int* prefix, int x) {
      int lo = 0, hi = rows - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= x)
          lo = mid;
        else
          hi = mid - 1;
      }
      return lo;
    };
    const int end_n = min(cu[rows], p.tokens), end_o = min(cup[rows], p.n_free);
    base_n = cu[rows];
    base_o = cup[rows];
    for (long long x = (long long)cup[0] + first; x < end_o; x += stride) {
      const int r = row_of(cup, (int)x);
      const long long col = pages_of(old_len[r], P) + (x - cup[r]);
      if (col < p.max_pages) p.block_table[(size_t)(r0 + r) * p.max_pages + col] = p.free_pages[x];
    }
    for (long long x = (long long)cu[0] + first; x < end_n; x += stride) {
      const int r = row_of(cu, (int)x);
      const int pos = add_capped(old_len[r], (int)x - cu[r]);
      const int col = pos / P, held = pages_of(old_len[r], P);
      int id = -1;
      if (col < p.max_pages) {
        // A page opened by this step is taken from the free list again: another
        // block may not have written its table entry yet.
        if (col < held)
          id = p.block_table[(size_t)(r0 + r) * p.max_pages + col];
        else if ((long long)cup[r] + (col - held) < p.n_free)
          id = p.free_pages[cup[r] + (col - held)];
      }
      const long long slot = (long long)id * P + pos % P;
      p.q_pos[x] = pos;
      p.slot[x] = id >= 0 && slot <= 0x7fffffffll ? (int)slot : -1;
    }
    __syncthreads();  // the arrays are overwritten by the next group
  }
  // Room behind the last row's tokens: position 0, not cached.
  for (long long x = (long long)base_n + first; x < p.tokens; x += stride) {
    p.q_pos[x] = 0;
    p.slot[x] = -1;
  }
  if (p.batch == 0 && blockIdx.x == 0 && tid == 0) p.cu_q[0] = p.cu_pages[0] = 0;
}

cudaError_t launch_chunk_meta(const ChunkMetaParams& p, cudaStream_t stream) {
  // One block until the tokens outgrow it (its scan is the latency), then up
  // to two per SM.
  const long long most = ((long long)std::max(p.tokens, p.n_free) + kChunkMetaThreads - 1) / kChunkMetaThreads;
  const int grid = (int)std::max(1ll, std::min(most, 296ll));
  chunk_meta_kernel<<<grid, kChunkMetaThreads, 0, stream>>>(p);
  return cudaGetLastError();
}

}  // namespace mb
