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
// token, 20 per row). Every block walks the rows in groups of four per
// thread and scans (tokens, pages) itself, so one launch without a grid barrier does
// the whole step; the tokens and opened pages of a group are spread over the
// blocks, each token finding its row by bisection in shared memory.
// Measured, replayed from a graph: 256 rows of one token 5.4 us, with six windows
// of 1024 tokens among them 6.0, 4096 rows of 0 to 4 tokens 9.4, 64 rows of 1024
// to 8192 tokens 7.9; called from Python 11.9 us each, of which the launch is 4
// and two thirds the host's.
#include "common.cuh"
#include "kernels.h"

namespace mb {

constexpr int kChunkMetaThreads = 1024, kChunkMetaRows = 4 * kChunkMetaThreads;  // a thread scans four rows

// Pages that hold n tokens.
__device__ __forceinline__ int pages_of(int n, int page_size) { return n / page_size + (n % page_size > 0); }

// Sum of two counts in [0, INT_MAX], capped there (associative, so a scan in
// any order gives the same prefix): an absurd count cannot wrap an index.
__device__ __forceinline__ int add_capped(int a, int b) {
  return (int)min((unsigned)a + (unsigned)b, 0x7fffffffu);
}

__global__ void __launch_bounds__(kChunkMetaThreads) chunk_meta_kernel(const ChunkMetaParams p) {
  __shared__ int cu[kChunkMetaRows + 1], cup[kChunkMetaRows + 1];
  __shared__ int warp_n[32], warp_o[32];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int first = blockIdx.x * kChunkMetaThreads + tid, stride = gridDim.x * kChunkMetaThreads;
  const int P = p.page_size;
  int base_n = 0, base_o = 0;  // tokens and pages of the groups before this one
  for (int r0 = 0, group = 0; r0 < p.batch; r0 += kChunkMetaRows, ++group) {
    const int rows = min(kChunkMetaRows, p.batch - r0);
    int n[4], c[4], o[4], sn = 0, so = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * tid + i;
      n[i] = r < rows ? max(p.lengths[r0 + r], 0) : 0;
      c[i] = r < rows ? max(p.kv_len[r0 + r], 0) : 0;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[i] = n[i] > 0 ? pages_of(add_capped(c[i], n[i]), P) - pages_of(c[i], P) : 0;
      sn = add_capped(sn, n[i]);
      so = add_capped(so, o[i]);
    }
    // Block scan of the threads' sums: within the warp, then every warp over
    // the warps' totals.
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
    __syncthreads();
    int tn = warp_n[lane], to = warp_o[lane];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int an = __shfl_up_sync(0xffffffffu, tn, d), ao = __shfl_up_sync(0xffffffffu, to, d);
      if (lane >= d) {
        tn = add_capped(tn, an);
        to = add_capped(to, ao);
      }
    }
    // Before this thread's rows: the groups, the warps and the lanes before it.
    const int pn = __shfl_sync(0xffffffffu, tn, max(w - 1, 0)), po = __shfl_sync(0xffffffffu, to, max(w - 1, 0));
    const int ln = __shfl_up_sync(0xffffffffu, sn, 1), lo = __shfl_up_sync(0xffffffffu, so, 1);
    int en = add_capped(base_n, add_capped(w > 0 ? pn : 0, lane > 0 ? ln : 0));
    int eo = add_capped(base_o, add_capped(w > 0 ? po : 0, lane > 0 ? lo : 0));
    if (tid == 0) {
      cu[0] = base_n;
      cup[0] = base_o;
    }
    const bool mine = group % gridDim.x == blockIdx.x;  // this block writes the group's rows
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * tid + i;
      en = add_capped(en, n[i]);
      eo = add_capped(eo, o[i]);
      cu[r + 1] = en;
      cup[r + 1] = eo;
      if (mine && r < rows) {
        p.cu_q[r0 + r + 1] = en;
        p.cu_pages[r0 + r + 1] = eo;
        p.new_len[r0 + r] = add_capped(c[i], n[i]);
        // More tokens or pages than the caller gave room for: what fits is done.
        if (en > p.tokens) report(kDevBadIndex);
        if (eo > p.n_free || (n[i] > 0 && pages_of(add_capped(c[i], n[i]), P) > p.max_pages)) report(kDevBadPage);
      }
    }
    if (mine && r0 == 0 && tid == 0) p.cu_q[0] = p.cu_pages[0] = 0;
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
      const long long col = pages_of(max(p.kv_len[r0 + r], 0), P) + (x - cup[r]);
      if (col < p.max_pages) p.block_table[(size_t)(r0 + r) * p.max_pages + col] = p.free_pages[x];
    }
    for (long long x = (long long)cu[0] + first; x < end_n; x += stride) {
      const int r = row_of(cu, (int)x);
      const int old = max(p.kv_len[r0 + r], 0), pos = add_capped(old, (int)x - cu[r]);
      const int col = pos / P, held = pages_of(old, P);
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
      const bool held_by_page = id >= 0 && slot <= 0x7fffffffll;
      if (!held_by_page) report(kDevBadPage);
      p.q_pos[x] = pos;
      p.slot[x] = held_by_page ? (int)slot : -1;
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
