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
// Work. The G q-heads of a kv-head read the same keys, so their queries share
// tiles: query row r of a tile is (token r / G, head r % G). A row with
// n_b G <= 16 is one "small" tile; a longer one is cut into "big" tiles of two
// sub-tiles of TS = 128 / G tokens (128 query rows) each. Every (tile,
// kv-head) is one item over 128-key tiles of the cache; items with many key
// tiles are split along the keys into pieces when the step has too few items
// to fill the SMs (chunk_plan_kernel), each piece leaves (O, max, sum) in fp32
// and the last piece to finish joins them in the pieces' order, so the result
// does not depend on who was last.
//
// One persistent CTA per SM takes pieces from a counter, longest first, and
// serves both kinds through one TMA ring, so that a rebuilt row's window runs
// beside the other rows' single tokens:
//   warp 0       producer: the piece's descriptor, Q, and its K/V tiles, each
//                gathered from its pages in 64-row boxes
//   warp 1       issues tcgen05.mma for big tiles (S = Q K^T and O += P V with
//                S, P and O in tensor memory); for small ones it only passes
//                the ring stages back
//   warp 2       zeroes the V rows behind the row's last token before the tile
//                is handed on (a page's unused slots may hold anything; their
//                weights are 0, and 0 * NaN is not); warp 3 is idle
//   warps 4-11   big: softmax of sub-tile 0 and 1 (thread = query row);
//                small: warp w takes keys 16 w .. 16 w + 15 of every tile with
//                mma.sync, its own running max and sum
//   warps 12-15  epilogue: big tiles' O out of tensor memory, small tiles' join
//                over the eight warps, the output or the piece's partial, and
//                the join over pieces
// Bounds: single tokens are bound by HBM (a 16-row tile needs 64 KB of K/V per
// 128 keys), chunks by the softmax's exponentials and the tensor pipe.
//
// Every wait is bounded (common.cuh); the first one that runs out stops its
// CTA, and no output of an incomplete item is written.
#include "common.cuh"
#include "kernels.h"
#include "tcgen05.cuh"

#include <atomic>

namespace mb {

// ------------------------------------------------------------------ the plan
// An entry is one piece of one tile of one row, for every kv-head:
//   a = {row, first token in the stream, tokens, position of the first token}
//   b = {keys the row holds, first key tile, key tiles, first partial slot or -1}
//   c = {pieces, piece, small, -}
struct ChunkEntry {
  int4 a, b, c;
};

constexpr int kChunkKeys = 128;      // keys per tile
constexpr int kChunkSmallRows = 16;  // query rows of a small tile (one mma.sync row block)
constexpr int kChunkPlanThreads = 1024;
constexpr int kChunkBuckets = 2048;  // key-tile counts up to 2046 exactly, longer ones together
// Shortest piece: below it a piece's own cost (its queries, its partial, the
// join) outweighs what another SM gains.
constexpr int kMinSplitTiles = 4;

struct ChunkPlanParams {
  const int32_t* cu_q;
  const int32_t* kv_len;
  int batch, tokens, G, Hkv, tile_tokens, key_limit, sms, max_entries, max_slots;
  ChunkEntry* entries;
  int* head;      // [0] entries, [1] next item, [2] CTAs done
  int* counters;  // [max_slots * Hkv] pieces finished, by first slot and kv-head
};

// Key tiles that query tile t of a row (n new tokens, len cached) visits.
__device__ __forceinline__ int key_tiles(int n, int len, int t, int tile_tokens, int key_limit) {
  const int end = min(n, (t + 1) * tile_tokens);
  const int keys = min(len - n + end, key_limit);
  return max(1, (max(keys, 0) + kChunkKeys - 1) / kChunkKeys);
}

// The work list of a step. Splitting: with E entries before it, the longest
// tiles are cut into pieces of at most c key tiles, c the smallest that leaves
// at most one wave of CTAs beyond the waves the unsplit items need anyway (so
// the partials stay few), and never below kMinSplitTiles. Order: rows by the
// length of their pieces, longest first; a row's tiles stay together, its last
// (longest) first, so that they read the row's keys from L2.
__global__ void __launch_bounds__(kChunkPlanThreads) chunk_plan_kernel(const ChunkPlanParams p) {
  __shared__ int pre[kChunkPlanThreads + 1], n_s[kChunkPlanThreads], len_s[kChunkPlanThreads], base_s[kChunkPlanThreads];
  __shared__ int hist[kChunkBuckets];
  __shared__ int warp_tot[32];
  __shared__ unsigned long long sum_s, over_s;
  __shared__ int max_s, fits_s, slots_s;
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  auto bucket = [](int kt) { return min(kt, kChunkBuckets - 1); };

  // Exclusive block scan of one count per thread into pre[0 .. threads].
  auto scan = [&](int v) {
    int x = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_tot[w] = x;
    __syncthreads();
    if (w == 0) {
      int t = warp_tot[lane];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, t, d);
        if (lane >= d) t += y;
      }
      warp_tot[lane] = t;
    }
    __syncthreads();
    pre[tid + 1] = x + (w > 0 ? warp_tot[w - 1] : 0);
    if (tid == 0) pre[0] = 0;
    __syncthreads();
  };
  auto tiles_of = [&](int n) {
    return n <= 0 ? 0 : (long long)n * p.G <= kChunkSmallRows ? 1 : (n + p.tile_tokens - 1) / p.tile_tokens;
  };
  // Rows r0 .. r0 + threads - 1 into n_s, len_s and the tile prefix.
  int held = -1;
  auto load_rows = [&](int r0) {
    if (held == r0) return;
    held = r0;
    int n = 0, len = 0;
    if (r0 + tid < p.batch) {
      const int lo = min(max(p.cu_q[r0 + tid], 0), p.tokens);
      n = min(max(p.cu_q[r0 + tid + 1], lo), p.tokens) - lo;
      len = max(p.kv_len[r0 + tid], 0);
      if (n > 0 && len > p.key_limit) report(kDevBadPage);
    }
    __syncthreads();
    n_s[tid] = n;
    len_s[tid] = len;
    scan(tiles_of(n));
  };
  auto row_of = [&](int x) {
    int lo = 0, hi = kChunkPlanThreads - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (pre[mid] <= x)
        lo = mid;
      else
        hi = mid - 1;
    }
    return lo;
  };

  // 1. Histogram of the tiles' key-tile counts.
  for (int i = tid; i < kChunkBuckets; i += kChunkPlanThreads) hist[i] = 0;
  if (tid == 0) {
    sum_s = over_s = 0;
    max_s = slots_s = 0;
  }
  __syncthreads();
  long long E = 0;
  for (int r0 = 0; r0 < p.batch; r0 += kChunkPlanThreads) {
    load_rows(r0);
    const int tiles = pre[kChunkPlanThreads];
    E += tiles;
    unsigned long long sum = 0, over = 0;
    int most = 0;
    for (int x = tid; x < tiles; x += kChunkPlanThreads) {
      const int r = row_of(x);
      const int kt = key_tiles(n_s[r], len_s[r], x - pre[r], p.tile_tokens, p.key_limit);
      atomicAdd(&hist[bucket(kt)], 1);
      sum += kt;
      if (kt >= kChunkBuckets - 1) over += kt;
      most = max(most, kt);
    }
    if (sum) {
      atomicAdd(&sum_s, sum);
      if (over) atomicAdd(&over_s, over);
      atomicMax(&max_s, most);
    }
  }
  __syncthreads();
  const int most = max_s;
  // 2. The piece length c: 32 candidates a round, one per warp.
  const long long waves = (E * p.Hkv + p.sms - 1) / p.sms + 1;
  const long long room = waves * p.sms / p.Hkv;  // entries allowed after splitting
  int c = max(most, 1);
  if (room > E) {
    int lo = (int)min((unsigned long long)c, max((sum_s + room - 1) / (unsigned long long)room,
                                                 (unsigned long long)kMinSplitTiles));
    int hi = c;  // c = most splits nothing, which always fits
    while (lo < hi) {
      const int cand = lo + (int)((long long)(hi - lo) * w / 32);
      unsigned long long pieces = 0;
      for (int kt = lane; kt < kChunkBuckets - 1 && kt <= most; kt += 32)
        pieces += (unsigned long long)hist[kt] * ((kt + cand - 1) / cand);
#pragma unroll
      for (int d = 16; d > 0; d >>= 1) pieces += __shfl_xor_sync(0xffffffffu, pieces, d);
      pieces += over_s / cand + hist[kChunkBuckets - 1];
      if (tid == 0) fits_s = hi;
      __syncthreads();
      if (lane == 0) {
        if (pieces <= (unsigned long long)room)
          atomicMin(&fits_s, cand);
        warp_tot[w] = cand;
      }
      __syncthreads();
      // The smallest candidate that fits bounds c from above, the one before it from below.
      const int fit = fits_s;
      int below = lo - 1;
      for (int i = 0; i < 32; ++i)
        if (warp_tot[i] < fit) below = max(below, warp_tot[i]);
      __syncthreads();
      hi = fit;
      lo = below + 1;
    }
    c = hi;
  }
  // Pieces of a tile, and of all of a row's tiles from tile t on.
  auto pieces_of = [&](int kt) { return kt <= c ? 1 : (kt + c - 1) / c; };
  auto pieces_from = [&](int r, int t, int tiles) {
    if (key_tiles(n_s[r], len_s[r], tiles - 1, p.tile_tokens, p.key_limit) <= c) return tiles - t;
    int s = 0;
    for (; t < tiles; ++t) s += pieces_of(key_tiles(n_s[r], len_s[r], t, p.tile_tokens, p.key_limit));
    return s;
  };
  auto sort_key = [&](int r, int tiles) {
    const int kt = key_tiles(n_s[r], len_s[r], tiles - 1, p.tile_tokens, p.key_limit);
    const int s = pieces_of(kt);
    return bucket((kt + s - 1) / s);
  };
  // 3. Where each piece length starts in the order, longest first.
  for (int i = tid; i < kChunkBuckets; i += kChunkPlanThreads) hist[i] = 0;
  __syncthreads();
  for (int r0 = 0; r0 < p.batch; r0 += kChunkPlanThreads) {
    load_rows(r0);
    const int tiles = pre[tid + 1] - pre[tid];
    if (tiles > 0) atomicAdd(&hist[sort_key(tid, tiles)], pieces_from(tid, 0, tiles));
    __syncthreads();
  }
  {
    const int i0 = kChunkBuckets - 1 - 2 * tid, i1 = i0 - 1;
    const int h0 = hist[i0], h1 = hist[i1];
    int x = h0 + h1;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) warp_tot[w] = x;
    __syncthreads();
    int before = x - h0 - h1;
    for (int i = 0; i < w; ++i) before += warp_tot[i];
    hist[i0] = before;
    hist[i1] = before + h0;
    if (tid == kChunkPlanThreads - 1) fits_s = before + h0 + h1;
    __syncthreads();
  }
  const int total = fits_s;
  const bool fits = total <= p.max_entries;  // offsets that overlap can ask for more tiles than the stream holds
  if (!fits && tid == 0) report(kDevBadIndex);
  if (tid == 0) {
    p.head[0] = fits ? total : 0;
    p.head[1] = p.head[2] = 0;
  }
  for (int i = tid; i < p.max_slots * p.Hkv; i += kChunkPlanThreads) p.counters[i] = 0;
  if (!fits) return;
  // 4. The entries.
  for (int r0 = 0; r0 < p.batch; r0 += kChunkPlanThreads) {
    load_rows(r0);
    {
      const int tiles = pre[tid + 1] - pre[tid];
      if (tiles > 0) base_s[tid] = atomicAdd(&hist[sort_key(tid, tiles)], pieces_from(tid, 0, tiles));
    }
    __syncthreads();
    for (int x = tid; x < pre[kChunkPlanThreads]; x += kChunkPlanThreads) {
      const int r = row_of(x), t = x - pre[r], tiles = pre[r + 1] - pre[r];
      const int n = n_s[r], len = len_s[r];
      const bool small = (long long)n * p.G <= kChunkSmallRows;
      const int kt = key_tiles(n, len, t, p.tile_tokens, p.key_limit);
      const int pieces = pieces_of(kt);
      int slot = -1;
      if (pieces > 1) {
        slot = atomicAdd(&slots_s, pieces);
        if (slot + pieces > p.max_slots) report(kDevBadIndex);  // cannot happen: see chunk_layout
      }
      const int first = base_s[r] + pieces_from(r, t + 1, tiles);
      const int q0 = t * p.tile_tokens;
      const int cu = min(max(p.cu_q[r0 + r], 0), p.tokens);
      for (int i = 0; i < pieces; ++i) {
        const int k0 = (int)((long long)kt * i / pieces), k1 = (int)((long long)kt * (i + 1) / pieces);
        ChunkEntry e;
        e.a = make_int4(r0 + r, cu + q0, min(n - q0, small ? n : p.tile_tokens), len - n + q0);
        e.b = make_int4(min(len, p.key_limit), k0, k1 - k0, slot + pieces <= p.max_slots ? slot : -1);
        e.c = make_int4(pieces, i, small, 0);
        p.entries[first + i] = e;
      }
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------- the attention
constexpr int kChunkThreads = 512;
constexpr int kChunkLaunchRegs = 128;  // 65536 / 512
struct ChunkRegs {  // control, epilogue and softmax warpgroups
  static constexpr int ctrl = 56, epi = 80, softmax = 184;
  static_assert(128 * ctrl + 128 * epi + 256 * softmax <= kChunkThreads * kChunkLaunchRegs,
                "the register split must fit the launch allocation");
};

template <int HD>
struct ChunkTile {
  static constexpr int NCB = HD / 64;               // 64-element column blocks
  static constexpr int BOX = 128 * 128;             // bytes of a 64-element x 128-row block
  static constexpr int QTILE = NCB * BOX;           // one sub-tile's queries
  static constexpr int SQBOX = 16 * 128;            // a small tile's queries: 16 rows
  static constexpr int SQ = NCB * SQBOX;
  static constexpr int KVTILE = NCB * BOX;          // one K (or V) tile
  static constexpr int STAGES = HD == 128 ? 2 : 5;
  static constexpr int BARS = 5632;
  static constexpr int SMEM = 2 * QTILE + 2 * SQ + 2 * STAGES * KVTILE + BARS + 1024;
  static_assert(8 * kChunkSmallRows * HD * 4 <= 2 * QTILE, "the small tiles' join lies in the big tiles' Q");
  static_assert(SMEM <= 232448, "shared memory of a CTA");
};

constexpr int kChunkMaxStages = 5;
// A piece as its CTA's warps see it.
struct ChunkWork {
  int h;             // kv-head, or -1: no work left
  int q0, ntok, pos0;
  int len;           // keys the row holds
  int k0, n;         // key tiles of the piece
  int n0, n1;        // ... that sub-tile 0 and 1 visit (big)
  int slot, pieces, piece, small;
};

struct ChunkShared {
  uint64_t work_full[2], work_empty[2];   // descriptor ring (producer -> everyone)
  uint64_t q_full[2], q_empty[2];         // by piece parity; q_empty: Q and the join area are free again
  uint64_t k_full[kChunkMaxStages], v_full[kChunkMaxStages], kv_empty[kChunkMaxStages];
  uint64_t v_tail[kChunkMaxStages];       // a V tile with rows behind the last token has landed (by such tile)
  uint64_t small_done[kChunkMaxStages];   // a small tile's keys are consumed (by small tile)
  uint64_t s_full[2], p_full[2];          // per sub-tile
  uint64_t o_full, o_empty;
  uint64_t stats_full[2];                 // by piece parity: max and sum (big), join area written (small)
  uint64_t mma_drain;
  uint32_t tmem_base;
  int abort;                              // set by the first wait that runs out
  int flag;                               // epilogue: this CTA joins the pieces
  int q_armed;
  ChunkWork work[2];
  float stats[2][2][2][128];              // [piece parity][sub-tile][max, sum][row]; small: [.][0][.][warp * 16 + row]
};
static_assert(sizeof(ChunkShared) <= ChunkTile<128>::BARS, "barrier block outgrew its share");

// Score of a masked key (-2^90) on the tcgen05 path, where masks are applied by
// arithmetic; real scores stay far above it.
constexpr float kChunkMasked = -1.2379401e27f;

template <int HD>
__global__ void __launch_bounds__(kChunkThreads, 1)
    chunk_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap sqmap,
                           const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                           const ChunkParams p) {
  using C = ChunkTile<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qs = smem;                        // [2][QTILE]; small tiles: the join area
  uint8_t* ks = qs + 2 * C::QTILE;           // [STAGES][KVTILE]
  uint8_t* vs = ks + C::STAGES * C::KVTILE;  // [STAGES][KVTILE]
  uint8_t* sq = vs + C::STAGES * C::KVTILE;  // [2][SQ]
  ChunkShared* sh = reinterpret_cast<ChunkShared*>(sq + 2 * C::SQ);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sh->work_full[s], 1);
      mbar_init(&sh->work_empty[s], 14);  // every warp but the producer and warp 3
      mbar_init(&sh->q_full[s], 1);
      mbar_init(&sh->q_empty[s], 1);
      mbar_init(&sh->s_full[s], 1);
      mbar_init(&sh->p_full[s], 4);
      mbar_init(&sh->stats_full[s], 8);
    }
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&sh->k_full[s], 1);
      mbar_init(&sh->v_full[s], 1);
      mbar_init(&sh->kv_empty[s], 1);
      mbar_init(&sh->v_tail[s], 1);
      mbar_init(&sh->small_done[s], 8);
    }
    mbar_init(&sh->o_full, 1);
    mbar_init(&sh->o_empty, 4);
    mbar_init(&sh->mma_drain, 1);
    sh->abort = 0;
    sh->q_armed = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&sh->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = sh->tmem_base;
  const int n_items = p.head[0] * p.Hkv;

  // Warp-uniform bounded wait; one that runs out stops every warp of the CTA.
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    return (bool)__all_sync(0xffffffffu, mbar_wait_abortable(bar, parity, code, &sh->abort));
  };
  // Piece k of this CTA from the descriptor ring; false at the end of the work.
  auto take = [&](int k, ChunkWork& wk) {
    if (!wait(&sh->work_full[k & 1], (k >> 1) & 1, kDevTimeoutFull)) return false;
    wk = sh->work[k & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh->work_empty[k & 1]);
    return wk.h >= 0;
  };
  // Whether key tile t of a row holding len keys has V rows to be zeroed, i.e.
  // the last 64-row box that holds a key is not full (a box without keys is
  // loaded as zeros). Such a tile's V lands on v_tail; warp 2 completes v_full.
  auto ragged = [](int t, int len) { return len % 64 != 0 && t == len / kChunkKeys; };

  if (warp < 4) {
    regs_dec<ChunkRegs::ctrl>();
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      if (lane == 0) {
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&sqmap);
        prefetch_tensormap(&kmap);
        prefetch_tensormap(&vmap);
      }
      // The next piece is taken and its entry read while this one's keys stream.
      int next = 0;
      ChunkEntry e{};
      auto fetch = [&](int k) {
        if (lane == 0) next = k == 0 ? (int)blockIdx.x : (int)gridDim.x + atomicAdd(&p.head[1], 1);
        next = __shfl_sync(0xffffffffu, next, 0);
        if (next < n_items) e = p.entries[next / p.Hkv];
      };
      fetch(0);
      bool ok = true;
      int J = 0, jc = 0;         // K/V tiles issued, those with V rows to be zeroed
      uint32_t tails = 0;        // bit i: the tile issued i tiles ago was one of them
      for (int k = 0;; ++k) {
        ok = wait(&sh->work_empty[k & 1], ((k >> 1) & 1) ^ 1, kDevTimeoutEmpty);
        if (!ok) break;
        if (next >= n_items) {
          if (lane == 0) {
            sh->work[k & 1].h = -1;
            mbar_arrive(&sh->work_full[k & 1]);
          }
          break;
        }
        ChunkWork wk;
        wk.h = next % p.Hkv;
        const int row = e.a.x;
        wk.q0 = e.a.y;
        wk.ntok = e.a.z;
        wk.pos0 = e.a.w;
        wk.len = e.b.x;
        wk.k0 = e.b.y;
        wk.n = e.b.z;
        wk.slot = e.b.w;
        wk.pieces = e.c.x;
        wk.piece = e.c.y;
        wk.small = e.c.z;
        if (wk.ntok > p.sub_tokens && !wk.small) {
          const int keys0 = min(wk.pos0 + p.sub_tokens, p.key_limit);
          const int end0 = max(1, (max(keys0, 0) + kChunkKeys - 1) / kChunkKeys);
          wk.n0 = min(max(end0 - wk.k0, 0), wk.n);
          wk.n1 = wk.n;
        } else {
          wk.n0 = wk.n;
          wk.n1 = 0;
        }
        if (lane == 0) {
          sh->work[k & 1] = wk;
          mbar_arrive(&sh->work_full[k & 1]);
        }
        // Q: the small buffer of this parity is free once piece k - 2 is done,
        // the big one (the small pieces' join area) once piece k - 1 is.
        if (k >= 2) ok = wait(&sh->q_empty[k & 1], ((k >> 1) & 1) ^ 1, kDevTimeoutEmpty);
        if (ok && !wk.small && k >= 1) ok = wait(&sh->q_empty[(k - 1) & 1], ((k - 1) >> 1) & 1, kDevTimeoutEmpty);
        if (!ok) break;
        if (lane == 0) {
          if (wk.small) {
            mbar_arrive_expect_tx(&sh->q_full[k & 1], C::NCB * p.small_rows * 128);
            for (int cb = 0; cb < C::NCB; ++cb)
              tma_load_3d(sq + (k & 1) * C::SQ + cb * C::SQBOX, &sqmap, &sh->q_full[k & 1], cb * 64, wk.h * p.G, wk.q0);
          } else {
            const int subs = wk.n1 > 0 ? 2 : 1;
            mbar_arrive_expect_tx(&sh->q_full[k & 1], subs * C::NCB * p.sub_tokens * p.G * 128);
            for (int s = 0; s < subs; ++s)
              for (int cb = 0; cb < C::NCB; ++cb)
                tma_load_3d(qs + s * C::QTILE + cb * C::BOX, &qmap, &sh->q_full[k & 1], cb * 64, wk.h * p.G,
                            wk.q0 + s * p.sub_tokens);
          }
          *reinterpret_cast<volatile int*>(&sh->q_armed) = k + 1;
        }
        fetch(k + 1);
        // K/V tiles. Page ids of the next 32 boxes at a time, one per lane.
        const int32_t* table = p.block_table + (size_t)row * p.max_pages;
        int y_lane = 0;
        int j = 0;
        for (; j < wk.n; ++j) {
          if (j % 16 == 0) {
            const long long tok = ((long long)wk.k0 + j) * kChunkKeys + lane * 64;
            y_lane = -64;  // wholly out of bounds: reads zeros
            if (tok < wk.len && tok < ((long long)wk.k0 + wk.n) * kChunkKeys) {
              const int col = (int)tok / p.page_size;
              const int pg = col < p.max_pages ? table[col] : -1;
              if (pg >= 0 && pg < p.num_pages)
                y_lane = (pg * p.Hkv + wk.h) * p.page_size + (int)tok % p.page_size;
              else
                report(kDevBadPage);
            }
          }
          const int y0 = __shfl_sync(0xffffffffu, y_lane, 2 * (j % 16));
          const int y1 = __shfl_sync(0xffffffffu, y_lane, 2 * (j % 16) + 1);
          const int st = (J + j) % C::STAGES;
          if (!(ok = wait(&sh->kv_empty[st], (((J + j) / C::STAGES) & 1) ^ 1, kDevTimeoutEmpty))) break;
          const bool tail = ragged(wk.k0 + j, wk.len);
          if (lane == 0) {
            mbar_arrive_expect_tx(&sh->k_full[st], C::KVTILE);
#pragma unroll
            for (int cb = 0; cb < C::NCB; ++cb) {
              uint8_t* dst = ks + st * C::KVTILE + cb * C::BOX;
              tma_load_2d(dst, &kmap, &sh->k_full[st], cb * 64, y0);
              tma_load_2d(dst + C::BOX / 2, &kmap, &sh->k_full[st], cb * 64, y1);
            }
            uint64_t* v_bar = tail ? &sh->v_tail[jc % C::STAGES] : &sh->v_full[st];
            mbar_arrive_expect_tx(v_bar, C::KVTILE);
#pragma unroll
            for (int cb = 0; cb < C::NCB; ++cb) {
              uint8_t* dst = vs + st * C::KVTILE + cb * C::BOX;
              tma_load_2d(dst, &vmap, v_bar, cb * 64, y0);
              tma_load_2d(dst + C::BOX / 2, &vmap, v_bar, cb * 64, y1);
            }
          }
          jc += tail;
          tails = tails << 1 | (uint32_t)tail;
          __syncwarp();
        }
        J += j;
        if (!ok) break;
      }
      if (lane == 0) {
        // Every load issued lands before the CTA exits, also when a wait ran out.
        drain_ring(sh->q_full, 2, *reinterpret_cast<volatile int*>(&sh->q_armed));
        drain_ring(sh->k_full, C::STAGES, J);
        drain_ring(sh->v_tail, C::STAGES, jc);
        for (int i = max(J - C::STAGES, 0); i < J; ++i)
          if (!(tails >> (J - 1 - i) & 1)) mbar_drain(&sh->v_full[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1);
        // The last CTA resets the counters: the plan serves the next layer too.
        __threadfence();
        if (atomicAdd(&p.head[2], 1) == (int)gridDim.x - 1) p.head[1] = p.head[2] = 0;
      }
    } else if (warp == 1) {
      // --------------------------------------------------------- MMA issue
      constexpr uint32_t ID_QK = umma_idesc_bf16(128, 128, 0, 0);
      constexpr uint32_t ID_PV = umma_idesc_bf16(128, HD, 0, 1);
      auto issue_qk = [&](int s, int st) {
        const uint64_t dq = umma_desc_sw128(smem_u32(qs + s * C::QTILE), 16, 1024);
        const uint64_t dk = umma_desc_sw128(smem_u32(ks + st * C::KVTILE), 16, 1024);
        if constexpr (HD == 128)
          umma_ss_k128_warp(tbase + 128 * s, dq, dk, ID_QK);
        else
          umma_ss_k64_warp(tbase + 128 * s, dq, dk, ID_QK);
        umma_commit_warp(&sh->s_full[s]);
      };
      bool ok = true;
      ChunkWork wk;
      // Running counts: K/V tiles, small tiles, each sub-tile's S tiles, big pieces.
      int J = 0, js = 0, jb[2] = {0, 0}, big = 0;
      for (int k = 0; ok && take(k, wk); ++k) {
        if (wk.small) {
          for (int j = 0; ok && j < wk.n; ++j, ++js) {
            ok = wait(&sh->small_done[js % C::STAGES], (js / C::STAGES) & 1, kDevTimeoutFull);
            if (ok && lane == 0) mbar_arrive(&sh->kv_empty[(J + j) % C::STAGES]);
          }
          J += wk.n;
          continue;
        }
        const int n_sub[2] = {wk.n0, wk.n1};
        if (!(ok = wait(&sh->q_full[k & 1], (k >> 1) & 1, kDevTimeoutFull))) break;
        if (!(ok = wait(&sh->k_full[J % C::STAGES], (J / C::STAGES) & 1, kDevTimeoutFull))) break;
        tc_fence_after();
        for (int s = 0; s < 2; ++s)
          if (n_sub[s] > 0) issue_qk(s, J % C::STAGES);
        if (wk.n == 1) umma_commit_warp(&sh->q_empty[k & 1]);  // the piece's last Q K^T
        for (int j = 0; ok && j < wk.n; ++j) {
          const int jj = J + j, st = jj % C::STAGES, st1 = (jj + 1) % C::STAGES;
          if (!(ok = wait(&sh->v_full[st], (jj / C::STAGES) & 1, kDevTimeoutFull))) break;
          bool k_next = false;
          const uint64_t dv = umma_desc_sw128(smem_u32(vs + st * C::KVTILE), C::BOX, 1024);
          for (int s = 0; s < 2; ++s) {
            if (j >= n_sub[s]) continue;
            if (!(ok = wait(&sh->p_full[s], (jb[s] + j) & 1, kDevTimeoutFull))) break;
            // The piece's first P V overwrites O: the previous epilogue must hold it.
            if (j == 0 && big > 0 && !(ok = wait(&sh->o_empty, (big - 1) & 1, kDevTimeoutFull))) break;
            tc_fence_after();
            umma_ts_t128_linear_warp(tbase + 256 + HD * s, tbase + 128 * s, dv, ID_PV, j > 0 ? 1u : 0u);
            if (j + 1 < n_sub[s]) {
              if (!k_next && !(ok = wait(&sh->k_full[st1], ((jj + 1) / C::STAGES) & 1, kDevTimeoutFull))) break;
              k_next = true;
              issue_qk(s, st1);
            }
          }
          if (!ok) break;
          if (j + 2 == wk.n) umma_commit_warp(&sh->q_empty[k & 1]);
          umma_commit_warp(&sh->kv_empty[st]);
        }
        if (!ok) break;
        umma_commit_warp(&sh->o_full);
        J += wk.n;
        jb[0] += wk.n0;
        jb[1] += wk.n1;
        ++big;
      }
      umma_drain_warp(&sh->mma_drain);  // before TMEM is freed, also when a wait ran out
    } else if (warp == 2) {
      // ------------------------------------- zeroing behind the last token
      ChunkWork wk;
      int J = 0, jc = 0;
      for (int k = 0; take(k, wk); ++k) {
        const int j = wk.len / kChunkKeys - wk.k0;
        if (j >= 0 && j < wk.n && ragged(wk.k0 + j, wk.len)) {
          const int st = (J + j) % C::STAGES;
          if (!wait(&sh->v_tail[jc % C::STAGES], (jc / C::STAGES) & 1, kDevTimeoutFull)) break;
          const int r0 = wk.len % kChunkKeys, rows = 64 - r0 % 64;
          uint8_t* v = vs + st * C::KVTILE;
          for (int i = lane; i < rows * C::NCB * 8; i += 32) {
            const int r = r0 + i / (C::NCB * 8), cb = i / 8 % C::NCB;
            *reinterpret_cast<uint4*>(v + cb * C::BOX + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();  // read by tcgen05.mma, overwritten by the next load
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->v_full[st]);
          ++jc;
        }
        J += wk.n;
      }
    }
  } else if (warp < 12) {
    regs_inc<ChunkRegs::softmax>();
    const int hh = (warp - 4) >> 2;  // big: sub-tile
    const int sub = warp & 3;        // TMEM lane quarter this warp may access
    const int r = sub * 32 + lane;   // query row of the sub-tile
    const int r_tok = r / p.G + hh * p.sub_tokens;
    const bool r_in = r < p.sub_tokens * p.G;
    const uint32_t lane_bits = (uint32_t)(sub * 32) << 16;
    const uint32_t t_s = tbase + 128 * hh + lane_bits;
    const uint32_t t_o = tbase + 256 + HD * hh + lane_bits;
    const int sw = warp - 4;  // small: its 16 keys of a tile
    const int gid = lane >> 2, tig = lane & 3;
    ChunkWork wk;
    int J = 0, js = 0, jb = 0;
    bool ok = true;
    for (int k = 0; ok && take(k, wk); ++k) {
      if (wk.small) {
        // ------------------------------------------------ small: mma.sync
        int kv_end[2];
        const int R = wk.ntok * p.G;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int rr = gid + 8 * half;
          kv_end[half] = rr < R ? min(wk.pos0 + rr / p.G + 1, wk.len) : 0;
        }
        if (!(ok = wait(&sh->q_full[k & 1], (k >> 1) & 1, kDevTimeoutFull))) break;
        uint32_t qa[HD / 16][4];
        {
          const uint32_t qb = smem_u32(sq + (k & 1) * C::SQ);
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            const int ch = 2 * kk + (lane >> 4);
            ldmatrix_x4(qa[kk][0], qa[kk][1], qa[kk][2], qa[kk][3],
                        qb + (ch >> 3) * C::SQBOX + swz128(lane & 15, ch & 7));
          }
        }
        float o[HD / 8][4];
#pragma unroll
        for (int d = 0; d < HD / 8; ++d) o[d][0] = o[d][1] = o[d][2] = o[d][3] = 0.f;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
        for (int j = 0; j < wk.n; ++j, ++js) {
          const int jj = J + j, st = jj % C::STAGES;
          const int tok0 = (wk.k0 + j) * kChunkKeys + sw * 16;
          if (!(ok = wait(&sh->k_full[st], (jj / C::STAGES) & 1, kDevTimeoutFull))) break;
          float s[2][4];
          const uint32_t kb = smem_u32(ks + st * C::KVTILE);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            s[t][0] = s[t][1] = s[t][2] = s[t][3] = 0.f;
            const uint32_t rr = sw * 16 + t * 8 + (lane & 7);
#pragma unroll
            for (int kp = 0; kp < HD / 32; ++kp) {
              uint32_t b0, b1, b2, b3;
              const int ch = kp * 4 + (lane >> 3);
              ldmatrix_x4(b0, b1, b2, b3, kb + (ch >> 3) * C::BOX + swz128(rr, ch & 7));
              mma_bf16_16816(s[t], qa[2 * kp], b0, b1);
              mma_bf16_16816(s[t], qa[2 * kp + 1], b2, b3);
            }
          }
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int half = x >> 1;
              s[t][x] = tok0 + t * 8 + tig * 2 + (x & 1) < kv_end[half] ? s[t][x] * p.scale_log2 : -INFINITY;
              mx[half] = fmaxf(mx[half], s[t][x]);
            }
          float alpha[2];
          bool moved = false;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 1));
            mx[half] = fmaxf(mx[half], __shfl_xor_sync(0xffffffffu, mx[half], 2));
            const float m_new = fmaxf(m[half], mx[half]);
            moved |= m_new > m[half];
            alpha[half] = m_new == -INFINITY ? 1.f : exp2f(m[half] - m_new);
            m[half] = m_new;
            const float m_use = m_new == -INFINITY ? 0.f : m_new;
            l[half] *= alpha[half];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              s[t][2 * half] = fast_exp2(s[t][2 * half] - m_use);
              s[t][2 * half + 1] = fast_exp2(s[t][2 * half + 1] - m_use);
              l[half] += s[t][2 * half] + s[t][2 * half + 1];
            }
          }
          if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int d = 0; d < HD / 8; ++d) {
              o[d][0] *= alpha[0];
              o[d][1] *= alpha[0];
              o[d][2] *= alpha[1];
              o[d][3] *= alpha[1];
            }
          }
          if (!(ok = wait(&sh->v_full[st], (jj / C::STAGES) & 1, kDevTimeoutFull))) break;
          const uint32_t pa[4] = {pack_bf16x2(s[0][0], s[0][1]), pack_bf16x2(s[0][2], s[0][3]),
                                  pack_bf16x2(s[1][0], s[1][1]), pack_bf16x2(s[1][2], s[1][3])};
          const uint32_t vb = smem_u32(vs + st * C::KVTILE);
          const uint32_t rr = sw * 16 + ((lane >> 3) & 1) * 8 + (lane & 7);
#pragma unroll
          for (int d = 0; d < HD / 8; d += 2) {
            uint32_t b0, b1, b2, b3;
            const int ch = d + (lane >> 4);
            ldmatrix_x4_trans(b0, b1, b2, b3, vb + (ch >> 3) * C::BOX + swz128(rr, ch & 7));
            mma_bf16_16816(o[d], pa, b0, b1);
            mma_bf16_16816(o[d + 1], pa, b2, b3);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->small_done[js % C::STAGES]);
        }
        if (!ok) break;
        J += wk.n;
        // Into the join area once piece k - 1 has left it.
        if (k >= 1 && !(ok = wait(&sh->q_empty[(k - 1) & 1], ((k - 1) >> 1) & 1, kDevTimeoutEmpty))) break;
        float* join = reinterpret_cast<float*>(qs) + (size_t)sw * kChunkSmallRows * HD;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          l[half] += __shfl_xor_sync(0xffffffffu, l[half], 1);
          l[half] += __shfl_xor_sync(0xffffffffu, l[half], 2);
          const int rr = gid + 8 * half;
          if (rr < R) {
            if (tig == 0) {
              sh->stats[k & 1][0][0][sw * 16 + rr] = m[half];
              sh->stats[k & 1][0][1][sw * 16 + rr] = l[half];
            }
            // Columns permuted by the row, in steps of 8, against bank conflicts.
#pragma unroll
            for (int d = 0; d < HD / 8; ++d)
              *reinterpret_cast<float2*>(&join[rr * HD + ((d ^ (rr & 7)) * 8 + tig * 2)]) =
                  make_float2(o[d][2 * half], o[d][2 * half + 1]);
          }
        }
        fence_proxy_async();  // the next big tile's Q lands here
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->stats_full[k & 1]);
        continue;
      }
      // --------------------------------------------------- big: softmax
      const int n = hh == 0 ? wk.n0 : wk.n1;
      const bool row_ok = r_in && r_tok < wk.ntok;
      const int hi = row_ok ? min(wk.pos0 + r_tok, wk.len - 1) : -1;  // last visible key
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j) {
        const int kv0 = (wk.k0 + j) * kChunkKeys;
        if (!(ok = wait(&sh->s_full[hh], (jb + j) & 1, kDevTimeoutFull))) break;
        tc_fence_after();
        uint32_t v[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(v + 32 * c));
        tmem_wait_ld();
        if (!(row_ok && kv0 + kChunkKeys - 1 <= hi)) {
          // Keys behind the last visible one go to kChunkMasked by arithmetic:
          // the minimum with a line that is huge up to it and hugely negative
          // past it (this also drops a NaN score), then the maximum with
          // kChunkMasked.
          const float big = 1.2676506e30f;  // 2^100
          const float hb = (hi >= kv0 ? (float)min(hi - kv0, kChunkKeys - 1) + 0.5f : -1000.f) * big;
#pragma unroll
          for (int e = 0; e < 128; ++e)
            v[e] = __float_as_uint(fmaxf(fminf(__uint_as_float(v[e]), fmaf(-(float)e, big, hb)), kChunkMasked));
        }
        // Row max and sum as independent chains.
        float mp[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) mp[q] = fmaxf(__uint_as_float(v[q]), __uint_as_float(v[8 + q]));
#pragma unroll
        for (int e = 16; e < 128; e += 16)
#pragma unroll
          for (int q = 0; q < 8; ++q) mp[q] = fmax3(mp[q], __uint_as_float(v[e + q]), __uint_as_float(v[e + 8 + q]));
        float mx = fmax3(fmax3(mp[0], mp[1], mp[2]), fmax3(mp[3], mp[4], mp[5]), fmaxf(mp[6], mp[7]));
        if (mx <= kChunkMasked) mx = -INFINITY;  // no key of this tile is visible to the row
        const float m_new = fmaxf(m_used, mx * p.scale_log2);
        // O is rescaled only when the maximum grew by more than 2^8; the final
        // division uses the same stale maximum, so the result is exact.
        float alpha = 1.f;
        const bool rescale = m_new > m_used + 8.f;
        if (rescale) {
          alpha = exp2f(m_used - m_new);
          m_used = m_new;
        }
        const float neg_mu = m_used == -INFINITY ? 0.f : -m_used;
        float ls[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) ls[q] = 0.f;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int e = 0; e < 32; e += 2) {
            float x0, x1;
            ffma2(x0, x1, __uint_as_float(v[32 * c + e]), __uint_as_float(v[32 * c + e + 1]), p.scale_log2,
                  p.scale_log2, neg_mu, neg_mu);
            const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
            const int q = 2 * ((e >> 1) & 3);
            fadd2(ls[q], ls[q + 1], ls[q], ls[q + 1], p0, p1);
            pk[e >> 1] = pack_bf16x2(p0, p1);
          }
          tmem_st16(t_s + 16 * c, pk);
        }
        l = l * alpha + (((ls[0] + ls[1]) + (ls[2] + ls[3])) + ((ls[4] + ls[5]) + (ls[6] + ls[7])));
        if (__any_sync(0xffffffffu, rescale && j > 0)) {
          const float a = (rescale && j > 0) ? alpha : 1.f;
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o + 32 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * a);
            tmem_st32(t_o + 32 * c, o);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->p_full[hh]);
      }
      if (!ok) break;
      sh->stats[k & 1][hh][0][r] = m_used;
      sh->stats[k & 1][hh][1][r] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->stats_full[k & 1]);
      jb += n;
      J += wk.n;
    }
  } else {
    regs_dec<ChunkRegs::epi>();
    // ------------------------------------------------------------ epilogue
    const int tid = threadIdx.x - 384;
    const int sub = warp & 3;
    const int r = sub * 32 + lane;
    const uint32_t lane_bits = (uint32_t)(sub * 32) << 16;
    auto sleepy = [&](uint64_t* bar, uint32_t parity) {
      return (bool)__all_sync(0xffffffffu, mbar_wait_sleepy_abortable(bar, parity, kDevTimeoutFull, &sh->abort));
    };
    ChunkWork wk;
    int big = 0;
    for (int k = 0;; ++k) {
      // The four warps leave together: they share named barriers below.
      wk.h = 0;
      bool ok = sleepy(&sh->work_full[k & 1], (k >> 1) & 1);
      if (ok) {
        const bool more = take(k, wk);
        ok = more || wk.h < 0;
      }
      if (named_barrier_or(1, 128, !ok) || wk.h < 0) break;
      ok = sleepy(&sh->stats_full[k & 1], (k >> 1) & 1) && (wk.small || sleepy(&sh->o_full, big & 1));
      if (named_barrier_or(1, 128, !ok)) break;
      const bool split = wk.pieces > 1;
      const int rows = wk.ntok * p.G;
      const size_t part = ((size_t)(wk.slot + wk.piece) * p.Hkv + wk.h) * p.part_rows;
      if (wk.small) {
        const float* join = reinterpret_cast<const float*>(qs);
        const float(*st)[128] = sh->stats[k & 1][0];
        for (int i = tid; i < rows * (HD / 4); i += 128) {
          const int rr = i / (HD / 4), c4 = i % (HD / 4);
          float M = -INFINITY;
#pragma unroll
          for (int w = 0; w < 8; ++w) M = fmaxf(M, st[0][w * 16 + rr]);
          const float Mu = M == -INFINITY ? 0.f : M;
          float L = 0.f;
          float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
          const int at = rr * HD + (((c4 >> 1) ^ (rr & 7)) * 8 + (c4 & 1) * 4);
#pragma unroll
          for (int w = 0; w < 8; ++w) {
            const float f = exp2f(st[0][w * 16 + rr] - Mu);
            const float4 x = *reinterpret_cast<const float4*>(&join[w * kChunkSmallRows * HD + at]);
            L += st[1][w * 16 + rr] * f;
            O.x += x.x * f;
            O.y += x.y * f;
            O.z += x.z * f;
            O.w += x.w * f;
          }
          if (split) {
            *reinterpret_cast<float4*>(&p.part_o[(part + rr) * HD + c4 * 4]) = O;
            if (c4 == 0) p.part_ml[part + rr] = make_float2(M, L);
          } else {
            const float inv = L > 0.f ? 1.f / L : 0.f;
            const int tok = wk.q0 + rr / p.G, h = wk.h * p.G + rr % p.G;
            uint2 u;
            u.x = pack_bf16x2(O.x * inv, O.y * inv);
            u.y = pack_bf16x2(O.z * inv, O.w * inv);
            *reinterpret_cast<uint2*>(p.out + ((size_t)tok * p.Hq + h) * HD + c4 * 4) = u;
          }
        }
        fence_proxy_async();  // the next big tile's Q lands here
        named_barrier(1, 128);
        if (tid == 0) mbar_arrive(&sh->q_empty[k & 1]);
      } else {
        tc_fence_after();
        for (int hh = 0; hh < 2; ++hh) {
          const int r_tok = r / p.G + hh * p.sub_tokens;
          const bool row_ok = r < p.sub_tokens * p.G && r_tok < wk.ntok;
          if (hh * p.sub_tokens >= wk.ntok) break;
          const float m_used = sh->stats[k & 1][hh][0][r];
          const float l = sh->stats[k & 1][hh][1][r];
          const float inv = l > 0.f ? 1.f / l : 0.f;
          const uint32_t t_o = tbase + 256 + HD * hh + lane_bits;
          const int tok = wk.q0 + r_tok, h = wk.h * p.G + r % p.G;
          uint4* dst = reinterpret_cast<uint4*>(p.out + ((size_t)tok * p.Hq + h) * HD);
          const size_t pr = part + hh * p.sub_tokens * p.G + r;
          float4* pdst = reinterpret_cast<float4*>(p.part_o + pr * HD);
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            tmem_ld32(t_o + 32 * c, o);
            tmem_wait_ld();
            if (!row_ok) {
            } else if (split) {
#pragma unroll
              for (int q = 0; q < 8; ++q) {
                float4 f;
                f.x = l > 0.f ? __uint_as_float(o[4 * q + 0]) : 0.f;
                f.y = l > 0.f ? __uint_as_float(o[4 * q + 1]) : 0.f;
                f.z = l > 0.f ? __uint_as_float(o[4 * q + 2]) : 0.f;
                f.w = l > 0.f ? __uint_as_float(o[4 * q + 3]) : 0.f;
                pdst[8 * c + q] = f;
              }
            } else {
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint4 u;
                u.x = pack_bf16x2(__uint_as_float(o[8 * q + 0]) * inv, __uint_as_float(o[8 * q + 1]) * inv);
                u.y = pack_bf16x2(__uint_as_float(o[8 * q + 2]) * inv, __uint_as_float(o[8 * q + 3]) * inv);
                u.z = pack_bf16x2(__uint_as_float(o[8 * q + 4]) * inv, __uint_as_float(o[8 * q + 5]) * inv);
                u.w = pack_bf16x2(__uint_as_float(o[8 * q + 6]) * inv, __uint_as_float(o[8 * q + 7]) * inv);
                dst[4 * c + q] = l > 0.f ? u : make_uint4(0, 0, 0, 0);
              }
            }
          }
          if (split && row_ok) p.part_ml[pr] = make_float2(m_used, l);
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->o_empty);
        ++big;
      }
      if (!split) continue;
      // Release this piece's partial and take a ticket; the last piece joins
      // them all, in their order.
      __threadfence();
      named_barrier(1, 128);
      if (tid == 0) sh->flag = atomicAdd(&p.counters[wk.slot * p.Hkv + wk.h], 1) == wk.pieces - 1;
      named_barrier(1, 128);
      if (!sh->flag) continue;
      __threadfence();
      const size_t first = ((size_t)wk.slot * p.Hkv + wk.h) * p.part_rows, step = (size_t)p.Hkv * p.part_rows;
      for (int i = tid; i < rows * (HD / 4); i += 128) {
        const int rr = i / (HD / 4), c4 = i % (HD / 4);
        float M = -INFINITY;
        for (int c = 0; c < wk.pieces; ++c) M = fmaxf(M, __ldcg(&p.part_ml[first + c * step + rr]).x);
        const float Mu = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int c = 0; c < wk.pieces; ++c) {
          const float2 ml = __ldcg(&p.part_ml[first + c * step + rr]);
          const float4 x = __ldcg(reinterpret_cast<const float4*>(&p.part_o[(first + c * step + rr) * HD + c4 * 4]));
          const float f = exp2f(ml.x - Mu);
          L += ml.y * f;
          O.x += x.x * f;
          O.y += x.y * f;
          O.z += x.z * f;
          O.w += x.w * f;
        }
        const float inv = L > 0.f ? 1.f / L : 0.f;
        const int tok = wk.q0 + rr / p.G, h = wk.h * p.G + rr % p.G;
        uint2 u;
        u.x = pack_bf16x2(O.x * inv, O.y * inv);
        u.y = pack_bf16x2(O.z * inv, O.w * inv);
        *reinterpret_cast<uint2*>(p.out + ((size_t)tok * p.Hq + h) * HD + c4 * 4) = u;
      }
      if (tid == 0) p.counters[wk.slot * p.Hkv + wk.h] = 0;  // ready for the next layer
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tbase, 512);
  }
}

// ------------------------------------------------------------------ host side
int chunk_sub_tokens(int G) { return 128 / G; }

// Workspace. Entries: a row's tiles are at most its tokens / tile_tokens
// rounded up, and splitting adds at most `extra` (the plan's room: one wave
// of CTAs, plus what the last wave leaves, over the kv-heads). A split tile
// has at least two pieces, so at most twice `extra` entries are pieces.
size_t chunk_layout(int batch, int tokens, int Hq, int Hkv, int head_dim, int sms, ChunkLayout* lay) {
  const int G = Hq / Hkv, tile_tokens = 2 * chunk_sub_tokens(G);
  const size_t extra = (size_t)(2 * sms) / Hkv + 1;
  auto up = [](size_t x) { return (x + 255) & ~size_t(255); };
  lay->max_entries = (size_t)std::min(batch, tokens) + (size_t)tokens / tile_tokens + extra;
  lay->max_slots = 2 * extra;
  lay->part_rows = (int)std::min<long long>((long long)tokens * G, tile_tokens * G);
  size_t off = 0;
  lay->head = off;     off = up(off + 4 * sizeof(int));
  lay->entries = off;  off = up(off + lay->max_entries * sizeof(ChunkEntry));
  lay->counters = off; off = up(off + lay->max_slots * Hkv * sizeof(int));
  lay->part_ml = off;  off = up(off + lay->max_slots * Hkv * lay->part_rows * sizeof(float2));
  lay->part_o = off;   off = up(off + lay->max_slots * Hkv * lay->part_rows * head_dim * sizeof(float));
  lay->total = off;
  return off;
}

cudaError_t launch_chunk_plan(const ChunkParams& p, const ChunkLayout& lay, uint8_t* ws, int sms,
                              cudaStream_t stream) {
  ChunkPlanParams q{};
  q.cu_q = p.cu_q;
  q.kv_len = p.kv_len;
  q.batch = p.batch;
  q.tokens = p.tokens;
  q.G = p.G;
  q.Hkv = p.Hkv;
  q.tile_tokens = 2 * p.sub_tokens;
  q.key_limit = p.key_limit;
  q.sms = sms;
  q.max_entries = (int)lay.max_entries;
  q.max_slots = (int)lay.max_slots;
  q.entries = reinterpret_cast<ChunkEntry*>(ws + lay.entries);
  q.head = reinterpret_cast<int*>(ws + lay.head);
  q.counters = reinterpret_cast<int*>(ws + lay.counters);
  chunk_plan_kernel<<<1, kChunkPlanThreads, 0, stream>>>(q);
  return cudaGetLastError();
}

// One-time set-up of an instantiation on the current device: its shared
// memory, and a check that it is launched with the registers that the
// setmaxnreg split draws on (an increase beyond them would never complete).
template <int HD>
static cudaError_t chunk_prepare() {
  static std::atomic<int> ready[kMaxDevices];
  const int dev = device_slot();
  if (dev >= 0 && ready[dev].load(std::memory_order_acquire)) return cudaSuccess;
  cudaFuncAttributes a{};
  cudaError_t e = cudaFuncGetAttributes(&a, chunk_attention_kernel<HD>);
  if (e != cudaSuccess) return e;
  if (a.numRegs < kChunkLaunchRegs) return cudaErrorInvalidConfiguration;
  e = cudaFuncSetAttribute(chunk_attention_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           ChunkTile<HD>::SMEM);
  if (e == cudaSuccess && dev >= 0) ready[dev].store(1, std::memory_order_release);
  return e;
}

template <int HD>
static cudaError_t launch_chunk(const CUtensorMap& qm, const CUtensorMap& sqm, const CUtensorMap& km,
                                const CUtensorMap& vm, const ChunkParams& p, unsigned grid, cudaStream_t stream) {
  cudaError_t e = chunk_prepare<HD>();
  if (e != cudaSuccess) return e;
  chunk_attention_kernel<HD><<<grid, kChunkThreads, ChunkTile<HD>::SMEM, stream>>>(qm, sqm, km, vm, p);
  return cudaGetLastError();
}

cudaError_t launch_chunk_attention(const CUtensorMap& qm, const CUtensorMap& sqm, const CUtensorMap& km,
                                   const CUtensorMap& vm, ChunkParams p, const ChunkLayout& lay, uint8_t* ws, int sms,
                                   cudaStream_t stream) {
  p.entries = reinterpret_cast<const ChunkEntry*>(ws + lay.entries);
  p.head = reinterpret_cast<int*>(ws + lay.head);
  p.counters = reinterpret_cast<int*>(ws + lay.counters);
  p.part_ml = reinterpret_cast<float2*>(ws + lay.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + lay.part_o);
  p.part_rows = lay.part_rows;
  const unsigned grid = (unsigned)std::min<size_t>((size_t)sms, lay.max_entries * p.Hkv);
  return p.head_dim == 128 ? launch_chunk<128>(qm, sqm, km, vm, p, grid, stream)
                           : launch_chunk<64>(qm, sqm, km, vm, p, grid, stream);
}

}  // namespace mb
