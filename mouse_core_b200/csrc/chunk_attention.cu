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
// sub-tiles of TS = 128 / G tokens (128 query rows) each. (A big tile with one
// sub-tile's tokens takes its even key tiles as the one and its odd ones as the
// other, "dual", and the epilogue joins the two: 3 rows of up to 20 query rows over
// 131000 keys take 141 us, and 154 without.) Every (tile,
// kv-head) is one item over 128-key tiles of the cache; items with many key
// tiles are split along the keys into pieces when the step has too few items
// to fill the SMs (chunk_plan_kernel): each piece leaves (O, max, sum) in fp32,
// and chunk_join_kernel joins them in the pieces' order, so the result does not
// depend on the schedule. (Joined by the last piece's CTA instead, a 256-row
// tile in 7 pieces kept one CTA 170 us longer than the rest.)
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
//                over the eight warps; the output or the piece's partial
// Bounds: single tokens are bound by HBM (a 16-row tile needs 64 KB of K/V per
// 128 keys); chunks by the chain of a sub-tile, S -> softmax -> P -> O -> next S:
// at head_dim 128 it takes 3700 cycles for a pair of sub-tiles whose products
// alone are 2100, at 64 (S issued ahead, but exponentials for half the products)
// 3650, and a piece costs 3000 more to start and to end.
// Measured, with the plan (16/8 heads of 128 in 128-token pages, or 32/8 of 64 in
// 64-token pages; 6.55 TB/s copied and 1677 TFLOP/s multiplied by the library):
//   256 single tokens over 64..4096 keys           366 us, 6.0 TB/s
//   128 rows of 0..4 tokens over 128..16380 (64)   124 us, 5.6 TB/s
//   48 rows, four of them windows of 1024           72 us
//   48 x 256 tokens over 1024..8192 keys           543 us, 878 TFLOP/s
//   64 windows of 500..1024 from empty (64)        402 us, 394 TFLOP/s
//   700 tokens over 60001 keys                     428 us, 810 TFLOP/s
//   3 rows of 1..5 tokens over 90000..131000 (64)  144 us, 4.7 TB/s
//
// Precision: scores, statistics, sums, O and the partials are fp32. The weights
// are rounded to bf16 for P V, whose V is bf16 (a wider P would need the tf32
// pipe at half the rate and V converted), and the output once: against 64 bits
// the outputs are off by 0.0020 to 0.0023 (relative, in the mean square), by
// 0.0016 to 0.0017 with the output's rounding alone.
//
// Every wait is bounded (common.cuh); the first one that runs out stops its
// CTA. A query row's output (or partial) is written only when the row is done,
// so every element of out is then the result or as it was; that of another row
// of the same item may be either. Split tiles are not joined.
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
// Up to eight query rows of a split tile, for the join: the tile's first
// partial slot, its pieces, its first token, the first of the rows, and the
// tile's rows.
struct alignas(16) ChunkSplit {
  int slot, pieces, q0;
  short row0, rows;
};
constexpr int kJoinRows = 8;

constexpr int kChunkKeys = 128;      // keys per tile
constexpr int kChunkSmallRows = 16;  // query rows of a small tile (one mma.sync row block)
constexpr int kChunkPlanThreads = 1024;
// Shortest piece: below it a piece's own cost (its queries, its partial, the
// join) outweighs what another SM gains. (Long steps take the same at half and
// twice this; a short one is spared the join's launch, 4 us.)
// (In kChunkTileCost's units: four tiles of the cheapest kind.)
constexpr int kMinPieceCost = 16;
// ... and little is gained by pieces shorter than an SM's share of the step, or
// half of it when there are few items: longest first evens those out. (A step
// of 800 items took 119 us cut at the share and 131 at half of it; 8 items over
// 131072 keys 199 and 151.)
constexpr int kManyItems = 4;  // items per SM

// What a key tile costs, in quarters of a small piece's, which is bound by its
// K/V (hd 64: 32 KB in 1440 cycles, hd 128: 64 KB in 2700). One sub-tile alone
// takes 1825 cycles, a pair 3650. (All alike, 48 rows with four windows among
// them take 88 us instead of 72; pairs at 8 and 6 quarters and single sub-tiles
// like small pieces 74, and 3 long rows of hd 64 147 instead of 142.)
enum ChunkKind { kSmallTile, kOneSub, kTwoSubs };
constexpr int kChunkTileCost[2][3] = {{4, 6, 10}, {4, 5, 7}};  // head_dim 64, 128

struct ChunkPlanParams {
  const int32_t* cu_q;
  const int32_t* kv_len;
  int batch, tokens, G, Hkv, tile_tokens, key_limit, sms, max_entries, max_slots, plan_key, cost[3];
  ChunkEntry* entries;
  ChunkSplit* splits;
  // [0] entries, [1] next item, [2] CTAs done, [3] splits, [4] whether a wait ran out, [5] the sizes' key, [6] join
  // blocks that saw [4]
  int* head;
};

// Key tiles that query tile t of a row (n new tokens, len cached ones) visits.
__device__ __forceinline__ int chunk_key_tiles(int n, int len, int t, bool small, int tile_tokens, int key_limit) {
  const int end = small ? n : min(n, (t + 1) * tile_tokens);
  return max(1, (max(min(len - n + end, key_limit), 0) + kChunkKeys - 1) / kChunkKeys);
}

// The work list of a step, in one block with a row per thread (5 us for 256
// rows, most of it the launch and the reads). Splitting: with
// E entries before it, the longest tiles are cut into pieces that cost at most
// c, c the smallest that leaves at most one wave of CTAs beyond the waves
// the unsplit items need anyway (so the partials stay few), and not below the
// two bounds above. Order: rows by the length of their longest piece, longest
// first; a row's tiles stay together, its last (longest) first, so that they
// read the row's keys from L2.
__global__ void __launch_bounds__(kChunkPlanThreads) chunk_plan_kernel(const ChunkPlanParams p) {
  constexpr int kBuckets = kChunkPlanThreads;  // piece lengths, the longest together
  __shared__ int hist[kBuckets], warp_tot[32], warp_max[32];
  __shared__ int base_s[kChunkPlanThreads], n_s[kChunkPlanThreads], len_s[kChunkPlanThreads];
  __shared__ int cu_s[kChunkPlanThreads], pre[kChunkPlanThreads + 1];
  __shared__ unsigned long long warp_sum[32];
  __shared__ unsigned fit_s[3];
  __shared__ int slots_s, splits_s;
  launch_dependents();  // the attention's CTAs set themselves up meanwhile
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5, nw = blockDim.x >> 5;
  const unsigned all = 0xffffffffu;

  // Row r0 + tid: its tokens, keys and tiles.
  int r0 = -1, n = 0, len = 0, tiles = 0, cu = 0;
  bool small = false;
  int cost = 0;  // of a key tile
  auto load = [&](int at) {
    if (at == r0) return;
    r0 = at;
    n = len = tiles = 0;
    if (r0 + tid < p.batch) {
      cu = min(max(p.cu_q[r0 + tid], 0), p.tokens);
      const int end = max(p.cu_q[r0 + tid + 1], cu);
      n = min(end, p.tokens) - cu;
      // Tokens behind the stream's end are left out, and with them the row's
      // last keys, which only they see (none may be left: len <= 0).
      len = max(p.kv_len[r0 + tid], 0) - (end - cu - n);
      small = n <= kChunkSmallRows / p.G;
      tiles = n <= 0 ? 0 : small ? 1 : (n + p.tile_tokens - 1) / p.tile_tokens;
      cost = p.cost[small ? kSmallTile : n > p.tile_tokens / 2 ? kTwoSubs : kOneSub];
    }
  };
  auto key_tiles = [&](int t) { return chunk_key_tiles(n, len, t, small, p.tile_tokens, p.key_limit); };
  auto warp_add = [&](unsigned long long v) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(all, v, d);
    return v;
  };

  // 1. Entries, their cost and the most of one, over all rows.
  if (tid < 3) fit_s[tid] = 0;
  if (tid == 0) slots_s = splits_s = 0;
  hist[tid] = 0;
  for (int i = tid + blockDim.x; i < kBuckets; i += blockDim.x) hist[i] = 0;
  unsigned long long count = 0, sum = 0;
  int most = 0;
  for (int at = 0; at < p.batch; at += blockDim.x) {
    load(at);
    if (n > 0 && len > p.key_limit) report(kDevBadPage);
    if (r0 + tid < p.batch && p.cu_q[r0 + tid + 1] > p.tokens) report(kDevBadIndex);
    count += tiles;
    if (count > p.max_entries) continue;  // too many already (below): bounds this loop, too
    for (int t = 0; t < tiles; ++t) sum += key_tiles(t) * cost;
    if (tiles > 0) most = max(most, key_tiles(tiles - 1) * cost);
  }
  count = warp_add(count);
  sum = warp_add(sum);
  most = __reduce_max_sync(all, most);
  if (lane == 0) {
    warp_tot[w] = (int)min(count, 0x7fffffffull);
    warp_sum[w] = sum;
    warp_max[w] = most;
  }
  __syncthreads();
  const long long E = (long long)warp_add(lane < nw ? (unsigned long long)warp_tot[lane] : 0);
  // Offsets that overlap can ask for more tiles than the stream holds. Such a
  // step has no plan; below, no 32-bit count of tiles or pieces can wrap.
  auto no_plan = [&]() {
    if (tid == 0) {
      report(kDevBadIndex);
      p.head[0] = p.head[1] = p.head[2] = p.head[3] = p.head[4] = p.head[6] = 0;
      p.head[5] = p.plan_key;
    }
  };
  if (E > p.max_entries) return no_plan();
  sum = warp_add(lane < nw ? warp_sum[lane] : 0);
  most = __reduce_max_sync(all, lane < nw ? warp_max[lane] : 0);
  // 2. The piece length c, by bisection.
  const long long waves = (E * p.Hkv + p.sms - 1) / p.sms + 1;
  const long long room = waves * p.sms / p.Hkv;  // entries allowed after splitting
  int hi = max(most, 1);                           // splits nothing, which always fits
  int lo = hi;
  if (room > E) {
    const unsigned long long share = sum * p.Hkv / (p.sms * (E * p.Hkv >= kManyItems * p.sms ? 1 : 2));
    lo = (int)min((unsigned long long)hi, max(max((sum + room - 1) / (unsigned long long)room, share),
                                              (unsigned long long)kMinPieceCost));
    // c >= sum / (room - E) always fits: pieces are at most sum / c + E.
    hi = (int)max((unsigned long long)lo, min((unsigned long long)hi, sum / (unsigned long long)(room - E) + 1));
  }
  for (int round = 0; lo < hi; ++round) {
    const int c = (lo + hi) >> 1;
    unsigned pieces = 0;
    for (int at = 0; at < p.batch; at += blockDim.x) {
      load(at);
      for (int t = 0; t < tiles; ++t) pieces += (unsigned)(key_tiles(t) * cost + c - 1) / c;
    }
    pieces = __reduce_add_sync(all, min(pieces, 1u << 21));  // (no sum wraps; so many never fit)
    if (lane == 0 && pieces) atomicAdd(&fit_s[round % 3], pieces);
    if (tid == 0) fit_s[(round + 1) % 3] = 0;  // (read by nobody now: two rounds old)
    __syncthreads();
    if ((long long)fit_s[round % 3] <= room)
      hi = c;
    else
      lo = c + 1;
  }
  const int c = hi;
  auto pieces_of = [&](int of) { return of <= c ? 1 : (of + c - 1) / c; };  // of a tile, by its cost
  auto row_pieces = [&]() {
    if (tiles == 0 || key_tiles(tiles - 1) * cost <= c) return tiles;
    int s = 0;
    for (int t = 0; t < tiles; ++t) s += pieces_of(key_tiles(t) * cost);
    return s;
  };
  // Of the row's longest piece (a row with a split tile counts as c: it has
  // pieces near it); 0 comes first.
  auto bucket = [&]() { return kBuckets - 1 - min(min(key_tiles(tiles - 1) * cost, c) / 4, kBuckets - 1); };
  // 3. Where each piece length starts in the order.
  __syncthreads();
  for (int at = 0; at < p.batch; at += blockDim.x) {
    load(at);
    if (tiles > 0) atomicAdd(&hist[bucket()], row_pieces());
  }
  __syncthreads();
  int total = 0;
  for (int at = 0; at < kBuckets; at += blockDim.x) {
    const int h = hist[at + tid];
    int x = h;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(all, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) warp_tot[w] = x;
    __syncthreads();
    int tot = lane < nw ? warp_tot[lane] : 0;
    const int before = __reduce_add_sync(all, lane < w ? tot : 0);
    hist[at + tid] = total + before + x - h;
    total += __reduce_add_sync(all, tot);
    __syncthreads();
  }
  if (total > p.max_entries) return no_plan();
  if (tid == 0) {
    p.head[0] = total;
    p.head[1] = p.head[2] = p.head[4] = p.head[6] = 0;
    p.head[5] = p.plan_key;
  }
  // 4. The entries: the group's tiles side by side, each finding its row by
  // bisection.
  for (int at = 0; at < p.batch; at += blockDim.x) {
    load(at);
    base_s[tid] = tiles > 0 ? atomicAdd(&hist[bucket()], row_pieces()) : 0;
    n_s[tid] = n;
    len_s[tid] = len;
    cu_s[tid] = cu;
    int x = tiles;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(all, x, d);
      if (lane >= d) x += y;
    }
    if (lane == 31) warp_tot[w] = x;
    __syncthreads();
    const int tot = lane < nw ? warp_tot[lane] : 0;
    pre[tid + 1] = x + __reduce_add_sync(all, lane < w ? tot : 0);
    if (tid == 0) pre[0] = 0;
    __syncthreads();
    const int row0 = r0;
    for (int e = tid; e < pre[blockDim.x]; e += blockDim.x) {
      int r = 0, hi_r = blockDim.x - 1;
      while (r < hi_r) {
        const int mid = (r + hi_r + 1) >> 1;
        if (pre[mid] <= e)
          r = mid;
        else
          hi_r = mid - 1;
      }
      const int t = e - pre[r], last = pre[r + 1] - pre[r] - 1;
      const int n_ = n_s[r], len_ = len_s[r];
      const bool small_ = n_ <= kChunkSmallRows / p.G;
      const int kt = chunk_key_tiles(n_, len_, t, small_, p.tile_tokens, p.key_limit);
      const int cost_ = p.cost[small_ ? kSmallTile : n_ > p.tile_tokens / 2 ? kTwoSubs : kOneSub];
      const int pieces = pieces_of(kt * cost_);
      // Behind the row's longer tiles t + 1 .. last.
      int first = base_s[r] + last - t;
      if (chunk_key_tiles(n_, len_, last, small_, p.tile_tokens, p.key_limit) * cost_ > c)
        for (int u = t + 1; u <= last; ++u)
          first += pieces_of(chunk_key_tiles(n_, len_, u, small_, p.tile_tokens, p.key_limit) * cost_) - 1;
      int slot = -1;
      if (pieces > 1) {
        slot = atomicAdd(&slots_s, pieces);
        if (slot + pieces > p.max_slots) {  // cannot happen: see chunk_layout
          report(kDevBadIndex);
          slot = -1;
        }
      }
      const int q0 = t * p.tile_tokens, ntok = small_ ? n_ : min(n_ - q0, p.tile_tokens);
      if (slot >= 0) {
        const int rows = ntok * p.G;
        int at_split = atomicAdd(&splits_s, (rows + kJoinRows - 1) / kJoinRows);
        for (int row = 0; row < rows; row += kJoinRows)
          p.splits[at_split++] = ChunkSplit{slot, pieces, cu_s[r] + q0, (short)row, (short)rows};
      }
      for (int i = 0, k0 = 0; i < pieces; ++i) {
        const int k = (kt - k0) / (pieces - i);  // even pieces
        ChunkEntry out;
        out.a = make_int4(row0 + r, cu_s[r] + q0, ntok, len_ - n_ + q0);
        out.b = make_int4(min(max(len_, 0), p.key_limit), k0, k, slot);
        out.c = make_int4(pieces, i, small_, 0);
        p.entries[first + i] = out;
        k0 += k;
      }
    }
    __syncthreads();
  }
  if (tid == 0) p.head[3] = splits_s;
}

// ------------------------------------------------------------- the attention
constexpr int kChunkThreads = 512;

template <int HD>
struct ChunkTile {
  static constexpr int NCB = HD / 64;             // 64-element column blocks
  static constexpr int BOX = 128 * 128;           // bytes of a 64-element x 128-row block
  static constexpr int QTILE = NCB * BOX;         // one sub-tile's queries
  static constexpr int SQBOX = 16 * 128;          // a small tile's queries: 16 rows
  static constexpr int SQ = NCB * SQBOX;
  static constexpr int KVTILE = NCB * BOX;        // one K (or V) tile
  static constexpr int STAGES = HD == 128 ? 2 : 5;
  static constexpr int STAGE_OUT = 4 * 32 * 128;  // epilogue: 32 rows x 128 bytes per warp
  static constexpr int BARS = 6144;
  static constexpr int SMEM = 2 * QTILE + 2 * SQ + 2 * STAGES * KVTILE + STAGE_OUT + BARS + 1024;
  static_assert(8 * kChunkSmallRows * HD * 4 <= 2 * QTILE, "the small tiles' join lies in the big tiles' Q");
  static_assert(SMEM <= 232448, "shared memory of a CTA");
  // Tensor memory: S of both sub-tiles, then O. With head_dim 64 there is room
  // for P beside S, so that the next S = Q K^T runs under a tile's exponentials;
  // with 128 P overwrites its S.
  static constexpr bool OWN_P = HD == 64;
  static constexpr uint32_t T_O = 256, T_P = OWN_P ? 384 : 0, P_STEP = OWN_P ? 64 : 128;
};

constexpr int kChunkMaxStages = 5;
// A piece as its CTA's warps see it.
struct ChunkWork {
  int h, row;        // kv-head, or -1: no work left; the step's row
  int q0, ntok, pos0;
  int len;           // keys the row holds
  int k0, n;         // key tiles of the piece
  int n0, n1;        // ... that sub-tile 0 and 1 visit (big)
  int slot, pieces, piece, small, dual;
};

struct ChunkShared {
  uint64_t work_full[2], work_empty[2];   // descriptor ring (producer -> everyone)
  uint64_t q_full[2][2], q_empty[2][2];   // by piece parity and sub-tile; q_empty: its Q, or the join area, is free
  uint64_t k_full[kChunkMaxStages], v_full[kChunkMaxStages];
  uint64_t k_empty[kChunkMaxStages], v_empty[kChunkMaxStages];
  uint64_t v_tail[kChunkMaxStages];       // a V tile with rows behind the last token has landed (by such tile)
  uint64_t small_done[kChunkMaxStages];   // a small tile's keys are consumed (by small tile)
  uint64_t s_full[2], p_full[2][2];       // per sub-tile; P in two halves of 64 keys
  uint64_t s_read[2], p_empty[2];         // OWN_P: S is in registers, P is consumed
  uint64_t o_full[2], o_empty[2];         // per sub-tile
  uint64_t stats_full[2][2];              // by piece parity and softmax warpgroup: max and sum, or join area, written
  uint64_t mma_drain;
  uint32_t tmem_base;
  int abort;                              // set by the first wait that runs out
  int q_armed[2];                         // pieces whose Q loads were issued
  ChunkWork work[2];
  alignas(16) int box_y[32];              // the pool rows of the next 16 tiles' boxes
  float stats[2][2][2][128];              // [piece parity][sub-tile][max, sum][row]; small: [.][0][.][warp * 16 + row]
};
static_assert(sizeof(ChunkShared) <= ChunkTile<128>::BARS, "barrier block outgrew its share");

// A number known at compile time.
template <int V>
struct Const {
  __device__ constexpr operator int() const { return V; }
};

// A position in a ring of N barriers and the parity of its phase.
template <int N>
struct ChunkRing {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void step() {
    if (++at == N) {
      at = 0;
      phase ^= 1;
    }
  }
};

template <int HD>
__global__ void __launch_bounds__(kChunkThreads, 1)
    chunk_attention_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap sqmap,
                           const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                           const ChunkParams p) {
  using C = ChunkTile<HD>;
  using Ring = ChunkRing<C::STAGES>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* qs = smem;                        // [2][QTILE]; small tiles: the join area
  uint8_t* ks = qs + 2 * C::QTILE;           // [STAGES][KVTILE]
  uint8_t* vs = ks + C::STAGES * C::KVTILE;  // [STAGES][KVTILE]
  uint8_t* sq = vs + C::STAGES * C::KVTILE;  // [2][SQ]
  uint8_t* so = sq + 2 * C::SQ;              // the epilogue's staging
  ChunkShared* sh = reinterpret_cast<ChunkShared*>(so + C::STAGE_OUT);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&sh->work_full[s], 1);
      mbar_init(&sh->work_empty[s], 14);  // every warp but the producer and warp 3
      for (int t = 0; t < 2; ++t) {
        mbar_init(&sh->q_full[s][t], 1);
        mbar_init(&sh->q_empty[s][t], 1);
        mbar_init(&sh->stats_full[s][t], 4);
        mbar_init(&sh->p_full[s][t], 4);
      }
      mbar_init(&sh->s_full[s], 1);
      mbar_init(&sh->s_read[s], 4);
      mbar_init(&sh->p_empty[s], 1);
      mbar_init(&sh->o_full[s], 1);
      mbar_init(&sh->o_empty[s], 4);
    }
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&sh->k_full[s], 1);
      mbar_init(&sh->v_full[s], 1);
      mbar_init(&sh->k_empty[s], 1);
      mbar_init(&sh->v_empty[s], 1);
      mbar_init(&sh->v_tail[s], 1);
      mbar_init(&sh->small_done[s], 8);
    }
    mbar_init(&sh->mma_drain, 1);
    sh->abort = 0;
    sh->q_armed[0] = sh->q_armed[1] = 0;
    fence_barrier_init();
  }
  if (warp == 1) tmem_alloc(&sh->tmem_base, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = sh->tmem_base;
  wait_for_prior_grid();  // the plan, when it was launched just before
  launch_dependents();    // the join waits for the SMs and then for this grid

  // Warp-uniform bounded wait; one that runs out stops every warp of the CTA.
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    return (bool)__all_sync(0xffffffffu, mbar_wait_or_abort(bar, parity, code, &sh->abort));
  };
  // The same off the critical path: it sleeps between polls and so leaves the
  // issue slots to the warps at work.
  auto sleepy = [&](uint64_t* bar, uint32_t parity) {
    return (bool)__all_sync(0xffffffffu, mbar_wait_sleepy_or_abort(bar, parity, kDevTimeoutFull, &sh->abort));
  };
  // Piece k of this CTA from the descriptor ring (h < 0: the end of the work);
  // take() is false at the end, too.
  auto take_any = [&](int k, ChunkWork& wk) {
    if (!wait(&sh->work_full[k & 1], (k >> 1) & 1, kDevTimeoutFull)) return false;
    wk = sh->work[k & 1];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh->work_empty[k & 1]);
    return true;
  };
  auto take = [&](int k, ChunkWork& wk) { return take_any(k, wk) && wk.h >= 0; };
  // Whether key tile t of a row holding len keys has V rows to be zeroed, i.e.
  // the last 64-row box that holds a key is not full (a box without keys is
  // loaded as zeros). Such a tile's V lands on v_tail; warp 2 completes v_full.
  auto ragged = [](int t, int len) { return len % 64 != 0 && t == len / kChunkKeys; };

  if (warp < 4) {
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      // Lane 0 waits and loads; the warp looks the boxes' pages up.
      if (lane == 0) {
        prefetch_tensormap(&qmap);
        prefetch_tensormap(&sqmap);
        prefetch_tensormap(&kmap);
        prefetch_tensormap(&vmap);
      }
      auto wait1 = [&](uint64_t* bar, uint32_t parity) {
        return mbar_wait_or_abort(bar, parity, kDevTimeoutEmpty, &sh->abort);
      };
      const bool planned = p.head[5] == p.plan_key;
      if (!planned) report(kDevBadIndex);
      const int n_items = planned ? p.head[0] * p.Hkv : 0;
      // The next piece is taken, and its entry read, when this one's last tiles
      // are loaded: early enough to hide the reads, late enough that a CTA
      // busy with a long piece does not hold on to another.
      int next = blockIdx.x;
      ChunkEntry e{};
      if (next < n_items) e = p.entries[next / p.Hkv];
      Ring kv, tail_at;
      int k_issued = 0, issued = 0, tails_issued = 0;  // K tiles, V tiles, and those with V rows to be zeroed
      uint32_t tails = 0;                              // bit i: the tile issued i tiles ago was one of them
      for (int k = 0;; ++k) {
        bool ok = true;
        ChunkWork wk{};
        // Q: the small buffer of this parity is free once piece k - 2 is done, a
        // sub-tile's (the small pieces' join area) once piece k - 1 is. The
        // second sub-tile's is loaded behind the first K/V tile, whose stage is
        // free earlier.
        auto load_q = [&](int s) {
          const int par = wk.small ? k & 1 : (k - 1) & 1;
          const uint32_t phase = wk.small ? ((k >> 1) & 1) ^ 1 : ((k - 1) >> 1) & 1;
          if (k >= (wk.small ? 2 : 1) && !wait1(&sh->q_empty[par][s], phase)) return false;
          if (wk.small && k >= 2 && !wait1(&sh->q_empty[par][1], phase)) return false;
          uint64_t* bar = &sh->q_full[k & 1][s];
          mbar_arrive_expect_tx(bar, C::NCB * (wk.small ? p.small_rows : p.sub_tokens * p.G) * 128);
          uint8_t* dst = wk.small ? sq + (k & 1) * C::SQ : qs + s * C::QTILE;
          const CUtensorMap* map = wk.small ? &sqmap : &qmap;
#pragma unroll
          for (int cb = 0; cb < C::NCB; ++cb, dst += wk.small ? C::SQBOX : C::BOX)
            tma_load_3d(dst, map, bar, cb * 64, wk.h * p.G, wk.q0 + s * p.sub_tokens);
          *reinterpret_cast<volatile int*>(&sh->q_armed[s]) = k + 1;
          return true;
        };
        if (lane == 0) {
          wk.h = next < n_items ? next % p.Hkv : -1;
          wk.row = e.a.x;
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
          wk.n0 = wk.n;
          wk.n1 = 0;
          if (wk.ntok > p.sub_tokens && !wk.small) {
            const int keys0 = min(wk.pos0 + p.sub_tokens, p.key_limit);
            wk.n0 = min(max(max(1, (max(keys0, 0) + kChunkKeys - 1) / kChunkKeys) - wk.k0, 0), wk.n);
            wk.n1 = wk.n;
          }
          wk.dual = !wk.small && wk.ntok <= p.sub_tokens && wk.n > 1;
          if (wk.dual) {
            wk.n0 = (wk.n + 1) / 2;
            wk.n1 = wk.n / 2;
          }
          ok = wait1(&sh->work_empty[k & 1], ((k >> 1) & 1) ^ 1);
          if (ok) {
            sh->work[k & 1] = wk;
            mbar_arrive(&sh->work_full[k & 1]);
          } else {
            wk.h = -1;
          }
        }
        const int h = __shfl_sync(0xffffffffu, wk.h, 0);
        if (h < 0) break;
        // K/V tiles in 64-row boxes, the pages of 16 tiles' boxes looked up at a
        // time (one per lane, while the 16 before are loaded). A box behind the
        // row's last key, or on no page, reads zeros (wholly out of bounds).
        const int n = __shfl_sync(0xffffffffu, wk.n, 0), k0 = __shfl_sync(0xffffffffu, wk.k0, 0);
        const int len = __shfl_sync(0xffffffffu, wk.len, 0), row = __shfl_sync(0xffffffffu, wk.row, 0);
        const int32_t* table = p.block_table + (size_t)row * p.max_pages;
        int page = -1, at = 0;
        auto look_up = [&](int j) {
          const long long tok = ((long long)k0 + j) * kChunkKeys + lane * 64;
          page = -2;  // behind the last key
          if (tok < len && tok < ((long long)k0 + n) * kChunkKeys) {
            const int col = (int)tok / p.page_size;
            at = (int)tok - col * p.page_size;
            page = col < p.max_pages ? table[col] : -1;
          }
        };
        look_up(0);
        if (lane == 0) {
          ok = load_q(0);
          if (ok && (wk.n1 == 0 || wk.dual)) {  // nothing to load: both advance with every piece
            mbar_arrive(&sh->q_full[k & 1][1]);
            *reinterpret_cast<volatile int*>(&sh->q_armed[1]) = k + 1;
          }
        }
        for (int j0 = 0; j0 < n; j0 += 16) {
          int y = -64;
          if (page >= 0 && page < p.num_pages)
            y = (page * p.Hkv + h) * p.page_size + at;
          else if (page != -2)
            report(kDevBadPage);
          sh->box_y[lane] = y;
          __syncwarp();
          if (j0 + 16 < n) look_up(j0 + 16);
          if (lane == 0 && ok) {
            for (int j = j0; j < min(n, j0 + 16); ++j) {
              if (j == max(n - 2, 0)) {
                next = (int)gridDim.x + atomicAdd(&p.head[1], 1);
                if (next < n_items) e = p.entries[next / p.Hkv];
              }
              const int2 ys = *reinterpret_cast<const int2*>(&sh->box_y[2 * (j - j0)]);
              // K and V stages are released apart: K's a tile earlier than V's.
              const bool tail = ragged(k0 + j, len);
              auto load = [&](uint64_t* bar, uint64_t* empty, const CUtensorMap* map, uint8_t* dst) {
                if (empty && !wait1(empty, kv.phase ^ 1)) return false;
                mbar_arrive_expect_tx(bar, C::KVTILE);
#pragma unroll
                for (int cb = 0; cb < C::NCB; ++cb) {
                  tma_load_2d(dst + cb * C::BOX, map, bar, cb * 64, ys.x);
                  tma_load_2d(dst + cb * C::BOX + C::BOX / 2, map, bar, cb * 64, ys.y);
                }
                return true;
              };
              if (!(ok = load(&sh->k_full[kv.at], C::OWN_P ? &sh->v_empty[kv.at] : &sh->k_empty[kv.at], &kmap,
                              ks + kv.at * C::KVTILE)))
                break;
              ++k_issued;
              if (!(ok = load(tail ? &sh->v_tail[tail_at.at] : &sh->v_full[kv.at], C::OWN_P ? nullptr : &sh->v_empty[kv.at], &vmap,
                              vs + kv.at * C::KVTILE)))
                break;
              kv.step();
              ++issued;
              if (tail) {
                tail_at.step();
                ++tails_issued;
              }
              tails = tails << 1 | (uint32_t)tail;
              if (j == 0 && wk.n1 > 0 && !wk.dual && !(ok = load_q(1))) break;
            }
          }
          __syncwarp();
        }
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
      }
      if (lane == 0) {
        // Every load issued lands before the CTA exits, also when a wait ran out.
        for (int s = 0; s < 2; ++s)
          for (int n = *reinterpret_cast<volatile int*>(&sh->q_armed[s]), i = max(n - 2, 0); i < n; ++i)
            mbar_drain(&sh->q_full[i & 1][s], (uint32_t)(i >> 1) & 1);
        drain_ring(sh->k_full, C::STAGES, k_issued);
        drain_ring(sh->v_tail, C::STAGES, tails_issued);
        for (int i = max(issued - C::STAGES, 0); i < issued; ++i)
          if (!(tails >> (issued - 1 - i) & 1)) mbar_drain(&sh->v_full[i % C::STAGES], (uint32_t)(i / C::STAGES) & 1);
        // The last CTA resets the counters: the plan serves the next layer too.
        __threadfence();
        if (planned && atomicAdd(&p.head[2], 1) == (int)gridDim.x - 1) p.head[1] = p.head[2] = 0;
      }
    } else if (warp == 1) {
      // --------------------------------------------------------- MMA issue
      constexpr uint32_t ID_QK = umma_idesc_bf16(128, 128, 0, 0);
      constexpr uint32_t ID_PV = umma_idesc_bf16(128, HD, 0, 1);
      auto issue_qk = [&](int s, int st, int q = -1) {
        tc_fence_after();
        const uint64_t dq = umma_desc_sw128(smem_u32(qs + (q < 0 ? s : q) * C::QTILE), 16, 1024);
        const uint64_t dk = umma_desc_sw128(smem_u32(ks + st * C::KVTILE), 16, 1024);
        if constexpr (HD == 128)
          umma_ss_k128_warp(tbase + 128 * s, dq, dk, ID_QK);
        else
          umma_ss_k64_warp(tbase + 128 * s, dq, dk, ID_QK);
        umma_commit_warp(&sh->s_full[s]);
      };
      ChunkWork wk;
      Ring kv, small_at;
      uint32_t tile_par = 0, o_par = 3;  // bit s: parity of sub-tile s's next P, of its O's last release
      bool early = false;  // this piece's first S of sub-tile 0 is under way already
      bool ok = take(0, wk);
      for (int k = 0; ok;) {
        if (wk.small) {
          for (int j = 0; j < wk.n; ++j, kv.step(), small_at.step()) {
            if (!(ok = wait(&sh->small_done[small_at.at], small_at.phase, kDevTimeoutFull))) break;
            if (lane == 0) {
              if (!C::OWN_P) mbar_arrive(&sh->k_empty[kv.at]);
              mbar_arrive(&sh->v_empty[kv.at]);
            }
          }
          ok = ok && take(++k, wk);
          continue;
        }
        Ring kv1 = kv;  // the stage behind kv
        kv1.step();
#pragma unroll 1
        for (int s = early ? 1 : 0; s < 2; ++s) {
          const int n_s = s == 0 ? wk.n0 : wk.n1, q = wk.dual ? 0 : s;
          // (Q is waited for even when this piece has no key for the sub-tile: it must have landed.)
          if (!(ok = wait(&sh->q_full[k & 1][s], (k >> 1) & 1, kDevTimeoutFull))) break;
          const Ring& first = wk.dual && s == 1 ? kv1 : kv;
          if (n_s > 0) {
            if (!(ok = wait(&sh->k_full[first.at], first.phase, kDevTimeoutFull))) break;
            issue_qk(s, first.at, q);
          }
          if (!C::OWN_P && (wk.dual || s == 1)) umma_commit_warp(&sh->k_empty[first.at]);
          if (!wk.dual && n_s <= 1) umma_commit_warp(&sh->q_empty[k & 1][s]);  // its last Q K^T
        }
        if (ok && wk.dual && wk.n <= 2) {
          umma_commit_warp(&sh->q_empty[k & 1][0]);
          umma_commit_warp(&sh->q_empty[k & 1][1]);
        }
        if (!ok) break;
        early = false;
        ChunkWork nx;
        nx.h = -1;
        for (int j = 0; j < wk.n; ++j) {
          kv1 = kv;  // the stage of the next S of the sub-tiles: one tile on, dual two
          kv1.step();
          if (wk.dual) kv1.step();
          const int ahead = wk.dual ? 2 : 1;
          if (!(ok = wait(&sh->v_full[kv.at], kv.phase, kDevTimeoutFull))) break;
          if (!C::OWN_P && !wk.dual && j + 1 < wk.n && !(ok = wait(&sh->k_full[kv1.at], kv1.phase, kDevTimeoutFull)))
            break;
          const uint64_t dv = umma_desc_sw128(smem_u32(vs + kv.at * C::KVTILE), C::BOX, 1024);
          // One sub-tile's step: O += P V for tile j and S = Q K^T for its next one.
          // (At head_dim 128 written out for each: the tensor pipe idles while
          // this warp works its way from one MMA to the next. At 64 the softmax is
          // the bound, and the shorter code is worth more.)
          auto step = [&](auto sub_tile) {
            const int s = sub_tile;
            const int n_s = wk.dual ? wk.n : s == 0 ? wk.n0 : wk.n1;
            if (j >= n_s || (wk.dual && (j & 1) != s)) return true;
            const uint32_t par = tile_par >> s & 1;
            auto next_s = [&]() {
              if ((C::OWN_P || wk.dual) && !wait(&sh->k_full[kv1.at], kv1.phase, kDevTimeoutFull)) return false;
              issue_qk(s, kv1.at, wk.dual ? 0 : (int)s);
              if (j + ahead + 1 == n_s) {
                umma_commit_warp(&sh->q_empty[k & 1][s]);
                if (wk.dual) umma_commit_warp(&sh->q_empty[k & 1][s ^ 1]);
              }
              return true;
            };
            if (C::OWN_P && j + ahead < n_s) {  // S is free once it is in registers
              if (!wait(&sh->s_read[s], par, kDevTimeoutFull) || !next_s()) return false;
            }
            if (s == 1 && j + 1 == wk.n && !wk.dual) {
              // While sub-tile 1 finishes the piece, sub-tile 0 starts the next
              // one as soon as its Q and K are there, so that the two stay out
              // of step (in step, their exponentials compete for the same unit).
              if (!take_any(k + 1, nx)) return false;
              const bool cand = nx.h >= 0 && !nx.small && !nx.dual && nx.n0 > 0;
              const uint32_t t0 = clock32();
              while (true) {
                if (cand && !early &&
                    __all_sync(0xffffffffu, mbar_test_wait(&sh->q_full[(k + 1) & 1][0], ((k + 1) >> 1) & 1) &&
                                                mbar_test_wait(&sh->k_full[kv1.at], kv1.phase))) {
                  issue_qk(0, kv1.at);
                  if (nx.n0 == 1) umma_commit_warp(&sh->q_empty[(k + 1) & 1][0]);
                  early = true;
                }
                if (__all_sync(0xffffffffu, mbar_test_wait(&sh->p_full[1][C::OWN_P], par))) break;
                if (__any_sync(0xffffffffu, wait_gave_up(t0, kDevTimeoutFull, &sh->abort))) return false;
              }
            } else if (!wait(&sh->p_full[s][C::OWN_P], par, kDevTimeoutFull)) {
              return false;
            }
            // O += P V in two halves: the first runs under the second's
            // exponentials. The piece's first one overwrites O, which the
            // previous epilogue must hold.
            const bool first = j < ahead && (wk.dual || j == 0);
            if (first && !wait(&sh->o_empty[s], o_par >> s & 1, kDevTimeoutFull)) return false;
            tc_fence_after();
            const uint32_t t_p = tbase + C::T_P + C::P_STEP * s, t_o = tbase + C::T_O + HD * s;
            if constexpr (C::OWN_P) {
              umma_ts_t128_linear_warp(t_o, t_p, dv, ID_PV, first ? 0u : 1u);
              umma_commit_warp(&sh->p_empty[s]);
            } else {
              umma_ts_t64_linear_warp(t_o, t_p, dv, ID_PV, first ? 0u : 1u);
              if (!wait(&sh->p_full[s][1], par, kDevTimeoutFull)) return false;
              tc_fence_after();
              umma_ts_t64_linear_warp(t_o, t_p + 32, dv + 512, ID_PV, 1u);
            }
            if (j + ahead >= n_s)
              umma_commit_warp(&sh->o_full[s]);
            else if (!C::OWN_P && !next_s())
              return false;
            tile_par ^= 1u << s;
            return true;
          };
          if constexpr (C::OWN_P) {
#pragma unroll 1
            for (int s = 0; ok && s < 2; ++s) ok = step(s);
          } else {
            ok = step(Const<0>{}) && step(Const<1>{});
          }
          if (!ok) break;
          if (!C::OWN_P && j + ahead < wk.n) umma_commit_warp(&sh->k_empty[kv1.at]);
          umma_commit_warp(&sh->v_empty[kv.at]);
          kv.step();
        }
        if (!ok) break;
        if ((wk.n1 == 0 || wk.dual) && !(ok = take_any(k + 1, nx))) break;
        o_par ^= (uint32_t)(wk.n0 > 0) | (uint32_t)(wk.n1 > 0) << 1;
        wk = nx;
        ++k;
        ok = wk.h >= 0;
      }
      umma_drain_warp(&sh->mma_drain);  // before TMEM is freed, also when a wait ran out
    } else if (warp == 2) {
      // ------------------------------------- zeroing behind the last token
      ChunkWork wk;
      Ring tail_at;
      int J = 0;  // tiles before this piece
      for (int k = 0; sleepy(&sh->work_full[k & 1], (k >> 1) & 1) && take(k, wk); ++k) {
        const int j = wk.len / kChunkKeys - wk.k0;
        if (j >= 0 && j < wk.n && ragged(wk.k0 + j, wk.len)) {
          const int st = (J + j) % C::STAGES;
          if (!wait(&sh->v_tail[tail_at.at], tail_at.phase, kDevTimeoutFull)) break;
          const int r0 = wk.len % kChunkKeys, rows = 64 - r0 % 64;
          uint8_t* v = vs + st * C::KVTILE;
#pragma unroll 1
          for (int i = lane; i < rows * C::NCB * 8; i += 32) {
            const int r = r0 + i / (C::NCB * 8), cb = i / 8 % C::NCB;
            *reinterpret_cast<uint4*>(v + cb * C::BOX + r * 128 + (i & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async();  // read by tcgen05.mma, overwritten by the next load
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh->v_full[st]);
          tail_at.step();
        }
        J += wk.n;
      }
    }
  } else if (warp < 12) {
    const int hh = (warp - 4) >> 2;  // big: sub-tile
    const int sub = warp & 3;        // TMEM lane quarter this warp may access
    const int r = sub * 32 + lane;   // query row of the sub-tile
    const int r_tok0 = r < p.sub_tokens * p.G ? r / p.G : 0x40000000;
    const uint32_t lane_bits = (uint32_t)(sub * 32) << 16;
    const uint32_t t_s = tbase + 128 * hh + lane_bits;
    const uint32_t t_p = tbase + C::T_P + C::P_STEP * hh + lane_bits;
    const uint32_t t_o = tbase + C::T_O + HD * hh + lane_bits;
    const int sw = warp - 4;  // small: its 16 keys of a tile
    const int gid = lane >> 2, tig = lane & 3;
    ChunkWork wk;
    Ring kv, small_at;       // (kv is kept by the small pieces only, from the tile count)
    int J = 0;               // tiles before this piece
    uint32_t tile_par = 0;   // parity of this sub-tile's next S
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
        if (!(ok = wait(&sh->q_full[k & 1][0], (k >> 1) & 1, kDevTimeoutFull))) break;
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
        kv.at = J % C::STAGES;
        kv.phase = (J / C::STAGES) & 1;
        int tok0 = wk.k0 * kChunkKeys + sw * 16;
        for (int j = 0; j < wk.n; ++j, kv.step(), small_at.step(), tok0 += kChunkKeys) {
          if (!(ok = wait(&sh->k_full[kv.at], kv.phase, kDevTimeoutFull))) break;
          float s[2][4];
          const uint32_t kb = smem_u32(ks + kv.at * C::KVTILE);
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
            alpha[half] = m_new == -INFINITY ? 1.f : fast_exp2(m[half] - m_new);
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
          if (!(ok = wait(&sh->v_full[kv.at], kv.phase, kDevTimeoutFull))) break;
          const uint32_t pa[4] = {pack_bf16x2(s[0][0], s[0][1]), pack_bf16x2(s[0][2], s[0][3]),
                                  pack_bf16x2(s[1][0], s[1][1]), pack_bf16x2(s[1][2], s[1][3])};
          const uint32_t vb = smem_u32(vs + kv.at * C::KVTILE);
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
          if (lane == 0) mbar_arrive(&sh->small_done[small_at.at]);
        }
        if (!ok) break;
        J += wk.n;
        // Into the join area once piece k - 1 has left it.
        if (k >= 1 && !(ok = wait(&sh->q_empty[(k - 1) & 1][0], ((k - 1) >> 1) & 1, kDevTimeoutEmpty) &&
                             wait(&sh->q_empty[(k - 1) & 1][1], ((k - 1) >> 1) & 1, kDevTimeoutEmpty)))
          break;
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
        if (lane == 0) mbar_arrive(&sh->stats_full[k & 1][hh]);
        continue;
      }
      // --------------------------------------------------- big: softmax
      const int n = hh == 0 ? wk.n0 : wk.n1;
      const int r_tok = r_tok0 + (wk.dual ? 0 : hh * p.sub_tokens);
      // Last visible key. (Rows without a token compute on and are dropped.)
      const int hi = r_tok < wk.ntok ? min(wk.pos0 + r_tok, wk.len - 1) : 0x7fffffff;
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j, tile_par ^= 1) {
        const int kv0 = (wk.k0 + (wk.dual ? 2 * j + hh : j)) * kChunkKeys;
        if (!(ok = wait(&sh->s_full[hh], tile_par, kDevTimeoutFull))) break;
        tc_fence_after();
        // S is read twice, 64 columns at a time in rolled loops: once for the
        // maximum, once for the exponentials. (All 128 columns held in registers
        // and unrolled, the kernel's loops outgrew the instruction cache: on
        // short pieces, where all its roles are busy, a quarter of the fetches
        // missed and tiles took twice as long.)
        const bool masked = __any_sync(0xffffffffu, kv0 + kChunkKeys - 1 > hi);
        // Scores of the keys behind the row's last visible one, whatever they
        // are, become -inf; the first pass writes them back for the second.
        auto load = [&](int half, uint32_t(&v)[64]) {
          tmem_ld32(t_s + 64 * half, *reinterpret_cast<uint32_t(*)[32]>(v));
          tmem_ld32(t_s + 64 * half + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
          tmem_wait_ld();
        };
        float mx = -INFINITY;
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t v[64];
          load(half, v);
          if (masked) {
            const int last = hi - kv0 - 64 * half;
#pragma unroll
            for (int e = 0; e < 64; ++e) v[e] = e <= last ? v[e] : __float_as_uint(-INFINITY);
            tmem_st32(t_s + 64 * half, *reinterpret_cast<uint32_t(*)[32]>(v));
            tmem_st32(t_s + 64 * half + 32, *reinterpret_cast<uint32_t(*)[32]>(v + 32));
            tmem_wait_st();
          }
          float mp[8];  // independent chains
#pragma unroll
          for (int q = 0; q < 8; ++q) mp[q] = fmax_nan(__uint_as_float(v[q]), __uint_as_float(v[8 + q]));
#pragma unroll
          for (int e = 16; e < 64; e += 16)
#pragma unroll
            for (int q = 0; q < 8; ++q) mp[q] = fmax3_nan(mp[q], __uint_as_float(v[e + q]), __uint_as_float(v[e + 8 + q]));
          mx = fmax3_nan(fmax3_nan(mp[0], mp[1], mp[2]), fmax3_nan(mp[3], mp[4], mp[5]), fmax3_nan(mp[6], mp[7], mx));
        }
        // O is rescaled only when the maximum grew by more than 2^8: the final
        // division uses the same stale maximum, so the result is exact. (A row
        // that sees no key of the tile keeps -inf; a NaN or +inf among the
        // visible scores makes the maximum, and with it the row, NaN.)
        const float m_tile = mx == -INFINITY ? mx : fmaf(mx, p.scale_log2, mx - mx);
        const bool grew = !(m_tile <= m_used + 8.f);
        // P's columns (and O) are free once the tile before is consumed.
        if (C::OWN_P) {
          if (!(ok = wait(&sh->p_empty[hh], tile_par ^ 1, kDevTimeoutEmpty))) break;
          tc_fence_after();
        }
        if (j == 0) {
          m_used = m_tile;
        } else if (__any_sync(0xffffffffu, grew)) {
          const float alpha = grew ? fast_exp2(m_used - m_tile) : 1.f;
          if (grew) m_used = fmax_nan(m_used, m_tile);  // (NaN stays)
          l *= alpha;
#pragma unroll 1
          for (int c = 0; c < HD / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(t_o + 16 * c, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16(t_o + 16 * c, o);
          }
          tmem_wait_st();
        }
        const float neg_mu = m_used == -INFINITY ? 0.f : -m_used;
        // P and its row sums. Without P columns of its own, P's first half lies
        // over the S columns 0 .. 31 and its second over 32 .. 63, both read.
#pragma unroll 1
        for (int half = 0; half < 2; ++half) {
          uint32_t v[64];
          load(half, v);
          if (C::OWN_P && half == 1) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->s_read[hh]);
          }
          float ls[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) ls[q] = 0.f;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 32; e += 2) {
              float x0, x1;
              ffma2(x0, x1, __uint_as_float(v[32 * c + e]), __uint_as_float(v[32 * c + e + 1]), p.scale_log2,
                    p.scale_log2, neg_mu, neg_mu);
              // (Some of them by a polynomial on the FMA pipe gained nothing: one
              // pair in four 545 us against 545 and 426 against 423 at head_dim 128,
              // one in eight 425 against 403 at 64.)
              const float p0 = fast_exp2(x0), p1 = fast_exp2(x1);
              const int q = 2 * ((e >> 1) & 3);
              fadd2(ls[q], ls[q + 1], ls[q], ls[q + 1], p0, p1);
              pk[e >> 1] = pack_bf16x2(p0, p1);
            }
            tmem_st16(t_p + 32 * half + 16 * c, pk);
          }
          l += ((ls[0] + ls[1]) + (ls[2] + ls[3])) + ((ls[4] + ls[5]) + (ls[6] + ls[7]));
          if (!C::OWN_P || half == 1) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh->p_full[hh][half]);
          }
        }
      }
      if (!ok) break;
      sh->stats[k & 1][hh][0][r] = m_used;
      sh->stats[k & 1][hh][1][r] = l;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->stats_full[k & 1][hh]);
      J += wk.n;
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int tid = threadIdx.x - 384;
    const int sub = warp & 3;
    const int r = sub * 32 + lane;
    const uint32_t lane_bits = (uint32_t)(sub * 32) << 16;
    // Where this lane's stores of a sub-tile's turned lines go, from the
    // sub-tile's first query row.
    int off[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int qr = sub * 32 + i * 4 + (lane >> 3);
      off[i] = (qr / p.G * p.Hq + qr % p.G) * HD + 8 * (lane & 7);
    }
    ChunkWork wk;
    uint32_t o_par = 0;  // bit s: parity of sub-tile s's next O
    bool ok = true;
    for (int k = 0;; ++k) {
      // The four warps leave together: they share named barriers.
      wk.h = 0;
      ok = ok && sleepy(&sh->work_full[k & 1], (k >> 1) & 1);
      if (ok) wk = sh->work[k & 1];
      if (named_barrier_or(1, 128, !ok) || wk.h < 0) break;
      const bool split = wk.pieces > 1;
      const int rows = wk.ntok * p.G;
      const size_t part = ((size_t)(wk.slot + wk.piece) * p.Hkv + wk.h) * p.part_rows;
      if (wk.small) {
        ok = sleepy(&sh->stats_full[k & 1][0], (k >> 1) & 1) && sleepy(&sh->stats_full[k & 1][1], (k >> 1) & 1);
        if (named_barrier_or(1, 128, !ok)) break;
        const float* join = reinterpret_cast<const float*>(qs);
        const float(*st)[128] = sh->stats[k & 1][0];
#pragma unroll 1
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
            const float f = fast_exp2(st[0][w * 16 + rr] - Mu);
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
            const float inv = L != 0.f ? 1.f / L : 0.f;
            const int tok = wk.q0 + rr / p.G, h = wk.h * p.G + rr % p.G;
            uint2 u;
            u.x = pack_bf16x2(O.x * inv, O.y * inv);
            u.y = pack_bf16x2(O.z * inv, O.w * inv);
            *reinterpret_cast<uint2*>(p.out + ((size_t)tok * p.Hq + h) * HD + c4 * 4) = u;
          }
        }
        fence_proxy_async();  // the next big tile's Q lands here
        named_barrier(1, 128);
        if (tid < 2) mbar_arrive(&sh->q_empty[k & 1][tid]);
      } else {
        // O out of tensor memory a row per lane, 128 bytes of it at a time,
        // turned in shared memory so that eight lanes store a whole line.
        uint8_t* stage = so + (warp - 12) * 4096;
        const int sub_rows = p.sub_tokens * p.G;
#pragma unroll 1
        for (int hh = 0; hh < 2; ++hh) {
          if (hh * p.sub_tokens >= wk.ntok) break;
          // Both sub-tiles' O are the same rows' in a dual piece.
          const int last = wk.dual ? 1 : hh;
          for (int s = hh; ok && s <= last; ++s) {
            ok = sleepy(&sh->stats_full[k & 1][s], (k >> 1) & 1);
            if (ok && (s == 0 ? wk.n0 : wk.n1) > 0) {  // else: no key tile of this piece
              ok = sleepy(&sh->o_full[s], o_par >> s & 1);
              o_par ^= 1u << s;
            }
          }
          if (!ok) break;
          tc_fence_after();
          const bool any = (hh == 0 ? wk.n0 : wk.n1) > 0;
          float m_used = sh->stats[k & 1][hh][0][r], l = sh->stats[k & 1][hh][1][r], f0 = 1.f, f1 = 0.f;
          if (wk.dual) {
            const float m1 = sh->stats[k & 1][1][0][r], l1 = sh->stats[k & 1][1][1][r], M = fmaxf(m_used, m1);
            f0 = l != 0.f ? fast_exp2(m_used - M) : 0.f;
            f1 = l1 != 0.f ? fast_exp2(m1 - M) : 0.f;
            m_used = M;
            l = l * f0 + l1 * f1;
          }
          const float inv = split ? 1.f : 1.f / l;
          const uint32_t t_o = tbase + C::T_O + HD * hh + lane_bits;
          const int live = min(sub_rows, rows - hh * sub_rows) - sub * 32;  // of this warp's 32 rows
          const size_t pr = part + hh * sub_rows + sub * 32;
          __nv_bfloat16* out = p.out + ((size_t)(wk.q0 + hh * p.sub_tokens) * p.Hq + wk.h * p.G) * HD;
          const int cols = split ? 32 : 64;  // of a 128-byte line
          // Where this lane's 16 bytes of line c0's eight turned stores go.
          uint8_t* dst = split ? reinterpret_cast<uint8_t*>(p.part_o + pr * HD + 4 * (lane & 7))
                               : reinterpret_cast<uint8_t*>(out);
#pragma unroll 1
          for (int c0 = 0; c0 < HD; c0 += cols) {
#pragma unroll 1
            for (int c = c0; c < c0 + cols; c += 16) {
              uint32_t o[16];
              tmem_ld16(t_o + c, o);
              tmem_wait_ld();
              if (wk.dual) {
                uint32_t o1[16];
                tmem_ld16(t_o + HD + c, o1);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; ++e)
                  o[e] = __float_as_uint((f0 > 0.f ? __uint_as_float(o[e]) * f0 : 0.f) +
                                         (f1 > 0.f ? __uint_as_float(o1[e]) * f1 : 0.f));
              }
              if (c == HD - 16 && any) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {  // the next piece may overwrite O
                  mbar_arrive(&sh->o_empty[hh]);
                  if (wk.dual) mbar_arrive(&sh->o_empty[1]);
                }
              }
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] = l != 0.f ? __float_as_uint(__uint_as_float(o[e]) * inv) : 0u;
              if (split) {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                  *reinterpret_cast<uint4*>(stage + lane * 128 + ((((c - c0) / 4 + q) ^ (lane & 7)) << 4)) =
                      make_uint4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
              } else {
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                  uint4 u;
                  u.x = pack_bf16x2(__uint_as_float(o[8 * q + 0]), __uint_as_float(o[8 * q + 1]));
                  u.y = pack_bf16x2(__uint_as_float(o[8 * q + 2]), __uint_as_float(o[8 * q + 3]));
                  u.z = pack_bf16x2(__uint_as_float(o[8 * q + 4]), __uint_as_float(o[8 * q + 5]));
                  u.w = pack_bf16x2(__uint_as_float(o[8 * q + 6]), __uint_as_float(o[8 * q + 7]));
                  *reinterpret_cast<uint4*>(stage + lane * 128 + ((((c - c0) / 8 + q) ^ (lane & 7)) << 4)) = u;
                }
              }
            }
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int row = i * 4 + (lane >> 3);
              const uint4 u = *reinterpret_cast<const uint4*>(stage + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
              if (row < live) *reinterpret_cast<uint4*>(dst + (split ? row * HD * 4 : off[i] * 2)) = u;
            }
            dst += 128;
            __syncwarp();
          }
          if (split && lane < live) p.part_ml[pr + lane] = make_float2(m_used, l);
        }
      }
      // Only now: nobody gets two pieces ahead of the epilogue, so max, sum and
      // join area by piece parity are enough.
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->work_empty[k & 1]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tbase, 512);
  }
  if (threadIdx.x == 0 && *reinterpret_cast<volatile int*>(&sh->abort)) p.head[4] = 1;  // nothing to join
}

// out of the split tiles: over a row's pieces, in their order, M = max m,
// out = sum O 2^(m - M) / sum l 2^(m - M). A warp per row.
template <int HD>
__global__ void __launch_bounds__(32 * kJoinRows, 4) chunk_join_kernel(const ChunkParams p) {
  constexpr int E = HD / 32;  // output elements per lane
  wait_for_prior_grid();
  const int lane = threadIdx.x & 31;
  if (p.head[5] != p.plan_key) return;
  if (p.head[4]) {
    // A wait ran out. The last block takes the mark back, once every thread of
    // the grid has read it: the next launch on this plan is joined again.
    __syncthreads();
    if (threadIdx.x == 0 && atomicAdd(&p.head[6], 1) == (int)gridDim.x - 1) p.head[4] = p.head[6] = 0;
    return;
  }
  const int units = p.head[3] * p.Hkv;
  const size_t step = (size_t)p.Hkv * p.part_rows;
  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int h = u % p.Hkv;
    const ChunkSplit sp = p.splits[u / p.Hkv];
    const int row = sp.row0 + (threadIdx.x >> 5);
    if (row >= sp.rows) continue;
    const size_t first = ((size_t)sp.slot * p.Hkv + h) * p.part_rows + row;
    float M = -INFINITY;
    for (int c = lane; c < sp.pieces; c += 32) M = fmaxf(M, p.part_ml[first + c * step].x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
    float L = 0.f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.f;
    const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll 2
    for (int c = 0; c < sp.pieces; ++c) {
      const float2 ml = p.part_ml[first + c * step];
      const float f = exp2f(ml.x - Mu);
      const float* src = p.part_o + (first + c * step) * HD + lane * E;
      L += ml.y * f;
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 x = *reinterpret_cast<const float2*>(src + e);
        o[e] += x.x * f;
        o[e + 1] += x.y * f;
      }
    }
    const float inv = L != 0.f ? 1.f / L : 0.f;
    __nv_bfloat16* dst = p.out + ((size_t)(sp.q0 + row / p.G) * p.Hq + h * p.G + row % p.G) * HD + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2)
      *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16x2(o[e] * inv, o[e + 1] * inv);
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
  lay->head = off;     off = up(off + 7 * sizeof(int));
  lay->entries = off;  off = up(off + lay->max_entries * sizeof(ChunkEntry));
  lay->splits = off;   off = up(off + extra * ((lay->part_rows + kJoinRows - 1) / kJoinRows) * sizeof(ChunkSplit));
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
  for (int i = 0; i < 3; ++i) q.cost[i] = kChunkTileCost[p.head_dim == 128][i];
  q.plan_key = p.plan_key;
  q.max_entries = (int)lay.max_entries;
  q.max_slots = (int)lay.max_slots;
  q.entries = reinterpret_cast<ChunkEntry*>(ws + lay.entries);
  q.head = reinterpret_cast<int*>(ws + lay.head);
  q.splits = reinterpret_cast<ChunkSplit*>(ws + lay.splits);
  int threads = 256;  // a power of two: the buckets are scanned in whole blocks of threads
  while (threads < kChunkPlanThreads && threads < p.batch) threads *= 2;
  chunk_plan_kernel<<<1, threads, 0, stream>>>(q);
  return cudaGetLastError();
}

// One-time set-up of an instantiation on the current device: its shared memory.
template <int HD>
static cudaError_t chunk_prepare() {
  static std::atomic<int> ready[kMaxDevices];
  const int dev = device_slot();
  if (dev >= 0 && ready[dev].load(std::memory_order_acquire)) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(chunk_attention_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       ChunkTile<HD>::SMEM);
  if (e == cudaSuccess && dev >= 0) ready[dev].store(1, std::memory_order_release);
  return e;
}

template <int HD>
static cudaError_t launch_chunk(const CUtensorMap& qm, const CUtensorMap& sqm, const CUtensorMap& km,
                                const CUtensorMap& vm, const ChunkParams& p, unsigned grid, bool after_plan,
                                cudaStream_t stream) {
  cudaError_t e = chunk_prepare<HD>();
  if (e != cudaSuccess) return e;
  // Right behind its plan the kernel starts early and waits for it in its
  // own prologue; otherwise it is an ordinary launch.
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kChunkThreads);
  cfg.dynamicSmemBytes = ChunkTile<HD>::SMEM;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = after_plan ? 1 : 0;
  e = cudaLaunchKernelEx(&cfg, chunk_attention_kernel<HD>, qm, sqm, km, vm, p);
  // A table whose longest tile costs no more than the shortest piece allowed needs no join.
  const int kind = p.tokens > p.sub_tokens ? kTwoSubs : p.tokens > kChunkSmallRows / p.G ? kOneSub : kSmallTile;
  const long long most = ((long long)p.key_limit + kChunkKeys - 1) / kChunkKeys * kChunkTileCost[HD == 128][kind];
  if (e != cudaSuccess || most <= kMinPieceCost) return e;
  cfg.gridDim = dim3(8 * grid);
  cfg.blockDim = dim3(32 * kJoinRows);
  cfg.dynamicSmemBytes = 0;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, chunk_join_kernel<HD>, p);
}

cudaError_t launch_chunk_attention(const CUtensorMap& qm, const CUtensorMap& sqm, const CUtensorMap& km,
                                   const CUtensorMap& vm, ChunkParams p, const ChunkLayout& lay, uint8_t* ws, int sms,
                                   bool after_plan, cudaStream_t stream) {
  p.entries = reinterpret_cast<const ChunkEntry*>(ws + lay.entries);
  p.head = reinterpret_cast<int*>(ws + lay.head);
  p.splits = reinterpret_cast<const ChunkSplit*>(ws + lay.splits);
  p.part_ml = reinterpret_cast<float2*>(ws + lay.part_ml);
  p.part_o = reinterpret_cast<float*>(ws + lay.part_o);
  p.part_rows = lay.part_rows;
  const unsigned grid = (unsigned)std::min<size_t>((size_t)sms, lay.max_entries * p.Hkv);
  return p.head_dim == 128 ? launch_chunk<128>(qm, sqm, km, vm, p, grid, after_plan, stream)
                           : launch_chunk<64>(qm, sqm, km, vm, p, grid, after_plan, stream);
}

}  // namespace mb
