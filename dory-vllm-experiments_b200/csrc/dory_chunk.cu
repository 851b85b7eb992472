// dory_chunk.cu — attention of a chunk of new tokens over the paged cache
// (dory_chunk_attention; the C ABI is in include/dory_decode.h).
//
// out[t][h] = gate * sum_c softmax_c(scale q.k_c) v_c over the positions c a token sees.
//
// Shape of the work.  The G query heads of a KV head see the same keys, so G x (128 / G) rows
// (token, head) fill the 128 rows of a tensor-core tile; an item of work is one or two such
// tiles (kTiles) of one sequence and KV head, with the 128-position cache tiles they see.  A
// unit is one cache tile of one item.  All units of the batch, in (sequence, KV head, item)
// order, are cut into equal consecutive pieces, one per SM: causal triangles, ragged lengths
// and a few rows over a long cache all balance by themselves.  An item cut between SMs leaves
// FP32 partial results (unnormalised sum, maximum, sum of weights) which a second small launch
// joins, so results do not depend on arrival order.
//
// chunk_kernel, one CTA per SM, warp roles:
//   scheduler  derives the SM's piece from query_start / seq_lens on the device (no host read,
//              so a captured graph follows new lengths) and hands items to the others;
//   loader     tensor copies: the queries, and K and V tiles page by page through the block
//              table into a ring (256-dim bf16 heads: two warps); pages outside the item's
//              positions, and bad block ids, load as zeros without touching memory;
//   conversion (FP8 caches, four warps) e4m3 tiles to f16 tiles, bf16 queries to scaled f16 ones;
//   products   tcgen05: S = Q K^T into tensor memory, O += P V with P read from there;
//   softmax    two warpgroups, a row (256-dim heads: half a row) per thread: scores to
//              registers, running maximum, exponentials, P back to tensor memory as 16-bit
//              floats, and at the end of an item O / sum, gate and store.
// With 64/128-dim heads an item has two tiles and the products of one overlap the softmax of
// the other.  With 256-dim heads tensor memory holds one tile's O and two score buffers.
//
// O is rescaled only when a row's maximum has grown by more than 2^8: the weights stay below
// 2^8, far from the range's end, and most tiles touch O not at all.
//
// Positions no row of the item sees (behind the sequence, before the window) may hold anything,
// so their V rows are zeroed in shared memory (0 x NaN would reach the sum).  A position that
// some rows see and others do not can still hold Inf or NaN: a row whose O comes out non-finite
// from finite weights is looked at by the join kernel, which computes it again from its own
// positions alone if it took part in a product with such a position without seeing it.
//
// What bounds it, measured (CUDA graph, 16-row pages, FP32 gate): long chunks the length of a cache
// tile's chain (scores, the row's maximum over all columns, the columns read again for the weights,
// product), which two tiles in turn do not hide: no unit is full (prompt of 8192, 32 query heads on
// 8, 128 dims: 543 us, 1,012 TFLOP/s, 63% of the library GEMM's rate; no exponentials, or half of
// the products, would save 5-13%).  64-dim heads have the same chain for half of the products (476
// us, 577 TFLOP/s); 256-dim heads the page copies as well (16 heads on 4: 669 us, 585 with 128-row
// pages); FP8 caches the conversion (597 us); short items their latency, 4-5 us each, and a call of
// few tokens the chain from launch to join (4 tokens over 640: 16.5 us).

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include <cudaTypedefs.h>

#include <mutex>
#include <type_traits>

#include "dory_common.h"
#include "dory_sm100.cuh"

namespace {

using namespace sm100;
using dory::aligned16;
using dory::device_sms;
using dory::fail;

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kM = 128;              // rows of a tensor-core tile
constexpr int kN = 128;              // positions of a cache tile
constexpr int kChunkBytes = kN * 128;  // 64 columns of a tile: 128 rows of 128 bytes
constexpr int kItemUnits = 3;        // cost of an item's output, in cache tiles
constexpr int kQueue = 4;            // items handed out ahead
constexpr int kBadRing = 16;         // tiles whose bad-page masks are kept
constexpr int kMaxPosition = 1 << 30;
constexpr float kSlack = 8.0f;       // log2 a row's maximum may grow before O is rescaled
// ~2 s, then give up.
constexpr long long kWaitLimitCycles = 4000000000LL;

struct ChunkArgs {
  const __nv_bfloat16* q;
  const void* kc;
  const void* vc;
  const int32_t* tables;
  const int32_t* query_start;
  const int32_t* seq_lens;
  const void* gate;
  __nv_bfloat16* out;
  uint32_t* err;
  int64_t q_t, q_h, out_t, gate_t, table_stride, sb, so, sh, blocks;
  float scale_log2, k_scale, v_scale;
  int T, S, max_blocks, NH, NKV, G, B, window, gate_dtype;
  int TB;             // tokens of a tile: 128 / G
  int copy_rows;      // rows of a tensor copy: the largest power of two dividing B, up to 128
  int copy_shift;     // its logarithm
  int table_span;     // positions the table names, at most kMaxPosition
  int32_t* joins;     // [CTAs][8] (Join): what each CTA leaves to the join kernel
  float2* part_ml;    // [2 CTAs][rows]: (maximum in log2 units, sum of weights)
  float* part_o;      // [2 CTAs][rows][HD]
};
struct Maps {
  CUtensorMap q, k, v;
};

__device__ __forceinline__ float load_gate(const ChunkArgs& a, int64_t i) {
  if (a.gate_dtype == DORY_DTYPE_F32) return static_cast<const float*>(a.gate)[i];
  if (a.gate_dtype == DORY_DTYPE_BF16)
    return __bfloat162float(static_cast<const __nv_bfloat16*>(a.gate)[i]);
  return __half2float(static_cast<const __half*>(a.gate)[i]);
}

// Two e4m3 values, the low byte the lower one, in f16: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two_bytes) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two_bytes)));
  return r;
}
// The first N values of a cache row's words.
template <bool KV8, int N>
__device__ __forceinline__ void unpack(const uint32_t* words, float* x) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    if (KV8) {
      const uint32_t h = e4m3x2_to_f16x2(words[i / 4] >> (8 * (i % 4)) & 0xffffu);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      x[i] = f.x;
      x[i + 1] = f.y;
    } else {
      x[i] = __uint_as_float(words[i / 2] << 16);
      x[i + 1] = __uint_as_float(words[i / 2] & 0xffff0000u);
    }
  }
}

// Rows [t0, t1) of sequence i, whatever the arrays hold: always within [0, T].
__device__ __forceinline__ void rows_of(const ChunkArgs& a, int i, int& t0, int& t1) {
  t0 = min(max(a.query_start[i], 0), a.T);
  t1 = min(max(a.query_start[i + 1], t0), a.T);
}

// The block of a sequence that holds position c, or -1 (reported) outside the cache.
__device__ __forceinline__ int64_t block_of(const ChunkArgs& a, const int32_t* table, int c) {
  const int b = c / a.B;
  const int64_t id = b < a.max_blocks ? table[b] : -1;
  if (id < 0 || id >= a.blocks) {
    atomicOr(a.err, DORY_DEVERR_BLOCK_OOB);
    return -1;
  }
  return id;
}

// ------------------------------------------------------------------------------------
// The tensor-core kernel
// ------------------------------------------------------------------------------------
constexpr int kWide128 = 1, kWide256 = 2;
template <int HD, bool KV8>
struct Shape {
  static constexpr int kTiles = HD == 256 ? 1 : 2;           // tensor-core tiles of an item
  static constexpr int kCols = HD < 128 ? HD : 128;          // columns of a ring stage
  static constexpr int kHalves = HD / kCols;                 // stages of a K (or V) tile
  static constexpr int kStageBytes = kCols / 64 * kChunkBytes;
  static constexpr int kStages = HD == 64 ? 8 : KV8 ? 3 : 5;
  // FP8 caches: tiles of bytes as they were copied, 128 dims a row, before their conversion
  static constexpr int kRawStages = KV8 ? 4 : 0, kRawBytes = kChunkBytes;
  static constexpr int kConvertWarps = KV8 ? 4 : 0;
  static constexpr int kTileBytes = kTiles * HD / 64 * kChunkBytes + kStages * kStageBytes +
                                    kRawStages * kRawBytes;
  static constexpr int kQBytes = kTiles * HD / 64 * kChunkBytes;
  static constexpr int kShares = HD == 256 ? kWide256 : kWide128;  // softmax warpgroups of a tile
  static constexpr int kScoreCols = kN / kShares;            // of a row, per softmax thread
  static constexpr int kOutCols = HD / kShares;
  static constexpr int kParts = kScoreCols > 32 ? 2 : 1;     // the weights are handed over in
  static constexpr int kPartCols = kScoreCols / kParts;
  static constexpr int kSoftmaxWarps = 4 * kShares * kTiles;
  // Copying warps: the 256-dim heads' four stages a tile keep one busier than the products
  // (16-row pages, prompt of 8192: 786 us, 692 with two; four: 662, but 640 in place of 587 with
  // 128-row pages); elsewhere the second only takes issue slots (542 us, 565).
  static constexpr int kLoaders = HD == 256 && !KV8 ? 2 : 1;
  static constexpr int kLoadWarp = kSoftmaxWarps, kMmaWarp = kLoadWarp + kLoaders,
                       kPlanWarp = kMmaWarp + 1;
  [[maybe_unused]] static constexpr int kConvert = kPlanWarp + 1;  // the first of these
  static constexpr int kThreads = (kConvert + kConvertWarps) * 32;
  static constexpr int kItemRows = kTiles * kM;
  // f16 weights are lifted by 2^7, to below 2^15 (kSlack), so that they are exact to 11 bits down
  // to 2^-21 of the row's largest and end at 2^-32 of it
  static constexpr float kLift = KV8 ? 7.0f : 0.0f;
  // Of four pairs of exponentials, those that go to the FP32 pipe: a piece of 32 columns takes two
  // warps of a scheduler 486 clocks with one, 562 with none, 532 with two (prompt of 8192: 542
  // us, 557, 557).  256-dim heads and FP8 caches wait for other things: none (1-2% better).
  static constexpr int kPolyOf4 = HD == 256 || KV8 ? 0 : 1;
  // tensor memory, in columns: two score buffers (P takes a buffer's first half), then O
  static constexpr int kO = 2 * kN;
  static constexpr int kOStride = HD <= 128 ? 128 : 0;       // between the tiles' O
};

enum : int { kItemEnd = 1 };
struct Item {
  int flags;
  int kv0, kvn;      // cache tiles of this piece: [kv0, kv0 + kvn)
  int tok0, ntok;    // query rows of the batch
  int pos0;          // position of the first (negative: before the sequence)
  int kvh, seq;
  int cap;           // positions of the sequence that the table names
  int slot;          // partial-result slot, -1: the whole item is here
  int tile;          // the tensor-core tile of its first rows: 1 only if they fill one at most
  int pad[5];
  __device__ int tiles(const ChunkArgs& a) const { return ntok > a.TB ? 2 : 1; }
};

template <int HD, bool KV8>
struct Control {  // shared memory behind the tiles
  alignas(8) uint64_t kv_full[Shape<HD, KV8>::kStages], kv_empty[Shape<HD, KV8>::kStages];
  uint64_t raw_full[4], raw_empty[4], q_raw[2];  // FP8 caches only
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2][2], o_full[2], item_full[kQueue],
      item_empty[kQueue], met[4 * Shape<HD, KV8>::kTiles], drained;
  Item items[kQueue];
  uint32_t bad[kBadRing];
  // what a row's f16 query was divided by; a second set for the tile's next item, which the
  // conversion may reach while softmax warps are still at the output of the item before
  float q_scale[2][KV8 ? Shape<HD, KV8>::kItemRows : 1];
  uint32_t tmem;
  int abort;
  // a row's maxima and sums, by share
  float swap[Shape<HD, KV8>::kTiles][Shape<HD, KV8>::kShares][Shape<HD, KV8>::kShares > 1 ? kM : 1];
};

__device__ __noinline__ bool wait_slow(uint32_t bar, uint32_t parity, volatile int* abort,
                                       uint32_t* err) {
  const long long start = clock64();
  while (!mbar_try(bar, parity)) {
    if (*abort) return false;
    if (clock64() - start > kWaitLimitCycles) {
      *abort = 1;
      atomicOr(err, DORY_DEVERR_WAIT_TIMEOUT);
      return false;
    }
  }
  return true;
}
// A whole warp's wait, the same answer in every lane.
__device__ __forceinline__ bool wait_bar(uint32_t b, uint32_t parity, int* abort, uint32_t* err) {
  bool ok = mbar_try(b, parity);
  if (!__all_sync(0xffffffffu, ok)) {
    if (!ok) ok = wait_slow(b, parity, abort, err);
    return __all_sync(0xffffffffu, ok);
  }
  return true;
}
__device__ __forceinline__ bool wait_warp(const uint64_t& bar, uint32_t parity, int* abort,
                                          uint32_t* err) {
  return wait_bar(smem_u32(&bar), parity, abort, err);
}

// The cache tiles that rows at positions [p0, p0 + n) see: their number and the first.
__device__ __forceinline__ int tiles_seen(int p0, int n, int cap, int window, int& first) {
  const int hi = min(p0 + n, cap), lo = window ? max(0, p0 - window + 1) : 0;
  first = 0;
  if (n <= 0 || hi <= lo) return 0;
  first = lo / kN;
  return (hi + kN - 1) / kN - first;
}
// Those of tile t of an item within this CTA's piece: [b, e).
template <int HD, bool KV8>
__device__ __forceinline__ void tile_range(const ChunkArgs& a, const Item& it, int t, int& b, int& e) {
  const int skip = (t - it.tile) * a.TB;
  const int n = tiles_seen(it.pos0 + skip, skip < 0 ? 0 : min(it.ntok - skip, a.TB), it.cap,
                           a.window, b);
  e = b + n;
  b = max(b, it.kv0);
  e = min(e, it.kv0 + it.kvn);
  if (e < b) e = b;
}

// ---- scheduler ----
struct Seq {
  int t0, n, pos, cap;  // first row, rows, position of the first, positions to see
};
__device__ __forceinline__ Seq sequence(const ChunkArgs& a, int i) {
  Seq s{0, 0, 0, 0};
  if (i < a.S) {
    int t1;
    rows_of(a, i, s.t0, t1);
    s.n = t1 - s.t0;
    const int len = min(max(a.seq_lens[i], 0), kMaxPosition);
    s.pos = len - s.n;
    s.cap = min(len, a.table_span);
  }
  return s;
}
// An item's units: its cache tiles (one at least: an item that sees nothing still writes its
// zeros), then kItemUnits for what it costs besides them.
__device__ __forceinline__ int item_units(const ChunkArgs& a, const Seq& s, int m, int tokens,
                                          int& first, int& tiles) {
  tiles = tiles_seen(s.pos + m * tokens, min(tokens, s.n - m * tokens), s.cap, a.window, first);
  return max(tiles, 1) + kItemUnits;
}
// Units of one KV head of every lane's sequence.
__device__ __forceinline__ int head_units(const ChunkArgs& a, const Seq& s, int tokens,
                                                int lane) {
  const int items = (s.n + tokens - 1) / tokens;
  int u = 0, first, tiles;
  if (items <= 4)
#pragma unroll 1
    for (int m = 0; m < items; ++m) u += item_units(a, s, m, tokens, first, tiles);
  uint32_t big = __ballot_sync(0xffffffffu, items > 4);
  while (big) {  // long sequences: the warp shares the items
    const int src = __ffs(big) - 1;
    big &= big - 1;
    Seq o;
    o.t0 = 0;
    o.n = __shfl_sync(0xffffffffu, s.n, src);
    o.pos = __shfl_sync(0xffffffffu, s.pos, src);
    o.cap = __shfl_sync(0xffffffffu, s.cap, src);
    int sum = 0;
    for (int m = lane; m * tokens < o.n; m += 32) sum += item_units(a, o, m, tokens, first, tiles);
    sum = __reduce_add_sync(0xffffffffu, sum);
    if (lane == src) u = sum;
  }
  return u;
}
__device__ __forceinline__ int scan_add(int x, int lane) {  // inclusive
#pragma unroll 1
  for (int k = 1; k < 32; k <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, k);
    if (lane >= k) x += y;
  }
  return x;
}

// A CTA's units [u0, u1), of `per` a CTA: its first item is number m of KV head kvh of sequence
// seq, from its unit off on.
struct Piece {
  int u0, u1, per, seq, kvh, m, off;
};
template <int HD, bool KV8>
__device__ Piece find_piece(const ChunkArgs& a, int lane) {
  const int tokens = Shape<HD, KV8>::kTiles * a.TB, cta = blockIdx.x;
  int total = 0, mine = 0;
  for (int base = 0; base < a.S; base += 32) {
    const int i = base + lane;
    // rows that two sequences own, or that are not there: nothing is done (nor do the units, 32
    // bits for disjoint rows, overflow)
    const bool broken = i < a.S && (a.query_start[i] < 0 || a.query_start[i + 1] > a.T ||
                                    a.query_start[i] > a.query_start[i + 1]);
    if (__any_sync(0xffffffffu, broken)) {
      if (cta == 0 && lane == 0) atomicOr(a.err, DORY_DEVERR_QUERY_START);
      total = 0;
      break;
    }
    mine = head_units(a, sequence(a, i), tokens, lane) * a.NKV;
    total += __reduce_add_sync(0xffffffffu, mine);
  }
  const int per = max((total + int(gridDim.x) - 1) / int(gridDim.x), 1);
  const int u0 = min(cta * per, total), u1 = min(u0 + per, total);
  Piece p{u0, u1, per, 0, 0, 0, 0};
  if (u0 < u1) {
    // the sequence, KV head and item that hold unit u0
    int before = 0, seq = 0;
    for (int base = 0; base < a.S; base += 32) {
      if (a.S > 32) mine = head_units(a, sequence(a, base + lane), tokens, lane) * a.NKV;
      const int upto = before + scan_add(mine, lane);
      const uint32_t past = __ballot_sync(0xffffffffu, upto > u0);
      if (past) {
        const int src = __ffs(past) - 1;
        before = __shfl_sync(0xffffffffu, upto - mine, src);
        seq = base + src;
        break;
      }
      before = __shfl_sync(0xffffffffu, upto, 31);
    }
    const Seq s = sequence(a, seq);
    const int per_head =
        __shfl_sync(0xffffffffu, head_units(a, lane ? Seq{0, 0, 0, 0} : s, tokens, lane), 0);
    int rest = u0 - before;
    int kvh = rest / per_head, m = 0;
    rest -= kvh * per_head;
    int first, tiles;
    for (int base = 0;; base += 32) {
      const bool real = (base + lane) * tokens < s.n;
      const int u = real ? item_units(a, s, base + lane, tokens, first, tiles) : 0;
      const int upto = scan_add(u, lane);
      const uint32_t past = __ballot_sync(0xffffffffu, upto > rest);
      if (past) {
        const int src = __ffs(past) - 1;
        rest -= __shfl_sync(0xffffffffu, upto - u, src);
        m = base + src;
        break;
      }
      rest -= __shfl_sync(0xffffffffu, upto, 31);
      if ((base + 32) * tokens >= s.n) break;  // not reached: rest lies within the head
    }
    p.seq = seq;
    p.kvh = kvh;
    p.m = m;
    p.off = rest;
  }
  return p;
}

// The parts of items that make up a piece, in order: f(item, its cache tiles or 1, its first unit's
// number), until it returns false.
template <int HD, bool KV8, class F>
__device__ __forceinline__ void walk(const ChunkArgs& a, const Piece& p, F f) {
  const int tokens = Shape<HD, KV8>::kTiles * a.TB, cta = blockIdx.x;
  if (p.u0 >= p.u1) return;
  const int u1 = p.u1;
  int seq = p.seq, kvh = p.kvh, m = p.m, off = p.off, turn = 0, first, tiles;
  Seq s = sequence(a, seq);
#pragma unroll 1
  for (int at = p.u0; at < u1;) {
    const int units = item_units(a, s, m, tokens, first, tiles);
    const int take = min(units - off, u1 - at);
    const int work = units - kItemUnits;  // cache tiles, or 1
    if (off < work) {
      Item it;
      it.flags = 0;
      it.kv0 = first + off;
      it.kvn = tiles ? min(take, work - off) : 0;
      it.tok0 = s.t0 + m * tokens;
      it.ntok = min(tokens, s.n - m * tokens);
      it.pos0 = s.pos + m * tokens;
      it.kvh = kvh;
      it.seq = seq;
      it.cap = s.cap;
      it.slot = off == 0 ? (take >= work ? -1 : 2 * cta + 1) : 2 * cta;
      // items of one tile's rows take the two in turn: one's output overlaps the next one
      it.tile = Shape<HD, KV8>::kTiles == 2 && it.ntok <= a.TB ? turn ^= 1 : 0;
      if (!f(it, work, at)) return;
    }
    at += take;
    off = 0;
    if (++m * tokens >= s.n) {
      m = 0;
      if (++kvh == a.NKV) {
        kvh = 0;
        if (at < u1) do s = sequence(a, ++seq); while (s.n == 0 && seq < a.S);
      }
    }
  }
}

// What a CTA leaves to the join kernel: the item whose first part ends its piece, and whether a
// row of an item that it holds whole came out non-finite from finite weights.
struct Join {
  int32_t parts, tok0, ntok, kvh;  // parts: CTAs that hold one; 0: no item
  int32_t odd, seq, pos0, cap;
};

template <int HD, bool KV8>
__device__ void plan_role(const ChunkArgs& a, Control<HD, KV8>& c, const Piece& p, int lane) {
  const int cta = blockIdx.x;
  Join* const join = reinterpret_cast<Join*>(a.joins) + cta;
  // Before anything can give up: the join must not find an earlier call's record.
  if (lane == 0) join->parts = join->odd = 0;
  int queued = 0;
  auto push = [&](const Item& it) {
    const int at = queued % kQueue;
    if (queued >= kQueue &&
        !wait_warp(c.item_empty[at], (queued / kQueue - 1) & 1, &c.abort, a.err))
      return false;
    if (lane == 0) {
      c.items[at] = it;
      mbar_arrive(smem_u32(&c.item_full[at]));
    }
    __syncwarp();
    ++queued;
    return true;
  };
  bool ok = true;
  walk<HD, KV8>(a, p, [&](const Item& it, int work, int at) {
    if (it.slot == 2 * cta + 1 && lane == 0) {
      join->parts = (at + work - 1) / p.per - cta + 1;
      join->tok0 = it.tok0;
      join->ntok = it.ntok;
      join->kvh = it.kvh;
      join->seq = it.seq;
      join->pos0 = it.pos0;
      join->cap = it.cap;
    }
    return ok = push(it);
  });
  if (!ok) return;
  if (cta == 0)  // lengths beyond the block table
    for (int i = lane; i < a.S; i += 32)
      if (a.seq_lens[i] > a.table_span && sequence(a, i).n) atomicOr(a.err, DORY_DEVERR_BLOCK_OOB);
  Item end;
  memset(&end, 0, sizeof(end));
  end.flags = kItemEnd;
  push(end);
}

// ---- loader ----
// What ring stage q of an item's n tiles holds.  Stages are used in the order K0 V0 K1 V1 ..;
// with 256-dim heads (two stages a tile, and K of the next tile wanted before V of this one)
// K0 K1 V0 K2 V1 .. Vn-1.
template <int HD, bool KV8>
__device__ __forceinline__ void stage_holds(int q, int n, bool& is_v, int& tile, int& half) {
  if (Shape<HD, KV8>::kTiles == 2) {
    is_v = q & 1;
    tile = q >> 1;
    half = 0;
    return;
  }
  const int r = q - 2, step = r >> 2;  // K of tile step + 1, then V of tile step
  half = q & 1;
  is_v = r >= 0 && (r & 2 || step + 1 >= n);
  tile = r < 0 ? 0 : is_v ? step : step + 1;
}
// The first stage of V of tile i.
template <int HD, bool KV8>
__device__ __forceinline__ uint32_t stage_of_v(int i, int n) {
  if (Shape<HD, KV8>::kTiles == 2) return 2 * i + 1;
  return i + 1 < n ? 4 * i + 4 : 4 * i + 2;
}

template <int HD, bool KV8>
__device__ void load_role(const ChunkArgs& a, const Maps& maps, Control<HD, KV8>& c, uint32_t tiles,
                          int part, int lane) {
  using Sh = Shape<HD, KV8>;
  // the ring the copies go to: the products' own, or the bytes' that wait for conversion
  constexpr int kRing = KV8 ? Sh::kRawStages : Sh::kStages;
  constexpr int kBytes = KV8 ? Sh::kRawBytes : Sh::kStageBytes;
  constexpr int kBoxes = KV8 ? 1 : Sh::kCols / 64;  // 128-byte boxes across a row
  // Two warps share a stage's copies: a box each of a row's two.
  constexpr int kOwnBoxes = kBoxes / Sh::kLoaders;
  static_assert(kOwnBoxes >= 1, "a box a warp");
  const uint32_t stages = tiles + Sh::kQBytes + (KV8 ? Sh::kStages * Sh::kStageBytes : 0);
  uint64_t* const full = KV8 ? c.raw_full : c.kv_full;
  uint64_t* const empty = KV8 ? c.raw_empty : c.kv_empty;
  const int copies = kN / a.copy_rows;
  int stage = 0, queued = 0, q_uses[2] = {0, 0};
  uint32_t phase = 1, tile_no = 0, issued = 0;  // phase of the stage's empty barrier: free at first
  bool ok = true;
  for (;;) {
    const int at = queued % kQueue;
    if (!(ok = wait_warp(c.item_full[at], (queued / kQueue) & 1, &c.abort, a.err))) break;
    const Item it = c.items[at];
    __syncwarp();
    if (elect_one()) mbar_arrive(smem_u32(&c.item_empty[at]));
    ++queued;
    if (uniform(it.flags) & kItemEnd) break;
    const int kvn = uniform(it.kvn), kv0 = uniform(it.kv0), kvh = uniform(it.kvh);
    if (!kvn) continue;
    const int lo = a.window ? max(0, it.pos0 - a.window + 1) : 0;
    const int hi = min(it.pos0 + it.ntok, it.cap);
    const int32_t* table = a.tables + int64_t(it.seq) * a.table_stride;
    // Lane x's copy of stage q: its block, or one beyond the cache, which loads as zeros.
    auto look_up = [&](int q, bool& bad) {
      bool is_v;
      int tile, half;
      stage_holds<HD, KV8>(q, kvn, is_v, tile, half);
      const int pos = (kv0 + tile) * kN + lane * a.copy_rows;
      int id = int(a.blocks);
      bad = false;
      if (lane < copies && tile < kvn && pos < hi && pos + a.copy_rows > lo) {
        const int entry = table[pos / a.B];
        bad = entry < 0 || entry >= a.blocks;
        if (!bad) id = entry;
      }
      return id;
    };
    bool bad;
    int id = look_up(0, bad);
    if (part == 0) {  // the queries
      const int tok0 = uniform(it.tok0), first = uniform(it.tile);
      const int end = first + uniform(it.tiles(a));
#pragma unroll
      for (int t = 0; t < Sh::kTiles; ++t) {
        if (t < first || t >= end) continue;
        if (!(ok = wait_warp(c.q_empty[t], (q_uses[t] & 1) ^ 1, &c.abort, a.err))) break;
        ++q_uses[t];
        if (elect_one()) {
          const uint32_t bar = smem_u32(KV8 ? &c.q_raw[t] : &c.q_full[t]);
          mbar_expect(bar, (HD / 64) * a.TB * a.G * 128);
#pragma unroll 1
          for (int k = 0; k < HD / 64; ++k)
            tma_load_3d(tiles + (t * (HD / 64) + k) * kChunkBytes, &maps.q, 64 * k, kvh * a.G,
                        tok0 + (t - first) * a.TB, bar);
        }
        __syncwarp();
      }
      if (!ok) break;
    }
#pragma unroll 1
    for (int q = 0; q < 2 * Sh::kHalves * kvn; ++q) {
      bool is_v;
      int tile, half;
      stage_holds<HD, KV8>(q, kvn, is_v, tile, half);
      if (part == 0 && !is_v && half == 0) {
        const uint32_t mask = __ballot_sync(0xffffffffu, bad);
        if (elect_one()) {
          c.bad[tile_no % kBadRing] = mask;
          if (mask) atomicOr(a.err, DORY_DEVERR_BLOCK_OOB);
        }
        __syncwarp();
        ++tile_no;
      }
      const int own = id;
      id = look_up(q + 1, bad);  // in flight while this stage's copies are issued
      const uint32_t bar = smem_u32(&full[stage]);
      const uint32_t dst = stages + stage * kBytes;
      const CUtensorMap* map = is_v ? &maps.v : &maps.k;
      // Every copy's block in registers first, then one elected run of copies: 28 clocks a copy
      // of 2 KB; a loop that fetches each block as it goes took 47, a copy a lane 66.
      int block[kN / 16], row[kN / 16];
#pragma unroll
      for (int x = 0; x < kN / 16; ++x) {
        block[x] = __shfl_sync(0xffffffffu, own, x);
        row[x] = 0;
      }
      if (a.copy_rows != a.B) {
        int r = (kv0 + tile) * kN % a.B;
#pragma unroll
        for (int x = 0; x < kN / 16; ++x) {
          row[x] = r;
          r += a.copy_rows;  // which divides both the tile and the page
          if (r == a.B) r = 0;
        }
      }
      if (!(ok = wait_warp(empty[stage], phase, &c.abort, a.err))) break;
      if (elect_one()) {
        mbar_expect(bar, kBytes / Sh::kLoaders);
#pragma unroll
        for (int x = 0; x < kN / 16; ++x) {
          if (x < copies)
#pragma unroll
            for (int k = 0; k < kOwnBoxes; ++k) {
              const int box = part * kOwnBoxes + k;
              tma_load_4d(dst + box * kChunkBytes + x * a.copy_rows * 128, map,
                          half * Sh::kCols + 64 * box, row[x], kvh, block[x], bar);
            }
        }
      }
      __syncwarp();
      ++issued;
      if (++stage == kRing) {
        stage = 0;
        phase ^= 1;
      }
    }
    if (!ok) break;
  }
  if (!ok) {  // given up: no copy may land after the CTA has gone
    const long long start = clock64();
#pragma unroll 1
    for (uint32_t i = issued > kRing ? issued - kRing : 0; i < issued; ++i)
      while (!mbar_try(smem_u32(&full[i % kRing]), (i / kRing) & 1) &&
             clock64() - start < 200000000LL) {
      }
    for (int t = 0; t < Sh::kTiles; ++t)
      while (q_uses[t] &&
             !mbar_try(smem_u32(KV8 ? &c.q_raw[t] : &c.q_full[t]), (q_uses[t] - 1) & 1) &&
             clock64() - start < 300000000LL) {
      }
  }
}

// ---- conversion, FP8 caches: four warps ----
// e4m3 is exact in f16, so K and V tiles become f16 tiles.  A query row becomes f16 after a
// scaling by a power of two that puts its largest element in [2^10, 2^11): bf16's 8 bits fit
// f16's 11, and only what lies 2^24 below the row's largest element loses any.  Both together
// let the scores and the sum be f16 products, the weights rounded to 11 bits.
template <int HD, bool KV8>
__device__ void convert_role(const ChunkArgs& a, Control<HD, KV8>& c, uint32_t tiles, int thread) {
  using Sh = Shape<HD, KV8>;
  const int lane = thread & 31;
  const uint32_t stages = tiles + Sh::kQBytes, raws = stages + Sh::kStages * Sh::kStageBytes;
  // A thread converts 16 dims at a time, one 16-byte piece of bytes to two of f16, of every 16th
  // row.  Of eight lanes four take half of a row and four the other half of its neighbour, so
  // that no two of them share a bank.
  const int piece = thread & 7, own_row = (thread >> 3) ^ (piece >> 2);
  const uint32_t own_src = own_row * 128 + ((piece ^ own_row) & 7) * 16;
  const uint32_t own_dst = (piece >> 2) * kChunkBytes + own_row * 128 +
                           (((piece & 3) * 2) ^ (own_row & 7)) * 16;
  int queued = 0, raw = 0, stage = 0;
  uint32_t raw_phase = 0, phase = 1, q_phase = 0;
  for (;;) {
    const int at = queued % kQueue;
    if (!wait_warp(c.item_full[at], (queued / kQueue) & 1, &c.abort, a.err)) return;
    const Item it = c.items[at];
    const int kvn = it.kvn;
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&c.item_empty[at]));
    ++queued;
    if (it.flags & kItemEnd) return;
    if (!kvn) continue;
    const int lo = a.window ? max(0, it.pos0 - a.window + 1) : 0;
    const int hi = min(it.pos0 + it.ntok, it.cap);
#pragma unroll 1
    for (int t = it.tile; t < it.tile + it.tiles(a); ++t) {  // a row a thread, in place
      if (!wait_warp(c.q_raw[t], q_phase >> t & 1, &c.abort, a.err)) return;
      const uint32_t row = tiles + t * (HD / 64) * kChunkBytes + thread * 128;
      float top = 0.0f;
#pragma unroll 1
      for (int x = 0; x < HD / 8; ++x) {
        uint32_t w[4];
        lds128(row + x / 8 * kChunkBytes + ((x ^ thread) & 7) * 16, w);
#pragma unroll
        for (int y = 0; y < 4; ++y)
          top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[y] << 16)),
                                 fabsf(__uint_as_float(w[y] & 0xffff0000u))));
      }
      // 2^(10 - exponent), within what FP32 holds; 1 for zero, infinite and NaN rows
      const int exponent = int(__float_as_uint(top) >> 23) - 127;
      const int up = top > 0.0f && exponent < 128 ? min(10 - exponent, 126) : 0;
      const float scale = __uint_as_float(uint32_t(up + 127) << 23);
#pragma unroll 1
      for (int x = 0; x < HD / 8; ++x) {
        uint32_t w[4];
        const uint32_t piece = row + x / 8 * kChunkBytes + ((x ^ thread) & 7) * 16;
        lds128(piece, w);
#pragma unroll
        for (int y = 0; y < 4; ++y)
          w[y] = pack_f16(__uint_as_float(w[y] << 16) * scale,
                          __uint_as_float(w[y] & 0xffff0000u) * scale);
        sts128(piece, w);
      }
      c.q_scale[q_phase >> t & 1][t * kM + thread] = __uint_as_float(uint32_t(127 - up) << 23);
      q_phase ^= 1u << t;
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&c.q_full[t]));
    }
#pragma unroll 1
    for (int q = 0; q < 2 * Sh::kHalves * kvn; ++q) {
      if (!wait_warp(c.raw_full[raw], raw_phase, &c.abort, a.err)) return;
      if (!wait_warp(c.kv_empty[stage], phase, &c.abort, a.err)) return;
      const uint32_t from = raws + raw * Sh::kRawBytes, to = stages + stage * Sh::kStageBytes;
      bool is_v;
      int tile, half;
      stage_holds<HD, KV8>(q, kvn, is_v, tile, half);
      const int seen_lo = lo - (it.kv0 + tile) * kN, seen_hi = hi - (it.kv0 + tile) * kN;
      // Rows 16 apart have the same swizzle, so a step is an addition to three addresses (FP8
      // prompt of 8192: 598 us then; 618 with the addresses formed row by row, 256-dim heads 796, 872).
      const uint32_t src = from + own_src, dst = to + own_dst;
      const int own_seen = own_row - seen_lo, n_seen = max(seen_hi - seen_lo, 0);
      constexpr int kAtOnce = HD == 256 ? 4 : 2;
#pragma unroll kAtOnce
      for (int k = 0; k < kN / 16; ++k) {
        uint32_t w[4], f[8];
        lds128(src + k * 16 * 128, w);
        const bool seen = uint32_t(own_seen + 16 * k) < uint32_t(n_seen);  // by a row of the item
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          if (!seen) w[y] = 0;
          f[2 * y] = e4m3x2_to_f16x2(w[y]);
          f[2 * y + 1] = e4m3x2_to_f16x2(w[y] >> 16);
        }
        sts128(dst + k * 16 * 128, f);
        sts128((dst ^ 16) + k * 16 * 128, f + 4);
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&c.kv_full[stage]));
        mbar_arrive(smem_u32(&c.raw_empty[raw]));
      }
      if (++raw == Sh::kRawStages) {
        raw = 0;
        raw_phase ^= 1;
      }
      if (++stage == Sh::kStages) {
        stage = 0;
        phase ^= 1;
      }
    }
  }
}

// Column, within a score buffer, of the weights of positions [16 x, 16 x + 16): each warpgroup
// puts its own over the scores it has read.
template <int HD, bool KV8>
__host__ __device__ constexpr int weight_column(int x) {
  constexpr int kSteps = Shape<HD, KV8>::kScoreCols / 16;
  return x / kSteps * Shape<HD, KV8>::kScoreCols + x % kSteps * 8;
}

// ---- products ----
// One warp, and the path that paces the kernel: each of its instructions delays both tiles (the
// product loops rolled up, say, cost 17%).  So barriers are plain addresses, descriptors one
// addition a product, and what needs no wait between shares an elected block.
template <int HD, bool KV8>
__device__ bool mma_items(const ChunkArgs& a, Control<HD, KV8>& c, uint32_t tiles) {
  using Sh = Shape<HD, KV8>;
  using C = Control<HD, KV8>;
  const uint32_t tmem = uniform(c.tmem), stages = tiles + Sh::kQBytes;
  const uint32_t control = tiles + Sh::kTileBytes;
  constexpr uint32_t kScores = instruction(!KV8, false, kM, kN);
  constexpr uint32_t kSum = instruction(!KV8, true, kM, Sh::kCols);
  int stage = 0, queued = 0;
  uint32_t phase = 0, q_phase = 0, p_phase = 0, p_count = 0, buffers = 0;
#define BAR(field, i) (control + uint32_t(offsetof(C, field)) + 8 * (i))
#define WAIT(bar, parity) \
  if (!wait_bar(bar, parity, &c.abort, a.err)) return false
  auto wait_stage = [&]() { return wait_bar(BAR(kv_full, stage), phase, &c.abort, a.err); };
  auto take = [&]() {
    const int was = stage;
    if (++stage == Sh::kStages) {
      stage = 0;
      phase ^= 1;
    }
    return was;
  };
  // By the elected lane: S (+)= Q K^T over one stage's columns.
  auto scores = [&](int t, int buffer, int st, int half, bool add) {
    const uint32_t q = desc_k_major(tiles + (t * (HD / 64) + half * (Sh::kCols / 64)) * kChunkBytes);
    const uint32_t k = desc_k_major(stages + st * Sh::kStageBytes);
#pragma unroll
    for (int x = 0; x < Sh::kCols / 64; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t step = (x * kChunkBytes + 32 * y) >> 4;
        mma_ss(tmem + buffer * kN, q + step, k + step, kScores, x + y > 0 ? 1u : uint32_t(add));
      }
  };
  // By the elected lane: O += P V for a part of a tile's positions, the same part of each softmax
  // warpgroup's.
  auto sum = [&](int o_col, int buffer, int st, int part, bool add) {
    constexpr int kSteps = Sh::kPartCols / 16;
    const uint32_t weights = tmem + buffer * kN + 8 * kSteps * part;
    const uint32_t v = desc_mn_major(stages + st * Sh::kStageBytes, kChunkBytes) +
                       (part * kSteps * 16 * 128 >> 4);
#pragma unroll
    for (int i = 0; i < kSteps * Sh::kShares; ++i) {
      const int x = i / kSteps * (Sh::kScoreCols / 16) + i % kSteps;  // in part 0
      mma_ts(tmem + o_col, weights + weight_column<HD, KV8>(x), v + (x * 16 * 128 >> 4), kSum,
             part + i > 0 ? 1u : uint32_t(add));
    }
  };
  for (;;) {
    const int at = queued % kQueue;
    WAIT(BAR(item_full, at), (queued / kQueue) & 1);
    const Item it = c.items[at];
    __syncwarp();
    if (elect_one()) mbar_arrive(BAR(item_empty, at));
    ++queued;
    if (uniform(it.flags) & kItemEnd) return true;
    const int kvn = uniform(it.kvn);
    if (!kvn) continue;
    const int j0 = uniform(it.kv0), j1 = j0 + kvn;
    const int filled = uniform(((1 << it.tiles(a)) - 1) << it.tile);
#pragma unroll
    for (int t = 0; t < Sh::kTiles; ++t)
      if (filled >> t & 1) WAIT(BAR(q_full, t), q_phase >> t & 1);
    q_phase ^= filled;
    auto free_queries = [&]() {  // by the elected lane, behind the item's last scores
#pragma unroll
      for (int t = 0; t < Sh::kTiles; ++t)
        if (filled >> t & 1) mma_commit(BAR(q_empty, t));
    };
    if constexpr (Sh::kTiles == 2) {
      int b[2], e[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        tile_range<HD, KV8>(a, it, t, b[t], e[t]);
        b[t] = uniform(b[t]);
        e[t] = uniform(e[t]);
      }
      if (!wait_stage()) return false;
      tc_fence_after();
      int k_st = take();
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (b[t] <= j0 && j0 < e[t]) {
            scores(t, t, k_st, 0, false);
            mma_commit(BAR(s_full, t));
          }
        mma_commit(BAR(kv_empty, k_st));
        if (j0 + 1 == j1) free_queries();
      }
      for (int j = j0; j < j1; ++j) {
        if (!wait_stage()) return false;
        const int v_st = take();
        const bool more = j + 1 < j1;
        k_st = -1;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const bool now = b[t] <= j && j < e[t];
          const bool next = more && b[t] <= j + 1 && j + 1 < e[t];
          if (now) {
#pragma unroll
            for (int part = 0; part + 1 < Sh::kParts; ++part) {
              WAIT(BAR(p_full, 2 * t + part), p_phase >> t & 1);
              tc_fence_after();
              if (elect_one()) sum(Sh::kO + t * Sh::kOStride, t, v_st, part, j > b[t]);
            }
          }
          if (next && k_st < 0) {  // ahead of the wait for the last weights
            if (!wait_stage()) return false;
            k_st = take();
          }
          if (now) {
            WAIT(BAR(p_full, 2 * t + Sh::kParts - 1), p_phase >> t & 1);
            p_phase ^= 1u << t;
          }
          tc_fence_after();
          if (elect_one()) {
            if (now) {
              sum(Sh::kO + t * Sh::kOStride, t, v_st, Sh::kParts - 1, j > b[t]);
              if (j + 1 == e[t]) mma_commit(BAR(o_full, t));
            }
            if (next) {
              scores(t, t, k_st, 0, false);
              mma_commit(BAR(s_full, t));
            }
          }
        }
        if (more && k_st < 0) {  // a tile of positions between the two tiles' windows
          if (!wait_stage()) return false;
          k_st = take();
        }
        if (elect_one()) {
          mma_commit(BAR(kv_empty, v_st));
          if (more) mma_commit(BAR(kv_empty, k_st));
          if (j + 2 == j1) free_queries();
        }
      }
    } else {
      auto next_scores = [&]() {
#pragma unroll
        for (int h = 0; h < Sh::kHalves; ++h) {
          if (!wait_stage()) return false;
          tc_fence_after();
          const int st = take();
          if (elect_one()) {
            scores(0, buffers & 1, st, h, h > 0);
            mma_commit(BAR(kv_empty, st));
            if (h + 1 == Sh::kHalves) mma_commit(BAR(s_full, buffers & 1));
          }
        }
        ++buffers;
        return true;
      };
      if (!next_scores()) return false;
      for (int j = j0; j < j1; ++j) {
        if (j + 1 < j1 && !next_scores()) return false;
        if (j + 2 >= j1 && (j + 2 == j1 || j0 + 1 == j1))
          if (elect_one()) free_queries();
        const int buffer = p_count & 1;
        const uint32_t parity = (p_count++ >> 1) & 1;
        int v_st[Sh::kHalves];
#pragma unroll
        for (int h = 0; h < Sh::kHalves; ++h) {
          if (!wait_stage()) return false;
          v_st[h] = take();
        }
#pragma unroll
        for (int part = 0; part < Sh::kParts; ++part) {
          WAIT(BAR(p_full, 2 * buffer + part), parity);
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int h = 0; h < Sh::kHalves; ++h) {
              sum(Sh::kO + h * Sh::kCols, buffer, v_st[h], part, j > j0);
              if (part + 1 == Sh::kParts) mma_commit(BAR(kv_empty, v_st[h]));
            }
            if (part + 1 == Sh::kParts) mma_commit(BAR(o_full, buffer));
          }
        }
      }
    }
  }
#undef WAIT
#undef BAR
}

// ---- softmax ----
// Two 16-bit gate values, in g.x, as FP32.
__device__ __forceinline__ void widen2(bool bf16, uint2& g) {
  const uint32_t w = g.x;
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w));
  g.x = bf16 ? w << 16 : __float_as_uint(h.x);
  g.y = bf16 ? w & 0xffff0000u : __float_as_uint(h.y);
}

// A bit for each of 32 columns that lies above `last` or below `first`.
__device__ __forceinline__ uint32_t outside(int last, int first) {
  const uint32_t above = last < 0 ? 0xffffffffu : last >= 31 ? 0u : 0xfffffffeu << last;
  const uint32_t below = first <= 0 ? 0u : first >= 32 ? 0xffffffffu : (1u << first) - 1u;
  return above | below;
}
// A bit for each of the 32 columns from `col` that belongs to a copy with a bad block id.
__device__ __forceinline__ uint32_t bad_columns(uint32_t bad, int col, int copy_shift) {
  return (bad >> (col >> copy_shift) & 1 ? 0x0000ffffu : 0u) |
         (bad >> ((col + 16) >> copy_shift) & 1 ? 0xffff0000u : 0u);
}

template <int HD, bool KV8>
__device__ void softmax_role(const ChunkArgs& a, Control<HD, KV8>& c, uint32_t tiles, int warp, int lane) {
  using Sh = Shape<HD, KV8>;
  constexpr bool kTwo = Sh::kTiles == 2;
  const int quad = warp & 3, row = quad * 32 + lane;
  const int t = (warp >> 2) / Sh::kShares, share = (warp >> 2) % Sh::kShares;
  // The warps that share rows, of one tile: a wait like any other, so that one of them can give up
  // (a block barrier would keep the other for good).
  uint32_t met = 0;
  auto meet = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(&c.met[t * 4 + quad]));
    met ^= 1;
    return wait_warp(c.met[t * 4 + quad], met ^ 1, &c.abort, a.err);
  };
  const uint32_t tmem = c.tmem + (uint32_t(quad * 32) << 16);
  const uint32_t o_addr = tmem + Sh::kO + t * Sh::kOStride + share * Sh::kOutCols;
  const uint32_t stages = tiles + Sh::kQBytes;
  const int row_tok = row / a.G, row_head = row - row_tok * a.G;
  const bool row_real = row < a.TB * a.G;
  int queued = 0;
  uint32_t scored = 0, summed = 0, tiles_seen_before = 0, stage_no = 0, q_set = 0;
  // The last sum given to the tensor cores is complete.  A parity can only be asked for with one
  // phase of its barrier outstanding.  Two tiles: a phase an item.  256-dim heads: a phase a
  // tile, on two barriers in turn, because scores j only vouch for the sum of tile j - 2.
  auto wait_sum = [&]() {
    const uint32_t last = summed - 1;
    return kTwo ? wait_warp(c.o_full[t], last & 1, &c.abort, a.err)
                : wait_warp(c.o_full[last & 1], (last >> 1) & 1, &c.abort, a.err);
  };
  for (;;) {
    const int at = queued % kQueue;
    if (!wait_warp(c.item_full[at], (queued / kQueue) & 1, &c.abort, a.err)) return;
    // left in shared memory: what the loop over the tiles does not use would only hold registers
    const Item& it = c.items[at];
    if (it.flags & kItemEnd) return;
    int b, e;
    tile_range<HD, KV8>(a, it, t, b, e);
    const int tok = (t - it.tile) * a.TB + row_tok;
    const bool live = row_real && tok >= 0 && tok < it.ntok;
    const bool warp_live = __any_sync(0xffffffffu, live);
    const int pos = it.pos0 + tok;
    const int see_hi = min(pos, it.cap - 1), see_lo = a.window ? max(0, pos - a.window + 1) : 0;
    if (live && a.gate && it.slot < 0) {  // the gate's row, wanted at the end
      const int size = a.gate_dtype == DORY_DTYPE_F32 ? 4 : 2;
      const char* at_gate =
          static_cast<const char*>(a.gate) +
          ((it.tok0 + tok) * a.gate_t + int64_t(it.kvh * a.G + row_head) * HD + share * Sh::kOutCols) * size;
      for (int x = 0; x < Sh::kOutCols * size; x += 128)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(at_gate + x));
    }
    // the tiles with positions before the first or behind the last that the item sees
    const int item_lo = a.window ? max(0, it.pos0 - a.window + 1) : 0;
    const int item_hi = min(it.pos0 + it.ntok, it.cap);
    const int ragged_lo = item_lo % kN ? item_lo / kN : -1;
    const int ragged_hi = item_hi > 0 && item_hi % kN ? item_hi / kN : -1;
    float sl = a.scale_log2, slack = kSlack / a.scale_log2;
    float m = -INFINITY, l = 0.0f;
    for (int j = b; j < e; ++j) {
      const int buffer = kTwo ? t : int(scored & 1);
      const uint32_t s_addr = tmem + buffer * kN;
      if (!wait_warp(c.s_full[buffer], kTwo ? scored & 1 : (scored >> 1) & 1, &c.abort, a.err))
        return;
      tc_fence_after();
      if (KV8 && j == b && live) {  // there since the first scores: they needed the queries
        sl = a.scale_log2 * a.k_scale * c.q_scale[q_set][t * kM + row];
        slack = kSlack / sl;
      }
      const uint32_t bad = c.bad[(tiles_seen_before + (j - it.kv0)) % kBadRing];
      // 256-dim heads: a warp may already be a tile ahead of another, so a barrier a buffer
      auto ready = [&](int part) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&c.p_full[buffer][part]));
      };
      // V rows of this tile that no row of the item sees, in copies that hold others it does
      if (!KV8 && (j == ragged_lo || j == ragged_hi)) {  // (FP8: the conversion sees to it)
        const int z_lo = (a.window ? max(0, it.pos0 - a.window + 1) : 0) - j * kN;
        const int z_hi = min(it.pos0 + it.ntok, it.cap) - j * kN;
        const int i = j - it.kv0;  // the tile's place in the piece, and so its V stages
        const uint32_t v_no = stage_no + stage_of_v<HD, KV8>(i, it.kvn);
        const int r1 = z_lo > 0 ? (z_lo & ~(a.copy_rows - 1)) : 0, r2 = max(z_lo, 0);
        const int r3 = min(z_hi, kN), r4 = (r3 + a.copy_rows - 1) & ~(a.copy_rows - 1);
        for (int h = 0; h < Sh::kHalves; ++h) {
          const uint32_t no = v_no + h;
          const int st = no % Sh::kStages;
          if (!wait_warp(c.kv_full[st], (no / Sh::kStages) & 1, &c.abort, a.err)) return;
          constexpr int kPieces = Sh::kCols / 8;  // 16-byte pieces of a row
          const int rows = (r2 - r1) + (r4 - r3);
          for (int x = (share * 4 + quad) * 32 + lane; x < rows * kPieces; x += Sh::kShares * 128) {
            int r = x / kPieces;
            const int piece = x % kPieces;
            r = r < r2 - r1 ? r1 + r : r3 + (r - (r2 - r1));
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             stages + st * Sh::kStageBytes + (piece / 8) * kChunkBytes + r * 128 +
                             (piece % 8) * 16),
                         "r"(0)
                         : "memory");
          }
        }
        fence_async_smem();
      }
      if (!warp_live) {
        for (int part = 0; part < Sh::kParts; ++part) ready(part);
      } else {
        const uint32_t own_scores = s_addr + share * Sh::kScoreCols;
        const int base = j * kN + share * Sh::kScoreCols;
        const int last = see_hi - base, first = see_lo - base;
        const bool edge = bad || __any_sync(0xffffffffu,
                                            live && (last < Sh::kScoreCols - 1 || first > 0));
        // scores x .. x + 31 of the row: asked for, and there, the hidden ones -infinity
        auto ask_scores = [&](int x, float* s) {
          tmem_ld32(own_scores + x, reinterpret_cast<uint32_t*>(s));
        };
        auto get_scores = [&](int x, float* s) {
          tmem_wait_ld32(reinterpret_cast<uint32_t*>(s));
          if (edge) {
            uint32_t hide = outside(last - x, first - x);
            if (bad) hide |= bad_columns(bad, share * Sh::kScoreCols + x, a.copy_shift);
#pragma unroll
            for (int y = 0; y < 32; ++y)
              if (hide >> y & 1) s[y] = -INFINITY;
          }
        };
        float mt = -INFINITY;
        if (!edge) {  // all columns on their way at once
          float s[Sh::kScoreCols], top[4];
#pragma unroll
          for (int x = 0; x < Sh::kScoreCols; x += 32)
            ask_scores(x, s + x);
          tmem_wait_ld32(reinterpret_cast<uint32_t*>(s));
#pragma unroll
          for (int x = 32; x < Sh::kScoreCols; x += 32) tmem_more32(reinterpret_cast<uint32_t*>(s + x));
#pragma unroll
          for (int x = 0; x < 4; ++x) top[x] = max3(s[3 * x], s[3 * x + 1], s[3 * x + 2]);
#pragma unroll
          for (int x = 12; x < Sh::kScoreCols; x += 2)
            top[x / 2 & 3] = max3(top[x / 2 & 3], s[x], s[x + 1]);
          mt = max2(max2(top[0], top[1]), max2(top[2], top[3]));
        } else {
#pragma unroll 1
          for (int x = 0; x < Sh::kScoreCols; x += 32) {
            float s[32];
            ask_scores(x, s);
            get_scores(x, s);
#pragma unroll
            for (int y = 0; y < 32; y += 2) mt = max3(mt, s[y], s[y + 1]);
          }
        }
        if constexpr (Sh::kShares > 1) {  // the rest of the row's columns
          c.swap[t][share][row] = mt;
          if (!meet()) return;
#pragma unroll
          for (int x = 1; x < Sh::kShares; ++x) mt = max2(mt, c.swap[t][(share + x) % Sh::kShares][row]);
          if (!kTwo && !meet()) return;  // a warp may go on to the next tile while another still reads
        }
        if (j == b) {
          m = mt;
        } else if (__any_sync(0xffffffffu, live && !(mt <= m + slack))) {  // NaN too
          // (a row that is none holds whatever was in shared memory: it must not decide)
          const float grown = max2(m, mt);
          const float f = m == -INFINITY ? 0.0f : exp2_approx((m - grown) * sl);
          l *= f;
          m = grown;
          if (!kTwo) {  // the sum over the tile before may still be running
            if (!wait_sum()) return;
            tc_fence_after();
          }
#pragma unroll 1
          for (int x = 0; x < Sh::kOutCols; x += 32) {
            uint32_t o[32];
            tmem_ld32(o_addr + x, o);
            tmem_wait_ld32(o);
#pragma unroll
            for (int y = 0; y < 32; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * f);
            tmem_st32(o_addr + x, o);
          }
          tmem_wait_st();
        }
        // +inf gives NaN, as inf - inf would in every weight
        const float ref = m == -INFINITY ? 0.0f : fmaf(m, sl, m - m) - Sh::kLift;
        const uint64_t sl2 = pair(sl, sl), ref2 = pair(-ref, -ref);
        uint64_t sums[2] = {0, 0};
        // The scores are read again, a piece at a time: a loop, not 128 unrolled columns, because
        // the instructions of a straight run have to come from L2 time and again.
#pragma unroll 1
        for (int x = 0; x < Sh::kScoreCols; x += 32) {
          float s[32];
          uint32_t p[16];
          ask_scores(x, s);
          get_scores(x, s);
#pragma unroll
          for (int y = 0; y < 32; y += 2) {
            const uint64_t z = fma2(pair(s[y], s[y + 1]), sl2, ref2);
            float p0, p1;
            if (y / 2 % 4 < Sh::kPolyOf4) {
              exp2_poly2(z, p0, p1);
            } else {
              split(z, p0, p1);
              p0 = exp2_approx(p0);
              p1 = exp2_approx(p1);
            }
            sums[y / 2 & 1] = add2(sums[y / 2 & 1], pair(p0, p1));
            p[y / 2] = KV8 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
          }
          tmem_st16(own_scores + x / 2, p);
          if (Sh::kParts > 1 && x + 32 == Sh::kPartCols) {
            tmem_wait_st();
            ready(0);
          }
        }
        float l0, l1;
        split(add2(sums[0], sums[1]), l0, l1);
        l += l0 + l1;
        tmem_wait_st();
        ready(Sh::kParts - 1);
      }
      ++scored;
      if (!kTwo) ++summed;
    }
    tiles_seen_before += it.kvn;
    q_set ^= it.kvn > 0 && t >= it.tile && t < it.tile + it.tiles(a);  // the tile had queries
    stage_no += 2 * Sh::kHalves * it.kvn;

    // the item's rows
    if (e > b) {
      if (kTwo) ++summed;
      if (!wait_sum()) return;
      tc_fence_after();
    }
    auto done = [&]() {  // with the item
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&c.item_empty[at]));
      ++queued;
    };
    if (!warp_live) {
      done();
      continue;
    }
    if constexpr (Sh::kShares > 1) {
      // the sums of the shares; each warp is past its last tile's maxima: the sum just waited for
      // needed every share's weights
      c.swap[t][share][row] = l;
      if (!meet()) return;
#pragma unroll
      for (int x = 1; x < Sh::kShares; ++x) l += c.swap[t][(share + x) % Sh::kShares][row];
      if (!meet()) return;
    }
    // Opaque here, or the compiler computes everything below that depends on them alone once,
    // ahead of the items, and spills it across the loop over the tiles.
    int own_lane = lane, own_row = (t - it.tile) * kM + row, col0 = share * Sh::kOutCols;
    asm volatile("" : "+r"(own_lane), "+r"(own_row), "+r"(col0));
    const float inv = l == 0.0f ? 0.0f : (KV8 ? a.v_scale : 1.0f) / l;
    const bool whole = it.slot < 0, gated = whole && a.gate;
    // O is read as product fragments: a lane has two columns of four rows, four lanes eight
    // columns side by side, so every load of the gate and store covers whole 32-byte sectors
    // (after neighbours have exchanged halves of their packed columns).  A row a thread takes
    // 32 lines an instruction: 20,500 clocks an item with an FP32 gate.
    const int quarter = own_lane & 3;
    const int where = row_head << 16 | tok;  // tok < 256
    uint64_t row_inv[4], odd[4];             // odd: NaN once a value of the row is not finite
    int64_t out_at[4];
    const char* gate_at[4];
    uint32_t alive = 0;
    const uint32_t lives = __ballot_sync(0xffffffffu, live);
    const int gate_size = a.gate_dtype == DORY_DTYPE_F32 ? 4 : 2;
#pragma unroll
    for (int r = 0; r < 4; ++r) {  // rows 8 r + lane / 4
      const int own = 8 * r + (own_lane >> 2);
      const bool there = lives >> own & 1;
      const int src = there ? own : __ffs(lives) - 1;  // any row's gate may be read in its place
      const int w = __shfl_sync(0xffffffffu, where, src);
      const float f = whole ? __shfl_sync(0xffffffffu, inv, src) : 1.0f;
      row_inv[r] = pair(f, f);
      alive |= uint32_t(there) << r;
      const int64_t token = it.tok0 + (w & 0xffff);
      const int64_t column = int64_t(it.kvh * a.G + (w >> 16)) * HD + col0;
      out_at[r] = whole ? token * a.out_t + column
                        : (int64_t(it.slot) * Sh::kItemRows + own_row - own_lane + src) * HD + col0;
      gate_at[r] = static_cast<const char*>(a.gate) +
                   (token * a.gate_t + column + 2 * quarter) * gate_size;
      odd[r] = 0;
    }
    // Code of its own for each type of gate (its elements' bytes; 0: none), without a test or a
    // branch in it (1024 single tokens: 308 us, 356 with them; prompt of 8192: 545, 558).  The
    // gate is asked for a piece ahead; two pieces cost more code than they save waiting.
    auto output = [&](auto bytes) {
      constexpr int kBytes = bytes.value;
      uint2 g[4][4];
      auto ask_gate = [&]() {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (kBytes == 4) g[r][i] = *reinterpret_cast<const uint2*>(gate_at[r] + 32 * i);
            if (kBytes == 2) g[r][i].x = *reinterpret_cast<const uint32_t*>(gate_at[r] + 16 * i);
          }
          gate_at[r] += 32 * kBytes;
        }
      };
      if (kBytes) ask_gate();
#pragma unroll 1
      for (int x = 0; x < Sh::kOutCols; x += 32) {
        float o[32];  // row r's columns 8 i + 2 quarter + y at 16 (r / 2) + 4 i + 2 (r % 2) + y
#pragma unroll
        for (int y = 0; y < 32; ++y) o[y] = 0.0f;
        if (e > b) {
          tmem_ld_fragment(o_addr + x, reinterpret_cast<uint32_t*>(o));
          tmem_ld_fragment(o_addr + (16u << 16) + x, reinterpret_cast<uint32_t*>(o + 16));
        }
        tmem_wait_ld32(reinterpret_cast<uint32_t*>(o));
        uint64_t v[4][4];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float* at_o = o + 16 * (r / 2) + 4 * i + 2 * (r % 2);
            v[r][i] = pair(at_o[0], at_o[1]);
            odd[r] = fma2(v[r][i], 0, odd[r]);
            if (whole) v[r][i] = mul2(v[r][i], row_inv[r]);
            if (kBytes == 2) widen2(a.gate_dtype == DORY_DTYPE_BF16, g[r][i]);
            if (kBytes)
              v[r][i] = mul2(v[r][i], pair(__uint_as_float(g[r][i].x), __uint_as_float(g[r][i].y)));
          }
        if (kBytes && x + 32 < Sh::kOutCols) ask_gate();
        if (kBytes || whole) {
          const bool second = quarter & 1;  // of two neighbours: takes the odd eights
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v0, v1;
              split(v[r][i], v0, v1);
              w[i] = pack_bf16(v0, v1);
            }
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const uint32_t got = __shfl_xor_sync(0xffffffffu, second ? w[i] : w[i + 1], 1);
              if (alive >> r & 1)
                *reinterpret_cast<uint2*>(a.out + out_at[r] + x + 8 * (i + second) +
                                          4 * (quarter >> 1)) =
                    second ? make_uint2(got, w[i + 1]) : make_uint2(w[i], got);
            }
          }
        } else {
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float v0, v1;
              split(v[r][i], v0, v1);
              if (alive >> r & 1)
                *reinterpret_cast<float2*>(a.part_o + out_at[r] + x + 8 * i + 2 * quarter) =
                    make_float2(v0, v1);
            }
        }
      }
    };
    if (!gated) output(std::integral_constant<int, 0>());
    else if (gate_size == 4) output(std::integral_constant<int, 4>());
    else output(std::integral_constant<int, 2>());
    __syncwarp();
    const int64_t slot_row = int64_t(max(it.slot, 0)) * Sh::kItemRows + own_row;
    if (live && !whole && share == 0)
      a.part_ml[slot_row] = make_float2(m == -INFINITY ? 0.0f : m * sl - Sh::kLift, l);
    if (whole) {  // (parts: the join kernel sees for itself)
      bool again = false;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float odd0, odd1;
        split(odd[r], odd0, odd1);
        const float sum = __shfl_sync(0xffffffffu, l, 8 * r + (own_lane >> 2));
        again |= (isnan(odd0) || isnan(odd1)) && (alive >> r & 1) && isfinite(sum);
      }
      if (__any_sync(0xffffffffu, again) && lane == 0)
        reinterpret_cast<Join*>(a.joins)[blockIdx.x].odd = 1;
    }
    done();
  }
}

template <int HD, bool KV8>
__global__ void __launch_bounds__(Shape<HD, KV8>::kThreads, 1)
    chunk_kernel(const __grid_constant__ ChunkArgs a, const __grid_constant__ Maps maps) {
  using Sh = Shape<HD, KV8>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Control<HD, KV8>& c = *reinterpret_cast<Control<HD, KV8>*>(smem + Sh::kTileBytes);
  const uint32_t tiles = smem_u32(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_launch();
  if (threadIdx.x == 0) {
    for (int i = 0; i < Sh::kStages; ++i) {
      mbar_init(smem_u32(&c.kv_full[i]), KV8 ? Sh::kConvertWarps : Sh::kLoaders);
      mbar_init(smem_u32(&c.kv_empty[i]), 1);
    }
    for (int i = 0; i < Sh::kRawStages; ++i) {
      mbar_init(smem_u32(&c.raw_full[i]), 1);
      mbar_init(smem_u32(&c.raw_empty[i]), Sh::kConvertWarps);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&c.q_raw[i]), 1);
      mbar_init(smem_u32(&c.q_full[i]), KV8 ? Sh::kConvertWarps : 1);
      mbar_init(smem_u32(&c.q_empty[i]), 1);
      mbar_init(smem_u32(&c.s_full[i]), 1);
      for (int part = 0; part < 2; ++part)
        mbar_init(smem_u32(&c.p_full[i][part]), 4 * Sh::kShares);
      mbar_init(smem_u32(&c.o_full[i]), 1);
    }
    for (int i = 0; i < kQueue; ++i) {
      mbar_init(smem_u32(&c.item_full[i]), 1);
      mbar_init(smem_u32(&c.item_empty[i]), Sh::kSoftmaxWarps + Sh::kLoaders + 1 + Sh::kConvertWarps);
    }
    for (int i = 0; i < 4 * Sh::kTiles; ++i) mbar_init(smem_u32(&c.met[i]), Sh::kShares);
    mbar_init(smem_u32(&c.drained), 1);
    c.abort = 0;
    fence_mbar_init();
    fence_async_smem();
  }
  if (warp == Sh::kMmaWarp) tmem_alloc(smem_u32(&c.tmem), 512);
  Piece piece;  // the others have nothing to do before it is known
  memset(&piece, 0, sizeof(piece));
  if (warp == Sh::kPlanWarp) piece = find_piece<HD, KV8>(a, lane);
  if (warp == Sh::kLoadWarp && lane == 0) {
    prefetch_map(&maps.q);
    prefetch_map(&maps.k);
    prefetch_map(&maps.v);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp < Sh::kSoftmaxWarps) {
    softmax_role<HD, KV8>(a, c, tiles, warp, lane);
  } else {
    if (warp < Sh::kLoadWarp + Sh::kLoaders) {
      load_role<HD, KV8>(a, maps, c, tiles, Sh::kLoaders == 1 ? 0 : uniform(warp - Sh::kLoadWarp),
                         lane);
    } else if (warp == Sh::kMmaWarp) {
      mma_items<HD, KV8>(a, c, tiles);
      // one lane issued every product: it is the one elected here too
      if (elect_one()) mma_commit(smem_u32(&c.drained));
      __syncwarp();  // no product or arrival is under way after this:
      const long long start = clock64();
      while (!mbar_try(smem_u32(&c.drained), 0) && clock64() - start < 1000000000LL) {
      }
    } else if (warp == Sh::kPlanWarp) {
      plan_role<HD, KV8>(a, c, piece, lane);
    } else if constexpr (KV8) {
      convert_role<HD, KV8>(a, c, tiles, threadIdx.x - Sh::kConvert * 32);
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == Sh::kMmaWarp) tmem_free(c.tmem, 512);
}

template <int N>
__device__ __forceinline__ void load_row(const float* p, float* v) {
  if constexpr (N == 2) {
    const float2 w = *reinterpret_cast<const float2*>(p);
    v[0] = w.x;
    v[1] = w.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 w = *reinterpret_cast<const float4*>(p + i);
      v[i] = w.x;
      v[i + 1] = w.y;
      v[i + 2] = w.z;
      v[i + 3] = w.w;
    }
  }
}

// ---- rows computed again ----
// A product takes 0 x NaN for a position that a row does not see, so a row can come out non-finite
// through a position of its tiles that only other rows see.  Such a row is computed from its own
// positions alone; one that sees a non-finite V itself, and took part in a product with no other,
// is as the formula has it and stays.

// 16 bytes of a V row: whether a value among them is Inf or NaN.
template <bool KV8>
__device__ __forceinline__ bool non_finite(const uint4& w) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    any |= KV8 ? __vcmpeq4(x[i] & 0x7f7f7f7fu, 0x7f7f7f7fu)
               : __vcmpeq2(x[i] & 0x7f807f80u, 0x7f807f80u);
  return any;
}

// The first position of [from, to) whose V holds Inf or NaN, or -1; by the warp.
template <int HD, bool KV8>
__device__ __noinline__ int find_bad(const ChunkArgs& a, int seq, int kvh, int from, int to) {
  constexpr int kSize = KV8 ? 1 : 2, kLanes = HD * kSize / 16;
  constexpr int kAt = 32 / kLanes, kAhead = 8;  // positions at once, loads in flight
  const int lane = threadIdx.x & 31;
  const int32_t* table = a.tables + int64_t(seq) * a.table_stride;
  const char* v = static_cast<const char*>(a.vc) + int64_t(kvh) * a.sh * kSize + lane % kLanes * 16;
#pragma unroll 1
  for (int c0 = from; c0 < to; c0 += kAhead * kAt) {
    uint4 w[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int c = c0 + u * kAt + lane / kLanes;
      w[u] = make_uint4(0, 0, 0, 0);
      if (c < to) {
        const int64_t id = table[c / a.B];  // c lies within the table; bad blocks count as zeros
        if (id >= 0 && id < a.blocks)
          w[u] = *reinterpret_cast<const uint4*>(v + (id * a.sb + int64_t(c % a.B) * a.so) * kSize);
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const uint32_t hits = __ballot_sync(0xffffffffu, non_finite<KV8>(w[u]));
      if (hits) return c0 + u * kAt + (__ffs(hits) - 1) / kLanes;
    }
  }
  return -1;
}

// Row (token tok of the item, query head) from positions [lo, hi) alone, by the warp.
template <int HD, bool KV8>
__device__ __noinline__ void redo_row(const ChunkArgs& a, const Item& it, int tok, int head, int lo,
                                      int hi) {
  constexpr int kSize = KV8 ? 1 : 2;
  constexpr int kPiece = 16 / kSize, kLanes = HD / kPiece;  // elements a lane, lanes a K row
  constexpr int kCols = HD / 32;                            // columns of O a lane
  constexpr int kAhead = 8;                                 // rows of K, of V in flight
  using Words = std::conditional_t<kCols * kSize == 16, uint4,
                                   std::conditional_t<kCols * kSize == 8, uint2, uint32_t>>;
  const int lane = threadIdx.x & 31, sub = lane % kLanes, column = lane * kCols;
  const int32_t* table = a.tables + int64_t(it.seq) * a.table_stride;
  const char* const keys =
      static_cast<const char*>(a.kc) + (int64_t(it.kvh) * a.sh + sub * kPiece) * kSize;
  const char* const values =
      static_cast<const char*>(a.vc) + (int64_t(it.kvh) * a.sh + column) * kSize;
  const float qk = a.scale_log2 * (KV8 ? a.k_scale : 1.0f);
  const int64_t token = it.tok0 + tok;
  float q[kPiece], m = -INFINITY, l = 0.0f, acc[kCols];
#pragma unroll
  for (int i = 0; i < kPiece; ++i)
    q[i] = __bfloat162float(a.q[token * a.q_t + head * a.q_h + sub * kPiece + i]);
#pragma unroll
  for (int i = 0; i < kCols; ++i) acc[i] = 0.0f;
  auto place = [&](int c) -> int64_t {  // bytes to position c's rows; -1: there are none
    if (c >= hi) return -1;
    const int64_t id = block_of(a, table, c);
    return id < 0 ? -1 : (id * a.sb + int64_t(c % a.B) * a.so) * kSize;
  };
  int64_t next = place(lo + lane);
#pragma unroll 1
  for (int c0 = lo; c0 < hi; c0 += 32) {
    const int64_t at = next;
    next = place(c0 + 32 + lane);  // on its way while this one is worked on
    // kLanes lanes take kLanes positions one after the other: lane x's own at step x % kLanes
    float s = -INFINITY;
#pragma unroll 1
    for (int step0 = 0; step0 < kLanes; step0 += kAhead) {
      uint4 w[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int64_t row = __shfl_sync(0xffffffffu, at, lane - sub + step0 + x);
        w[x] = *reinterpret_cast<const uint4*>(keys + (row < 0 ? 0 : row));
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const uint32_t words[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
        float k[kPiece], dot = 0.0f;
        unpack<KV8, kPiece>(words, k);
#pragma unroll
        for (int i = 0; i < kPiece; ++i) dot += q[i] * k[i];
#pragma unroll
        for (int y = kLanes / 2; y; y >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, y);
        if (sub == step0 + x && at >= 0) s = dot * qk;
      }
    }
    if (__any_sync(0xffffffffu, isnan(s))) {  // and so is every weight
      l = s = NAN;
      break;
    }
    float top = s;
#pragma unroll
    for (int y = 16; y; y >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
    const float m_new = fmaxf(m, top), base = m_new == -INFINITY ? 0.0f : m_new;
    const float w = exp2f(s - base), shrink = exp2f(m - base);
    m = m_new;
    l = l * shrink + w;
#pragma unroll
    for (int i = 0; i < kCols; ++i) acc[i] *= shrink;
#pragma unroll 1
    for (int k0 = 0; k0 < 32; k0 += kAhead) {
      Words words[kAhead];
      bool there[kAhead];
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const int64_t row = __shfl_sync(0xffffffffu, at, k0 + x);
        there[x] = row >= 0;
        words[x] = *reinterpret_cast<const Words*>(values + (row < 0 ? 0 : row));
      }
#pragma unroll
      for (int x = 0; x < kAhead; ++x) {
        const float wk = __shfl_sync(0xffffffffu, w, k0 + x);
        float v[kCols];
        unpack<KV8, kCols>(reinterpret_cast<const uint32_t*>(&words[x]), v);
        if (there[x])  // whatever the caches' first row, read in its place, holds
#pragma unroll
          for (int i = 0; i < kCols; ++i) acc[i] += wk * v[i];
      }
    }
  }
#pragma unroll
  for (int y = 16; y; y >>= 1) l += __shfl_xor_sync(0xffffffffu, l, y);
  const float inv = l == 0.0f ? 0.0f : (KV8 ? a.v_scale : 1.0f) / l;  // 0: it sees nothing
  const int64_t to = int64_t(head) * HD + column;
#pragma unroll
  for (int i = 0; i < kCols; ++i) {
    float y = acc[i] * inv;
    if (a.gate) y *= load_gate(a, token * a.gate_t + to + i);
    a.out[token * a.out_t + to + i] = __float2bfloat16_rn(y);
  }
}

// Looks at row r of an item, which came out non-finite, and computes it again if it has to be;
// false: it stays.  `guess`: a position that may be non-finite, for the block's warps.
template <int HD, bool KV8>
__device__ __noinline__ bool mend_row(const ChunkArgs& a, const Item& it, int r, volatile int* guess) {
  const int t = r / kM, in_tile = r % kM, row_tok = in_tile / a.G;
  const int tok = t * a.TB + row_tok, head = it.kvh * a.G + in_tile - row_tok * a.G;
  const int pos = it.pos0 + tok;
  // the positions whose products the row's tile took part in, and those that the row sees
  int first;
  const int tiles =
      tiles_seen(it.pos0 + t * a.TB, min(it.ntok - t * a.TB, a.TB), it.cap, a.window, first);
  const int p0 = max(first * kN, a.window ? it.pos0 - a.window + 1 : 0);
  const int p1 = max(min((first + tiles) * kN, min(it.pos0 + it.ntok, it.cap)), p0);
  const int lo = min(max(a.window ? pos - a.window + 1 : 0, p0), p1);
  const int hi = max(min(pos + 1, p1), lo);
  if (find_bad<HD, KV8>(a, it.seq, it.kvh, p0, lo) < 0 &&
      find_bad<HD, KV8>(a, it.seq, it.kvh, hi, p1) < 0) {
    // The warps of a block look for it in different places; what one finds serves all.
    const int step = (hi - lo + 15) / 16;
    for (int i = 0; i < 16; ++i) {
      const int g = *guess;  // never set, perhaps
      if (g >= lo && g < hi && find_bad<HD, KV8>(a, it.seq, it.kvh, g, g + 1) >= 0) return false;
      const int from = lo + (i + (threadIdx.x >> 5)) % 16 * step;
      const int found = find_bad<HD, KV8>(a, it.seq, it.kvh, from, min(from + step, hi));
      if (found < 0) continue;
      *guess = found;
      return false;
    }
    // neither: a sum that overflowed FP32 against a reference below the row's maximum
  }
  redo_row<HD, KV8>(a, it, tok, head, lo, hi);
  return true;
}

constexpr int kJoinSlices = 8;
// What a warp of join_kernel does where rows came out non-finite: it looks at its rows of the item
// that was joined (`cut`), and of the items that CTA blockIdx.x held whole (`whole`).
template <int HD, bool KV8>
__device__ __noinline__ void look_through(const ChunkArgs& a, int row0, bool cut, bool whole) {
  __shared__ int guess;
  const int lane = threadIdx.x & 31;
  auto rows = [&](const Item& it) {
#pragma unroll 1
    for (int r = row0; r < Shape<HD, KV8>::kItemRows; r += 16 * kJoinSlices) {
      const int t = r / kM, in_tile = r % kM, row_tok = in_tile / a.G;
      const int tok = t * a.TB + row_tok;
      if (in_tile >= a.TB * a.G || tok >= it.ntok || it.tok0 + tok >= a.T) continue;
      const int64_t column = int64_t(it.kvh * a.G + in_tile - row_tok * a.G) * HD + lane * (HD / 32);
      bool bad = false;
#pragma unroll
      for (int x = 0; x < HD / 32; ++x)
        bad |= !isfinite(__bfloat162float(a.out[(it.tok0 + tok) * a.out_t + column + x]));
      if (__any_sync(0xffffffffu, bad)) mend_row<HD, KV8>(a, it, r, &guess);
    }
  };
  if (cut) {
    const Join& j = reinterpret_cast<const Join*>(a.joins)[blockIdx.x];
    Item it;
    it.tok0 = j.tok0;
    it.ntok = j.ntok;
    it.kvh = j.kvh;
    it.seq = j.seq;
    it.pos0 = j.pos0;
    it.cap = j.cap;
    rows(it);
  }
  if (whole)
    walk<HD, KV8>(a, find_piece<HD, KV8>(a, lane), [&](const Item& it, int, int) {
      if (it.slot < 0) rows(it);
      return true;
    });
}

// Joins the parts of the items that were cut between CTAs: block (c, s) takes the item that
// starts at the end of CTA c's piece, a warp a row.  Then, where one of them, or of the rows of CTA
// c's whole items, is not finite, it looks through those.
template <int HD, bool KV8>
__global__ void __launch_bounds__(512, HD == 256 ? 1 : 2) join_kernel(const __grid_constant__ ChunkArgs a) {
  using Sh = Shape<HD, KV8>;
  constexpr int kPer = HD / 32;  // columns of a lane
  grid_wait();
  const int4 join = *reinterpret_cast<const int4*>(a.joins + blockIdx.x * 8);
  const int odd = a.joins[blockIdx.x * 8 + 4];
  const int parts = join.x, tok0 = join.y, ntok = join.z, kvh = join.w;
  if (!parts && !odd) return;
  const int lane = threadIdx.x & 31, row0 = blockIdx.y * 16 + (threadIdx.x >> 5);
  bool cut_odd = false;
  for (int r = row0; parts && r < Sh::kItemRows; r += 16 * kJoinSlices) {
    const int t = r / kM, in_tile = r % kM, row_tok = in_tile / a.G;
    const int tok = t * a.TB + row_tok;
    if (in_tile >= a.TB * a.G || tok >= ntok || tok0 + tok >= a.T) continue;
    auto slot = [&](int i) {
      return int64_t(i == 0 ? 2 * blockIdx.x + 1 : 2 * (blockIdx.x + i)) * Sh::kItemRows + r;
    };
    const int token = tok0 + tok;
    const int64_t column = int64_t(kvh * a.G + in_tile - row_tok * a.G) * HD + lane * kPer;
    float m = -INFINITY, l = 0.0f, acc[kPer], gate[kPer];
#pragma unroll
    for (int x = 0; x < kPer; ++x) {  // the gate on its way with the parts
      acc[x] = 0.0f;
      gate[x] = a.gate ? load_gate(a, token * a.gate_t + column + x) : 1.0f;
    }
    for (int i = 0; i < parts; i += 4) {  // four parts on their way at once
      float2 ml[4];
      float o[4][kPer];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        ml[y] = make_float2(0.0f, 0.0f);
        if (i + y < parts) {
          ml[y] = a.part_ml[slot(i + y)];
          load_row<kPer>(a.part_o + slot(i + y) * HD + lane * kPer, o[y]);
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        if (ml[y].y == 0.0f) continue;  // not there, or saw nothing
        const float top = max2(m, ml[y].x);
        const float keep = exp2_approx(m - top), w = exp2_approx(ml[y].x - top);
        m = top;
        l = l * keep + w * ml[y].y;
#pragma unroll
        for (int x = 0; x < kPer; ++x) acc[x] = acc[x] * keep + w * o[y][x];
      }
    }
    float zero = 0.0f;  // NaN if a sum is not finite
#pragma unroll
    for (int x = 0; x < kPer; ++x) zero = fmaf(acc[x], 0.0f, zero);
    cut_odd |= isnan(zero) && isfinite(l);
    const float inv = l == 0.0f ? 0.0f : (KV8 ? a.v_scale : 1.0f) / l;
#pragma unroll
    for (int x = 0; x < kPer; x += 2) {
      const float y0 = acc[x] * inv * gate[x], y1 = acc[x + 1] * inv * gate[x + 1];
      *reinterpret_cast<uint32_t*>(a.out + token * a.out_t + column + x) = pack_bf16(y0, y1);
    }
  }
  cut_odd = __any_sync(0xffffffffu, cut_odd);
  if (cut_odd || odd) {
    __syncwarp();  // the warp's stores come first
    look_through<HD, KV8>(a, row0, cut_odd, odd);
  }
}

// ------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------
struct ScratchLayout {
  int64_t joins, ml, o, total;
};
ScratchLayout scratch_layout(int ctas, int head_dim) {
  const int64_t rows = head_dim == 256 ? kM : 2 * kM;
  ScratchLayout s;
  s.joins = 256;  // [0, 256): header; word 0 = device error flags
  s.ml = s.joins + (int64_t(ctas) * 32 + 255) / 256 * 256;
  s.o = s.ml + 2 * ctas * rows * 8;
  s.total = s.o + 2 * ctas * rows * head_dim * 4;
  return s;
}

PFN_cuTensorMapEncodeTiled_v12000 encoder() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// A map of elements of `esize` bytes (bf16 or bytes) with the 128-byte swizzle.  A dimension of
// one element needs no stride of its own: any valid one does.
bool encode(CUtensorMap* map, const void* base, int esize, int rank, const int64_t* dims,
            const int64_t* strides, const int* box) {
  cuuint64_t d[5], st[5];
  cuuint32_t b[5], es[5];
  for (int i = 0; i < rank; ++i) {
    d[i] = cuuint64_t(dims[i]);
    b[i] = cuuint32_t(box[i]);
    es[i] = 1;
    if (i > 0) st[i - 1] = dims[i] == 1 ? 128 : cuuint64_t(strides[i]) * esize;
  }
  auto fn = encoder();
  return fn && fn(map, esize == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                  cuuint32_t(rank), const_cast<void*>(base),
                  d, st, b, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Whether n elements of `size` bytes from a and m from b share memory.
bool meet(const void* a, int64_t n, int size, const void* b, int64_t m, int b_size) {
  const auto x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return x < y + uintptr_t(m * b_size) && y < x + uintptr_t(n * size);
}

template <int HD, bool KV8>
int32_t launch(const ChunkArgs& a, const Maps& maps, int device, int ctas, cudaStream_t stream) {
  using Sh = Shape<HD, KV8>;
  constexpr int kBytes = Sh::kTileBytes + int(sizeof(Control<HD, KV8>));
  static_assert(kBytes <= 232448, "more shared memory than a CTA may have");
  static bool ready[64] = {false};
  if (!ready[device]) {
    const cudaError_t e = cudaFuncSetAttribute(
        chunk_kernel<HD, KV8>, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
    if (e != cudaSuccess)
      return fail(DORY_ERR_CUDA, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
    ready[device] = true;
  }
  chunk_kernel<HD, KV8><<<ctas, Sh::kThreads, kBytes, stream>>>(a, maps);
  int32_t status = dory::launched(cudaSuccess);
  if (status != DORY_OK) return status;
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(ctas, kJoinSlices);
  cfg.blockDim = dim3(512);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return dory::launched(cudaLaunchKernelEx(&cfg, join_kernel<HD, KV8>, a));
}

}  // namespace

extern "C" {

int64_t dory_chunk_params_bytes(void) { return int64_t(sizeof(DoryChunkParams)); }

int64_t dory_chunk_scratch_bytes(int32_t num_heads, int32_t num_kv_heads, int32_t head_dim) {
  if (num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads ||
      num_heads / num_kv_heads > 64 || (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return 0;
  int device;
  const int sms = device_sms(&device);
  return scratch_layout(sms > 0 ? sms : 148, head_dim).total;
}

int32_t dory_chunk_attention(const DoryChunkParams* P, void* stream) {
  if (!P) return fail(DORY_ERR_INVALID_ARGUMENT, "null params");
  const DoryChunkParams& p = *P;
  if (p.num_heads < 1 || p.num_kv_heads < 1 || p.num_heads % p.num_kv_heads)
    return fail(DORY_ERR_INVALID_ARGUMENT, "query heads must be a multiple of KV heads");
  if (p.num_tokens < 0 || p.num_seqs < 0)
    return fail(DORY_ERR_INVALID_ARGUMENT, "negative token or sequence count");
  if (p.window < 0) return fail(DORY_ERR_INVALID_ARGUMENT, "negative window");
  const int G = p.num_heads / p.num_kv_heads;
  if (G > 64) return fail(DORY_ERR_UNSUPPORTED, "%d query heads per KV head (max 64)", G);
  if (p.head_dim != 64 && p.head_dim != 128 && p.head_dim != 256)
    return fail(DORY_ERR_UNSUPPORTED, "head_dim %d (supported: 64, 128, 256)", p.head_dim);
  if (p.block_size < 16 || p.block_size % 16)
    return fail(DORY_ERR_UNSUPPORTED, "block_size %d is not a multiple of 16", p.block_size);
  if (p.kv_dtype != 0 && p.kv_dtype != DORY_DTYPE_BF16 && p.kv_dtype != DORY_DTYPE_FP8_E4M3)
    return fail(DORY_ERR_INVALID_ARGUMENT, "kv_dtype %d (bf16 or fp8 e4m3)", p.kv_dtype);
  const bool kv8 = p.kv_dtype == DORY_DTYPE_FP8_E4M3;
  if (kv8 && p.head_dim == 64)
    return fail(DORY_ERR_UNSUPPORTED, "FP8 caches take 128/256-dim heads");
  if (kv8 && !(p.k_scale > 0.0f && p.v_scale > 0.0f && p.k_scale < 3.4e38f && p.v_scale < 3.4e38f))
    return fail(DORY_ERR_INVALID_ARGUMENT, "FP8 caches need positive, finite k/v scales");
  if (!(p.softmax_scale > 0.0f && p.softmax_scale < 3.4e38f))
    return fail(DORY_ERR_INVALID_ARGUMENT, "softmax_scale must be positive and finite");
  if (p.gate && (p.gate_dtype < 0 || p.gate_dtype > 2))
    return fail(DORY_ERR_INVALID_ARGUMENT, "gate dtype");
  if (p.num_tokens == 0 || p.num_seqs == 0) return DORY_OK;  // nothing is read or written
  if (p.num_cache_blocks < 1 || p.max_blocks < 1)
    return fail(DORY_ERR_INVALID_ARGUMENT, "the cache and the block tables must not be empty");
  if (!p.q || !p.key_cache || !p.value_cache || !p.block_tables || !p.query_start ||
      !p.seq_lens || !p.out || !p.scratch)
    return fail(DORY_ERR_INVALID_ARGUMENT, "null tensor argument");
  // The stride of a dimension of one element is not used.
  const int64_t q_t = p.num_tokens > 1 ? p.q_stride_token : 0;
  const int64_t out_t = p.num_tokens > 1 ? p.out_stride_token : 0;
  const int64_t gate_t = p.num_tokens > 1 ? p.gate_stride_token : 0;
  const int64_t q_h = p.num_heads > 1 ? p.q_stride_head : 0;
  const int64_t sb = p.num_cache_blocks > 1 ? p.stride_block : 0;
  const int64_t sh = p.num_kv_heads > 1 ? p.stride_head : 0;
  const int64_t cache_mask = kv8 ? 15 : 7;
  if (!aligned16(p.q) || !aligned16(p.out) || ((q_t | q_h) & 7) || (out_t & 7))
    return fail(DORY_ERR_ALIGNMENT, "q and out need 16-byte aligned bases and rows");
  if (!aligned16(p.key_cache) || !aligned16(p.value_cache) ||
      ((sb | p.stride_offset | sh) & cache_mask))
    return fail(DORY_ERR_ALIGNMENT, "key/value caches need 16-byte aligned bases and strides");
  if (p.gate && (!aligned16(p.gate) || (gate_t & 7)))
    return fail(DORY_ERR_ALIGNMENT, "gate needs a 16-byte aligned base and rows");
  if (!aligned16(p.scratch))
    return fail(DORY_ERR_ALIGNMENT, "scratch needs a 16-byte aligned base");
  const int64_t need = dory_chunk_scratch_bytes(p.num_heads, p.num_kv_heads, p.head_dim);
  if (p.scratch_bytes < need)
    return fail(DORY_ERR_INVALID_ARGUMENT, "scratch too small (%lld < %lld bytes)",
                (long long)p.scratch_bytes, (long long)need);
  // A row may be computed again (redo_row) after others, and itself, have been stored.
  const int64_t width = int64_t(p.num_heads) * p.head_dim, last = p.num_tokens - 1;
  const int gate_size = p.gate_dtype == DORY_DTYPE_F32 ? 4 : 2;
  if (meet(p.out, last * out_t + width, 2, p.q,
           last * q_t + (p.num_heads - 1) * q_h + p.head_dim, 2) ||
      (p.gate && meet(p.out, last * out_t + width, 2, p.gate, last * gate_t + width, gate_size)))
    return fail(DORY_ERR_INVALID_ARGUMENT, "out must lie apart from q and gate");

  ChunkArgs a;
  memset(&a, 0, sizeof(a));
  a.q = static_cast<const __nv_bfloat16*>(p.q);
  a.kc = p.key_cache;
  a.vc = p.value_cache;
  a.tables = p.block_tables;
  a.query_start = p.query_start;
  a.seq_lens = p.seq_lens;
  a.gate = p.gate;
  a.out = static_cast<__nv_bfloat16*>(p.out);
  a.err = static_cast<uint32_t*>(p.scratch);
  a.q_t = q_t;
  a.q_h = q_h;
  a.out_t = out_t;
  a.gate_t = gate_t;
  a.table_stride = p.table_stride;
  a.sb = sb;
  a.so = p.stride_offset;
  a.sh = sh;
  a.blocks = p.num_cache_blocks;
  a.scale_log2 = p.softmax_scale * kLog2e;
  a.k_scale = p.k_scale;
  a.v_scale = p.v_scale;
  a.T = p.num_tokens;
  a.S = p.num_seqs;
  a.max_blocks = p.max_blocks;
  a.NH = p.num_heads;
  a.NKV = p.num_kv_heads;
  a.G = G;
  a.B = p.block_size;
  a.window = p.window < kMaxPosition ? p.window : kMaxPosition;
  a.gate_dtype = p.gate_dtype;
  a.TB = kM / G;
  a.copy_rows = p.block_size & -p.block_size;
  if (a.copy_rows > kN) a.copy_rows = kN;
  while ((1 << a.copy_shift) < a.copy_rows) ++a.copy_shift;
  const int64_t span = int64_t(p.max_blocks) * p.block_size;
  a.table_span = span < kMaxPosition ? int(span) : kMaxPosition;
  // The device counts units in 32 bits.
  const int64_t most = (int64_t(p.num_tokens) / (a.TB * (p.head_dim == 256 ? 1 : 2)) + p.num_seqs + 1) *
                       (a.table_span / kN + 2 + kItemUnits);
  if (most > (int64_t(1) << 30) / p.num_kv_heads)
    return fail(DORY_ERR_UNSUPPORTED, "more work than one call counts (tokens x positions)");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int device;
  const int ctas = device_sms(&device);
  if (ctas <= 0) return fail(DORY_ERR_CUDA, "no current CUDA device");
  uint8_t* scratch = static_cast<uint8_t*>(p.scratch);
  const ScratchLayout layout = scratch_layout(ctas, p.head_dim);
  a.joins = reinterpret_cast<int32_t*>(scratch + layout.joins);
  a.part_ml = reinterpret_cast<float2*>(scratch + layout.ml);
  a.part_o = reinterpret_cast<float*>(scratch + layout.o);
  Maps maps;
  const int64_t q_dims[3] = {p.head_dim, p.num_heads, p.num_tokens};
  const int64_t q_strides[3] = {1, q_h, q_t};
  const int q_box[3] = {64, G, a.TB};
  const int64_t c_dims[4] = {p.head_dim, p.block_size, p.num_kv_heads, p.num_cache_blocks};
  const int64_t c_strides[4] = {1, p.stride_offset, sh, sb};
  const int esize = kv8 ? 1 : 2;
  const int c_box[4] = {128 / esize, a.copy_rows, 1, 1};
  if (!encode(&maps.q, p.q, 2, 3, q_dims, q_strides, q_box) ||
      !encode(&maps.k, p.key_cache, esize, 4, c_dims, c_strides, c_box) ||
      !encode(&maps.v, p.value_cache, esize, 4, c_dims, c_strides, c_box))
    return fail(DORY_ERR_UNSUPPORTED, "no tensor map for the query or cache view (strides must be "
                                      "positive)");
  if (kv8)
    return p.head_dim == 128 ? launch<128, true>(a, maps, device, ctas, s)
                             : launch<256, true>(a, maps, device, ctas, s);
  if (p.head_dim == 64) return launch<64, false>(a, maps, device, ctas, s);
  if (p.head_dim == 128) return launch<128, false>(a, maps, device, ctas, s);
  return launch<256, false>(a, maps, device, ctas, s);
}

}  // extern "C"
