// Attention of a step's new tokens over a paged key/value cache, for sm_100a:
// token i of a request with `ctx` older tokens sees keys [0, ctx) and the new
// keys that its ancestor mask names (or new keys 0 .. i without a mask). One new
// token is plain decoding, a tree of drafts or a chunk of a prompt are many.
//
// Rows. The query heads of one key/value head share its keys, so the rows of a
// (request, key/value head) are its new tokens times the group's heads, row =
// token * G + head, cut into blocks of 256. What bounds it is reading K and V once
// up to about 200 rows, and the softmax's exponentials beyond.
//
// Work. A block's keys are tiles of 128; the tiles of all blocks, in order of
// (block, head, tile), are one list that is cut into equal shares, one per CTA
// (one per SM); every CTA adds up the requests' tiles itself to find where its
// share begins, which costs about a microsecond where a planning launch of its
// own cost five. Beginning a block costs a CTA about as much as kBlockCost tiles,
// which the list holds ahead of each block's. So a batch of uneven lengths and a single long request alike keep
// every SM reading to the end. A block whose tiles lie in several shares is
// joined at the end: each CTA publishes its rows of O with their maxima and sums,
// and when all have, each joins its slice of the rows, in a fixed order.
//
// A CTA is that of attention.cu (TMA producer, MMA issuer, two softmax
// warpgroups with their own TMEM scores and accumulator) with two uses of the
// warpgroups:
//   - above 128 rows: warpgroup t takes rows 128 t .. of the block, and both visit
//     every tile;
//   - up to 128 rows: both hold the same rows and visit every other tile.
// With few rows most of a 128-row tile would idle while a few threads worked
// through 128 columns each: a tile's product costs the same however many of its
// rows count. So up to 64 / 32 rows the tile holds 2 / 4 copies of them, copy k in
// its own TMEM lanes, and copy k's warps take only quarter (half) k of the
// columns, P being zero elsewhere. Every copy is a split of the keys of its own
// with its own maximum, sum and O; they meet in shared memory at the end of the
// block, together with the two warpgroups'.
//
// Measured, per call back to back (and in a replayed graph, on the GPU alone): 64 requests
// of up to 8192 keys, 32 heads over 8 of 128, one token each: 304-321 us, 5.1-5.4 TB/s
// (285-288); 384 of up to 2000 keys 580 us, 4.1 TB/s (550); 16 requests of up to 5000 keys
// with trees of up to 64 drafts 116 us (112-116, up to 140 after other work); two of
// 100003 and 81102 keys with up to 12 drafts, 16 heads over 2, 69 us (67); one of 777 keys,
// one token, 18.4 us (16.5-21); 2048 new tokens over 8192, 418 us, 740 TFLOPS (414); 256 of
// up to 200 keys 127 us (125), which is beginning blocks. Heads of 64: the decode 234 us
// (224), the drafts 96, the long two 50.
// Pages of 16 tokens cost the decode a fifth: a box of 2 KB takes about 100 cycles to issue
// and there are 32 to a tile. Issued from one lane of a converged warp they cost less on
// the GPU (344 -> 313 us) but the few boxes of larger pages more
// (288 -> 308), and code for both slowed either. Asking tiles into L2 ahead of the ring
// adds boxes and lost 3-25 %. A warp that fetches the next block's Q during the joins
// changed nothing.
//
// Pages: a tile is gathered by one TMA box per page and 64-element slab (a page
// of 128 tokens or more is one box), each lane of the producer warp issuing one.
// Keys past the request's length are loaded from past the last page, which fills
// zeros. Values that are not finite are handled as in attention_prefill.cu, and scores of
// NaN reach their row however its keys are split (see join_parts).
#include <algorithm>
#include <atomic>
#include <climits>
#include <cstring>
#include <type_traits>

#include "attention_common.cuh"

namespace b2g {

// One row block: where it is and how many tiles its rows need.
struct TreeEntry {
  int32_t request, block;   // block of 256 rows of the request
  int32_t tiles;            // KV tiles, at least one
  int32_t ctx;              // older tokens: length - new tokens (negative if it is shorter)
  int32_t fresh;            // new tokens
  int32_t first;            // first new token's row among all
  int32_t len;              // keys
};

// Where a share begins: head of `e` and unit of that; `before` units lie before the block.
struct ShareStart {
  int64_t units, before, here;  // here: units of the share
  TreeEntry e;
  int32_t hk, unit;
};

struct alignas(64) TreeParams {
  CUtensorMap tmK, tmV;  // 4-D (d, slot, head, page), 64 x min(page, 128) x 1 x 1 boxes
  const void* Q;
  int64_t q_t, q_h;
  void* O;
  int64_t o_t, o_h;
  const void* V;
  int64_t v_p, v_t, v_h;
  const int32_t* tables;
  int64_t table_stride;
  const int64_t* mask;
  float* lse;
  int* status;
  const int32_t* cu;
  const int32_t* lens;
  // Parts of unfinished blocks, four per CTA: of the block that its share begins
  // inside and of the one that it ends inside, of each warpgroup
  float* part;             // [4 per CTA][D / 4][part_rows] float4: O, rows side by side
  float2* part_ml;         // [4 per CTA][part_rows] {max (log2 units), sum}
  uint32_t* counters;      // two per CTA, zero at rest: published, joined
  int32_t mask_words, part_rows, requests;
  int32_t most;            // keys that a table has room for
  int32_t HQ, HK, G, tokens, page_size, num_pages;
  int64_t most_units;      // units of a head that the call can ask for at most
  int32_t inject;          // test hook: joins wait for a part that nobody publishes
  float scale_log2;
  uint64_t timeout_ns;
};

// Tiles that beginning a block counts as in the cut of the shares. What it costs depends on
// rows, pages and head dim, but one count serves them. Interleaved, for 0 / 4 / 8 / 16, us:
//   heads of 128: 16 drafted trees 127 / 117 / 116 / 112, two long caches 77 / 72 / 69 / 62,
//     384 requests of up to 2000 keys 591 / 587 / 581 / 587, 256 of up to 200 keys 155 / 129 /
//     127 / 124, 64 of up to 600 with 8 drafts 89 / 72 / 73 / 75, 2048 new tokens over 8192
//     415 / 415 / 418 / 423
//   heads of 64: the trees 101 / 99 / 96 / 104, the long caches 55 / 50 / 50 / 50, 64 requests
//     of up to 8192 keys 238 / 234 / 234 / 235
constexpr int32_t kBlockCost = 8;

template <int D>
struct TreePlan {
  static constexpr uint32_t kSoftmaxWarps = 8;
  static constexpr uint32_t kFirstSoftmax = 2;  // after the producer and the MMA issuer
  static constexpr uint32_t kThreads = 32 * (kFirstSoftmax + kSoftmaxWarps);
  static constexpr uint32_t kSlabs = D / 64;
  static constexpr uint32_t kTile = kSlabs * kSlabBytes;  // Q, K or V tile
  static constexpr uint32_t kSlots = D == 128 ? 5 : 10;   // ring of K and V tiles in turn
  static constexpr uint32_t kQOff = 0;                    // two tiles
  static constexpr uint32_t kJoinOff = kTile;  // up to 128 rows the second Q tile is the join buffer
  static constexpr uint32_t kRingOff = 2 * kTile;
  static constexpr uint32_t kMlOff = kRingOff + kSlots * kTile;   // float2 [8 warps][32 rows]
  static constexpr uint32_t kBarOff = kMlOff + 8 * 32 * 8;
  // q_full, q_empty, full[S], empty[S], s_full[2], p_full[2][2], o_done[2], o_free[2]
  static constexpr uint32_t kNumBars = 2 + 2 * kSlots + 10;
  static constexpr uint32_t kMiscOff = kBarOff + kNumBars * 8;  // tmem slot, abort flag
  static constexpr uint32_t kOddOff = kMiscOff + 16;            // [2 blocks][8 warps]
  static constexpr uint32_t kBytes = kOddOff + 64;
  // the carve-up starts on a 1024-byte boundary; what is left of the 227 KB is
  // there for rounding up to it, and the kernel refuses to run if that is too little
  static constexpr uint32_t kMaxDyn = 232448;
  static constexpr uint32_t kDynBytes = kBytes + 1024 <= kMaxDyn ? kBytes + 1024 : kMaxDyn;
  static constexpr uint32_t kS = 0, kO = 256, kTileCols = 128;
  static_assert(kBytes <= kMaxDyn, "shared memory");
  static_assert(2 * (kThreads / 32) * 8 <= 512 && 512 + sizeof(ShareStart) <= 8 * 32 * 8, "scratch");
};

// ------------------------------------------------------------------- plan --
// Request r: its new tokens and keys, cut to what the call has room for.
__device__ __forceinline__ TreeEntry tree_request(const TreeParams& p, int32_t r, bool report) {
  TreeEntry e;
  const int32_t lo = p.cu[r], hi = p.cu[r + 1], len = p.lens[r];
  e.request = r;
  e.block = 0;
  e.tiles = 0;
  e.first = min(max(lo, 0), p.tokens);
  e.fresh = min(max(hi, e.first), p.tokens) - e.first;
  e.len = min(max(len, 0), p.most);
  e.ctx = e.len - e.fresh;
  if (report) {
    if (lo < 0 || hi < lo || hi > p.tokens) fmha_report(p, B2G_STATUS_TOKENS);
    if (len > p.most) fmha_report(p, B2G_STATUS_PAGE_TABLE);
  }
  return e;
}

__device__ __forceinline__ int32_t tree_blocks(const TreeParams& p, const TreeEntry& e) {
  return static_cast<int32_t>((static_cast<int64_t>(e.fresh) * p.G + 255) / 256);
}

// Tiles of keys that a block's rows see some of; without a mask its last token
// sees no newer one.
__device__ __forceinline__ int32_t tree_tiles(const TreeParams& p, const TreeEntry& e, int32_t block) {
  int32_t end = e.len;
  if (p.mask == nullptr) {
    const int32_t rows = min(e.fresh * p.G, (block + 1) * 256);
    end = min(end, e.ctx + (rows - 1) / p.G + 1);
  }
  return max((end + 127) / 128, 1);
}

// Units before CTA c's of `ctas` equal shares, and the CTA whose share holds unit
// u. A 64-bit division takes several hundred cycles, so 32-bit ones where they do.
__device__ __forceinline__ int64_t mul_div(int64_t a, int64_t b, int64_t d) {
  const int64_t n = a * b;
  if (((n | d) >> 32) == 0) return static_cast<uint32_t>(n) / static_cast<uint32_t>(d);
  return n / d;
}
__device__ __forceinline__ int64_t share_begin(int64_t units, int32_t c, int32_t ctas) {
  return mul_div(units, c, ctas);
}
__device__ __forceinline__ int32_t share_of(int64_t u, int64_t units, int32_t ctas) {
  // the last c whose share begins at or before u: c < (u + 1) ctas / units
  const int64_t n = (u + 1) * ctas - 1;
  return static_cast<int32_t>(mul_div(n, 1, units));
}

// The share of this CTA. All threads of the block take part; `sums` is scratch in
// shared memory for two int64 per warp, and `out` shared too.
template <uint32_t kThreads>
__device__ __forceinline__ void find_share(const TreeParams& p, int64_t* sums, ShareStart* out) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr uint32_t kWarps = kThreads / 32;
  auto tiles_of = [&](int32_t r, bool report) {
    if (r >= p.requests) return static_cast<int64_t>(0);
    const TreeEntry e = tree_request(p, r, report);
    const int32_t blocks = tree_blocks(p, e);
    int64_t n = 0;
    for (int32_t b = 0; b < blocks; ++b) n += tree_tiles(p, e, b) + kBlockCost;
    return n;
  };
  int64_t first = 0, sum = 0;  // this thread's first request, and all of them
  for (int32_t r0 = 0; r0 < p.requests; r0 += static_cast<int32_t>(kThreads)) {
    const int64_t n = tiles_of(r0 + static_cast<int32_t>(threadIdx.x), blockIdx.x == 0);
    if (r0 == 0) first = n;
    sum += n;
  }
  int64_t scan = first;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t up = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= static_cast<uint32_t>(d)) scan += up;
  }
  if (lane == 31u) sums[warp] = scan;
  if (lane == 0u) sums[kWarps + warp] = sum;
  // before the barrier: the thread that finds the share stores its length after it
  if (threadIdx.x == 0) out->here = 0;
  __syncthreads();
  int64_t total = 0, base = 0, upto = 0;
#pragma unroll
  for (uint32_t i = 0; i < kWarps; ++i) {
    total += sums[kWarps + i];
    if (i < warp) base += sums[i];
    upto += sums[i];
  }
  // Offsets that decrease name rows more than once: what passes all that the call's shapes
  // hold (hours of work from a few tokens) is not run. The status has been set above.
  if (total > p.most_units) total = 0;
  const int64_t units = total * p.HK;
  const int64_t ctas = min(units, static_cast<int64_t>(gridDim.x));
  const int64_t u =
      ctas > 0 ? share_begin(units, static_cast<int32_t>(blockIdx.x), static_cast<int32_t>(ctas)) : 0;
  if (threadIdx.x == 0) out->units = units;
  if (static_cast<int64_t>(blockIdx.x) >= ctas) return;
  int64_t n = first, before = base + scan - first;  // units a head of this thread's request, and before it
  for (int32_t r0 = 0;;) {
    if (n > 0 && before * p.HK <= u && u < (before + n) * p.HK) {
      const int32_t r = r0 + static_cast<int32_t>(threadIdx.x);
      TreeEntry e = tree_request(p, r, false);
      e.tiles = tree_tiles(p, e, 0);
      while (u >= (before + e.tiles + kBlockCost) * p.HK) {
        before += e.tiles + kBlockCost;
        e.tiles = tree_tiles(p, e, ++e.block);
      }
      const int64_t in = u - before * p.HK;  // less than (tiles + kBlockCost) * HK
      out->here = share_begin(units, static_cast<int32_t>(blockIdx.x) + 1,
                              static_cast<int32_t>(ctas)) - u;
      out->before = before * p.HK;
      out->e = e;
      out->hk = static_cast<int32_t>(mul_div(in, 1, e.tiles + kBlockCost));
      out->unit = static_cast<int32_t>(in - static_cast<int64_t>(out->hk) * (e.tiles + kBlockCost));
    }
    r0 += static_cast<int32_t>(kThreads);
    // the same for all threads: whether the share begins in a later round of requests
    if (r0 >= p.requests || u < upto * p.HK) break;
    n = tiles_of(r0 + static_cast<int32_t>(threadIdx.x), false);
    scan = n;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t up = __shfl_up_sync(0xffffffffu, scan, d);
      if (lane >= static_cast<uint32_t>(d)) scan += up;
    }
    __syncthreads();
    if (lane == 31u) sums[warp] = scan;
    __syncthreads();
    before = upto + scan - n;
#pragma unroll
    for (uint32_t i = 0; i < kWarps; ++i) {
      if (i < warp) before += sums[i];
      upto += sums[i];
    }
  }
}

// ----------------------------------------------------------------- kernel --
// The part of one (block, key/value head) that lies in this CTA's share.
struct Segment {
  TreeEntry e;
  int64_t unit0;    // the unit of the block and head's first tile
  int32_t hk;
  int32_t j0, j1;   // tiles
  int32_t row0, rows;
  bool two;         // above 128 rows: a row tile per warpgroup
  uint32_t slots;   // warpgroups with tiles to visit
};

// Walks a share: the segments of its `left` units.
struct SegmentWalk {
  TreeEntry e;
  int64_t left, before;  // before: units before the block
  int32_t hk, unit;

  __device__ __forceinline__ void begin(const ShareStart& s) {
    left = s.here;
    before = s.before;
    e = s.e;
    hk = s.hk;
    unit = s.unit;
  }

  __device__ __forceinline__ bool next(const TreeParams& p, Segment& s) {
    while (left > 0) {
      if (hk == p.HK) {  // the next block, of this request or of the next that has new tokens
        before += static_cast<int64_t>(e.tiles + kBlockCost) * p.HK;
        hk = 0;
        if (e.block + 1 < tree_blocks(p, e)) {
          ++e.block;
        } else {
          do e = tree_request(p, e.request + 1, false);
          while (e.fresh == 0);
        }
        e.tiles = tree_tiles(p, e, e.block);
      }
      const int32_t of_head = e.tiles + kBlockCost, from = unit;
      const int32_t to = static_cast<int32_t>(min(static_cast<int64_t>(of_head), from + left));
      left -= to - from;
      unit = 0;
      s.hk = hk++;
      if (to <= kBlockCost) continue;  // the share ends before the block's first tile
      s.e = e;
      s.unit0 = before + static_cast<int64_t>(s.hk) * of_head + kBlockCost;
      s.j0 = max(from - kBlockCost, 0);
      s.j1 = to - kBlockCost;
      s.row0 = e.block * 256;
      s.rows = min(256, e.fresh * p.G - s.row0);
      s.two = s.rows > 128;
      s.slots = s.two || s.j1 - s.j0 > 1 ? 2u : 1u;
      return true;
    }
    return false;
  }
};

// What the join of a block that lies in several shares needs of it.
struct OpenBlock {
  int32_t owner;  // the CTA whose share has its first tile (-1: none)
  int32_t parts;  // shares
  int32_t first, hk, row0, rows;
  int32_t each;   // parts that a share has of it
};

// The place of tile j's K and V among a segment's loads (n tiles).
__device__ __forceinline__ uint32_t k_order(bool two, int32_t j) {
  return static_cast<uint32_t>(two || j == 0 ? 2 * j : 2 * j - 1);
}
__device__ __forceinline__ uint32_t v_order(bool two, int32_t j, int32_t n) {
  return static_cast<uint32_t>(two || j + 1 == n ? 2 * j + 1 : 2 * j + 2);
}

// log2 of the copies that a segment's row tile holds of its rows.
__device__ __forceinline__ uint32_t tree_log_copies(const Segment& s) {
  return s.two || s.rows > 64 ? 0u : s.rows > 32 ? 1u : 2u;
}

__device__ __forceinline__ uint64_t mask_word(const TreeParams& p, const TreeEntry& e, int32_t i,
                                              int32_t w) {
  return static_cast<uint64_t>(p.mask[static_cast<int64_t>(e.first + i) * p.mask_words + w]);
}

// Bits of the 32 keys from kb on that new token i of the segment's request sees.
// (`word0` is the first word of its mask)
__device__ __forceinline__ uint32_t seen_bits(const TreeParams& p, const TreeEntry& e, int32_t i,
                                              uint64_t word0, int32_t kb) {
  auto low = [](int32_t n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; };
  const int32_t r = kb - e.ctx;  // rank of the first key among the new ones
  if (p.mask == nullptr) return low(min(i + 1, e.fresh) - r);
  uint32_t bits = low(-r);  // older tokens
  if (r > -32) {
    auto word = [&](int32_t w) {
      if (w <= 0) return w == 0 ? word0 : 0ull;
      return w < p.mask_words ? mask_word(p, e, i, w) : 0ull;
    };
    const int32_t w = r >> 6, sh = r & 63;  // arithmetic: word -1 holds ranks -64 .. -1
    uint64_t v = word(w) >> sh;
    if (sh > 32) v |= word(w + 1) << (64 - sh);
    bits |= static_cast<uint32_t>(v) & ~low(-r);
  }
  return bits & low(e.fresh - r);
}

// Adds to n values of a row of O (of new token i, from dim d0 on) what is not
// finite among the values that the token sees; see attention_prefill.cu.
template <int D, typename T, typename OutT>
__device__ __noinline__ void add_odd_cache_values(const TreeParams& p, const Segment& s, int32_t i,
                                                  int32_t d0, int32_t n, OutT* out) {
  for (int32_t kb = s.j0 * 128; kb < min(s.j1 * 128, s.e.len); kb += 32) {
    uint32_t bits = seen_bits(p, s.e, i, p.mask != nullptr ? mask_word(p, s.e, i, 0) : 0ull, kb);
    while (bits != 0u) {
      const int32_t key = kb + __ffs(static_cast<int>(bits)) - 1;
      bits &= bits - 1u;
      const int32_t page =
          p.tables[s.e.request * p.table_stride + key / p.page_size];
      if (page < 0 || page >= p.num_pages) continue;
      const T* v = static_cast<const T*>(p.V) + page * p.v_p + (key % p.page_size) * p.v_t +
                   s.hk * p.v_h + d0;
      for (int32_t d = 0; d < n; ++d) {
        const float x = static_cast<float>(v[d]);
        if (!isfinite(x)) out[d] = static_cast<OutT>(static_cast<float>(out[d]) + x);
      }
    }
  }
}

__device__ __forceinline__ void softmax_warps_meet() {
  asm volatile("bar.sync 1, 256;" ::: "memory");
}

// Joins share k of a block: a lane to a row, E float4 columns by P parts at a time,
// whose loads are all in flight together (with eight warps on the SM their latency
// and that of the arithmetic between them is what bounds this, so what depends on
// the row alone is done once). More than P parts go in rounds with a running
// maximum. With many parts and fewer than eight runs of columns, warps split a run's parts
// and the first of them adds up what they leave in shared memory (`sums`, six floats
// by 32 lanes each). Indices past the end repeat the last one: every load is
// unconditional. All warps meet the same number of times. A part without anything is
// one whose sum is zero: scores that are all NaN leave a maximum of -inf too, and have
// to come out as NaN.
template <int D, bool kBF16, int E, int P>
__device__ __noinline__ void join_parts(const TreeParams& p, const OpenBlock& b, int32_t k,
                                        int32_t warp8, int32_t lane, float* sums) {
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr int32_t kRuns = D / 4 / E;  // runs of E columns in a row
  const int32_t all = (b.rows + 31) / 32 * kRuns, parts = b.parts * b.each;
  const int32_t from = all * k / b.parts, to = all * (k + 1) / b.parts;
  const int32_t ls = E > 1 || parts <= 16 || to - from >= 8 ? 0 : to - from >= 4 ? 1 : to - from >= 2 ? 2 : 3;
  const int32_t split = warp8 & ((1 << ls) - 1);  // of the run's parts, this warp's
  const int32_t step = p.part_rows * (D / 4);      // float4s of a part
  for (int32_t u0 = from; u0 < to; u0 += 8 >> ls) {
    const int32_t u1 = u0 + (warp8 >> ls), u = min(u1, to - 1);
    const int32_t r0 = u / kRuns * 32 + lane, r = min(r0, b.rows - 1), v = u % kRuns * E;
    const float2* ml = p.part_ml + 4 * b.owner * p.part_rows + r;
    const float4* po = reinterpret_cast<const float4*>(p.part) + 4 * b.owner * step + v * p.part_rows + r;
    float m = -INFINITY, l = 0.0f;
    float4 sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int32_t c0 = split; c0 < parts; c0 += P << ls) {
      float2 x[P];
      float4 o[P][E];
#pragma unroll
      for (int c = 0; c < P; ++c) {
        const int32_t i = min(c0 + (c << ls), parts - 1);
        const int32_t share = b.each == 2 ? i >> 1 : i;
        // the owner's part lies in its second pair of slots, the others' in their first
        const int32_t id = 4 * share + (share == 0 ? 2 : 0) + (b.each == 2 ? i & 1 : 0);
        x[c] = __ldcg(ml + id * p.part_rows);
#pragma unroll
        for (int e = 0; e < E; ++e) o[c][e] = __ldcg(po + id * step + e * p.part_rows);
      }
      float top = m;
#pragma unroll
      for (int c = 0; c < P; ++c) top = fmaxf(top, x[c].x);
      const float ref = top == -INFINITY ? 0.0f : top;  // nothing so far, or only NaN
      const float was = fast_exp2(m - ref);
      m = top;
      l *= was;
#pragma unroll
      for (int e = 0; e < E; ++e)
        sum[e] = make_float4(sum[e].x * was, sum[e].y * was, sum[e].z * was, sum[e].w * was);
#pragma unroll
      for (int c = 0; c < P; ++c) {
        // a part without anything may never have been written
        if (c0 + (c << ls) >= parts || x[c].y == 0.0f) continue;
        const float f = fast_exp2(x[c].x - ref);
        l = fmaf(x[c].y, f, l);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          sum[e].x = fmaf(o[c][e].x, f, sum[e].x);
          sum[e].y = fmaf(o[c][e].y, f, sum[e].y);
          sum[e].z = fmaf(o[c][e].z, f, sum[e].z);
          sum[e].w = fmaf(o[c][e].w, f, sum[e].w);
        }
      }
    }
    if (E == 1 && ls > 0) {
      float* mine = sums + warp8 * 6 * 32 + lane;
      mine[0] = m;
      mine[32] = l;
      mine[64] = sum[0].x;
      mine[96] = sum[0].y;
      mine[128] = sum[0].z;
      mine[160] = sum[0].w;
      softmax_warps_meet();
      if (split == 0) {
        float top = -INFINITY;
        for (int c = 0; c < (1 << ls); ++c) top = fmaxf(top, mine[c * 192]);
        const float ref = top == -INFINITY ? 0.0f : top;
        m = top;
        l = 0.0f;
        sum[0] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int c = 0; c < (1 << ls); ++c) {
          const float* x = mine + c * 192;
          const float f = fast_exp2(x[0] - ref);
          l = fmaf(x[32], f, l);
          sum[0].x = fmaf(x[64], f, sum[0].x);
          sum[0].y = fmaf(x[96], f, sum[0].y);
          sum[0].z = fmaf(x[128], f, sum[0].z);
          sum[0].w = fmaf(x[160], f, sum[0].w);
        }
      }
      softmax_warps_meet();
    }
    if (split != 0 || u1 >= to || r0 >= b.rows) continue;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int32_t g = b.row0 + r, t = g / p.G, h = b.hk * p.G + g - t * p.G;
    T* dst = static_cast<T*>(p.O) + static_cast<int64_t>(b.first + t) * p.o_t + h * p.o_h + 4 * v;
    uint2 out[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      out[e] = make_uint2(pack2<kBF16>(sum[e].x * inv, sum[e].y * inv),
                          pack2<kBF16>(sum[e].z * inv, sum[e].w * inv));
    if constexpr (E == 1) {
      *reinterpret_cast<uint2*>(dst) = out[0];
    } else {
#pragma unroll
      for (int e = 0; e < E; e += 2)
        reinterpret_cast<uint4*>(dst)[e / 2] = make_uint4(out[e].x, out[e].y, out[e + 1].x, out[e + 1].y);
    }
    if (v == 0 && p.lse != nullptr)
      p.lse[static_cast<int64_t>(h) * p.tokens + b.first + t] =
          l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.693147180559945309f;
  }
}

template <int D, bool kBF16>
__global__ void __launch_bounds__(TreePlan<D>::kThreads, 1)
    tree_kernel(const __grid_constant__ TreeParams p) {
  using TP = TreePlan<D>;
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr uint32_t NS = TP::kSlots;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  if (static_cast<uint32_t>(smem - smem_raw) + TP::kBytes > TP::kDynBytes) {
    if (threadIdx.x == 0) fmha_report(p, B2G_STATUS_SMEM_BASE);
    return;
  }
  const uint32_t sbase = smem_u32(smem);
  const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  const uint32_t bar0 = sbase + TP::kBarOff;
  const uint32_t q_full = bar0, q_empty = bar0 + 8u;
  auto full = [&](uint32_t s) { return bar0 + 8u * (2 + s); };
  auto empty = [&](uint32_t s) { return bar0 + 8u * (2 + NS + s); };
  const uint32_t bar1 = bar0 + 8u * (2 + 2 * NS);
  auto s_full = [&](uint32_t t) { return bar1 + 8u * t; };
  auto p_full = [&](uint32_t t, uint32_t half) { return bar1 + 8u * (2 + 2 * t + half); };
  auto o_done = [&](uint32_t t) { return bar1 + 8u * (6 + t); };
  auto o_free = [&](uint32_t t) { return bar1 + 8u * (8 + t); };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + TP::kMiscOff);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + TP::kMiscOff + 4);

  if (threadIdx.x == 0) {
    mbar_init(q_full, TP::kSoftmaxWarps);
    mbar_init(q_empty, 1);
    for (uint32_t s = 0; s < NS; ++s) {
      mbar_init(full(s), 1);
      mbar_init(empty(s), 1);
    }
    for (uint32_t t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t, 0), 4);
      mbar_init(p_full(t, 1), 4);
      mbar_init(o_done(t), 1);
      mbar_init(o_free(t), 4);
    }
    *abort_flag = 0u;
    fence_mbarrier_init();
    prefetch_tensormap(&p.tmK);
    prefetch_tensormap(&p.tmV);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(tmem_slot), 512);
    tmem_relinquish<1>();
  }
  ShareStart* start = reinterpret_cast<ShareStart*>(smem + TP::kMlOff + 512);
  find_share<TP::kThreads>(p, reinterpret_cast<int64_t*>(smem + TP::kMlOff), start);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  const ShareStart share = *start;
  const int64_t units = share.units;
  const int32_t ctas =
      static_cast<int32_t>(min(units, static_cast<int64_t>(gridDim.x)));
  const int32_t me = static_cast<int32_t>(blockIdx.x);
  SegmentWalk walk;
  walk.begin(share);
  Segment w;

  if (warp == 0) {
    // ------------------------------------------------------------ producer --
    // K and V tiles in turn through one ring. Lane l of the warp issues box l: a
    // tile is `boxes` pages (or one, of a large page) by kSlabs slabs.
    const int32_t box_rows = min(p.page_size, 128);
    const uint32_t boxes = 128u / static_cast<uint32_t>(box_rows);
    const uint32_t box = lane % boxes, slab = lane / boxes;
    const bool issues = slab < TP::kSlabs;
    uint32_t ld = 0;  // tiles loaded
    bool alive = true;
    while (alive && walk.next(p, w)) {
      const int32_t* table = p.tables + w.e.request * p.table_stride;
      // this lane's page of tile j, as the table has it; -2 for keys past the end
      auto page_of = [&](int32_t j) {
        const int32_t key = j * 128 + static_cast<int32_t>(box) * box_rows;
        return issues && key < w.e.len ? table[key / p.page_size] : -2;
      };
      auto load = [&](const CUtensorMap* map, int32_t j, int32_t page) {
        const uint32_t s = ld % NS;
        if (!__all_sync(0xffffffffu, fmha_wait(empty(s), ((ld / NS) & 1u) ^ 1u, abort_flag, p,
                                               B2G_SITE_EMPTY))) {
          alive = false;
          return;
        }
        if (lane == 0) mbar_arrive_expect_tx(full(s), TP::kTile);
        __syncwarp();
        if (issues) {
          if (page < 0 || page >= p.num_pages) {  // past the last page: the box reads zeros
            if (page != -2) fmha_report(p, B2G_STATUS_PAGE_TABLE);
            page = p.num_pages;
          }
          tma_load_4d(sbase + TP::kRingOff + s * TP::kTile + slab * kSlabBytes +
                          box * static_cast<uint32_t>(box_rows) * 128u,
                      map, full(s), static_cast<int32_t>(slab) * 64,
                      p.page_size > 128 ? (j * 128) % p.page_size : 0, w.hk, page);
        }
        ++ld;
      };
      // In the order in which the products take them: with two row tiles K and V of
      // a tile, else K a tile ahead of V. Pages are read two tiles ahead.
      int32_t page = page_of(w.j0), page1 = w.j0 + 1 < w.j1 ? page_of(w.j0 + 1) : -2;
      load(&p.tmK, w.j0, page);
      for (int32_t j = w.j0; alive && j < w.j1; ++j) {
        const int32_t page2 = j + 2 < w.j1 ? page_of(j + 2) : -2;
        if (w.two) load(&p.tmV, j, page);
        if (alive && j + 1 < w.j1) load(&p.tmK, j + 1, page1);
        if (alive && !w.two) load(&p.tmV, j, page);
        page = page1;
        page1 = page2;
      }
    }
    // every load issued lands before the CTA can exit
    for (uint32_t i = ld > NS ? ld - NS : 0u; i < ld; ++i) {
      uint32_t spins = 0;
      while (!mbar_try_wait(full(i % NS), (i / NS) & 1u) && spins < (1u << 20)) ++spins;
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------- MMA issue --
    // The whole warp runs this and one lane issues; see attention_prefill.cu.
    {
      constexpr uint32_t idesc_s = fmha_idesc_s<D, kBF16>();
      constexpr uint32_t idesc_pv = fmha_idesc_pv<D, kBF16>();
      uint32_t last_bar = 0, last_par = 0;  // the newest commit: all earlier MMAs precede it
      uint32_t base = 0, ic = 0;            // ring loads before the segment, segments
      uint32_t steps0 = 0, steps1 = 0;      // tiles of each warpgroup (phases of s_full, p_full)
      uint32_t items0 = 0, items1 = 0;      // segments of each (phases of o_done, o_free)
      bool alive = true;
      auto wait = [&](uint32_t bar, uint32_t parity, int site) {
        return __all_sync(0xffffffffu, fmha_wait(bar, parity & 1u, abort_flag, p, site)) != 0;
      };
      auto commit = [&](uint32_t bar) {
        if (elect_one()) tc_commit<1>(bar);
      };
      const uint64_t q_desc = sdesc_kmajor_sw128(sbase + TP::kQOff);
      const uint64_t k_desc = sdesc_kmajor_sw128(sbase + TP::kRingOff);
      const uint64_t v_desc = sdesc_mnmajor_sw128(sbase + TP::kRingOff, kSlabBytes, 1024u);
      while (alive && uniform(static_cast<int32_t>(walk.next(p, w))) != 0) {
        const int32_t n = uniform(w.j1 - w.j0);
        const bool two = uniform(static_cast<int32_t>(w.two)) != 0;
        const uint32_t slots = two || n > 1 ? 2u : 1u;
        // S = Q K^T of tile j for warpgroup t
        auto issue_s = [&](uint32_t t, int32_t j, uint32_t s) {
          const uint64_t qd = q_desc + (two ? t * (TP::kTile >> 4) : 0u);
          const uint64_t kd = k_desc + s * (TP::kTile >> 4);
#pragma unroll
          for (uint32_t kk = 0; kk < D / 16; ++kk) {
            const uint32_t at = (kk >> 2) * (kSlabBytes >> 4) + 2u * (kk & 3u);
            if (elect_one())
              mma_f16<1>(tmem_base + TP::kS + t * TP::kTileCols, qd + at, kd + at, idesc_s,
                         kk > 0 ? 1u : 0u);
          }
          commit(s_full(t));
          // the tile of K is free after its last product, Q after the block's
          if (!two || t == 1u) {
            commit(empty(s));
            if (j + 1 == n) commit(q_empty);
          }
        };
        if (!wait(q_full, ic, B2G_SITE_FULL)) break;
        for (uint32_t t = 0; t < slots; ++t) {
          const int32_t j = two ? 0 : static_cast<int32_t>(t);
          const uint32_t ld = base + k_order(two, j);
          if (!wait(full(ld % NS), ld / NS, B2G_SITE_FULL)) {
            alive = false;
            break;
          }
          tc_fence_after();
          issue_s(t, j, ld % NS);
        }
        // warpgroup t's PV of tile j, then S of its next one
        auto slot_step = [&](uint32_t t, int32_t j, uint32_t& steps, uint32_t& items) {
          const int32_t next = j + (two ? 1 : 2);
          const bool first = two ? j == 0 : j < 2, more = next < n;
          const uint32_t lv = base + v_order(two, j, n), lk = base + k_order(two, next);
          if (!wait(full(lv % NS), lv / NS, B2G_SITE_FULL)) return false;
          // with a row tile to each warpgroup K of the next tile is there by now
          if (two && more && !wait(full(lk % NS), lk / NS, B2G_SITE_FULL)) return false;
          if (first && items > 0 && !wait(o_free(t), items - 1u, B2G_SITE_ACC_EMPTY)) return false;
          const uint64_t vd = v_desc + (lv % NS) * (TP::kTile >> 4);
          const uint32_t p_col = tmem_base + TP::kS + t * TP::kTileCols;
#pragma unroll
          for (uint32_t half = 0; half < 2; ++half) {
            if (!wait(p_full(t, half), steps, B2G_SITE_ACC_FULL)) return false;
            tc_fence_after();
#pragma unroll
            for (uint32_t k4 = 0; k4 < 4; ++k4) {
              const uint32_t kk = half * 4u + k4;
              if (elect_one())
                mma_f16_ts(tmem_base + TP::kO + t * TP::kTileCols, p_col + kk * 8u,
                           vd + kk * (2048u >> 4), idesc_pv, (!first || kk > 0) ? 1u : 0u);
            }
          }
          ++steps;
          if (!two) commit(empty(lv % NS));
          if (more) {
            if (!two && !wait(full(lk % NS), lk / NS, B2G_SITE_FULL)) return false;
            tc_fence_after();
            issue_s(t, next, lk % NS);
            last_bar = s_full(t);
            last_par = steps & 1u;
          } else {
            commit(o_done(t));
            last_bar = o_done(t);
            last_par = items & 1u;
            ++items;
          }
          if (two && t == 1u) commit(empty(lv % NS));
          return true;
        };
        for (int32_t j = 0; alive && j < n; ++j) {
          if (two || (j & 1) == 0) alive = slot_step(0u, j, steps0, items0);
          if (alive && (two || (j & 1) != 0)) alive = slot_step(1u, j, steps1, items1);
        }
        base += 2u * static_cast<uint32_t>(n);
        ++ic;
      }
      // all MMAs issued by this warp finish before TMEM can be freed
      if (last_bar != 0u) {
        uint32_t spins = 0;
        while (!mbar_try_wait(last_bar, last_par) && spins < (1u << 22)) ++spins;
      }
    }
  } else {
    // ------------------------------------ Q, softmax, epilogue and the join --
    const uint32_t w8 = warp - TP::kFirstSoftmax;
    const uint32_t t = w8 >> 2;                // warpgroup
    const uint32_t quarter = warp & 3u;        // TMEM lane quarter of the warp
    const uint32_t row = quarter * 32u + lane;
    const uint32_t taddr = tmem_base + ((quarter * 32u) << 16);
    const uint32_t s_col = taddr + TP::kS + t * TP::kTileCols;
    const uint32_t o_col = taddr + TP::kO + t * TP::kTileCols;
    float2* ml = reinterpret_cast<float2*>(smem + TP::kMlOff);  // [warpgroup][quarter][lane]
    volatile uint32_t* odd_words = reinterpret_cast<volatile uint32_t*>(smem + TP::kOddOff);
    uint32_t step = 0, ti = 0;        // this warpgroup's tiles and segments
    uint32_t base = 0, ic = 0;        // ring loads before the segment, segments of the CTA
    bool alive = true;
    // The eight warps meet at a hardware barrier, which has no limit of its own: so a
    // warp whose wait ran out does not leave, but goes on without waiting (its results
    // no longer count, the status says so) and reaches every meeting like the others.
    auto wait_all = [&](uint32_t bar, uint32_t parity, int site) {
      if (alive && __all_sync(0xffffffffu, fmha_wait(bar, parity & 1u, abort_flag, p, site)) == 0)
        alive = false;
    };
    auto meet = [&]() { softmax_warps_meet(); };
    // blocks of this share that other shares hold parts of: the first and the last
    OpenBlock open_first = {-1}, open_last = {-1};

    while (walk.next(p, w)) {
      const bool whole = w.j0 == 0 && w.j1 == w.e.tiles;
      const uint32_t lc = tree_log_copies(w);
      const uint32_t copies = 1u << lc, per = 4u >> lc;  // copies of the rows, warps of a copy
      const uint32_t copy = quarter >> (2u - lc);
      const int32_t lrow = static_cast<int32_t>((quarter & (per - 1u)) * 32u + lane);  // row in the tile
      const int32_t brow = lrow + (w.two ? static_cast<int32_t>(t) * 128 : 0);  // row in the block
      const bool real = brow < w.rows;
      const int32_t grow = w.row0 + brow;                // row of the (request, head)
      const int32_t tok = grow / p.G, head = w.hk * p.G + grow - tok * p.G;

      // Q into shared memory: with one row tile each warpgroup copies half of every row
      if (ic > 0) wait_all(q_empty, ic - 1u, B2G_SITE_EMPTY);
      {
        constexpr uint32_t kVecs = static_cast<uint32_t>(D) / 8;  // 16-byte pieces of a row
        const uint32_t v0 = w.two ? 0u : t * (kVecs / 2), v1 = w.two ? kVecs : v0 + kVecs / 2;
        const uint4* src = reinterpret_cast<const uint4*>(
            static_cast<const T*>(p.Q) + (w.e.first + static_cast<int64_t>(real ? tok : 0)) * p.q_t +
            (real ? head : 0) * p.q_h);
        const uint32_t dst = sbase + TP::kQOff + (w.two ? t * TP::kTile : 0u) + row * 128u;
        constexpr uint32_t kBatch = kVecs / 2;
        for (uint32_t v = v0; v < v1; v += kBatch) {
          uint4 x[kBatch];
#pragma unroll
          for (uint32_t i = 0; i < kBatch; ++i) x[i] = real ? src[v + i] : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (uint32_t i = 0; i < kBatch; ++i) {
            // 128-byte swizzle: 16-byte piece c of row r sits at piece c ^ (r % 8)
            const uint32_t a = dst + ((v + i) >> 3) * kSlabBytes + ((((v + i) & 7u) ^ (row & 7u)) << 4);
            const uint32_t r4[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
            st_shared_v4(a, r4);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
      }

      // the lanes without a row stay quiet: their maximum never moves
      float m_run = real ? -INFINITY : INFINITY, l_run = 0.0f;
      uint32_t odd = 0;
      const int32_t n = w.j1 - w.j0;
      const int32_t stride = w.two ? 1 : 2;
      const uint64_t word0 = p.mask != nullptr && real ? mask_word(p, w.e, tok, 0) : 0ull;
      for (int32_t j = w.two ? 0 : static_cast<int32_t>(t); j < n; j += stride, ++step) {
        const int32_t kb = (w.j0 + j) * 128;
        const bool masked = kb + 128 > w.e.ctx;  // some row may not see some key
        // Above one copy a row's weights are zero outside its columns, so every tile
        // is looked through; above 128 rows the first warpgroup does it for both.
        if ((masked || copies > 1u) && !(w.two && t == 1u)) {
          const uint32_t load = base + v_order(w.two, j, n);
          wait_all(full(load % NS), load / NS, B2G_SITE_FULL);
          const bool mine = clear_odd_values<D, kBF16>(
              sbase + TP::kRingOff + (load % NS) * TP::kTile + row * 128u, lane);
          const uint32_t found = __ballot_sync(0xffffffffu, mine);
          if (found != 0u) fence_proxy_async_smem();
          odd |= found;
        }
        wait_all(s_full(t), step, B2G_SITE_ACC_FULL);
        tc_fence_after();
        if (j + stride >= n && lane == 0) odd_words[(ic & 1u) * 8u + t * 4u + quarter] = odd;
        uint32_t seen[4] = {~0u, ~0u, ~0u, ~0u};
        const bool first = j < stride;
        const uint32_t c0 = copy * per;
        if (masked && real) {
#pragma unroll
          for (uint32_t c = 0; c < 4; ++c)
            if (c < per)
              seen[c] = seen_bits(p, w.e, tok, word0, kb + 32 * static_cast<int32_t>(c0 + c));
        }
        if (per == 4u)
          tile_softmax<D, kBF16, 4>(s_col, o_col, 0u, p.scale_log2, masked, seen, first, m_run,
                                    l_run, p_full(t, 0), p_full(t, 1), lane);
        else if (per == 2u)
          tile_softmax<D, kBF16, 2>(s_col, o_col, c0, p.scale_log2, masked, seen, first, m_run,
                                    l_run, p_full(t, 0), p_full(t, 1), lane);
        else
          tile_softmax<D, kBF16, 1>(s_col, o_col, c0, p.scale_log2, masked, seen, first, m_run,
                                    l_run, p_full(t, 0), p_full(t, 1), lane);
      }

      const bool active = t < w.slots;
      if (active) {
        wait_all(o_done(t), ti, B2G_SITE_ACC_FULL);
        tc_fence_after();
        ++ti;
      }
      // where the rows go: O, or this share's unfinished rows
      const bool direct = w.two || (!whole && copies == 1u);  // no join in this CTA
      const int32_t part_id =
          4 * me + (w.j0 == 0 ? 2 : 0) + (direct && !w.two ? static_cast<int32_t>(t) : 0);
      float4* part = reinterpret_cast<float4*>(p.part) +
                     static_cast<int64_t>(part_id) * p.part_rows * (D / 4);
      float2* part_ml = p.part_ml + static_cast<int64_t>(part_id) * p.part_rows;
      constexpr float kLn2 = 0.693147180559945309f;
      auto store_sums = [&](float m, float l) {  // of this thread's row
        if (!whole) {
          part_ml[brow] = make_float2(m, l);
        } else if (p.lse != nullptr) {
          p.lse[static_cast<int64_t>(head) * p.tokens + w.e.first + tok] =
              l == 0.0f ? -INFINITY : (m + __log2f(l)) * kLn2;
        }
      };
      if (direct && !active) {
        if (real) store_sums(m_run, l_run);  // a sum of nothing: its O is never read
      } else if (direct) {
        uint32_t o[D];
#pragma unroll
        for (uint32_t d = 0; d < static_cast<uint32_t>(D); d += 32u)
          tmem_ld_32x32b_x32(o_col + d, *reinterpret_cast<uint32_t(*)[32]>(&o[d]));
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_free(t));
        // two row tiles of one V: the first warpgroup looked; else each at its own
        const volatile uint32_t* m = odd_words + (ic & 1u) * 8u + (w.two ? 0u : t * 4u);
        const bool any_odd = (m[0] | m[1] | m[2] | m[3]) != 0u;
        if (real) {
          store_sums(m_run, l_run);
          if (whole) {
            const float inv = l_run == 0.0f ? 0.0f : 1.0f / l_run;
            T* dst = static_cast<T*>(p.O) + static_cast<int64_t>(w.e.first + tok) * p.o_t + head * p.o_h;
#pragma unroll
            for (int v = 0; v < D / 8; ++v) {
              uint4 u;
              uint32_t* uw = &u.x;
#pragma unroll
              for (int i = 0; i < 4; ++i)
                uw[i] = pack2<kBF16>(__uint_as_float(o[8 * v + 2 * i]) * inv,
                                     __uint_as_float(o[8 * v + 2 * i + 1]) * inv);
              reinterpret_cast<uint4*>(dst)[v] = u;
            }
            if (any_odd) add_odd_cache_values<D, T>(p, w, tok, 0, D, dst);
          } else {
#pragma unroll
            for (int v = 0; v < D / 4; ++v)
              part[v * p.part_rows + brow] =
                  make_float4(__uint_as_float(o[4 * v]), __uint_as_float(o[4 * v + 1]),
                              __uint_as_float(o[4 * v + 2]), __uint_as_float(o[4 * v + 3]));
            if (any_odd)
              for (int v = 0; v < D / 4; ++v)
                add_odd_cache_values<D, T>(p, w, tok, 4 * v, 4, &part[v * p.part_rows + brow].x);
          }
        }
      } else {
        // the copies and the two warpgroups meet: maxima and sums first, then O in
        // column chunks through shared memory, already scaled by the writers
        ml[(t * 4u + quarter) * 32u + lane] = make_float2(m_run, l_run);
        meet();
        const volatile uint32_t* ow = odd_words + (ic & 1u) * 8u;
        bool any_odd = (ow[0] | ow[1] | ow[2] | ow[3]) != 0u;
        if (w.slots == 2u) any_odd |= (ow[4] | ow[5] | ow[6] | ow[7]) != 0u;
        const uint32_t parts = w.slots * copies;  // at most eight
        // warp of part c that holds this row, or row r
        auto warp_of = [&](uint32_t c, uint32_t r) {
          return ((c >> lc) << 2) + ((c & (copies - 1u)) << (2u - lc)) + (r >> 5);
        };
        // (a maximum of -inf: nothing seen, with sums of zero, or only NaN, with sums of NaN)
        float m_tot = -INFINITY, l_tot = 0.0f, ref;
        {
          float2 x[8];
#pragma unroll
          for (uint32_t c = 0; c < 8; ++c)
            x[c] = c < parts ? ml[warp_of(c, static_cast<uint32_t>(lrow)) * 32u + lane]
                             : make_float2(-INFINITY, 0.0f);
#pragma unroll
          for (uint32_t c = 0; c < 8; ++c) m_tot = fmaxf(m_tot, x[c].x);
          ref = m_tot == -INFINITY ? 0.0f : m_tot;
#pragma unroll
          for (uint32_t c = 0; c < 8; ++c) l_tot = fmaf(x[c].y, fast_exp2(x[c].x - ref), l_tot);
        }
        float scale = fast_exp2(m_run - ref);
        if (whole) scale = l_tot == 0.0f ? 0.0f : scale / l_tot;
        if (t == 0u && copy == 0u && real) store_sums(m_tot, l_tot);
        // A round takes 32 columns, or as many as the buffer holds of fewer rows: it
        // is [8 warps][row][columns], the float4s of a row permuted so that eight
        // rows at once spread over the banks.
        const uint32_t lw = w.rows <= 8 ? 3u : w.rows <= 16 ? 4u : 5u;  // log2 rows of a warp
        constexpr uint32_t kLogTile = D == 128 ? 15 : 14;
        static_assert(TP::kTile == 1u << kLogTile, "join buffer");
        const uint32_t lv = min(D == 128 ? 5u : 4u, kLogTile - 3u - 4u - lw);  // log2 float4s of a round
        const uint32_t vecs = 1u << lv, cols = vecs * 4u;
        const uint32_t buf = sbase + TP::kJoinOff;
        auto at = [&](uint32_t wq, uint32_t r, uint32_t v) {
          return buf + ((((wq << lw) + r) << lv) + (v ^ (r & (vecs - 1u) & 7u))) * 16u;
        };
        for (uint32_t d = 0; d < static_cast<uint32_t>(D); d += cols) {
          if (active) {
#pragma unroll 1
            for (uint32_t d2 = 0; d2 < cols; d2 += 16u) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(o_col + d + d2, o);
              tmem_wait_ld();
              if (real) {
#pragma unroll
                for (uint32_t v = 0; v < 4; ++v) {
                  uint32_t x[4];
#pragma unroll
                  for (uint32_t i = 0; i < 4; ++i)
                    x[i] = __float_as_uint(__uint_as_float(o[4 * v + i]) * scale);
                  st_shared_v4(at(t * 4u + quarter, lane, d2 / 4u + v), x);
                }
              }
            }
            if (d + cols == static_cast<uint32_t>(D)) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(o_free(t));
            }
          }
          meet();
          // four columns of a row to a thread: neighbours along the row where it goes to
          // O, neighbouring rows where it goes to the unfinished ones
          auto sum_of = [&](uint32_t r, uint32_t v) {
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
            for (uint32_t c = 0; c < parts; ++c) {
              uint32_t x[4];
              ld_shared_v4(at(warp_of(c, r), r & 31u, v), x);
              sum.x += __uint_as_float(x[0]);
              sum.y += __uint_as_float(x[1]);
              sum.z += __uint_as_float(x[2]);
              sum.w += __uint_as_float(x[3]);
            }
            return sum;
          };
          if (whole) {
            for (uint32_t i = (threadIdx.x - 32u * TP::kFirstSoftmax); i < static_cast<uint32_t>(w.rows) << lv; i += 256u) {
              const uint32_t r = i >> lv, v = i & (vecs - 1u);
              const float4 sum = sum_of(r, v);
              const int32_t g = w.row0 + static_cast<int32_t>(r), tk = g / p.G;
              const int32_t col = static_cast<int32_t>(d + 4u * v);
              T* dst = static_cast<T*>(p.O) + static_cast<int64_t>(w.e.first + tk) * p.o_t +
                       (w.hk * p.G + g - tk * p.G) * p.o_h + col;
              *reinterpret_cast<uint2*>(dst) =
                  make_uint2(pack2<kBF16>(sum.x, sum.y), pack2<kBF16>(sum.z, sum.w));
              if (any_odd) add_odd_cache_values<D, T>(p, w, tk, col, 4, dst);
            }
          } else {
            for (uint32_t v = w8; v < vecs; v += 8u) {
              for (uint32_t r = lane; r < static_cast<uint32_t>(w.rows); r += 32u) {
                const int32_t col = static_cast<int32_t>(d + 4u * v);
                float4* dst = part + (col / 4) * p.part_rows + r;
                *dst = sum_of(r, v);
                if (any_odd)
                  add_odd_cache_values<D, T>(p, w, (w.row0 + static_cast<int32_t>(r)) / p.G, col, 4,
                                             &dst->x);
              }
            }
          }
          meet();  // the buffer is free again
        }
      }
      if (!whole) {
        OpenBlock b;
        b.owner = share_of(w.unit0, units, ctas);
        b.parts = share_of(w.unit0 + w.e.tiles - 1, units, ctas) - b.owner + 1;
        b.first = w.e.first;
        b.hk = w.hk;
        b.row0 = w.row0;
        b.rows = w.rows;
        b.each = direct && !w.two ? 2 : 1;
        (w.j1 == w.e.tiles ? open_first : open_last) = b;
      }
      base += 2u * static_cast<uint32_t>(n);
      ++ic;
    }

    // The blocks that this share had a part of: this CTA's parts are published, and
    // when all of a block's are, each of its CTAs joins a slice of the block's
    // values, in the order of the shares.
    if (open_first.owner >= 0 || open_last.owner >= 0) {
      meet();
      const int32_t owner = lane == 0 ? open_first.owner : open_last.owner;
      if (w8 == 0u && lane < 2u && owner >= 0) {
        __threadfence();
        atomicAdd(&p.counters[2 * owner], 1u);
      }
    }
#pragma unroll 1
    for (int slot = 0; slot < 2; ++slot) {
      const OpenBlock b = slot == 0 ? open_first : open_last;
      if (b.owner < 0) continue;
      if (w8 == 0u && lane == 0) {
        uint32_t* count = p.counters + 2 * b.owner;
        const uint64_t t0 = globaltimer_ns();
        bool there = true;
        while (ld_acquire_gpu(count) < static_cast<uint32_t>(b.parts + p.inject)) {
          if (*abort_flag != 0u || globaltimer_ns() - t0 > p.timeout_ns) {
            fmha_report(p, B2G_STATUS_TIMEOUT | B2G_SITE_FLAG);
            *abort_flag = 1u;
            there = false;
            break;
          }
        }
        // the last CTA to have seen the count leaves both words at zero
        if (there && atomicAdd(&count[1], 1u) + 1u == static_cast<uint32_t>(b.parts)) {
          count[0] = 0u;
          count[1] = 0u;
        }
        __threadfence();
      }
      meet();
      if (*abort_flag != 0u) continue;
      const int32_t k = me - b.owner, wi = static_cast<int32_t>(w8), ln = static_cast<int32_t>(lane);
      float* sums = reinterpret_cast<float*>(smem + TP::kJoinOff);
      // Few parts: more columns to a thread instead of loads of parts that are not there.
      // With the last form alone, 16 drafted trees take 154 us instead of 116, 2048 new
      // tokens over 8192 461 instead of 418; two long caches, 74 parts a block, are alike.
      const int32_t parts = b.parts * b.each;
      if (parts <= 2)
        join_parts<D, kBF16, 4, 2>(p, b, k, wi, ln, sums);
      else if (parts <= 4)
        join_parts<D, kBF16, 2, 4>(p, b, k, wi, ln, sums);
      else
        join_parts<D, kBF16, 1, 8>(p, b, k, wi, ln, sums);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<1>(tmem_base, 512);
  }
}

// ------------------------------------------------------------------- host --
namespace {

struct TreeWorkspace {
  size_t part, part_ml, total;
  int32_t part_rows;
};

TreeWorkspace tree_workspace(int64_t tokens, int group, int head_dim, int sms) {
  TreeWorkspace w;
  auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
  w.part_rows = static_cast<int32_t>(std::min<int64_t>(256, tokens * group));
  w.part_ml = workspace_flag_bytes(sms);
  w.part = w.part_ml + up(sizeof(float2) * 4 * static_cast<size_t>(sms) * w.part_rows);
  w.total = w.part + sizeof(float) * 4 * static_cast<size_t>(sms) * w.part_rows * head_dim;
  return w;
}

bool encode_cache(CUtensorMap* map, const void* base, int dtype, int D, int page_size, int heads,
                  int64_t pages, const int64_t* st /* page, slot, head (elements) */) {
  auto enc = tma_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(page_size),
                              static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(pages)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(st[1]) * 2u,
                                 static_cast<cuuint64_t>(st[2]) * 2u,
                                 static_cast<cuuint64_t>(st[0]) * 2u};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(std::min(page_size, 128)), 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t =
      dtype == B2G_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, t, 4, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, bool kBF16>
int launch_tree(const TreeParams& prm, int sms, cudaStream_t stream) {
  using TP = TreePlan<D>;
  auto kern = tree_kernel<D, kBF16>;
  static std::atomic<bool> attr_set[64];  // per instantiation and device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return B2G_ENODEVICE;
  }
  if (!attr_set[dev].load()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(TP::kDynBytes)) != cudaSuccess)
      return static_cast<int>(cudaGetLastError());
    attr_set[dev].store(true);
  }
  // one CTA per SM: the CTAs that share a block wait for one another, so all of
  // them have to be resident, which a cooperative launch guarantees
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(sms), 1, 1);
  cfg.blockDim = dim3(TP::kThreads, 1, 1);
  cfg.dynamicSmemBytes = TP::kDynBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeCooperative;
  attr[0].val.cooperative = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, prm);
  if (e != cudaSuccess) cudaGetLastError();
  return e == cudaSuccess ? B2G_OK : static_cast<int>(e);
}

}  // namespace

}  // namespace b2g

extern "C" size_t b2g_attention_tree_workspace_bytes(int requests, int64_t tokens, int heads_q,
                                                     int heads_k, int head_dim) {
  const int sms = b2g::current_device_sms();
  if (sms <= 0 || requests < 0 || tokens < 0 || heads_k < 1 || heads_q < heads_k || head_dim < 1)
    return 0;
  return b2g::tree_workspace(tokens, heads_q / heads_k, head_dim, sms).total;
}

extern "C" int b2g_attention_tree(const void* q, const void* k_cache, const void* v_cache, void* o,
                                  const int64_t* strides, const int32_t* block_tables,
                                  int64_t table_stride, int max_pages, const int32_t* seq_lens,
                                  const int32_t* cu_seqlens, const int64_t* tree_mask,
                                  int mask_words, int requests, int64_t tokens, int heads_q,
                                  int heads_k, int head_dim, int64_t num_pages, int page_size,
                                  int dtype, float sm_scale, float* lse, void* workspace,
                                  size_t workspace_bytes, int* status, void* stream) {
  using namespace b2g;
  if (tokens < 0 || tokens > INT_MAX - 256 || requests < 0) return B2G_ESHAPE;
  if (tokens == 0 || requests == 0) return B2G_OK;
  const int rc = check_serving_attention(heads_q, heads_k, head_dim, dtype, sm_scale, strides, 10,
                                         {q, k_cache, v_cache, o});
  if (rc != B2G_OK) return rc;
  if (block_tables == nullptr || seq_lens == nullptr || cu_seqlens == nullptr) return B2G_EINVAL;
  if (tree_mask != nullptr && mask_words < 1) return B2G_EINVAL;
  if (num_pages < 1 || num_pages > INT_MAX - 1 || max_pages < 0) return B2G_ESHAPE;
  if (page_size != 8 && page_size != 16 && page_size != 32 && page_size != 64 &&
      (page_size < 1 || page_size % 128 != 0))
    return B2G_ESHAPE;
  const int group = heads_q / heads_k;
  if (tokens * group > INT_MAX - 512) return B2G_ESHAPE;
  if (requests > 1 && table_stride < max_pages) return B2G_ESTRIDE;
  if (reinterpret_cast<uintptr_t>(tree_mask) % 8 != 0 ||
      reinterpret_cast<uintptr_t>(lse) % alignof(float) != 0)
    return B2G_EALIGN;
  const int sms = current_device_sms();
  if (sms <= 0) return B2G_ENODEVICE;
  const TreeWorkspace wl = tree_workspace(tokens, group, head_dim, sms);
  if (workspace == nullptr || workspace_bytes < wl.total) return B2G_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return B2G_EALIGN;
  uint8_t* ws = static_cast<uint8_t*>(workspace);

  TreeParams prm;
  std::memset(&prm, 0, sizeof(prm));
  if (!encode_cache(&prm.tmK, k_cache, dtype, head_dim, page_size, heads_k, num_pages, strides + 2) ||
      !encode_cache(&prm.tmV, v_cache, dtype, head_dim, page_size, heads_k, num_pages, strides + 5))
    return B2G_ETENSORMAP;
  prm.Q = q;
  prm.q_t = strides[0];
  prm.q_h = strides[1];
  prm.V = v_cache;
  prm.v_p = strides[5];
  prm.v_t = strides[6];
  prm.v_h = strides[7];
  prm.O = o;
  prm.o_t = strides[8];
  prm.o_h = strides[9];
  prm.tables = block_tables;
  prm.table_stride = table_stride;
  prm.mask = tree_mask;
  prm.mask_words = mask_words;
  prm.lse = lse;
  prm.status = status;
  prm.cu = cu_seqlens;
  prm.lens = seq_lens;
  prm.requests = requests;
  prm.most = static_cast<int32_t>(
      std::min<int64_t>(static_cast<int64_t>(max_pages) * page_size, INT_MAX - 256));
  // a block for every 256 rows, a ragged one for each request, each with all tiles
  prm.most_units =
      (tokens * group / 256 + std::min<int64_t>(requests, tokens)) *
      (std::max<int64_t>((static_cast<int64_t>(prm.most) + 127) / 128, 1) + kBlockCost);
  prm.part = reinterpret_cast<float*>(ws + wl.part);
  prm.part_ml = reinterpret_cast<float2*>(ws + wl.part_ml);
  prm.part_rows = wl.part_rows;
  prm.counters = reinterpret_cast<uint32_t*>(ws);
  prm.HQ = heads_q;
  prm.HK = heads_k;
  prm.G = group;
  prm.tokens = static_cast<int32_t>(tokens);
  prm.page_size = page_size;
  prm.num_pages = static_cast<int32_t>(num_pages);
  prm.scale_log2 = sm_scale * 1.4426950408889634f;
  prm.timeout_ns = wait_timeout_ns();
  prm.inject = inject_flag_timeout() ? 1 : 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool bf16 = dtype == B2G_DT_BF16;
  if (head_dim == 128)
    return bf16 ? launch_tree<128, true>(prm, sms, s) : launch_tree<128, false>(prm, sms, s);
  return bf16 ? launch_tree<64, true>(prm, sms, s) : launch_tree<64, false>(prm, sms, s);
}
