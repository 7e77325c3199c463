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
// (one per SM). So a batch of uneven lengths and a single long request alike keep
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
// Pages: a tile is gathered by one TMA box per page and 64-element slab (a page
// of 128 tokens or more is one box), each lane of the producer warp issuing one.
// Keys past the request's length are loaded from past the last page, which fills
// zeros. Values that are not finite are handled as in attention.cu.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cstring>
#include <type_traits>

#include "attention_common.cuh"

namespace b2g {

// One row block: where it is and how many tiles its rows need.
struct alignas(32) TreeEntry {
  int32_t request, block;   // block of 256 rows of the request
  int32_t tiles;            // KV tiles, at least one
  int32_t before;           // tiles of the blocks before this one (per key/value head)
  int32_t ctx;              // older tokens: length - new tokens (negative if it is shorter)
  int32_t fresh;            // new tokens
  int32_t first;            // first new token's row among all
  int32_t len;              // keys
};

struct TreeMeta {
  int32_t entries, pad;
  int64_t units;  // tiles of all blocks and key/value heads
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
  const TreeEntry* plan;
  const TreeMeta* meta;
  const int4* start;       // per CTA: entry, head, tile of its first unit
  float* part;             // [2 per CTA][part_rows][D] unfinished O
  float2* part_ml;         // [2 per CTA][part_rows] {max (log2 units), sum}
  uint32_t* counters;      // two per CTA, zero at rest: published, joined
  int32_t mask_words, part_rows;
  int32_t HQ, HK, G, tokens, page_size, num_pages;
  float scale_log2;
  uint64_t timeout_ns;
};

template <int D>
struct TreePlan {
  static constexpr uint32_t kSoftmaxWarps = 8;
  static constexpr uint32_t kThreads = 64 + 32 * kSoftmaxWarps;
  static constexpr uint32_t kSlabs = D / 64;
  static constexpr uint32_t kTile = kSlabs * kSlabBytes;  // Q, K or V tile
  static constexpr uint32_t kSlots = D == 128 ? 5 : 10;   // ring of K and V tiles in turn
  static constexpr uint32_t kQOff = 0;                    // two tiles
  static constexpr uint32_t kJoinOff = kTile;  // up to 128 rows the second Q tile is the join buffer
  static constexpr uint32_t kJoinCols = D / 4; // columns joined at a time (8 warps x 32 rows x 4 B)
  static constexpr uint32_t kRingOff = 2 * kTile;
  static constexpr uint32_t kMlOff = kRingOff + kSlots * kTile;   // float2 [8 warps][32 rows]
  static constexpr uint32_t kBarOff = kMlOff + 8 * 32 * 8;
  // q_full, q_empty, full[S], empty[S], s_full[2], p_full[2][2], o_done[2], o_free[2], join
  static constexpr uint32_t kNumBars = 2 + 2 * kSlots + 11;
  static constexpr uint32_t kMiscOff = kBarOff + kNumBars * 8;  // tmem slot, abort flag
  static constexpr uint32_t kOddOff = kMiscOff + 16;            // [2 blocks][8 warps]
  static constexpr uint32_t kBytes = kOddOff + 64;
  // the carve-up starts on a 1024-byte boundary; what is left of the 227 KB is
  // there for rounding up to it, and the kernel refuses to run if that is too little
  static constexpr uint32_t kMaxDyn = 232448;
  static constexpr uint32_t kDynBytes = kBytes + 1024 <= kMaxDyn ? kBytes + 1024 : kMaxDyn;
  static constexpr uint32_t kS = 0, kO = 256, kTileCols = 128;
  static_assert(kBytes <= kMaxDyn, "shared memory");
  static_assert(8 * 32 * kJoinCols * 4 == kTile, "join buffer");
};

// The CTA whose share holds unit u, of `ctas` equal shares of `units`.
__device__ __forceinline__ int32_t share_of(int64_t u, int64_t units, int32_t ctas) {
  return static_cast<int32_t>(((u + 1) * ctas - 1) / units);
}

// ------------------------------------------------------------------- plan --
// The row blocks of all requests with running sums of their tiles, and where each
// CTA's share begins. One CTA, latency-bound: a scan over the requests, then a
// search per share.
constexpr int kTreePlanThreads = 1024;
constexpr int kTreePlanShared = 4096;  // running sums kept in shared memory for the searches

struct TreePlanParams {
  const int32_t* cu;
  const int32_t* lens;
  TreeEntry* plan;
  TreeMeta* meta;
  int4* start;
  int* status;
  int64_t most;  // keys that a table has room for
  int32_t requests, tokens, G, HK, capacity, ctas, chain;
};

__global__ void __launch_bounds__(kTreePlanThreads) tree_plan_kernel(const TreePlanParams p) {
  __shared__ int32_t before[kTreePlanShared];
  __shared__ int64_t warp_e[kTreePlanThreads / 32], warp_u[kTreePlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_launch_dependents();
  int64_t e_base = 0, u_base = 0;
  for (int r0 = 0; r0 < p.requests; r0 += kTreePlanThreads) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    TreeEntry t = {};
    int32_t blocks = 0;
    auto tiles_of = [&](int32_t block) {
      int32_t end = t.len;
      if (p.chain) {  // the block's last token sees no newer one
        const int64_t last = min(static_cast<int64_t>(t.fresh) * p.G, (block + 1) * static_cast<int64_t>(256)) - 1;
        end = min(end, t.ctx + static_cast<int32_t>(last / p.G) + 1);
      }
      return max((end + 127) / 128, 1);
    };
    int64_t e = 0, u = 0;
    if (r < p.requests) {
      const int32_t lo = p.cu[r], hi = p.cu[r + 1];
      const int32_t len = p.lens[r];
      t.request = r;
      t.first = min(max(lo, 0), p.tokens);
      t.fresh = min(max(hi, t.first), p.tokens) - t.first;
      t.len = static_cast<int32_t>(min(static_cast<int64_t>(max(len, 0)), p.most));
      t.ctx = t.len - t.fresh;
      if (p.status != nullptr) {
        if (lo < 0 || hi < lo || hi > p.tokens) atomicCAS(p.status, 0, B2G_STATUS_TOKENS);
        if (len > p.most) atomicCAS(p.status, 0, B2G_STATUS_PAGE_TABLE);
      }
      blocks = static_cast<int32_t>((static_cast<int64_t>(t.fresh) * p.G + 255) / 256);
      e = blocks;
      for (int32_t b = 0; b < blocks; ++b) u += tiles_of(b);
    }
    int64_t es = e, us = u;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t ue = __shfl_up_sync(0xffffffffu, es, d), uu = __shfl_up_sync(0xffffffffu, us, d);
      if (lane >= d) {
        es += ue;
        us += uu;
      }
    }
    __syncthreads();
    if (lane == 31) {
      warp_e[warp] = es;
      warp_u[warp] = us;
    }
    __syncthreads();
    int64_t e_sum = 0, u_sum = 0;
    for (int w = 0; w < kTreePlanThreads / 32; ++w) {
      if (w < warp) {
        es += warp_e[w];
        us += warp_u[w];
      }
      e_sum += warp_e[w];
      u_sum += warp_u[w];
    }
    int64_t at = e_base + es - e, sum = u_base + us - u;
    for (int32_t b = 0; b < blocks; ++b, ++at) {
      t.block = b;
      t.tiles = tiles_of(b);
      t.before = static_cast<int32_t>(sum);
      sum += t.tiles;
      if (at < p.capacity) p.plan[at] = t;
      if (at < kTreePlanShared) before[at] = t.before;
    }
    e_base += e_sum;
    u_base += u_sum;
  }
  __syncthreads();
  // offsets that decrease can ask for more blocks than there is room for
  const int32_t entries = static_cast<int32_t>(min(e_base, static_cast<int64_t>(p.capacity)));
  if (entries < e_base) u_base = p.plan[entries - 1].before + p.plan[entries - 1].tiles;
  const int64_t units = u_base * p.HK;
  if (threadIdx.x == 0) {
    p.meta->entries = entries;
    p.meta->units = units;
  }
  const int64_t ctas = min(units, static_cast<int64_t>(p.ctas));
  for (int c = threadIdx.x; c < ctas; c += kTreePlanThreads) {
    const int64_t u = units * c / ctas;
    int lo = 0, hi = entries - 1;  // the last entry that begins at or before u
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      const int64_t b = mid < kTreePlanShared ? before[mid] : p.plan[mid].before;
      if (b * p.HK <= u) lo = mid;
      else hi = mid - 1;
    }
    const int64_t in = u - static_cast<int64_t>(p.plan[lo].before) * p.HK;
    const int32_t tiles = p.plan[lo].tiles;
    p.start[c] = make_int4(lo, static_cast<int32_t>(in / tiles), static_cast<int32_t>(in % tiles), 0);
  }
}

// ----------------------------------------------------------------- kernel --
// The part of one (block, key/value head) that lies in this CTA's share.
struct Segment {
  TreeEntry e;
  int32_t entry, hk;
  int32_t j0, j1;   // tiles
  int32_t row0, rows;
  bool two;         // above 128 rows: a row tile per warpgroup
  uint32_t slots;   // warpgroups with tiles to visit
};

// Walks a share: the segments of `left` units from (entry, hk, tile).
struct SegmentWalk {
  int32_t entry, hk, tile;
  int64_t left;

  __device__ __forceinline__ bool next(const TreeParams& p, Segment& s) {
    if (left <= 0) return false;
    const int4* src = reinterpret_cast<const int4*>(p.plan + entry);
    const int4 a = src[0], b = src[1];
    s.e.request = a.x;
    s.e.block = a.y;
    s.e.tiles = a.z;
    s.e.before = a.w;
    s.e.ctx = b.x;
    s.e.fresh = b.y;
    s.e.first = b.z;
    s.e.len = b.w;
    s.entry = entry;
    s.hk = hk;
    s.j0 = tile;
    s.j1 = static_cast<int32_t>(min(static_cast<int64_t>(s.e.tiles), tile + left));
    left -= s.j1 - s.j0;
    s.row0 = s.e.block * 256;
    s.rows = min(256, s.e.fresh * p.G - s.row0);
    s.two = s.rows > 128;
    s.slots = s.two || s.j1 - s.j0 > 1 ? 2u : 1u;
    tile = 0;
    if (++hk == p.HK) {
      hk = 0;
      ++entry;
    }
    return true;
  }
};

// Bits of the 32 keys from kb on that new token i of the segment's request sees.
__device__ __forceinline__ uint32_t seen_bits(const TreeParams& p, const TreeEntry& e, int32_t i,
                                              int32_t kb) {
  auto low = [](int32_t n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; };
  const int32_t r = kb - e.ctx;  // rank of the first key among the new ones
  if (p.mask == nullptr) return low(min(i + 1, e.fresh) - r);
  uint32_t bits = low(-r);  // older tokens
  if (r > -32) {
    const int64_t* words = p.mask + static_cast<int64_t>(e.first + i) * p.mask_words;
    auto word = [&](int32_t w) {
      return w >= 0 && w < p.mask_words ? static_cast<uint64_t>(words[w]) : 0ull;
    };
    const int32_t w = r >> 6, sh = r & 63;  // arithmetic: word -1 holds ranks -64 .. -1
    uint64_t v = word(w) >> sh;
    if (sh > 32) v |= word(w + 1) << (64 - sh);
    bits |= static_cast<uint32_t>(v) & ~low(-r);
  }
  return bits & low(e.fresh - r);
}

// Adds to n values of a row of O (of new token i, from dim d0 on) what is not
// finite among the values that the token sees; see attention.cu.
template <int D, typename T, typename OutT>
__device__ __noinline__ void add_odd_cache_values(const TreeParams& p, const Segment& s, int32_t i,
                                                  int32_t d0, int32_t n, OutT* out) {
  for (int32_t kb = s.j0 * 128; kb < min(s.j1 * 128, s.e.len); kb += 32) {
    uint32_t bits = seen_bits(p, s.e, i, kb);
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

// One tile's softmax for a thread's row: NCH chunks of 32 score columns from
// chunk c0 on, weights for those and zeros for the others into P. Keeps the
// running maximum (log2 units) and sum.
template <int D, bool kBF16, int NCH>
__device__ __forceinline__ void tree_softmax(uint32_t s_col, uint32_t o_col, uint32_t c0, float sl2,
                                             bool masked, const uint32_t (&seen)[4], bool first,
                                             float& m_run, float& l_run, uint32_t p_bar0,
                                             uint32_t p_bar1, uint32_t lane) {
  constexpr int kRegs = NCH == 4 ? 4 : NCH;
  uint32_t s[32 * kRegs];
#pragma unroll
  for (int c = 0; c < NCH; ++c)
    tmem_ld_32x32b_x32(s_col + 32u * (c0 + c), *reinterpret_cast<uint32_t(*)[32]>(&s[32 * c]));
  tmem_wait_ld();
  if (masked) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (!((seen[c] >> i) & 1u)) s[32 * c + i] = __float_as_uint(-INFINITY);
  }
  float m8[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) m8[i] = fmaxf(__uint_as_float(s[i]), __uint_as_float(s[i + 8]));
#pragma unroll
  for (int c = 16; c < 32 * NCH; c += 16)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      m8[i] = fmax3(m8[i], __uint_as_float(s[c + i]), __uint_as_float(s[c + 8 + i]));
  const float mx = fmax3(fmax3(m8[0], m8[1], m8[2]), fmax3(m8[3], m8[4], m8[5]),
                         fmaxf(m8[6], m8[7]));
  constexpr float kRescaleLog2 = 8.0f;  // see attention.cu
  const float m_cand = mx * sl2;
  const bool move = m_cand > m_run + kRescaleLog2;
  const float m_new = move ? m_cand : m_run;
  float alpha = 1.0f;
  if (move) alpha = poly_exp2(m_run - m_new);
  if (!first && __any_sync(0xffffffffu, move)) {
#pragma unroll 1
    for (uint32_t d = 0; d < static_cast<uint32_t>(D); d += 16u) {
      uint32_t o[16];
      tmem_ld_32x32b_x16(o_col + d, o);
      tmem_wait_ld();
#pragma unroll
      for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * alpha);
      tmem_st_32x32b_x16(o_col + d, o);
    }
  }
  const float off = m_new == -INFINITY ? 0.0f : -m_new;
  const float2 sl2x2 = make_float2(sl2, sl2), negm = make_float2(off, off);
  float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f),
                   make_float2(0.f, 0.f)};
  uint32_t buf[2][32];
  if constexpr (NCH == 4) tmem_ld_32x32b_x32(s_col + 64u, buf[0]);
  if constexpr (NCH < 4) {
    uint32_t zero[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) zero[i] = 0u;
#pragma unroll
    for (uint32_t c = 0; c < 4; ++c)
      if (c < c0 || c >= c0 + NCH) tmem_st_32x32b_x16(s_col + 16u * c, zero);
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    if (NCH == 4 && c == 2) {
      tmem_wait_ld();
      regs_ready(buf[0]);
      tmem_ld_32x32b_x32(s_col + 96u, buf[1]);
    }
    if (NCH == 4 && c == 3) {
      tmem_wait_ld();
      regs_ready(buf[1]);
    }
    uint32_t cur[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) cur[i] = c < 2 ? s[32 * c + i] : buf[c & 1][i];
    if (c >= 2 && masked) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (!((seen[c] >> i) & 1u)) cur[i] = __float_as_uint(-INFINITY);
    }
    uint32_t pk[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float2 x = __ffma2_rn(
          make_float2(__uint_as_float(cur[2 * i]), __uint_as_float(cur[2 * i + 1])), sl2x2, negm);
      const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
      acc[i & 3] = __fadd2_rn(acc[i & 3], e);
      pk[i] = pack2<kBF16>(e.x, e.y);
    }
    tmem_st_32x32b_x16(s_col + 16u * (c0 + static_cast<uint32_t>(c)), pk);
    if (c + 1 == NCH || (NCH == 4 && c == 1)) {
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (c == 1 || NCH < 4) mbar_arrive(p_bar0);
        if (c + 1 == NCH) mbar_arrive(p_bar1);
      }
    }
  }
  const float2 a01 = __fadd2_rn(acc[0], acc[1]), a23 = __fadd2_rn(acc[2], acc[3]);
  const float2 a = __fadd2_rn(a01, a23);
  l_run = fmaf(l_run, alpha, a.x + a.y);
  m_run = m_new;
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
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  const uint32_t bar0 = sbase + TP::kBarOff;
  const uint32_t q_full = bar0, q_empty = bar0 + 8u;
  auto full = [&](uint32_t s) { return bar0 + 8u * (2 + s); };
  auto empty = [&](uint32_t s) { return bar0 + 8u * (2 + NS + s); };
  const uint32_t bar1 = bar0 + 8u * (2 + 2 * NS);
  auto s_full = [&](uint32_t t) { return bar1 + 8u * t; };
  auto p_full = [&](uint32_t t, uint32_t half) { return bar1 + 8u * (2 + 2 * t + half); };
  auto o_done = [&](uint32_t t) { return bar1 + 8u * (6 + t); };
  auto o_free = [&](uint32_t t) { return bar1 + 8u * (8 + t); };
  const uint32_t join = bar1 + 8u * 10;
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
    mbar_init(join, TP::kSoftmaxWarps);
    *abort_flag = 0u;
    fence_mbarrier_init();
    prefetch_tensormap(&p.tmK);
    prefetch_tensormap(&p.tmV);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(tmem_slot), 512);
    tmem_relinquish<1>();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  grid_dependency_wait();  // the plan is complete

  const int64_t units = p.meta->units;
  const int32_t ctas =
      static_cast<int32_t>(min(units, static_cast<int64_t>(gridDim.x)));
  const int32_t me = static_cast<int32_t>(blockIdx.x);
  SegmentWalk walk = {0, 0, 0, 0};
  if (me < ctas) {
    const int4 st = p.start[me];
    walk.entry = st.x;
    walk.hk = st.y;
    walk.tile = st.z;
    walk.left = units * (me + 1) / ctas - units * me / ctas;
  }
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
      // this lane's page of tile j; num_pages, past the end, where there is none
      auto page_of = [&](int32_t j) {
        const int32_t key = j * 128 + static_cast<int32_t>(box) * box_rows;
        if (!issues || key >= w.e.len) return p.num_pages;
        const int32_t page = table[key / p.page_size];
        if (page >= 0 && page < p.num_pages) return page;
        fmha_report(p, B2G_STATUS_PAGE_TABLE);
        return p.num_pages;
      };
      int32_t page = page_of(w.j0);
      for (int32_t j = w.j0; alive && j < w.j1; ++j) {
        const int32_t next = j + 1 < w.j1 ? page_of(j + 1) : 0;
        const int32_t slot_row = p.page_size > 128 ? (j * 128) % p.page_size : 0;
        for (uint32_t kv = 0; kv < 2; ++kv, ++ld) {
          const uint32_t s = ld % NS;
          if (!__all_sync(0xffffffffu, fmha_wait(empty(s), ((ld / NS) & 1u) ^ 1u, abort_flag, p,
                                                 B2G_SITE_EMPTY))) {
            alive = false;
            break;
          }
          if (lane == 0) mbar_arrive_expect_tx(full(s), TP::kTile);
          __syncwarp();
          if (issues)
            tma_load_4d(sbase + TP::kRingOff + s * TP::kTile + slab * kSlabBytes +
                            box * static_cast<uint32_t>(box_rows) * 128u,
                        kv == 0 ? &p.tmK : &p.tmV, full(s), static_cast<int32_t>(slab) * 64,
                        slot_row, w.hk, page);
        }
        page = next;
      }
    }
    // every load issued lands before the CTA can exit
    for (uint32_t i = ld > NS ? ld - NS : 0u; i < ld; ++i) {
      uint32_t spins = 0;
      while (!mbar_try_wait(full(i % NS), (i / NS) & 1u) && spins < (1u << 20)) ++spins;
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------- MMA issue --
    if (lane == 0) {
      constexpr uint32_t idesc_s = fmha_idesc_s<D, kBF16>();
      constexpr uint32_t idesc_pv = fmha_idesc_pv<D, kBF16>();
      uint32_t last_bar = 0, last_par = 0;  // the newest commit: all earlier MMAs precede it
      uint32_t base = 0, ic = 0;            // ring loads before the segment, segments
      uint32_t steps[2] = {0u, 0u};         // tiles of each warpgroup (phases of s_full, p_full)
      uint32_t titems[2] = {0u, 0u};        // segments of each (phases of o_done, o_free)
      bool alive = true;
      while (alive && walk.next(p, w)) {
        const int32_t n = w.j1 - w.j0;
        auto ready = [&](uint32_t load) {
          return fmha_wait(full(load % NS), (load / NS) & 1u, abort_flag, p, B2G_SITE_FULL);
        };
        // S = Q K^T of step j for warpgroup t
        auto issue_s = [&](uint32_t t, int32_t j) {
          const uint32_t k_base =
              sbase + TP::kRingOff + ((base + 2u * static_cast<uint32_t>(j)) % NS) * TP::kTile;
          const uint32_t q_base = sbase + TP::kQOff + (w.two ? t * TP::kTile : 0u);
#pragma unroll
          for (uint32_t kk = 0; kk < D / 16; ++kk) {
            const uint64_t ad = sdesc_kmajor_sw128(q_base + (kk >> 2) * kSlabBytes) + 2u * (kk & 3u);
            const uint64_t bd = sdesc_kmajor_sw128(k_base + (kk >> 2) * kSlabBytes) + 2u * (kk & 3u);
            mma_f16<1>(tmem_base + TP::kS + t * TP::kTileCols, ad, bd, idesc_s, kk > 0 ? 1u : 0u);
          }
          tc_commit<1>(s_full(t));
          last_bar = s_full(t);
          last_par = steps[t] & 1u;
          // the tile of K is free after its last product, Q after the block's
          if (!w.two || t == 1u) {
            tc_commit<1>(empty((base + 2u * static_cast<uint32_t>(j)) % NS));
            if (j + 1 == n) tc_commit<1>(q_empty);
          }
        };
        if (!fmha_wait(q_full, ic & 1u, abort_flag, p, B2G_SITE_FULL)) break;
        for (uint32_t t = 0; t < w.slots; ++t) {
          const int32_t j = w.two ? 0 : static_cast<int32_t>(t);
          if (!ready(base + 2u * static_cast<uint32_t>(j))) {
            alive = false;
            break;
          }
          tc_fence_after();
          issue_s(t, j);
        }
        for (int32_t j = 0; alive && j < n; ++j) {
          const uint32_t v_load = base + 2u * static_cast<uint32_t>(j) + 1u;
          if (!ready(v_load)) {
            alive = false;
            break;
          }
          const uint32_t v_base = sbase + TP::kRingOff + (v_load % NS) * TP::kTile;
          const uint32_t t_begin = w.two ? 0u : static_cast<uint32_t>(j) & 1u;
          const uint32_t t_end = w.two ? 2u : t_begin + 1u;
          const int32_t next = j + (w.two ? 1 : 2);
          const bool first = w.two ? j == 0 : j < 2;
          for (uint32_t t = t_begin; alive && t < t_end; ++t) {
            const uint32_t p_col = tmem_base + TP::kS + t * TP::kTileCols;
            if (first && titems[t] > 0 &&
                !fmha_wait(o_free(t), (titems[t] - 1u) & 1u, abort_flag, p, B2G_SITE_ACC_EMPTY)) {
              alive = false;
              break;
            }
            for (uint32_t half = 0; half < 2; ++half) {
              if (!fmha_wait(p_full(t, half), steps[t] & 1u, abort_flag, p, B2G_SITE_ACC_FULL)) {
                alive = false;
                break;
              }
              tc_fence_after();
#pragma unroll
              for (uint32_t k4 = 0; k4 < 4; ++k4) {
                const uint32_t kk = half * 4u + k4;
                const uint64_t bd = sdesc_mnmajor_sw128(v_base + kk * 2048u, kSlabBytes, 1024u);
                mma_f16_ts(tmem_base + TP::kO + t * TP::kTileCols, p_col + kk * 8u, bd, idesc_pv,
                           (!first || kk > 0) ? 1u : 0u);
              }
            }
            if (!alive) break;
            ++steps[t];
            if (next >= n) {
              tc_commit<1>(o_done(t));
              last_bar = o_done(t);
              last_par = titems[t] & 1u;
              ++titems[t];
              continue;
            }
            if (!ready(base + 2u * static_cast<uint32_t>(next))) {
              alive = false;
              break;
            }
            tc_fence_after();
            issue_s(t, next);
          }
          if (alive) tc_commit<1>(empty(v_load % NS));
        }
        base += 2u * static_cast<uint32_t>(n);
        ++ic;
      }
      // all MMAs issued by this thread finish before TMEM can be freed
      if (last_bar != 0u) {
        uint32_t spins = 0;
        while (!mbar_try_wait(last_bar, last_par) && spins < (1u << 22)) ++spins;
      }
    }
  } else {
    // ------------------------------------ Q, softmax, epilogue and the join --
    const uint32_t t = (warp - 2u) >> 2;       // warpgroup
    const uint32_t quarter = warp & 3u;        // TMEM lane quarter of the warp
    const uint32_t row = quarter * 32u + lane;
    const uint32_t taddr = tmem_base + ((quarter * 32u) << 16);
    const uint32_t s_col = taddr + TP::kS + t * TP::kTileCols;
    const uint32_t o_col = taddr + TP::kO + t * TP::kTileCols;
    float2* ml = reinterpret_cast<float2*>(smem + TP::kMlOff);  // [warpgroup][quarter][lane]
    volatile uint32_t* odd_words = reinterpret_cast<volatile uint32_t*>(smem + TP::kOddOff);
    uint32_t step = 0, ti = 0;        // this warpgroup's tiles and segments
    uint32_t base = 0, ic = 0;        // ring loads before the segment, segments of the CTA
    uint32_t joins = 0;               // uses of the join barrier
    bool alive = true;
    auto wait_all = [&](uint32_t bar, uint32_t parity, int site) {
      if (__all_sync(0xffffffffu, fmha_wait(bar, parity & 1u, abort_flag, p, site)) == 0)
        alive = false;
      return alive;
    };
    // all eight warps meet
    auto meet = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(join);
      return wait_all(join, joins++, B2G_SITE_FLAG);
    };
    // blocks of this share that other shares hold parts of: the first and the last
    int32_t open_entry[2] = {-1, -1}, open_hk[2] = {0, 0};

    while (alive && walk.next(p, w)) {
      const bool whole = w.j0 == 0 && w.j1 == w.e.tiles;
      const uint32_t copies = w.two || w.rows > 64 ? 1u : w.rows > 32 ? 2u : 4u;
      const uint32_t per = 4u / copies;                  // warps of a copy
      const uint32_t copy = quarter / per;
      const int32_t lrow = static_cast<int32_t>((quarter % per) * 32u + lane);  // row in the tile
      const int32_t brow = lrow + (w.two ? static_cast<int32_t>(t) * 128 : 0);  // row in the block
      const bool real = brow < w.rows;
      const int32_t grow = w.row0 + brow;                // row of the (request, head)
      const int32_t tok = grow / p.G, head = w.hk * p.G + grow % p.G;

      // Q into shared memory: with one row tile each warpgroup copies half of every row
      if (ic > 0 && !wait_all(q_empty, ic - 1u, B2G_SITE_EMPTY)) break;
      {
        constexpr uint32_t kVecs = static_cast<uint32_t>(D) / 8;  // 16-byte pieces of a row
        const uint32_t v0 = w.two ? 0u : t * (kVecs / 2), v1 = w.two ? kVecs : v0 + kVecs / 2;
        const uint4* src = reinterpret_cast<const uint4*>(
            static_cast<const T*>(p.Q) + (w.e.first + static_cast<int64_t>(real ? tok : 0)) * p.q_t +
            (real ? head : 0) * p.q_h);
        const uint32_t dst = sbase + TP::kQOff + (w.two ? t * TP::kTile : 0u) + row * 128u;
        for (uint32_t v = v0; v < v1; v += 4) {
          uint4 x[4];
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) x[i] = real ? src[v + i] : make_uint4(0, 0, 0, 0);
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i) {
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

      float m_run = -INFINITY, l_run = 0.0f;
      uint32_t odd = 0;
      const int32_t n = w.j1 - w.j0;
      const int32_t stride = w.two ? 1 : 2;
      for (int32_t j = w.two ? 0 : static_cast<int32_t>(t); j < n; j += stride, ++step) {
        const int32_t kb = (w.j0 + j) * 128;
        const bool masked = kb + 128 > w.e.ctx;  // some row may not see some key
        // Above one copy a row's weights are zero outside its columns, so every tile
        // is looked through; above 128 rows the first warpgroup does it for both.
        if ((masked || copies > 1u) && !(w.two && t == 1u)) {
          const uint32_t load = base + 2u * static_cast<uint32_t>(j) + 1u;
          if (!wait_all(full(load % NS), load / NS, B2G_SITE_FULL)) break;
          const bool mine = clear_odd_values<D, kBF16>(
              sbase + TP::kRingOff + (load % NS) * TP::kTile + row * 128u, lane);
          const uint32_t found = __ballot_sync(0xffffffffu, mine);
          if (found != 0u) fence_proxy_async_smem();
          odd |= found;
        }
        if (!wait_all(s_full(t), step, B2G_SITE_ACC_FULL)) break;
        tc_fence_after();
        if (j + stride >= n && lane == 0) odd_words[(ic & 1u) * 8u + t * 4u + quarter] = odd;
        uint32_t seen[4] = {~0u, ~0u, ~0u, ~0u};
        const bool first = j < stride;
        const uint32_t c0 = copy * per;
        if (masked && real) {
#pragma unroll
          for (uint32_t c = 0; c < 4; ++c)
            if (c < per)
              seen[c] = seen_bits(p, w.e, tok, kb + 32 * static_cast<int32_t>(c0 + c));
        }
        if (per == 4u)
          tree_softmax<D, kBF16, 4>(s_col, o_col, 0u, p.scale_log2, masked, seen, first, m_run,
                                    l_run, p_full(t, 0), p_full(t, 1), lane);
        else if (per == 2u)
          tree_softmax<D, kBF16, 2>(s_col, o_col, c0, p.scale_log2, masked, seen, first, m_run,
                                    l_run, p_full(t, 0), p_full(t, 1), lane);
        else
          tree_softmax<D, kBF16, 1>(s_col, o_col, c0, p.scale_log2, masked, seen, first, m_run,
                                    l_run, p_full(t, 0), p_full(t, 1), lane);
      }
      if (!alive) break;

      const bool active = t < w.slots;
      if (active) {
        if (!wait_all(o_done(t), ti, B2G_SITE_ACC_FULL)) break;
        tc_fence_after();
        ++ti;
      }
      // where the rows go: O, or this share's unfinished rows
      const int32_t part_id = 2 * me + (w.j0 == 0 ? 1 : 0);
      float* part = p.part + static_cast<int64_t>(part_id) * p.part_rows * D;
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
      if (w.two) {
        uint32_t o[D];
#pragma unroll
        for (uint32_t d = 0; d < static_cast<uint32_t>(D); d += 32u)
          tmem_ld_32x32b_x32(o_col + d, *reinterpret_cast<uint32_t(*)[32]>(&o[d]));
        tmem_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(o_free(t));
        const volatile uint32_t* m = odd_words + (ic & 1u) * 8u;
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
            float* dst = part + static_cast<int64_t>(brow) * D;
#pragma unroll
            for (int v = 0; v < D / 4; ++v)
              reinterpret_cast<uint4*>(dst)[v] =
                  make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
            if (any_odd) add_odd_cache_values<D, T>(p, w, tok, 0, D, dst);
          }
        }
      } else {
        // the copies and the two warpgroups meet: maxima and sums first, then O in
        // column chunks through shared memory, already scaled by the writers
        ml[(t * 4u + quarter) * 32u + lane] = make_float2(m_run, l_run);
        if (!meet()) break;
        const volatile uint32_t* ow = odd_words + (ic & 1u) * 8u;
        bool any_odd = (ow[0] | ow[1] | ow[2] | ow[3]) != 0u;
        if (w.slots == 2u) any_odd |= (ow[4] | ow[5] | ow[6] | ow[7]) != 0u;
        float m_tot = -INFINITY, l_tot = 0.0f;
        for (uint32_t c = 0; c < w.slots * copies; ++c)
          m_tot = fmaxf(m_tot, ml[((c / copies) * 4u + (c % copies) * per + quarter % per) * 32u + lane].x);
        for (uint32_t c = 0; c < w.slots * copies; ++c) {
          const float2 x = ml[((c / copies) * 4u + (c % copies) * per + quarter % per) * 32u + lane];
          if (m_tot > -INFINITY) l_tot = fmaf(x.y, fast_exp2(x.x - m_tot), l_tot);
        }
        float scale = m_tot > -INFINITY ? fast_exp2(m_run - m_tot) : 0.0f;
        if (whole) scale = l_tot == 0.0f ? 0.0f : scale / l_tot;
        if (t == 0u && copy == 0u && real) store_sums(m_tot, l_tot);
        constexpr uint32_t JC = TP::kJoinCols, JV = JC / 4;  // columns, float4s of a row and round
        const uint32_t buf = sbase + TP::kJoinOff;
        // float4 v of row r: the rows of eight lanes spread over the banks
        auto at = [&](uint32_t wq, uint32_t r, uint32_t v) {
          return buf + ((wq * 32u + r) * JV + (v ^ (r & (JV - 1u)))) * 16u;
        };
        for (uint32_t d = 0; d < static_cast<uint32_t>(D); d += JC) {
          if (active) {
            uint32_t o[JC];
            if constexpr (JC == 32) tmem_ld_32x32b_x32(o_col + d, *reinterpret_cast<uint32_t(*)[32]>(&o[0]));
            else tmem_ld_32x32b_x16(o_col + d, *reinterpret_cast<uint32_t(*)[16]>(&o[0]));
            tmem_wait_ld();
            if (d + JC == static_cast<uint32_t>(D)) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(o_free(t));
            }
            if (real) {
#pragma unroll
              for (uint32_t v = 0; v < JV; ++v) {
                uint32_t x[4];
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i)
                  x[i] = __float_as_uint(__uint_as_float(o[4 * v + i]) * scale);
                st_shared_v4(at(t * 4u + quarter, lane, v), x);
              }
            }
          }
          if (!meet()) break;
          // four columns of one row to a thread
          for (uint32_t i = threadIdx.x - 64u; i < static_cast<uint32_t>(w.rows) * JV; i += 256u) {
            const uint32_t r = i / JV, v = i % JV;
            float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
            for (uint32_t c = 0; c < w.slots * copies; ++c) {
              uint32_t x[4];
              ld_shared_v4(at((c / copies) * 4u + (c % copies) * per + (r >> 5), r & 31u, v), x);
              sum.x += __uint_as_float(x[0]);
              sum.y += __uint_as_float(x[1]);
              sum.z += __uint_as_float(x[2]);
              sum.w += __uint_as_float(x[3]);
            }
            const int32_t g = w.row0 + static_cast<int32_t>(r), tk = g / p.G;
            const int32_t col = static_cast<int32_t>(d + 4u * v);
            if (whole) {
              T* dst = static_cast<T*>(p.O) + static_cast<int64_t>(w.e.first + tk) * p.o_t +
                       (w.hk * p.G + g % p.G) * p.o_h + col;
              *reinterpret_cast<uint2*>(dst) =
                  make_uint2(pack2<kBF16>(sum.x, sum.y), pack2<kBF16>(sum.z, sum.w));
              if (any_odd) add_odd_cache_values<D, T>(p, w, tk, col, 4, dst);
            } else {
              float* dst = part + static_cast<int64_t>(r) * D + col;
              *reinterpret_cast<float4*>(dst) = sum;
              if (any_odd) add_odd_cache_values<D, T>(p, w, tk, col, 4, dst);
            }
          }
          if (!meet()) break;  // the buffer is free again
        }
        if (!alive) break;
      }
      if (!whole) {
        // publish: every warp's rows are written, then the owner's count goes up
        if (!meet()) break;
        const int64_t u0 = static_cast<int64_t>(w.e.before) * p.HK + static_cast<int64_t>(w.hk) * w.e.tiles;
        if (warp == 2u && lane == 0) {
          __threadfence();
          atomicAdd(&p.counters[2 * share_of(u0, units, ctas)], 1u);
        }
        const int slot = w.j1 == w.e.tiles ? 0 : 1;
        open_entry[slot] = w.entry;
        open_hk[slot] = w.hk;
      }
      base += 2u * static_cast<uint32_t>(n);
      ++ic;
    }

    // The blocks that this share had a part of: when every part is published, each
    // of the CTAs joins its slice of the block's values, in the order of the shares.
#pragma unroll 1
    for (int slot = 0; alive && slot < 2; ++slot) {
      if (open_entry[slot] < 0) continue;
      const TreeEntry e = p.plan[open_entry[slot]];
      const int32_t hk = open_hk[slot];
      const int64_t u0 = static_cast<int64_t>(e.before) * p.HK + static_cast<int64_t>(hk) * e.tiles;
      const int32_t owner = share_of(u0, units, ctas);
      const int32_t parts = share_of(u0 + e.tiles - 1, units, ctas) - owner + 1;
      uint32_t* count = p.counters + 2 * owner;
      bool there = true;
      if (lane == 0) {
        const uint64_t t0 = globaltimer_ns();
        while (ld_acquire_gpu(count) < static_cast<uint32_t>(parts)) {
          if (*abort_flag != 0u || globaltimer_ns() - t0 > p.timeout_ns) {
            fmha_report(p, B2G_STATUS_TIMEOUT | B2G_SITE_FLAG);
            *abort_flag = 1u;
            there = false;
            break;
          }
        }
      }
      if (!__all_sync(0xffffffffu, there)) {
        alive = false;
        break;
      }
      const int32_t row0 = e.block * 256, rows = min(256, e.fresh * p.G - row0);
      constexpr int32_t kV = D / 4;
      const int64_t all = static_cast<int64_t>(rows) * kV;
      const int32_t k = me - owner;
      const int64_t stop = all * (k + 1) / parts;
      for (int64_t i = all * k / parts + (threadIdx.x - 64u); i < stop; i += 256) {
        const int32_t r = static_cast<int32_t>(i / kV), v = static_cast<int32_t>(i % kV);
        auto id = [&](int32_t c) { return static_cast<int64_t>(c == 0 ? 2 * owner + 1 : 2 * (owner + c)); };
        float m = -INFINITY;
#pragma unroll 4
        for (int32_t c = 0; c < parts; ++c) m = fmaxf(m, __ldcg(&p.part_ml[id(c) * p.part_rows + r]).x);
        float l = 0.0f;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        if (m > -INFINITY) {
#pragma unroll 4
          for (int32_t c = 0; c < parts; ++c) {
            const float2 x = __ldcg(&p.part_ml[id(c) * p.part_rows + r]);
            const float4 o = __ldcg(reinterpret_cast<const float4*>(
                p.part + (id(c) * p.part_rows + r) * D) + v);
            const float f = fast_exp2(x.x - m);
            l = fmaf(x.y, f, l);
            sum.x = fmaf(o.x, f, sum.x);
            sum.y = fmaf(o.y, f, sum.y);
            sum.z = fmaf(o.z, f, sum.z);
            sum.w = fmaf(o.w, f, sum.w);
          }
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const int32_t g = row0 + r, tk = g / p.G, h = hk * p.G + g % p.G;
        T* dst = static_cast<T*>(p.O) + static_cast<int64_t>(e.first + tk) * p.o_t + h * p.o_h + 4 * v;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<kBF16>(sum.x * inv, sum.y * inv),
                                                    pack2<kBF16>(sum.z * inv, sum.w * inv));
        if (v == 0 && p.lse != nullptr)
          p.lse[static_cast<int64_t>(h) * p.tokens + e.first + tk] =
              l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.693147180559945309f;
      }
      // the last CTA to have read the parts leaves both counts at zero
      if (!meet()) break;
      if (warp == 2u && lane == 0) {
        __threadfence();
        if (atomicAdd(&count[1], 1u) + 1u == static_cast<uint32_t>(parts)) {
          count[0] = 0u;
          count[1] = 0u;
        }
      }
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
  size_t meta, start, plan, part, part_ml, total;
  int64_t capacity;  // row blocks
  int32_t part_rows;
};

TreeWorkspace tree_workspace(int requests, int64_t tokens, int group, int head_dim, int sms) {
  TreeWorkspace w;
  auto up = [](size_t v) { return (v + 255) & ~static_cast<size_t>(255); };
  w.capacity = tokens * group / 256 + std::min<int64_t>(requests, tokens);
  w.part_rows = static_cast<int32_t>(std::min<int64_t>(256, tokens * group));
  w.meta = workspace_flag_bytes(sms);
  w.start = w.meta + 256;
  w.plan = w.start + up(sizeof(int4) * static_cast<size_t>(sms));
  w.part_ml = w.plan + up(sizeof(TreeEntry) * static_cast<size_t>(w.capacity));
  w.part = w.part_ml + up(sizeof(float2) * 2 * static_cast<size_t>(sms) * w.part_rows);
  w.total = w.part + sizeof(float) * 2 * static_cast<size_t>(sms) * w.part_rows * head_dim;
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
  // them have to be resident
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(sms), 1, 1);
  cfg.blockDim = dim3(TP::kThreads, 1, 1);
  cfg.dynamicSmemBytes = TP::kDynBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
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
  return b2g::tree_workspace(requests, tokens, heads_q / heads_k, head_dim, sms).total;
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
  const TreeWorkspace wl = tree_workspace(requests, tokens, group, head_dim, sms);
  if (workspace == nullptr || workspace_bytes < wl.total) return B2G_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return B2G_EALIGN;
  uint8_t* ws = static_cast<uint8_t*>(workspace);

  TreeParams prm;
  std::memset(&prm, 0, sizeof(prm));
  if (!encode_cache(&prm.tmK, k_cache, dtype, head_dim, page_size, heads_k, num_pages, strides + 2) ||
      !encode_cache(&prm.tmV, v_cache, dtype, head_dim, page_size, heads_k, num_pages, strides + 5))
    return B2G_ETENSORMAP;
  TreePlanParams pl;
  pl.cu = cu_seqlens;
  pl.lens = seq_lens;
  pl.plan = reinterpret_cast<TreeEntry*>(ws + wl.plan);
  pl.meta = reinterpret_cast<TreeMeta*>(ws + wl.meta);
  pl.start = reinterpret_cast<int4*>(ws + wl.start);
  pl.status = status;
  pl.most = std::min<int64_t>(static_cast<int64_t>(max_pages) * page_size, INT_MAX - 256);
  pl.requests = requests;
  pl.tokens = static_cast<int32_t>(tokens);
  pl.G = group;
  pl.HK = heads_k;
  pl.capacity = static_cast<int32_t>(wl.capacity);
  pl.ctas = sms;
  pl.chain = tree_mask == nullptr;
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
  prm.plan = pl.plan;
  prm.meta = pl.meta;
  prm.start = pl.start;
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
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  tree_plan_kernel<<<1, kTreePlanThreads, 0, s>>>(pl);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return static_cast<int>(e);
  const bool bf16 = dtype == B2G_DT_BF16;
  if (head_dim == 128)
    return bf16 ? launch_tree<128, true>(prm, sms, s) : launch_tree<128, false>(prm, sms, s);
  return bf16 ? launch_tree<64, true>(prm, sms, s) : launch_tree<64, false>(prm, sms, s);
}
