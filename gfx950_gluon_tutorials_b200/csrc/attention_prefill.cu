// Causal attention over packed prompts for sm_100a: row i of a prompt sees keys
// j <= i. The CTA is that of attention.cu: TMA producer, MMA issuer and two softmax
// warpgroups, each with its 128-row query tile, TMEM scores and accumulator.
//
// Items. A 128-row tile that starts at row m of its prompt needs m / 128 + 1 KV
// tiles, of which only the last is masked, by a triangle (which hides the keys past
// the prompt's end too: they lie after every row that is stored). What the two
// warpgroups work on at one time depends on the heads:
//   - kHeads: the same 128 rows of two query heads. With an even number of query
//     heads per key/value head they share K and V, and both end with the same tile,
//     so neither waits for the other and a prompt's ragged end leaves none idle.
//   - kRows: two 128-row tiles of one head, for an odd number of heads per
//     key/value head, where neighbouring heads would need two tiles of K and V (one
//     prompt of 12031 tokens, 24 heads of 128 not grouped: 860 us so, 1199 with two
//     heads and their own K and V each).
//   - with an odd number, blocks of up to 128 rows are kHeads items too, whose heads
//     may then differ in K and V: every KV tile takes two ring stages.
// The blocks are listed in order of falling work and dealt to the CTAs in turns of
// alternating direction, which evens out their sums. Up to kOwnBlocks of them every
// CTA makes the list for itself (one prompt of 61 tokens: 8.3 us on the GPU against 9.8
// with a planning launch; 256 blocks are compared with one another in about as long as
// the launch takes), above that a planning kernel does.
//
// What bounds it: the two products and the exponentials of a tile, as in
// attention.cu, and for short prompts the hand-over from item to item. 12031 tokens,
// 32 heads over 8, 128: 945-1078 us (1250-1100 TFLOPS; the power cap moves it, 1689 is
// the measured rate of a plain product); 24 prompts of 1 to 1100 tokens 144 us per call, 128
// in a replayed graph whose inputs stay in L2; 96 of up to 300, 24 heads of 64: 73-74 us
// either way (1.8 TB/s of what has to move). Measured and
// not kept: half of a row's columns to each of two threads (16 softmax warps) 1213-1341
// us for the first; one wait for all of P instead of one for each half, 5-8 % slower; a
// quarter of the exponentials as poly_exp2, no gain at 128 and 9 % at 64, for a sum of
// weights that is right to 1e-5 only.
//
// What is masked must not count whatever it holds, and 0 * NaN would: the keys of
// the last KV tile may be another prompt's, or later tokens of the same one. So
// the softmax warps look through that tile of V before its PV product, set what
// is not finite to zero, and the epilogue adds it to the rows that do see it.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cstring>
#include <type_traits>

#include "attention_common.cuh"

namespace b2g {

struct alignas(64) PrefillParams {
  CUtensorMap tmQ, tmK, tmV;  // 4-D (d, token, head, 1), 64 x 128 x 1 x 1 boxes, 128B swizzle
  void* O;
  int64_t o_t, o_h;
  const void* V;
  int64_t v_t, v_h;
  float* lse;                 // [HQ][tokens] or null
  int* status;
  const int32_t* cu;
  const int4* plan;           // blocks: {first token, its row in the prompt, prompt's rows, 0}; null: own list
  const int2* counts;         // kRows blocks (first in the plan), kHeads blocks
  int32_t HQ, G, tokens, prompts, block;
  uint32_t hq_inv, pairs_inv;  // 2^32 / HQ and / (head pairs), rounded up; 0: divide
  float scale_log2;
  uint64_t timeout_ns;
};

constexpr uint32_t kOwnBlocks = 256;   // most blocks that a CTA lists for itself
constexpr int32_t kPlanLevels = 4096;  // levels of work: KV tiles of 128 keys, half a million tokens

template <int D>
struct PrefillPlan {
  static constexpr uint32_t kSoftmaxWarps = 8;
  static constexpr uint32_t kThreads = 64 + 32 * kSoftmaxWarps;
  static constexpr uint32_t kSlabs = D / 64;
  static constexpr uint32_t kTile = kSlabs * kSlabBytes;
  static constexpr uint32_t kStages = D == 128 ? 2 : 4;  // depth of the K ring and of the V ring
  static constexpr uint32_t kQOff = 0;                   // Q0, Q1
  static constexpr uint32_t kKOff = kQOff + 2 * kTile;
  static constexpr uint32_t kVOff = kKOff + kStages * kTile;
  static constexpr uint32_t kBarOff = kVOff + kStages * kTile;
  // q_full, q_empty, k_full[S], k_empty[S], v_full[S], v_empty[S], s_full[2],
  // p_full[2][2] (tile, key half), o_done[2], o_free[2]
  static constexpr uint32_t kNumBars = 2 + 4 * kStages + 10;
  static constexpr uint32_t kMiscOff = kBarOff + kNumBars * 8;  // tmem slot, abort flag
  static constexpr uint32_t kOddOff = kMiscOff + 16;            // [3][2 items][4 warps], see odd_words
  // a CTA's own list: int4 sorted[kOwnBlocks], unsorted[kOwnBlocks], int32 keys[kOwnBlocks]
  static constexpr uint32_t kListOff = (kOddOff + 96 + 15) / 16 * 16;
  static constexpr uint32_t kStoreOff = (kListOff + kOwnBlocks * 36 + 127) / 128 * 128;
  static constexpr uint32_t kBytes = kStoreOff + kSoftmaxWarps * 2048;  // [warps][32 rows][32 values]
  static constexpr uint32_t kDynBytes = kBytes + 1024;  // + alignment slack
  static constexpr uint32_t kS = 0, kO = 256, kTileCols = 128;  // TMEM columns, as in attention.cu
  static_assert(kDynBytes <= 232448, "shared memory");
};

// Adds the values that are not finite of tokens [t0, t1) of V, which the product
// left out, to a stored row of O. The weights that multiply them are positive, so
// they carry over as they are.
template <int D, typename T>
__device__ __noinline__ void add_odd_values(const PrefillParams& p, int32_t t0, int32_t hk,
                                            int32_t t1, T* orow) {
  for (int32_t t = t0; t < t1; ++t) {
    const T* v = static_cast<const T*>(p.V) + hk * p.v_h + t * p.v_t;
    for (int d = 0; d < D; ++d) {
      const float x = static_cast<float>(v[d]);
      if (!isfinite(x)) orow[d] = static_cast<T>(static_cast<float>(orow[d]) + x);
    }
  }
}

// ------------------------------------------------------------------- plan --
// The blocks of all prompts in order of falling work (KV tiles), kRows blocks
// first, by a counting sort over kPlanLevels work levels each: blocks of equal level
// come in any order, and longer prompts than the levels reach share the first. One
// CTA; latency-bound (three passes over the offsets). The order only decides which
// CTA works when, never a result.
constexpr int kPlanThreads = 1024;

// Rows of prompt b and its first token. Offsets are 0 <= cu[0] <= cu[1] <= ... <= tokens;
// others are cut to that and reported.
__device__ __forceinline__ int32_t prompt_rows(const int32_t* cu, int b, int32_t tokens,
                                               int* status, int32_t& begin) {
  const int32_t lo = cu[b], hi = cu[b + 1];
  begin = min(max(lo, 0), tokens);
  if ((lo < 0 || hi < lo || hi > tokens) && status != nullptr)
    atomicCAS(status, 0, B2G_STATUS_TOKENS);
  return min(max(hi, begin), tokens) - begin;
}

// Where the block at `row` of a prompt belongs: kRows blocks first, falling work is
// rising level.
__device__ __forceinline__ int32_t block_level(int32_t row, int32_t rows, int32_t block) {
  const bool two = block == 256 && rows - row > 128;
  const int32_t kv = row / 128 + (two ? 2 : 1);
  return kPlanLevels - min(kv, kPlanLevels) + (two ? 0 : kPlanLevels);
}

struct PackedPlanParams {
  const int32_t* cu;
  int4* plan;
  int2* counts;
  int* status;
  int32_t prompts, tokens;
  int32_t capacity;  // of plan; only offsets that decrease can ask for more
  int32_t block;     // rows of a block: 128 (all kHeads), or 256 (kRows, and kHeads up to 128)
};

__global__ void __launch_bounds__(kPlanThreads) packed_plan_kernel(const PackedPlanParams p) {
  __shared__ int32_t level[2 * kPlanLevels];  // blocks of a level, then where they go
  __shared__ int32_t warp_sum[kPlanThreads / 32];
  __shared__ int64_t warp_asked[kPlanThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  grid_launch_dependents();
  for (int i = threadIdx.x; i < 2 * kPlanLevels; i += kPlanThreads) level[i] = 0;
  __syncthreads();
  // a warp to a prompt, a lane to a block
  int64_t asked = 0;
  for (int b = warp; b < p.prompts; b += kPlanThreads / 32) {
    int32_t begin;
    const int32_t rows = prompt_rows(p.cu, b, p.tokens, p.status, begin);
    asked += (rows + p.block - 1) / p.block;
    for (int32_t row = lane * p.block; row < rows; row += 32 * p.block)
      atomicAdd(&level[block_level(row, rows, p.block)], 1);
  }
  if (lane == 0) warp_asked[warp] = asked;
  __syncthreads();
  // Offsets that decrease can ask for more blocks than the 32-bit sums below hold, whose
  // places in the plan would then mean nothing: no block is run.
  asked = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) asked += warp_asked[w];
  if (asked > INT_MAX) {
    if (threadIdx.x == 0) *p.counts = make_int2(0, 0);
    return;
  }
  // exclusive sums over the levels, eight to a thread
  constexpr int kPer = 2 * kPlanLevels / kPlanThreads;
  int32_t mine[kPer], sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    mine[i] = sum;
    sum += level[threadIdx.x * kPer + i];
  }
  int32_t upto = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int32_t u = __shfl_up_sync(0xffffffffu, upto, d);
    if (lane >= d) upto += u;
  }
  if (lane == 31) warp_sum[warp] = upto;
  __syncthreads();
  int32_t base = upto - sum, total = 0, twos = 0;
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w < warp) base += warp_sum[w];
    total += warp_sum[w];
    if (w < kPlanThreads / 64) twos += warp_sum[w];  // the first half of the levels
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i) level[threadIdx.x * kPer + i] = base + mine[i];
  if (threadIdx.x == 0) {
    twos = min(twos, p.capacity);
    *p.counts = make_int2(twos, min(total, p.capacity) - twos);
  }
  __syncthreads();
  for (int b = warp; b < p.prompts; b += kPlanThreads / 32) {
    int32_t begin;
    const int32_t rows = prompt_rows(p.cu, b, p.tokens, p.status, begin);
    for (int32_t row = lane * p.block; row < rows; row += 32 * p.block) {
      const int32_t at = atomicAdd(&level[block_level(row, rows, p.block)], 1);
      if (at < p.capacity) p.plan[at] = make_int4(begin + row, row, rows, 0);
    }
  }
}

// The same list, made by one CTA of the attention kernel for itself: up to kOwnBlocks
// blocks of at most as many prompts as it has threads. All CTAs have to come to the
// same order, so blocks of equal level keep the order of the prompts: a block's place
// is the number of blocks before it. Returns the counts; all threads take part.
template <int kThreads>
__device__ __forceinline__ int2 list_own_blocks(const PrefillParams& p, int4* sorted, int4* raw,
                                                int32_t* keys) {
  static_assert(kOwnBlocks <= kThreads, "one block to a thread");
  __shared__ int32_t warp_sum[kThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = static_cast<int>(threadIdx.x);
  int32_t begin = 0, rows = 0;
  if (b < p.prompts)
    rows = prompt_rows(p.cu, b, p.tokens, blockIdx.x == 0 ? p.status : nullptr, begin);
  const int32_t n = (rows + p.block - 1) / p.block;
  int32_t at = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int32_t up = __shfl_up_sync(0xffffffffu, at, d);
    if (lane >= d) at += up;
  }
  if (lane == 31) warp_sum[warp] = at;
  __syncthreads();
  int32_t total = 0;
  for (int w = 0; w < kThreads / 32; ++w) {
    if (w < warp) at += warp_sum[w];
    total += warp_sum[w];
  }
  total = min(total, static_cast<int32_t>(kOwnBlocks));  // decreasing offsets can ask for more
  at -= n;
  for (int32_t i = 0; i < n && at + i < total; ++i) {
    raw[at + i] = make_int4(begin + i * p.block, i * p.block, rows, 0);
    keys[at + i] = block_level(i * p.block, rows, p.block);
  }
  __syncthreads();
  const bool mine = b < total;
  const int32_t key = mine ? keys[b] : 0;
  if (mine) {
    int32_t place = 0;
#pragma unroll 4
    for (int32_t f = 0; f < total; ++f) {
      const int32_t other = keys[f];
      place += other < key || (other == key && f < b) ? 1 : 0;
    }
    sorted[place] = raw[b];
  }
  const int32_t twos = __syncthreads_count(mine && key < kPlanLevels);
  return make_int2(twos, total - twos);
}

// ----------------------------------------------------------------- kernel --
// What the two warpgroups work on: up to two query tiles ("slots").
struct PrefillItem {
  int32_t m0, k0;    // first token of the rows, of the prompt
  int32_t rows;      // of the prompt from m0 on
  int32_t head;      // of slot 0
  int32_t n;         // KV tiles of the last slot
  uint32_t slots;
  bool by_rows;      // slot 1: the next 128 rows, not the next head
  bool shared;       // one K and V for both

  __device__ __forceinline__ int32_t tiles(uint32_t t) const {
    return by_rows && slots == 2u && t == 0u ? n - 1 : n;
  }
  __device__ __forceinline__ int32_t row0(uint32_t t) const {
    return m0 + (by_rows ? static_cast<int32_t>(t) * 128 : 0);
  }
  __device__ __forceinline__ int32_t head_of(uint32_t t) const {
    return head + (by_rows ? 0 : static_cast<int32_t>(t));
  }
  // ring stage of slot t's KV tile j, and stages of the item
  __device__ __forceinline__ uint32_t stage(uint32_t t, int32_t j) const {
    return static_cast<uint32_t>(shared ? j : 2 * j + static_cast<int32_t>(t));
  }
  __device__ __forceinline__ uint32_t stages() const {
    return static_cast<uint32_t>(shared ? n : 2 * n);
  }
};

// n / d with inv = 2^32 / d rounded up, exact while n d < 2^32, or 0.
__device__ __forceinline__ int32_t quotient(int32_t n, int32_t d, uint32_t inv) {
  return inv != 0u ? static_cast<int32_t>(__umulhi(static_cast<uint32_t>(n), inv)) : n / d;
}

// Walks a CTA's items. What it needs of the list stays in shared memory or is
// prefetched an item ahead: registers are the softmax's.
struct PrefillWalk {
  int32_t item;
  uint32_t turn;

  __device__ __forceinline__ bool next(const PrefillParams& p, const int4* own, const int2* counts,
                                       PrefillItem& w) {
    const int4* list = p.plan == nullptr ? own : p.plan;
    const int32_t pairs = (p.HQ + 1) / 2, row_blocks = counts->x, row_items = row_blocks * p.HQ;
    const int32_t items = row_items + counts->y * pairs;
    auto block_of = [&](int32_t i) {
      return i < row_items ? quotient(i, p.HQ, p.hq_inv)
                           : row_blocks + quotient(i - row_items, pairs, p.pairs_inv);
    };
    if (item >= items) return false;
    const int32_t block = block_of(item);
    const int4 e = list[block];
    w.by_rows = item < row_items;
    w.m0 = e.x;
    w.k0 = e.x - e.y;
    w.rows = e.z - e.y;
    if (w.by_rows) {
      w.head = item - block * p.HQ;
      w.slots = 2;
      w.shared = true;
      w.n = e.y / 128 + 2;
    } else {
      w.head = 2 * (item - row_items - (block - row_blocks) * pairs);
      w.slots = w.head + 1 < p.HQ ? 2u : 1u;
      w.shared = (p.G & 1) == 0 || w.slots == 1u || w.head / p.G == (w.head + 1) / p.G;
      w.n = e.y / 128 + 1;
    }
    const int32_t g = static_cast<int32_t>(gridDim.x), c = static_cast<int32_t>(blockIdx.x);
    item += (turn & 1u) ? 2 * c + 1 : 2 * (g - c) - 1;
    ++turn;
    if (p.plan != nullptr && item < items)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(p.plan + block_of(item)));
    return true;
  }
};

template <int D, bool kBF16>
__global__ void __launch_bounds__(PrefillPlan<D>::kThreads, 1)
    prefill_kernel(const __grid_constant__ PrefillParams p) {
  using PP = PrefillPlan<D>;
  using T = typename std::conditional<kBF16, __nv_bfloat16, __half>::type;
  constexpr uint32_t KS = PP::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  const uint32_t sbase = smem_u32(smem);
  const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;

  const uint32_t bar0 = sbase + PP::kBarOff;
  const uint32_t q_full = bar0, q_empty = bar0 + 8u;  // q_empty: the item's last S is done with Q
  auto k_full = [&](uint32_t s) { return bar0 + 8u * (2 + s); };
  auto k_empty = [&](uint32_t s) { return bar0 + 8u * (2 + KS + s); };
  auto v_full = [&](uint32_t s) { return bar0 + 8u * (2 + 2 * KS + s); };
  auto v_empty = [&](uint32_t s) { return bar0 + 8u * (2 + 3 * KS + s); };
  const uint32_t bar1 = bar0 + 8u * (2 + 4 * KS);
  auto s_full = [&](uint32_t t) { return bar1 + 8u * t; };
  auto p_full = [&](uint32_t t, uint32_t half) { return bar1 + 8u * (2 + 2 * t + half); };
  auto o_done = [&](uint32_t t) { return bar1 + 8u * (6 + t); };
  auto o_free = [&](uint32_t t) { return bar1 + 8u * (8 + t); };  // the epilogue has read O
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + PP::kMiscOff);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(smem + PP::kMiscOff + 4);

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (uint32_t s = 0; s < KS; ++s) {
      mbar_init(k_full(s), 1);
      mbar_init(k_empty(s), 1);
      mbar_init(v_full(s), 1);
      mbar_init(v_empty(s), 1);
    }
    for (uint32_t t = 0; t < 2; ++t) {
      mbar_init(s_full(t), 1);
      mbar_init(p_full(t, 0), 4);  // one arrival per softmax warp of the slot
      mbar_init(p_full(t, 1), 4);
      mbar_init(o_done(t), 1);
      mbar_init(o_free(t), 4);
    }
    *abort_flag = 0u;
    fence_mbarrier_init();
    prefetch_tensormap(&p.tmQ);
    prefetch_tensormap(&p.tmK);
    prefetch_tensormap(&p.tmV);
  }
  if (warp == 1) {
    tmem_alloc<1>(smem_u32(tmem_slot), 512);
    tmem_relinquish<1>();
  }
  int4* own_list = reinterpret_cast<int4*>(smem + PP::kListOff);
  int2* counts = reinterpret_cast<int2*>(smem + PP::kMiscOff + 8);
  if (p.plan == nullptr) {
    const int2 c = list_own_blocks<PP::kThreads>(
        p, own_list, own_list + kOwnBlocks, reinterpret_cast<int32_t*>(own_list + 2 * kOwnBlocks));
    if (threadIdx.x == 0) *counts = c;
  } else {
    grid_dependency_wait();  // the plan is complete
    if (threadIdx.x == 0) *counts = *p.counts;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
  PrefillWalk walk = {static_cast<int32_t>(blockIdx.x), 0u};
  PrefillItem w;

  if (warp == 0) {
    // ------------------------------------------------------------ producer --
    if (lane == 0) {
      uint32_t base = 0, ic = 0;  // ring stages before the item, items
      uint32_t nk = 0, nv = 0;    // K and V loads issued
      bool alive = true;
      while (alive && walk.next(p, own_list, counts, w)) {
        if (ic > 0 && !fmha_wait(q_empty, (ic - 1u) & 1u, abort_flag, p, B2G_SITE_EMPTY)) break;
        mbar_arrive_expect_tx(q_full, w.slots * PP::kTile);
        for (uint32_t t = 0; t < w.slots; ++t)
          for (uint32_t r = 0; r < PP::kSlabs; ++r)
            tma_load_4d(sbase + PP::kQOff + t * PP::kTile + r * kSlabBytes, &p.tmQ, q_full, r * 64,
                        w.row0(t), w.head_of(t), 0);
        ++ic;
        for (int32_t j = 0; alive && j < w.n; ++j) {
          for (uint32_t t = 0; t < (w.shared ? 1u : 2u); ++t) {
            const uint32_t st = base + w.stage(t, j), s = st % KS, ph = ((st / KS) & 1u) ^ 1u;
            const int32_t hk = w.head_of(t) / p.G;
            if (!fmha_wait(k_empty(s), ph, abort_flag, p, B2G_SITE_EMPTY)) {
              alive = false;
              break;
            }
            mbar_arrive_expect_tx(k_full(s), PP::kTile);
            for (uint32_t r = 0; r < PP::kSlabs; ++r)
              tma_load_4d(sbase + PP::kKOff + s * PP::kTile + r * kSlabBytes, &p.tmK, k_full(s),
                          r * 64, w.k0 + j * 128, hk, 0);
            ++nk;
            if (!fmha_wait(v_empty(s), ph, abort_flag, p, B2G_SITE_EMPTY)) {
              alive = false;
              break;
            }
            mbar_arrive_expect_tx(v_full(s), PP::kTile);
            for (uint32_t r = 0; r < PP::kSlabs; ++r)
              tma_load_4d(sbase + PP::kVOff + s * PP::kTile + r * kSlabBytes, &p.tmV, v_full(s),
                          r * 64, w.k0 + j * 128, hk, 0);
            ++nv;
          }
        }
        base += w.stages();
      }
      // every load issued lands before the CTA can exit: the last Q and the K and V
      // loads of the last KS stages (older ones were consumed)
      uint32_t spins = 0;
      if (ic > 0)
        while (!mbar_try_wait(q_full, (ic - 1u) & 1u) && spins < (1u << 20)) ++spins;
      for (uint32_t i = nk > KS ? nk - KS : 0u; i < nk; ++i) {
        spins = 0;
        while (!mbar_try_wait(k_full(i % KS), (i / KS) & 1u) && spins < (1u << 20)) ++spins;
      }
      for (uint32_t i = nv > KS ? nv - KS : 0u; i < nv; ++i) {
        spins = 0;
        while (!mbar_try_wait(v_full(i % KS), (i / KS) & 1u) && spins < (1u << 20)) ++spins;
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------- MMA issue --
    // Per slot the order is S_0, PV_0, S_1, PV_1, ... (P lies in S's columns, and
    // one thread's MMAs run in issue order); the slots take turns, so one's softmax
    // runs during the other's products. The whole warp runs this and one lane issues
    // (see elect_one), what is there long before P is waited for before it, and
    // descriptors are sums: with a single-thread branch the issue took longer than the
    // products (12031 tokens x 32 heads: 1124 us then, 945-963 so).
    {
      constexpr uint32_t idesc_s = fmha_idesc_s<D, kBF16>();
      constexpr uint32_t idesc_pv = fmha_idesc_pv<D, kBF16>();
      uint32_t last_bar = 0, last_par = 0;  // the newest commit: all earlier MMAs precede it
      uint32_t base = 0, ic = 0;            // ring stages before the item, items
      uint32_t steps0 = 0, steps1 = 0;      // tiles of each slot (phases of s_full, p_full)
      uint32_t items0 = 0, items1 = 0;      // items of each slot (phases of o_done, o_free)
      bool alive = true;
      auto wait = [&](uint32_t bar, uint32_t parity, int site) {
        return __all_sync(0xffffffffu, fmha_wait(bar, parity & 1u, abort_flag, p, site)) != 0;
      };
      auto commit = [&](uint32_t bar) {
        if (elect_one()) tc_commit<1>(bar);
      };
      const uint64_t q_desc = sdesc_kmajor_sw128(sbase + PP::kQOff);
      const uint64_t k_desc = sdesc_kmajor_sw128(sbase + PP::kKOff);
      const uint64_t v_desc = sdesc_mnmajor_sw128(sbase + PP::kVOff, kSlabBytes, 1024u);
      // S of slot t with the K tile of stage s
      auto issue_s = [&](uint32_t t, uint32_t s) {
        const uint64_t qd = q_desc + t * (PP::kTile >> 4), kd = k_desc + s * (PP::kTile >> 4);
#pragma unroll
        for (uint32_t kk = 0; kk < D / 16; ++kk) {
          const uint32_t at = (kk >> 2) * (kSlabBytes >> 4) + 2u * (kk & 3u);
          if (elect_one())
            mma_f16<1>(tmem_base + PP::kS + t * PP::kTileCols, qd + at, kd + at, idesc_s,
                       kk > 0 ? 1u : 0u);
        }
        commit(s_full(t));
      };
      // (uniform: where the compiler cannot see that the warp stays converged, issuing is
      // as slow as from one thread)
      while (alive && uniform(static_cast<int32_t>(walk.next(p, own_list, counts, w))) != 0) {
        w.n = uniform(w.n);
        w.slots = uniform(w.slots);
        w.shared = uniform(static_cast<int32_t>(w.shared)) != 0;
        w.by_rows = uniform(static_cast<int32_t>(w.by_rows)) != 0;
        const uint32_t dual = w.shared ? 0u : 1u;
        if (!wait(q_full, ic, B2G_SITE_FULL)) break;
        for (uint32_t t = 0; t < w.slots; ++t) {
          const uint32_t st = base + dual * t, s = st % KS;
          if (!wait(k_full(s), st / KS, B2G_SITE_FULL)) {
            alive = false;
            break;
          }
          tc_fence_after();
          issue_s(t, s);
          if (dual || t + 1u == w.slots) commit(k_empty(s));
        }
        if (w.n == 1) commit(q_empty);
        // slot t's step j: PV of its tile, then S of its next one
        auto slot_step = [&](uint32_t t, int32_t j, uint32_t& steps, uint32_t& items) {
          const int32_t n = w.tiles(t);
          if (j >= n) return true;
          const uint32_t st = base + (static_cast<uint32_t>(j) << dual) + dual * t, s = st % KS;
          const uint32_t st1 = st + 1u + dual, s1 = st1 % KS;
          const bool more = j + 1 < n, last = dual || t + 1u == w.slots;
          if (!wait(v_full(s), st / KS, B2G_SITE_FULL)) return false;
          if (more && !wait(k_full(s1), st1 / KS, B2G_SITE_FULL)) return false;
          if (j == 0 && items > 0 && !wait(o_free(t), items - 1u, B2G_SITE_ACC_EMPTY)) return false;
          const uint64_t vd = v_desc + s * (PP::kTile >> 4);
          const uint32_t p_col = tmem_base + PP::kS + t * PP::kTileCols;
#pragma unroll
          for (uint32_t half = 0; half < 2; ++half) {
            if (!wait(p_full(t, half), steps, B2G_SITE_ACC_FULL)) return false;
            tc_fence_after();
#pragma unroll
            for (uint32_t k4 = 0; k4 < 4; ++k4) {
              const uint32_t kk = half * 4u + k4;
              if (elect_one())
                mma_f16_ts(tmem_base + PP::kO + t * PP::kTileCols, p_col + kk * 8u,
                           vd + kk * (2048u >> 4), idesc_pv, (j > 0 || kk > 0) ? 1u : 0u);
            }
          }
          ++steps;
          if (more) {
            issue_s(t, s1);
            last_bar = s_full(t);
            last_par = steps & 1u;
            if (last) commit(k_empty(s1));
          } else {
            commit(o_done(t));
            last_bar = o_done(t);
            last_par = items & 1u;
            ++items;
          }
          if (last) commit(v_empty(s));
          return true;
        };
        for (int32_t j = 0; alive && j < w.n; ++j) {
          alive = slot_step(0u, j, steps0, items0) &&
                  (w.slots == 1u || slot_step(1u, j, steps1, items1));
          if (j + 2 == w.n) commit(q_empty);  // the item's last S is issued
        }
        base += w.stages();
        ++ic;
      }
      // all MMAs issued by this thread finish before TMEM can be freed
      if (last_bar != 0u) {
        uint32_t spins = 0;
        while (!mbar_try_wait(last_bar, last_par) && spins < (1u << 22)) ++spins;
      }
    }
  } else {
    // --------------------------------------------- softmax and epilogue --
    // Warpgroup t has slot t; thread i of warp w has row 32 (w % 4) + i of its tile.
    const uint32_t t = (warp - 2u) >> 2;
    const uint32_t quarter = warp & 3u;
    const uint32_t row = quarter * 32u + lane;
    const uint32_t taddr = tmem_base + ((quarter * 32u) << 16);
    const uint32_t s_col = taddr + PP::kS + t * PP::kTileCols;
    const uint32_t o_col = taddr + PP::kO + t * PP::kTileCols;
    // Which of a warp's 32 rows of the last V tile hold values that are not finite:
    // [0], [1] as each slot found them in its own, [2] slot 0's for slot 1; by the
    // parity of the reader's items, so that a word is rewritten only after the reader
    // has taken part in another item.
    volatile uint32_t* odd_words = reinterpret_cast<volatile uint32_t*>(smem + PP::kOddOff);
    uint32_t step = 0, ti = 0;      // this slot's tiles and items
    uint32_t base = 0, pairs = 0;   // ring stages before the item, items of both slots
    bool alive = true;
    auto wait_all = [&](uint32_t bar, uint32_t parity, int site) {
      return __all_sync(0xffffffffu, fmha_wait(bar, parity & 1u, abort_flag, p, site)) != 0;
    };
    bool have = walk.next(p, own_list, counts, w);
    while (alive && have) {
      const uint32_t stage0 = base;
      base += w.stages();
      if (t >= w.slots) {
        have = walk.next(p, own_list, counts, w);
        continue;
      }
      const int32_t n = w.tiles(t);
      float m_run = -INFINITY, l_run = 0.0f;  // offset in log2 units, sum of weights
      for (int32_t j = 0; j < n; ++j, ++step) {
        const bool diagonal = j + 1 == n;
        uint32_t odd = 0;
        // a V tile that both slots read last is slot 0's to look through
        if (diagonal && (t == 0u || w.by_rows || !w.shared)) {
          const uint32_t st = stage0 + w.stage(t, j), s = st % KS;
          if (!wait_all(v_full(s), st / KS, B2G_SITE_FULL)) {
            alive = false;
            break;
          }
          const bool mine =
              clear_odd_values<D, kBF16>(sbase + PP::kVOff + s * PP::kTile + row * 128u, lane);
          odd = __ballot_sync(0xffffffffu, mine);
          if (odd != 0u) fence_proxy_async_smem();  // the PV product reads the zeros
        }
        if (!wait_all(s_full(t), step, B2G_SITE_ACC_FULL)) {
          alive = false;
          break;
        }
        tc_fence_after();
        uint32_t seen[4];
        if (diagonal) {
          if (lane == 0) {
            odd_words[(t * 2u + (ti & 1u)) * 4u + quarter] = odd;
            if (t == 0u) odd_words[(4u + (pairs & 1u)) * 4u + quarter] = odd;
          }
#pragma unroll
          for (uint32_t c = 0; c < 4; ++c)  // keys 32 c .. up to the row's own
            seen[c] = c < quarter ? ~0u : c > quarter ? 0u : 0xffffffffu >> (31u - lane);
        }
        tile_softmax<D, kBF16, 4>(s_col, o_col, 0u, p.scale_log2, diagonal, seen, j == 0, m_run,
                                  l_run, p_full(t, 0), p_full(t, 1), lane);
      }
      if (!alive) break;

      // epilogue: O into registers, the columns released to the next item's first PV,
      // then the scaled rows stored. What the next item is gets worked out while the
      // last PV runs.
      const int32_t head = w.head_of(t), m0 = w.m0, row0 = w.row0(t);
      const int32_t rows = w.rows - (row0 - m0);  // of this tile that there are
      const uint32_t two = w.slots - 1u;
      have = walk.next(p, own_list, counts, w);
      if (!wait_all(o_done(t), ti, B2G_SITE_ACC_FULL)) break;
      tc_fence_after();
      uint32_t o[D];
#pragma unroll
      for (uint32_t d = 0; d < static_cast<uint32_t>(D); d += 32u)
        tmem_ld_32x32b_x32(o_col + d, *reinterpret_cast<uint32_t(*)[32]>(&o[d]));
      tmem_wait_ld();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(o_free(t));
      const float inv_l = l_run == 0.0f ? 0.0f : 1.0f / l_run;
      // 32 columns at a time through shared memory, so that four lanes store 64
      // neighbouring bytes of a row (a row per lane costs a memory transaction per lane
      // and 16 bytes). 16-byte piece c of row r sits at piece c ^ (r / 2 % 4), which
      // spreads eight rows and eight pieces alike over the banks.
      const uint32_t stage = sbase + PP::kStoreOff + (warp - 2u) * 2048u;
      const uint32_t srow = lane >> 2, sc = lane & 3u;  // of the first of four stores
      T* dst = static_cast<T*>(p.O) + static_cast<int64_t>(row0 + static_cast<int32_t>(quarter * 32u + srow)) * p.o_t +
               head * p.o_h + 8u * sc;
#pragma unroll
      for (uint32_t d = 0; d < static_cast<uint32_t>(D); d += 32u) {
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) {
          uint32_t u[4];
#pragma unroll
          for (uint32_t i = 0; i < 4; ++i)
            u[i] = pack2<kBF16>(__uint_as_float(o[d + 8 * c + 2 * i]) * inv_l,
                                __uint_as_float(o[d + 8 * c + 2 * i + 1]) * inv_l);
          st_shared_v4(stage + lane * 64u + ((c ^ ((lane >> 1) & 3u)) << 4), u);
        }
        __syncwarp();
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
          const uint32_t r = srow + 8u * i;
          uint32_t u[4];
          ld_shared_v4(stage + r * 64u + ((sc ^ ((r >> 1) & 3u)) << 4), u);
          if (static_cast<int32_t>(quarter * 32u + r) < rows)
            *reinterpret_cast<uint4*>(dst + static_cast<int64_t>(8u * i) * p.o_t + d) =
                make_uint4(u[0], u[1], u[2], u[3]);
        }
        __syncwarp();
      }
      if (static_cast<int32_t>(row) < rows) {
        const int32_t token = row0 + static_cast<int32_t>(row);
        uint32_t any = 0;
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
          any |= odd_words[(t * 2u + (ti & 1u)) * 4u + q];
          if (t == 1u) any |= odd_words[(4u + (pairs & 1u)) * 4u + q];
        }
        if (any != 0u)  // (the warp's stores above are visible to it: __syncwarp)
          add_odd_values<D>(p, m0, head / p.G, token + 1,
                            static_cast<T*>(p.O) + static_cast<int64_t>(token) * p.o_t + head * p.o_h);
        if (p.lse != nullptr) {
          constexpr float kLn2 = 0.693147180559945309f;
          p.lse[static_cast<int64_t>(head) * p.tokens + token] =
              l_run == 0.0f ? -INFINITY : (m_run + __log2f(l_run)) * kLn2;
        }
      }
      ++ti;
      pairs += two;
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

template <int D, bool kBF16>
int launch_prefill(const PrefillParams& prm, int64_t items, int sms, cudaStream_t stream) {
  using PP = PrefillPlan<D>;
  auto kern = prefill_kernel<D, kBF16>;
  // at least half the SM's shared memory, so that two CTAs never share an SM (each
  // holds all 512 TMEM columns)
  const uint32_t dyn = std::max(PP::kDynBytes, 120u * 1024u);
  static std::atomic<bool> attr_set[64];  // per instantiation and device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return B2G_ENODEVICE;
  }
  if (!attr_set[dev].load()) {
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             static_cast<int>(dyn)) != cudaSuccess)
      return static_cast<int>(cudaGetLastError());
    attr_set[dev].store(true);
  }
  // after a planning kernel: set up while it runs, grid_dependency_wait orders the rest
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(std::min<int64_t>(items, sms)), 1, 1);
  cfg.blockDim = dim3(PP::kThreads, 1, 1);
  cfg.dynamicSmemBytes = dyn;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = prm.plan != nullptr ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, prm);
  if (e != cudaSuccess) cudaGetLastError();
  return e == cudaSuccess ? B2G_OK : static_cast<int>(e);
}

// Rows of a block, see packed_plan_kernel; most blocks that `tokens` in `prompts` can
// have: one for every `rows` tokens and a ragged one for each prompt.
int block_rows(int group) { return group % 2 == 0 ? 128 : 256; }
int64_t packed_blocks(int prompts, int64_t tokens, int rows) {
  return tokens / rows + std::min<int64_t>(prompts, tokens);
}
size_t packed_workspace(int64_t blocks, int sms) {
  return workspace_flag_bytes(sms) + 256 + static_cast<size_t>(blocks) * sizeof(int4);
}

}  // namespace

}  // namespace b2g

extern "C" size_t b2g_attention_prefill_workspace_bytes(int prompts, int64_t tokens, int heads_q) {
  (void)heads_q;
  const int sms = b2g::current_device_sms();
  if (sms <= 0 || prompts < 0 || tokens < 0) return 0;
  return b2g::packed_workspace(b2g::packed_blocks(prompts, tokens, 128), sms);
}

extern "C" int b2g_attention_prefill(const void* q, const void* k, const void* v, void* o,
                                     const int64_t* strides, const int32_t* cu_seqlens,
                                     int prompts, int64_t tokens, int heads_q, int heads_k,
                                     int head_dim, int dtype, float sm_scale, float* lse,
                                     void* workspace, size_t workspace_bytes, int* status,
                                     void* stream) {
  using namespace b2g;
  if (tokens < 0 || tokens > INT_MAX - 256 || prompts < 0) return B2G_ESHAPE;
  if (tokens == 0 || prompts == 0) return B2G_OK;
  const int rc = check_serving_attention(heads_q, heads_k, head_dim, dtype, sm_scale, strides, 8,
                                         {q, k, v, o});
  if (rc != B2G_OK) return rc;
  if (cu_seqlens == nullptr) return B2G_EINVAL;
  if (reinterpret_cast<uintptr_t>(lse) % alignof(float) != 0) return B2G_EALIGN;
  const int group = heads_q / heads_k;
  const int64_t blocks = packed_blocks(prompts, tokens, block_rows(group));
  if (blocks * heads_q > INT_MAX / 4) return B2G_ESHAPE;
  const int sms = current_device_sms();
  if (sms <= 0) return B2G_ENODEVICE;
  if (workspace == nullptr || workspace_bytes < packed_workspace(blocks, sms))
    return B2G_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % 256 != 0) return B2G_EALIGN;

  PrefillParams prm;
  std::memset(&prm, 0, sizeof(prm));
  // (token, head) strides as a batch of one: (batch, head, sequence, dim)
  auto encode = [&](CUtensorMap* map, const void* base, int heads, const int64_t* st) {
    const int64_t four[4] = {st[0] * tokens, st[1], st[0], 1};
    return encode_bshd_view(map, base, dtype, head_dim, static_cast<int>(tokens), heads, 1, four);
  };
  if (!encode(&prm.tmQ, q, heads_q, strides) || !encode(&prm.tmK, k, heads_k, strides + 2) ||
      !encode(&prm.tmV, v, heads_k, strides + 4))
    return B2G_ETENSORMAP;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  prm.cu = cu_seqlens;
  prm.prompts = prompts;
  prm.block = block_rows(group);
  if (blocks > static_cast<int64_t>(kOwnBlocks) || prompts > PrefillPlan<128>::kThreads) {
    uint8_t* ws = static_cast<uint8_t*>(workspace) + workspace_flag_bytes(sms);
    PackedPlanParams pl;
    pl.cu = cu_seqlens;
    pl.counts = reinterpret_cast<int2*>(ws);
    pl.plan = reinterpret_cast<int4*>(ws + 256);
    pl.status = status;
    pl.prompts = prompts;
    pl.tokens = static_cast<int32_t>(tokens);
    pl.capacity = static_cast<int32_t>(blocks);
    pl.block = prm.block;
    prm.plan = pl.plan;
    prm.counts = pl.counts;
    packed_plan_kernel<<<1, kPlanThreads, 0, s>>>(pl);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  prm.O = o;
  prm.o_t = strides[6];
  prm.o_h = strides[7];
  prm.V = v;
  prm.v_t = strides[4];
  prm.v_h = strides[5];
  prm.lse = lse;
  prm.status = status;
  prm.HQ = heads_q;
  prm.G = group;
  prm.tokens = static_cast<int32_t>(tokens);
  // every item number is below blocks * HQ
  auto inverse = [&](int64_t d) {
    const bool exact = d > 1 && blocks * heads_q * d < (static_cast<int64_t>(1) << 32);
    return exact ? static_cast<uint32_t>(((static_cast<int64_t>(1) << 32) + d - 1) / d) : 0u;
  };
  prm.hq_inv = inverse(heads_q);
  prm.pairs_inv = inverse((heads_q + 1) / 2);
  prm.scale_log2 = sm_scale * 1.4426950408889634f;
  prm.timeout_ns = wait_timeout_ns();
  const bool bf16 = dtype == B2G_DT_BF16;
  const int64_t items = blocks * heads_q;  // at most
  if (head_dim == 128)
    return bf16 ? launch_prefill<128, true>(prm, items, sms, s)
                : launch_prefill<128, false>(prm, items, sms, s);
  return bf16 ? launch_prefill<64, true>(prm, items, sms, s)
              : launch_prefill<64, false>(prm, items, sms, s);
}
