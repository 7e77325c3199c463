// A paged key/value cache's bookkeeping and stores.
//
// map_step_kernel: from the lengths of a step's requests (tokens already cached
// c_r, new tokens n_r, pages held h_r) to where its new tokens go:
//   fresh_r  = max(0, ceil((c_r + n_r) / P) - h_r)         pages to take
//   first_r  = sum of fresh_s over s < r                    (exclusive scan)
//   page k of the step = free[num_free - 1 - k]             (the list is a stack)
//   token i of request r sits at position p = c_r + i, in page p / P of r, at
//   slot page * P + p % P.
// What bounds it is the launch and one pass of dependent loads; every CTA scans all
// requests itself (3 ints each, from L2) and then writes its own share of the
// tokens and table entries, so there is one launch and no hand-over between CTAs.
//
// kv_write_kernel: cache[slot] = k, v. Every byte is read once and written once;
// bound by DRAM bandwidth, so 16-byte accesses with several in flight per thread.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>

#include "b2g.h"
#include "capi_internal.h"

namespace b2g {

struct MapStepParams {
  const int32_t* cached;
  const int32_t* fresh_tokens;
  const int32_t* held;
  int32_t* tables;
  int64_t table_stride;
  const int32_t* free_pages;
  int64_t free_capacity;
  const int32_t* num_free;
  int64_t* slots;
  int32_t* positions;
  int32_t* cu;
  int32_t* seq_lens;
  int32_t* held_out;
  int32_t* num_free_out;
  int* status;
  int32_t requests, max_pages, page_size, num_tokens;
};

constexpr int kMapThreads = 512;
constexpr int kMapMaxRequests = 8192;  // two int32 prefix sums per request in shared memory
constexpr int kMapStaticBytes = 2 * (kMapThreads / 32) * 8;  // warp_tok and warp_pag

__device__ __forceinline__ void report(int* status, int code) {
  if (status != nullptr) atomicCAS(status, 0, code);
}

// First index in the non-decreasing ends[0..n) whose value exceeds x (n if none).
__device__ __forceinline__ int first_above(const int32_t* ends, int n, int32_t x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (ends[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kMapThreads) map_step_kernel(const MapStepParams p) {
  extern __shared__ int32_t ends[];  // [requests] token ends, then [requests] page ends
  int32_t* page_ends = ends + p.requests;
  __shared__ int64_t warp_tok[kMapThreads / 32], warp_pag[kMapThreads / 32];
  static_assert(sizeof(warp_tok) + sizeof(warp_pag) == kMapStaticBytes, "static shared memory");
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t limit = p.num_tokens;
  int64_t tok_base = 0, pag_base = 0;  // sums over the chunks before this one (same in all threads)
  for (int r0 = 0; r0 < p.requests; r0 += kMapThreads) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    int64_t tok = 0, pag = 0, length = 0, held = 0;
    if (r < p.requests) {
      const int64_t c = max(p.cached[r], 0);
      tok = max(p.fresh_tokens[r], 0);
      held = min(max(p.held[r], 0), p.max_pages);
      length = c + tok;
      int64_t need = (length + p.page_size - 1) / p.page_size;
      if (need > p.max_pages) {
        need = p.max_pages;
        if (blockIdx.x == 0) report(p.status, B2G_STATUS_PAGE_TABLE);
      }
      pag = max(need - held, static_cast<int64_t>(0));
    }
    // inclusive scans over the chunk: shuffles within a warp, then over the warps' sums
    int64_t t = tok, g = pag;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t ut = __shfl_up_sync(0xffffffffu, t, d), ug = __shfl_up_sync(0xffffffffu, g, d);
      if (lane >= d) {
        t += ut;
        g += ug;
      }
    }
    __syncthreads();  // the previous chunk's sums have been read
    if (lane == 31) {
      warp_tok[warp] = t;
      warp_pag[warp] = g;
    }
    __syncthreads();
    int64_t chunk_tok = 0, chunk_pag = 0;
#pragma unroll
    for (int w = 0; w < kMapThreads / 32; ++w) {
      if (w < warp) {
        t += warp_tok[w];
        g += warp_pag[w];
      }
      chunk_tok += warp_tok[w];
      chunk_pag += warp_pag[w];
    }
    if (r < p.requests) {
      const int32_t end = static_cast<int32_t>(min(tok_base + t, limit));
      ends[r] = end;
      page_ends[r] = static_cast<int32_t>(min(pag_base + g, static_cast<int64_t>(INT_MAX)));
      if (blockIdx.x == 0) {
        p.cu[r + 1] = end;
        p.seq_lens[r] = static_cast<int32_t>(min(length, static_cast<int64_t>(INT_MAX)));
        p.held_out[r] = static_cast<int32_t>(held + pag);
      }
    }
    tok_base += chunk_tok;
    pag_base += chunk_pag;
  }
  __syncthreads();
  const int32_t have = static_cast<int32_t>(
      min(static_cast<int64_t>(max(*p.num_free, 0)), p.free_capacity));
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    p.cu[0] = 0;
    p.num_free_out[0] =
        static_cast<int32_t>(max(have - pag_base, static_cast<int64_t>(INT_MIN)));
    if (tok_base > limit) report(p.status, B2G_STATUS_TOKENS);
  }
  const int32_t pages = static_cast<int32_t>(min(pag_base, static_cast<int64_t>(INT_MAX)));
  const int64_t step = static_cast<int64_t>(gridDim.x) * kMapThreads;
  const int64_t me = static_cast<int64_t>(blockIdx.x) * kMapThreads + threadIdx.x;
  for (int64_t k = me; k < pages; k += step) {
    const int r = first_above(page_ends, p.requests, static_cast<int32_t>(k));
    const int32_t first = r > 0 ? page_ends[r - 1] : 0;
    const int32_t held = min(max(p.held[r], 0), p.max_pages);
    const int64_t at = have - 1 - k;
    p.tables[r * p.table_stride + held + (k - first)] = at >= 0 ? p.free_pages[at] : -1;
  }
  for (int64_t i = me; i < limit; i += step) {
    const int r = first_above(ends, p.requests, static_cast<int32_t>(i));
    int64_t slot = -1;
    int32_t pos = 0;
    if (r < p.requests) {
      const int32_t held = min(max(p.held[r], 0), p.max_pages);
      const int64_t pl = max(p.cached[r], 0) + i - (r > 0 ? ends[r - 1] : 0);
      const int64_t pg = pl / p.page_size;
      pos = static_cast<int32_t>(min(pl, static_cast<int64_t>(INT_MAX)));
      int32_t page = -1;
      if (pg < held) {
        page = p.tables[r * p.table_stride + pg];
      } else if (pg < p.max_pages) {
        const int64_t at = have - 1 - ((r > 0 ? page_ends[r - 1] : 0) + pg - held);
        if (at >= 0) page = p.free_pages[at];
      }
      if (page >= 0) slot = static_cast<int64_t>(page) * p.page_size + pl % p.page_size;
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
  }
}

struct KvWriteParams {
  const void* src[2];  // k, v
  void* dst[2];        // caches
  int64_t src_token[2], src_head[2];                // in vectors
  int64_t dst_page[2], dst_slot[2], dst_head[2];    // in vectors
  const int64_t* slots;
  int* status;
  int64_t num_slots;
  uint32_t rows;                   // tokens * heads
  uint32_t heads, row, page_size;  // row: vectors of a (token, head)
};

// A warp to a row of K and the same one of V, kUnroll vectors of each in flight per
// lane: the loads do not wait for the slot, only the stores do. One division per row
// and 32-bit ones (with an index division per vector the 134 MB of 16384 tokens x 8
// heads x 128 took 32.6 us on the GPU, so 22.6: 5.95 TB/s; per call 24.6).
template <typename Vec>
__global__ void __launch_bounds__(256) kv_write_kernel(const KvWriteParams p) {
  constexpr uint32_t kUnroll = 4;
  const uint32_t lane = threadIdx.x & 31u;
  const uint32_t warps = gridDim.x * (blockDim.x / 32u);
  for (uint32_t r = blockIdx.x * (blockDim.x / 32u) + threadIdx.x / 32u; r < p.rows; r += warps) {
    const uint32_t tok = r / p.heads, h = r - tok * p.heads;
    const int64_t slot = p.slots[tok];
    const Vec* src[2];
#pragma unroll
    for (int s = 0; s < 2; ++s)
      src[s] = static_cast<const Vec*>(p.src[s]) + tok * p.src_token[s] + h * p.src_head[s];
    const bool there = slot >= 0 && slot < p.num_slots;
    for (uint32_t c0 = lane; c0 < p.row; c0 += 32u * kUnroll) {
      Vec val[2][kUnroll];
#pragma unroll
      for (uint32_t u = 0; u < kUnroll; ++u)
        if (c0 + 32u * u < p.row)
#pragma unroll
          for (int s = 0; s < 2; ++s) val[s][u] = src[s][c0 + 32u * u];
      if (!there) {
        if (slot >= p.num_slots) report(p.status, B2G_STATUS_SLOT);
        break;
      }
      int64_t page, in;
      if (((slot | p.num_slots) >> 31) == 0) {
        page = static_cast<uint32_t>(slot) / p.page_size;
        in = static_cast<uint32_t>(slot) - static_cast<uint32_t>(page) * p.page_size;
      } else {
        page = slot / p.page_size;
        in = slot - page * p.page_size;
      }
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        Vec* dst = static_cast<Vec*>(p.dst[s]) + page * p.dst_page[s] + in * p.dst_slot[s] + h * p.dst_head[s];
#pragma unroll
        for (uint32_t u = 0; u < kUnroll; ++u)
          if (c0 + 32u * u < p.row) dst[c0 + 32u * u] = val[s][u];
      }
    }
  }
}

namespace {

template <typename Vec>
int launch_kv_write(const KvWriteParams& p, int sms, cudaStream_t stream) {
  const unsigned blocks = (p.rows + 7) / 8;
  kv_write_kernel<Vec><<<std::min(blocks, static_cast<unsigned>(sms) * 8u), 256, 0, stream>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B2G_OK : static_cast<int>(e);
}

}  // namespace

}  // namespace b2g

extern "C" int b2g_kv_map_step(const int32_t* cached_lens, const int32_t* new_lens,
                               const int32_t* page_counts, int32_t* block_tables,
                               int64_t table_stride, int requests, int max_pages,
                               const int32_t* free_pages, int64_t free_capacity,
                               const int32_t* num_free, int page_size, int64_t num_tokens,
                               int64_t* slots, int32_t* positions, int32_t* cu_seqlens,
                               int32_t* seq_lens, int32_t* page_counts_out,
                               int32_t* num_free_out, int* status, void* stream) {
  using namespace b2g;
  if (requests < 0 || max_pages < 0 || page_size < 1 || num_tokens < 0 || free_capacity < 0)
    return B2G_ESHAPE;
  if (num_tokens > INT_MAX - 1 || free_capacity > INT_MAX) return B2G_ESHAPE;
  if (requests > kMapMaxRequests) return B2G_ECAPACITY;
  if (cu_seqlens == nullptr || num_free == nullptr || num_free_out == nullptr) return B2G_EINVAL;
  if (requests > 0 && (cached_lens == nullptr || new_lens == nullptr || page_counts == nullptr ||
                       seq_lens == nullptr || page_counts_out == nullptr))
    return B2G_EINVAL;
  if (requests > 0 && max_pages > 0 && block_tables == nullptr) return B2G_EINVAL;
  if (free_capacity > 0 && free_pages == nullptr) return B2G_EINVAL;
  if (num_tokens > 0 && (slots == nullptr || positions == nullptr)) return B2G_EINVAL;
  if (requests > 1 && table_stride < max_pages) return B2G_ESTRIDE;
  if (reinterpret_cast<uintptr_t>(slots) % 8 != 0) return B2G_EALIGN;
  const int sms = current_device_sms();
  if (sms <= 0) return B2G_ENODEVICE;
  MapStepParams p;
  p.cached = cached_lens;
  p.fresh_tokens = new_lens;
  p.held = page_counts;
  p.tables = block_tables;
  p.table_stride = table_stride;
  p.free_pages = free_pages;
  p.free_capacity = free_capacity;
  p.num_free = num_free;
  p.slots = slots;
  p.positions = positions;
  p.cu = cu_seqlens;
  p.seq_lens = seq_lens;
  p.held_out = page_counts_out;
  p.num_free_out = num_free_out;
  p.status = status;
  p.requests = requests;
  p.max_pages = max_pages;
  p.page_size = page_size;
  p.num_tokens = static_cast<int32_t>(num_tokens);
  const int smem = std::max(requests, 1) * 2 * static_cast<int>(sizeof(int32_t));
  // what a launch may take unasked (48 KB) holds the kernel's static arrays too
  if (smem + kMapStaticBytes > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(
        map_step_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
        kMapMaxRequests * 2 * static_cast<int>(sizeof(int32_t)));
    if (e != cudaSuccess) {
      cudaGetLastError();
      return static_cast<int>(e);
    }
  }
  const int64_t want = (std::max<int64_t>(num_tokens, requests) + kMapThreads - 1) / kMapThreads;
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(want, 1), sms));
  map_step_kernel<<<grid, kMapThreads, smem, static_cast<cudaStream_t>(stream)>>>(p);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B2G_OK : static_cast<int>(e);
}

extern "C" int b2g_kv_write(const void* k, const void* v, void* k_cache, void* v_cache,
                            const int64_t* strides, const int64_t* slots, int64_t tokens,
                            int heads, int head_dim, int64_t num_pages, int page_size, int dtype,
                            int* status, void* stream) {
  using namespace b2g;
  if (strides == nullptr) return B2G_EINVAL;
  if (dtype != B2G_DT_F16 && dtype != B2G_DT_BF16) return B2G_EINVAL;
  if (tokens < 0 || heads < 1 || head_dim < 1 || num_pages < 0 || page_size < 1) return B2G_ESHAPE;
  if (tokens > INT_MAX / heads || num_pages > INT64_MAX / page_size) return B2G_ESHAPE;
  if (tokens == 0) return B2G_OK;
  if (k == nullptr || v == nullptr || slots == nullptr) return B2G_EINVAL;
  if (num_pages > 0 && (k_cache == nullptr || v_cache == nullptr)) return B2G_EINVAL;
  if (reinterpret_cast<uintptr_t>(slots) % 8 != 0) return B2G_EALIGN;
  const int64_t* st = strides;  // k, v: (token, head); k_cache, v_cache: (page, slot, head)
  const int sms = current_device_sms();
  if (sms <= 0) return B2G_ENODEVICE;
  // heads that lie side by side in all four tensors make one longer row
  int64_t row = head_dim;
  if (st[1] == head_dim && st[3] == head_dim && st[6] == head_dim && st[9] == head_dim) {
    row = static_cast<int64_t>(heads) * head_dim;
    if (row > INT_MAX) return B2G_ESHAPE;
    heads = 1;
  }
  // the widest vector that every address of the call is a multiple of
  uint64_t all = static_cast<uint64_t>(row) * 2;
  for (int i = 0; i < 10; ++i)
    if (heads > 1 || (i != 1 && i != 3 && i != 6 && i != 9))
      all |= static_cast<uint64_t>(st[i]) * 2;
  for (const void* ptr : {k, v, static_cast<const void*>(k_cache), static_cast<const void*>(v_cache)})
    all |= reinterpret_cast<uintptr_t>(ptr);
  if (all & 1) return B2G_EALIGN;
  const int bytes = all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
  const int64_t per = bytes / 2;
  KvWriteParams p;
  p.src[0] = k;
  p.src[1] = v;
  p.dst[0] = k_cache;
  p.dst[1] = v_cache;
  for (int s = 0; s < 2; ++s) {
    p.src_token[s] = st[2 * s] / per;
    p.src_head[s] = heads > 1 ? st[2 * s + 1] / per : 0;
    p.dst_page[s] = st[4 + 3 * s] / per;
    p.dst_slot[s] = st[5 + 3 * s] / per;
    p.dst_head[s] = heads > 1 ? st[6 + 3 * s] / per : 0;
  }
  p.slots = slots;
  p.status = status;
  p.num_slots = num_pages * page_size;
  p.heads = static_cast<uint32_t>(heads);
  p.row = static_cast<uint32_t>(row / per);
  p.rows = static_cast<uint32_t>(tokens * heads);
  p.page_size = static_cast<uint32_t>(page_size);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (bytes) {
    case 16: return launch_kv_write<uint4>(p, sms, s);
    case 8: return launch_kv_write<uint2>(p, sms, s);
    case 4: return launch_kv_write<uint32_t>(p, sms, s);
    default: return launch_kv_write<uint16_t>(p, sms, s);
  }
}
