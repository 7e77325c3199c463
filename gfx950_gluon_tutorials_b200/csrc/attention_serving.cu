// Attention forward of a serving step: causal over packed prompts, and drafted
// tokens over a paged cache. One warp per (token, query head): the head's row of Q
// in registers, one key at a time with a running maximum and sum.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <initializer_list>
#include <cstdint>

#include "b2g.h"
#include "capi_internal.h"

namespace b2g {

struct RowsParams {
  const void *q, *k, *v;
  void* o;
  int64_t q_t, q_h, o_t, o_h;              // token, head strides
  int64_t k_p, k_t, k_h, v_p, v_t, v_h;    // page, token, head strides
  const int32_t* cu;
  const int32_t* seq_lens;   // paged form
  const int32_t* tables;     // paged form, else null
  int64_t table_stride, num_pages;
  const int64_t* mask;
  float* lse;
  int* status;
  int32_t mask_words, max_pages, page_size, requests, tokens, HQ, HK;
  float scale;
};

template <int D, typename T>
__global__ void rows_kernel(const RowsParams p) {
  constexpr int E = D / 32;
  const int lane = threadIdx.x & 31;
  const int64_t row = (blockIdx.x * static_cast<int64_t>(blockDim.x) + threadIdx.x) >> 5;
  if (row >= static_cast<int64_t>(p.tokens) * p.HQ) return;
  const int tok = static_cast<int>(row / p.HQ), h = static_cast<int>(row % p.HQ);
  const int hk = h / (p.HQ / p.HK);
  int lo = 0, hi = p.requests;  // the request with cu[r] <= tok < cu[r + 1]
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (p.cu[mid + 1] > tok) hi = mid;
    else lo = mid + 1;
  }
  if (row == 0 && lane == 0) {  // offsets are 0 <= c[0] <= c[1] <= ... <= tokens
    int last = 0;
    for (int r = 0; r <= p.requests; ++r) {
      if (p.cu[r] < last || p.cu[r] > p.tokens)
        if (p.status) atomicCAS(p.status, 0, B2G_STATUS_TOKENS);
      last = p.cu[r];
      if (p.tables && r < p.requests && p.seq_lens[r] > static_cast<int64_t>(p.max_pages) * p.page_size)
        if (p.status) atomicCAS(p.status, 0, B2G_STATUS_PAGE_TABLE);
    }
  }
  if (lo >= p.requests || p.cu[lo] > tok) return;
  const int first = max(p.cu[lo], 0), i = tok - first;
  const int n = min(p.cu[lo + 1], p.tokens) - first;
  const int len = p.tables ? min(max(p.seq_lens[lo], 0), p.max_pages * p.page_size) : n;
  const int ctx = len - n;
  float qr[E], acc[E];
  const T* qp = static_cast<const T*>(p.q) + tok * p.q_t + h * p.q_h;
  for (int e = 0; e < E; ++e) {
    qr[e] = static_cast<float>(qp[lane * E + e]) * p.scale;
    acc[e] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int j = 0; j < len; ++j) {
    const int rank = j - ctx;
    if (rank >= 0) {
      if (p.mask == nullptr) {
        if (rank > i) break;
      } else {
        if (rank >= 64 * p.mask_words) break;
        if (!((p.mask[static_cast<int64_t>(tok) * p.mask_words + (rank >> 6)] >> (rank & 63)) & 1)) continue;
      }
    }
    const T *kp = static_cast<const T*>(p.k) + hk * p.k_h, *vp = static_cast<const T*>(p.v) + hk * p.v_h;
    if (p.tables) {
      const int page = p.tables[lo * p.table_stride + j / p.page_size];
      if (page < 0 || page >= p.num_pages) {
        if (p.status) atomicCAS(p.status, 0, B2G_STATUS_PAGE_TABLE);
        continue;
      }
      kp += page * p.k_p + (j % p.page_size) * p.k_t;
      vp += page * p.v_p + (j % p.page_size) * p.v_t;
    } else {
      kp += (first + j) * p.k_t;
      vp += (first + j) * p.v_t;
    }
    float s = 0.0f;
    for (int e = 0; e < E; ++e) s += qr[e] * static_cast<float>(kp[lane * E + e]);
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float mn = fmaxf(m, s);
    const float a = mn == -INFINITY ? 1.0f : expf(m - mn);
    const float w = mn == -INFINITY ? 0.0f : expf(s - mn);
    l = l * a + w;
    for (int e = 0; e < E; ++e) acc[e] = acc[e] * a + w * static_cast<float>(vp[lane * E + e]);
    m = mn;
  }
  T* op = static_cast<T*>(p.o) + tok * p.o_t + h * p.o_h;
  for (int e = 0; e < E; ++e) op[lane * E + e] = static_cast<T>(l == 0.0f ? 0.0f : acc[e] / l);
  if (p.lse != nullptr && lane == 0)
    p.lse[static_cast<int64_t>(h) * p.tokens + tok] = l == 0.0f ? -INFINITY : m + logf(l);
}

namespace {
int launch_rows(const RowsParams& p, int head_dim, int dtype, cudaStream_t s) {
  const int64_t rows = static_cast<int64_t>(p.tokens) * p.HQ;
  const unsigned grid = static_cast<unsigned>((rows + 7) / 8);
  if (head_dim == 128) {
    if (dtype == B2G_DT_BF16) rows_kernel<128, __nv_bfloat16><<<grid, 256, 0, s>>>(p);
    else rows_kernel<128, __half><<<grid, 256, 0, s>>>(p);
  } else {
    if (dtype == B2G_DT_BF16) rows_kernel<64, __nv_bfloat16><<<grid, 256, 0, s>>>(p);
    else rows_kernel<64, __half><<<grid, 256, 0, s>>>(p);
  }
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? B2G_OK : static_cast<int>(e);
}

}  // namespace

}  // namespace b2g

extern "C" size_t b2g_attention_tree_workspace_bytes(int, int64_t, int, int, int) { return 0; }

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
  if (num_pages < 1 || num_pages > INT_MAX || max_pages < 0) return B2G_ESHAPE;
  if (page_size != 8 && page_size != 16 && page_size != 32 && page_size != 64 &&
      (page_size < 1 || page_size % 128 != 0))
    return B2G_ESHAPE;
  if (requests > 1 && table_stride < max_pages) return B2G_ESTRIDE;
  if (reinterpret_cast<uintptr_t>(tree_mask) % 8 != 0) return B2G_EALIGN;
  if (current_device_sms() <= 0) return B2G_ENODEVICE;
  RowsParams p = {};
  p.q = q; p.k = k_cache; p.v = v_cache; p.o = o;
  p.q_t = strides[0]; p.q_h = strides[1];
  p.k_p = strides[2]; p.k_t = strides[3]; p.k_h = strides[4];
  p.v_p = strides[5]; p.v_t = strides[6]; p.v_h = strides[7];
  p.o_t = strides[8]; p.o_h = strides[9];
  p.cu = cu_seqlens; p.seq_lens = seq_lens; p.tables = block_tables; p.table_stride = table_stride;
  p.max_pages = max_pages; p.num_pages = num_pages; p.page_size = page_size;
  p.mask = tree_mask; p.mask_words = mask_words; p.lse = lse; p.status = status;
  p.requests = requests; p.tokens = static_cast<int32_t>(tokens); p.HQ = heads_q; p.HK = heads_k;
  p.scale = sm_scale;
  return launch_rows(p, head_dim, dtype, static_cast<cudaStream_t>(stream));
}
