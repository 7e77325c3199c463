// What the attention kernels share: the softmax's exponentials, the bounded
// waits, the instruction descriptors of the two products and the tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>

#include <cmath>
#include <cstdint>

#include "b2g.h"
#include "capi_internal.h"
#include "ptx.cuh"

// Suspend-time hint of the slow path of the bounded waits (0: plain probes,
// which hand over between the roles a little sooner).
#ifndef B2G_FMHA_WAIT_HINT_NS
#define B2G_FMHA_WAIT_HINT_NS 0
#endif

namespace b2g {

// A 128-row operand tile lies in shared memory as slabs of 64 elements, each 128
// rows of 128 bytes.
constexpr uint32_t kSlabBytes = 128 * 128;

// exp2 on the FMA pipe for x <= 8 (a share of the softmax exponentials, so that
// they do not all queue on the MUFU unit): x = i + f with i = round(x) and
// f in [-0.5, 0.5]; 2^f from a cubic fitted here to minimise the relative error
// on that interval (iteratively reweighted least squares; max relative error
// 7.5e-5 in fp32 for x in [-125.5, 8], below half an fp16 ULP); 2^i added to
// the exponent field. Inputs below -126 (masked keys are -inf) are clamped
// there: with 2^f in [0.70, 1.42] the biased exponent 126 or 127 plus
// i >= -126 stays >= 0, so the result is a tiny non-negative number, never a
// carry into the sign bit (at the clamp the exponent field reaches 0, so the
// result is the subnormal 0.99986 * 2^-126 rather than 0.99993 * 2^-126).
// b2g_selftest_poly_exp2 evaluates it on caller data for the tests.
__device__ __forceinline__ float poly_exp2(float x) {
  constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to an integer
  x = fmaxf(x, -126.0f);
  const float t = x + kRound;
  const float fi = t - kRound;
  const float f = x - fi;
  float p = fmaf(0.05517134442925453f, f, 0.24261033535003662f);
  p = fmaf(p, f, 0.6932609677314758f);
  p = fmaf(p, f, 0.9999281167984009f);
  const int32_t i = static_cast<int32_t>(__float_as_uint(t) - __float_as_uint(kRound));
  return __uint_as_float(static_cast<uint32_t>(static_cast<int32_t>(__float_as_uint(p)) + (i << 23)));
}

// poly_exp2 on a pair, with the packed (two-lane) fp32 add and FMA: per pair
// two clamps, five packed operations and two integer adds.
__device__ __forceinline__ float2 poly_exp2x2(float2 x) {
  constexpr float kRound = 12582912.0f;
  x.x = fmaxf(x.x, -126.0f);
  x.y = fmaxf(x.y, -126.0f);
  const float2 t = __fadd2_rn(x, make_float2(kRound, kRound));
  const float2 fi = __fadd2_rn(t, make_float2(-kRound, -kRound));
  const float2 f = __ffma2_rn(fi, make_float2(-1.0f, -1.0f), x);
  float2 q = __ffma2_rn(make_float2(0.05517134442925453f, 0.05517134442925453f), f,
                        make_float2(0.24261033535003662f, 0.24261033535003662f));
  q = __ffma2_rn(q, f, make_float2(0.6932609677314758f, 0.6932609677314758f));
  q = __ffma2_rn(q, f, make_float2(0.9999281167984009f, 0.9999281167984009f));
  // t's bit pattern is that of 1.5 * 2^23 plus round(x), and the former ends in
  // nine zero bits: shifted left by 23 it leaves round(x) * 2^23, the exponent step
  return make_float2(__uint_as_float(__float_as_uint(q.x) + (__float_as_uint(t.x) << 23)),
                     __uint_as_float(__float_as_uint(q.y) + (__float_as_uint(t.y) << 23)));
}

// 2^x for x <= 8 to fp32 rounding, on the FMA pipe: as poly_exp2, but 2^f is the series of
// e^(f ln 2) up to f^7, whose next term is 5e-9 at f = 0.5.
__device__ __forceinline__ float series_exp2(float x) {
  constexpr float kRound = 12582912.0f;
  x = fmaxf(x, -126.0f);
  const float t = x + kRound;
  const float f = x - (t - kRound);
  float p = 1.525273380e-05f;  // ln(2)^7 / 7!
  p = fmaf(p, f, 1.540353039e-04f);
  p = fmaf(p, f, 1.333355815e-03f);
  p = fmaf(p, f, 9.618129108e-03f);
  p = fmaf(p, f, 5.550410866e-02f);
  p = fmaf(p, f, 2.402265070e-01f);
  p = fmaf(p, f, 6.931471806e-01f);
  p = fmaf(p, f, 1.0f);
  return __uint_as_float(__float_as_uint(p) + (__float_as_uint(t) << 23));
}

// After tcgen05.wait::ld: ties these registers to this point, so that no use
// of a value loaded asynchronously is scheduled before the wait (no code).
__device__ __forceinline__ void regs_ready(uint32_t (&r)[32]) {
#pragma unroll
  for (int i = 0; i < 32; ++i) asm volatile("" : "+r"(r[i]));
}

__device__ __forceinline__ float fmax3(float a, float b, float c) {
  float m;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}

template <int D, bool kBF16>
__host__ __device__ constexpr uint32_t fmha_idesc_s() {
  // D fp32 | A, B fmt | both K-major | N = 128 keys | M = 128 rows
  constexpr uint32_t f = kBF16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
}

template <int D, bool kBF16>
__host__ __device__ constexpr uint32_t fmha_idesc_pv() {
  // D fp32 | A, B fmt | A K-major (TMEM), B MN-major (V, d contiguous) | N = D | M = 128
  constexpr uint32_t f = kBF16 ? 1u : 0u;
  return (1u << 4) | (f << 7) | (f << 10) | (1u << 16) | ((static_cast<uint32_t>(D) >> 3) << 17) |
         ((128u >> 4) << 24);
}

template <typename P>
__device__ __forceinline__ void fmha_report(const P& p, int code) {
  if (p.status != nullptr) atomicCAS(p.status, 0, code);
}

// Bounded mbarrier wait: sleeping probes, then the deadline and the CTA's
// abort flag between them. P: a kernel's parameters, with status and timeout_ns.
template <typename P>
__device__ __noinline__ bool fmha_wait_slow(uint32_t bar, uint32_t parity,
                                            volatile uint32_t* abort_flag, const P& p,
                                            int site) {
  const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
  while (true) {
#if B2G_FMHA_WAIT_HINT_NS > 0
    if (mbar_try_wait_sleep(bar, parity, B2G_FMHA_WAIT_HINT_NS)) return true;
#else
    if (mbar_try_wait(bar, parity)) return true;
#endif
    if (*abort_flag != 0u) return false;
    if (globaltimer_ns() - t0 > p.timeout_ns) {
      fmha_report(p, B2G_STATUS_TIMEOUT | site);
      *abort_flag = 1u;
      return false;
    }
  }
}

template <typename P>
__device__ __forceinline__ bool fmha_wait(uint32_t bar, uint32_t parity,
                                          volatile uint32_t* abort_flag, const P& p,
                                          int site) {
  if (mbar_try_wait(bar, parity)) return true;
  return fmha_wait_slow(bar, parity, abort_flag, p, site);
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool kBF16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (kBF16) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
}

// Sets what is not finite among the D values of one V row in shared memory to
// zero; returns whether there was any. The row's slabs of 128 bytes (64 elements) lie
// kSlabBytes apart; swizzling only permutes 16-byte chunks within a slab, so the
// order does not matter, and starting at a chunk of its own keeps a warp's lanes
// off one another's banks.
template <int D, bool kBF16>
__device__ __forceinline__ bool clear_odd_values(uint32_t row_addr, uint32_t lane) {
  constexpr uint32_t kExp = kBF16 ? 0x7F807F80u : 0x7C007C00u;  // all ones: infinity or NaN
  constexpr uint32_t kUp = kBF16 ? 0x00800080u : 0x04000400u;   // carries all ones into bit 15
  uint32_t odd = 0;
#pragma unroll
  for (uint32_t i = 0; i < static_cast<uint32_t>(D) / 8; ++i) {
    const uint32_t a = row_addr + (i >> 3) * kSlabBytes + (((i + lane) & 7u) << 4);
    uint32_t x[4];
    ld_shared_v4(a, x);
#pragma unroll
    for (int w = 0; w < 4; ++w) odd |= ((x[w] & kExp) + kUp) & 0x80008000u;
  }
  if (odd == 0u) return false;
  for (uint32_t i = 0; i < static_cast<uint32_t>(D) / 8; ++i) {
    const uint32_t a = row_addr + (i >> 3) * kSlabBytes + ((i & 7u) << 4);
    uint32_t x[4];
    ld_shared_v4(a, x);
    for (int w = 0; w < 4; ++w) {
      const uint32_t hit = ((x[w] & kExp) + kUp) & 0x80008000u;
      if (hit & 0x8000u) x[w] &= 0xFFFF0000u;
      if (hit & 0x80000000u) x[w] &= 0x0000FFFFu;
    }
    st_shared_v4(a, x);
  }
  return true;
}

// One tile's softmax for a thread's row: NCH chunks of 32 score columns from
// chunk c0 on, weights for those and zeros for the others into P. Keeps the
// running maximum (log2 units) and sum.
template <int D, bool kBF16, int NCH>
__device__ __forceinline__ void tile_softmax(uint32_t s_col, uint32_t o_col, uint32_t c0, float sl2,
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
  // Right to fp32 rounding, since what it scales stays in the sum (poly_exp2's 7e-5 came out
  // in the lse of a row with many keys just below the one that moved it). The series costs
  // the tiles in which no row moves nothing; one hardware exponential is evaluated for all of
  // them instead (decode of 64 requests of up to 8192 keys, interleaved: 319.5 us so, 325).
  float alpha = 1.0f;
  if (move) alpha = series_exp2(m_run - m_new);
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

// 4-D view (d, sequence, head, batch) of one operand, 64 x 128 boxes.
inline bool encode_bshd_view(CUtensorMap* map, const void* base, int dtype, int D, int S, int H, int B,
                      const int64_t* st /* batch, head, seq, dim (elements) */) {
  auto enc = tma_encoder();
  if (enc == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(S),
                              static_cast<cuuint64_t>(H), static_cast<cuuint64_t>(B)};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(st[2]) * 2u,
                                 static_cast<cuuint64_t>(st[1]) * 2u,
                                 static_cast<cuuint64_t>(st[0]) * 2u};
  const cuuint32_t box[4] = {64, 128, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType t =
      dtype == B2G_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return enc(map, t, 4, const_cast<void*>(base), dims, strides, box, estr,
             CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace b2g
