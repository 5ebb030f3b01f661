// Parts of the bf16 attention kernels (attention.hip, kv_attention.h): operand
// types, direct-to-LDS loads, the LDS layout of key and value tiles, and the
// arithmetic around the softmax.
#pragma once

#include "common.h"

using namespace bwpp;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef short v8s_t __attribute__((ext_vector_type(8)));
typedef unsigned int u32x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s_t lds_v4s_t;

namespace {

typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

// Eight fp32 probabilities (registers r0 .. r0 + 7 of an accumulator) as two
// bf16 terms: the upper 16 bits, and the rounded rest.  The rest is kept
// above zero wherever p is (by 2^-23 p), so that p * inf stays inf.
__device__ __forceinline__ void split_bf16x8(const f32x16_t *s, int r0, bf16x8_t &hi, bf16x8_t &lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float p0 = (*s)[r0 + 2 * i], p1 = (*s)[r0 + 2 * i + 1];
    const uint32_t u0 = __float_as_uint(p0) & 0xffff0000u, u1 = __float_as_uint(p1) & 0xffff0000u;
    h[i] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
    l[i] = pack_bf16x2(__builtin_fmaf(p0, 1.00000012f, -__uint_as_float(u0)),
                       __builtin_fmaf(p1, 1.00000012f, -__uint_as_float(u1)));
  }
  hi = __builtin_bit_cast(bf16x8_t, make_uint4(h[0], h[1], h[2], h[3]));
  lo = __builtin_bit_cast(bf16x8_t, make_uint4(l[0], l[1], l[2], l[3]));
}

// m ln 2 + ln l, rounded once: l = 2^k f with f in [0.71, 1.42), so that logf's
// error is one of a small number, ln 2 in two terms, and every rounding on the
// way carried to the end (B1 H16 S1664 d64, error against 64 bits: 5.4e-8 with
// plain arithmetic, 4.3e-8 in the generic path).
__device__ __forceinline__ float lse_of(float m, float l) {
#pragma clang fp contract(off)
  constexpr float kHi = 0.693147182f, kLo = -1.90465421e-9f;
  if (!(l < INFINITY)) return l;
  const uint32_t u = __float_as_uint(l);
  const int k = (int)(u - 0x3f3504f3u) >> 23;
  const float e = (float)k, lf = logf(__uint_as_float(u - ((uint32_t)k << 23)));
  const float a = m * kHi, b = e * kHi, t = a + b, td = t - a, r = t + lf, rd = r - t;
  const float lo = ((a - (t - td)) + (b - td)) + ((t - (r - rd)) + (lf - rd));  // of the two sums
  return r + (lo + (__builtin_fmaf(m, kHi, -a) + __builtin_fmaf(e, kHi, -b) + (m + e) * kLo));
}

// Running maximum of |v| as bit patterns, two bf16 lanes at a time (0x7f80
// and above: infinity or NaN).
__device__ __forceinline__ u16x2_t max_abs_bf16(u16x2_t m, v8s_t v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u16x2_t w = {(unsigned short)(v[2 * i] & 0x7fff), (unsigned short)(v[2 * i + 1] & 0x7fff)};
    m = __builtin_elementwise_max(m, w);
  }
  return m;
}

// The running maximum is raised when a tile exceeds it by this much (log2).
constexpr float kLazy = 8.0f;

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

// 16 bytes per lane global -> LDS (M0 = destination of lane 0, lane l at
// +16 l), from a wave-uniform 64-bit base in SGPRs plus a 32-bit per-lane
// byte offset; inline asm keeps the compiler from adding vmcnt(0) before every
// LDS read (completion is awaited with wait_vmcnt + a barrier).  M0 cannot
// be declared clobbered (it is reserved); these kernels use M0 for nothing
// else, which the generated code confirms (only these s_mov_b32 m0 write it).
__device__ __forceinline__ void g2lds16_so(const void *sbase, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_addr), "v"(voff), "s"(sbase)
               : "memory");
}

template <int D>
struct AttnTile {
  static constexpr int kSlots = D <= 64 ? 8 : 16;  // 16-byte chunks per LDS row (D / 8 of them in use)
  static constexpr int kRowB = 16 * kSlots;
  // Chunk c of K row r: the 16 rows of a quarter-wave's ds_read_b128 fall
  // on 16 distinct 16-byte slots of the 64 banks.
  static __device__ __forceinline__ uint32_t k_swz(uint32_t r) { return kSlots == 8 ? (r >> 1) & 7u : r & 15u; }
  // Chunk c of V row r: the 4 rows x 4 chunks of a half-wave's transposing
  // reads likewise; unchanged by steps of 8 rows.
  static __device__ __forceinline__ uint32_t v_swz(uint32_t r) {
    return kSlots == 8 ? 4u * ((r >> 1) & 1u) : 4u * (r & 3u);
  }
};

}  // namespace
