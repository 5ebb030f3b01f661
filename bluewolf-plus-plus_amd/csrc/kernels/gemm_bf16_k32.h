// A second main loop for bf16 products on 256 x 256 tiles, with an epilogue of
// the caller's (gemm_bf16.h describes those), on v_mfma_f32_16x16x32_bf16.
//
// The chip is held back by power here, not by its matrix pipes (8192^3, random
// data: 1.7 to 1.9 GHz of 2.4), so a product takes the time that its energy
// takes.  A 16 x 16 x 32 MFMA reads and writes its accumulators once for 32 k, a
// 32 x 32 x 16 one for 16; and K-contiguous rows are fetched a pair of K tiles at
// a time, both halves of a 128-byte line one after the other (the second from the
// L1 cache).  8192^3, op(B) transposed: 873 us on gemm_bf16_pipe, 793 on this loop,
// 771 with the pairs; row-major B 852 -> 780.
//
// Eight waves in 2 x 4, each 128 x 64 (8 x 4 tiles); K tiles of 32, one MFMA deep,
// in a ring of four LDS stages.  Step kt multiplies tile kt from registers while
// tile kt + 1's operands are read from LDS into the other register set and tiles
// kt + 4 (pairs: kt + 3 and kt + 4, in odd steps) are fetched into the stages that
// are free.  The step's barrier comes after its first MFMAs: tile kt + 1 is in LDS
// for every wave, and nobody reads tile kt's stage any more.  Past the last tile
// the loop goes on fetching the last one and reading stages that nothing uses, so
// every step is the same.
//
// BM = 128 (half tiles): where 256-row tiles would leave CUs idle.
//
// SPLIT: fp32 operands as bf16 terms, v = v1 + v2 + v3 (8 + 8 + 8 bits of the
// significand, exact but for underflow), each a plane of its own, and the product
// as six bf16 ones, smallest first: a3 b1, a1 b3, a2 b2, a2 b1, a1 b2, a1 b1 (the
// three left out are 2^-25 of it or less).  The six run as one K six times as long,
// at 4 times the fp32 matrix rate and more.  An infinity or NaN lies in v1 alone;
// the terms that multiply the other side's v2 and v3 take v1 from a plane where
// such values are 0, so the sum is that of fp32 (no infinity meets a remainder).
//
// M and N are any as long as an operand's 16-byte chunks are whole (rows and
// columns past them re-read the last ones; the epilogue leaves them out); K is a
// multiple of 32, and so is a K split's range.
#pragma once

#include "gemm_bf16.h"

namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct Frag16 {  // v_mfma_f32_16x16x32_bf16
  static constexpr int kSize = 16, kRegs = 4;
  static __device__ __forceinline__ uint32_t row(int lane) { return (uint32_t)(lane & 15); }
  static __device__ __forceinline__ uint32_t col(int lane, int r) { return (uint32_t)(4 * (lane >> 4) + r); }
};

// Positions of 16-byte chunks in LDS.  A K-contiguous tile has rows of four:
// chunk c of a row at c ^ kc16_swz(row), so that the lanes a ds_read_b128 serves
// together (four runs of four rows, two of the next chunk) hit 16 positions of the
// 64 banks.  An MN-contiguous one has k-rows of 32: the transposing reads of 16
// columns at k and k + 8 meet in different halves.
__device__ __forceinline__ uint32_t kc16_swz(uint32_t row) {
  const uint32_t r = (row >> 2) & 3u;
  return r ^ ((r & 1u) << 1);
}
__device__ __forceinline__ uint32_t mnc16_swz(uint32_t k) { return 4u * (k & 3u) ^ 2u * ((k >> 3) & 1u); }

// Byte offset from the tile's origin of this lane's chunk in 1 KiB block `blk`;
// `lim` rows or columns exist.
template <bool MNC, int W>
__device__ __forceinline__ uint32_t tile16_off(uint32_t ld, uint32_t blk, int lane, uint32_t lim) {
  const uint32_t q = blk * 64u + (uint32_t)lane;
  if constexpr (!MNC) {
    const uint32_t row = q >> 2, c = (q & 3u) ^ kc16_swz(row);
    return 2u * (min(row, lim - 1u) * ld + 8u * c);
  } else {
    const uint32_t k = q / (W / 8u), c = (q % (W / 8u)) ^ mnc16_swz(k);
    return 2u * (k * ld + min(8u * c, lim - 8u));
  }
}
// MFMA operand: rows (columns) rb + lane % 16, k = 8 (lane / 16) .. + 7.
template <bool MNC, int W>
__device__ __forceinline__ bf16x8_t read16(const unsigned char *tile, uint32_t rb, int lane) {
  if constexpr (!MNC) {
    const uint32_t row = rb + (uint32_t)(lane & 15), c = (uint32_t)(lane >> 4);
    return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const uint4 *>(tile + row * 64u + 16u * (c ^ kc16_swz(row))));
  } else {
    const uint32_t g = (uint32_t)(lane >> 4), L = (uint32_t)(lane & 15);
    const uint32_t col = rb + 4u * (L & 3u), c = col >> 3, sub = (col & 7u) * 2u;
    const uint32_t k0 = 8u * g + (L >> 2);
    const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t *)(tile + k0 * (2u * W) + 16u * (c ^ mnc16_swz(k0)) + sub));
    const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t *)(tile + (k0 + 4u) * (2u * W) + 16u * (c ^ mnc16_swz(k0 + 4u)) + sub));
    typedef short v8s_t __attribute__((ext_vector_type(8)));
    const v8s_t v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8_t, v);
  }
}

// The block's tile and K range: each XCD (blocks go to the eight in turn) takes one
// run of them, K range by K range, so that its L2 holds the panels they share (777 x
// 1021 from 8003 columns in eight ranges of 28 tiles, fp32 in terms: 146 -> 102 us).
__device__ __forceinline__ void k32_tile(const BwppGemmArgs &a, uint32_t &tm, uint32_t &tn, uint32_t &split) {
  const uint32_t x = blockIdx.x & 7u, each = gridDim.x >> 3, more = gridDim.x & 7u;
  uint32_t b = x * each + min(x, more) + (blockIdx.x >> 3);
  const uint32_t tiles = a.tiles_m * a.tiles_n;
  split = a.ksplit > 1 ? b / tiles : 0u;
  b -= split * tiles;
  const uint32_t per_group = a.group_m * a.tiles_n, g = b / per_group, first = g * a.group_m;
  const uint32_t rows = min(a.group_m, a.tiles_m - first), idx = b - g * per_group;
  tm = first + idx % rows;
  tn = idx / rows;
}

template <bool TA, bool TB, int BM, bool PAIRS, bool SPLIT, class EPI>
__device__ __forceinline__ void gemm_bf16_k32(const BwppGemmArgs &a, const EPI &epi, const BwppSplitTerms &terms = {}) {
  constexpr int BN = 256, WM = 2, WN = 4, NW = WM * WN, STAGES = 4;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int S0 = FM;  // MFMAs ahead of a step's barrier
  constexpr int kTileA = BM * 64, kStage = kTileA + BN * 64;
  constexpr int kDmaA = BM / 16 / NW, kDmaB = BN / 16 / NW, kDma = kDmaA + kDmaB;
  constexpr int kReads = FM + FN, kMfma = FM * FN;
  constexpr int kRing = STAGES * kStage, kEpi = BM * (BN + 8) * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kRing > kEpi ? kRing : kEpi];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  uint32_t tm, tn, split;
  const uint16_t *A = static_cast<const uint16_t *>(a.a), *B = static_cast<const uint16_t *>(a.b);
  k32_tile(a, tm, tn, split);
  const uint32_t kbeg = a.ksplit > 1 ? split * a.kchunk : 0u;
  const uint32_t klen = a.ksplit > 1 ? min(a.K - kbeg, a.kchunk) : a.K;
  const uint32_t m0 = tm * BM, n0 = tn * BN;
  // (a plane of terms has zeros up to a multiple of 32, either way)
  const uint32_t am = SPLIT ? (a.M + 31u) & ~31u : a.M, bn = SPLIT ? (a.N + 31u) & ~31u : a.N;
  const uint32_t nk1 = klen / 32, nk = SPLIT ? 6 * nk1 : nk1;
  A += TA ? (size_t)kbeg * a.lda + m0 : (size_t)m0 * a.lda + kbeg;
  B += TB ? (size_t)n0 * a.ldb + kbeg : (size_t)kbeg * a.ldb + n0;
  const size_t stepA = TA ? (size_t)32 * a.lda : 32, stepB = TB ? 32 : (size_t)32 * a.ldb;
  uint32_t offA[kDmaA], offB[kDmaB];
#pragma unroll
  for (int i = 0; i < kDmaA; ++i) offA[i] = tile16_off<TA, BM>(a.lda, (uint32_t)(wave * kDmaA + i), lane, am - m0);
#pragma unroll
  for (int i = 0; i < kDmaB; ++i) offB[i] = tile16_off<!TB, BN>(a.ldb, (uint32_t)(wave * kDmaB + i), lane, bn - n0);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
  const uint32_t ldsA = lds0 + (uint32_t)(wave * kDmaA) * 1024u, ldsB = lds0 + kTileA + (uint32_t)(wave * kDmaB) * 1024u;
  auto dma = [&](int d, uint32_t kt, uint32_t st) {
    const uint16_t *At = A, *Bt = B;
    if constexpr (SPLIT) {
      const uint32_t t = (kt >= nk1) + (kt >= 2 * nk1) + (kt >= 3 * nk1) + (kt >= 4 * nk1) + (kt >= 5 * nk1);
      kt -= t * nk1;
      At += (terms.a_planes >> (4 * t) & 15u) * terms.a_stride;
      Bt += (terms.b_planes >> (4 * t) & 15u) * terms.b_stride;
    }
    if (d < kDmaA) g2lds16_so(At + kt * stepA, offA[d], ldsA + st * kStage + (uint32_t)d * 1024u);
    else g2lds16_so(Bt + kt * stepB, offB[d - kDmaA], ldsB + st * kStage + (uint32_t)(d - kDmaA) * 1024u);
  };
  f32x4_t acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  bf16x8_t fa[2][FM], fb[2][FN];
  auto read = [&](auto set, int r, const unsigned char *st) {
    constexpr int b = decltype(set)::value;
    if (r < FM) fa[b][r] = read16<TA, BM>(st, (uint32_t)(wm * TM + r * 16), lane);
    else fb[b][r - FM] = read16<!TB, BN>(st + kTileA, (uint32_t)(wn * TN + (r - FM) * 16), lane);
  };
  auto mfma = [&](auto set, int s) {
    constexpr int b = decltype(set)::value;
    const int i = s / FM, j = s % FM;
    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[b][i], fa[b][j], acc[i][j], 0, 0, 0);
  };
  const uint32_t last = nk - 1;
#pragma unroll
  for (int st = 0; st < STAGES; ++st)
#pragma unroll
    for (int d = 0; d < kDma; ++d) dma(d, min((uint32_t)st, last), (uint32_t)st);
  wait_vmcnt<(STAGES - 1) * kDma>();
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kReads; ++r) read(std::integral_constant<int, 0>{}, r, smem);
  uint32_t cur = 0;  // stage of tile kt
  auto step = [&](uint32_t kt, auto set) {
    constexpr int b = decltype(set)::value;
    const uint32_t nst = cur + 1 == STAGES ? 0 : cur + 1, kd = min(kt + STAGES, last);
    const unsigned char *nx = smem + nst * kStage;
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < S0; ++s) mfma(set, s);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): tile kt's operands are in registers
    // Tile kt + 1: what was issued after it may be in flight.
    if constexpr (PAIRS && b == 1) wait_vmcnt<1>();
    else wait_vmcnt<2 * kDma>();
    __syncthreads();
    constexpr int kRest = kMfma - S0, kGap = kRest / kReads > 0 ? kRest / kReads : 1, kGapD = kRest / kDma;
#pragma unroll
    for (int s = S0; s < kMfma; ++s) {
      const int t = s - S0;
      if (t % kGap == 0 && t / kGap < kReads) read(std::integral_constant<int, 1 - b>{}, t / kGap, nx);
      if (t % kGapD == kGapD / 2 && t / kGapD < kDma) {
        if constexpr (!PAIRS) {
          dma(t / kGapD, kd, cur);
        } else if constexpr (b == 1) {
          dma(t / kGapD, min(kt - 1 + STAGES, last), cur - 1);
          dma(t / kGapD, kd, cur);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      mfma(set, s);
      __builtin_amdgcn_sched_barrier(0);
    }
    cur = nst;
  };
  using T0 = std::integral_constant<int, 0>;
  using T1 = std::integral_constant<int, 1>;
  for (uint32_t kt = 0; kt + 1 < nk; kt += 2) {
    step(kt, T0{});
    step(kt + 1, T1{});
  }
  if (nk & 1) step(last, T0{});
  wait_vmcnt<0>();  // the fetches past the end
  __syncthreads();
  epi.template run<Frag16, BM, BN, WM, WN>(acc, smem, m0, n0, tn, split, tid, wm, wn);
}

}  // namespace
