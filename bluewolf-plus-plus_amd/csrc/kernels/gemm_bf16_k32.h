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
template <bool MNC>
__device__ __forceinline__ uint32_t tile16_off(uint32_t ld, uint32_t blk, int lane, uint32_t lim) {
  const uint32_t q = blk * 64u + (uint32_t)lane;
  if constexpr (!MNC) {
    const uint32_t row = q >> 2, c = (q & 3u) ^ kc16_swz(row);
    return 2u * (min(row, lim - 1u) * ld + 8u * c);
  } else {
    const uint32_t k = q / 32u, c = (q % 32u) ^ mnc16_swz(k);
    return 2u * (k * ld + min(8u * c, lim - 8u));
  }
}
// MFMA operand: rows (columns) rb + lane % 16, k = 8 (lane / 16) .. + 7.
template <bool MNC>
__device__ __forceinline__ bf16x8_t read16(const unsigned char *tile, uint32_t rb, int lane) {
  if constexpr (!MNC) {
    const uint32_t row = rb + (uint32_t)(lane & 15), c = (uint32_t)(lane >> 4);
    return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const uint4 *>(tile + row * 64u + 16u * (c ^ kc16_swz(row))));
  } else {
    const uint32_t g = (uint32_t)(lane >> 4), L = (uint32_t)(lane & 15);
    const uint32_t col = rb + 4u * (L & 3u), c = col >> 3, sub = (col & 7u) * 2u;
    const uint32_t k0 = 8u * g + (L >> 2);
    const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t *)(tile + k0 * 512u + 16u * (c ^ mnc16_swz(k0)) + sub));
    const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t *)(tile + (k0 + 4u) * 512u + 16u * (c ^ mnc16_swz(k0 + 4u)) + sub));
    typedef short v8s_t __attribute__((ext_vector_type(8)));
    const v8s_t v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8_t, v);
  }
}

template <bool TA, bool TB, bool PAIRS, class EPI>
__device__ __forceinline__ void gemm_bf16_k32(const BwppGemmArgs &a, const EPI &epi) {
  constexpr int BM = 256, BN = 256, WM = 2, WN = 4, NW = WM * WN, STAGES = 4;
  constexpr int S0 = 8;  // MFMAs ahead of a step's barrier
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 16, FN = TN / 16;
  constexpr int kTile = 256 * 64, kStage = 2 * kTile, kDma = 32 / NW, kHalfD = kDma / 2;
  constexpr int kReads = FM + FN, kMfma = FM * FN;
  constexpr int kRing = STAGES * kStage, kEpi = BM * (BN + 8) * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kRing > kEpi ? kRing : kEpi];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  uint32_t tm, tn;
  const uint16_t *A = static_cast<const uint16_t *>(a.a), *B = static_cast<const uint16_t *>(a.b);
  const uint32_t tiles = a.tiles_m * a.tiles_n;
  const uint32_t split = a.ksplit > 1 ? blockIdx.x / tiles : 0u;
  tile_coords(a, tm, tn, blockIdx.x - split * tiles);
  const uint32_t kbeg = a.ksplit > 1 ? split * a.kchunk : 0u;
  const uint32_t klen = a.ksplit > 1 ? min(a.K - kbeg, a.kchunk) : a.K;
  const uint32_t m0 = tm * BM, n0 = tn * BN;
  const uint32_t nk = klen / 32;
  A += TA ? (size_t)kbeg * a.lda + m0 : (size_t)m0 * a.lda + kbeg;
  B += TB ? (size_t)n0 * a.ldb + kbeg : (size_t)kbeg * a.ldb + n0;
  const size_t stepA = TA ? (size_t)32 * a.lda : 32, stepB = TB ? 32 : (size_t)32 * a.ldb;
  uint32_t offA[kHalfD], offB[kHalfD];
#pragma unroll
  for (int i = 0; i < kHalfD; ++i) {
    offA[i] = tile16_off<TA>(a.lda, (uint32_t)(wave * kHalfD + i), lane, a.M - m0);
    offB[i] = tile16_off<!TB>(a.ldb, (uint32_t)(wave * kHalfD + i), lane, a.N - n0);
  }
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
  const uint32_t ldsA = lds0 + (uint32_t)(wave * kHalfD) * 1024u, ldsB = ldsA + kTile;
  auto dma = [&](int d, uint32_t kt, uint32_t st) {
    if (d < kHalfD) g2lds16_so(A + kt * stepA, offA[d], ldsA + st * kStage + (uint32_t)d * 1024u);
    else g2lds16_so(B + kt * stepB, offB[d - kHalfD], ldsB + st * kStage + (uint32_t)(d - kHalfD) * 1024u);
  };
  f32x4_t acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  bf16x8_t fa[2][FM], fb[2][FN];
  auto read = [&](auto set, int r, const unsigned char *st) {
    constexpr int b = decltype(set)::value;
    if (r < FM) fa[b][r] = read16<TA>(st, (uint32_t)(wm * TM + r * 16), lane);
    else fb[b][r - FM] = read16<!TB>(st + kTile, (uint32_t)(wn * TN + (r - FM) * 16), lane);
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
