// The bf16 matrix products' main loops: full 256-row tiles (gemm.hip), and tiles
// for any M, N and K (gemm.hip, xent.h), these with an epilogue of the caller's:
// EpiStore stores C = acc (+ bias) (-> SiLU) in bf16, or a K split's raw sums;
// any other gets the accumulators.
#pragma once

#include <type_traits>

#include "common.h"
#include "../kargs.h"

using namespace bwpp;

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

namespace {

constexpr uint32_t kEpiAdd = 1u, kEpiSilu = 2u;

__device__ __forceinline__ void tile_coords(const BwppGemmArgs &a, uint32_t &tm, uint32_t &tn,
                                            uint32_t b = blockIdx.x) {
  const uint32_t T = a.tiles_m * a.tiles_n;
  if ((T & 7u) == 0) b = (b & 7u) * (T >> 3) + (b >> 3);
  const uint32_t gm = a.group_m;
  const uint32_t per_group = gm * a.tiles_n;
  const uint32_t g = b / per_group;
  const uint32_t first = g * gm;
  const uint32_t rows = min(gm, a.tiles_m - first);
  const uint32_t idx = b - g * per_group;
  tm = first + idx % rows;
  tn = idx / rows;
}

// x / (1 + e^-x) with the hardware exp2 and reciprocal (about 2 ulp):
// e^-x overflows to +inf for x < -88 and the result is then -0, as the
// reference's x / (1 + expf(-x)).
__device__ __forceinline__ float silu(float x) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f));
}

// A caller's epilogue has kStore = false and
//   run<Frag32, BM, BN, WM, WN>(acc, smem, m0, n0, tn, split, tid, wm, wn)
// with f32x16_t acc[FN][FM]: register r of acc[i][j] in lane l is row m0 + wm TM
// + 32 j + Frag32::row(l) and column n0 + wn TN + 32 i + Frag32::col(l, r) (TM =
// BM / WM, TN = BN / WN).  smem is free (BM (BN + 8) bf16 at least).
struct Frag32 {  // v_mfma_f32_32x32x16_bf16
  static constexpr int kSize = 32, kRegs = 16;
  static __device__ __forceinline__ uint32_t row(int lane) { return (uint32_t)(lane & 31); }
  static __device__ __forceinline__ uint32_t col(int lane, int r) { return (uint32_t)(8 * (r / 4) + 4 * (lane >> 5) + r % 4); }
};
struct EpiStore {
  static constexpr bool kStore = true;
};

// ------------------------------------------------- bf16, pipelined (full tiles)
//
// Register-free staging: every operand byte goes global -> LDS with
// global_load_lds (16 bytes per lane; the lanes of one instruction fill
// 1 KiB of LDS in lane order, each lane from its own global address), into
// a ring of STAGES stages of BK = 32 (the 8-wave kernels: three, two K
// tiles in flight while the third is multiplied).
//   K-contiguous operand ("KC": A, or B with TB): LDS [rows][32 k],
//     64-byte rows of four 16-byte chunks, chunk c of row r at
//     c ^ ((r >> 2) & 3), so the 16 rows read by 16 lanes of a ds_read_b128
//     hit 16 distinct 16-byte bank groups.
//   MN-contiguous operand ("MNC": row-major B, or A with TA): LDS
//     [32 k][W], 2 W-byte rows, chunk c of row k at c ^ (4 * (k & 3)); the
//     MFMA operand (8 consecutive k of one row/column per lane) is read with
//     two ds_read_b64_tr_b16: in each 16-lane group, lane L fetches 4
//     elements of k-row kb + L/4 at column c0 + 4 * (L % 4), and the
//     hardware returns to lane j the 4 k-values of column c0 + j.
// Needs M a multiple of 256, N of 256 (of 8 for the 384-wide tiles), K of
// 32, and 16-byte aligned rows.

typedef short v4s_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s_t lds_v4s_t;

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  // s_waitcnt with expcnt / lgkmcnt at their maxima (gfx9 encoding).
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4) | (15 << 8));
}

constexpr int kPipeBK = 32;

__device__ __forceinline__ uint32_t kc_off(uint32_t row, uint32_t c) {
  return row * 64u + 16u * (c ^ ((row >> 2) & 3u));
}
// MN-contiguous tile W elements wide: 2 W-byte k-rows of W / 8 chunks, chunk
// c of row k at c ^ mnc_swz(k): the 4 k-rows x 4 chunks of a half-wave's
// transposing reads fall on 16 distinct 16-byte slots of the 64 banks.
template <int W>
__device__ __forceinline__ uint32_t mnc_swz(uint32_t k) {
  static_assert(W % 128 == 0 || W == 64 || W == 32, "k-rows of 4, 8 or a multiple of 16 chunks");
  return W == 32 ? 0u : W == 64 ? 4u * ((k >> 1) & 1u) : 4u * (k & 3u);
}
template <int W>
__device__ __forceinline__ uint32_t mnc_off(uint32_t k, uint32_t c) {
  return k * (2u * W) + 16u * (c ^ mnc_swz<W>(k));
}

// 16 bytes per lane, global -> LDS (M0 holds the wave's LDS destination;
// lane l lands at M0 + 16 * l).  Issued as inline asm so that the
// compiler's conservative LDS-DMA tracking (an s_waitcnt vmcnt(0) before
// every later LDS read) does not flatten the stage ring: completion is
// awaited explicitly with wait_vmcnt() + a barrier before a stage is read.
__device__ __forceinline__ void g2lds16(const void *gptr, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_addr), "v"(gptr)
               : "memory");
}
// The same from a wave-uniform base (SGPRs) plus a 32-bit byte offset per
// lane: one VGPR per lane instead of a 64-bit address.
__device__ __forceinline__ void g2lds16_so(const void *sbase, uint32_t voff, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_addr), "v"(voff), "s"(sbase)
               : "memory");
}

// Source of this lane's 16-byte chunk in 1 KiB block `blk` of an operand
// tile of W rows (KC) or W columns (MNC) whose first K index is 0 (the
// caller adds the K advance).  CLAMP: rows (KC) or columns (MNC) from
// `lim` on re-read the last ones (a tile that overhangs N; those results
// are never stored).
template <bool MNC, int W, bool CLAMP = false>
__device__ __forceinline__ const uint16_t *tile_src(const uint16_t *g, uint32_t ld, uint32_t r0, uint32_t blk,
                                                    int lane, uint32_t lim = 0) {
  const uint32_t q = blk * 64u + (uint32_t)lane;
  if constexpr (!MNC) {
    const uint32_t row = q >> 2, c = (q & 3u) ^ ((row >> 2) & 3u);
    uint32_t r = r0 + row;
    if constexpr (CLAMP) r = min(r, lim - 1u);
    return g + (size_t)r * ld + 8u * c;
  } else {
    constexpr uint32_t kChunks = W / 8;
    const uint32_t k = q / kChunks, c = (q % kChunks) ^ (4u * (k & 3u));
    uint32_t col = r0 + 8u * c;
    if constexpr (CLAMP) col = min(col, lim - 8u);
    return g + (size_t)k * ld + col;
  }
}

// The same chunk as a byte offset from the tile's origin (row or column
// r0 at K = 0), in 32-bit arithmetic: ld * 2 * (rows of a KC tile) must
// stay below 2^32.
template <bool MNC, int W, bool CLAMP = false>
__device__ __forceinline__ uint32_t tile_off(uint32_t ld, uint32_t r0, uint32_t blk, int lane, uint32_t lim = 0) {
  const uint32_t q = blk * 64u + (uint32_t)lane;
  if constexpr (!MNC) {
    const uint32_t row = q >> 2, c = (q & 3u) ^ ((row >> 2) & 3u);
    uint32_t r = row;
    if constexpr (CLAMP) r = min(r, lim - 1u - r0);
    return 2u * (r * ld + 8u * c);
  } else {
    constexpr uint32_t kChunks = W / 8;
    const uint32_t k = q / kChunks, c = (q % kChunks) ^ (4u * (k & 3u));
    uint32_t col = 8u * c;
    if constexpr (CLAMP) col = min(col, lim - 8u - r0);
    return 2u * (k * ld + col);
  }
}

// MFMA operand (8 bf16: rows rb + lane%32, k = 16*ks + 8*(lane/32) .. +7)
// of a tile W rows (KC) or W columns (MNC) wide.
template <bool MNC, int W>
__device__ __forceinline__ bf16x8_t read_operand(const unsigned char *tile, uint32_t rb, int ks, int lane) {
  if constexpr (!MNC) {
    const uint32_t row = rb + (uint32_t)(lane & 31);
    const uint32_t c = (uint32_t)(2 * ks + (lane >> 5));
    return __builtin_bit_cast(bf16x8_t, *reinterpret_cast<const uint4 *>(tile + kc_off(row, c)));
  } else {
    const uint32_t g = (uint32_t)((lane >> 4) & 3), L = (uint32_t)(lane & 15);
    const uint32_t col = rb + 16u * (g & 1u) + 4u * (L & 3u);
    const uint32_t c = col >> 3;
    const uint32_t sub = (col & 7u) * 2u;
    const uint32_t k0 = (uint32_t)(16 * ks) + 8u * (g >> 1) + (L >> 2);
    const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_v4s_t *)(tile + mnc_off<W>(k0, c) + sub));
    const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (lds_v4s_t *)(tile + mnc_off<W>(k0 + 4u, c) + sub));
    typedef short v8s_t __attribute__((ext_vector_type(8)));
    const v8s_t v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(bf16x8_t, v);
  }
}

template <bool V>
using bool_tag = std::integral_constant<bool, V>;

// 256 x BN output tile (BN 256 or 384), WM x WN waves (4 or 8); each wave
// owns a (256/WM) x (BN/WN) sub-tile.  STAGES K tiles of 32 in the LDS
// ring (STAGES - 1 in flight while one is multiplied).
//
// Schedule of one K tile (two 16-deep MFMA k-steps), per wave:
//   phase A: the k-step-0 MFMAs, interleaved with the LDS reads of k-step 1
//            and the DMA of K tile kt + STAGES - 1 into the stage freed by
//            kt - 1;
//   then:    lgkmcnt(0) (this wave is done reading tile kt), vmcnt down to
//            the tiles younger than kt + 1, barrier (tile kt + 1 is in LDS
//            for every wave, and nobody reads tile kt any more);
//   phase B: the k-step-1 MFMAs, interleaved with the LDS reads of k-step 0
//            of tile kt + 1.
// The MFMA pipe thus always has work queued while LDS reads and DMA issue,
// and there is one barrier per K tile.  sched_barrier(0) pins the order the
// source gives (the DMA is inline asm, which the scheduler cannot classify).
//
// BN = 384 (a 384-wide B tile: a sixth fewer L2 -> LDS bytes per FLOP than
// 256 x 256, and fewer LDS operand bytes per MFMA): the ring's 40 KiB
// stages fit three deep, the epilogue stages C through LDS in two halves
// of 128 rows, and N need only be a multiple of 8 -- a tile column that
// overhangs N re-reads B's last columns (or rows) and stores only n < N.
template <bool TA, bool TB, int WM, int WN, int BN = 256, int STAGES = 4>
__device__ __forceinline__ void gemm_bf16_pipe(const BwppGemmArgs &a) {
  constexpr int BM = 256;
  constexpr int NW = WM * WN, NT = 64 * NW;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
  constexpr int kTileA = BM * kPipeBK * 2, kTileB = BN * kPipeBK * 2;  // bytes per operand tile
  constexpr int LPA = kTileA / 1024 / NW, LPB = kTileB / 1024 / NW;     // 1 KiB DMA blocks per wave
  static_assert(LPA * NW * 1024 == kTileA && LPB * NW * 1024 == kTileB, "DMA blocks split evenly over the waves");
  static_assert(TN % 32 == 0 && TM % 32 == 0 && STAGES >= 2 && STAGES <= 4, "tile shape");
  constexpr bool kEdgeN = BN != 256;
  // Lean register use (the 8-wave 384-wide tile holds 192 accumulator
  // VGPRs): DMA sources as 32-bit offsets from wave-uniform tile origins,
  // and one set of A operands, each re-read for the next k-step as soon as
  // its last MFMA of the current one has issued (MFMAs in A-operand order).
  constexpr bool kLean = BN != 256;
  constexpr int kStage = kTileA + kTileB;
  constexpr int kCld = BN + 8;
  constexpr int kRing = STAGES * kStage;
  constexpr int kHalves = BM * kCld * 2 + BN * 2 > 163840 ? 2 : 1;  // epilogue passes over the rows
  static_assert(kHalves == 1 || WM == kHalves, "one wave row per epilogue half");
  constexpr int kHR = BM / kHalves;  // rows per epilogue half
  constexpr int kEpi = kHR * kCld * 2;
  constexpr int kBiasOff = kRing > kEpi ? kRing : kEpi;  // bias row (bf16) after both
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kBiasOff + BN * 2];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  uint32_t tm, tn;
  tile_coords(a, tm, tn);
  const uint32_t m0 = tm * BM, n0 = tn * BN;
  const uint16_t *A = static_cast<const uint16_t *>(a.a);
  const uint16_t *B = static_cast<const uint16_t *>(a.b);
  const uint32_t nk = a.K / kPipeBK;
  const uint16_t *bias = static_cast<const uint16_t *>(a.bias);
  const bool add = (a.epilogue & kEpiAdd) && bias;
  const bool act = (a.epilogue & kEpiSilu) != 0;

  const uint16_t *bias_s = reinterpret_cast<const uint16_t *>(smem + kBiasOff);

  // Per-lane DMA sources at K = 0, advanced by a fixed step per K tile.
  const uint16_t *srcA[kLean ? 1 : LPA], *srcB[kLean ? 1 : LPB];
  uint32_t offA[kLean ? LPA : 1], offB[kLean ? LPB : 1];  // lean: bytes from baseA / baseB
  const uint16_t *baseA = A + (TA ? (size_t)m0 : (size_t)m0 * a.lda);
  const uint16_t *baseB = B + (TB ? (size_t)n0 * a.ldb : (size_t)n0);
#pragma unroll
  for (int i = 0; i < LPA; ++i) {
    if constexpr (kLean) offA[i] = tile_off<TA, BM>(a.lda, m0, (uint32_t)(wave * LPA + i), lane);
    else srcA[i] = tile_src<TA, BM>(A, a.lda, m0, (uint32_t)(wave * LPA + i), lane);
  }
#pragma unroll
  for (int i = 0; i < LPB; ++i) {
    if constexpr (kLean) offB[i] = tile_off<!TB, BN, kEdgeN>(a.ldb, n0, (uint32_t)(wave * LPB + i), lane, a.N);
    else srcB[i] = tile_src<!TB, BN>(B, a.ldb, n0, (uint32_t)(wave * LPB + i), lane);
  }
  const size_t stepA = TA ? (size_t)kPipeBK * a.lda : (size_t)kPipeBK;
  const size_t stepB = TB ? (size_t)kPipeBK : (size_t)kPipeBK * a.ldb;
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
  const uint32_t ldsA = lds_base + (uint32_t)(wave * LPA) * 1024u;
  const uint32_t ldsB = lds_base + (uint32_t)kTileA + (uint32_t)(wave * LPB) * 1024u;

  // DMA instruction d (0 .. LPA+LPB-1) of K tile kt.
  auto dma = [&](int d, uint32_t kt) {
    const uint32_t st = (kt % STAGES) * kStage;
    if constexpr (kLean) {
      if (d < LPA)
        g2lds16_so(baseA + kt * stepA, offA[d], ldsA + st + (uint32_t)d * 1024u);
      else
        g2lds16_so(baseB + kt * stepB, offB[d - LPA], ldsB + st + (uint32_t)(d - LPA) * 1024u);
    } else {
      if (d < LPA)
        g2lds16(srcA[d] + kt * stepA, ldsA + st + (uint32_t)d * 1024u);
      else
        g2lds16(srcB[d - LPA] + kt * stepB, ldsB + st + (uint32_t)(d - LPA) * 1024u);
    }
  };

  f32x16_t acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  // fa/fb[0]: operands of k-step 0, [1]: of k-step 1 (lean: one fa set).
  bf16x8_t fa[kLean ? 1 : 2][FM], fb[2][FN];
  constexpr int kReads = FM + FN, kMfma = FM * FN, kDma = LPA + LPB;
  static_assert(kReads <= kMfma && kDma <= kMfma, "interleave needs an MFMA slot per read and DMA");
  // Wait until at most the y youngest K tiles' DMA are still in flight.
  auto wait_younger = [&](uint32_t y) {
    if constexpr (STAGES >= 4) {
      if (y >= 2) {
        wait_vmcnt<2 * kDma>();
        return;
      }
    }
    if (STAGES >= 3 && y >= 1) wait_vmcnt<kDma>();
    else wait_vmcnt<0>();
  };

  auto stage_ptr = [&](uint32_t kt) { return smem + (kt % STAGES) * kStage; };
  auto read = [&](auto buf, int r, const unsigned char *As, int ks) {
    constexpr int b = decltype(buf)::value ? 1 : 0;
    if (r < FM)
      fa[kLean ? 0 : b][r] = read_operand<TA, BM>(As, (uint32_t)(wm * TM + r * 32), ks, lane);
    else
      fb[b][r - FM] = read_operand<!TB, BN>(As + kTileA, (uint32_t)(wn * TN + (r - FM) * 32), ks, lane);
  };
  auto mfma = [&](auto buf, int s) {
    constexpr int b = decltype(buf)::value ? 1 : 0;
    const int i = kLean ? s % FN : s / FM, j = kLean ? s / FN : s % FM;
    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[b][i], fa[kLean ? 0 : b][j], acc[i][j], 0, 0, 0);
  };

  // The tile's BN bias values (16-byte aligned) are copied to LDS by the
  // first lanes of wave 0, ahead of its first K tile, so the prologue wait
  // and barrier publish them and the epilogue never waits on a global load.
  if (add && wave == 0 && lane < BN / 8) {
    uint32_t nb = n0 + 8u * (uint32_t)lane;
    if constexpr (kEdgeN) nb = min(nb, a.N - 8u);
    g2lds16(bias + nb, lds_base + (uint32_t)kBiasOff);
  }
#pragma unroll
  for (int st = 0; st < STAGES - 1; ++st)
    if ((uint32_t)st < nk) {
#pragma unroll
      for (int d = 0; d < kDma; ++d) dma(d, (uint32_t)st);
    }
  wait_younger(nk >= (uint32_t)(STAGES - 1) ? (uint32_t)(STAGES - 2) : (nk > 0 ? nk - 1 : 0u));
  __syncthreads();
  if (nk > 0) {
#pragma unroll
    for (int r = 0; r < kReads; ++r) read(bool_tag<false>{}, r, stage_ptr(0), 0);
  }

  // One K tile; DMA: issue tile kt + STAGES - 1, NEXT: a tile kt + 1 exists.
  auto ktile = [&](uint32_t kt, auto dma_tag, auto next_tag) {
    constexpr bool kDmaOn = decltype(dma_tag)::value, kNext = decltype(next_tag)::value;
    const unsigned char *cur = stage_ptr(kt);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < kMfma; ++s) {
      mfma(bool_tag<false>{}, s);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kLean) {
        if (s < FN) {
          read(bool_tag<true>{}, FM + s, cur, 1);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (s % FN == FN - 1) {  // the last MFMA of fa[s / FN] has issued
          read(bool_tag<true>{}, s / FN, cur, 1);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else if (s < kReads) {
        read(bool_tag<true>{}, s, cur, 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (kDmaOn) {
        if (s < kDma) {
          dma(s, kt + STAGES - 1);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if constexpr (kNext) {
      // Tiles issued after kt + 1 may stay in flight.
      const uint32_t younger = min(nk - 2 - kt, (uint32_t)(STAGES - 2));
      __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): done reading tile kt
      wait_younger(younger);
      __syncthreads();
    }
    const unsigned char *nxt = stage_ptr(kt + 1);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int s = 0; s < kMfma; ++s) {
      mfma(bool_tag<true>{}, s);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (kNext && kLean) {
        if (s < FN) {
          read(bool_tag<false>{}, FM + s, nxt, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        if (s % FN == FN - 1) {
          read(bool_tag<false>{}, s / FN, nxt, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
      } else if constexpr (kNext) {
        if (s < kReads) {
          read(bool_tag<false>{}, s, nxt, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  };

  uint32_t kt = 0;
  for (; kt + STAGES - 1 < nk; ++kt) ktile(kt, bool_tag<true>{}, bool_tag<true>{});
  for (; kt + 1 < nk; ++kt) ktile(kt, bool_tag<false>{}, bool_tag<true>{});
  if (kt < nk) ktile(kt, bool_tag<false>{}, bool_tag<false>{});
  __syncthreads();

  // Epilogue through LDS (see gemm_bf16), in kHalves passes of kHR rows.
  uint16_t *cs = reinterpret_cast<uint16_t *>(smem);
  uint16_t *C = static_cast<uint16_t *>(a.c);
  const int lrow = lane & 31, lhalf = lane >> 5;
  constexpr int kRowChunks = BN / 8;
#pragma unroll
  for (int hv = 0; hv < kHalves; ++hv) {
    if (hv > 0) __syncthreads();  // the previous half has left LDS
    if (kHalves == 1 || wm == hv) {
#pragma unroll
      for (int i = 0; i < FN; ++i) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int nl = wn * TN + i * 32 + q * 8 + lhalf * 4;
          float bv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
          if (add) {
            const uint2 raw = *reinterpret_cast<const uint2 *>(bias_s + nl);
            bv[0] = __uint_as_float(raw.x << 16);
            bv[1] = __uint_as_float(raw.x & 0xffff0000u);
            bv[2] = __uint_as_float(raw.y << 16);
            bv[3] = __uint_as_float(raw.y & 0xffff0000u);
          }
#pragma unroll
          for (int j = 0; j < FM; ++j) {
            const int ml = wm * TM - hv * kHR + j * 32 + lrow;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float t = acc[i][j][q * 4 + e] + bv[e];
              if (act) t = silu(t);
              v[e] = t;
            }
            uint2 o;
            o.x = pack_bf16x2(v[0], v[1]);
            o.y = pack_bf16x2(v[2], v[3]);
            *reinterpret_cast<uint2 *>(cs + ml * kCld + nl) = o;
          }
        }
      }
    }
    __syncthreads();
#pragma unroll 4
    for (int it = 0; it < kHR * kRowChunks / NT; ++it) {
      const int q = tid + it * NT;
      const int row = q / kRowChunks, c = q % kRowChunks;
      if (!kEdgeN || n0 + (uint32_t)c * 8u < a.N)
        *reinterpret_cast<uint4 *>(C + (size_t)(m0 + hv * kHR + row) * a.ldc + n0 + c * 8) =
            *reinterpret_cast<const uint4 *>(cs + row * kCld + c * 8);
    }
  }
}

// ------------------------------------------ bf16, pipelined, any M, N and K
//
// The same LDS-DMA ring with smaller tiles, for what the 256-wide tiles leave
// idle CUs or padding: ragged M, N and K, few rows (decoding), and products
// with fewer tiles than CUs, whose K is then cut into ksplit ranges (raw
// partial tiles, added in order by bwpp_gemm_bf16_splitk_reduce).  Rows or
// columns past M / N re-read the last ones and are not stored; the chunks
// past K of the last stage are zeroed in LDS, in both operands, before it is
// multiplied.
//
// BM x BN tiles on WM x WN waves; KPS K tiles of 32 per stage, STAGES stages.
// Small blocks, several per CU: a block waits for its stage and reads its
// operands while another multiplies, which is worth more here than the
// 256-wide kernels' hand-ordered loop.  32 x 64 streams op(B) with 48 KiB in
// flight per block (16 x 4096 x 11008: 17.5 us, 5.2 TB/s; 210 on the 256 x 256
// edge tile).  64 x 128 and 128 x 128 wait for their stages, with 4 and 8
// MFMAs per wave between barriers and one to two blocks a CU: over 1337 x
// 1024 x 3000 (18.1 us; 94 before) and its weight gradient (21.8) the matrix
// pipe is busy 12-15 % of the cycles and LDS 7-13 %, without bank conflicts.
//
// REG: the operands go through registers instead (16-byte loads at any
// 2-byte address, the same LDS layout), for rows that are not 16-byte
// aligned or extents that are no multiple of 8: one stage ahead, so bound by
// the load latency where few blocks share a CU (4095 x 8191 x 2048: 170 us,
// 1085 on the edge tile's element-wise loads; 257 x 255 x 4097 split 8 ways
// 13.2, 1385).
template <bool MNC, int W>
__device__ __forceinline__ uint32_t ring_off(uint32_t ld, uint32_t blk, int lane, uint32_t lim, uint32_t klim) {
  // Byte offset of this lane's chunk of 1 KiB block `blk` (over the stage's
  // 32-deep K tiles) from the tile's origin; lim rows / columns and klim k
  // exist (multiples of 8 where chunks run along them).
  constexpr uint32_t kBlocks = W / 16;
  const uint32_t sub = blk / kBlocks, q = (blk % kBlocks) * 64u + (uint32_t)lane;
  if constexpr (!MNC) {
    const uint32_t row = q >> 2, c = (q & 3u) ^ ((row >> 2) & 3u);
    return 2u * (min(row, lim - 1u) * ld + min(sub * 32u + 8u * c, klim - 8u));
  } else {
    constexpr uint32_t kChunks = W / 8;
    const uint32_t k = q / kChunks, c = (q % kChunks) ^ mnc_swz<W>(k);
    return 2u * (min(sub * 32u + k, klim - 1u) * ld + min(8u * c, lim - 8u));
  }
}

typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4a2_t __attribute__((ext_vector_type(4), aligned(2)));
// 16 bytes at any 2-byte address (unaligned accesses are on for HSA code).
__device__ __forceinline__ u32x4_t load16_b16(const uint16_t *p) { return *reinterpret_cast<const u32x4a2_t *>(p); }
// v's bf16 elements moved down by n (0 .. 7; 8 and more: all gone), zeros
// behind them.  (No array: the compiler indexed it, in scratch.)
__device__ __forceinline__ u32x4_t shift_down_b16(u32x4_t v, uint32_t n) {
  const bool s4 = n & 4u, s2 = n & 2u, s1 = n & 1u;
  const uint32_t a0 = s4 ? v[2] : v[0], a1 = s4 ? v[3] : v[1], a2 = s4 ? 0u : v[2], a3 = s4 ? 0u : v[3];
  const uint32_t b0 = s2 ? a1 : a0, b1 = s2 ? a2 : a1, b2 = s2 ? a3 : a2, b3 = s2 ? 0u : a3;
  const uint32_t c0 = s1 ? (b0 >> 16 | b1 << 16) : b0, c1 = s1 ? (b1 >> 16 | b2 << 16) : b1;
  const uint32_t c2 = s1 ? (b2 >> 16 | b3 << 16) : b2, c3 = s1 ? b3 >> 16 : b3;
  const uint32_t keep = n < 8u ? 0xffffffffu : 0u;
  return u32x4_t{c0 & keep, c1 & keep, c2 & keep, c3 & keep};
}
// This lane's chunk of block `blk` of a stage (ring_off's chunk), for rows
// at any address and extents of any size: a chunk that would pass its row's
// end is read as the row's last 8 elements and moved down when it is stored
// (ring_fix); rows past the last re-read that.  lim rows / columns, klim k.
template <bool MNC, int W>
struct RingChunk {
  uint32_t row;  // row of the stored operand within the stage
  int col;       // first element along it
  __device__ __forceinline__ RingChunk(uint32_t blk, int lane) {
    constexpr uint32_t kBlocks = W / 16, kChunks = W / 8;
    const uint32_t sub = blk / kBlocks, q = (blk % kBlocks) * 64u + (uint32_t)lane;
    if constexpr (!MNC) {
      row = q >> 2;
      col = (int)(sub * 32u + 8u * ((q & 3u) ^ ((row >> 2) & 3u)));
    } else {
      row = sub * 32u + q / kChunks;
      col = (int)(8u * ((q % kChunks) ^ mnc_swz<W>(q / kChunks)));
    }
  }
  __device__ __forceinline__ int at(uint32_t lim, uint32_t klim) const { return min(col, (int)(MNC ? lim : klim) - 8); }
  __device__ __forceinline__ u32x4_t load(const uint16_t *g, uint32_t ld, uint32_t lim, uint32_t klim) const {
    return load16_b16(g + ((int64_t)min(row, (MNC ? klim : lim) - 1u) * ld + at(lim, klim)));
  }
  __device__ __forceinline__ u32x4_t fix(u32x4_t v, uint32_t lim, uint32_t klim) const {
    const u32x4_t r = shift_down_b16(v, (uint32_t)(col - at(lim, klim)));
    const uint32_t keep = MNC && row >= klim ? 0u : 0xffffffffu;
    return u32x4_t{r[0] & keep, r[1] & keep, r[2] & keep, r[3] & keep};
  }
};

// Zeroes the chunks of a staged operand (KPS K tiles, kTileBytes apart)
// whose k is krem or more.
template <bool MNC, int W, int KPS, int NT>
__device__ __forceinline__ void ring_zero(unsigned char *tile, uint32_t stride, uint32_t krem, int tid) {
#pragma unroll
  for (int sub = 0; sub < KPS; ++sub) {
    for (uint32_t i = (uint32_t)tid; i < W * 4u; i += NT) {
      const uint32_t row = i >> 2;
      const uint32_t k = MNC ? i / (W / 8) : 8u * ((i & 3u) ^ ((row >> 2) & 3u));
      if ((uint32_t)sub * 32u + k >= krem)
        *reinterpret_cast<uint4 *>(tile + sub * stride + 16u * i) = make_uint4(0, 0, 0, 0);
    }
  }
}

template <bool TA, bool TB, int BM, int BN, int WM, int WN, int KPS, int STAGES, bool REG, class EPI = EpiStore>
__device__ __forceinline__ void gemm_bf16_ring(const BwppGemmArgs &a, const EPI &epi = EPI{}) {
  constexpr int NW = WM * WN, NT = 64 * NW, BK = 32 * KPS;
  constexpr int TM = BM / WM, TN = BN / WN, FM = TM / 32, FN = TN / 32;
  constexpr int kTileA = BM * 64, kTileB = BN * 64, kSub = kTileA + kTileB, kStage = KPS * kSub;
  constexpr int LPA = KPS * (BM / 16) / NW, LPB = KPS * (BN / 16) / NW, kDma = LPA + LPB;
  static_assert(LPA * NW == KPS * (BM / 16) && LPB * NW == KPS * (BN / 16), "DMA blocks split evenly");
  constexpr int kCld = BN + 8, kRing = STAGES * kStage, kOut = BM * kCld * 2;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[kRing > kOut ? kRing : kOut];
  __shared__ float bias_s[BN];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave / WN, wn = wave % WN;
  const uint32_t tiles = a.tiles_m * a.tiles_n;
  const uint32_t split = a.ksplit > 1 ? blockIdx.x / tiles : 0u;
  uint32_t tm, tn;
  tile_coords(a, tm, tn, blockIdx.x - split * tiles);
  const uint32_t m0 = tm * BM, n0 = tn * BN;
  const uint32_t kbeg = a.ksplit > 1 ? split * a.kchunk : 0u;
  const uint32_t klen = a.ksplit > 1 ? min(a.K - kbeg, a.kchunk) : a.K;
  const uint32_t ns = (klen + BK - 1) / BK, krem = klen - (ns - 1) * BK;  // k of the last stage
  const uint16_t *A = static_cast<const uint16_t *>(a.a) +
                      (TA ? (size_t)kbeg * a.lda + m0 : (size_t)m0 * a.lda + kbeg);
  const uint16_t *B = static_cast<const uint16_t *>(a.b) +
                      (TB ? (size_t)n0 * a.ldb + kbeg : (size_t)kbeg * a.ldb + n0);
  const size_t stepA = TA ? (size_t)BK * a.lda : (size_t)BK, stepB = TB ? (size_t)BK : (size_t)BK * a.ldb;

  const uint16_t *bias = static_cast<const uint16_t *>(a.bias);
  const bool add = (a.epilogue & kEpiAdd) && bias && a.ksplit <= 1;
  const bool act = (a.epilogue & kEpiSilu) != 0;
  if (tid < BN) bias_s[tid] = add ? bf16_bits_to_f32(bias[min(n0 + (uint32_t)tid, a.N - 1u)]) : 0.0f;
  wait_vmcnt<0>();  // no load of the compiler's outstanding beside the DMA

  f32x16_t acc[FN][FM];
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  auto multiply = [&](const unsigned char *st) {
#pragma unroll
    for (int ks = 0; ks < 2 * KPS; ++ks) {
      const unsigned char *sub = st + (ks / 2) * kSub;
      bf16x8_t fa[FM], fb[FN];
#pragma unroll
      for (int j = 0; j < FM; ++j) fa[j] = read_operand<TA, BM>(sub, (uint32_t)(wm * TM + j * 32), ks % 2, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i)
        fb[i] = read_operand<!TB, BN>(sub + kTileA, (uint32_t)(wn * TN + i * 32), ks % 2, lane);
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int j = 0; j < FM; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fb[i], fa[j], acc[i][j], 0, 0, 0);
    }
  };

  if constexpr (!REG) {
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
    uint32_t offA[LPA], offB[LPB];
    uint32_t dstA[LPA], dstB[LPB];  // wave-uniform
#pragma unroll
    for (int i = 0; i < LPA; ++i) {
      const uint32_t blk = (uint32_t)(wave * LPA + i);
      offA[i] = ring_off<TA, BM>(a.lda, blk, lane, a.M - m0, 0xffffffffu);
      dstA[i] = lds0 + blk / (BM / 16) * kSub + blk % (BM / 16) * 1024u;
    }
#pragma unroll
    for (int i = 0; i < LPB; ++i) {
      const uint32_t blk = (uint32_t)(wave * LPB + i);
      offB[i] = ring_off<!TB, BN>(a.ldb, blk, lane, a.N - n0, 0xffffffffu);
      dstB[i] = lds0 + blk / (BN / 16) * kSub + kTileA + blk % (BN / 16) * 1024u;
    }
    auto issue = [&](uint32_t t) {
      const uint32_t st = (t % STAGES) * kStage;
      const uint16_t *At = A + t * stepA, *Bt = B + t * stepB;
      if (t + 1 < ns || krem == BK) {
#pragma unroll
        for (int i = 0; i < LPA; ++i) g2lds16_so(At, offA[i], dstA[i] + st);
#pragma unroll
        for (int i = 0; i < LPB; ++i) g2lds16_so(Bt, offB[i], dstB[i] + st);
      } else {  // the last stage, short of k
#pragma unroll
        for (int i = 0; i < LPA; ++i)
          g2lds16_so(At, ring_off<TA, BM>(a.lda, (uint32_t)(wave * LPA + i), lane, a.M - m0, krem), dstA[i] + st);
#pragma unroll
        for (int i = 0; i < LPB; ++i)
          g2lds16_so(Bt, ring_off<!TB, BN>(a.ldb, (uint32_t)(wave * LPB + i), lane, a.N - n0, krem), dstB[i] + st);
      }
    };
#pragma unroll
    for (int t = 0; t < STAGES - 1; ++t)
      if ((uint32_t)t < ns) issue((uint32_t)t);
    for (uint32_t t = 0; t < ns; ++t) {
      // Stages t + 1 .. t + STAGES - 2 may still be in flight.
      const uint32_t younger = min(ns - 1 - t, (uint32_t)(STAGES - 2));
      if (STAGES >= 4 && younger >= 2) wait_vmcnt<2 * kDma>();
      else if (STAGES >= 3 && younger >= 1) wait_vmcnt<kDma>();
      else wait_vmcnt<0>();
      __syncthreads();  // stage t is in LDS, and nobody reads stage t - 1 any more
      if (t + STAGES - 1 < ns) issue(t + STAGES - 1);
      unsigned char *st = smem + __builtin_amdgcn_readfirstlane((t % STAGES) * kStage);
      if (t + 1 == ns && krem < BK) {
        ring_zero<TA, BM, KPS, NT>(st, kSub, krem, tid);
        ring_zero<!TB, BN, KPS, NT>(st + kTileA, kSub, krem, tid);
        __syncthreads();
      }
      multiply(st);
    }
  } else {
    // Through registers: stage t + 1 is loaded while stage t is multiplied,
    // then written to the other LDS buffer.
    static_assert(STAGES == 2, "two LDS buffers");
    u32x4_t ra[LPA], rb[LPB];
    const bool edge = (TA && a.M - m0 < BM) || (!TB && a.N - n0 < BN);  // block-uniform: chunks pass M or N
    auto klim = [&](uint32_t t) { return t + 1 == ns ? krem : (uint32_t)BK; };
    // The loads take no branch (their values would be merged, and waited
    // for, where the paths meet).
    auto load = [&](uint32_t t) {
#pragma unroll
      for (int i = 0; i < LPA; ++i)
        ra[i] = RingChunk<TA, BM>((uint32_t)(wave * LPA + i), lane).load(A + t * stepA, a.lda, a.M - m0, klim(t));
#pragma unroll
      for (int i = 0; i < LPB; ++i)
        rb[i] = RingChunk<!TB, BN>((uint32_t)(wave * LPB + i), lane).load(B + t * stepB, a.ldb, a.N - n0, klim(t));
    };
    auto store = [&](uint32_t t) {
      if (edge || klim(t) < BK) {
#pragma unroll
        for (int i = 0; i < LPA; ++i)
          ra[i] = RingChunk<TA, BM>((uint32_t)(wave * LPA + i), lane).fix(ra[i], a.M - m0, klim(t));
#pragma unroll
        for (int i = 0; i < LPB; ++i)
          rb[i] = RingChunk<!TB, BN>((uint32_t)(wave * LPB + i), lane).fix(rb[i], a.N - n0, klim(t));
      }
      unsigned char *st = smem + (t & 1u) * kStage + 16 * lane;
#pragma unroll
      for (int i = 0; i < LPA; ++i) {
        const int blk = wave * LPA + i;
        *reinterpret_cast<u32x4_t *>(st + blk / (BM / 16) * kSub + blk % (BM / 16) * 1024) = ra[i];
      }
#pragma unroll
      for (int i = 0; i < LPB; ++i) {
        const int blk = wave * LPB + i;
        *reinterpret_cast<u32x4_t *>(st + blk / (BN / 16) * kSub + kTileA + blk % (BN / 16) * 1024) = rb[i];
      }
    };
    load(0);
    store(0);
    __syncthreads();
    for (uint32_t t = 0; t < ns; ++t) {
      if (t + 1 < ns) load(t + 1);
      multiply(smem + (t & 1u) * kStage);
      if (t + 1 < ns) store(t + 1);
      __syncthreads();
    }
  }

  if constexpr (!EPI::kStore) {
    __syncthreads();
    epi.template run<Frag32, BM, BN, WM, WN>(acc, smem, m0, n0, tn, split, tid, wm, wn);
    return;
  }
  const int lrow = lane & 31, lhalf = lane >> 5;
  if (a.ksplit > 1) {
    // Raw sums, rows of N rounded up to 4 floats.
    const uint32_t np = (a.N + 3u) & ~3u;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const uint32_t m = m0 + (uint32_t)(wm * TM + j * 32 + lrow);
      float *row = a.part + ((size_t)split * a.M + m) * np;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const uint32_t n = n0 + (uint32_t)(wn * TN + i * 32 + q * 8 + lhalf * 4);
          if (m < a.M && n < np)
            *reinterpret_cast<float4 *>(row + n) = make_float4(acc[i][j][4 * q], acc[i][j][4 * q + 1],
                                                               acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]);
        }
    }
    return;
  }
  __syncthreads();
  uint16_t *cs = reinterpret_cast<uint16_t *>(smem);  // [BM][BN + 8]
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int nl = wn * TN + i * 32 + q * 8 + lhalf * 4;
      const float4 bv = *reinterpret_cast<const float4 *>(bias_s + nl);
#pragma unroll
      for (int j = 0; j < FM; ++j) {
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float t = acc[i][j][4 * q + e] + (e == 0 ? bv.x : e == 1 ? bv.y : e == 2 ? bv.z : bv.w);
          v[e] = act ? silu(t) : t;
        }
        uint2 o;
        o.x = pack_bf16x2(v[0], v[1]);
        o.y = pack_bf16x2(v[2], v[3]);
        *reinterpret_cast<uint2 *>(cs + (wm * TM + j * 32 + lrow) * kCld + nl) = o;
      }
    }
  __syncthreads();
  uint16_t *C = static_cast<uint16_t *>(a.c);
#pragma unroll 2
  for (int it = 0; it < BM * (BN / 8) / NT; ++it) {
    const int q = tid + it * NT, row = q / (BN / 8), c = q % (BN / 8);
    const uint32_t m = m0 + (uint32_t)row, n = n0 + 8u * (uint32_t)c;
    if (m >= a.M || n >= a.N) continue;
    const uint16_t *h = cs + row * kCld + c * 8;
    if (n + 8 <= a.N) {
      *reinterpret_cast<u32x4a2_t *>(C + (size_t)m * a.ldc + n) = *reinterpret_cast<const u32x4_t *>(h);
    } else {
      for (uint32_t e = 0; e < 8 && n + e < a.N; ++e) C[(size_t)m * a.ldc + n + e] = h[e];
    }
  }
}

}  // namespace
