// Cross entropy of hidden states against a vocabulary, for gfx950, without
// keeping the logits:
//
//   z = scale x W                        [tokens x vocabulary]
//   lse_t = log sum_v exp z_tv           loss_t = lse_t - z_t,target
//   dz_tv = g_t (exp(z_tv - lse_t) - [v = target]),   dx = scale dz W^T,
//   dW = scale x^T dz
//
// Measured: 4 x 1024 x 16384 loss 11.8 us (W at 2.8 TB/s, and two launches), 2048 x
// 4096 x 50001 loss 666 (1260 TFLOP/s), 4096 x 2048 x 32768 train 1828 and 4096 x 4096
// x 131072 13.0 ms (1203 and 1350 TFLOP/s of the four products a call that does not
// keep the logits makes); the wide products run at the rate that the chip's power
// allows (gemm_bf16_k32.h).
//
// A target outside the vocabulary leaves its row out: loss and gradients 0.
//
// bf16: the logits' product runs on the matrix cores (gemm_bf16_k32.h's loop on 256 x
// 256 tiles, gemm_bf16.h's on 32 x 64 to 128 x 128 and for any sizes)
// and stays in its accumulators.  The forward's epilogue reduces each tile's
// rows to (max, sum of exp), a pair per row and tile, and a second kernel
// joins the pairs.  The gradient's epilogue turns the same product, made
// again from x and W, into dz, rounded to bf16 as the next two products'
// operand (each element off by at most half a step, 2^-8 of it; dx and dW add
// thousands of them, and are rounded to bf16 themselves).  A row's largest element
// by far is its target's p - 1: what its rounding leaves is kept, a float a token,
// and added by the kernels that sum dx's planes and make dW.  It does so for
// one piece of the vocabulary at a time, small enough to stay in the Infinity
// Cache between its writer and its readers.  dx is summed over the pieces in
// fp32 planes (one per K split) and rounded once; each piece's dW is final.
// fp32, few tokens: the logits of a piece go through memory once, in fp32 (8 to 16
// bytes a logit beside 2 dim FLOPs at a sixteenth of the bf16 rate).  More: x, W and
// dz as three bf16 terms each (gemm_bf16_k32.h), and all as in bf16; the gradient's
// epilogue leaves dz's terms, and dW is fp32.  What it costs beside the products is
// a pass over W a call (4 bytes read and 8 written an element, 17 us for 8003 x
// 1021).  777 x 1021 x 8003 train: 604 us on fp32 matrix instructions, 424 so, and
// off by 3e-7 of the result; 4096 x 2048 x 8000 4450 and 2630.  A dz that overflows
// to an infinity leaves NaN where fp32 products could leave the infinity.
//
// Maxima and sums are fp32, the last logarithm 64-bit (once a row): lse is off
// by a few 2^-24 of itself.  exp(z - max) is taken as exp2 of the rounded
// difference, which is exact for the logits that count.
#pragma once

#include "gemm_bf16_k32.h"

namespace xent {

constexpr float kLog2e = 1.44269504088896341f;

// exp(z - m) with m the maximum of some z's; an infinite maximum (no logit,
// or an infinite one) counts from 0.
__device__ __forceinline__ float finite_or_0(float m) { return __builtin_isfinite(m) ? m : 0.0f; }
__device__ __forceinline__ float exp_diff(float z, float ref) { return __builtin_amdgcn_exp2f((z - ref) * kLog2e); }
__device__ __forceinline__ void join(float &m, float &s, float m2, float s2) {
  const float mm = fmaxf(m, m2), ref = finite_or_0(mm);
  // (a part without logits is (-inf, 0))
  s = s * exp_diff(m, ref) + s2 * exp_diff(m2, ref);
  m = mm;
}

// f(i, r, n) for the registers of a wave's fragments in one row, n its column.
template <class FR, int FN, class F>
__device__ __forceinline__ void each_column(uint32_t n_first, int lane, F f) {
#pragma unroll
  for (int i = 0; i < FN; ++i)
#pragma unroll
    for (int r = 0; r < FR::kRegs; ++r) f(i, r, n_first + (uint32_t)(i * FR::kSize) + FR::col(lane, r));
}
// Over the lanes that share a row.
template <class FR>
__device__ __forceinline__ float row_max(float v) {
  if constexpr (FR::kSize == 16) v = fmaxf(v, xor_f32(v, 16));
  return fmaxf(v, xor_f32(v, 32));
}
template <class FR>
__device__ __forceinline__ float row_sum(float v) {
  if constexpr (FR::kSize == 16) v += xor_f32(v, 16);
  return v + xor_f32(v, 32);
}

// Per row of the tile: maximum and sum of exp, and the target's logit.
struct EpiStats {
  static constexpr bool kStore = false;
  const BwppXentArgs &a;

  template <class FR, int BM, int BN, int WM, int WN, class V, int FN, int FM>
  __device__ __forceinline__ void run(V (&acc)[FN][FM], unsigned char *smem, uint32_t m0, uint32_t n0, uint32_t tn,
                                      uint32_t, int tid, int wm, int wn) const {
    constexpr int TM = BM / WM, TN = BN / WN;
    const int lane = tid & 63;
    float2 *pair = reinterpret_cast<float2 *>(smem);  // [BM][WN]
    const uint32_t nw = n0 + (uint32_t)(wn * TN);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const uint32_t ml = (uint32_t)(wm * TM + j * FR::kSize) + FR::row(lane), m = m0 + ml;
      const uint32_t t = m < a.g.M ? (uint32_t)a.target[m] : 0xffffffffu;
      if (n0 + BN > a.g.N)  // the last tile column: no logits past N
        each_column<FR, FN>(nw, lane, [&](int i, int r, uint32_t n) {
          acc[i][j][r] = n < a.g.N ? acc[i][j][r] * a.scale : -__builtin_inff();
        });
      else
        each_column<FR, FN>(nw, lane, [&](int i, int r, uint32_t) { acc[i][j][r] *= a.scale; });
      const uint32_t tl = t - a.n_base;  // the target's column of this product
      if (__any(t < a.vocab && tl - nw < (uint32_t)TN))
        each_column<FR, FN>(nw, lane, [&](int i, int r, uint32_t n) {
          if (t < a.vocab && n == tl && n < a.g.N) a.zt[m] = acc[i][j][r];
        });
      float mx = -__builtin_inff(), s = 0.0f;
      each_column<FR, FN>(nw, lane, [&](int i, int r, uint32_t) { mx = fmaxf(mx, acc[i][j][r]); });
      mx = row_max<FR>(mx);
      const float ref = finite_or_0(mx);
      each_column<FR, FN>(nw, lane, [&](int i, int r, uint32_t) { s += exp_diff(acc[i][j][r], ref); });
      s = row_sum<FR>(s);
      if (lane < FR::kSize) pair[ml * WN + wn] = make_float2(mx, s);
    }
    __syncthreads();
    if (tid < BM && m0 + (uint32_t)tid < a.g.M) {
      float2 p = pair[tid * WN];
#pragma unroll
      for (int w = 1; w < WN; ++w) {
        const float2 q = pair[tid * WN + w];
        join(p.x, p.y, q.x, q.y);
      }
      reinterpret_cast<float2 *>(a.part)[(size_t)(a.part_base + tn) * a.g.M + m0 + (uint32_t)tid] = p;
    }
  }
};

// dz scale in bf16.
struct EpiGrad {
  static constexpr bool kStore = false;
  const BwppXentArgs &a;

  template <class FR, int BM, int BN, int WM, int WN, class V, int FN, int FM>
  __device__ __forceinline__ void run(V (&acc)[FN][FM], unsigned char *smem, uint32_t m0, uint32_t n0, uint32_t, uint32_t,
                                      int tid, int wm, int wn) const {
    constexpr int TM = BM / WM, TN = BN / WN, NT = 64 * WM * WN, kCld = BN + 8;
    const int lane = tid & 63;
    uint16_t *cs = reinterpret_cast<uint16_t *>(smem);  // [BM][BN + 8]
    const uint32_t nw = n0 + (uint32_t)(wn * TN);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const uint32_t ml = (uint32_t)(wm * TM + j * FR::kSize) + FR::row(lane), m = m0 + ml;
      uint32_t t = 0xffffffffu;
      float lse = 0.0f, g = 0.0f;
      if (m < a.g.M) {
        t = (uint32_t)a.target[m];
        lse = a.lse[m];
        g = (a.dloss ? a.dloss[a.dloss_scalar ? 0u : m] : 1.0f) * a.scale;
      }
      const bool live = t < a.vocab;
      each_column<FR, FN>(nw, lane, [&](int i, int r, uint32_t) { acc[i][j][r] = exp_diff(acc[i][j][r] * a.scale, lse); });
      const uint32_t tl = t - a.n_base;
      if (__any(live && tl - nw < (uint32_t)TN))
        each_column<FR, FN>(nw, lane, [&](int i, int r, uint32_t n) {
          if (live && n == tl) {
            acc[i][j][r] -= 1.0f;
            const float v = g * acc[i][j][r], rest = v - bf16_bits_to_f32(f32_to_bf16_bits(v));
            if (a.rest) a.rest[m] = __builtin_isfinite(rest) ? rest : 0.0f;
          }
        });
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int r = 0; r < FR::kRegs; r += 4) {  // four columns
          float v[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = live ? g * acc[i][j][r + e] : 0.0f;
          uint2 o;
          o.x = pack_bf16x2(v[0], v[1]);
          o.y = pack_bf16x2(v[2], v[3]);
          *reinterpret_cast<uint2 *>(cs + ml * kCld + wn * TN + i * FR::kSize + FR::col(lane, r)) = o;
        }
    }
    __syncthreads();
    // Whole chunks: the last one's columns past N, which the row has room for,
    // get values of columns that were read again, and are never used.
#pragma unroll 4
    for (int it = 0; it < BM * (BN / 8) / NT; ++it) {
      const int q = tid + it * NT, row = q / (BN / 8), c = q % (BN / 8);
      const uint32_t m = m0 + (uint32_t)row, n = n0 + 8u * (uint32_t)c;
      if (m < a.rows_up && n < a.g.N)  // rows past M: zeros
        *reinterpret_cast<uint4 *>(a.dl + (size_t)m * a.ldl + n) = *reinterpret_cast<const uint4 *>(cs + row * kCld + c * 8);
    }
  }
};

// What dW's epilogues share.
struct DwRest {
  const BwppXentArgs &a;

  // dW += x^T (what rounding left of the targets' dz): of a row of dz the target's
  // p - 1 is by far the largest element, and its rounding nearly all of the error
  // that dz's brings (dx and dW off by 0.0025 of their norm with it, 0.0017, their
  // own rounding, without).  Of the tokens first .. end - 1 those whose target is in
  // the tile, in order, 32 at a time as one more K step: a one-hot operand of the
  // remainders (bf16: 2^-9 of 2^-9) and the rows of x, both laid out as the main
  // loop's K tiles.  256 T / V tokens a tile on average: no longer at 4096 x 2048 x
  // 32768 (465 us), 2 to 6 us at 120 x 1216 x 19298 (19 -> 24) and the like.  The steps
  // wait for their loads, so it shows where a tile has many: dW and the logits again,
  // targets uniform, half one id, all of one id or of 256: 8192 x 4096 x 2048 342, 469,
  // 615 us; 8192 x 4096 x 32000 3270, 3770, 4260; 4096 x 2048 x 32768 906, 949, 945.
  template <class FR, int BM, int BN, int WM, int WN, class V, int FN, int FM>
  __device__ __forceinline__ void add_rest(V (&acc)[FN][FM], unsigned char *smem, uint32_t m0, uint32_t n0, uint32_t first,
                                           uint32_t end, int tid, int wm, int wn) const {
    asm volatile("" : "+v"(tid));  // nothing below is computed ahead of the main loop, whose registers are full
    static_assert(FR::kSize == 32 || (BM == 256 && BN == 256), "as the main loops lay out their tiles");
    constexpr int TM = BM / WM, TN = BN / WN, NW = WM * WN, NT = 64 * NW;
    constexpr uint32_t kEach = 8, kWindow = NT * kEach;  // tokens a thread, and the block, looks at
    unsigned char *ta = smem, *tb = smem + BM * 64;       // K tiles of 32
    uint32_t *list = reinterpret_cast<uint32_t *>(smem + (BM + BN) * 64);  // [kWindow] tokens of the window, and their columns
    uint32_t *totals = list + kWindow;                                     // [NW]
    const int lane = tid & 63, wave = tid >> 6;
    const bool xa = a.x_is_a;
    const uint32_t v0 = a.n_base + (xa ? n0 : m0), d0 = xa ? m0 : n0;
    const uint32_t lim = (xa ? a.g.M : a.g.N) - d0;
    const uint16_t *x = static_cast<const uint16_t *>(xa ? a.g.a : a.g.b);
    const uint64_t ldx = xa ? a.g.lda : a.g.ldb;
    unsigned char *xs = xa ? ta : tb, *hot = xa ? tb : ta;
    const uint32_t wx = xa ? BM : BN, wh = xa ? BN : BM;
    // Byte offset of chunk c of k-row k in a tile of that width.
    auto pos = [&](bool in_a, uint32_t k, uint32_t c) {
      if constexpr (FR::kSize == 16) return k * 512u + 16u * (c ^ mnc16_swz(k));
      else return in_a ? mnc_off<BM>(k, c) : mnc_off<BN>(k, c);
    };
    for (uint32_t w0 = first; w0 < end; w0 += kWindow) {
      uint32_t mine = 0, column[kEach];  // bit e: token w0 + kEach tid + e
#pragma unroll
      for (uint32_t e = 0; e < kEach; ++e) {
        const uint32_t m = w0 + kEach * (uint32_t)tid + e;
        const uint32_t t = m < end ? (uint32_t)a.target[m] : 0xffffffffu;
        column[e] = t - v0;
        if (t < a.vocab && column[e] < wh) mine |= 1u << e;
      }
      const uint32_t n = (uint32_t)__popc(mine);
      uint32_t before = n;  // of the wave's lanes up to this one
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const uint32_t o = (uint32_t)__shfl_up((int)before, d);
        if (lane >= d) before += o;
      }
      if (lane == 63) totals[wave] = before;
      __syncthreads();
      uint32_t at = before - n, count = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const uint32_t c = totals[w];
        if (w < wave) at += c;
        count += c;
      }
#pragma unroll
      for (uint32_t e = 0; e < kEach; ++e)
        if (mine >> e & 1u) list[at++] = column[e] << 16 | (kEach * (uint32_t)tid + e);
      __syncthreads();
      for (uint32_t b = 0; b < count; b += 32) {
        const bool one = tid < 32 && b + (uint32_t)tid < count;
        const uint32_t entry = one ? list[b + (uint32_t)tid] : 0u;
        const float rest = one ? a.rest[w0 + (entry & 0xffffu)] : 0.0f;
#pragma unroll 1
        for (uint32_t q = (uint32_t)tid; q < 4u * wh; q += NT) *reinterpret_cast<u32x4_t *>(hot + 16u * q) = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll 1
        for (uint32_t q = (uint32_t)tid; q < 4u * wx; q += NT) {
          const uint32_t k = q / (wx / 8u), c = q % (wx / 8u);
          u32x4_t v = {0u, 0u, 0u, 0u};
          if (b + k < count)
            v = *reinterpret_cast<const u32x4_t *>(x + (uint64_t)(w0 + (list[b + k] & 0xffffu)) * ldx + d0 +
                                                   min(8u * c, lim - 8u));
          *reinterpret_cast<u32x4_t *>(xs + pos(xa, k, c)) = v;
        }
        __syncthreads();
        if (one) {
          const uint32_t v = entry >> 16;
          *reinterpret_cast<uint16_t *>(hot + pos(!xa, (uint32_t)tid, v >> 3) + 2u * (v & 7u)) = f32_to_bf16_bits(rest);
        }
        __syncthreads();
        if constexpr (FR::kSize == 16) {
          bf16x8_t fb[FN];
#pragma unroll
          for (int i = 0; i < FN; ++i) fb[i] = read16<true, BN>(tb, (uint32_t)(wn * TN + i * 16), lane);
#pragma unroll
          for (int j = 0; j < FM; ++j) {
            const bf16x8_t fa = read16<true, BM>(ta, (uint32_t)(wm * TM + j * 16), lane);
#pragma unroll
            for (int i = 0; i < FN; ++i) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fb[i], fa, acc[i][j], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);  // one operand in registers at a time
          }
        } else {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int j = 0; j < FM; ++j) {
              const bf16x8_t fa = read_operand<true, BM>(ta, (uint32_t)(wm * TM + j * 32), ks, lane);
#pragma unroll
              for (int i = 0; i < FN; ++i)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    read_operand<true, BN>(tb, (uint32_t)(wn * TN + i * 32), ks, lane), fa, acc[i][j], 0, 0, 0);
            }
        }
        __syncthreads();
      }
    }
    __syncthreads();
  }
};

// bf16 rows (dW), at any address and row stride: on 256-wide tiles, or where those
// are few on the smaller ones.
struct EpiRows : DwRest {
  static constexpr bool kStore = false;

  template <class FR, int BM, int BN, int WM, int WN, class V, int FN, int FM>
  __device__ __forceinline__ void run(V (&acc)[FN][FM], unsigned char *smem, uint32_t m0, uint32_t n0, uint32_t, uint32_t,
                                      int tid, int wm, int wn) const {
    constexpr int TM = BM / WM, TN = BN / WN, NT = 64 * WM * WN, kCld = BN + 8;
    const int lane = tid & 63;
    uint16_t *cs = reinterpret_cast<uint16_t *>(smem);  // [BM][BN + 8]
    add_rest<FR, BM, BN, WM, WN>(acc, smem, m0, n0, 0, a.rows, tid, wm, wn);
#pragma unroll
    for (int j = 0; j < FM; ++j)
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int r = 0; r < FR::kRegs; r += 4) {
          uint2 o;
          o.x = pack_bf16x2(acc[i][j][r], acc[i][j][r + 1]);
          o.y = pack_bf16x2(acc[i][j][r + 2], acc[i][j][r + 3]);
          *reinterpret_cast<uint2 *>(cs + ((uint32_t)(wm * TM + j * FR::kSize) + FR::row(lane)) * kCld + wn * TN +
                                     i * FR::kSize + FR::col(lane, r)) = o;
        }
    __syncthreads();
    uint16_t *C = static_cast<uint16_t *>(a.g.c);
#pragma unroll 4
    for (int it = 0; it < BM * (BN / 8) / NT; ++it) {
      const int q = tid + it * NT, row = q / (BN / 8), c = q % (BN / 8);
      const uint32_t m = m0 + (uint32_t)row, n = n0 + 8u * (uint32_t)c;
      if (m >= a.rows_out || n >= a.cols_out) continue;
      const uint16_t *h = cs + row * kCld + c * 8;
      uint16_t *dst = C + (size_t)m * a.g.ldc + n;
      if (n + 8 <= a.cols_out) {
        *reinterpret_cast<u32x4a2_t *>(dst) = *reinterpret_cast<const u32x4_t *>(h);
      } else {
        for (uint32_t e = 0; e < 8 && n + e < a.cols_out; ++e) dst[e] = h[e];
      }
    }
  }
};

// dW where those are few too: K (tokens) in ranges, each an fp32 plane [rows_out]
// [cols_out] with the remainders of its own tokens, so that a batch with one target
// brings a tile as many steps as the main loop has, not a block T / 32.  Beside
// dispatch_matmul without remainders (dW off by 0.0021 to 0.0028 of its norm, 0.0017
// so), us a pass of loss and gradients: 300 x 256 x 1000 29.5 -> 31, 1505 x 1024 x
// 3144 104 -> 106, 8000 x 512 x 1000 99 -> 104, 20000 x 64 x 15400 742 -> 770, 635 x
// 2560 x 2240 104 -> 103.  (256-wide tiles in ranges: 48, 122, 112, 809, 122.)
struct EpiRowSums : DwRest {
  static constexpr bool kStore = false;

  template <class FR, int BM, int BN, int WM, int WN, class V, int FN, int FM>
  __device__ __forceinline__ void run(V (&acc)[FN][FM], unsigned char *smem, uint32_t m0, uint32_t n0, uint32_t, uint32_t split,
                                      int tid, int wm, int wn) const {
    constexpr int TM = BM / WM, TN = BN / WN;
    const int lane = tid & 63;
    const uint32_t first = split * a.g.kchunk;
    add_rest<FR, BM, BN, WM, WN>(acc, smem, m0, n0, first, min(a.rows, first + a.g.kchunk), tid, wm, wn);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const uint32_t m = m0 + (uint32_t)(wm * TM + j * FR::kSize) + FR::row(lane);
      if (m >= a.rows_out) continue;
      float *row = a.raw + ((size_t)split * a.rows_out + m) * a.cols_out;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int r = 0; r < FR::kRegs; r += 4) {
          const uint32_t n = n0 + (uint32_t)(wn * TN + i * FR::kSize) + FR::col(lane, r);
          if (n + 4 <= a.cols_out) {
            store4(row + n, make_float4(acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < a.cols_out) row[n + e] = acc[i][j][r + e];
          }
        }
    }
  }
};

// dz scale in three bf16 planes (v1 + v2 + v3 = dz to 24 bits).
struct EpiGradTerms {
  static constexpr bool kStore = false;
  const BwppXentArgs &a;

  template <class FR, int BM, int BN, int WM, int WN, class V, int FN, int FM>
  __device__ __forceinline__ void run(V (&acc)[FN][FM], unsigned char *smem, uint32_t m0, uint32_t n0, uint32_t, uint32_t,
                                      int tid, int wm, int wn) const {
    constexpr int TM = BM / WM, TN = BN / WN, NT = 64 * WM * WN, kCld = BN + 8;
    const int lane = tid & 63;
    uint16_t *cs = reinterpret_cast<uint16_t *>(smem);  // [BM][BN + 8]
    const uint32_t nw = n0 + (uint32_t)(wn * TN);
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const uint32_t m = m0 + (uint32_t)(wm * TM + j * FR::kSize) + FR::row(lane);
      uint32_t t = 0xffffffffu;
      float lse = 0.0f, g = 0.0f;
      if (m < a.g.M) {
        t = (uint32_t)a.target[m];
        lse = a.lse[m];
        g = (a.dloss ? a.dloss[a.dloss_scalar ? 0u : m] : 1.0f) * a.scale;
      }
      const bool live = t < a.vocab;
      const uint32_t tl = t - a.n_base;
      each_column<FR, FN>(nw, lane, [&](int i, int r, uint32_t n) {
        const float p = exp_diff(acc[i][j][r] * a.scale, lse);
        acc[i][j][r] = live && n < a.g.N ? g * (n == tl ? p - 1.0f : p) : 0.0f;
      });
    }
#pragma unroll 1
    for (int plane = 0; plane < 3; ++plane) {
      if (plane > 0) __syncthreads();  // the plane before has left LDS
#pragma unroll
      for (int j = 0; j < FM; ++j)
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
          for (int r = 0; r < FR::kRegs; r += 4) {
            uint2 o;
            o.x = pack_bf16x2(acc[i][j][r], acc[i][j][r + 1]);
            o.y = pack_bf16x2(acc[i][j][r + 2], acc[i][j][r + 3]);
            *reinterpret_cast<uint2 *>(cs + ((uint32_t)(wm * TM + j * FR::kSize) + FR::row(lane)) * kCld + wn * TN +
                                       i * FR::kSize + FR::col(lane, r)) = o;
            acc[i][j][r] -= __uint_as_float(o.x << 16);  // exact
            acc[i][j][r + 1] -= __uint_as_float(o.x & 0xffff0000u);
            acc[i][j][r + 2] -= __uint_as_float(o.y << 16);
            acc[i][j][r + 3] -= __uint_as_float(o.y & 0xffff0000u);
          }
      __syncthreads();
      uint16_t *dl = a.dl + plane * a.dl_stride;
#pragma unroll 4
      for (int it = 0; it < BM * (BN / 8) / NT; ++it) {
        const int q = tid + it * NT, row = q / (BN / 8), c = q % (BN / 8);
        const uint32_t m = m0 + (uint32_t)row, n = n0 + 8u * (uint32_t)c;
        if (m < a.rows_up && n < a.cols_up)
          *reinterpret_cast<uint4 *>(dl + (size_t)m * a.ldl + n) = *reinterpret_cast<const uint4 *>(cs + row * kCld + c * 8);
      }
    }
  }
};

// fp32 rows (dW), at any address and row stride.
struct EpiRowsF32 {
  static constexpr bool kStore = false;
  const BwppXentArgs &a;

  template <class FR, int BM, int BN, int WM, int WN, class V, int FN, int FM>
  __device__ __forceinline__ void run(V (&acc)[FN][FM], unsigned char *, uint32_t m0, uint32_t n0, uint32_t, uint32_t,
                                      int tid, int wm, int wn) const {
    constexpr int TM = BM / WM, TN = BN / WN;
    const int lane = tid & 63;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const uint32_t m = m0 + (uint32_t)(wm * TM + j * FR::kSize) + FR::row(lane);
      if (m >= a.rows_out) continue;
      float *row = static_cast<float *>(a.g.c) + (size_t)m * a.g.ldc;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int r = 0; r < FR::kRegs; r += 4) {
          const uint32_t n = n0 + (uint32_t)(wn * TN + i * FR::kSize) + FR::col(lane, r);
          if (n + 4 <= a.cols_out) {
            store4(row + n, make_float4(acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < a.cols_out) row[n + e] = acc[i][j][r + e];
          }
        }
    }
  }
};

// fp32 sums, one plane per K split, added to what is there where asked.
struct EpiSums {
  static constexpr bool kStore = false;
  const BwppXentArgs &a;

  template <class FR, int BM, int BN, int WM, int WN, class V, int FN, int FM>
  __device__ __forceinline__ void run(V (&acc)[FN][FM], unsigned char *, uint32_t m0, uint32_t n0, uint32_t, uint32_t split,
                                      int tid, int wm, int wn) const {
    constexpr int TM = BM / WM, TN = BN / WN;
    const int lane = tid & 63;
#pragma unroll
    for (int j = 0; j < FM; ++j) {
      const uint32_t m = m0 + (uint32_t)(wm * TM + j * FR::kSize) + FR::row(lane);
      float *row = a.raw + ((size_t)split * a.g.M + m) * a.g.N;
      if (m >= a.g.M) continue;
#pragma unroll
      for (int i = 0; i < FN; ++i)
#pragma unroll
        for (int r = 0; r < FR::kRegs; r += 4) {
          const uint32_t n = n0 + (uint32_t)(wn * TN + i * FR::kSize) + FR::col(lane, r);
          float4 v = make_float4(acc[i][j][r], acc[i][j][r + 1], acc[i][j][r + 2], acc[i][j][r + 3]);
          if (n + 4 <= a.g.N) {
            if (a.accumulate) {
              const float4 o = load4(row + n);
              v = make_float4(v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w);
            }
            store4(row + n, v);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (n + e < a.g.N) row[n + e] = acc[i][j][r + e] + (a.accumulate ? row[n + e] : 0.0f);
          }
        }
    }
  }
};

// ------------------------------------------------------------ row kernels

__device__ __forceinline__ bool live(const BwppXentRowArgs &a, uint32_t row) {
  return (uint32_t)a.target[row] < a.vocab;
}

template <class T>
__device__ __forceinline__ T to(float v);
template <>
__device__ __forceinline__ float to<float>(float v) { return v; }
template <>
__device__ __forceinline__ uint16_t to<uint16_t>(float v) { return f32_to_bf16_bits(v); }

// y = x, rows that are left out 0 (their values, infinities and NaN among
// them, stay out of dW's sums), and so rows past the last (rows_up) and columns
// (ldy).
template <class T>
__device__ __forceinline__ void copy_rows(const BwppXentRowArgs &a) {
  for (uint32_t row = blockIdx.x; row < a.rows_up; row += gridDim.x) {
    const bool on = row < a.rows && live(a, row);
    const T *x = static_cast<const T *>(a.x) + row * a.ldx;
    T *y = static_cast<T *>(a.y) + row * a.ldy;
    for (uint32_t c = threadIdx.x; c < a.ldy; c += 256) y[c] = on && c < a.cols ? x[c] : T(0);
  }
}
// Rows that are left out: 0.
template <class T>
__device__ __forceinline__ void zero_rows(const BwppXentRowArgs &a) {
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    if (live(a, row)) continue;
    T *y = static_cast<T *>(a.y) + row * a.ldy;
    for (uint32_t c = threadIdx.x; c < a.cols; c += 256) y[c] = T(0);
  }
}

// Joins a row's pairs: `lanes` (a power of two, 64 at most) rows a block, its 16
// waves each over a part of the pairs, a wave's lanes beyond the rows over parts of
// that (4 rows with 256 pairs: one load a lane); then loss and lse, and with a
// single block the sums over the rows too.
extern "C" __global__ __launch_bounds__(1024) void bwpp_xent_join(const BwppXentRowArgs a) {
  __shared__ float2 p[16][64];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t row = blockIdx.x * a.lanes + (lane & (a.lanes - 1)), subs = 64u / a.lanes;
  float m = -__builtin_inff(), s = 0.0f;
  if (row < a.rows) {
    const float2 *part = reinterpret_cast<const float2 *>(a.part) + row;
#pragma unroll 4
    for (uint32_t i = wave * subs + lane / a.lanes; i < a.nparts; i += 16 * subs) {
      const float2 q = part[(size_t)i * a.rows];
      join(m, s, q.x, q.y);
    }
  }
  for (uint32_t d = a.lanes; d < 64; d *= 2) join(m, s, xor_f32(m, (int)d), xor_f32(s, (int)d));
  p[wave][lane] = make_float2(m, s);
  __syncthreads();
  if (wave != 0) return;
  double total = 0.0;
  uint32_t n = 0;
  if (row < a.rows && lane < a.lanes) {
#pragma unroll
    for (int w = 1; w < 16; ++w) join(m, s, p[w][lane].x, p[w][lane].y);
    const double lse = (double)finite_or_0(m) + log((double)s);
    const bool on = live(a, row);
    const float loss = on ? (float)(lse - (double)a.zt[row]) : 0.0f;
    if (a.lse) a.lse[row] = (float)lse;
    if (a.loss) a.loss[row] = loss;
    total = loss;
    n = on ? 1u : 0u;
  }
  if (a.sums && gridDim.x == 1) {
    for (int d = 1; d < 64; d *= 2) {
      total += __shfl_xor(total, d, 64);
      n += (uint32_t)__shfl_xor((int)n, d, 64);
    }
    if (lane == 0) {
      a.sums[0] = (float)total;
      a.sums[1] = (float)n;
    }
  }
}

// Sum of the losses (64-bit) and number of rows that count, one block.
extern "C" __global__ __launch_bounds__(1024) void bwpp_xent_sums(const BwppXentRowArgs a) {
  __shared__ double ts[16];
  __shared__ uint32_t ns[16];
  double total = 0.0;
  uint32_t n = 0;
  for (uint64_t row = threadIdx.x; row < a.rows; row += 1024) {
    const bool on = live(a, (uint32_t)row);
    total += on ? (double)a.loss[row] : 0.0;
    n += on ? 1u : 0u;
  }
  for (int d = 1; d < 64; d *= 2) {
    total += __shfl_xor(total, d, 64);
    n += (uint32_t)__shfl_xor((int)n, d, 64);
  }
  if ((threadIdx.x & 63) == 0) {
    ts[threadIdx.x >> 6] = total;
    ns[threadIdx.x >> 6] = n;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 16; ++w) {
      total += ts[w];
      n += ns[w];
    }
    a.sums[0] = (float)total;
    a.sums[1] = (float)n;
  }
}

// fp32 logits of a piece (src, unscaled; 16-byte rows with room up to 4 columns):
// one pair per row into part[rows].  A thread keeps up to 8 chunks of four logits
// at a time: their maximum first, then their sum (one exp a logit).
extern "C" __global__ __launch_bounds__(256) void bwpp_xent_stats_f32(const BwppXentRowArgs a) {
  __shared__ float ms[4], ss[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t chunks = (a.cols + 3) / 4;
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float *z = a.src + (uint64_t)row * a.lds;
    float m = -__builtin_inff(), s = 0.0f;
    for (uint32_t c0 = threadIdx.x; c0 < chunks; c0 += 256 * 8) {
      float4 v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t c = min(c0 + 256 * k, chunks - 1);
        v[k] = *reinterpret_cast<const float4 *>(z + 4 * (uint64_t)c);
      }
      float mc = -__builtin_inff();
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const uint32_t c = c0 + 256 * k, n = 4 * c;
        float *e = &v[k].x;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[i] = c < chunks && n + i < a.cols ? e[i] * a.scale : -__builtin_inff();
          mc = fmaxf(mc, e[i]);
        }
      }
      const float ref = finite_or_0(mc);
      float sc = 0.0f;
#pragma unroll
      for (int k = 0; k < 8; ++k) sc += (exp_diff(v[k].x, ref) + exp_diff(v[k].y, ref)) + (exp_diff(v[k].z, ref) + exp_diff(v[k].w, ref));
      join(m, s, mc, sc);
    }
    for (int d = 1; d < 64; d *= 2) join(m, s, xor_f32(m, d), xor_f32(s, d));
    if (lane == 0) {
      ms[wave] = m;
      ss[wave] = s;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < 4; ++w) join(m, s, ms[w], ss[w]);
      reinterpret_cast<float2 *>(a.part)[row] = make_float2(m, s);
      const uint32_t t = (uint32_t)a.target[row], tl = t - a.n_base;
      if (t < a.vocab && tl < a.cols) a.zt[row] = z[tl] * a.scale;
    }
    __syncthreads();
  }
}

// fp32 logits of a piece (y, unscaled; rows as above) -> dz scale, in place.
extern "C" __global__ __launch_bounds__(256) void bwpp_xent_grad_f32(const BwppXentRowArgs a) {
  const uint32_t chunks = (a.cols + 3) / 4;
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    float *z = static_cast<float *>(a.y) + (uint64_t)row * a.ldy;
    const uint32_t t = (uint32_t)a.target[row], tl = t - a.n_base;
    const bool on = t < a.vocab;
    const float lse = a.lse_in[row], g = (a.dloss ? a.dloss[a.dloss_scalar ? 0u : row] : 1.0f) * a.scale;
#pragma unroll 4
    for (uint32_t c = threadIdx.x; c < chunks; c += 256) {
      float4 v = *reinterpret_cast<const float4 *>(z + 4 * (uint64_t)c);
      float *e = &v.x;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float p = exp_diff(e[i] * a.scale, lse);
        e[i] = on ? g * (4 * c + i == tl ? p - 1.0f : p) : 0.0f;
      }
      *reinterpret_cast<float4 *>(z + 4 * (uint64_t)c) = v;
    }
  }
}

// Planes of fp32 sums -> rows of T, rows that are left out 0 (no targets: every row
// counts); bf16 dx: with W's row of the target times what rounding left of its dz
// (DwRest::add_rest).
template <class T>
__device__ __forceinline__ void sum_planes(const BwppXentRowArgs &a) {
  const uint64_t plane = (uint64_t)a.rows * a.cols;
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const bool on = !a.target || live(a, row);
    T *y = static_cast<T *>(a.y) + row * a.ldy;
    const float *src = a.src + (uint64_t)row * a.cols;
    const bool add = sizeof(T) == 2 && on && a.rest;
    const float rest = add ? a.rest[row] : 0.0f;
    const uint16_t *w = static_cast<const uint16_t *>(a.w) + (add ? (uint32_t)a.target[row] * a.ldw : 0u);
    for (uint32_t c = (blockIdx.y * 256u + threadIdx.x) * 4u; c < a.cols; c += gridDim.y * 1024u) {
      const uint32_t n = min(4u, a.cols - c);
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      if (n == 4) {
#pragma unroll 4
        for (uint32_t i = 0; i < a.nparts; ++i) {
          const float4 o = load4(src + i * plane + c);
          v[0] += o.x, v[1] += o.y, v[2] += o.z, v[3] += o.w;
        }
      } else {
        for (uint32_t i = 0; i < a.nparts; ++i)
#pragma unroll
          for (uint32_t e = 0; e < 3; ++e) v[e] += e < n ? src[i * plane + c + e] : 0.0f;
      }
      if (n == 4) {
        typedef uint16_t H4 __attribute__((ext_vector_type(4), aligned(2)));
        if constexpr (sizeof(T) == 2) {
          if (add) {
            const H4 h = *reinterpret_cast<const H4 *>(w + c);
#pragma unroll
            for (uint32_t e = 0; e < 4; ++e) v[e] += rest * bf16_bits_to_f32(h[e]);
          }
          const H4 o = {to<T>(on ? v[0] : 0.0f), to<T>(on ? v[1] : 0.0f), to<T>(on ? v[2] : 0.0f), to<T>(on ? v[3] : 0.0f)};
          *reinterpret_cast<H4 *>(y + c) = o;
        } else {
          store4(y + c, on ? make_float4(v[0], v[1], v[2], v[3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        }
      } else {
        for (uint32_t e = 0; e < n; ++e) {
          const float more = add ? rest * bf16_bits_to_f32(w[c + e]) : 0.0f;
          y[c + e] = to<T>(on ? (e == 0 ? v[0] : e == 1 ? v[1] : v[2]) + more : 0.0f);
        }
      }
    }
  }
}
extern "C" __global__ __launch_bounds__(256) void bwpp_xent_round_bf16(const BwppXentRowArgs a) { sum_planes<uint16_t>(a); }
extern "C" __global__ __launch_bounds__(256) void bwpp_xent_round_f32(const BwppXentRowArgs a) { sum_planes<float>(a); }
// W [dim][vocab]: its columns are gathered, every element from a line of its own.
// An XCD takes 32 columns of dx at a time for all tokens: those 32 rows of W stay in
// its L2 (4096 x 2048 from two planes: 90 us, 83 with 16 columns, 20 without the
// gather).  blockIdx: XCD, then `lanes` tokens (a multiple of 8), then the
// XCD's next columns.
extern "C" __global__ __launch_bounds__(256) void bwpp_xent_round_bf16_dv(const BwppXentRowArgs a) {
  const uint64_t plane = (uint64_t)a.rows * a.cols;
  const uint32_t groups = (a.rows + a.lanes - 1u) / a.lanes, q = blockIdx.x >> 3;
  const uint32_t chunk = (blockIdx.x & 7u) + 8u * (q / groups), c = chunk * 32u + (threadIdx.x & 31u);
  if (c >= a.cols) return;
  const uint16_t *w = static_cast<const uint16_t *>(a.w) + c * a.ldw;
#pragma unroll 8
  for (uint32_t i = 0; i < a.lanes; i += 8) {
    const uint32_t row = q % groups * a.lanes + i + threadIdx.x / 32u;
    if (row >= a.rows) continue;
    const uint32_t t = (uint32_t)a.target[row];
    float v = 0.0f;
    if (t < a.vocab) {
      const float *src = a.src + (uint64_t)row * a.cols + c;
      v = a.rest[row] * bf16_bits_to_f32(w[t]);
#pragma unroll 8
      for (uint32_t p = 0; p < a.nparts; ++p) v += src[p * plane];
    }
    static_cast<uint16_t *>(a.y)[row * a.ldy + c] = to<uint16_t>(v);
  }
}

// fp32 rows (x, any strides) -> four bf16 planes [rows_up][ldy]: v1, v1 where it
// is finite, v2, v3 (gemm_bf16_k32.h); zeros past the rows and columns and, with
// targets, in rows that are left out.
extern "C" __global__ __launch_bounds__(256) void bwpp_xent_terms(const BwppXentRowArgs a) {
  const uint32_t step = 256u / a.lanes, c0 = (threadIdx.x & (a.lanes - 1u)) * 8u;  // `lanes` threads a row
  for (uint32_t row = blockIdx.x * step + threadIdx.x / a.lanes; row < a.rows_up; row += gridDim.x * step) {
    const bool on = row < a.rows && (!a.target || live(a, row));
    const float *x = static_cast<const float *>(a.x) + row * a.ldx;
    uint16_t *y = static_cast<uint16_t *>(a.y) + row * a.ldy;
    for (uint32_t c = c0; c < a.ldy; c += a.lanes * 8u) {
      float v[8];
      if (on && c + 8 <= a.cols) {
        const float4 p = load4(x + c), q = load4(x + c + 4);
        v[0] = p.x, v[1] = p.y, v[2] = p.z, v[3] = p.w, v[4] = q.x, v[5] = q.y, v[6] = q.z, v[7] = q.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = on && c + e < a.cols ? x[c + e] : 0.0f;
      }
      uint16_t t1[8], tf[8], t2[8], t3[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const bool fin = __builtin_isfinite(v[e]);
        uint16_t h = f32_to_bf16_bits(v[e]);
        if (fin && !__builtin_isfinite(bf16_bits_to_f32(h))) h = (uint16_t)(__float_as_uint(v[e]) >> 16);  // no overflow
        const float r = fin ? v[e] - bf16_bits_to_f32(h) : 0.0f;
        t1[e] = h;
        tf[e] = fin ? h : 0;
        t2[e] = f32_to_bf16_bits(r);
        t3[e] = f32_to_bf16_bits(r - bf16_bits_to_f32(t2[e]));
      }
      auto store = [&](int plane, const uint16_t (&t)[8]) {
        uint4 o;
        o.x = t[0] | (uint32_t)t[1] << 16, o.y = t[2] | (uint32_t)t[3] << 16;
        o.z = t[4] | (uint32_t)t[5] << 16, o.w = t[6] | (uint32_t)t[7] << 16;
        *reinterpret_cast<uint4 *>(y + plane * a.plane + c) = o;
      };
      store(0, t1);
      store(1, tf);
      store(2, t2);
      store(3, t3);
    }
  }
}

// Zeros (dW of no rows): 2-byte units, rows of up to 2^32 of them (64-bit columns: a
// 32-bit one would pass the end of such a row and start again).
extern "C" __global__ __launch_bounds__(256) void bwpp_xent_clear(const BwppXentRowArgs a) {
  for (uint32_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    uint16_t *y = static_cast<uint16_t *>(a.y) + row * a.ldy;
    for (uint64_t c = blockIdx.y * 256u + threadIdx.x; c < a.cols; c += gridDim.y * 256u) y[c] = 0;
  }
}

#define BWPP_XENT_ROWS(TN, T)                                                                                       \
  extern "C" __global__ __launch_bounds__(256) void bwpp_xent_copy_##TN(const BwppXentRowArgs a) { copy_rows<T>(a); } \
  extern "C" __global__ __launch_bounds__(256) void bwpp_xent_zero_##TN(const BwppXentRowArgs a) { zero_rows<T>(a); }
BWPP_XENT_ROWS(bf16, uint16_t)
BWPP_XENT_ROWS(f32, float)

// bwpp_xent_<stats|grad|sums>_<tile>_t0<TB>: p = 256 x 256 (K in steps of
// 32), sp and sh = 256 x 256 and 128 x 256 for fp32 in terms; any sizes: r32 = 32 x 64, r64 = 64 x 64,
// r128 = 128 x 128, _u with operands through registers.  bwpp_xent_rows_<tile>_t10 and
// rowsums: dW.
#define BWPP_XENT_K32(NAME, EPI, TA, TB, BM, SPLIT)                                                       \
  extern "C" __global__ __attribute__((amdgpu_flat_work_group_size(512, 512), amdgpu_waves_per_eu(2, 2))) \
  void bwpp_xent_##NAME(const BwppXentArgs a) {                                                           \
    gemm_bf16_k32<TA != 0, TB != 0, BM, TB != 0, SPLIT, EPI>(a.g, EPI{a}, a.terms);                       \
  }
#define BWPP_XENT_RING(KIND, EPI, TB, NAME, BM, BN, WM, WN, KPS, STAGES, WPE, KPSU, WPEU)                       \
  extern "C" __global__ __launch_bounds__(64 * WM * WN, WPE) void bwpp_xent_##KIND##_##NAME##_t0##TB(           \
      const BwppXentArgs a) {                                                                                   \
    gemm_bf16_ring<false, TB != 0, BM, BN, WM, WN, KPS, STAGES, false, EPI>(a.g, EPI{a});                       \
  }                                                                                                             \
  extern "C" __global__ __launch_bounds__(64 * WM * WN, WPEU) void bwpp_xent_##KIND##_##NAME##_t0##TB##_u(      \
      const BwppXentArgs a) {                                                                                   \
    gemm_bf16_ring<false, TB != 0, BM, BN, WM, WN, KPSU, 2, true, EPI>(a.g, EPI{a});                            \
  }
// A transposed (dW: both operands are rows of tokens in the workspace, whole chunks).
#define BWPP_XENT_RING_T(KIND, EPI, NAME, BM, BN, WM, WN, KPS, STAGES, WPE)                                     \
  extern "C" __global__ __launch_bounds__(64 * WM * WN, WPE) void bwpp_xent_##KIND##_##NAME##_t10(              \
      const BwppXentArgs a) {                                                                                   \
    gemm_bf16_ring<true, false, BM, BN, WM, WN, KPS, STAGES, false, EPI>(a.g, EPI{a});                          \
  }
#define BWPP_XENT_TB(TB)                                                    \
  BWPP_XENT_K32(stats_p_t0##TB, EpiStats, 0, TB, 256, false)                \
  BWPP_XENT_K32(grad_p_t0##TB, EpiGrad, 0, TB, 256, false)                  \
  BWPP_XENT_K32(sums_p_t0##TB, EpiSums, 0, TB, 256, false)                  \
  BWPP_XENT_K32(stats_sp_t0##TB, EpiStats, 0, TB, 256, true)                \
  BWPP_XENT_K32(grad_sp_t0##TB, EpiGradTerms, 0, TB, 256, true)             \
  BWPP_XENT_K32(sums_sp_t0##TB, EpiSums, 0, TB, 256, true)                  \
  BWPP_XENT_K32(stats_sh_t0##TB, EpiStats, 0, TB, 128, true)                \
  BWPP_XENT_K32(grad_sh_t0##TB, EpiGradTerms, 0, TB, 128, true)             \
  BWPP_XENT_K32(sums_sh_t0##TB, EpiSums, 0, TB, 128, true)                  \
  BWPP_XENT_RING(stats, EpiStats, TB, r32, 32, 64, 1, 2, 4, 4, 1, 4, 1)     \
  BWPP_XENT_RING(grad, EpiGrad, TB, r32, 32, 64, 1, 2, 4, 4, 1, 4, 1)       \
  BWPP_XENT_RING(sums, EpiSums, TB, r32, 32, 64, 1, 2, 4, 4, 1, 4, 1)       \
  BWPP_XENT_RING(stats, EpiStats, TB, r64, 64, 64, 2, 2, 2, 4, 2, 4, 2)     \
  BWPP_XENT_RING(grad, EpiGrad, TB, r64, 64, 64, 2, 2, 2, 4, 2, 4, 2)       \
  BWPP_XENT_RING(sums, EpiSums, TB, r64, 64, 64, 2, 2, 2, 4, 2, 4, 2)       \
  BWPP_XENT_RING(stats, EpiStats, TB, r128, 128, 128, 2, 2, 1, 3, 2, 2, 2)  \
  BWPP_XENT_RING(grad, EpiGrad, TB, r128, 128, 128, 2, 2, 1, 3, 2, 2, 2)    \
  BWPP_XENT_RING(sums, EpiSums, TB, r128, 128, 128, 2, 2, 1, 3, 2, 2, 2)
BWPP_XENT_TB(0)
BWPP_XENT_TB(1)
BWPP_XENT_K32(rows_p_t10, EpiRows, 1, 0, 256, false)
BWPP_XENT_RING_T(rows, EpiRows, r32, 32, 64, 1, 2, 4, 4, 1)
BWPP_XENT_RING_T(rows, EpiRows, r64, 64, 64, 2, 2, 2, 4, 2)
BWPP_XENT_RING_T(rows, EpiRows, r128, 128, 128, 2, 2, 1, 3, 2)
BWPP_XENT_RING_T(rowsums, EpiRowSums, r32, 32, 64, 1, 2, 4, 4, 1)
BWPP_XENT_RING_T(rowsums, EpiRowSums, r64, 64, 64, 2, 2, 2, 4, 2)
BWPP_XENT_RING_T(rowsums, EpiRowSums, r128, 128, 128, 2, 2, 1, 3, 2)
BWPP_XENT_K32(rows_sp_t10, EpiRowsF32, 1, 0, 256, true)
BWPP_XENT_K32(rows_sh_t10, EpiRowsF32, 1, 0, 128, true)
BWPP_XENT_K32(sums_sp_t10, EpiSums, 1, 0, 256, true)
BWPP_XENT_K32(sums_sh_t10, EpiSums, 1, 0, 128, true)

}  // namespace xent
