// Rotary positions for gfx950: q and k rows turned pair by pair by an angle
// that grows with the token's position.
//
//   f_i = base^(-2 i / n)          n = rot_dim, i = 0 .. n/2 - 1, scaled for
//                                  long contexts (all by 1 / s, or by parts)
//   a   = p f_i
//   (y_a, y_b) = m (x_a cos a - x_b sin a, x_b cos a + x_a sin a)
//
// over the pairs (a, b) = (i, i + n/2) ("half") or (2i, 2i + 1)
// ("interleaved"); columns from n on are copied.  The gradient is the
// transpose: the same turn backwards (the sine's sign) with the same m.
//
// Bound by HBM: each row is read and written once.  A block takes a tile of
// tokens and a group of heads: its threads first compute the tile's cosines
// and sines into LDS, once for all heads, then stream the rows.  The angle is
// reduced in 64 bits, in quarter turns (position 10^6 at f = 1 keeps 2^-32 of
// a turn; in 32 bits it would lose 2^-5), the remainder's sine and cosine come
// from their Taylor series in 32 bits (|z| <= pi/4: terms up to z^11 and z^10
// leave 2^-37 and 2^-33), then one rounding to the output type.
//
// A thread's item is a chunk of C pairs of one row: 16-byte loads of each
// half for bf16 with C = 8 and fp32 with C = 4 (any address), two 16-byte
// loads side by side when interleaved; C = 4 of bf16 and C = 1 are for
// rotated widths those do not divide.
//
// 4 x 4096 tokens of 32 + 8 heads of 128, bf16: 71 us (335 MB, 4.7 TB/s; a copy of as
// many bytes, not in the caches, 65).  8 x 1 tokens: 4.7 us, a launch.  3 x 1001 x 24
// heads of 80, 40 turned, fp32: 11.9 us (46 MB, 3.9 TB/s).
#pragma once

#include "common.h"
#include "rotary_math.h"
#include "../kargs.h"

using namespace bwpp;

namespace rotary_pos {

constexpr int kMaxAngles = 2048;  // (token, pair) angles of a block: 16 KiB of LDS

template <class T, bool INTER, int C>
__device__ __forceinline__ void rotary(const BwppRotaryArgs &a) {
  __shared__ float2 cs[kMaxAngles];
  const uint32_t tid = threadIdx.x, NT = 256;
  const uint32_t t0 = blockIdx.x % ((a.tokens + a.tile - 1) / a.tile) * a.tile;
  const uint64_t b = blockIdx.x / ((a.tokens + a.tile - 1) / a.tile);
  const uint32_t nt = min(a.tile, a.tokens - t0);
  const uint32_t h0 = blockIdx.y * a.hgroup, nh = min(a.hgroup, a.heads - h0);
  // Angles: a thread keeps its pair and walks the tokens.
  const uint32_t per = a.pairs < NT ? NT / a.pairs : 1u;  // tokens side by side
  if (tid < per * a.pairs || a.pairs >= NT) {
    for (uint32_t i = a.pairs < NT ? tid % a.pairs : tid; i < a.pairs; i += NT) {
      const double f = quarter_turns(a, i);
      for (uint32_t t = a.pairs < NT ? tid / a.pairs : 0u; t < nt; t += per) {
        const int32_t p = a.positions ? a.positions[b * a.pos_bs + t0 + t] : 0;
        // int64: pos0 + token may pass 2^31
        const double pos = a.positions ? (double)p : (double)((int64_t)a.pos0 + (int64_t)(t0 + t));
        cs[t * a.pairs + i] = cos_sin(a, pos * f);
      }
    }
  }
  __syncthreads();

  const uint32_t chunks = a.pairs / C + a.tail_chunks;
  // A thread keeps its chunk where the chunks divide among the threads.
  const uint32_t rows = nt * nh;
  const uint32_t magic = 0xffffffffu / nh + 1u;  // row / nh by a multiply: rows * nh < 2^32 (nh <= 256)
  const uint32_t side = chunks < NT ? NT / chunks : 1u;  // rows side by side
  if (chunks < NT && tid >= side * chunks) return;
  for (uint32_t c = chunks < NT ? tid % chunks : tid; c < chunks; c += NT) {
    for (uint32_t row = chunks < NT ? tid / chunks : 0u; row < rows; row += side) {
      const uint32_t t = nh > 1 ? __umulhi(row, magic) : row;
      const uint32_t hd = h0 + (row - t * nh);
      const bool isq = hd < a.q_heads;
      const uint64_t tok = t0 + t, hh = isq ? hd : hd - a.q_heads;
      const T *src = isq ? static_cast<const T *>(a.q) + (b * a.q_bs + tok * a.q_ts + hh * a.q_hs)
                         : static_cast<const T *>(a.k) + (b * a.k_bs + tok * a.k_ts + hh * a.k_hs);
      T *dst = isq ? static_cast<T *>(a.qo) + (b * a.qo_bs + tok * a.qo_ts + hh * a.qo_hs)
                   : static_cast<T *>(a.ko) + (b * a.ko_bs + tok * a.ko_ts + hh * a.ko_hs);
      if (c >= a.pairs / C) {  // columns that are not rotated
        if (!(a.copy & (isq ? 1u : 2u))) continue;
        const uint32_t c0 = 2 * a.pairs + (c - a.pairs / C) * C;
        if (c0 + C <= a.dim) {
          float v[C];
          Vec<T, C>::load(src + c0, v);
          Vec<T, C>::store(dst + c0, v);
        } else {
          for (uint32_t e = c0; e < a.dim; ++e) dst[e] = src[e];
        }
        continue;
      }
      const float2 *ang = cs + t * a.pairs + c * C;
      if constexpr (INTER) {
        float v[2 * C], o[2 * C];
        Vec<T, 2 * C>::load(src + 2 * c * C, v);
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const float2 w = ang[e];
          o[2 * e] = v[2 * e] * w.x - v[2 * e + 1] * w.y;
          o[2 * e + 1] = v[2 * e + 1] * w.x + v[2 * e] * w.y;
        }
        Vec<T, 2 * C>::store(dst + 2 * c * C, o);
      } else {
        float x[C], y[C], u[C], v[C];
        Vec<T, C>::load(src + c * C, x);
        Vec<T, C>::load(src + a.pairs + c * C, y);
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const float2 w = ang[e];
          u[e] = x[e] * w.x - y[e] * w.y;
          v[e] = y[e] * w.x + x[e] * w.y;
        }
        Vec<T, C>::store(dst + c * C, u);
        Vec<T, C>::store(dst + a.pairs + c * C, v);
      }
    }
  }
}

#define BWPP_ROTARY(NAME, T, INTER, C) \
  extern "C" __global__ __launch_bounds__(256) void bwpp_rotary_##NAME(const BwppRotaryArgs a) { rotary<T, INTER, C>(a); }
BWPP_ROTARY(bf16_half_8, uint16_t, false, 8)
BWPP_ROTARY(bf16_half_4, uint16_t, false, 4)
BWPP_ROTARY(bf16_half_1, uint16_t, false, 1)
BWPP_ROTARY(bf16_inter_8, uint16_t, true, 8)
BWPP_ROTARY(bf16_inter_4, uint16_t, true, 4)
BWPP_ROTARY(bf16_inter_1, uint16_t, true, 1)
BWPP_ROTARY(f32_half_4, float, false, 4)
BWPP_ROTARY(f32_half_1, float, false, 1)
BWPP_ROTARY(f32_inter_4, float, true, 4)
BWPP_ROTARY(f32_inter_1, float, true, 1)

}  // namespace rotary_pos
