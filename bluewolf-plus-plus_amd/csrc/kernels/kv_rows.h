// Attention over a paged cache for many query rows, any head dim up to 256,
// fp32 or bf16, any alignment, on the fp32 matrix cores (32 x 32 x 2): what
// kv_flash.h does not take.
//
// A block of four waves has a tile of 128 rows, a wave 32 of them.  Tiles of 32
// keys and values come through registers, a tile ahead, into LDS as fp32, rows
// of 32 DB columns (zeros behind the head's) and 4 more, so that the 16 rows of
// a quarter-wave's 16-byte read fall on distinct banks.  S^T = K Q^T takes 4
// columns a lane from LDS; of its result lane l has row l % 32 against keys
// 8 (r >> 2) + 4 (l / 32) + (r & 3), which is how O^T += V^T P^T takes its "B"
// operand, 2 keys a product.  The matrix products bound it: 2 x 1024 tokens of
// prompts, 32 : 8 heads of 128, fp32 257 us, 99 TFLOP/s (a large library product
// reaches 137).  On the 16-row tiles, which read keys for every 16 rows: 461 us.
#pragma once

#include "attention_common.h"
#include "kv_items.h"
#include "kv_attention.h"
#include "../kargs.h"

namespace kv {

template <class T, int DB>
__device__ __forceinline__ void attend_rows_f32(const BwppCacheAttnArgs &a) {
  constexpr uint32_t kRows = 128, kKeys = 32, kChunks = 8 * DB, kPitch = 32 * DB + 4;
  __shared__ __attribute__((aligned(16))) float ks[kKeys][kPitch], vs[kKeys][kPitch];
  __shared__ uint32_t pages[kPages];
  const BwppCacheArgs &c = a.c;
  const uint32_t lane = threadIdx.x & 63u, wave = uni(threadIdx.x >> 6), lq = lane & 31u, lh = lane >> 5;
  const uint32_t D = c.dim, g = a.group, Dp = (D + 3u) & ~3u, pmask = (1u << c.page_shift) - 1u;
  const float scale = a.flip ? -a.scale_log2 : a.scale_log2;

  for_items<kRows, 64>(a, [&](const Item &it, uint32_t slot) {
    const uint32_t row0 = it.tile * kRows + 32u * wave, row = min(row0 + lq, it.R - 1u), tok = row / g;
    float qf[4 * DB][4];
    {
      const T *Q = static_cast<const T *>(a.q) + (uint64_t)(it.q.first + tok) * a.q_ts + (uint64_t)(it.head * g + row % g) * a.q_hs;
#pragma unroll
      for (int j = 0; j < 4 * DB; ++j) load4(Q, 8u * j + 4u * lh, D, qf[j]);  // zeros past the head's columns
    }
    const T *K = static_cast<const T *>(c.k) + (uint64_t)it.head * c.head_s;
    const T *V = static_cast<const T *>(c.v) + (uint64_t)it.head * c.head_s;
    f32x16_t o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    // Keys below `all` are seen by all of the wave's rows (`all_block`: the block's), from `none` on by none.
    const uint32_t t0 = min(row0, it.R - 1u) / g, t1 = min(row0 + 31u, it.R - 1u) / g;
    const uint32_t all = a.mask ? it.q.held : it.q.held + t0 + 1u;
    const uint32_t all_block = a.mask ? it.q.held : it.q.held + it.tile * kRows / g + 1u;
    const uint32_t none = row0 >= it.R ? 0u : a.mask ? it.kend : min(it.kend, it.q.held + t1 + 1u);

    for (uint32_t seg = it.kbeg; seg < it.kend;) {
      bool bad;
      const uint32_t end = uni(load_pages<256>(c, it, seg, pages, bad)), first = seg >> c.page_shift;
      float kr[DB][4], vr[DB][4];
      auto fetch = [&](uint32_t k0) {
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          const uint32_t x = threadIdx.x + 256u * i, key = min(k0 + x / kChunks, it.kend - 1), col = 4u * (x % kChunks);
          const uint32_t page = pages[(key >> c.page_shift) - first] & ~kNoPage;
          const uint64_t off = (uint64_t)page * c.page_s + (uint64_t)(key & pmask) * c.tok_s;
          load4(K + off, col, D, kr[i]);
          load4(V + off, col, D, vr[i]);
        }
      };
      fetch(seg);
      for (uint32_t k0 = seg; k0 < end; k0 += kKeys) {
        const bool fresh = bad || k0 + kKeys > it.kend || k0 + kKeys > all_block;  // the same in every wave
        bool odd = false;
        __syncthreads();  // done with the last tile
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          const uint32_t x = threadIdx.x + 256u * i;
          *reinterpret_cast<float4 *>(&ks[x / kChunks][4u * (x % kChunks)]) = make_float4(kr[i][0], kr[i][1], kr[i][2], kr[i][3]);
          *reinterpret_cast<float4 *>(&vs[x / kChunks][4u * (x % kChunks)]) = make_float4(vr[i][0], vr[i][1], vr[i][2], vr[i][3]);
          if (fresh)
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= !(fabsf(vr[i][e]) < INFINITY);
        }
        bool found = false;  // infinite or NaN values: 0 times those would reach rows that do not see them
        if (fresh) found = __syncthreads_or(odd) != 0;
        else __syncthreads();
        if (k0 + kKeys < end) fetch(k0 + kKeys);
        const bool mine = k0 < none, masked = fresh && (bad || k0 + kKeys > it.kend || k0 + kKeys > all);
        uint32_t vis = ~0u;
        if (masked) {
          if (k0 + kKeys > it.q.held) {
            vis = mask_bits32(a, it.q.first, tok, (int64_t)k0 - (int64_t)it.q.held);
            if (k0 < it.q.held) vis |= (1u << (it.q.held - k0)) - 1u;  // fewer than 32
          }
          vis &= keys_with_page(c, it, k0, first, pages);
        }
        f32x16_t s;
        if (mine) {
#pragma unroll
          for (int r = 0; r < 16; ++r) s[r] = 0.0f;
          // Operands are read ahead of their products; the order is held by hand.
          auto read = [&](int j) { return *reinterpret_cast<const float4 *>(&ks[lq][8u * j + 4u * lh]); };
          float4 k4[2] = {read(0), read(1)};
#pragma unroll
          for (int j = 0; j < 4 * DB; ++j) {
            __builtin_amdgcn_sched_barrier(0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k4[j % 2].x, qf[j][0], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k4[j % 2].y, qf[j][1], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k4[j % 2].z, qf[j][2], s, 0, 0, 0);
            s = __builtin_amdgcn_mfma_f32_32x32x2f32(k4[j % 2].w, qf[j][3], s, 0, 0, 0);
            if (j + 2 < 4 * DB) k4[j % 2] = read(j + 2);
          }
          __builtin_amdgcn_sched_barrier(0);
          const uint32_t w = vis >> (4u * lh);
          float mx = -INFINITY;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[r] = w >> (8 * (r >> 2) + (r & 3)) & 1u ? s[r] * scale : -INFINITY;
            mx = fmaxf(mx, s[r]);
          }
          mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
          float alpha = 1.0f;
          if (mx > m + kLazy) {
            alpha = __builtin_amdgcn_exp2f(m - mx);  // 0 when m is -inf
            m = mx;
          }
          const float use = m == -INFINITY ? 0.0f : m;
          float sum = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[r] = __builtin_amdgcn_exp2f(s[r] - use);
            sum += s[r];
          }
          l = l * alpha + sum;  // of this lane's keys; lane ^ 32 has the others
          if (__ballot(alpha != 1.0f)) {
#pragma unroll
            for (int d = 0; d < DB; ++d)
#pragma unroll
              for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
          }
        }
        if (found) {
          // What the rows that see them get, key by key; then zeros in their place.
          if (mine)
            for (uint32_t k = 0; k < kKeys; ++k) {
              float p = 0.0f;
#pragma unroll
              for (int r = 0; r < 16; ++r) p = (uint32_t)r == 4u * (k >> 3) + (k & 3u) ? s[r] : p;
              p = __shfl(p, (int)(lq + 32u * (k >> 2 & 1u)), 64);
              const bool see = vis >> k & 1u;
#pragma unroll
              for (int d = 0; d < DB; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                  if (r % 4 == 0) asm volatile("" ::: "memory");  // few reads at a time: registers
                  const float v = vs[k][32 * d + 8 * (r >> 2) + 4 * lh + (r & 3)];
                  if (see && !(fabsf(v) < INFINITY)) o[d][r] += p * v;
                }
            }
          __syncthreads();
          for (uint32_t x = threadIdx.x; x < kKeys * 32u * DB; x += 256u) {
            float &v = vs[x / (32u * DB)][x % (32u * DB)];
            if (!(fabsf(v) < INFINITY)) v = 0.0f;
          }
          __syncthreads();
        }
        if (mine) {
          constexpr int N = 16 * DB, kAhead = 6;
          auto read = [&](int i) { return vs[8 * (i / DB >> 2) + 4 * lh + (i / DB & 3)][32 * (i % DB) + lq]; };
          float v[kAhead];
#pragma unroll
          for (int i = 0; i < kAhead; ++i) v[i] = read(i);
#pragma unroll
          for (int i = 0; i < N; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            o[i % DB] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[i % kAhead], s[i / DB], o[i % DB], 0, 0, 0);
            if (i + kAhead < N) v[i % kAhead] = read(i + kAhead);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      seg = end;
    }
    l += __shfl_xor(l, 32, 64);
    if (row0 + lq >= it.R) return;
    const uint32_t rw = 32u * wave + lq;
    const uint64_t t = it.q.first + tok, hh = it.head * g + row % g, sr = (uint64_t)slot * kRows + rw;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const uint32_t col = 32u * d + 8u * q4 + 4u * lh;
        if (col >= D) continue;
        if (it.whole) {
          const float u[4] = {o[d][4 * q4] * inv, o[d][4 * q4 + 1] * inv, o[d][4 * q4 + 2] * inv, o[d][4 * q4 + 3] * inv};
          store4(static_cast<T *>(a.o) + t * a.o_ts + hh * a.o_hs, col, D, u);
        } else {
          *reinterpret_cast<float4 *>(a.part_o + sr * Dp + col) =
              make_float4(o[d][4 * q4], o[d][4 * q4 + 1], o[d][4 * q4 + 2], o[d][4 * q4 + 3]);
        }
      }
    if (lh == 0) {
      if (!it.whole) *reinterpret_cast<float2 *>(a.part_ml + 2 * sr) = make_float2(m, l);
      else if (a.lse) a.lse[t * (uint64_t)(c.heads * g) + hh] = l == 0.0f ? -INFINITY : lse_of(m == -INFINITY ? 0.0f : m, l);
    }
  });
}

}  // namespace kv

#define BWPP_ATTEND_ROWS_F32(NAME, T, DB)                                                                             \
  extern "C" __global__ __launch_bounds__(256, DB <= 4 ? 2 : 1) void bwpp_cache_attend_##NAME(const BwppCacheAttnArgs a) { \
    kv::attend_rows_f32<T, DB>(a);                                                                                    \
  }
BWPP_ATTEND_ROWS_F32(f32_rows_d32, float, 1)
BWPP_ATTEND_ROWS_F32(f32_rows_d64, float, 2)
BWPP_ATTEND_ROWS_F32(f32_rows_d96, float, 3)
BWPP_ATTEND_ROWS_F32(f32_rows_d128, float, 4)
BWPP_ATTEND_ROWS_F32(f32_rows_d160, float, 5)
BWPP_ATTEND_ROWS_F32(f32_rows_d192, float, 6)
BWPP_ATTEND_ROWS_F32(f32_rows_d224, float, 7)
BWPP_ATTEND_ROWS_F32(f32_rows_d256, float, 8)
BWPP_ATTEND_ROWS_F32(bf16_rows_d32, uint16_t, 1)
BWPP_ATTEND_ROWS_F32(bf16_rows_d64, uint16_t, 2)
BWPP_ATTEND_ROWS_F32(bf16_rows_d96, uint16_t, 3)
BWPP_ATTEND_ROWS_F32(bf16_rows_d128, uint16_t, 4)
BWPP_ATTEND_ROWS_F32(bf16_rows_d160, uint16_t, 5)
BWPP_ATTEND_ROWS_F32(bf16_rows_d192, uint16_t, 6)
BWPP_ATTEND_ROWS_F32(bf16_rows_d224, uint16_t, 7)
BWPP_ATTEND_ROWS_F32(bf16_rows_d256, uint16_t, 8)
