// Attention of new tokens over a paged cache, any head dim up to 256, fp32 or
// bf16, any alignment; and the join of items that several blocks shared.
//
//   o[t][h] = sum_p w_p v_p / sum_p w_p,  w_p = e^(scale q[t][h] . k_p)
//
// over the held tokens and those new tokens of the sequence that token t sees
// (its mask bits, or those up to itself).  The query heads that share a key
// head are rows of one tile, so keys and values are read once for all.
//
// A wave holds 16 query rows.  Per 16 keys it computes S^T = K Q^T with fp32
// matrix instructions (16 x 16 x 4, exact products): lane l's keys come
// straight from memory, 4 elements of key l % 16 a load, and are the "A"
// operand as they stand, since a product may take the head's columns in any
// order as long as q's are in the same.  The accumulator then has row l % 16
// against keys 4 (l / 16) .. + 3, which is how the "B" operand of
// O^T += V^T P^T wants the probabilities, and V's rows are loaded 4 columns a
// lane (column 64 j + 4 i + c is row i of product (j, c)).  So nothing passes
// through LDS but the sums at the end.
//
// A block's four waves take every fourth tile of its 16 rows' keys, and their
// sums meet in LDS.  More rows are kv_rows.h's.  Long caches are bound by HBM
// (64 sequences of up to 16000 tokens, 32 : 8 heads of 128, fp32: 351 us, 5.8
// TB/s), short ones by the chain share, pages, tiles, sums and the join's launch
// (6 trees of 13 tokens over up to 2901, 12 heads of 80: 14.7 and 6.6 us).
#pragma once

#include "attention_common.h"
#include "kv_cache.h"
#include "kv_items.h"
#include "rotary_math.h"
#include "../kargs.h"

typedef float f32x4_t __attribute__((ext_vector_type(4)));

namespace kv {

constexpr uint32_t kThreads = 256;

// Four elements from column c of a row of `dim`, zeros past it.
template <class T>
__device__ __forceinline__ void load4(const T *row, uint32_t c, uint32_t dim, float (&o)[4]) {
  if (c + 4 <= dim) {
    rotary_pos::Vec<T, 4>::load(row + c, o);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float e[1] = {0.0f};
      if (c + (uint32_t)i < dim) rotary_pos::Vec<T, 1>::load(row + c + i, e);
      o[i] = e[0];
    }
  }
}

template <class T>
__device__ __forceinline__ void store4(T *row, uint32_t c, uint32_t dim, const float (&v)[4]) {
  if (c + 4 <= dim) {
    rotary_pos::Vec<T, 4>::store(row + c, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e[1] = {v[i]};
      if (c + (uint32_t)i < dim) rotary_pos::Vec<T, 1>::store(row + c + i, e);
    }
  }
}

template <class T, int DC>
__device__ __forceinline__ void attend_split(const BwppCacheAttnArgs &a) {
  constexpr uint32_t kRows = 16, kUnit = 64, kTile = 16, kStep = 4 * kTile;
  constexpr int KC = 4 * DC, kLd = 64 * DC + 4;
  __shared__ float os[4][16][kLd];
  __shared__ float ml[4][16][2];
  const BwppCacheArgs &c = a.c;
  const uint32_t lane = threadIdx.x & 63u, wave = uni(threadIdx.x >> 6), i16 = lane & 15u, grp = lane >> 4;
  const uint32_t D = c.dim, g = a.group, Dp = (D + 3u) & ~3u, pmask = (1u << c.page_shift) - 1u;
  const float scale = a.flip ? -a.scale_log2 : a.scale_log2;

  for_items<kRows, kUnit>(a, [&](const Item &it, uint32_t slot) {
    const uint32_t row = min(it.tile * kRows + i16, it.R - 1u), tok = row / g, hq = it.head * g + row % g;
    float qf[KC][4];
    {
      const T *Q = static_cast<const T *>(a.q) + (uint64_t)(it.q.first + tok) * a.q_ts + (uint64_t)hq * a.q_hs;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        if (16u * j < D) load4(Q, 16u * j + 4u * grp, D, qf[j]);
        else qf[j][0] = qf[j][1] = qf[j][2] = qf[j][3] = 0.0f;
      }
    }
    const T *K = static_cast<const T *>(c.k) + (uint64_t)it.head * c.head_s;
    const T *V = static_cast<const T *>(c.v) + (uint64_t)it.head * c.head_s;
    const int32_t *table = c.table + (uint64_t)it.s * c.ld_table;

    f32x4_t o[DC][4];
#pragma unroll
    for (int j = 0; j < DC; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[j][e] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f;

    uint32_t k0 = it.kbeg + kTile * wave;
    // A lane's key of the tile at k: its row's offset, kNoSlot past the keys or
    // outside the pool.  Page numbers are fetched one tile ahead.
    auto page = [&](uint32_t k) { return k + i16 < it.kend ? (uint32_t)table[(k + i16) >> c.page_shift] : ~0u; };
    auto offset = [&](uint32_t k, uint32_t pg) {
      return pg < c.pages ? (uint64_t)pg * c.page_s + (uint64_t)((k + i16) & pmask) * c.tok_s : kNoSlot;
    };
    float kf[KC][4];
    auto load_keys = [&](uint64_t off) {
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        kf[j][0] = kf[j][1] = kf[j][2] = kf[j][3] = 0.0f;
        if (16u * j < D && off != kNoSlot) load4(K + off, 16u * j + 4u * grp, D, kf[j]);
      }
    };
    uint64_t off = kNoSlot;
    uint32_t next_page = ~0u;
    if (k0 < it.kend) {
      off = offset(k0, page(k0));
      next_page = page(k0 + kStep);
      load_keys(off);
    }
    for (; k0 < it.kend; k0 += kStep) {
      float vf[4][DC][4];
      bool live[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const uint64_t ov = __shfl(off, 4 * grp + r, 64);
        live[r] = ov != kNoSlot;
#pragma unroll
        for (int j = 0; j < DC; ++j) {
          vf[r][j][0] = vf[r][j][1] = vf[r][j][2] = vf[r][j][3] = 0.0f;
          if (live[r] && 64u * j + 4u * i16 < D) load4(V + ov, 64u * j + 4u * i16, D, vf[r][j]);
        }
      }
      f32x4_t s0 = {0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0;
#pragma unroll
      for (int j = 0; j < KC; ++j) {
        if (16u * j >= D) continue;
        s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][0], qf[j][0], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][1], qf[j][1], s1, 0, 0, 0);
        s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][2], qf[j][2], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[j][3], qf[j][3], s1, 0, 0, 0);
      }
      off = offset(k0 + kStep, next_page);
      next_page = page(k0 + 2 * kStep);
      load_keys(off);
      // Visible keys of this lane's row among its four.
      uint32_t vis = (live[0] ? 1u : 0u) | (live[1] ? 2u : 0u) | (live[2] ? 4u : 0u) | (live[3] ? 8u : 0u);
      const bool fresh = k0 + kTile > it.q.held;  // new tokens among the keys
      if (fresh) {
        uint32_t bits = mask_bits32(a, it.q.first, tok, (int64_t)k0 - (int64_t)it.q.held);
        if (k0 < it.q.held) bits |= (1u << (it.q.held - k0)) - 1u;  // fewer than 16
        vis &= bits >> (4u * grp);
      }
      float p[4], mx = -INFINITY;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = vis >> r & 1u ? (s0[r] + s1[r]) * scale : -INFINITY;
        mx = fmaxf(mx, p[r]);
      }
      mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      float alpha = 1.0f;
      if (mx > m + kLazy) {
        alpha = __builtin_amdgcn_exp2f(m - mx);  // 0 when m is -inf
        m = mx;
      }
      const float use = m == -INFINITY ? 0.0f : m;
      float sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[r] = __builtin_amdgcn_exp2f(p[r] - use);
        sum += p[r];
      }
      l = l * alpha + sum;  // of this lane's keys: the lanes of a row are added at the end
      if (__ballot(alpha != 1.0f)) {
#pragma unroll
        for (int j = 0; j < DC; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[j][e] *= alpha;
      }
      // 0 times an infinite or NaN v would reach rows that do not see it.
      bool odd = false;
      if (fresh) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < DC; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= !(fabsf(vf[r][j][e]) < INFINITY);
      }
      if (fresh && __ballot(odd)) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          for (uint32_t k4 = 0; k4 < 4; ++k4) {  // key 4 k4 + r
            const float pk = __shfl(p[r], 16 * k4 + i16, 64);
            const bool see = __shfl(vis >> r & 1u, 16 * k4 + i16, 64) != 0;
#pragma unroll
            for (int j = 0; j < DC; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int rr = 0; rr < 4; ++rr) {
                  const float v = __shfl(vf[r][j][e], 16 * k4 + 4 * grp + rr, 64);
                  if (see) o[j][e][rr] += pk * v;
                }
          }
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
          for (int j = 0; j < DC; ++j) {
            if (64u * j >= D) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              o[j][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[r][j][e], p[r], o[j][e], 0, 0, 0);
          }
      }
    }
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);

    // Results: row i16 has columns 64 j + 4 (4 grp + rr) + e in o[j][e][rr].
    auto put = [&](uint32_t rw, uint32_t col, const float (&v)[4], float mm, float ll, bool head) {
      // rw: row of the tile
      const uint32_t rr = it.tile * kRows + rw;
      if (rr >= it.R || col >= D) return;
      if (!it.whole) {
        float *po = a.part_o + ((uint64_t)slot * kRows + rw) * Dp + col;
        *reinterpret_cast<float4 *>(po) = make_float4(v[0], v[1], v[2], v[3]);
        if (head) *reinterpret_cast<float2 *>(a.part_ml + ((uint64_t)slot * kRows + rw) * 2) = make_float2(mm, ll);
        return;
      }
      const uint64_t t = it.q.first + rr / g, hh = it.head * g + rr % g;
      const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
      const float u[4] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
      store4(static_cast<T *>(a.o) + t * a.o_ts + hh * a.o_hs, col, D, u);
      if (head && a.lse) a.lse[t * (uint64_t)(c.heads * g) + hh] = ll == 0.0f ? -INFINITY : lse_of(mm == -INFINITY ? 0.0f : mm, ll);
    };
    {
#pragma unroll
      for (int j = 0; j < DC; ++j)
#pragma unroll
        for (int rr = 0; rr < 4; ++rr)
          *reinterpret_cast<float4 *>(&os[wave][i16][64 * j + 4 * (4 * grp + rr)]) =
              make_float4(o[j][0][rr], o[j][1][rr], o[j][2][rr], o[j][3][rr]);
      if (grp == 0) ml[wave][i16][0] = m, ml[wave][i16][1] = l;
      __syncthreads();
      for (uint32_t i = threadIdx.x; i < 16u * (Dp / 4u); i += kThreads) {
        const uint32_t rw = i / (Dp / 4u), col = 4u * (i % (Dp / 4u));
        float mm = -INFINITY, ll = 0.0f, v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w) mm = fmaxf(mm, ml[w][rw][0]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float mw = ml[w][rw][0];
          // no key seen (offset -inf): sums of 0 (or NaN, kept)
          const float f = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - mm);
          ll += ml[w][rw][1] * f;
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += os[w][rw][col + e] * f;
        }
        put(rw, col, v, mm, ll, col == 0);
      }
      __syncthreads();
    }
  });
}

// Four columns at E places of an item's tile, joined from its parts, P of which
// are fetched at once.
template <int E, int P, class Sums, class Pair, class Put>
__device__ __forceinline__ void join_columns(uint32_t i0, uint32_t end, uint32_t parts, Sums sums, Pair pair, Put put) {
  float4 u[E][P], v[E];
  float2 w[E][P];
  float m[E], l[E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    v[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    m[e] = -INFINITY;
    l[e] = 0.0f;
  }
  for (uint32_t k = 0; k < parts; k += P) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t i = i0 + e * kThreads;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const bool there = i < end && k + j < parts;
        w[e][j] = there ? pair(k + j, i) : make_float2(-INFINITY, 0.0f);
        u[e][j] = there ? sums(k + j, i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
      float top = m[e];
#pragma unroll
      for (int j = 0; j < P; ++j) top = fmaxf(top, w[e][j].x);
      // no key seen (offset -inf): sums of 0 (or NaN, kept)
      auto factor = [&](float o) { return o == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(o - top); };
      const float f = factor(m[e]);
      l[e] *= f;
      v[e] = make_float4(v[e].x * f, v[e].y * f, v[e].z * f, v[e].w * f);
      m[e] = top;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        const float fj = factor(w[e][j].x);
        l[e] += w[e][j].y * fj;
        v[e].x += u[e][j].x * fj, v[e].y += u[e][j].y * fj, v[e].z += u[e][j].z * fj, v[e].w += u[e][j].w * fj;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (i0 + e * kThreads < end) put(i0 + e * kThreads, v[e], m[e], l[e]);
}

// Joins the parts of divided items.  The blocks of a border (blockIdx.x + 1, a
// column of the grid) work on the item that it divides, with those of the other
// borders inside it, each on an even share of its tile's places (a row's four
// columns): parts times places of a block are much the same for any lengths.
// A chain of latencies (costs, pairs with sums, store), so 16 sums a thread are
// fetched at once: 8 trees of 48 tokens, tiles of 256 rows, 32 MB of parts 13 us (17
// with 16 rows for a block of each item's first border); 2 x 2048 tokens of prompts
// 20 (33).
template <class T, uint32_t kRows, uint32_t kUnit>
__device__ __forceinline__ void join(const BwppCacheAttnArgs &a) {
  typedef Work<kRows, kUnit> W;
  const BwppCacheArgs &c = a.c;
  const Costs<kRows, kUnit> costs(a);
  const uint32_t b = blockIdx.x + 1;
  const uint64_t S = share_of(a, costs.total), x = S * b;
  if (costs.whole || x >= costs.total) return;
  Seq q;
  uint64_t before, begin, end;
  const uint32_t seq = costs.at(a, x, q, before);
  const Place item = W::find(a, false, seq, q, x - before, begin, end);
  if (item.unit == 0) return;
  // Its borders first .. last; before them one may lie in it and divide nothing (unit 0).
  uint32_t first = (uint32_t)((double)(before + begin) / (double)S);
  if (S * first < before + begin) ++first;
  first = min(max(first, 1u), b);
  while (first < b && W::unit(a, q, item.tile, S * first - before - begin, end - begin) == 0) ++first;
  uint32_t last = (uint32_t)((double)(before + end - 1) / (double)S);
  if (S * last >= before + end) --last;  // (a quotient rounded up)
  last = min(max(last, b), a.blocks - 1u);  // (costs past 2^52: only sequences that overlap have them)
  const uint32_t g = a.group, D = c.dim, n4 = (D + 3u) / 4u, Dp = 4u * n4;
  const uint32_t places = min(kRows, q.n * g - item.tile * kRows) * n4, parts = last - first + 2;
  const uint32_t sharers = (last - first + 1) * gridDim.y, per = (places + sharers - 1) / sharers;
  const uint32_t i0 = per * ((b - first) * gridDim.y + blockIdx.y), i1 = min(i0 + per, places);
  // part 0 in slot 2 (first - 1) + 1, part k in slot 2 (first + k - 1)
  auto slot_row = [&](uint32_t k) { return (uint64_t)(k == 0 ? 2 * first - 1 : 2 * (first + k - 1)) * kRows; };
  auto sums = [&](uint32_t k, uint32_t i) { return *reinterpret_cast<const float4 *>(a.part_o + slot_row(k) * Dp + 4u * i); };
  auto pair = [&](uint32_t k, uint32_t i) { return *reinterpret_cast<const float2 *>(a.part_ml + 2 * (slot_row(k) + i / n4)); };
  auto put = [&](uint32_t i, const float4 &v, float m, float l) {
    const uint32_t r = i / n4, col = 4u * (i % n4), rr = item.tile * kRows + r;
    const uint64_t t = q.first + rr / g, hh = item.head * g + rr % g;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const float u[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
    store4(static_cast<T *>(a.o) + t * a.o_ts + hh * a.o_hs, col, D, u);
    if (col == 0 && a.lse) a.lse[t * (uint64_t)(c.heads * g) + hh] = l == 0.0f ? -INFINITY : lse_of(m == -INFINITY ? 0.0f : m, l);
  };
  const uint32_t i = i0 + threadIdx.x;
  if (per <= kThreads) {
    if (i < i1) join_columns<1, 16>(i, i1, parts, sums, pair, put);
  } else if (parts <= 4) {
    for (uint32_t e = i; e < i1; e += 4 * kThreads) join_columns<4, 4>(e, i1, parts, sums, pair, put);
  } else {
    for (uint32_t e = i; e < i1; e += 2 * kThreads) join_columns<2, 8>(e, i1, parts, sums, pair, put);
  }
}

}  // namespace kv

#define BWPP_ATTEND(NAME, T, DC)                                                                                    \
  extern "C" __global__ __launch_bounds__(256, DC <= 2 ? 2 : 1) void bwpp_cache_attend_##NAME(const BwppCacheAttnArgs a) { \
    kv::attend_split<T, DC>(a);                                                                                     \
  }
BWPP_ATTEND(f32_d64, float, 1)
BWPP_ATTEND(f32_d128, float, 2)
BWPP_ATTEND(f32_d192, float, 3)
BWPP_ATTEND(f32_d256, float, 4)
BWPP_ATTEND(bf16_d64, uint16_t, 1)
BWPP_ATTEND(bf16_d128, uint16_t, 2)
BWPP_ATTEND(bf16_d192, uint16_t, 3)
BWPP_ATTEND(bf16_d256, uint16_t, 4)

#define BWPP_JOIN(NAME, T, ROWS) \
  extern "C" __global__ __launch_bounds__(256, 4) void bwpp_cache_join_##NAME(const BwppCacheAttnArgs a) { kv::join<T, ROWS, 64>(a); }
BWPP_JOIN(f32_16, float, 16)
BWPP_JOIN(f32_128, float, 128)
BWPP_JOIN(bf16_16, uint16_t, 16)
BWPP_JOIN(bf16_32, uint16_t, 32)
BWPP_JOIN(bf16_128, uint16_t, 128)
BWPP_JOIN(bf16_256, uint16_t, 256)
