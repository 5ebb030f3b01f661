// Attention over a paged cache for bf16 rows of 16-byte chunks, head dims of
// multiples of 16, on the bf16 matrix cores: the scheme of attention.hip
// (S^T = K Q^T, softmax on the accumulator registers, O^T += V^T P^T with V
// read transposed from LDS) over pages.
//
// A wave holds 32 query rows, which are the tokens of a tile times the query
// heads of one key head, so a key is read once for all of them.
//
// Few rows (attend_few): reading K and V once bounds it.  A block of NW waves
// has one tile of 32 rows; every wave streams key tiles of 32 of its own
// (every NW-th of the block's) through a DMA ring of its own, and the waves'
// triples meet in LDS at the end of an item.  64 sequences of up to 32768
// tokens, 32 : 8 heads of 128: 300 us, 6.5 TB/s (through the caches 334); of up to
// 16000, pages of 16 tokens 164 us (6.2), d = 64 92 us (5.5).  Four waves a block
// measured no better.
//
// More rows (attend_rows): the matrix products and the softmax bound it, and
// with them power (2 x 2048 tokens over up to 32000, 32 : 8 heads of 128: 362 to 379 us
// with the join, 880 to 920 TFLOP/s, the matrix pipe busy in 49 % of the cycles at 1.7 to
// 2.0 GHz; a large library product reaches 1215).  Each of a block's waves has
// 32 rows of the tile, and key tiles of 64 come through a two-stage ring that all
// of them read (four stages: the same times): four waves, two blocks a CU, or, for
// more than 128 rows and head dims up to 128, eight (of the attention alone: four
// 386 us, eight 379; 8 trees of 48 tokens 62 and 57).  P enters its product as two
// bf16 terms, except for d = 128, where it is rounded to one: so do attention.hip's
// kernels for many queries (two terms or fp32 for every other dim).  For d = 128 two
// would cost 475 and 64 us, and the result's error (rms, of its norm) is 0.0022 with
// one, 0.0017, its own rounding, with two.  For the other dims the second term costs
// 26 to 33 % of prompts and 7 to 20 % of trees (2 x 2048 tokens over 32000 d = 64 1102
// -> 1458 us, d = 256 4398 -> 5559; 8 trees of 48 54 -> 64 and 176 -> 197), and one
// term was off by up to nine times the bound of two.
//
// Page numbers of an item's keys are copied to LDS, 1024 at a time, before its
// tiles: no load of the compiler's is outstanding beside the DMA, whose
// completion is counted by hand.  Where a key tile lies in one page its base
// is a scalar and the lanes' offsets in the tile never change; smaller pages
// take an address per lane and row.
#pragma once

#include "attention_common.h"
#include "kv_cache.h"
#include "kv_items.h"
#include "../kargs.h"

namespace kv {

// 16 bytes a lane from memory to LDS (see g2lds16_so), from a scalar base or a
// 64-bit address a lane.  The LDS address passes through a scalar register by
// name: one chosen by the compiler may be VCC, and the code objects' check of M0
// takes plain ones.  ONCE: past the caches (Item::once).
template <bool ONCE>
__device__ __forceinline__ void dma16_so(const void *sbase, uint32_t voff, uint32_t lds_addr) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"{s33}"(lds_addr), "v"(voff), "s"(sbase) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{s33}"(lds_addr), "v"(voff), "s"(sbase) : "memory");
}
template <bool ONCE>
__device__ __forceinline__ void dma16_v(const void *addr, uint32_t lds_addr) {
  if constexpr (ONCE)
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off nt" ::"{s33}"(lds_addr), "v"(addr) : "memory");
  else
    asm volatile("s_mov_b32 m0, %0\n\tglobal_load_lds_dwordx4 %1, off" ::"{s33}"(lds_addr), "v"(addr) : "memory");
}

// A tile of key or value rows in LDS: dense rows of D / 8 chunks of 16 bytes,
// chunk c of row r at c ^ swz(r).
template <int D>
struct Rows {
  static constexpr uint32_t kSlots = D / 8, kRowB = 16 * kSlots;
  static constexpr uint32_t kPow = kSlots & (~kSlots + 1);         // chunks that may change places
  static constexpr uint32_t kMask = (kPow < 16 ? kPow : 16) - 1;
  static constexpr uint32_t kShift = kPow >= 16 ? 0 : kPow == 8 ? 1 : kPow == 4 ? 2 : 3;  // rows that differ by their address
  // The 16 rows of a quarter-wave's ds_read_b128 fall on distinct bank groups.
  static __device__ __forceinline__ uint32_t k_swz(uint32_t r) { return (r >> kShift) & kMask; }
  // Rows of a half-wave's transposing reads likewise; unchanged by steps of 8 rows.
  static __device__ __forceinline__ uint32_t v_swz(uint32_t r) {
    return kSlots % 16 == 0 ? 4u * (r & 3u) : kSlots % 8 == 0 ? 4u * ((r >> 1) & 1u) : 0u;
  }
};

// A wave's 32 query rows and what it has of their results.  Lane l has row
// l % 32; of a block of 32 keys it has the scores of keys 8 (r >> 2) + 4 (l >>
// 5) + (r & 3) in register r.
template <int D, int KB>
struct Wave32 {
  using R = Rows<D>;
  static constexpr int KS = D / 16, DB = (D + 31) / 32, kKeys = 32 * KB;
  static constexpr uint32_t kTile = kKeys * R::kRowB, kStage = 2 * kTile;
  static constexpr int kAhead = 4;  // operands read ahead of their products
  bf16x8_t q[KS];
  f32x16_t o[DB];
  float m, l, c;
  uint32_t lq, lh, koff[KS], voff[DB];

  __device__ __forceinline__ void place() {
    const uint32_t lane = threadIdx.x & 63u, grp = lane >> 4, L = lane & 15u;
    lq = lane & 31u;
    lh = lane >> 5;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) koff[ks] = lq * R::kRowB + 16u * ((2u * ks + lh) ^ R::k_swz(lq));
    const uint32_t kbase = 4u * (grp >> 1) + (L >> 2);
#pragma unroll
    for (int d = 0; d < DB; ++d) {
      const uint32_t col = 32u * d + 16u * (grp & 1u) + 4u * (L & 3u);
      voff[d] = kTile + kbase * R::kRowB + 16u * ((col >> 3) ^ R::v_swz(kbase)) + (col & 7u) * 2u;
    }
  }
  // Starts an item: the query row at Q (any valid row where the lane has none).
  __device__ __forceinline__ void start(const uint16_t *Q, float scale_log2, uint32_t flip) {
    c = scale_log2;
    const uint32_t sign = flip ? 0x80008000u : 0u;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      uint4 v = *reinterpret_cast<const uint4 *>(Q + 16 * ks + 8 * lh);
      v.x ^= sign, v.y ^= sign, v.z ^= sign, v.w ^= sign;
      q[ks] = __builtin_bit_cast(bf16x8_t, v);
    }
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) o[d][r] = 0.0f;
    m = -INFINITY;
    l = 0.0f;
  }

  // Scores and probabilities (in s) of the key tile at `st`.  masked: vis has bit k
  // of word kb where this lane's row sees key 32 kb + k; otherwise all are seen.
  __device__ __forceinline__ void scores(const unsigned char *st, bool masked, const uint32_t (&vis)[KB], f32x16_t (&s)[KB]) {
    // kAhead reads of K on the way; the order is held by hand (left to itself the
    // compiler reads each operand right before its product and waits for it).
    constexpr int N = KB * KS, A = N < kAhead ? N : kAhead;
    uint4 kf[kAhead];
    auto read = [&](int i) { return *reinterpret_cast<const uint4 *>(st + koff[i % KS] + 32u * (i / KS) * R::kRowB); };
#pragma unroll
    for (int i = 0; i < A; ++i) kf[i] = read(i);
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __builtin_amdgcn_sched_barrier(0);
      s[i / KS] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, kf[i % kAhead]), q[i % KS], s[i / KS], 0, 0, 0);
      if (i + A < N) kf[i % kAhead] = read(i + A);
    }
    __builtin_amdgcn_sched_barrier(0);
    if (masked) {  // wave-uniform
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint32_t w = vis[kb] >> (4u * lh);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = w >> (8 * (r >> 2) + (r & 3)) & 1u ? s[kb][r] : -INFINITY;
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[kb][r]);
    {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
      mx = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])) * c;
    }
    float alpha = 1.0f;
    if (mx > m + kLazy) {
      alpha = __builtin_amdgcn_exp2f(m - mx);  // 0 when m is -inf
      m = mx;
    }
    const float use = m == -INFINITY ? 0.0f : m;
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], c, -use));
        s[kb][r] = p;
        sum += p;
      }
    l = l * alpha + sum;  // of this lane's keys; lane ^ 32 has the others
    if (__ballot(alpha != 1.0f)) {
#pragma unroll
      for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[d][r] *= alpha;
    }
  }

  // O^T += V^T P^T.  P enters as two bf16 terms, 2^-16 of p together, or rounded to
  // one, 2^-8 (the sum of p has it whole).
  template <int TERMS>
  __device__ __forceinline__ void products(const unsigned char *st, const f32x16_t (&s)[KB]) {
    constexpr int N = KB * 2 * DB, A = N < kAhead ? N : kAhead;
    v8s_t vf[kAhead];
    auto read = [&](int i) {  // block i % DB of 32 columns, keys 16 (i / DB) ..
      const unsigned char *p = st + voff[i % DB] + 16u * (i / DB) * R::kRowB;
      const v4s_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t *)p);
      const v4s_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s_t *)(p + 8u * R::kRowB));
      return v8s_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
#pragma unroll
    for (int i = 0; i < A; ++i) vf[i] = read(i);
    bf16x8_t ph, pl;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int d = i % DB, kb = i / DB / 2, r0 = 8 * (i / DB % 2);
      if (d == 0) {
        if constexpr (TERMS == 2) {
          split_bf16x8(&s[kb], r0, ph, pl);
        } else {
          const uint4 w = make_uint4(pack_bf16x2(s[kb][r0], s[kb][r0 + 1]), pack_bf16x2(s[kb][r0 + 2], s[kb][r0 + 3]),
                                     pack_bf16x2(s[kb][r0 + 4], s[kb][r0 + 5]), pack_bf16x2(s[kb][r0 + 6], s[kb][r0 + 7]));
          ph = __builtin_bit_cast(bf16x8_t, w);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf[i % kAhead]), ph, o[d], 0, 0, 0);
      if constexpr (TERMS == 2)
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, vf[i % kAhead]), pl, o[d], 0, 0, 0);
      if (i + A < N) vf[i % kAhead] = read(i + A);
    }
    __builtin_amdgcn_sched_barrier(0);
  }

  // Infinite and NaN values of a tile with masked keys: 0 times those would reach
  // rows that do not see them.  Where odd_values finds one, add_odd adds what the
  // rows that see them get, key by key, and clear_odd puts zeros in their place,
  // before the products.  `share` of `shares` that look through the tile.
  static __device__ __forceinline__ bool odd_values(const unsigned char *st, uint32_t share, uint32_t shares) {
    u16x2_t big = {0, 0};
    for (uint32_t i = share * 64u + (threadIdx.x & 63u); i < kTile / 16u; i += shares * 64u)
      big = max_abs_bf16(big, *reinterpret_cast<const v8s_t *>(st + kTile + 16u * i));
    return __ballot(big[0] >= 0x7f80u || big[1] >= 0x7f80u) != 0;
  }
  __device__ __forceinline__ void add_odd(const unsigned char *st, const uint32_t (&vis)[KB], const f32x16_t (&s)[KB]) {
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
      for (uint32_t k = 0; k < 32; ++k) {
        float mine = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) mine = (uint32_t)r == 4u * (k >> 3) + (k & 3u) ? s[kb][r] : mine;
        const float pk = __shfl(mine, (int)(lq + 32u * (k >> 2 & 1u)), 64);
        const bool see = vis[kb] >> k & 1u;
        const uint32_t row = 32u * kb + k;
        const unsigned char *vr = st + kTile + row * R::kRowB;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            if (r % 4 == 0) asm volatile("" ::: "memory");  // few reads at a time: registers
            const uint32_t col = 32u * d + 8u * (r >> 2) + 4u * lh + (r & 3);
            if (col >= (uint32_t)D) continue;
            const float v = bf16_bits_to_f32(*reinterpret_cast<const uint16_t *>(
                vr + 16u * ((col >> 3) ^ R::v_swz(row)) + 2u * (col & 7u)));
            if (see && !(fabsf(v) < INFINITY)) o[d][r] += pk * v;
          }
      }
  }
  static __device__ __forceinline__ void clear_odd(unsigned char *st, uint32_t share, uint32_t shares) {
    for (uint32_t i = share * 64u + (threadIdx.x & 63u); i < kTile / 16u; i += shares * 64u) {
      v8s_t *p = reinterpret_cast<v8s_t *>(st + kTile + 16u * i);
      v8s_t v = *p;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (v[e] & 0x7f80) == 0x7f80 ? (short)0 : v[e];
      *p = v;
    }
  }
  // The row's whole sum in both of its lanes.
  __device__ __forceinline__ void finish() {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
    l = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
};

// Rows of keys and values from their pages to LDS: one wave's share (every
// STEP-th from `from` on) of the DMA instructions of a tile of KEYS keys.
template <int D, int KEYS, int FROM_WAVES>
struct Fetch {
  using R = Rows<D>;
  static constexpr uint32_t kDma = KEYS * R::kSlots / 64, kMine = (kDma + FROM_WAVES - 1) / FROM_WAVES;
  static constexpr uint32_t kTile = KEYS * R::kRowB;
  const uint16_t *K, *V;  // the item's key head
  static constexpr bool kKeep = kMine <= 8;  // offsets are kept in registers, more of them made again
  uint32_t kept[kKeep ? 2 * kMine : 1];
  uint32_t wave, tok_s;   // wave: of FROM_WAVES that share the tile

  static __device__ __forceinline__ uint32_t slot(uint32_t i, uint32_t w) { return (i * FROM_WAVES + w) * 64u + (threadIdx.x & 63u); }
  __device__ __forceinline__ void place(const BwppCacheArgs &c, uint32_t w) {
    wave = w;
    tok_s = (uint32_t)c.tok_s;
    if constexpr (kKeep) {
#pragma unroll
      for (uint32_t i = 0; i < kMine; ++i) kept[2 * i] = offset(i, false), kept[2 * i + 1] = offset(i, true);
    }
  }
  // Bytes from the tile's first row to a lane's chunk.
  __device__ __forceinline__ uint32_t offset(uint32_t i, bool values) const {
    const uint32_t q = slot(i, wave), r = q / R::kSlots, pc = q % R::kSlots;
    return 2u * (r * tok_s + 8u * (pc ^ (values ? R::v_swz(r) : R::k_swz(r))));
  }
  __device__ __forceinline__ uint32_t koff(uint32_t i) const { return kKeep ? kept[kKeep ? 2 * i : 0] : offset(i, false); }
  __device__ __forceinline__ uint32_t voff(uint32_t i) const { return kKeep ? kept[kKeep ? 2 * i + 1 : 0] : offset(i, true); }
  __device__ __forceinline__ void issue(const BwppCacheArgs &c, const Item &it, uint32_t k0, uint32_t first,
                                        const uint32_t *pages, uint32_t lds) const {
    if (it.once) rows<true>(c, it, k0, first, pages, lds);
    else rows<false>(c, it, k0, first, pages, lds);
  }
  template <bool ONCE>
  __device__ __forceinline__ void rows(const BwppCacheArgs &c, const Item &it, uint32_t k0, uint32_t first,
                                       const uint32_t *pages, uint32_t lds) const {
    const uint32_t pmask = (1u << c.page_shift) - 1u, n = min((uint32_t)KEYS, it.kend - k0);
    if (pmask + 1u >= (uint32_t)KEYS) {
      const uint32_t page = uni(pages[(k0 >> c.page_shift) - first]) & ~kNoPage;
      const uint64_t base = page * c.page_s + (uint64_t)(k0 & pmask) * c.tok_s;
      if (n == (uint32_t)KEYS) {
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
          if (kDma % FROM_WAVES && i * FROM_WAVES + wave >= kDma) break;
          dma16_so<ONCE>(K + base, koff(i), lds + (i * FROM_WAVES + wave) * 1024u);
          dma16_so<ONCE>(V + base, voff(i), lds + kTile + (i * FROM_WAVES + wave) * 1024u);
        }
      } else {  // rows past the last key re-read it
#pragma unroll
        for (uint32_t i = 0; i < kMine; ++i) {
          if (kDma % FROM_WAVES && i * FROM_WAVES + wave >= kDma) break;
          const uint32_t r = slot(i, wave) / R::kSlots, back = r < n ? 0u : 2u * (r - (n - 1)) * tok_s;
          dma16_so<ONCE>(K + base, koff(i) - back, lds + (i * FROM_WAVES + wave) * 1024u);
          dma16_so<ONCE>(V + base, voff(i) - back, lds + kTile + (i * FROM_WAVES + wave) * 1024u);
        }
      }
    } else {
#pragma unroll
      for (uint32_t i = 0; i < kMine; ++i) {
        if (kDma % FROM_WAVES && i * FROM_WAVES + wave >= kDma) break;
        const uint32_t r = slot(i, wave) / R::kSlots, key = k0 + min(r, n - 1);
        const uint32_t page = pages[(key >> c.page_shift) - first] & ~kNoPage;
        // less the row's offset, which koff and voff have
        const uint64_t row = (uint64_t)page * (uint32_t)c.page_s + (uint64_t)(key & pmask) * tok_s;
        const uint32_t mine = 2u * r * tok_s;
        dma16_v<ONCE>(reinterpret_cast<const char *>(K + row) + (koff(i) - mine), lds + (i * FROM_WAVES + wave) * 1024u);
        dma16_v<ONCE>(reinterpret_cast<const char *>(V + row) + (voff(i) - mine), lds + kTile + (i * FROM_WAVES + wave) * 1024u);
      }
    }
  }
};

__device__ __forceinline__ float4 scaled(const float4 &t, float f) { return make_float4(t.x * f, t.y * f, t.z * f, t.w * f); }

// Four columns of a row of the tile: to the output or, of a part, to its slot.
template <int D, uint32_t ROWS>
__device__ __forceinline__ void put(const BwppCacheAttnArgs &a, const Item &it, uint32_t slot, uint32_t row, uint32_t col,
                                    const float4 &t, float m, float l, bool head) {
  const uint32_t rr = it.tile * ROWS + row;
  if (rr >= it.R) return;
  if (!it.whole) {
    const uint64_t sr = (uint64_t)slot * ROWS + row;
    *reinterpret_cast<float4 *>(a.part_o + sr * D + col) = t;
    if (head) *reinterpret_cast<float2 *>(a.part_ml + 2 * sr) = make_float2(m, l);
    return;
  }
  const uint64_t tok = it.q.first + rr / a.group, hh = it.head * a.group + rr % a.group;
  const float4 u = scaled(t, l == 0.0f ? 0.0f : 1.0f / l);
  *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(a.o) + tok * a.o_ts + hh * a.o_hs + col) =
      make_uint2(pack_bf16x2(u.x, u.y), pack_bf16x2(u.z, u.w));
  if (head && a.lse)
    a.lse[tok * (uint64_t)(a.c.heads * a.group) + hh] = l == 0.0f ? -INFINITY : lse_of(m == -INFINITY ? 0.0f : m, l);
}

template <int D, int KB>
__device__ __forceinline__ const uint16_t *query_row(const BwppCacheAttnArgs &a, const Item &it, uint32_t row, uint32_t &tok) {
  const uint32_t r = min(row, it.R - 1u);
  tok = r / a.group;
  return static_cast<const uint16_t *>(a.q) + (uint64_t)(it.q.first + tok) * a.q_ts +
         (uint64_t)(it.head * a.group + r % a.group) * a.q_hs;
}

template <int D, int NW>
__device__ __forceinline__ void attend_few(const BwppCacheAttnArgs &a) {
  typedef Wave32<D, 1> W;
  typedef Fetch<D, 32, 1> F;
  constexpr uint32_t kStage = W::kStage, kStages = kStage * 3 <= 36864 ? 36864 / kStage : 2, kDma = 2 * F::kDma;
  constexpr uint32_t kRing = kStages * kStage, kCld = D + 4, kMerge = NW * 32 * kCld * 4;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[(NW * kRing > kMerge ? NW * kRing : kMerge) + 64];
  __shared__ uint32_t pages[kPages];
  __shared__ float mls[NW][32][2];
  const BwppCacheArgs &c = a.c;
  const uint32_t wave = uni(threadIdx.x >> 6);
  unsigned char *ring = smem + wave * kRing;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)ring;
  W w;
  w.place();
  F fetch;
  fetch.place(c, 0);

  for_items<32, 64>(a, [&](const Item &it, uint32_t slot) {
    uint32_t tok;
    const uint16_t *Q = query_row<D, 1>(a, it, it.tile * 32u + w.lq, tok);
    w.start(Q, a.scale_log2, a.flip);
    fetch.K = static_cast<const uint16_t *>(c.k) + (uint64_t)it.head * c.head_s;
    fetch.V = static_cast<const uint16_t *>(c.v) + (uint64_t)it.head * c.head_s;
    for (uint32_t seg = it.kbeg; seg < it.kend;) {
      bool bad;
      const uint32_t end = uni(load_pages<64 * NW>(c, it, seg, pages, bad)), first = seg >> c.page_shift;
      wait_vmcnt<0>();  // no load of the compiler's outstanding beside the DMA
      const uint32_t ntile = (end - seg + 31u) / 32u, mine = ntile > wave ? (ntile - wave + NW - 1) / NW : 0u;
      auto key0 = [&](uint32_t j) { return seg + 32u * (NW * j + wave); };
      auto issue = [&](uint32_t j) { fetch.issue(c, it, key0(j), first, pages, lds0 + (j % kStages) * kStage); };
#pragma unroll
      for (uint32_t j = 0; j < kStages - 1; ++j)
        if (j < mine) issue(j);
      for (uint32_t j = 0; j < mine; ++j) {
        const uint32_t k0 = key0(j), younger = min(mine - 1 - j, kStages - 2);
        if (kStages >= 4 && younger >= 2) wait_vmcnt<(kStages >= 4 ? 2 * kDma : 0)>();
        else if (kStages >= 3 && younger >= 1) wait_vmcnt<(kStages >= 3 ? kDma : 0)>();
        else wait_vmcnt<0>();
        __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0): done reading the stage that is refilled now
        if (j + kStages - 1 < mine) issue(j + kStages - 1);
        unsigned char *st = ring + uni((j % kStages) * kStage);
        uint32_t vis[1] = {~0u};
        const bool masked = bad || k0 + 32u > it.kend || k0 + 32u > it.q.held;
        if (masked) {
          if (k0 + 32u > it.q.held) {
            vis[0] = mask_bits32(a, it.q.first, tok, (int64_t)k0 - (int64_t)it.q.held);
            if (k0 < it.q.held) vis[0] |= (1u << (it.q.held - k0)) - 1u;  // fewer than 32
            wait_vmcnt<0>();  // the mask's loads
          }
          vis[0] &= keys_with_page(c, it, k0, first, pages);
        }
        f32x16_t s[1];
        w.scores(st, masked, vis, s);
        if (masked && W::odd_values(st, 0, 1)) {
          w.add_odd(st, vis, s);
          W::clear_odd(st, 0, 1);
        }
        w.template products<2>(st, s);
      }
      seg = end;
    }
    w.finish();
    // The waves' triples: O (this lane's row, column 32 d + 8 (r >> 2) + 4 lh +
    // (r & 3)) and (offset, sum).
    __syncthreads();
    float *os = reinterpret_cast<float *>(smem) + wave * (32 * kCld);
#pragma unroll
    for (int d = 0; d < W::DB; ++d)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4)
        if (32 * d + 8 * q4 + 4 * (int)w.lh < D)
          *reinterpret_cast<float4 *>(os + w.lq * kCld + 32 * d + 8 * q4 + 4 * (int)w.lh) =
              make_float4(w.o[d][4 * q4], w.o[d][4 * q4 + 1], w.o[d][4 * q4 + 2], w.o[d][4 * q4 + 3]);
    if (w.lh == 0) {
      mls[wave][w.lq][0] = w.m;
      mls[wave][w.lq][1] = w.l;
    }
    __syncthreads();
    const uint32_t rows = min(32u, it.R - it.tile * 32u);
    for (uint32_t i = threadIdx.x; i < rows * (D / 4); i += 64 * NW) {
      const uint32_t row = i / (D / 4), d4 = 4u * (i % (D / 4));
      float m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int v = 0; v < NW; ++v) m = fmaxf(m, mls[v][row][0]);
      float4 t = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int v = 0; v < NW; ++v) {
        const float mw = mls[v][row][0];
        // no key seen (offset -inf): sums of 0 (or NaN, kept)
        const float f = mw == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(mw - m);
        const float4 u = *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(smem) + (v * 32 + row) * kCld + d4);
        l += mls[v][row][1] * f;
        t.x += u.x * f, t.y += u.y * f, t.z += u.z * f, t.w += u.w * f;
      }
      put<D, 32>(a, it, slot, row, d4, t, m, l, d4 == 0);
    }
    __syncthreads();  // before the rings are filled again
  });
}

template <int D, int NW>
__device__ __forceinline__ void attend_rows(const BwppCacheAttnArgs &a) {
  constexpr int KB = 2, TERMS = D == 128 ? 1 : 2;  // of P
  constexpr uint32_t kRows = 32 * NW, kKeys = 32 * KB;
  typedef Wave32<D, KB> W;
  typedef Fetch<D, 32 * KB, NW> F;
  constexpr uint32_t kStage = W::kStage;
  __shared__ __attribute__((aligned(1024))) unsigned char smem[2 * kStage + 64];
  __shared__ uint32_t pages[kPages];
  const BwppCacheArgs &c = a.c;
  const uint32_t wave = uni(threadIdx.x >> 6);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)smem;
  W w;
  w.place();
  F fetch;
  fetch.place(c, wave);

  for_items<kRows, 64>(a, [&](const Item &it, uint32_t slot) {
    uint32_t tok;
    const uint32_t row0 = it.tile * kRows + 32u * wave;
    const uint16_t *Q = query_row<D, KB>(a, it, row0 + w.lq, tok);
    w.start(Q, a.scale_log2, a.flip);
    fetch.K = static_cast<const uint16_t *>(c.k) + (uint64_t)it.head * c.head_s;
    fetch.V = static_cast<const uint16_t *>(c.v) + (uint64_t)it.head * c.head_s;
    // Keys below `all` are seen by all of the wave's rows (`all_block`: the block's), from `none` on by none.
    const uint32_t t0 = min(row0, it.R - 1u) / a.group, t1 = min(row0 + 31u, it.R - 1u) / a.group;
    const uint32_t all = a.mask ? it.q.held : it.q.held + t0 + 1u;
    const uint32_t all_block = a.mask ? it.q.held : it.q.held + it.tile * kRows / a.group + 1u;
    const uint32_t none = row0 >= it.R ? 0u : a.mask ? it.kend : min(it.kend, it.q.held + t1 + 1u);
    for (uint32_t seg = it.kbeg; seg < it.kend;) {
      bool bad;
      const uint32_t end = uni(load_pages<64 * NW>(c, it, seg, pages, bad)), first = seg >> c.page_shift;
      wait_vmcnt<0>();  // no load of the compiler's outstanding beside the DMA
      const uint32_t ntile = (end - seg + kKeys - 1) / kKeys;
      fetch.issue(c, it, seg, first, pages, lds0);
      for (uint32_t j = 0; j < ntile; ++j) {
        const uint32_t k0 = seg + kKeys * j;
        wait_vmcnt<0>();
        __syncthreads();
        if (j + 1 < ntile) fetch.issue(c, it, k0 + kKeys, first, pages, lds0 + ((j + 1) & 1u) * kStage);
        unsigned char *st = smem + uni((j & 1u) * kStage);
        const bool none_odd = !bad && k0 + kKeys <= it.kend && k0 + kKeys <= all_block;  // the same in every wave
        const bool mine = k0 < none, masked = !none_odd && (bad || k0 + kKeys > it.kend || k0 + kKeys > all);
        uint32_t vis[KB];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) vis[kb] = ~0u;
        if (masked) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            const uint32_t k = k0 + 32u * kb;
            if (k + 32u > it.q.held) {
              vis[kb] = mask_bits32(a, it.q.first, tok, (int64_t)k - (int64_t)it.q.held);
              if (k < it.q.held) vis[kb] |= (1u << (it.q.held - k)) - 1u;  // fewer than 32
            }
            vis[kb] &= keys_with_page(c, it, k, first, pages);
          }
        }
        f32x16_t s[KB];
        if (mine) w.scores(st, masked, vis, s);
        if (!none_odd && __syncthreads_or(W::odd_values(st, wave, NW))) {
          if (mine) w.add_odd(st, vis, s);
          __syncthreads();
          W::clear_odd(st, wave, NW);
          __syncthreads();
        }
        if (mine) w.template products<TERMS>(st, s);
      }
      seg = end;
      // (the next pages' first barrier comes before any stage is filled again)
    }
    w.finish();
#pragma unroll
    for (int d = 0; d < W::DB; ++d)
#pragma unroll
      for (int q4 = 0; q4 < 4; ++q4) {
        const uint32_t col = 32u * d + 8u * q4 + 4u * w.lh;
        if (col < (uint32_t)D)
          put<D, kRows>(a, it, slot, 32u * wave + w.lq, col,
                      make_float4(w.o[d][4 * q4], w.o[d][4 * q4 + 1], w.o[d][4 * q4 + 2], w.o[d][4 * q4 + 3]), w.m, w.l,
                      d == 0 && q4 == 0 && w.lh == 0);
      }
  });
}

}  // namespace kv

#define BWPP_ATTEND_FEW(D)                                                                                  \
  extern "C" __global__ __launch_bounds__(128) void bwpp_cache_attend_few_d##D(const BwppCacheAttnArgs a) { \
    kv::attend_few<D, 2>(a);                                                                                \
  }
#define BWPP_ATTEND_ROWS(ROWS, D, NW, BLOCKS)                                                                             \
  extern "C" __global__ __launch_bounds__(64 * NW, BLOCKS) void bwpp_cache_attend_r##ROWS##_d##D(const BwppCacheAttnArgs a) { \
    kv::attend_rows<D, NW>(a);                                                                                            \
  }
BWPP_ATTEND_FEW(64)
BWPP_ATTEND_FEW(80)
BWPP_ATTEND_FEW(96)
BWPP_ATTEND_FEW(128)
BWPP_ATTEND_FEW(160)
BWPP_ATTEND_FEW(192)
BWPP_ATTEND_FEW(256)
BWPP_ATTEND_ROWS(128, 64, 4, 2)
BWPP_ATTEND_ROWS(128, 80, 4, 2)
BWPP_ATTEND_ROWS(128, 96, 4, 2)
BWPP_ATTEND_ROWS(128, 128, 4, 2)
BWPP_ATTEND_ROWS(128, 160, 4, 1)
BWPP_ATTEND_ROWS(128, 192, 4, 1)
BWPP_ATTEND_ROWS(128, 256, 4, 1)
BWPP_ATTEND_ROWS(256, 64, 8, 1)
BWPP_ATTEND_ROWS(256, 80, 8, 1)
BWPP_ATTEND_ROWS(256, 96, 8, 1)
BWPP_ATTEND_ROWS(256, 128, 8, 1)
