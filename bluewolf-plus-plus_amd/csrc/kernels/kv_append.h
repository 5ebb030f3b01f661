// New tokens into a paged cache: q and k turned by their positions (the
// rotation of rotary.h), k and v written to their pages, q to its output; and
// the accepted tokens of a drafted tree moved together.
//
// Append is bound by HBM: a row is read and written once, cosines and sines are
// made once a tile of tokens, whose sequences are found by bisection over starts
// sampled in LDS (four prompts of up to 4096 tokens, 32 : 8 heads of 128, bf16:
// 48 us, 4.7 TB/s; a copy reaches 5.15).  Few tokens have a block for each eight
// heads, and cost a launch and a chain of latencies (8 tokens 6.8 us); so does
// keep (64 sequences, 6 of 48 tokens: 6.4 us).
#pragma once

#include "common.h"
#include "kv_cache.h"
#include "rotary_math.h"
#include "../kargs.h"

using namespace bwpp;

namespace kv {

constexpr int kMaxAngles = 2048;  // (token, pair) angles of a block: 16 KiB of LDS
constexpr int kMaxTile = 64;      // tokens of a block
constexpr int kSamples = 256;     // starts of sequences in LDS

// Sequence of row t: the last one that starts at or before it.
__device__ __forceinline__ uint32_t find_seq(const BwppCacheArgs &c, const uint32_t *samples, uint32_t step, uint32_t t) {
  uint32_t lo = 0, hi = (c.batch + step - 1) / step;  // samples[lo] <= t (or lo = 0), samples[hi] > t
  while (hi - lo > 1) {
    const uint32_t m = (lo + hi) / 2;
    if (samples[m] <= t) lo = m;
    else hi = m;
  }
  lo *= step;
  hi = min(lo + step, c.batch);
  while (hi - lo > 1) {
    const uint32_t m = (lo + hi) / 2;
    if (start_at(c, m) <= t) lo = m;
    else hi = m;
  }
  return lo;
}

// A block takes a tile of tokens and a group of the rows of a token: q's
// heads, k's, v's.
template <class T, bool INTER, int C>
__device__ __forceinline__ void append(const BwppCacheAppendArgs &a) {
  using namespace rotary_pos;
  const BwppRotaryArgs &r = a.r;
  const BwppCacheArgs &c = a.c;
  __shared__ float2 cs[kMaxAngles];
  __shared__ uint64_t place[kMaxTile];  // in the pools
  __shared__ int64_t pos[kMaxTile];
  __shared__ uint32_t live[kMaxTile];
  __shared__ uint32_t samples[kSamples];
  const uint32_t tid = threadIdx.x, NT = 256;
  const uint32_t t0 = blockIdx.x * r.tile, nt = min(r.tile, c.tokens - t0);
  const uint32_t h0 = blockIdx.y * r.hgroup, nh = min(r.hgroup, r.heads - h0);

  const uint32_t step = (c.batch + kSamples - 1) / kSamples;
  if ((uint64_t)tid * step < c.batch) samples[tid] = start_at(c, tid * step);
  __syncthreads();
  if (tid < nt) {
    const uint32_t t = t0 + tid, s = find_seq(c, samples, step, t);
    const Seq q = seq_at(c, s);
    const bool in = t >= q.first && t - q.first < q.n;
    const int32_t held = c.held[s];  // not cut to the table: the position goes on past it
    const uint64_t slot = (uint64_t)(held < 0 ? 0 : held) + (t - q.first);
    live[tid] = in;
    place[tid] = in ? slot_row(c, s, slot) : kNoSlot;
    pos[tid] = r.positions ? (int64_t)r.positions[t] : (int64_t)slot;
  }
  __syncthreads();

  // Angles: a thread keeps its pair and walks the tokens.
  if (r.pairs && h0 < r.heads - c.heads) {
    const uint32_t per = r.pairs < NT ? NT / r.pairs : 1u;  // tokens side by side
    if (tid < per * r.pairs || r.pairs >= NT) {
      for (uint32_t i = r.pairs < NT ? tid % r.pairs : tid; i < r.pairs; i += NT) {
        const double f = quarter_turns(r, i);
        for (uint32_t t = r.pairs < NT ? tid / r.pairs : 0u; t < nt; t += per)
          cs[t * r.pairs + i] = cos_sin(r, (double)pos[t] * f);
      }
    }
    __syncthreads();
  }

  const uint32_t chunks = r.pairs / C + r.tail_chunks;
  const uint32_t rows = nt * nh;
  const uint32_t magic = 0xffffffffu / nh + 1u;  // row / nh by a multiply: rows * nh < 2^32 (nh <= 256)
  const uint32_t side = chunks < NT ? NT / chunks : 1u;  // rows side by side
  if (chunks < NT && tid >= side * chunks) return;
  for (uint32_t ch = chunks < NT ? tid % chunks : tid; ch < chunks; ch += NT) {
    for (uint32_t row = chunks < NT ? tid / chunks : 0u; row < rows; row += side) {
      const uint32_t t = nh > 1 ? __umulhi(row, magic) : row;
      const uint32_t hd = h0 + (row - t * nh);
      const uint64_t tok = t0 + t;
      const bool isq = hd < r.q_heads, isv = hd >= r.heads - c.heads;
      if (!live[t] || (!isq && place[t] == kNoSlot)) continue;
      const T *src;
      T *dst;
      if (isq) {
        src = static_cast<const T *>(r.q) + (tok * r.q_ts + (uint64_t)hd * r.q_hs);
        dst = static_cast<T *>(r.qo) + (tok * r.qo_ts + (uint64_t)hd * r.qo_hs);
      } else {
        const uint64_t hh = isv ? hd - (r.heads - c.heads) : hd - r.q_heads;
        src = isv ? static_cast<const T *>(a.v_in) + (tok * a.v_ts + hh * a.v_hs)
                  : static_cast<const T *>(r.k) + (tok * r.k_ts + hh * r.k_hs);
        dst = static_cast<T *>(isv ? c.v : c.k) + (place[t] + hh * c.head_s);
      }
      if (ch >= r.pairs / C) {  // columns that are not rotated
        if (isq && !r.copy) continue;
        const uint32_t c0 = 2 * r.pairs + (ch - r.pairs / C) * C;
        if (c0 + C <= r.dim) copy_row<T, C>(src + c0, dst + c0);
        else
          for (uint32_t e = c0; e < r.dim; ++e) dst[e] = src[e];
        continue;
      }
      if (isv) {
        if constexpr (INTER) {
          copy_row<T, 2 * C>(src + 2 * ch * C, dst + 2 * ch * C);
        } else {
          copy_row<T, C>(src + ch * C, dst + ch * C);
          copy_row<T, C>(src + r.pairs + ch * C, dst + r.pairs + ch * C);
        }
        continue;
      }
      const float2 *ang = cs + t * r.pairs + ch * C;
      if constexpr (INTER) {
        float v[2 * C], o[2 * C];
        Vec<T, 2 * C>::load(src + 2 * ch * C, v);
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const float2 w = ang[e];
          o[2 * e] = v[2 * e] * w.x - v[2 * e + 1] * w.y;
          o[2 * e + 1] = v[2 * e + 1] * w.x + v[2 * e] * w.y;
        }
        Vec<T, 2 * C>::store(dst + 2 * ch * C, o);
      } else {
        float x[C], y[C], u[C], v[C];
        Vec<T, C>::load(src + ch * C, x);
        Vec<T, C>::load(src + r.pairs + ch * C, y);
#pragma unroll
        for (int e = 0; e < C; ++e) {
          const float2 w = ang[e];
          u[e] = x[e] * w.x - y[e] * w.y;
          v[e] = y[e] * w.x + x[e] * w.y;
        }
        Vec<T, C>::store(dst + ch * C, u);
        Vec<T, C>::store(dst + r.pairs + ch * C, v);
      }
    }
  }
}

// Slot held + i of a sequence takes what lies at held + kept[i].  A thread owns
// a chunk of one head's keys or values and reads kRound of its rows before it
// writes any, so within a round the order of kept does not matter; in later
// rounds an entry must not be below its index (then no row is overwritten
// before it is read).
template <class U>
__device__ __forceinline__ void keep(const BwppCacheKeepArgs &a) {
  constexpr uint32_t kRound = 16;
  const BwppCacheArgs &c = a.c;
  __shared__ uint64_t from[kRound], to[kRound];
  const uint32_t s = blockIdx.x;
  const int32_t h = c.held[s], cnt = a.counts[s];
  const uint32_t held = h < 0 ? 0u : min((uint32_t)h, c.capacity);
  const uint32_t n = cnt < 0 ? 0u : min((uint32_t)cnt, a.max_kept);
  const uint32_t item = blockIdx.y * blockDim.x + threadIdx.x, per = c.heads * a.chunks;
  const bool mine = item < 2 * per;
  const uint32_t which = item >= per, rest = which ? item - per : item;
  U *pool = reinterpret_cast<U *>(which ? c.v : c.k);
  const uint64_t col = ((uint64_t)(rest / a.chunks) * c.head_s) / a.unit + rest % a.chunks;
  for (uint32_t i0 = 0; i0 < n; i0 += kRound) {
    __syncthreads();
    if (threadIdx.x < kRound) {
      const uint32_t i = i0 + threadIdx.x;
      uint64_t f = kNoSlot, t = kNoSlot;
      if (i < n) {
        const int32_t k = a.kept[(uint64_t)s * a.ld_kept + i];
        if (k >= 0 && (uint32_t)k != i) {
          f = slot_row(c, s, (uint64_t)held + (uint32_t)k);
          t = slot_row(c, s, (uint64_t)held + i);
        }
      }
      if (f == kNoSlot || t == kNoSlot) f = t = kNoSlot;
      from[threadIdx.x] = f == kNoSlot ? f : f / a.unit;
      to[threadIdx.x] = t == kNoSlot ? t : t / a.unit;
    }
    __syncthreads();
    if (!mine) continue;
    U v[kRound];
#pragma unroll
    for (uint32_t i = 0; i < kRound; ++i)
      v[i] = from[i] != kNoSlot ? pool[from[i] + col] : U{};
#pragma unroll
    for (uint32_t i = 0; i < kRound; ++i)
      if (to[i] != kNoSlot) pool[to[i] + col] = v[i];
  }
}

}  // namespace kv

#define BWPP_APPEND(NAME, T, INTER, C)                                                             \
  extern "C" __global__ __launch_bounds__(256) void bwpp_cache_append_##NAME(const BwppCacheAppendArgs a) { \
    kv::append<T, INTER, C>(a);                                                                    \
  }
BWPP_APPEND(bf16_half_8, uint16_t, false, 8)
BWPP_APPEND(bf16_half_4, uint16_t, false, 4)
BWPP_APPEND(bf16_half_1, uint16_t, false, 1)
BWPP_APPEND(bf16_inter_8, uint16_t, true, 8)
BWPP_APPEND(bf16_inter_4, uint16_t, true, 4)
BWPP_APPEND(bf16_inter_1, uint16_t, true, 1)
BWPP_APPEND(f32_half_4, float, false, 4)
BWPP_APPEND(f32_half_1, float, false, 1)
BWPP_APPEND(f32_inter_4, float, true, 4)
BWPP_APPEND(f32_inter_1, float, true, 1)

#define BWPP_KEEP(NAME, U) \
  extern "C" __global__ __launch_bounds__(256) void bwpp_cache_keep_##NAME(const BwppCacheKeepArgs a) { kv::keep<U>(a); }
BWPP_KEEP(16, uint4)
BWPP_KEEP(4, uint32_t)
BWPP_KEEP(2, uint16_t)
