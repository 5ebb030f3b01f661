// Who computes what in the attention over a paged cache.
//
// Lengths lie in device memory and differ from sequence to sequence, so the
// work is shared out on the device: a fixed number of blocks, whatever the
// lengths, and a captured launch follows the lengths of its replay.  An item is
// a tile of ROWS query rows of one (sequence, key head) with all the keys that
// it sees, in units of UNIT keys.  Items stand in the order of sequences, heads
// and tiles, each with a cost: its keys (of a causal tile up to its last
// token) and item_keys more for what an item costs by itself.  Block b of G takes
// what lies between the costs W b / G and W (b + 1) / G of the total W, rounded
// to whole units.  An item whose keys fall to several blocks is left by each
// as a triple (exponent offset, sum of p, sum of p v) and joined by a second
// launch: the sharer where it begins leaves it in slot 2 b + 1, the others,
// for which it is the first item, in slot 2 b.  Where all sequences are short
// items are left whole, since parts cost more than an even share gains (and
// where the table's width says so, there is no second launch).  The sharers of
// one XCD are neighbours: the tiles of a head meet its keys in one L2.  Finding
// the share takes a block 2.4 us, its first pages and rows of q as much (8 trees
// of 48 tokens over up to 16384, tiles of 256 rows: of 54 us 33 are key tiles).
//
// Costs are whole numbers below 2^52, g times keys (g query heads a key head);
// quotients are taken in doubles (64-bit integer ones cost a microsecond
// here), the same in every block, so a sharer and its successor find the same
// border.  Only starts that descend can bring more, up to 2^62: then quotients
// may be off, and are cut to what there is.
#pragma once

#include "kv_cache.h"

namespace kv {

constexpr uint32_t kLeast = 64;  // a block's share is at least as many keys

// A place in the order of the work.
struct Place {
  uint32_t s, head, tile, unit;
};
__device__ __forceinline__ bool earlier(const Place &a, const Place &b) {
  if (a.s != b.s) return a.s < b.s;
  if (a.head != b.head) return a.head < b.head;
  return a.tile != b.tile ? a.tile < b.tile : a.unit < b.unit;
}
struct Share {
  Place from, to;
  Seq q;       // from's sequence
  uint32_t b;  // whose it is
  bool large;  // the sequences' keys and values are more than the caches hold
};

template <uint32_t ROWS, uint32_t UNIT>
struct Work {
  static __device__ __forceinline__ uint32_t tiles(const Seq &q, uint32_t g) { return (q.n * g + ROWS - 1) / ROWS; }
  static __device__ __forceinline__ uint64_t before(const BwppCacheAttnArgs &a, const Seq &q, uint64_t t) {  // cost of tiles 0 .. t - 1
    return t * ((uint64_t)a.group * (q.held + a.item_keys)) + ROWS * (t * (t + 1) / 2);
  }
  // Keys that a tile may see.
  static __device__ __forceinline__ uint32_t keys(const BwppCacheAttnArgs &a, const Seq &q, uint32_t tile) {
    const uint32_t g = a.group;
    const uint32_t last = a.mask ? q.n : (min((tile + 1) * ROWS, q.n * g) - 1) / g + 1;
    return min(q.held + last, a.c.capacity);
  }
  static __device__ __forceinline__ uint32_t units(const BwppCacheAttnArgs &a, const Seq &q, uint32_t tile) {
    return (keys(a, q, tile) + UNIT - 1) / UNIT;
  }
  // Where cost x of sequence s (all its heads) falls, and the costs where that
  // item begins and ends.
  static __device__ __forceinline__ Place find(const BwppCacheAttnArgs &a, bool whole, uint32_t s, const Seq &q, uint64_t x,
                                               uint64_t &begin, uint64_t &end) {
    const uint32_t T = tiles(q, a.group);
    const uint64_t head_cost = before(a, q, T);
    uint32_t head = min((uint32_t)((double)x / (double)head_cost), a.c.heads - 1u);
    if (head * head_cost > x) --head;  // (a quotient rounded up)
    const uint64_t rest = x - head * head_cost;
    uint32_t lo = 0, hi = T;  // before(lo) <= rest < before(hi)
    while (hi - lo > 1) {
      const uint32_t m = (lo + hi) / 2;
      if (before(a, q, m) <= rest) lo = m;
      else hi = m;
    }
    const uint64_t b0 = before(a, q, lo), b1 = before(a, q, lo + 1);
    begin = head * head_cost + b0;
    end = head * head_cost + b1;
    return {s, head, lo, whole ? 0u : unit(a, q, lo, rest - b0, b1 - b0)};
  }
  static __device__ __forceinline__ uint32_t unit(const BwppCacheAttnArgs &a, const Seq &q, uint32_t tile, uint64_t off,
                                                  uint64_t cost) {
    const uint32_t n = units(a, q, tile), u = (uint32_t)((double)off * (double)n / (double)cost);
    return min(u, n ? n - 1u : 0u);
  }
};

__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 | lo;
}

// Costs of all sequences, in every wave by itself (no barrier: a short call is
// a chain of latencies): a lane adds up a run of `per` sequences.
template <uint32_t ROWS, uint32_t UNIT>
struct Costs {
  uint32_t per;
  Seq q;           // of the lane's first sequence
  uint64_t first;  // costs before the lane's
  uint64_t mine, total;
  bool whole;      // every sequence is so short that its items are not shared

  static __device__ __forceinline__ uint64_t of(const BwppCacheAttnArgs &a, const Seq &q) {
    return a.c.heads * Work<ROWS, UNIT>::before(a, q, Work<ROWS, UNIT>::tiles(q, a.group));
  }
  // Keys of a sequence that its table holds: a table of at most whole_keys slots
  // leaves every item whole, and such a call has no workspace for parts.
  static __device__ __forceinline__ uint32_t keys_of(const BwppCacheAttnArgs &a, const Seq &q) {
    return q.n ? min(q.held + q.n, a.c.capacity) : 0u;
  }
  __device__ __forceinline__ Costs(const BwppCacheAttnArgs &a) {
    const uint32_t lane = threadIdx.x & 63u;
    per = (a.c.batch + 63u) / 64u;
    const uint32_t s0 = min(lane * per, a.c.batch), s1 = min(s0 + per, a.c.batch);
    q = {0, 0, 0};
    if (s0 < s1) q = seq_at(a.c, s0);
    mine = of(a, q);
    uint32_t most = keys_of(a, q);
#pragma unroll 4
    for (uint32_t s = s0 + 1; s < s1; ++s) {
      const Seq t = seq_at(a.c, s);
      mine += of(a, t);
      most = max(most, keys_of(a, t));
    }
    whole = __ballot(most > a.whole_keys) == 0;
    uint64_t sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const uint64_t up = __shfl_up(sum, d, 64);
      if (lane >= (uint32_t)d) sum += up;
    }
    first = sum - mine;
    total = lane_of(sum, 63);
  }
  // The sequence of cost x < total, and the costs before it.
  __device__ __forceinline__ uint32_t at(const BwppCacheAttnArgs &a, uint64_t x, Seq &at, uint64_t &begin) const {
    const int lane = __builtin_ctzll(__ballot(x >= first && x - first < mine));
    uint32_t s = (uint32_t)lane * per;
    begin = lane_of(first, lane);
    at = {(uint32_t)__builtin_amdgcn_readlane((int)q.first, lane), (uint32_t)__builtin_amdgcn_readlane((int)q.n, lane),
          (uint32_t)__builtin_amdgcn_readlane((int)q.held, lane)};
    for (uint64_t c = of(a, at); x - begin >= c; c = of(a, at)) {
      begin += c;
      at = seq_at(a.c, ++s);  // (the run's last sequence ends past x)
    }
    return s;
  }
};

// The share of a total cost: as much for each block, kLeast at least.
__device__ __forceinline__ uint64_t share_of(const BwppCacheAttnArgs &a, uint64_t total) {
  const uint64_t even = (uint64_t)((double)total * a.inv_blocks) + 1, least = (uint64_t)a.group * kLeast;
  return even < least ? least : even;
}

// The share of this block.
template <uint32_t ROWS, uint32_t UNIT>
__device__ __forceinline__ Share find_share(const BwppCacheAttnArgs &a) {
  typedef Work<ROWS, UNIT> W;
  constexpr uint32_t kXcds = 8;  // blocks go to them in turn
  const Costs<ROWS, UNIT> costs(a);
  const uint64_t S = share_of(a, costs.total);
  const uint32_t sharers = min((uint32_t)((double)costs.total / (double)S) + 1u, a.blocks), per = (sharers + kXcds - 1) / kXcds;
  Share share = {{a.c.batch, 0, 0, 0}, {a.c.batch, 0, 0, 0}, {0, 0, 0}, blockIdx.x % kXcds * per + blockIdx.x / kXcds,
                 costs.total > a.large_cost};
  const uint64_t x0 = S * share.b, x1 = x0 + S;
  if (blockIdx.x / kXcds >= per || x0 >= costs.total) return share;
  uint64_t begin, end, before;
  uint32_t s = costs.at(a, x0, share.q, before);
  share.from = W::find(a, costs.whole, s, share.q, x0 - before, begin, end);
  if (x1 < costs.total) {
    Seq q;
    s = costs.at(a, x1, q, before);
    share.to = W::find(a, costs.whole, s, q, x1 - before, begin, end);
  }
  return share;
}

}  // namespace kv
