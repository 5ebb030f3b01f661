// A block's items of the attention over a paged cache, their page numbers and
// masks.
#pragma once

#include "kv_cache.h"
#include "kv_schedule.h"
#include "../kargs.h"

namespace kv {

__device__ __forceinline__ uint32_t uni(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// 32 bits: which of the sequence's new tokens j0 .. j0 + 31 its token i sees
// (those below zero: none).
__device__ __forceinline__ uint32_t mask_bits32(const BwppCacheAttnArgs &a, uint32_t first, uint32_t i, int64_t j0) {
  if (!a.mask) {
    const int64_t seen = (int64_t)i + 1 - j0;
    return seen <= 0 ? 0u : seen >= 32 ? ~0u : (1u << seen) - 1u;
  }
  uint64_t two = 0;
  const uint32_t *row = a.mask + (uint64_t)(first + i) * a.mask_words;
  const int64_t w = j0 >> 5;
  if (w >= 0 && w < (int64_t)a.mask_words) two = row[w];
  if (w + 1 >= 0 && w + 1 < (int64_t)a.mask_words) two |= (uint64_t)row[w + 1] << 32;
  return (uint32_t)(two >> (j0 & 31));
}

constexpr uint32_t kPages = 1024;          // page numbers in LDS
constexpr uint32_t kNoPage = 0x80000000u;  // outside the pool: page 0 is read, and not seen

// An item as a wave sees it.
struct Item {
  Seq q;
  uint32_t s, head, tile, kbeg, kend, R;
  bool whole;
  bool once;  // its keys and values are read by no other tile, and of more than the caches hold
};

// Page numbers of the keys from k on, as many as LDS holds; returns the end of
// these keys (a multiple of the tiles, or kend) and whether some have no page.
// Every thread of the block calls it.
template <uint32_t THREADS>
__device__ __forceinline__ uint32_t load_pages(const BwppCacheArgs &c, const Item &it, uint32_t k, uint32_t *pages, bool &bad) {
  const uint32_t first = k >> c.page_shift, n = min(kPages, ((it.kend - 1) >> c.page_shift) - first + 1);
  const int32_t *table = c.table + (uint64_t)it.s * c.ld_table + first;
  int none = 0;
  uint32_t p = threadIdx.x < n ? (uint32_t)table[threadIdx.x] : 0u;  // under way with the query rows
  __syncthreads();  // done with the last ones
  for (uint32_t i = threadIdx.x; i < n;) {
    none |= p >= c.pages;
    pages[i] = p < c.pages ? p : kNoPage;
    i += THREADS;
    if (i < n) p = (uint32_t)table[i];
  }
  bad = __syncthreads_or(none) != 0;
  const uint64_t end = (uint64_t)(first + n) << c.page_shift;
  return (uint32_t)min(end, (uint64_t)it.kend);
}

// Which of the keys k0 .. k0 + 31 lie in a page (of those below kend), the same in every lane.
__device__ __forceinline__ uint32_t keys_with_page(const BwppCacheArgs &c, const Item &it, uint32_t k0, uint32_t first,
                                                   const uint32_t *pages) {
  const uint32_t k = k0 + (threadIdx.x & 31u);
  const bool ok = k < it.kend && !(pages[(min(k, it.kend - 1) >> c.page_shift) - first] & kNoPage);
  return (uint32_t)__ballot(ok);
}

// Walks a block's share: f(item, slot of its part).
template <uint32_t ROWS, uint32_t UNIT, class F>
__device__ __forceinline__ void for_items(const BwppCacheAttnArgs &a, F f) {
  typedef Work<ROWS, UNIT> W;
  const Share share = find_share<ROWS, UNIT>(a);
  const uint32_t b = uni(share.b), large = uni(share.large);
  Place at = {uni(share.from.s), uni(share.from.head), uni(share.from.tile), uni(share.from.unit)};
  const Place to = {uni(share.to.s), uni(share.to.head), uni(share.to.tile), uni(share.to.unit)};
  Item it = {};
  auto sequence = [&](const Seq &q) {
    it.q = {uni(q.first), uni(q.n), uni(q.held)};
    it.s = at.s;
    it.R = it.q.n * a.group;
    it.once = large && it.R <= ROWS;
  };
  sequence(share.q);
  // A part of an item that began in another block is written even if it has no
  // keys: the join reads it.
  bool part = at.unit != 0;
  for (; part || earlier(at, to); part = false) {
    const bool same = at.s == to.s && at.head == to.head && at.tile == to.tile;
    const uint32_t keys = W::keys(a, it.q, at.tile), total = (keys + UNIT - 1) / UNIT, u1 = same ? to.unit : total;
    it.head = at.head;
    it.tile = at.tile;
    it.whole = at.unit == 0 && u1 == total;
    it.kbeg = at.unit * UNIT;
    it.kend = min(u1 * UNIT, keys);
    f(it, 2u * b + (at.unit == 0 ? 1u : 0u));
    at.unit = 0;
    if (++at.tile >= W::tiles(it.q, a.group)) {
      at.tile = 0;
      if (++at.head >= a.c.heads) {
        at.head = 0;
        do {
          ++at.s;
          if (at.s >= a.c.batch) break;
          sequence(seq_at(a.c, at.s));
        } while (it.q.n == 0);
      }
    }
  }
}

}  // namespace kv
