// A paged cache of keys and values, as the kernels that write and read it see
// it.  Sequence s holds held[s] tokens; its new tokens are rows starts[s] ..
// starts[s + 1] - 1 of the batch's operands and take the slots behind them.
// Slot p lies in page table[s][p / page_tokens] at place p % page_tokens.
//
// Lengths, starts and page numbers come from device memory and may hold
// anything: starts and lengths are cut to the operands and the table, and a
// slot whose page number lies outside the pool does not exist (nothing is
// written there, no query sees it).  So no value makes a kernel leave its
// operands.
#pragma once

#include "common.h"
#include "../kargs.h"

using namespace bwpp;

namespace kv {

constexpr uint64_t kNoSlot = ~0ull;

struct Seq {
  uint32_t first, n, held;
};

__device__ __forceinline__ uint32_t start_at(const BwppCacheArgs &c, uint32_t i) {
  const int32_t v = c.starts[i];
  return v < 0 ? 0u : min((uint32_t)v, c.tokens);
}

__device__ __forceinline__ Seq seq_at(const BwppCacheArgs &c, uint32_t s) {
  const uint32_t a = start_at(c, s), b = start_at(c, s + 1);
  const int32_t h = c.held[s];
  return {a, b > a ? b - a : 0u, h < 0 ? 0u : min((uint32_t)h, c.capacity)};
}

// Page number of a slot of sequence s (any 32 bits), slot < capacity.
__device__ __forceinline__ uint32_t page_of(const BwppCacheArgs &c, uint32_t s, uint32_t slot) {
  return (uint32_t)c.table[(uint64_t)s * c.ld_table + (slot >> c.page_shift)];
}

// First element of head 0's row at a slot of that page, kNoSlot outside the pool.
__device__ __forceinline__ uint64_t row_at(const BwppCacheArgs &c, uint32_t page, uint32_t slot) {
  if (page >= c.pages) return kNoSlot;
  return (uint64_t)page * c.page_s + (uint64_t)(slot & ((1u << c.page_shift) - 1u)) * c.tok_s;
}

__device__ __forceinline__ uint64_t slot_row(const BwppCacheArgs &c, uint32_t s, uint64_t slot) {
  if (slot >= c.capacity || c.pages == 0) return kNoSlot;  // (without pages there may be no table)
  return row_at(c, page_of(c, s, (uint32_t)slot), (uint32_t)slot);
}

}  // namespace kv
