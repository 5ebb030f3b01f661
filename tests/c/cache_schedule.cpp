// Who computes what in the attention over a paged cache (kv_schedule.h,
// kv_items.h), block by block on the host.
//
//   cache_schedule rows blocks whole_keys item_keys group heads page_shift max_pages mask
//                  held:new held:new ...
//
// Follows every block's share and prints "items N divided M"; ends with status 1
// where an item's keys are not all taken, once each, where two parts lie in one
// slot or a part in no block's, or where blocks divide an item although the table
// is too narrow for the workspace that its parts need.
#include "kv_items.h"

#include <algorithm>
#include <map>
#include <tuple>

namespace {

struct Part {
  uint32_t kbeg, kend, slot;
  bool whole;
};

int wrong(const char *what, uint32_t s, uint32_t head, uint32_t tile) {
  printf("sequence %u head %u tile %u: %s\n", s, head, tile, what);
  return 1;
}

template <uint32_t ROWS>
int follow(const BwppCacheAttnArgs &a) {
  std::map<std::tuple<uint32_t, uint32_t, uint32_t>, std::vector<Part>> items;
  for (uint32_t b = 0; b < a.blocks; ++b)
    host_wave::run(b, [&] {
      kv::for_items<ROWS, 64>(a, [&](const kv::Item &it, uint32_t slot) {
        if (threadIdx.x == 0) items[{it.s, it.head, it.tile}].push_back({it.kbeg, it.kend, slot, it.whole});
      });
    });
  size_t expected = 0, divided = 0;
  std::map<uint32_t, int> slots;
  for (uint32_t s = 0; s < a.c.batch; ++s) {
    const kv::Seq q = kv::seq_at(a.c, s);
    for (uint32_t head = 0; head < a.c.heads; ++head)
      for (uint32_t tile = 0; tile < kv::Work<ROWS, 64>::tiles(q, a.group); ++tile, ++expected) {
        auto found = items.find({s, head, tile});
        if (found == items.end()) return wrong("nobody's", s, head, tile);
        std::vector<Part> &parts = found->second;
        std::sort(parts.begin(), parts.end(), [](const Part &x, const Part &y) {
          return x.kbeg != y.kbeg ? x.kbeg < y.kbeg : x.kend < y.kend;
        });
        const uint32_t keys = kv::Work<ROWS, 64>::keys(a, q, tile);
        uint32_t at = 0;
        for (const Part &p : parts) {
          if (p.kbeg != at) return wrong("keys that nobody or two blocks take", s, head, tile);
          at = p.kend;
          if (p.whole != (parts.size() == 1)) return wrong("a part that is taken for a whole", s, head, tile);
          if (!p.whole && (p.slot >= 2 * a.blocks || slots[p.slot]++)) return wrong("slot of a part", s, head, tile);
        }
        if (at != keys) return wrong("keys left", s, head, tile);
        if (parts.size() > 1) ++divided;
      }
  }
  if (items.size() != expected) return wrong("items that no sequence has", 0, 0, 0);
  printf("items %zu divided %zu\n", expected, divided);
  if (divided && a.c.capacity <= a.whole_keys) return wrong("divided, and the call has no workspace", 0, 0, 0);
  return 0;
}

}  // namespace

int main(int argc, char **argv) {
  if (argc < 11) return 2;
  auto num = [&](int i) { return (uint32_t)strtoul(argv[i], nullptr, 10); };
  const uint32_t rows = num(1);
  BwppCacheAttnArgs a = {};
  a.blocks = num(2);
  a.inv_blocks = 1.0 / a.blocks;
  a.whole_keys = num(3);
  a.item_keys = num(4);
  a.group = num(5);
  a.c.heads = num(6);
  a.c.page_shift = num(7);
  const uint64_t slots = (uint64_t)num(8) << a.c.page_shift;
  a.c.capacity = (uint32_t)std::min<uint64_t>(slots, 0x7fffffffu);
  const uint32_t some_mask = 0;
  a.mask = num(9) ? &some_mask : nullptr;  // (not read: whether there is one decides which keys a tile has)
  a.large_cost = ~0ull;
  std::vector<int32_t> held, starts = {0};
  for (int i = 10; i < argc; ++i) {
    char *end;
    held.push_back((int32_t)strtol(argv[i], &end, 10));
    starts.push_back(starts.back() + (int32_t)strtol(end + 1, nullptr, 10));
  }
  a.c.held = held.data();
  a.c.starts = starts.data();
  a.c.batch = (uint32_t)held.size();
  a.c.tokens = (uint32_t)starts.back();
  switch (rows) {
    case 16: return follow<16>(a);
    case 32: return follow<32>(a);
    case 128: return follow<128>(a);
    case 256: return follow<256>(a);
  }
  return 2;
}
