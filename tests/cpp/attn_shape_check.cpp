// The line of units of an attention call (attn_shape.h), walked by every CTA as the kernels walk it.
//   line  tb log2_tile window n_kv ctas cap packed rows extra join  n_seq  cu_q[n_seq + 1]  kv_len[n_seq]    prints "tiles items joined bad" or what is wrong
//   meet  a wide_a stride_a b wide_b stride_b rows                                     prints 0 or 1
//   few   max_rows g pairs                                                             prints 0 or 1
//   sizes rows n_seq n_head n_kv head_dim n_pages page_size max_pages paged            prints "ok", "invalid: ..." or "unsupported: ..."
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <set>
#include <vector>

#include "attn_shape.h"

using namespace infr;

static int line(int argc, char** argv) {
  std::vector<long long> v;
  for (int i = 2; i < argc; ++i) v.push_back(std::atoll(argv[i]));
  const int tb = (int)v[0], log2_tile = (int)v[1], window = (int)v[2], n_kv = (int)v[3], grid = (int)v[4], cap = (int)v[5], rows = (int)v[7], extra = (int)v[8], join = (int)v[9], n_seq = (int)v[10];
  const bool packed = v[6] != 0;
  const long long *cu = v.data() + 11, *kv = cu + n_seq + 1;
  struct Item {
    int s, b, head;
    AttnBlock blk;
    long long ub;
  };
  bool bad = false;
  std::vector<Item> items;
  std::set<std::pair<int, int>> written;  // (row, head)
  long long units = 0, tiles = 0;
  for (int s = 0; s < n_seq; ++s) {
    const AttnSeq q = attn_seq((int)cu[s], (int)cu[s + 1], (int)kv[s], packed, rows, cap, &bad);
    if (q.q0 < 0 || q.q_len < 0 || q.q0 + q.q_len > rows) return std::puts("rows out of range"), 1;
    for (int b = 0; b < attn_blocks(q.q_len, tb); ++b)
      for (int h = 0; h < n_kv; ++h) {
        const AttnBlock k = attn_block(q, b, tb, log2_tile, window);
        if (k.nt < 1 || k.nt > tb || k.t0 + k.nt > q.q_len || k.lo < 0 || (!packed && k.hi > cap) || (packed && k.hi > q.q_len) || k.ntile < 1)
          return std::puts("block out of range"), 1;
        // every key of every row is in the block's tiles
        for (int t = k.t0; t < k.t0 + k.nt; ++t) {
          const int pos = q.past + t, lo = window > 0 && pos - window + 1 > 0 ? pos - window + 1 : 0;
          if (pos >= 0 && (lo < k.lo || pos >= k.hi || (lo >> log2_tile) < k.tile0 || (pos >> log2_tile) >= k.tile0 + k.ntile)) return std::puts("key lost"), 1;
          written.insert({q.q0 + t, h});
        }
        items.push_back({s, b, h, k, units + extra});
        units += extra + k.ntile;
        tiles += k.ntile;
      }
  }
  int most = 0;
  for (const Item& i : items) most = i.blk.ntile + extra > most ? i.blk.ntile + extra : most;
  const int C = attn_ctas(units, grid, most, join);
  const AttnLine l = {C ? units / C : 0, C ? (int)(units % C) : 0};
  for (long long a : {units, 7 * units + 3, units / 3, (1ll << 45) + units})
    for (long long b : {units + 1, units / 2 + 5, (1ll << 30) + 3})
      if (a / b < (1 << 20) && attn_small_div(a, b) != a / b) return std::puts("small_div"), 1;
  std::map<long long, std::set<int>> slots;  // by the item's first unit
  std::map<long long, long long> covered;
  std::set<int> used;
  std::map<int, long long> counter;  // join counter -> item
  long long at = 0;
  for (int c = 0; c < C; ++c) {
    const long long u0 = attn_begin(l, c), u1 = attn_begin(l, c + 1);
    if (u0 != at || u1 <= u0) return std::puts("units not shared"), 1;
    at = u1;
    for (const Item& it : items) {
      const long long a = u0 > it.ub ? u0 : it.ub, e = u1 < it.ub + it.blk.ntile ? u1 : it.ub + it.blk.ntile;
      if (a >= e) continue;
      covered[it.ub] += e - a;
      if (attn_cta_of(l, a) != c || attn_cta_of(l, e - 1) != c) return std::puts("cta_of"), 1;
      const int first = attn_cta_of(l, it.ub), last = attn_cta_of(l, it.ub + it.blk.ntile - 1);
      if (a == it.ub && e == it.ub + it.blk.ntile) {
        if (first != c || last != c) return std::puts("a whole item is not whole"), 1;
        continue;
      }
      const int slot = 2 * c + (c == first ? 1 : 0);
      if (!used.insert(slot).second) return std::puts("slot used twice"), 1;
      slots[it.ub].insert(c);
      auto ins = counter.insert({first, it.ub});
      if (!ins.second && ins.first->second != it.ub) return std::puts("counter shared"), 1;
      if ((int)slots[it.ub].size() > last - first + 1) return std::puts("too many parts"), 1;
    }
  }
  if (units && at != units) return std::puts("units left"), 1;
  for (const Item& it : items) {
    if (covered[it.ub] != it.blk.ntile) return std::puts("tiles lost"), 1;
    const int first = attn_cta_of(l, it.ub), last = attn_cta_of(l, it.ub + it.blk.ntile - 1);
    if (slots.count(it.ub) && (int)slots[it.ub].size() != last - first + 1) return std::puts("parts missing"), 1;
  }
  std::printf("%lld %zu %zu %d\n", tiles, items.size(), slots.size(), (int)bad);
  return 0;
}

int main(int argc, char** argv) {
  if (argc > 2 && !std::strcmp(argv[1], "line")) return line(argc, argv);
  if (argc == 9 && !std::strcmp(argv[1], "meet")) {
    uint64_t x[7];
    for (int i = 0; i < 7; ++i) x[i] = std::strtoull(argv[i + 2], nullptr, 10);
    return std::printf("%d\n", attn_rows_meet(x[0], x[1], x[2], x[3], x[4], x[5], x[6])), 0;
  }
  if (argc == 5 && !std::strcmp(argv[1], "few")) return std::printf("%d\n", attn_few_rows(std::strtoull(argv[2], nullptr, 10), (uint32_t)std::atoi(argv[3]), std::strtoull(argv[4], nullptr, 10))), 0;
  if (argc != 11) return 2;
  uint32_t v[9];
  for (int i = 0; i < 9; ++i) v[i] = (uint32_t)std::strtoul(argv[i + 2], nullptr, 10);
  bool unsupported = false;
  const char* why = attn_sizes_error({v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8] != 0}, &unsupported);
  if (why) std::printf("%s: %s\n", unsupported ? "unsupported" : "invalid", why);
  else std::puts("ok");
  return 0;
}
