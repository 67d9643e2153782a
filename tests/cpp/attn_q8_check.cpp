// The sizes of pages of 8 bits (attn_shape.h).
//   bytes  n_pages page_size n_kv head_dim width                   prints attn_cache_bytes
//   unpack n_seq max_pages n_pages page_size n_kv head_dim         prints "by_sequence pages table side", or "no"
//   few    max_rows g head_dim pairs                               prints limit and 0 or 1
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "attn_shape.h"

using namespace infr;

int main(int argc, char** argv) {
  unsigned long long v[6] = {};
  if (argc < 2) return 2;
  for (int i = 2; i < argc && i < 8; ++i) v[i - 2] = std::strtoull(argv[i], nullptr, 10);
  AttnSizes s = {};
  s.paged = true;
  if (!std::strcmp(argv[1], "bytes")) {
    s.n_pages = (uint32_t)v[0], s.page_size = (uint32_t)v[1], s.n_kv = (uint32_t)v[2], s.head_dim = (uint32_t)v[3];
    std::printf("%llu\n", (unsigned long long)attn_cache_bytes(s, (uint32_t)v[4]));
  } else if (!std::strcmp(argv[1], "unpack")) {
    s.n_seq = (uint32_t)v[0], s.max_pages = (uint32_t)v[1], s.n_pages = (uint32_t)v[2], s.page_size = (uint32_t)v[3], s.n_kv = (uint32_t)v[4], s.head_dim = (uint32_t)v[5];
    AttnUnpacked u;
    if (!attn_unpacked(s, &u)) return std::puts("no"), 0;
    std::printf("%d %llu %llu %llu\n", (int)u.by_sequence, (unsigned long long)u.pages, (unsigned long long)u.table, (unsigned long long)u.side);
  } else if (!std::strcmp(argv[1], "few")) {
    std::printf("%u %d\n", attn_q8_rows_limit((uint32_t)v[2]), (int)attn_q8_few_rows(v[0], (uint32_t)v[1], (uint32_t)v[2], v[3]));
  } else {
    return 2;
  }
  return 0;
}
