// The far ends of what an attention call may be given (attn_shape.h).
//   bytes rows n_seq n_head n_kv head_dim n_pages page_size max_pages paged     prints "ok" or what is refused, and the cache's bytes
//   blocks tb rows n_seq                                     blocks counted where cu_q is 0, rows, 0, rows, ...: their number, or rows + 1; 1 where found bad
//   window past q_len tb log2_tile window most               "ok", or what a row loses of a sequence's keys at that window, as asked for and as the kernels get it
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <initializer_list>

#include "attn_shape.h"

using namespace infr;

int main(int argc, char** argv) {
  if (argc == 11 && !std::strcmp(argv[1], "bytes")) {
    uint32_t v[9];
    for (int i = 0; i < 9; ++i) v[i] = (uint32_t)std::strtoul(argv[i + 2], nullptr, 10);
    const AttnSizes s = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7], v[8] != 0};
    bool unsupported = false;
    const char* why = attn_sizes_error(s, &unsupported);
    return std::printf("%s %llu\n", why ? "refused" : "ok", why ? 0ull : (unsigned long long)attn_cache_bytes(s)), 0;
  }
  if (argc == 5 && !std::strcmp(argv[1], "blocks")) {
    const int tb = std::atoi(argv[2]), rows = std::atoi(argv[3]), n_seq = std::atoi(argv[4]);
    long long carry = 0;
    bool bad = false;
    for (int s = 0; s < n_seq; ++s) {
      carry = attn_blocks_on(carry + attn_blocks(attn_seq(s % 2 ? rows : 0, s % 2 ? 0 : rows, 0, true, rows, 0, &bad).q_len, tb), rows);
      if (carry < 0 || carry > (long long)rows + 1) return std::puts("lost count"), 1;
    }
    return std::printf("%lld %d\n", carry, (int)bad), 0;
  }
  if (argc == 8 && !std::strcmp(argv[1], "window")) {
    const int past = std::atoi(argv[2]), q_len = std::atoi(argv[3]), tb = std::atoi(argv[4]), log2_tile = std::atoi(argv[5]);
    const long long asked = std::atoll(argv[6]);
    const AttnSeq s = {0, q_len, past};
    for (int window : {(int)asked, attn_window((uint32_t)asked, (uint32_t)std::strtoul(argv[7], nullptr, 10))})
      for (int b = 0; b < attn_blocks(q_len, tb); ++b) {
        const AttnBlock k = attn_block(s, b, tb, log2_tile, window);
        const int full_lo = attn_full_lo(s, k, window), full_hi = attn_full_hi(s, k);
        if (k.lo < 0 || k.lo > k.hi || k.ntile < 1 || full_lo < 0) return std::puts("block"), 0;
        for (int t = k.t0; t < k.t0 + k.nt; ++t) {
          const long long pos = (long long)past + t, lo = asked > 0 && pos - asked + 1 > 0 ? pos - asked + 1 : 0;
          if (pos < 0) continue;
          if (lo != attn_first_key((int)pos, window)) return std::puts("first key"), 0;
          if (lo < k.lo || pos >= k.hi || (lo >> log2_tile) < k.tile0 || (pos >> log2_tile) >= k.tile0 + k.ntile) return std::puts("key lost"), 0;
          if (full_lo < lo || full_hi > pos + 1) return std::puts("hidden key taken for seen"), 0;
        }
      }
    return std::puts("ok"), 0;
  }
  return 2;
}
