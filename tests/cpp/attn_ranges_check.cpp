// The far ends of what an attention call may be given (attn_shape.h).
//   bytes rows n_seq n_head n_kv head_dim n_pages page_size max_pages paged     prints "ok" or what is refused, and the cache's bytes
#include <cstdio>
#include <cstdlib>
#include <cstring>

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
  return 2;
}
