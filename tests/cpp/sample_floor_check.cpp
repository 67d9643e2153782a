// Which logits of a row have a weight (sample_shape.h): reads "top temperature" pairs as f32 bits, prints the floor's.
#include <cstdint>
#include <cstdio>
#include <cstring>

#include "sample_shape.h"

int main() {
  unsigned a, b;
  while (std::scanf("%x %x", &a, &b) == 2) {
    float top, t;
    std::memcpy(&top, &a, 4);
    std::memcpy(&t, &b, 4);
    const float f = infr::sample_floor(top, t);
    uint32_t u;
    std::memcpy(&u, &f, 4);
    std::printf("%08x\n", u);
  }
  return 0;
}
