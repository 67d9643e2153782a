// Which logits of a row have a weight: numbers that the sampler (sample.cu) and a host program agree on.
#pragma once
#include <math.h>

#ifdef __CUDACC__
#define INFR_SAMPLE_HD __host__ __device__ inline
#else
#define INFR_SAMPLE_HD inline
#endif

namespace infr {

constexpr double SAMPLE_REACH = 45.0;  // weights down to e^-45, a little below 2^-64

// The least f32 number from which on a logit is at most SAMPLE_REACH temperatures below the largest, `top`.  Rounded up, so that no number below that is among
// them: where a step of f32 at `top` is many temperatures, the next one below it is thousands of octaves down, past what a weight's exponent holds.
// (An infinite largest value leaves those like it.)
INFR_SAMPLE_HD float sample_floor(float top, float temperature) {
  if (top > 3.402823466e38f) return top;
  const double reach = (double)top - SAMPLE_REACH * (double)temperature;
  if (!(reach > -3.402823466e38)) return -3.402823466e38f;
  const float near = (float)reach;
  return (double)near < reach ? nextafterf(near, 3.402823466e38f) : near;
}

}  // namespace infr
