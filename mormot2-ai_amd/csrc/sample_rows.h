// sample_rows.h - sizes shared by ihip_enqueue_sample_rows' kernels and the host.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define IHIP_HD_SAMPLE static inline __host__ __device__ __attribute__((always_inline))
#else
#define IHIP_HD_SAMPLE static inline
#endif

// the bits below the point of a weight (at most 1) as a whole number, so that the sum over
// a vocabulary stays below 2^62
IHIP_HD_SAMPLE int sample_weight_bits(int32_t vocab)
{
  int n = 0;
  while (((int64_t)1 << n) < vocab) n++;
  return 61 - n;
}
