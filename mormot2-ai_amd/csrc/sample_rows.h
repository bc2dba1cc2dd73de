// sample_rows.h - sizes shared by ihip_enqueue_sample_rows' kernels and the host.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define IHIP_HD_SAMPLE static inline __host__ __device__ __attribute__((always_inline))
#else
#define IHIP_HD_SAMPLE static inline
#endif

// rows of one launch whose candidates go into bins by all blocks, and the bins of each
#define SAMPLE_HEAVY 512
#define SAMPLE_BINS 2048
// tokens that a block sorts at once
#define SAMPLE_CAP 1024
// bytes of their bins, and of the tokens found in those that matter
#define SAMPLE_HEAVY_BYTES (SAMPLE_HEAVY * (SAMPLE_BINS * 8 + (1 + SAMPLE_CAP) * 4))

// the bits below the point of a weight (at most 1) as a whole number, so that the sum over
// a vocabulary stays below 2^62, and 2^52 holds one
IHIP_HD_SAMPLE int sample_weight_bits(int32_t vocab)
{
  int n = 0;
  while (((int64_t)1 << n) < vocab) n++;
  return 61 - n < 51 ? 61 - n : 51;
}
