// paged_q8.hip - attention over 8-bit pages: one new token of each sequence, the keys
// and values as 8-bit codes with a single scale for each head of a token.
#include "paged_attention.h"

using namespace ihip;

#define PAGED_ATTENTION_Q8(D)                                                                         \
  extern "C" __global__ __launch_bounds__(256, D <= 256 ? 2 : 1) void paged_attention_q8_##D(PagedAttn8Args a)          \
  {                                                                                                   \
    paged_attention_t<3, D, true>(a);                                                                 \
  }                                                                                                   \
  extern "C" __global__ __launch_bounds__(256) void paged_attention_q8_##D##_part(PagedAttn8Args a)   \
  {                                                                                                   \
    paged_attention_t<3, D, false>(a);                                                                \
  }
PAGED_ATTENTION_Q8(64)
PAGED_ATTENTION_Q8(128)
PAGED_ATTENTION_Q8(256)
PAGED_ATTENTION_Q8(512)
