// paged_q8.hip - attention over 8-bit pages: one new token of each sequence, the keys
// and values as 8-bit codes with a single scale for each head of a token.
#include "paged_attention.h"

using namespace ihip;

// HBM bound: 64 sequences of 100 to 16384 keys, 16 heads of 128 over 8, 1.12 GB: 237 us, 4.7
// TB/s; one of 1152 keys is a chain of round trips (12.9 us). The codes become halves and
// the values are turned in registers, as much vector work as a step's loads take, which two
// blocks a CU cover for heads of 128 (one 272 us); heads of 64 and of 256 keep all in the
// registers of one block a CU (194 us, two 209; 445 us, two that spill 492), and so do sizes
// between them (96: 297 us, two 310).
#define PAGED_ATTENTION_Q8(D)                                                                              \
  extern "C" __global__ __launch_bounds__(256, D == 128 ? 2 : 1) void paged_attention_q8_##D(PagedAttn8Args a)  \
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
