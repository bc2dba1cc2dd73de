// paged.h - where a paged cache (ihip_pages) holds a key: the index arithmetic
// of the kernels, shared with the host so that its bounds can be tested there.
#pragma once

#include <stdint.h>

#ifdef __HIP__
#define IHIP_HD static inline __host__ __device__ __attribute__((always_inline))
#else
#define IHIP_HD static inline
#endif

// the keys a query of a sequence of `length` tokens sees: [*lo, *hi), empty for
// a length below 1; a length beyond the table's width is cut to it
IHIP_HD void paged_range(int32_t length, int64_t window, int64_t max_pages, int32_t page_size,
                         int64_t* lo, int64_t* hi)
{
  int64_t n = length > 0 ? length : 0;
  const int64_t most = max_pages * page_size;
  if (n > most) n = most;
  *hi = n;
  *lo = window > 0 && n > window ? n - window : 0;
}

// how many tokens a group of the sequences [first, end) of `seqs` reads together: those of
// its `shared` that its tables hold, none where fewer than two sequences are its
IHIP_HD int64_t paged_common(int32_t first, int32_t end, int32_t shared, int32_t seqs, int64_t max_pages,
                             int32_t page_size)
{
  if (first < 0 || end > seqs || end <= first || end - first < 2 || shared <= 0) return 0;
  const int64_t most = max_pages * page_size;
  return shared < most ? shared : most;
}

// the columns (a member's query head each) that a block of the prefixes' kernel for heads of up
// to d takes, in tiles of 16: its registers' share, and the size of the pieces that it leaves
#define PAGED_SHARED_TILES(d, q8) ((d) <= 64 ? 4 : (d) <= 128 || ((d) == 256 && !(q8)) ? 2 : 1)

// the row of q and y of a sequence whose rows of the step are [first, end): the
// last of them, or -1 where it has none or its last is not among the `rows`
IHIP_HD int32_t paged_row(int32_t first, int32_t end, int32_t rows)
{
  return end > first && end >= 1 && end <= rows ? end - 1 : -1;
}

// the first value of token `at` of page `page`, in values from the pool's start
// (of KV head 0), or -1 where the page is outside the pool
IHIP_HD int64_t paged_value(int32_t page, int32_t at, int64_t pages, int64_t page_stride,
                            int64_t slot_stride)
{
  if (page < 0 || page >= pages) return -1;
  return (int64_t)page * page_stride + (int64_t)at * slot_stride;
}

// the same of a slot number (page * page_size + token)
IHIP_HD int64_t paged_slot_value(int32_t slot, int32_t page_size, int64_t pages,
                                 int64_t page_stride, int64_t slot_stride)
{
  if (slot < 0) return -1;
  const uint32_t page = (uint32_t)slot / (uint32_t)page_size;
  return paged_value((int32_t)page, (int32_t)((uint32_t)slot - page * (uint32_t)page_size), pages,
                     page_stride, slot_stride);
}
