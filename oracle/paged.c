/* paged.c - the whole-number arithmetic of the paged cache's and the draws' kernels, compiled for
 * the host, so that its bounds are tested without a device. */
#include "../mormot2-ai_amd/csrc/paged.h"
#include "../mormot2-ai_amd/csrc/sample_rows.h"

void orc_paged_range(int32_t length, int64_t window, int64_t max_pages, int32_t page_size,
                     int64_t* lo, int64_t* hi)
{
  paged_range(length, window, max_pages, page_size, lo, hi);
}

int64_t orc_paged_value(int32_t page, int32_t at, int64_t pages, int64_t page_stride,
                        int64_t slot_stride)
{
  return paged_value(page, at, pages, page_stride, slot_stride);
}

int64_t orc_paged_slot_value(int32_t slot, int32_t page_size, int64_t pages, int64_t page_stride,
                             int64_t slot_stride)
{
  return paged_slot_value(slot, page_size, pages, page_stride, slot_stride);
}

int64_t orc_paged_common(int32_t first, int32_t end, int32_t shared, int32_t seqs, int64_t max_pages, int32_t page_size)
{
  return paged_common(first, end, shared, seqs, max_pages, page_size);
}

int32_t orc_sample_weight_bits(int32_t vocab) { return sample_weight_bits(vocab); }

int32_t orc_paged_row(int32_t first, int32_t end, int32_t rows) { return paged_row(first, end, rows); }
