// fa_quant_read_args.h -- the by-value kernel argument block of the rows read back
// from a quantised cache (host and device).
#pragma once
#include <stdint.h>

#include "fa_udiv.h"

namespace fa {

// Strides of the caches are in bytes, of the scales in elements.
struct QuantReadArgs {
    const uint8_t* c[2];           // the caches, k and v
    int64_t c_sp[2], c_si[2], c_sh[2];
    const void* s[2];              // the scales
    int64_t s_sp[2], s_sb[2], s_sh[2];
    void* o[2];
    int64_t total, row0;           // rows; first of the launch
    const int64_t* slots;          // of the rows, or null
    int64_t num_slots;
    const int* cu;
    int B;
    const int* table;              // null: contiguous, the sequence's row is its page
    int64_t t_stride;
    const int* batch_idx;
    int rows, num_pages, page_size;  // rows of the page table, or pages when contiguous
    int64_t capacity;              // keys addressable per sequence
    UDiv page, sblk, chunks, per_row;  // division by page_size, scale_block, hd / 8, Hk * hd / 8
};

}  // namespace fa
