// fa_quant_args.h -- the by-value kernel argument blocks of the quantised
// cache: page table update, quantising append, attention (host and device).
#pragma once
#include <stdint.h>

#include "fa_udiv.h"

namespace fa {

// Cache types, as FA_DTYPE_FP8_E4M3, FA_DTYPE_INT8 and FA_DTYPE_FP4_E2M1.
enum : int { CT_E4M3 = 3, CT_INT8 = 4, CT_FP4 = 5 };

constexpr int kQuantMaxB = 2048;  // sequences of an attention launch, and entries of a list that is cut: they live in LDS

// Packed rows of a block of the 4-bit decode kernel; most that a call of blocks may have: (block, kv head) pairs, and
// those times 64 keys (fa_quant_list.h)
constexpr int kBlockRows = 32, kBlockSegs = 512, kBlockUnits = 16384;
static_assert(kBlockSegs <= kQuantMaxB, "blocks live in the list of sequences");

struct PageTableArgs {
    int* table;
    int64_t t_stride;
    int table_rows, max_pages;
    const int* batch_idx;
    const int* before;
    const int* after;
    int* free_pages;
    int free_cap;
    const int* num_free;
    int* num_free_out;
    int* cu_new;
    int64_t* slots;
    int64_t total_new;
    int B, page_size;
    UDiv page;
};

struct QuantAppendArgs {
    const void* x[2];              // k_new, v_new
    int64_t x_si[2], x_sh[2];
    uint8_t* c[2];                 // the caches
    int64_t c_sp[2], c_si[2], c_sh[2];
    float* s[2];                   // the scales
    int64_t s_sp[2], s_sb[2], s_sh[2];
    const int64_t* slots;
    int64_t total_new, num_slots;  // num_slots: num_pages * page_size
    int Hk, hd, page_size, scale_block;
    int rows_per_unit;             // rows among which a unit looks for the beginning of a run
    int64_t row0;                  // first row of the launch
    UDiv block, page, chunks;      // division by scale_block, page_size and hd / 8
};

// Strides are in elements; cache elements are bytes.
struct QuantFwdArgs {
    const void* q;
    int64_t q_sb, q_si, q_sh;
    const uint8_t* k;
    int64_t k_sp, k_si, k_sh;
    const uint8_t* v;
    int64_t v_sp, v_si, v_sh;
    const float* ks;
    int64_t ks_sp, ks_sb, ks_sh;
    const float* vs;
    int64_t vs_sp, vs_sb, vs_sh;
    void* out;
    int64_t o_sb, o_si, o_sh;
    float* lse;
    int64_t lse_sb, lse_sh;        // (B,H,Sq): b*lse_sb + h*lse_sh + i; ragged (H,T): h*lse_sh + cu_q[b] + i
    const int* seqlens;
    const int* cu_q;
    const int* table;              // null: contiguous, the sequence's row is its page
    int64_t t_stride;
    const int* batch_idx;
    int rows;                      // rows of the page table, or pages when contiguous (bound of batch_idx)
    int num_pages, max_pages, page_size;
    UDiv page, sblk;               // division by page_size and scale_block
    int capacity;                  // keys addressable per sequence
    float scale;                   // softmax_scale
    float softcap;                 // 0 = off
    int B, Sq, H, Hk, g, hd, total_q;
    int row0;                      // row of sequence 0 without batch_idx
    int wl, wr;                    // normalised window, -1 = unbounded, causal => wr = 0
    int bf16;                      // q and out: 0 = fp16, 1 = bf16
    int dec_rows;                  // sequences of at most as many packed rows take the decode kernel
    int blocks;                    // 4-bit codes: blocks of 32 packed rows that its list may have, 0: one for a sequence
    int* block_pref;               // [0..B]: block prefix, with `blocks`
    // scratch of the decode kernel
    int* sched;                    // [0..B]: tile prefix
    float* part_lse;               // [worker][2][16 * row tiles]
    float* part_o;                 // [worker][2][16 * row tiles][kernel head dim]
    // prefill kernel: whether its items are cut, and the scratch of that
    int cut;
    int* pf_cut;                   // [workgroup][4]: the cut item that begins there
    float* pf_lse;                 // [workgroup][2][rows of an item]
    float* pf_o;                   // [workgroup][2][rows of an item][kernel head dim]
};

}  // namespace fa
