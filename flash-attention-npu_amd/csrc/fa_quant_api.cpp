// fa_quant_api.cpp -- host side of the quantised cache's C entry points:
// fa_update_page_table, fa_quant_append, fa_quant_fwd. Checks, plans and launches
// only: no device memory is read, allocated or waited for.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "fa_quant_plan.h"

namespace fa {
hipError_t launch_page_table(const PageTableArgs& a, hipStream_t stream);
int quant_decode_workers(int kd, int grid);
hipError_t launch_quant_append(QuantAppendArgs a, int dtype, int ct, hipStream_t stream);
hipError_t launch_quant_decode(const QuantFwdArgs& a, int ct, int kd, int nr, int grid, hipStream_t stream);
hipError_t launch_quant_prefill(const QuantFwdArgs& a, int ct, int kd, int rows, int grid, hipStream_t stream);
}  // namespace fa

namespace {

int workers(int kd, int, int cus) { return fa::quant_decode_workers(kd, cus); }

fa_status_t check_table(const fa_page_table_params* p) {
    FA_CHECK(p != nullptr, "params must not be null");
    FA_CHECK(p->abi_version == FA_MI355X_ABI_VERSION, "abi_version %d does not match library ABI %d", p->abi_version,
             FA_MI355X_ABI_VERSION);
    FA_CHECK(p->batch >= 1, "batch size must be positive");
    FA_CHECK(p->page_size >= 1, "page_size must be positive");
    FA_CHECK(p->table_rows >= 0 && p->max_pages >= 0, "page_table sizes must not be negative");
    FA_CHECK(p->cache_batch_idx || p->table_rows >= p->batch, "page_table must have a row per request");
    FA_CHECK((int64_t)p->max_pages * p->page_size <= INT_MAX, "page_table rows hold at most 2^31 - 1 tokens");
    // the kernel's counters of pages go a few thousand past the last
    FA_CHECK((int64_t)p->batch * p->max_pages <= 1 << 30, "the requests of a step have at most 2^30 pages");
    FA_CHECK(p->page_table || (int64_t)p->table_rows * p->max_pages == 0, "page_table is required");
    FA_CHECK(p->page_table_row_stride >= p->max_pages || p->table_rows <= 1, "page_table rows must not overlap");
    FA_CHECK(p->free_capacity >= 0 && (p->free_pages || p->free_capacity == 0), "free_pages is required");
    FA_CHECK(p->cache_seqlens && p->new_seqlens && p->num_free && p->num_free_out && p->cu_seqlens_new,
             "cache_seqlens, new_seqlens, num_free, num_free_out and cu_seqlens_new are required");
    FA_CHECK(p->total_new >= 0 && p->total_new <= INT_MAX, "total_new must be in [0, 2^31)");
    FA_CHECK(p->slot_mapping || p->total_new == 0, "slot_mapping is required");
    return FA_OK;
}

}  // namespace

extern "C" {

fa_status_t fa_update_page_table(const fa_page_table_params* p, void* stream) {
    fa_status_t st = check_table(p);
    if (st != FA_OK) return st;
    fa::PageTableArgs a{};
    a.table = p->page_table;
    a.t_stride = p->page_table_row_stride;
    a.table_rows = p->table_rows;
    a.max_pages = p->max_pages;
    a.batch_idx = p->cache_batch_idx;
    a.before = p->cache_seqlens;
    a.after = p->new_seqlens;
    a.free_pages = p->free_pages;
    a.free_cap = p->free_capacity;
    a.num_free = p->num_free;
    a.num_free_out = p->num_free_out;
    a.cu_new = p->cu_seqlens_new;
    a.slots = p->slot_mapping;
    a.total_new = p->total_new;
    a.B = p->batch;
    a.page_size = p->page_size;
    a.page = fa::udiv_make((uint32_t)p->page_size);
    hipError_t e = fa::launch_page_table(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(FA_EHIP, "page table launch failed: %s", hipGetErrorString(e));
    return FA_OK;
}

fa_status_t fa_quant_append(const fa_quant_append_params* p, void* stream) {
    fa_status_t st = check_append(p, Codes::Eight);
    if (st != FA_OK) return st;
    if (p->total_new == 0 || p->num_pages == 0) return FA_OK;
    const hipError_t e = fa::launch_quant_append(append_args(p), p->dtype, p->cache_dtype, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(FA_EHIP, "append launch failed: %s", hipGetErrorString(e));
    return FA_OK;
}

fa_status_t fa_quant_fwd_workspace_size(const fa_quant_fwd_params* p, size_t* bytes) {
    if (!bytes) return fail(FA_EINVAL, "bytes must not be null");
    fa_status_t st = check_fwd(p, Codes::Eight);
    if (st != FA_OK) return st;
    *bytes = p->seqlen_q > 0 ? make_plan(p, workers).total : 0;
    return FA_OK;
}

fa_status_t fa_quant_fwd(const fa_quant_fwd_params* p, void* stream) {
    fa_status_t st = check_fwd(p, Codes::Eight);
    if (st != FA_OK) return st;
    return attend(p, stream, workers, fa::launch_quant_decode, fa::launch_quant_prefill);
}

}  // extern "C"
