// fa_fp4_api.cpp -- host side of the 4-bit cache's C entry points, fa_fp4_append and
// fa_fp4_fwd, and of fa_quant_read. Checks, plans and launches only: no device memory
// is read, allocated or waited for.
#include <hip/hip_runtime.h>

#include <climits>
#include <cstdint>

#include "fa_quant_plan.h"
#include "fa_quant_read_args.h"

namespace fa {
hipError_t launch_fp4_append(QuantAppendArgs a, int dtype, hipStream_t stream);
int fp4_decode_workers(int kd, int nr, int cus);
hipError_t launch_fp4_decode(const QuantFwdArgs& a, int ct, int kd, int nr, int grid, hipStream_t stream);
hipError_t launch_fp4_prefill(const QuantFwdArgs& a, int ct, int kd, int rows, int grid, hipStream_t stream);
hipError_t launch_quant_read(QuantReadArgs a, int dtype, int ct, hipStream_t stream);
}  // namespace fa

namespace {

fa_status_t check_read(const fa_quant_read_params* p) {
    FA_CHECK(p != nullptr, "params must not be null");
    FA_CHECK(p->abi_version == FA_MI355X_ABI_VERSION, "abi_version %d does not match library ABI %d", p->abi_version,
             FA_MI355X_ABI_VERSION);
    FA_CHECK(p->dtype == FA_DTYPE_FP32 || p->dtype == FA_DTYPE_FP16 || p->dtype == FA_DTYPE_BF16,
             "rows are read as fp32, fp16 or bf16");
    const fa_status_t st = check_cache(p->cache_dtype == FA_DTYPE_FP4_E2M1 ? Codes::Four : Codes::Eight, p->cache_dtype, p->nheads_k,
                                       p->headdim, p->num_pages, p->page_size, p->scale_block);
    if (st != FA_OK) return st;
    FA_CHECK(p->total >= 0 && p->total <= INT_MAX, "number of rows must be in [0, 2^31)");
    if (p->total == 0) return FA_OK;
    FA_CHECK(p->k_out && p->v_out && aligned16(p->k_out) && aligned16(p->v_out), "k_out and v_out are required, 16-byte aligned");
    FA_CHECK(p->num_pages == 0 || (p->k && p->v && p->k_scale && p->v_scale), "the caches and the scales are required");
    FA_CHECK(aligned16(p->k) && aligned16(p->v), "the caches must be 16-byte aligned");
    FA_CHECK(multiples(16, p->k_page_stride, p->k_row_stride, p->k_head_stride) &&
                 multiples(16, p->v_page_stride, p->v_row_stride, p->v_head_stride),
             "strides of the caches must be multiples of 16");
    FA_CHECK((p->slot_mapping != nullptr) != (p->cu_seqlens_k != nullptr), "either slot_mapping or cu_seqlens_k is required");
    if (p->cu_seqlens_k) {
        FA_CHECK(p->batch >= 1, "batch size must be positive");
        if (p->page_table) {
            FA_CHECK(p->table_rows >= 1 && p->max_pages >= 1, "page_table must have rows and columns");
            FA_CHECK(p->cache_batch_idx || p->table_rows >= p->batch, "page_table must have a row per sequence");
        } else {
            FA_CHECK(p->cache_batch_idx || p->num_pages >= p->batch, "the cache must have a row per sequence");
        }
    }
    return FA_OK;
}

}  // namespace

extern "C" {

fa_status_t fa_fp4_append(const fa_quant_append_params* p, void* stream) {
    const fa_status_t st = check_append(p, Codes::Four);
    if (st != FA_OK) return st;
    if (p->total_new == 0 || p->num_pages == 0) return FA_OK;
    const hipError_t e = fa::launch_fp4_append(append_args(p), p->dtype, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(FA_EHIP, "append launch failed: %s", hipGetErrorString(e));
    return FA_OK;
}

fa_status_t fa_quant_read(const fa_quant_read_params* p, void* stream) {
    const fa_status_t st = check_read(p);
    if (st != FA_OK) return st;
    if (p->total == 0) return FA_OK;
    fa::QuantReadArgs a{};
    a.c[0] = static_cast<const uint8_t*>(p->k);
    a.c_sp[0] = p->k_page_stride;
    a.c_si[0] = p->k_row_stride;
    a.c_sh[0] = p->k_head_stride;
    a.c[1] = static_cast<const uint8_t*>(p->v);
    a.c_sp[1] = p->v_page_stride;
    a.c_si[1] = p->v_row_stride;
    a.c_sh[1] = p->v_head_stride;
    a.s[0] = p->k_scale;
    a.s_sp[0] = p->k_scale_page_stride;
    a.s_sb[0] = p->k_scale_block_stride;
    a.s_sh[0] = p->k_scale_head_stride;
    a.s[1] = p->v_scale;
    a.s_sp[1] = p->v_scale_page_stride;
    a.s_sb[1] = p->v_scale_block_stride;
    a.s_sh[1] = p->v_scale_head_stride;
    a.o[0] = p->k_out;
    a.o[1] = p->v_out;
    a.total = p->total;
    a.slots = p->slot_mapping;
    a.num_slots = (int64_t)p->num_pages * p->page_size;
    a.cu = p->cu_seqlens_k;
    a.B = p->batch;
    a.table = p->page_table;
    a.t_stride = p->page_table_row_stride;
    a.batch_idx = p->cache_batch_idx;
    a.rows = p->page_table ? p->table_rows : p->num_pages;
    a.num_pages = p->num_pages;
    a.page_size = p->page_size;
    a.capacity = (int64_t)(p->page_table ? p->max_pages : 1) * p->page_size;
    a.page = fa::udiv_make((uint32_t)p->page_size);
    a.sblk = fa::udiv_make((uint32_t)p->scale_block);
    a.chunks = fa::udiv_make((uint32_t)p->headdim / 8);
    a.per_row = fa::udiv_make((uint32_t)p->nheads_k * (uint32_t)(p->headdim / 8));
    const hipError_t e = fa::launch_quant_read(a, p->dtype, p->cache_dtype, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(FA_EHIP, "read launch failed: %s", hipGetErrorString(e));
    return FA_OK;
}

fa_status_t fa_fp4_fwd_workspace_size(const fa_quant_fwd_params* p, size_t* bytes) {
    if (!bytes) return fail(FA_EINVAL, "bytes must not be null");
    const fa_status_t st = check_fwd(p, Codes::Four);
    if (st != FA_OK) return st;
    *bytes = p->seqlen_q > 0 ? make_plan(p, fa::fp4_decode_workers, true).total : 0;
    return FA_OK;
}

fa_status_t fa_fp4_fwd(const fa_quant_fwd_params* p, void* stream) {
    const fa_status_t st = check_fwd(p, Codes::Four);
    if (st != FA_OK) return st;
    return attend(p, stream, fa::fp4_decode_workers, fa::launch_fp4_decode, fa::launch_fp4_prefill, true);
}

}  // extern "C"
