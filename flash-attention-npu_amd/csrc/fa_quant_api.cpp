// fa_quant_api.cpp -- host side of the quantised cache's C entry points:
// fa_update_page_table, fa_quant_append, fa_quant_fwd. Checks, plans and launches
// only: no device memory is read, allocated or waited for.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/fa_mi355x.h"
#include "fa_quant_args.h"

namespace fa {
fa_status_t report_error(fa_status_t st, const char* msg);
hipError_t launch_page_table(const PageTableArgs& a, hipStream_t stream);
hipError_t launch_quant_append(QuantAppendArgs a, int dtype, int ct, hipStream_t stream);
int64_t quant_decode_batch(int kd, int Hk, int64_t capacity);
int quant_decode_workers(int kd, int grid);
hipError_t launch_quant_decode(const QuantFwdArgs& a, int ct, int kd, int nr, int grid, hipStream_t stream);
int quant_prefill_rows(int kd, bool many);
hipError_t launch_quant_prefill(const QuantFwdArgs& a, int ct, int kd, int rows, int grid, hipStream_t stream);
int compute_units();
}  // namespace fa

namespace {

fa_status_t fail(fa_status_t st, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return fa::report_error(st, buf);
}

#define FA_CHECK(cond, ...)                              \
    do {                                                 \
        if (!(cond)) return fail(FA_EINVAL, __VA_ARGS__); \
    } while (0)

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
bool multiples(int64_t n, int64_t a, int64_t b, int64_t c) { return a % n == 0 && b % n == 0 && c % n == 0; }

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

// What the append and the attention ask of a cache alike. strides: k, v (page,
// row, head).
fa_status_t check_cache(int cache_dtype, int dtype, int nheads_k, int headdim, int num_pages, int page_size,
                        int scale_block) {
    FA_CHECK(dtype == FA_DTYPE_FP16 || dtype == FA_DTYPE_BF16, "FlashAttention only support fp16 and bf16 data type");
    FA_CHECK(cache_dtype == FA_DTYPE_INT8 || cache_dtype == FA_DTYPE_FP8_E4M3,
             "a quantised cache holds int8 or float8_e4m3fn");
    FA_CHECK(nheads_k >= 1 && nheads_k <= 65535, "number of key/value heads must be in [1, 65535]");
    FA_CHECK(headdim >= 16 && headdim % 16 == 0 && headdim <= 256,
             "head dimension of a quantised cache must be a multiple of 16, at most 256, got %d", headdim);
    FA_CHECK(num_pages >= 0, "num_pages must not be negative");
    FA_CHECK(scale_block >= 16 && scale_block % 16 == 0, "a scale must cover a multiple of 16 tokens, got %d", scale_block);
    FA_CHECK(page_size >= scale_block && page_size % scale_block == 0,
             "page size %d must be a multiple of the %d tokens of a scale", page_size, scale_block);
    return FA_OK;
}

fa_status_t check_append(const fa_quant_append_params* p) {
    FA_CHECK(p != nullptr, "params must not be null");
    FA_CHECK(p->abi_version == FA_MI355X_ABI_VERSION, "abi_version %d does not match library ABI %d", p->abi_version,
             FA_MI355X_ABI_VERSION);
    fa_status_t st = check_cache(p->cache_dtype, p->dtype, p->nheads_k, p->headdim, p->num_pages, p->page_size, p->scale_block);
    if (st != FA_OK) return st;
    FA_CHECK(p->total_new >= 0 && p->total_new <= INT_MAX, "number of new rows must be in [0, 2^31)");
    if (p->total_new == 0 || p->num_pages == 0) return FA_OK;
    FA_CHECK(p->k_new && p->v_new && p->k && p->v && p->k_scale && p->v_scale && p->slot_mapping,
             "k, v, the caches, the scales and slot_mapping are required");
    FA_CHECK(aligned16(p->k_new) && aligned16(p->v_new) && aligned16(p->k) && aligned16(p->v),
             "k, v and the caches must be 16-byte aligned");
    FA_CHECK(multiples(8, p->knew_row_stride, p->knew_head_stride, 0) && multiples(8, p->vnew_row_stride, p->vnew_head_stride, 0),
             "strides of k and v must be multiples of 8 elements");
    // a pass of the kernel addresses up to 128 rows in 32 bits
    FA_CHECK(p->knew_row_stride >= 0 && p->knew_row_stride < (1 << 24) && p->vnew_row_stride >= 0 && p->vnew_row_stride < (1 << 24),
             "row strides of k and v must be in [0, 2^24)");
    FA_CHECK(multiples(16, p->k_page_stride, p->k_row_stride, p->k_head_stride) &&
                 multiples(16, p->v_page_stride, p->v_row_stride, p->v_head_stride),
             "strides of the caches must be multiples of 16");
    return FA_OK;
}

int kernel_headdim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

int64_t batch_of_launch(const fa_quant_fwd_params* p) {
    const int64_t capacity = (int64_t)(p->page_table ? p->max_pages : 1) * p->page_size;
    return std::min<int64_t>(fa::kQuantMaxB, fa::quant_decode_batch(kernel_headdim(p->headdim), p->nheads_k, capacity));
}

fa_status_t check_fwd(const fa_quant_fwd_params* p) {
    FA_CHECK(p != nullptr, "params must not be null");
    FA_CHECK(p->abi_version == FA_MI355X_ABI_VERSION, "abi_version %d does not match library ABI %d", p->abi_version,
             FA_MI355X_ABI_VERSION);
    fa_status_t st = check_cache(p->cache_dtype, p->dtype, p->nheads_k, p->headdim, p->num_pages, p->page_size, p->scale_block);
    if (st != FA_OK) return st;
    FA_CHECK(p->batch >= 1, "batch size must be positive");
    FA_CHECK(p->nheads >= 1 && p->nheads % p->nheads_k == 0, "Number of heads in key/value must divide number of heads in query");
    FA_CHECK(p->seqlen_q >= 0 && p->total_q >= 0, "seqlen_q and total_q must not be negative");
    FA_CHECK(p->softcap >= 0.f, "softcap must be >= 0");
    FA_CHECK(p->cache_seqlens, "cache_seqlens is required");
    FA_CHECK(p->num_pages >= 1, "the cache must have a page");
    if (p->page_table) {
        FA_CHECK(p->table_rows >= 1 && p->max_pages >= 1, "page_table must have rows and columns");
        FA_CHECK(p->cache_batch_idx || p->table_rows >= p->batch, "page_table must have a row per sequence");
        FA_CHECK((int64_t)p->max_pages * p->page_size <= INT_MAX, "page_table rows hold at most 2^31 - 1 tokens");
    } else {
        FA_CHECK(p->cache_batch_idx || p->num_pages >= p->batch, "the cache must have a row per sequence");
    }
    // positions of rows and keys count from -2^30 to 2^30
    FA_CHECK((int64_t)(p->page_table ? p->max_pages : 1) * p->page_size <= 1 << 30, "a sequence holds at most 2^30 tokens");
    const int64_t rows = p->cu_seqlens_q ? (int64_t)p->total_q : (int64_t)p->batch * p->seqlen_q;
    if (rows == 0 || p->seqlen_q == 0) return FA_OK;
    FA_CHECK(batch_of_launch(p) >= 1, "a sequence has too many key/value heads and tokens");
    FA_CHECK(rows <= 1 << 30 && rows * (p->nheads / p->nheads_k) <= 1 << 30, "too many query rows");
    FA_CHECK(p->q && p->out && p->softmax_lse && p->k && p->v && p->k_scale && p->v_scale,
             "q, out, softmax_lse, the caches and the scales are required");
    FA_CHECK(aligned16(p->q) && aligned16(p->out) && aligned16(p->k) && aligned16(p->v),
             "q, out and the caches must be 16-byte aligned");
    FA_CHECK(multiples(8, p->q_batch_stride, p->q_row_stride, p->q_head_stride) &&
                 multiples(8, p->out_batch_stride, p->out_row_stride, p->out_head_stride),
             "strides of q and out must be multiples of 8 elements");
    FA_CHECK(multiples(16, p->k_page_stride, p->k_row_stride, p->k_head_stride) &&
                 multiples(16, p->v_page_stride, p->v_row_stride, p->v_head_stride),
             "strides of the caches must be multiples of 16");
    // the rows of 16 keys are addressed in 32 bits
    FA_CHECK(p->k_row_stride >= 0 && p->k_row_stride < (1 << 27) && p->v_row_stride >= 0 && p->v_row_stride < (1 << 27),
             "row strides of the caches must be in [0, 2^27)");
    return FA_OK;
}

constexpr int kDecodeRows = 32;  // packed rows of a kv head that the decode kernel takes

struct Plan {
    int kd;          // kernel head dim
    int nb;          // sequences of a launch
    int g;
    int dec_rows;    // sequences of at most so many packed rows run on the decode kernel
    bool prefill;    // some may have more
    int nr, grid;    // decode: 16-row tiles, workgroups
    int pf_rows, pf_grid;
    bool cut;        // prefill: the items are cut over the workgroups
    size_t off_lse, off_o, off_pcut, off_plse, off_po, total;
};

size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

Plan make_plan(const fa_quant_fwd_params* p) {
    Plan pl{};
    pl.kd = kernel_headdim(p->headdim);
    pl.nb = (int)std::min<int64_t>(p->batch, batch_of_launch(p));
    pl.g = p->nheads / p->nheads_k;
    // of a ragged batch seqlen_q is a bound, and may be beyond the 2^30 rows of a call
    const int64_t rows = std::min<int64_t>((int64_t)p->seqlen_q * pl.g, 1 << 30);
    pl.prefill = rows > kDecodeRows;
    // Of a ragged batch with longer sequences the ones at their next token or two: with 32 rows in place of
    // 16 the two row tiles of the decode kernel cost a mixed batch 2 us of 185, where its shorter ones
    // are single tokens; 64 sequences of 2 to 7 tokens of 8 heads take 353 us in place of 403.
    pl.dec_rows = !pl.prefill ? (int)rows : p->cu_seqlens_q ? 16 : 0;
    pl.nr = pl.dec_rows <= 16 ? 1 : 2;
    const int cus = fa::compute_units();
    const size_t nb = pl.nb;
    pl.grid = cus;
    size_t off = 0;
    if (pl.dec_rows) {
        const size_t parts = (size_t)fa::quant_decode_workers(pl.kd, pl.grid) * 2 * 16 * pl.nr;
        pl.off_lse = off = align256(sizeof(int) * (nb + 1));
        pl.off_o = off = align256(off + sizeof(float) * parts);
        off = align256(off + sizeof(float) * parts * pl.kd);
    }
    if (pl.prefill) {
        // ragged batches go by their mean
        const int64_t each = p->cu_seqlens_q ? (int64_t)p->total_q * pl.g / p->batch : rows;
        const int bm = pl.pf_rows = fa::quant_prefill_rows(pl.kd, each > 192);
        int64_t entries = (int64_t)nb * ((rows + bm - 1) / bm);
        // ragged: a part tile more per sequence than the rows fill
        if (p->cu_seqlens_q) entries = std::min(entries, (int64_t)p->total_q * pl.g / bm + (int64_t)nb);
        const int64_t items = entries * p->nheads_k;
        // Cutting costs its pieces' sums a way through memory (chunks of 2048 onto 4096 keys,
        // four items to a workgroup: 921 -> 971 us). It pays where items differ in
        // length or a last round would leave workgroups without one. The host sees the latter,
        // and of the former only ragged queries: key lengths that differ under queries of
        // one length leave whole items to be shared out by their number.
        const int64_t rounds = (items + cus - 1) / cus;
        pl.cut = entries <= fa::kQuantMaxB && items < 8 * cus && (p->cu_seqlens_q || rounds * cus * 12 > items * 13);
        pl.pf_grid = pl.cut ? cus : (int)std::min<int64_t>(items, cus);
        if (pl.cut) {
            pl.off_pcut = off;
            pl.off_plse = off = align256(off + sizeof(int) * 4 * pl.pf_grid);
            pl.off_po = off = align256(off + sizeof(float) * 2 * pl.pf_grid * bm);
            off = align256(off + sizeof(float) * 2 * pl.pf_grid * bm * pl.kd);
        }
    }
    pl.total = off;
    return pl;
}

// A window of 2^30 - 1 reaches every key, and the masks' bounds then stay in 32 bits: key_hi
// + 1 is at most (2^30 - 1) + (2^30 - 1) + 1, key_lo at least -2^30 - (2^30 - 1).
int window_bound(int32_t w) { return w < 0 ? -1 : std::min(w, (1 << 30) - 1); }

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
    fa_status_t st = check_append(p);
    if (st != FA_OK) return st;
    if (p->total_new == 0 || p->num_pages == 0) return FA_OK;
    fa::QuantAppendArgs a{};
    a.x[0] = p->k_new;
    a.x_si[0] = p->knew_row_stride;
    a.x_sh[0] = p->knew_head_stride;
    a.x[1] = p->v_new;
    a.x_si[1] = p->vnew_row_stride;
    a.x_sh[1] = p->vnew_head_stride;
    a.c[0] = static_cast<uint8_t*>(p->k);
    a.c_sp[0] = p->k_page_stride;
    a.c_si[0] = p->k_row_stride;
    a.c_sh[0] = p->k_head_stride;
    a.c[1] = static_cast<uint8_t*>(p->v);
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
    a.slots = p->slot_mapping;
    a.total_new = p->total_new;
    a.num_slots = (int64_t)p->num_pages * p->page_size;
    a.Hk = p->nheads_k;
    a.hd = p->headdim;
    a.page_size = p->page_size;
    a.scale_block = p->scale_block;
    hipError_t e = fa::launch_quant_append(a, p->dtype, p->cache_dtype, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(FA_EHIP, "append launch failed: %s", hipGetErrorString(e));
    return FA_OK;
}

fa_status_t fa_quant_fwd_workspace_size(const fa_quant_fwd_params* p, size_t* bytes) {
    if (!bytes) return fail(FA_EINVAL, "bytes must not be null");
    fa_status_t st = check_fwd(p);
    if (st != FA_OK) return st;
    *bytes = p->seqlen_q > 0 ? make_plan(p).total : 0;
    return FA_OK;
}

fa_status_t fa_quant_fwd(const fa_quant_fwd_params* p, void* stream) {
    fa_status_t st = check_fwd(p);
    if (st != FA_OK) return st;
    const int64_t rows = p->cu_seqlens_q ? (int64_t)p->total_q : (int64_t)p->batch * p->seqlen_q;
    if (rows == 0 || p->seqlen_q == 0) return FA_OK;
    const Plan pl = make_plan(p);
    if (pl.total > 0) {
        if (!p->workspace || p->workspace_bytes < pl.total)
            return fail(FA_EWORKSPACE, "workspace of %zu bytes required, %zu given", pl.total, p->workspace ? p->workspace_bytes : (size_t)0);
        if (reinterpret_cast<uintptr_t>(p->workspace) & 255u) return fail(FA_EWORKSPACE, "workspace must be 256-byte aligned");
    }
    fa::QuantFwdArgs a{};
    a.q = p->q;
    a.q_sb = p->q_batch_stride;
    a.q_si = p->q_row_stride;
    a.q_sh = p->q_head_stride;
    a.k = static_cast<const uint8_t*>(p->k);
    a.k_sp = p->k_page_stride;
    a.k_si = p->k_row_stride;
    a.k_sh = p->k_head_stride;
    a.v = static_cast<const uint8_t*>(p->v);
    a.v_sp = p->v_page_stride;
    a.v_si = p->v_row_stride;
    a.v_sh = p->v_head_stride;
    a.ks = p->k_scale;
    a.ks_sp = p->k_scale_page_stride;
    a.ks_sb = p->k_scale_block_stride;
    a.ks_sh = p->k_scale_head_stride;
    a.vs = p->v_scale;
    a.vs_sp = p->v_scale_page_stride;
    a.vs_sb = p->v_scale_block_stride;
    a.vs_sh = p->v_scale_head_stride;
    a.out = p->out;
    a.o_sb = p->out_batch_stride;
    a.o_si = p->out_row_stride;
    a.o_sh = p->out_head_stride;
    a.lse = p->softmax_lse;
    a.lse_sb = p->cu_seqlens_q ? 0 : (int64_t)p->nheads * p->seqlen_q;
    a.lse_sh = p->cu_seqlens_q ? p->total_q : p->seqlen_q;
    a.seqlens = p->cache_seqlens;
    a.cu_q = p->cu_seqlens_q;
    a.table = p->page_table;
    a.t_stride = p->page_table_row_stride;
    a.batch_idx = p->cache_batch_idx;
    a.rows = p->page_table ? p->table_rows : p->num_pages;
    a.num_pages = p->num_pages;
    a.max_pages = p->page_table ? p->max_pages : 1;
    a.page_size = p->page_size;
    a.page = fa::udiv_make((uint32_t)p->page_size);
    a.sblk = fa::udiv_make((uint32_t)p->scale_block);
    a.capacity = (int)((int64_t)a.max_pages * p->page_size);
    a.scale = p->softmax_scale;
    a.softcap = p->softcap;
    a.Sq = p->seqlen_q;
    a.H = p->nheads;
    a.Hk = p->nheads_k;
    a.g = pl.g;
    a.hd = p->headdim;
    a.total_q = p->total_q;
    a.wl = window_bound(p->window_size_left);
    a.wr = p->is_causal ? 0 : window_bound(p->window_size_right);
    a.bf16 = p->dtype == FA_DTYPE_BF16;
    a.dec_rows = pl.dec_rows;
    char* ws = static_cast<char*>(p->workspace);
    a.sched = reinterpret_cast<int*>(ws);
    a.part_lse = reinterpret_cast<float*>(ws + pl.off_lse);
    a.part_o = reinterpret_cast<float*>(ws + pl.off_o);
    a.cut = pl.cut;
    a.pf_cut = reinterpret_cast<int*>(ws + pl.off_pcut);
    a.pf_lse = reinterpret_cast<float*>(ws + pl.off_plse);
    a.pf_o = reinterpret_cast<float*>(ws + pl.off_po);
    // a batch of more sequences than a launch lists runs in parts, one after another
    // on the stream and on the same scratch
    for (int64_t b0 = 0; b0 < p->batch; b0 += pl.nb) {
        fa::QuantFwdArgs c = a;
        c.B = (int)std::min<int64_t>(p->batch - b0, pl.nb);
        c.row0 = (int)b0;
        c.seqlens = a.seqlens + b0;
        if (a.cu_q) {
            c.cu_q = a.cu_q + b0;
        } else {
            c.q = static_cast<const uint16_t*>(a.q) + b0 * a.q_sb;
            c.out = static_cast<uint16_t*>(a.out) + b0 * a.o_sb;
            c.lse = a.lse + b0 * a.lse_sb;
        }
        if (a.batch_idx) c.batch_idx = a.batch_idx + b0;
        hipError_t e = hipSuccess;
        if (pl.dec_rows) e = fa::launch_quant_decode(c, p->cache_dtype, pl.kd, pl.nr, pl.grid, static_cast<hipStream_t>(stream));
        if (e == hipSuccess && pl.prefill) e = fa::launch_quant_prefill(c, p->cache_dtype, pl.kd, pl.pf_rows, pl.pf_grid, static_cast<hipStream_t>(stream));
        if (e != hipSuccess) return fail(FA_EHIP, "attention launch failed: %s", hipGetErrorString(e));
    }
    return FA_OK;
}

}  // extern "C"
