// fa_quant_plan.h -- what the entries of the 8-bit and of the 4-bit cache share on
// the host: the checks of a call, the plan of an attention call (which kernels run
// its sequences, their scratch) and the launches of its parts.
#pragma once
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

#include "fa_checks.h"
#include "fa_quant_args.h"

namespace fa {
int64_t quant_decode_batch(int kd, int Hk, int64_t capacity);
int quant_prefill_rows(int kd, bool many);
int compute_units();
}  // namespace fa

namespace {

enum class Codes { Eight, Four };  // the caches that an entry takes

// What the entries ask of a cache alike.
inline fa_status_t check_cache(Codes codes, int cache_dtype, int nheads_k, int headdim, int num_pages, int page_size, int scale_block) {
    if (codes == Codes::Eight)
        FA_CHECK(cache_dtype == FA_DTYPE_INT8 || cache_dtype == FA_DTYPE_FP8_E4M3,
                 "a quantised cache holds int8 or float8_e4m3fn");
    else
        FA_CHECK(cache_dtype == FA_DTYPE_FP4_E2M1, "a 4-bit cache holds float4_e2m1");
    FA_CHECK(nheads_k >= 1 && nheads_k <= 65535, "number of key/value heads must be in [1, 65535]");
    FA_CHECK(num_pages >= 0, "num_pages must not be negative");
    if (codes == Codes::Four) {
        FA_CHECK(headdim >= 32 && headdim % 32 == 0 && headdim <= 256,
                 "head dimension of a 4-bit cache must be a multiple of 32, at most 256, got %d", headdim);
        FA_CHECK(page_size >= 16 && page_size % 16 == 0, "page size of a 4-bit cache must be a multiple of 16, got %d", page_size);
        FA_CHECK(scale_block == 1, "each token of a 4-bit cache has scales of its own, got one for %d", scale_block);
        return FA_OK;
    }
    FA_CHECK(headdim >= 16 && headdim % 16 == 0 && headdim <= 256,
             "head dimension of a quantised cache must be a multiple of 16, at most 256, got %d", headdim);
    FA_CHECK(scale_block >= 16 && scale_block % 16 == 0, "a scale must cover a multiple of 16 tokens, got %d", scale_block);
    FA_CHECK(page_size >= scale_block && page_size % scale_block == 0,
             "page size %d must be a multiple of the %d tokens of a scale", page_size, scale_block);
    return FA_OK;
}

inline fa_status_t check_append(const fa_quant_append_params* p, Codes codes) {
    FA_CHECK(p != nullptr, "params must not be null");
    FA_CHECK(p->abi_version == FA_MI355X_ABI_VERSION, "abi_version %d does not match library ABI %d", p->abi_version,
             FA_MI355X_ABI_VERSION);
    FA_CHECK(p->dtype == FA_DTYPE_FP16 || p->dtype == FA_DTYPE_BF16, "FlashAttention only support fp16 and bf16 data type");
    const fa_status_t st = check_cache(codes, p->cache_dtype, p->nheads_k, p->headdim, p->num_pages, p->page_size, p->scale_block);
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

inline int kernel_headdim(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }

inline int64_t batch_of_launch(const fa_quant_fwd_params* p) {
    const int64_t capacity = (int64_t)(p->page_table ? p->max_pages : 1) * p->page_size;
    return std::min<int64_t>(fa::kQuantMaxB, fa::quant_decode_batch(kernel_headdim(p->headdim), p->nheads_k, capacity));
}

inline fa_status_t check_fwd(const fa_quant_fwd_params* p, Codes codes) {
    FA_CHECK(p != nullptr, "params must not be null");
    FA_CHECK(p->abi_version == FA_MI355X_ABI_VERSION, "abi_version %d does not match library ABI %d", p->abi_version,
             FA_MI355X_ABI_VERSION);
    FA_CHECK(p->dtype == FA_DTYPE_FP16 || p->dtype == FA_DTYPE_BF16, "FlashAttention only support fp16 and bf16 data type");
    const fa_status_t st = check_cache(codes, p->cache_dtype, p->nheads_k, p->headdim, p->num_pages, p->page_size, p->scale_block);
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
    FA_CHECK(codes == Codes::Eight || (p->k_scale_block_stride >= 0 && p->k_scale_block_stride < (1 << 27) &&
                                       p->v_scale_block_stride >= 0 && p->v_scale_block_stride < (1 << 27)),
             "token strides of the scales of a 4-bit cache must be in [0, 2^27)");
    return FA_OK;
}

constexpr int kDecodeRows = 32;  // packed rows of a kv head that the decode kernel takes

struct Plan {
    int kd;          // kernel head dim
    int nb;          // sequences of a launch
    int g;
    int dec_rows;    // sequences of at most so many packed rows run on the decode kernel
    bool prefill;    // some may have more
    int nr, grid;    // decode: 16-row tiles, compute units
    int pf_rows, pf_grid;
    bool cut;        // prefill: the items are cut over the workgroups
    int blocks;      // 4-bit codes: blocks of rows that the decode kernel's list may have
    size_t off_blk;
    size_t off_lse, off_o, off_pcut, off_plse, off_po, total;
};

inline size_t align256(size_t x) { return (x + 255) & ~size_t(255); }

// The waves that share the list of tiles, by the kernel head dim, 16-row tiles and compute units
using Workers = int (*)(int kd, int nr, int cus);

// in_blocks: the decode kernel takes longer sequences in blocks of their rows (fa_quant_list.h)
inline Plan make_plan(const fa_quant_fwd_params* p, Workers workers, bool in_blocks = false) {
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
    // (ragged: where most sequences are at their next token, their kernel is meant, and blocks are seldom taken)
    if (pl.prefill && in_blocks && (!p->cu_seqlens_q || (int64_t)p->total_q * pl.g >= (int64_t)fa::kBlockRows * p->batch)) {
        const int64_t most = p->cu_seqlens_q ? (int64_t)p->total_q * pl.g / fa::kBlockRows + pl.nb
                                             : pl.nb * ((rows + fa::kBlockRows - 1) / fa::kBlockRows);
        if (most * p->nheads_k <= fa::kBlockSegs) {
            pl.blocks = (int)most;
            pl.nr = 2;
            if (p->batch == 1) pl.dec_rows = 0;  // its only sequence is hardly shorter than a block: no launch for that
        }
    }
    const int cus = fa::compute_units();
    const size_t nb = pl.nb;
    pl.grid = cus;
    size_t off = 0;
    if (pl.dec_rows || pl.blocks) {
        const size_t parts = (size_t)workers(pl.kd, pl.nr, pl.grid) * 2 * 16 * pl.nr;
        pl.off_blk = sizeof(int) * (std::max(nb, (size_t)pl.blocks) + 1);
        pl.off_lse = off = align256(pl.off_blk + (pl.blocks ? sizeof(int) * (nb + 1) : 0));
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
inline int window_bound(int32_t w) { return w < 0 ? -1 : std::min(w, (1 << 30) - 1); }

inline fa::QuantAppendArgs append_args(const fa_quant_append_params* p) {
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
    a.s[0] = static_cast<float*>(p->k_scale);
    a.s_sp[0] = p->k_scale_page_stride;
    a.s_sb[0] = p->k_scale_block_stride;
    a.s_sh[0] = p->k_scale_head_stride;
    a.s[1] = static_cast<float*>(p->v_scale);
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
    return a;
}

using LaunchDecode = hipError_t (*)(const fa::QuantFwdArgs& a, int ct, int kd, int nr, int grid, hipStream_t stream);
using LaunchPrefill = hipError_t (*)(const fa::QuantFwdArgs& a, int ct, int kd, int rows, int grid, hipStream_t stream);

// A checked attention call
inline fa_status_t attend(const fa_quant_fwd_params* p, void* stream, Workers workers, LaunchDecode decode, LaunchPrefill prefill,
                          bool in_blocks = false) {
    const int64_t rows = p->cu_seqlens_q ? (int64_t)p->total_q : (int64_t)p->batch * p->seqlen_q;
    if (rows == 0 || p->seqlen_q == 0) return FA_OK;
    const Plan pl = make_plan(p, workers, in_blocks);
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
    a.ks = static_cast<const float*>(p->k_scale);
    a.ks_sp = p->k_scale_page_stride;
    a.ks_sb = p->k_scale_block_stride;
    a.ks_sh = p->k_scale_head_stride;
    a.vs = static_cast<const float*>(p->v_scale);
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
    a.blocks = pl.blocks;
    char* ws = static_cast<char*>(p->workspace);
    a.sched = reinterpret_cast<int*>(ws);
    a.block_pref = reinterpret_cast<int*>(ws + pl.off_blk);
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
        if (pl.dec_rows || pl.blocks) e = decode(c, p->cache_dtype, pl.kd, pl.nr, pl.grid, static_cast<hipStream_t>(stream));
        if (e == hipSuccess && pl.prefill) e = prefill(c, p->cache_dtype, pl.kd, pl.pf_rows, pl.pf_grid, static_cast<hipStream_t>(stream));
        if (e != hipSuccess) return fail(FA_EHIP, "attention launch failed: %s", hipGetErrorString(e));
    }
    return FA_OK;
}

}  // namespace
