// fa_rotary_api.cpp -- host side of the rotary C entry points: fa_rotary_table, fa_rotary.
// Checks and launches only: no device memory is read, allocated or waited for.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>

#include "fa_checks.h"
#include "fa_rotary_args.h"
#include "fa_rotary_rows.h"

namespace fa {
hipError_t launch_rotary_table(const RotaryTableArgs& a, int dtype, hipStream_t stream);
hipError_t launch_rotary(RotaryArgs a, int dtype, bool inter, bool wide_table, hipStream_t stream);
}  // namespace fa

namespace {

constexpr double kTwoPi = 6.283185307179586476925;

fa_status_t check_rotary_dim(int rd) {
    FA_CHECK(rd >= 16 && rd % 16 == 0 && rd <= 2 * fa::kMaxAngles, "rotary_dim must be a multiple of 16, at most 256, got %d", rd);
    return FA_OK;
}

fa_status_t check_table(const fa_rotary_table_params* p) {
    FA_CHECK(p != nullptr, "params must not be null");
    FA_CHECK(p->abi_version == FA_MI355X_ABI_VERSION, "abi_version %d does not match library ABI %d", p->abi_version,
             FA_MI355X_ABI_VERSION);
    FA_CHECK(p->dtype == FA_DTYPE_FP32 || p->dtype == FA_DTYPE_FP16 || p->dtype == FA_DTYPE_BF16,
             "rotary tables hold fp32, fp16 or bf16");
    const fa_status_t st = check_rotary_dim(p->rotary_dim);
    if (st != FA_OK) return st;
    FA_CHECK(p->num_positions >= 0, "the number of positions must not be negative");
    FA_CHECK(p->base > 0 && std::isfinite(p->base), "base must be positive");
    FA_CHECK(p->scaling >= FA_ROTARY_PLAIN && p->scaling <= FA_ROTARY_BY_PARTS, "unknown scaling of the positions");
    FA_CHECK(p->factor > 0 && std::isfinite(p->factor), "factor must be positive");
    FA_CHECK(std::isfinite(p->attention_factor), "attention_factor must be finite");
    if (p->scaling == FA_ROTARY_BY_PARTS) {
        FA_CHECK(p->original_length > 0 && std::isfinite(p->original_length), "original_length must be positive");
        FA_CHECK(std::isfinite(p->low) && std::isfinite(p->high) && p->low < p->high, "low must be less than high");
    }
    if (p->num_positions == 0) return FA_OK;
    FA_CHECK(p->positions && p->cos && p->sin, "positions, cos and sin are required");
    FA_CHECK(aligned16(p->cos) && aligned16(p->sin), "cos and sin must be 16-byte aligned");
    return FA_OK;
}

fa_status_t check_rotary(const fa_rotary_params* p) {
    FA_CHECK(p != nullptr, "params must not be null");
    FA_CHECK(p->abi_version == FA_MI355X_ABI_VERSION, "abi_version %d does not match library ABI %d", p->abi_version,
             FA_MI355X_ABI_VERSION);
    FA_CHECK(p->dtype == FA_DTYPE_FP16 || p->dtype == FA_DTYPE_BF16, "FlashAttention only support fp16 and bf16 data type");
    FA_CHECK(p->table_dtype == FA_DTYPE_FP32 || p->table_dtype == p->dtype, "cos and sin must have the dtype of q, or fp32");
    const fa_status_t st = check_rotary_dim(p->rotary_dim);
    if (st != FA_OK) return st;
    FA_CHECK(p->headdim % 8 == 0 && p->headdim <= 65536, "head dimension must be a multiple of 8, at most 65536, got %d", p->headdim);
    FA_CHECK(p->rotary_dim <= p->headdim, "rotary_dim %d exceeds the head dimension %d", p->rotary_dim, p->headdim);
    FA_CHECK(p->nheads >= 1 && p->nheads <= 65535, "number of heads must be in [1, 65535]");
    FA_CHECK(p->nheads_k >= 0 && p->nheads_k <= 65535, "number of key/value heads must be in [0, 65535]");
    FA_CHECK((int64_t)(p->nheads + p->nheads_k) * p->headdim <= 1 << 27, "a row has too many heads");
    FA_CHECK(p->batch >= 0 && p->seqlen >= 0 && p->total >= 0, "batch size, seqlen and total must not be negative");
    FA_CHECK(!p->cu_seqlens || p->batch >= 1, "cu_seqlens must have a sequence");
    FA_CHECK(p->cu_seqlens || (int64_t)p->batch * p->seqlen <= INT_MAX, "a call turns less than 2^31 rows");
    if ((p->cu_seqlens ? (int64_t)p->total : (int64_t)p->batch * p->seqlen) == 0) return FA_OK;
    FA_CHECK(p->seqlen_ro >= 1, "cos and sin must have a row");
    FA_CHECK(p->q && p->q_out && p->cos && p->sin, "q, its result, cos and sin are required");
    FA_CHECK(!p->nheads_k || (p->k && p->k_out), "k and its result are required");
    const bool in_place = p->q == p->q_out;
    FA_CHECK(!p->nheads_k || in_place == (p->k == p->k_out), "q and k are turned in place, or neither is");
    FA_CHECK(!in_place || (p->q_batch_stride == p->q_out_batch_stride && p->q_row_stride == p->q_out_row_stride &&
                           p->q_head_stride == p->q_out_head_stride &&
                           (!p->nheads_k || (p->k_batch_stride == p->k_out_batch_stride && p->k_row_stride == p->k_out_row_stride &&
                                             p->k_head_stride == p->k_out_head_stride))),
             "results in place have the strides of q and k");
    FA_CHECK(aligned16(p->q) && aligned16(p->q_out) && aligned16(p->cos) && aligned16(p->sin) &&
                 (!p->nheads_k || (aligned16(p->k) && aligned16(p->k_out))),
             "q, k, their results, cos and sin must be 16-byte aligned");
    FA_CHECK(p->q_batch_stride % 8 == 0 && p->q_row_stride % 8 == 0 && p->q_head_stride % 8 == 0 && p->q_out_batch_stride % 8 == 0 &&
                 p->q_out_row_stride % 8 == 0 && p->q_out_head_stride % 8 == 0 &&
                 (!p->nheads_k || (p->k_batch_stride % 8 == 0 && p->k_row_stride % 8 == 0 && p->k_head_stride % 8 == 0 &&
                                   p->k_out_batch_stride % 8 == 0 && p->k_out_row_stride % 8 == 0 && p->k_out_head_stride % 8 == 0)),
             "strides of q, k and their results must be multiples of 8 elements");
    FA_CHECK(p->cos_row_stride % 8 == 0 && p->sin_row_stride % 8 == 0, "row strides of cos and sin must be multiples of 8 elements");
    if (in_place) {
        const int64_t B = p->cu_seqlens ? 1 : p->batch, S = p->cu_seqlens ? p->total : p->seqlen;
        const fa::RotaryRows q{{B, S, p->nheads}, {p->q_batch_stride, p->q_row_stride, p->q_head_stride}, p->headdim};
        const fa::RotaryRows k{{B, S, p->nheads_k}, {p->k_batch_stride, p->k_row_stride, p->k_head_stride}, p->headdim};
        FA_CHECK(fa::rows_once(q) && fa::rows_once(k), "q and k turned in place must not repeat rows");
        FA_CHECK(!p->nheads_k || fa::rows_apart(q, k, ((int64_t)(uintptr_t)p->k - (int64_t)(uintptr_t)p->q) / 2),
                 "q and k turned in place must not hold the same memory");
    }
    return FA_OK;
}

}  // namespace

extern "C" {

fa_status_t fa_rotary_table(const fa_rotary_table_params* p, void* stream) {
    const fa_status_t st = check_table(p);
    if (st != FA_OK) return st;
    if (p->num_positions == 0) return FA_OK;
    fa::RotaryTableArgs a{};
    a.positions = p->positions;
    a.wide = p->positions_int64 != 0;
    a.n = p->num_positions;
    a.half = p->rotary_dim / 2;
    a.factor = (float)p->attention_factor;
    a.cos = p->cos;
    a.sin = p->sin;
    const double rd = p->rotary_dim;
    const double base = p->scaling == FA_ROTARY_NTK ? p->base * std::pow(p->factor, rd / (rd - 2)) : p->base;
    for (int i = 0; i < a.half; ++i) {
        double f = std::pow(base, -2.0 * i / rd);
        if (p->scaling == FA_ROTARY_LINEAR) {
            f /= p->factor;
        } else if (p->scaling == FA_ROTARY_BY_PARTS) {
            const double turns = p->original_length * f / kTwoPi;
            const double keep = std::fmin(std::fmax((turns - p->low) / (p->high - p->low), 0.0), 1.0);
            f *= keep + (1.0 - keep) / p->factor;
        }
        FA_CHECK(std::isfinite(f), "angle %d of base, factor and original_length is not finite", i);
        a.turns[i] = 4.0 * (f / kTwoPi);
    }
    const hipError_t e = fa::launch_rotary_table(a, p->dtype, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(FA_EHIP, "rotary table launch failed: %s", hipGetErrorString(e));
    return FA_OK;
}

fa_status_t fa_rotary(const fa_rotary_params* p, void* stream) {
    const fa_status_t st = check_rotary(p);
    if (st != FA_OK) return st;
    fa::RotaryArgs a{};
    a.rows = p->cu_seqlens ? (int64_t)p->total : (int64_t)p->batch * p->seqlen;
    if (a.rows == 0) return FA_OK;
    a.x[0] = p->q;
    a.x_sb[0] = p->q_batch_stride;
    a.x_si[0] = p->q_row_stride;
    a.x_sh[0] = p->q_head_stride;
    a.o[0] = p->q_out;
    a.o_sb[0] = p->q_out_batch_stride;
    a.o_si[0] = p->q_out_row_stride;
    a.o_sh[0] = p->q_out_head_stride;
    a.x[1] = p->k;
    a.x_sb[1] = p->k_batch_stride;
    a.x_si[1] = p->k_row_stride;
    a.x_sh[1] = p->k_head_stride;
    a.o[1] = p->k_out;
    a.o_sb[1] = p->k_out_batch_stride;
    a.o_si[1] = p->k_out_row_stride;
    a.o_sh[1] = p->k_out_head_stride;
    a.heads0 = p->nheads;
    a.heads = p->nheads + p->nheads_k;
    a.hd = p->headdim;
    a.rd = p->rotary_dim;
    a.in_place = p->q == p->q_out;
    a.sign = p->conjugate ? -1.f : 1.f;
    a.cos = p->cos;
    a.sin = p->sin;
    a.c_stride = p->cos_row_stride;
    a.s_stride = p->sin_row_stride;
    a.seqlen_ro = p->seqlen_ro;
    a.positions = p->positions;
    a.wide = p->positions_int64 != 0;
    a.p_sb = p->positions_batch_stride;
    a.p_si = p->positions_row_stride;
    a.offsets = p->seqlen_offsets;
    // a row is less than 2^31 behind its sequence's first, and so are the tables' rows: farther offsets all lead outside
    a.offset = std::clamp<int64_t>(p->seqlen_offset, -(1ll << 31), 1ll << 31);
    a.cu = p->cu_seqlens;
    a.B = p->batch;
    a.seqlen = fa::udiv_make((uint32_t)(p->cu_seqlens ? 1 : p->seqlen));
    const hipError_t e = fa::launch_rotary(a, p->dtype, p->interleaved != 0, p->table_dtype == FA_DTYPE_FP32, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(FA_EHIP, "rotation launch failed: %s", hipGetErrorString(e));
    return FA_OK;
}

}  // extern "C"
