// Host-only harness for the checks of the 4-bit cache's, the read's and the rotary C entries
// (flash-attention-npu_amd/csrc/fa_fp4_api.cpp, fa_rotary_api.cpp), built with g++ and AddressSanitizer /
// UndefinedBehaviorSanitizer by tests/test_fp4_host.py. The launchers are stubs that hold what reaches them
// against what the kernels assume: extreme fields are refused or arrive within those bounds, with no
// signed overflow on the way.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <random>

#include "fa_mi355x.h"
#include "fa_quant_args.h"
#include "fa_quant_read_args.h"
#include "fa_rotary_args.h"

extern "C" const char* hipGetErrorString(hipError_t) { return "stub"; }

static int failures = 0;
#define CHECK(cond, ...)                                  \
    do {                                                  \
        if (!(cond)) {                                    \
            if (++failures <= 20) {                       \
                std::printf("FAIL %s:%d: ", __FILE__, __LINE__); \
                std::printf(__VA_ARGS__);                 \
                std::printf("\n");                        \
            }                                             \
        }                                                 \
    } while (0)

namespace {
int g_decode, g_prefill, g_append, g_read, g_table, g_rotary;
}

namespace fa {
fa_status_t report_error(fa_status_t st, const char*) { return st; }
int compute_units() { return 256; }
int64_t quant_decode_batch(int, int, int64_t) { return 1 << 20; }
int fp4_decode_workers(int kd, int nr, int cus) { return 4 * cus * (kd == 256 || nr == 2 ? 2 : 3); }
int quant_prefill_rows(int kd, bool many) { return many && kd < 256 ? 256 : 128; }
static void check_cache(int hd, int page, int Hk) {
    CHECK(hd >= 32 && hd <= 256 && hd % 32 == 0 && page >= 16 && page % 16 == 0 && Hk >= 1 && Hk <= 65535, "cache %d %d %d", hd, page, Hk);
}
hipError_t launch_fp4_append(QuantAppendArgs a, int dtype, hipStream_t) {
    ++g_append;
    check_cache(a.hd, a.page_size, a.Hk);
    CHECK(dtype <= 1 && a.total_new >= 1 && a.total_new <= INT_MAX && a.num_slots >= a.page_size, "append");
    return hipSuccess;
}
hipError_t launch_fp4_decode(const QuantFwdArgs& a, int ct, int kd, int nr, int grid, hipStream_t) {
    ++g_decode;
    check_cache(a.hd, a.page_size, a.Hk);
    CHECK(ct == CT_FP4 && a.hd <= kd && a.B >= 1 && a.B <= 2048 && a.dec_rows <= 16 * nr && grid == 256 && a.capacity <= 1 << 30, "decode");
    return hipSuccess;
}
hipError_t launch_fp4_prefill(const QuantFwdArgs& a, int ct, int kd, int rows, int grid, hipStream_t) {
    ++g_prefill;
    check_cache(a.hd, a.page_size, a.Hk);
    CHECK(ct == CT_FP4 && a.hd <= kd && a.B >= 1 && a.B <= 2048 && (rows == 128 || rows == 256) && grid >= 1 && grid <= 256, "prefill");
    return hipSuccess;
}
hipError_t launch_quant_read(QuantReadArgs a, int dtype, int, hipStream_t) {
    ++g_read;
    CHECK(dtype <= 2 && a.total >= 1 && a.total <= INT_MAX && (a.slots != nullptr) != (a.cu != nullptr) && a.chunks.d >= 2 && a.chunks.d <= 32 &&
              a.per_row.d % a.chunks.d == 0 && a.per_row.d <= 65535 * 32 && a.capacity >= a.page_size && (!a.cu || a.B >= 1), "read");
    return hipSuccess;
}
hipError_t launch_rotary_table(const RotaryTableArgs& a, int dtype, hipStream_t) {
    ++g_table;
    CHECK(dtype <= 2 && a.n >= 1 && a.half >= 8 && a.half <= kMaxAngles && a.half % 8 == 0, "table");
    for (int i = 0; i < a.half; ++i) CHECK(a.turns[i] >= 0 && !std::isnan(a.turns[i]), "angle %d: %g", i, a.turns[i]);
    return hipSuccess;
}
hipError_t launch_rotary(RotaryArgs a, int dtype, bool, bool, hipStream_t) {
    ++g_rotary;
    CHECK(dtype <= 1 && a.rows >= 1 && a.rows <= INT_MAX && a.rd >= 16 && a.rd % 16 == 0 && a.rd <= a.hd && a.rd <= 256 && a.hd % 8 == 0 &&
              a.heads0 >= 1 && a.heads >= a.heads0 && (int64_t)a.heads * a.hd <= 1 << 27 && a.seqlen_ro >= 1, "rotary");
    CHECK(a.cu ? a.B >= 1 : a.seqlen.d >= 1, "sequences");
    return hipSuccess;
}
}  // namespace fa

static char* at(uintptr_t x) { return reinterpret_cast<char*>(x); }

template <typename P>
static void fill_cache(P& p) {
    p.abi_version = FA_MI355X_ABI_VERSION;
    p.nheads_k = 2, p.headdim = 64, p.num_pages = 9, p.page_size = 64, p.scale_block = 1;
    p.k = p.v = at(1ull << 40);
    p.k_page_stride = p.v_page_stride = 64 * 64;
    p.k_row_stride = p.v_row_stride = 64;
    p.k_head_stride = p.v_head_stride = 32;
    p.k_scale = p.v_scale = at(1ull << 41);
}

int main() {
    std::mt19937_64 g(1);
    const int64_t sizes[] = {INT_MIN, -1, 0, 1, 2, 8, 15, 16, 17, 24, 32, 48, 64, 96, 128, 256, 257, 2048, 65535, 65536, 1 << 20, 1 << 24, 1 << 30, INT_MAX};
    auto pick = [&]() { return (int32_t)sizes[g() % (sizeof(sizes) / sizeof(sizes[0]))]; };
    auto long_pick = [&]() { return g() % 3 ? (int64_t)pick() : g() % 2 ? INT64_MAX - (int64_t)(g() % 3) : INT64_MIN; };
    const double odd[] = {0.0, -1.0, 1.0, 1e-300, 1e300, NAN, INFINITY, 32.0, 1e4};
    int accepted = 0, refused = 0;
    auto count = [&](fa_status_t st) { (st == FA_OK ? accepted : refused)++; };
    for (int k = 0; k < 200000; ++k) {
        fa_quant_fwd_params f{};
        fill_cache(f);
        f.dtype = FA_DTYPE_BF16, f.cache_dtype = FA_DTYPE_FP4_E2M1, f.batch = 3, f.seqlen_q = 1, f.nheads = 8;
        f.q = at(1ull << 42), f.out = at(1ull << 43), f.softmax_lse = reinterpret_cast<float*>(at(1ull << 44));
        f.cache_seqlens = f.page_table = reinterpret_cast<int32_t*>(at(1ull << 45));
        f.page_table_row_stride = f.max_pages = 4, f.table_rows = 1 << 20;
        if (g() % 2) f.cu_seqlens_q = f.page_table, f.total_q = pick();
        int32_t* ff[] = {&f.batch, &f.seqlen_q, &f.nheads, &f.nheads_k, &f.headdim, &f.num_pages, &f.page_size, &f.scale_block, &f.table_rows,
                         &f.max_pages, &f.window_size_left, &f.window_size_right, &f.cache_dtype};
        for (int n = (int)(g() % 3); n >= 0; --n) *ff[g() % 13] = pick();
        if (f.batch > 10000) f.batch = 10000 + f.batch % 7;
        size_t bytes = 0;
        if (fa_fp4_fwd_workspace_size(&f, &bytes) == FA_OK) {
            f.workspace = at(1ull << 46), f.workspace_bytes = bytes;
            CHECK(fa_fp4_fwd(&f, nullptr) == FA_OK, "accepted, then refused");
            ++accepted;
        } else {
            ++refused;
        }
        fa_quant_append_params a{};
        fill_cache(a);
        a.dtype = FA_DTYPE_FP16, a.cache_dtype = FA_DTYPE_FP4_E2M1, a.total_new = 7;
        a.k_new = a.v_new = at(1ull << 42);
        a.slot_mapping = reinterpret_cast<int64_t*>(at(1ull << 44));
        int32_t* fa_[] = {&a.nheads_k, &a.headdim, &a.num_pages, &a.page_size, &a.scale_block, &a.cache_dtype, &a.dtype};
        for (int n = (int)(g() % 3); n > 0; --n) *fa_[g() % 7] = pick();
        if (g() % 3 == 0) a.total_new = long_pick();
        count(fa_fp4_append(&a, nullptr));
        fa_quant_read_params r{};
        fill_cache(r);
        r.dtype = FA_DTYPE_FP32, r.cache_dtype = g() % 2 ? FA_DTYPE_FP4_E2M1 : FA_DTYPE_INT8, r.total = 7;
        if (r.cache_dtype == FA_DTYPE_INT8) r.scale_block = 16;
        r.k_out = r.v_out = at(1ull << 42);
        if (g() % 2) r.slot_mapping = reinterpret_cast<int64_t*>(at(1ull << 44));
        else r.cu_seqlens_k = r.page_table = reinterpret_cast<int32_t*>(at(1ull << 45)), r.batch = 2, r.table_rows = 2, r.max_pages = 4;
        int32_t* fr[] = {&r.nheads_k, &r.headdim, &r.num_pages, &r.page_size, &r.scale_block, &r.batch, &r.table_rows, &r.max_pages, &r.dtype, &r.cache_dtype};
        for (int n = (int)(g() % 3); n > 0; --n) *fr[g() % 10] = pick();
        if (g() % 3 == 0) r.total = long_pick();
        count(fa_quant_read(&r, nullptr));
        fa_rotary_table_params t{};
        t.abi_version = FA_MI355X_ABI_VERSION, t.dtype = FA_DTYPE_FP32, t.rotary_dim = 64, t.scaling = (int)(g() % 4);
        t.base = 1e4, t.factor = 4, t.original_length = 100, t.low = 1, t.high = 32, t.attention_factor = 1, t.num_positions = 9;
        t.positions = t.cos = t.sin = at(1ull << 42);
        double* fd[] = {&t.base, &t.factor, &t.original_length, &t.low, &t.high, &t.attention_factor};
        for (int n = (int)(g() % 3); n > 0; --n) *fd[g() % 6] = odd[g() % 9];
        if (g() % 4 == 0) t.rotary_dim = pick();
        if (g() % 4 == 0) t.num_positions = long_pick();
        count(fa_rotary_table(&t, nullptr));
        fa_rotary_params p{};
        p.abi_version = FA_MI355X_ABI_VERSION, p.dtype = FA_DTYPE_BF16, p.table_dtype = FA_DTYPE_FP32, p.batch = 2, p.seqlen = 5, p.total = 9;
        p.nheads = 4, p.nheads_k = (int)(g() % 2), p.headdim = 64, p.rotary_dim = 32, p.seqlen_ro = 8;
        p.q = p.k = p.cos = p.sin = at(1ull << 42);
        p.q_out = p.k_out = at(1ull << 43);
        if (g() % 2) p.cu_seqlens = reinterpret_cast<int32_t*>(at(1ull << 45));
        int32_t* fp[] = {&p.batch, &p.seqlen, &p.total, &p.nheads, &p.nheads_k, &p.headdim, &p.rotary_dim, &p.seqlen_ro, &p.dtype, &p.table_dtype};
        for (int n = (int)(g() % 3); n > 0; --n) *fp[g() % 10] = pick();
        if (g() % 4 == 0) p.seqlen_offset = long_pick();
        count(fa_rotary(&p, nullptr));
    }
    CHECK(accepted > 200000 && refused > 200000, "%d accepted, %d refused", accepted, refused);
    CHECK(g_decode > 1000 && g_prefill > 1000 && g_append > 1000 && g_read > 1000 && g_table > 1000 && g_rotary > 1000, "launches %d %d %d %d %d %d",
          g_decode, g_prefill, g_append, g_read, g_table, g_rotary);
    std::printf("%d accepted, %d refused, %d failures\n", accepted, refused, failures);
    return failures != 0;
}
