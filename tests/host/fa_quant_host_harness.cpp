// Host-only harness for the checks and plans of the quantised cache's C entries
// (flash-attention-npu_amd/csrc/fa_quant_api.cpp), built with g++ and AddressSanitizer /
// UndefinedBehaviorSanitizer by tests/test_quant_sanitize.py. The launchers are
// recording stubs: the harness checks that every sequence goes through each kernel
// that may have to take it exactly once, with pointers moved to the launch's first
// sequence and at most 2048 sequences a launch, that the scratch of each launch lies
// within the workspace that was asked for, and that extreme fields are refused or
// planned without a signed overflow.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <cstdio>
#include <cstring>
#include <random>
#include <vector>

#include "fa_mi355x.h"
#include "fa_quant_args.h"

extern "C" const char* hipGetErrorString(hipError_t) { return "stub"; }

namespace {
char g_error[512];
struct Launch {
    int kernel;  // 0 decode, 1 prefill
    fa::QuantFwdArgs a;
    int nr, grid, rows;
};
std::vector<Launch> g_launch;
int g_tables, g_appends;
int64_t g_batch = 1 << 20;  // sequences x heads that the decode stub takes in one launch
}  // namespace

namespace fa {
fa_status_t report_error(fa_status_t st, const char* msg) {
    snprintf(g_error, sizeof(g_error), "%s", msg);
    return st;
}
int compute_units() { return 256; }
int64_t quant_decode_batch(int, int, int64_t) { return g_batch; }
int quant_decode_workers(int kd, int grid) { return grid * (kd == 256 ? 4 : 8); }
int quant_prefill_rows(int kd, bool many) { return many && kd < 256 ? 256 : 128; }
hipError_t launch_page_table(const PageTableArgs&, hipStream_t) {
    ++g_tables;
    return hipSuccess;
}
hipError_t launch_quant_append(QuantAppendArgs, int, int, hipStream_t) {
    ++g_appends;
    return hipSuccess;
}
hipError_t launch_quant_decode(const QuantFwdArgs& a, int, int, int nr, int grid, hipStream_t) {
    g_launch.push_back({0, a, nr, grid, 0});
    return hipSuccess;
}
hipError_t launch_quant_prefill(const QuantFwdArgs& a, int, int, int rows, int grid, hipStream_t) {
    g_launch.push_back({1, a, 0, grid, rows});
    return hipSuccess;
}
}  // namespace fa

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

static char* at(uintptr_t x) { return reinterpret_cast<char*>(x); }

static fa_quant_fwd_params base() {
    fa_quant_fwd_params p{};
    p.abi_version = FA_MI355X_ABI_VERSION;
    p.dtype = FA_DTYPE_BF16;
    p.cache_dtype = FA_DTYPE_INT8;
    p.batch = 3;
    p.seqlen_q = 1;
    p.nheads = 8;
    p.nheads_k = 2;
    p.headdim = 128;
    p.num_pages = 9;
    p.page_size = 64;
    p.scale_block = 16;
    p.q = at(1ull << 40);
    p.out = at(1ull << 41);
    p.softmax_lse = reinterpret_cast<float*>(at(1ull << 42));
    p.q_batch_stride = p.out_batch_stride = 1024;
    p.q_row_stride = p.out_row_stride = 1024;
    p.q_head_stride = p.out_head_stride = 128;
    p.k = p.v = at(1ull << 43);
    p.k_page_stride = p.v_page_stride = 64 * 256;
    p.k_row_stride = p.v_row_stride = 256;
    p.k_head_stride = p.v_head_stride = 128;
    p.k_scale = p.v_scale = reinterpret_cast<float*>(at(1ull << 44));
    p.cache_seqlens = reinterpret_cast<int32_t*>(at(1ull << 45));
    p.page_table = reinterpret_cast<int32_t*>(at(1ull << 46));
    p.page_table_row_stride = 4;
    p.table_rows = 3;
    p.max_pages = 4;
    p.softmax_scale = 0.1f;
    p.window_size_left = p.window_size_right = -1;
    return p;
}

// Plans the call and, if it is accepted, runs it on a workspace of the size asked for.
static fa_status_t run(fa_quant_fwd_params p) {
    size_t bytes = 0;
    fa_status_t st = fa_quant_fwd_workspace_size(&p, &bytes);
    g_launch.clear();
    if (st != FA_OK) return st;
    const uintptr_t ws = 1ull << 47;
    p.workspace = at(ws);
    p.workspace_bytes = bytes;
    st = fa_quant_fwd(&p, nullptr);
    CHECK(st == FA_OK, "accepted, then refused: %s", g_error);
    const int64_t rows = p.cu_seqlens_q ? (int64_t)p.total_q : (int64_t)p.batch * p.seqlen_q;
    if (rows == 0 || p.seqlen_q == 0) {
        CHECK(g_launch.empty(), "launches for no rows");
        return st;
    }
    const int kd = p.headdim <= 64 ? 64 : p.headdim <= 128 ? 128 : 256;
    int64_t next[2] = {0, 0};
    for (const Launch& l : g_launch) {
        const fa::QuantFwdArgs& a = l.a;
        const int64_t b0 = next[l.kernel];
        CHECK(a.B >= 1 && a.B <= 2048 && a.B <= std::max<int64_t>(g_batch, 1) && b0 + a.B <= p.batch, "launch of %d from %lld", a.B, (long long)b0);
        CHECK(a.row0 == b0 && a.seqlens == p.cache_seqlens + b0, "rows of a launch");
        if (p.cu_seqlens_q) {
            CHECK(a.cu_q == p.cu_seqlens_q + b0 && a.q == p.q && a.lse == p.softmax_lse, "ragged launch");
        } else {
            CHECK(a.q == static_cast<const uint16_t*>(p.q) + b0 * p.q_batch_stride && a.out == static_cast<uint16_t*>(p.out) + b0 * p.out_batch_stride &&
                      a.lse == p.softmax_lse + b0 * p.nheads * p.seqlen_q, "launch's rows");
        }
        CHECK(!p.cache_batch_idx || a.batch_idx == p.cache_batch_idx + b0, "batch_idx");
        CHECK(a.wl >= -1 && a.wl < 1 << 30 && a.wr >= -1 && a.wr < 1 << 30, "windows %d %d", a.wl, a.wr);
        next[l.kernel] += a.B;
        const auto end = [&](const void* q, int64_t n) { return (int64_t)((uintptr_t)q - ws) + n; };
        if (l.kernel == 0) {
            const int64_t parts = (int64_t)fa::quant_decode_workers(kd, l.grid) * 2 * 16 * l.nr;
            CHECK(end(a.sched, 4 * (a.B + 1)) <= end(a.part_lse, 0) && end(a.part_lse, 4 * parts) <= end(a.part_o, 0) &&
                      end(a.part_o, 4 * parts * kd) <= (int64_t)bytes, "decode scratch");
        } else {
            CHECK(l.grid >= 1 && l.grid <= 256, "prefill grid %d", l.grid);
            if (a.cut) {
                CHECK(l.grid == 256, "a cut line has all workgroups");
                CHECK(end(a.pf_cut, 16 * l.grid) <= end(a.pf_lse, 0) && end(a.pf_lse, 8ll * l.grid * l.rows) <= end(a.pf_o, 0) &&
                          end(a.pf_o, 8ll * l.grid * l.rows * kd) <= (int64_t)bytes && ((uintptr_t)a.pf_cut & 15) == 0, "prefill scratch");
                if (next[0] > 0) CHECK(a.pf_cut == nullptr || (uintptr_t)a.pf_cut >= (uintptr_t)(a.part_o), "scratch of both kernels");
            }
        }
    }
    const int64_t packed = (int64_t)p.seqlen_q * (p.nheads / p.nheads_k);
    const bool decode = packed <= 32 || p.cu_seqlens_q, prefill = packed > 32;
    CHECK(next[0] == (decode ? p.batch : 0) && next[1] == (prefill ? p.batch : 0), "sequences %lld and %lld of %d", (long long)next[0],
          (long long)next[1], p.batch);
    return st;
}

int main() {
    std::mt19937_64 g(1);
    const int64_t sizes[] = {INT_MIN, -1, 0, 1, 2, 3, 15, 16, 17, 31, 32, 33, 48, 64, 128, 255, 256, 257, 2047, 2048, 2049, 4096, 5000, 65535,
                             65536, 1 << 20, 1 << 24, 1 << 27, 1 << 30, (1 << 30) + 1, INT_MAX};
    auto pick = [&]() { return (int32_t)sizes[g() % (sizeof(sizes) / sizeof(sizes[0]))]; };
    int accepted = 0, refused = 0;
    for (int k = 0; k < 400000; ++k) {
        fa_quant_fwd_params p = base();
        g_batch = g() % 8 ? 1 << 20 : 1 + (int64_t)(g() % 100);
        if (g() % 2) p.cu_seqlens_q = reinterpret_cast<int32_t*>(at(1ull << 48)), p.total_q = pick();
        if (g() % 3 == 0) p.page_table = nullptr, p.num_pages = 1 << 20;
        if (g() % 3 == 0) p.cache_batch_idx = reinterpret_cast<int32_t*>(at(1ull << 49));
        int32_t* fields[] = {&p.batch, &p.seqlen_q, &p.nheads, &p.nheads_k, &p.headdim, &p.num_pages, &p.page_size, &p.scale_block, &p.total_q,
                             &p.table_rows, &p.max_pages, &p.window_size_left, &p.window_size_right};
        for (int n = (int)(g() % 4); n >= 0; --n) *fields[g() % 13] = pick();
        if (g() % 2) p.table_rows = std::max(p.table_rows, p.batch);
        // a launch each for more sequences than these is not worth its time here
        if (p.batch > 200000) p.batch = 200000 + p.batch % 7;
        (run(p) == FA_OK ? accepted : refused)++;
    }
    CHECK(accepted > 50000 && refused > 50000, "%d accepted, %d refused", accepted, refused);
    // the decode stub has room for no sequence: refused
    g_batch = 0;
    CHECK(run(base()) == FA_EINVAL, "no room for a sequence");
    for (int k = 0; k < 100000; ++k) {
        fa_page_table_params t{};
        t.abi_version = FA_MI355X_ABI_VERSION;
        t.batch = t.page_size = t.table_rows = t.max_pages = 4;
        t.page_table_row_stride = 4;
        t.page_table = t.free_pages = t.num_free_out = t.cu_seqlens_new = reinterpret_cast<int32_t*>(at(1ull << 40));
        t.cache_seqlens = t.new_seqlens = t.num_free = t.page_table;
        t.slot_mapping = reinterpret_cast<int64_t*>(at(1ull << 41));
        int32_t* fields[] = {&t.batch, &t.page_size, &t.table_rows, &t.max_pages, &t.free_capacity};
        for (int n = (int)(g() % 3); n >= 0; --n) *fields[g() % 5] = pick();
        t.total_new = g() % 4 ? pick() : INT64_MAX - (int64_t)(g() % 3);
        t.page_table_row_stride = g() % 4 ? t.max_pages : (int64_t)pick();
        if (fa_update_page_table(&t, nullptr) == FA_OK)
            CHECK(t.batch >= 1 && (int64_t)t.batch * t.max_pages <= 1 << 30 && t.total_new >= 0 && t.total_new <= INT_MAX, "table");
        fa_quant_append_params a{};
        a.abi_version = FA_MI355X_ABI_VERSION;
        a.dtype = FA_DTYPE_FP16;
        a.cache_dtype = FA_DTYPE_FP8_E4M3;
        a.nheads_k = 2, a.headdim = 64, a.num_pages = 5, a.page_size = 64, a.scale_block = 32, a.total_new = 7;
        a.k_new = a.v_new = a.k = a.v = at(1ull << 42);
        a.k_scale = a.v_scale = reinterpret_cast<float*>(at(1ull << 43));
        a.slot_mapping = reinterpret_cast<int64_t*>(at(1ull << 44));
        int32_t* more[] = {&a.nheads_k, &a.headdim, &a.num_pages, &a.page_size, &a.scale_block};
        for (int n = (int)(g() % 3); n >= 0; --n) *more[g() % 5] = pick();
        if (g() % 3 == 0) a.total_new = g() % 4 ? pick() : INT64_MAX;
        fa_quant_append(&a, nullptr);
    }
    CHECK(g_tables > 1000 && g_appends > 1000, "%d tables, %d appends", g_tables, g_appends);
    std::printf("%d accepted, %d refused, %d tables, %d appends, %d failures\n", accepted, refused, g_tables, g_appends, failures);
    return failures != 0;
}
