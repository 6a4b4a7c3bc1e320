// fa_page_table.hip -- the page table of a paged cache, brought from one step's
// request lengths to the next on the GPU: fa_update_page_table.
//
// Request b holds have = ceil(before / P) pages and needs need = ceil(after / P).
// With rel and take the two differences (each at least 0), and prefix sums over the
// requests in their order, released page r goes to place n0 + r of the free stack
// (n0 ids on it) and needed page t comes from place top - 1 - t, top = n0 + all
// released. Token i of request b has slot table[(before + i) / P] * P + (before +
// i) % P. Nothing below n0 is written and no entry of the table that the step
// still uses, so a step taken twice gives the same.
//
// What bounds it is latency: a few dependent reads, one launch. Every workgroup
// makes the prefix sums for itself in LDS (lengths and released ids are a few KB,
// read from L2) and then writes its share of stack, table and slots; an id that
// this step both releases and takes is found in the table, where its owner's row
// is not written, so no workgroup waits for another. Measured: 64 requests 6 us
// (10 with the call: the host dispatches and allocates three results), 1024 of which an eighth
// end 18, 96 prompts of 512 to 8192 tokens 10; as two launches the last two took 77 and 75.
#include "fa_common.h"
#include "fa_quant_args.h"

#include <algorithm>

namespace fa {

namespace {

constexpr int NT = 1024;

// Sums of counts, none negative. Pages of all requests fit in 32 bits (the host checks),
// new tokens need not, the lengths being the caller's: their sums (SAT) end at 2^31 - 1.
template <bool SAT>
__device__ __forceinline__ int add(int x, int y) {
    return SAT ? __builtin_elementwise_add_sat(x, y) : x + y;
}

// exclusive prefix over the workgroup of v, total in `sum`
template <bool SAT = false>
__device__ __forceinline__ int block_scan(int v, int* s_w, int& sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(incl, o);
        if (lane >= o) incl = add<SAT>(incl, u);
    }
    int excl = incl - v;
    if constexpr (SAT) {
        const int u = __shfl_up(incl, 1);
        excl = lane > 0 ? u : 0;
    }
    __syncthreads();
    if (lane == 63) s_w[wave] = incl;
    __syncthreads();
    int pre = 0;
    sum = 0;
    for (int w = 0; w < NT / 64; ++w) {
        pre = add<SAT>(pre, w < wave ? s_w[w] : 0);
        sum = add<SAT>(sum, s_w[w]);
    }
    return add<SAT>(pre, excl);
}

struct Req {
    int row;           // of the table, -1: none
    int have, need;    // pages
    int fresh;         // new tokens
};

__device__ __forceinline__ Req request(const PageTableArgs& a, int b) {
    Req r{-1, 0, 0, 0};
    if (b >= a.B) return r;
    const int before = max(a.before[b], 0), after = max(a.after[b], 0);
    r.fresh = max(after - before, 0);
    r.row = a.batch_idx ? a.batch_idx[b] : b;
    if (r.row < 0 || r.row >= a.table_rows) {
        r.row = -1;
        return r;
    }
    r.have = min((int)udiv(a.page, (uint32_t)before) + (before % a.page_size ? 1 : 0), a.max_pages);
    r.need = min((int)udiv(a.page, (uint32_t)after) + (after % a.page_size ? 1 : 0), a.max_pages);
    return r;
}

constexpr int MAXB = 4096;  // requests whose sums fit in LDS

// Inclusive prefix of s[1..n] over the workgroup, in place (s[0] = 0); s_w is scratch.
template <bool SAT = false>
__device__ __forceinline__ void scan_lds(int* s, int n, int* s_w) {
    int carry = 0;
    for (int b0 = 0; b0 < n; b0 += NT) {
        const int b = b0 + threadIdx.x, v = b < n ? s[b + 1] : 0;
        int sum;
        const int pre = add<SAT>(carry, block_scan<SAT>(v, s_w, sum));
        carry = add<SAT>(carry, sum);
        if (b < n) s[b + 1] = add<SAT>(pre, v);
    }
    if (threadIdx.x == 0) s[0] = 0;
    __syncthreads();
}

__global__ void __launch_bounds__(NT) fa_page_table_kernel(PageTableArgs a) {
    // prefixes of released entries, ids among them, needed pages and new tokens;
    // row (-1: none) and the smaller of have and need of each request
    __shared__ int s_rel[MAXB + 1], s_val[MAXB + 1], s_take[MAXB + 1], s_fresh[MAXB + 1], s_row[MAXB], s_min[MAXB], s_w[NT / 64];
    const int tid = threadIdx.x, B = a.B;
    const int64_t first = (int64_t)blockIdx.x * NT + tid, stride = (int64_t)gridDim.x * NT;
    const int n0 = min(max(a.num_free[0], 0), a.free_cap);
    for (int b = tid; b < B; b += NT) {
        const Req r = request(a, b);
        s_rel[b + 1] = s_val[b + 1] = max(r.have - r.need, 0);
        s_take[b + 1] = max(r.need - r.have, 0);
        s_fresh[b + 1] = r.fresh;
        s_row[b] = r.row;
        s_min[b] = min(r.have, r.need);
    }
    scan_lds(s_rel, B, s_w);
    scan_lds(s_take, B, s_w);
    scan_lds<true>(s_fresh, B, s_w);
    const int raw = s_rel[B], taken = s_take[B], fresh = s_fresh[B];
    // released entry f of the requests in turn: its request, place among the request's, id
    auto entry = [&](int f, int& b, int& j) -> int {
        b = seq_of(s_rel, B, f);
        j = f - s_rel[b];
        return a.table[(int64_t)s_row[b] * a.t_stride + s_min[b] + j];
    };
    if (raw > 0) {
        for (int f = tid; f < raw; f += 4 * NT) {  // four reads at once
            int id[4], b[4], j;
#pragma unroll
            for (int u = 0; u < 4; ++u) id[u] = f + u * NT < raw ? entry(f + u * NT, b[u], j) : 0;
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (id[u] < 0) atomicSub(&s_val[b[u] + 1], 1);
        }
        __syncthreads();
        scan_lds(s_val, B, s_w);
        for (int64_t f = first; f < raw; f += stride) {
            int b, j;
            const int id = entry((int)f, b, j);
            if (id < 0) continue;
            int rank = j;
            if (s_val[b + 1] - s_val[b] != s_rel[b + 1] - s_rel[b]) {  // -1 among them
                rank = 0;
                for (int u = 0; u < j; ++u) {
                    int bb, jj;
                    rank += entry(s_rel[b] + u, bb, jj) >= 0;
                }
            }
            const int64_t at = (int64_t)n0 + s_val[b] + rank;
            if (at < a.free_cap) a.free_pages[at] = id;
        }
    }
    const int released = raw > 0 ? s_val[B] : 0;
    const int top = (int)min((int64_t)n0 + released, (int64_t)a.free_cap);
    // the id that needed page t comes to
    auto page_at = [&](int t) -> int {
        const int at = top - 1 - t;
        if (at < 0) return -1;
        if (at < n0) return a.free_pages[at];
        const int b = seq_of(s_val, B, at - n0);
        int k = at - n0 - s_val[b], bb, jj;
        if (s_val[b + 1] - s_val[b] == s_rel[b + 1] - s_rel[b]) return entry(s_rel[b] + k, bb, jj);
        for (int u = s_rel[b]; u < s_rel[b + 1]; ++u) {
            const int id = entry(u, bb, jj);
            if (id >= 0 && k-- == 0) return id;
        }
        return -1;
    };
    for (int64_t t = first; t < taken; t += stride) {
        const int b = seq_of(s_take, B, (int)t);
        a.table[(int64_t)s_row[b] * a.t_stride + s_min[b] + ((int)t - s_take[b])] = page_at((int)t);
    }
    for (int64_t i = first; i < a.total_new; i += stride) {
        int64_t slot = -1;
        if (i < fresh) {
            const int b = seq_of(s_fresh, B, (int)i);
            const int64_t at = (int64_t)max(a.before[b], 0) + (i - s_fresh[b]);
            if (s_row[b] >= 0 && at < (int64_t)a.max_pages * a.page_size) {
                const int j = (int)udiv(a.page, (uint32_t)at), have = s_min[b];  // the request grows
                const int id = j < have ? a.table[(int64_t)s_row[b] * a.t_stride + j] : page_at(s_take[b] + j - have);
                if (id >= 0) slot = (int64_t)id * a.page_size + (at - (int64_t)j * a.page_size);
            }
        }
        a.slots[i] = slot;
    }
    if (blockIdx.x == 0) {
        for (int b = tid; b <= B; b += NT) a.cu_new[b] = s_fresh[b];
        if (tid == 0) a.num_free_out[0] = top - taken;
    }
}

// For more requests: one workgroup writes the stack, the table and the prefix of
// the new tokens, ...
__global__ void __launch_bounds__(NT) fa_page_table_large_kernel(PageTableArgs a) {
    __shared__ int s_w[NT / 64];
    const int n0 = min(max(a.num_free[0], 0), a.free_cap);
    int released = 0;
    for (int b0 = 0; b0 < a.B; b0 += NT) {
        const Req r = request(a, b0 + threadIdx.x);
        const int* row = a.table + (int64_t)max(r.row, 0) * a.t_stride;
        int n = 0, sum;
        for (int j = r.need; j < r.have; ++j) n += row[j] >= 0;
        int64_t at = (int64_t)n0 + released + block_scan(n, s_w, sum);
        for (int j = r.need; j < r.have; ++j) {
            const int id = row[j];
            if (id < 0) continue;
            if (at < a.free_cap) a.free_pages[at] = id;
            ++at;
        }
        released += sum;
    }
    const int top = (int)min((int64_t)n0 + released, (int64_t)a.free_cap);
    __syncthreads();  // the stack is whole
    int taken = 0, fresh = 0;
    for (int b0 = 0; b0 < a.B; b0 += NT) {
        const int b = b0 + threadIdx.x;
        const Req r = request(a, b);
        int sum;
        const int t0 = taken + block_scan(max(r.need - r.have, 0), s_w, sum);
        taken += sum;
        int* row = a.table + (int64_t)max(r.row, 0) * a.t_stride;
        for (int j = r.have; j < r.need; ++j) {
            const int at = top - 1 - (t0 + j - r.have);
            row[j] = at >= 0 ? a.free_pages[at] : -1;
        }
        const int f0 = add<true>(fresh, block_scan<true>(r.fresh, s_w, sum));
        fresh = add<true>(fresh, sum);
        if (b < a.B) a.cu_new[b] = f0;
    }
    if (threadIdx.x == 0) {
        a.cu_new[a.B] = fresh;
        a.num_free_out[0] = top - taken;
    }
}

// ... and a second launch the slots, from what the first left.
__global__ void __launch_bounds__(256) fa_slot_kernel(PageTableArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.total_new) return;
    int64_t slot = -1;
    if (i < a.cu_new[a.B]) {
        const int b = seq_of(a.cu_new, a.B, (int)i);
        const int row = a.batch_idx ? a.batch_idx[b] : b;
        const int64_t at = (int64_t)max(a.before[b], 0) + (i - a.cu_new[b]);
        if (row >= 0 && row < a.table_rows && at < (int64_t)a.max_pages * a.page_size) {
            const int j = (int)udiv(a.page, (uint32_t)at);
            const int id = a.table[(int64_t)row * a.t_stride + j];
            if (id >= 0) slot = (int64_t)id * a.page_size + (at - (int64_t)j * a.page_size);
        }
    }
    a.slots[i] = slot;
}

}  // namespace

hipError_t launch_page_table(const PageTableArgs& a, hipStream_t stream) {
    if (a.B <= MAXB) {
        // two slots a thread, pages of 128 requests a workgroup: few enough that
        // what they all do stays small
        const int64_t grid = std::max<int64_t>((a.total_new + 2 * NT - 1) / (2 * NT), (a.B + 127) / 128);
        hipLaunchKernelGGL(fa_page_table_kernel, dim3((unsigned)std::min<int64_t>(grid, 256)), dim3(NT), 0, stream, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(fa_page_table_large_kernel, dim3(1), dim3(NT), 0, stream, a);
    if (a.total_new > 0)
        hipLaunchKernelGGL(fa_slot_kernel, dim3((unsigned)((a.total_new + 255) / 256)), dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace fa
