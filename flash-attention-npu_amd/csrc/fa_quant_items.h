// fa_quant_items.h -- the work items of the prefill kernel over 8-bit codes: their
// list, their cut over the workgroups, and the merge of the pieces.
#pragma once
#include "fa_quant.h"
#include "fa_pipe.h"
#include "fa_quant_split.h"

#include <type_traits>

namespace fa {

namespace {

struct Rows {
    int rows, mt;
    QuantSeq q;
};

template <int BM>
__device__ __forceinline__ Rows rows_of(const QuantFwdArgs& a, int b) {
    Rows r;
    r.q = quant_seq(a, b);
    if (r.q.hi < r.q.lo) r.q.hi = r.q.lo;
    r.rows = r.q.sq * a.g > a.dec_rows ? r.q.sq * a.g : 0;
    r.mt = (r.rows + BM - 1) / BM;
    return r;
}

// Keys that rows [row0, row0 + n) see; those of a tile from base on
struct Keys {
    int lo, hi;
};
__device__ __forceinline__ Keys keys_of(const QuantFwdArgs& a, const QuantSeq& q, int row0, int n) {
    const int diag0 = q.sk - q.sq;
    Keys k;
    k.lo = max(0, key_lo(row0 / a.g + diag0, a.wl, 0));
    k.hi = max(k.lo, min(q.sk, key_hi((row0 + n - 1) / a.g + diag0, a.wr, 0) + 1));
    return k;
}
template <int BN>
__device__ __forceinline__ int tiles_of(const Keys& k) {
    return (k.hi - (k.lo & ~15) + BN - 1) / BN;  // tiles start at a block of 16 keys
}

template <typename T, typename X>
__device__ __forceinline__ int find_in(const T* s, int n, X x) {  // the last i of [0, n) with s[i] <= x
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// The list: an entry is a tile of BM rows of a sequence, an item an entry of one kv
// head. Every workgroup makes the list alike, in LDS.
// Ragged items, or few, are cut (fa_quant_split.h).
template <int BM, int BN, int NW>
__device__ void build_list(const QuantFwdArgs& a, int* s_pref, int64_t* s_line) {
    constexpr int NT = NW * 64;
    const int tid = threadIdx.x;
    for (int b = tid; b < a.B; b += NT) s_pref[b + 1] = rows_of<BM>(a, b).mt;
    __syncthreads();
    if (tid < 64) prefix_sums(s_pref, a.B);
    __syncthreads();
    if (!a.cut) return;
    const int n = min(s_pref[a.B], kQuantMaxB);
    for (int e = tid; e < n; e += NT) {
        const int b = find_in(s_pref, a.B, e);
        const Rows r = rows_of<BM>(a, b);
        const int mt = e - s_pref[b];
        const Keys k = keys_of(a, r.q, mt * BM, min(BM, r.rows - mt * BM));
        s_line[e + 1] = kStart + (int64_t)tiles_of<BN>(k) * (BN / 32);
    }
    __syncthreads();
    if (tid < 64) prefix_sums(s_line, n);
    __syncthreads();
}

// An item that was cut, left by the worker that holds its start for the merge
struct CutItem {
    int pieces, b, mt, hk;
};

// Merge of the pieces of cut items: the first is the second slot of the worker that
// left the item, the others the first slots of those after it. A thread for each row
// and 8 columns.
template <int DT, int HD, int BM>
__global__ void __launch_bounds__(256) fa_quant_prefill_merge_kernel(QuantFwdArgs a) {
    constexpr int DCH = HD / 8, RPB = 256 / DCH, BPT = BM / RPB;
    const int blk = blockIdx.x % BPT, w = blockIdx.x / BPT;
    const CutItem c = reinterpret_cast<const CutItem*>(a.pf_cut)[w];
    if (c.pieces == 0) return;
    const int sq = quant_seq(a, c.b).sq;
    const int rr = blk * RPB + threadIdx.x / DCH, d0 = threadIdx.x % DCH * 8, r = c.mt * BM + rr;
    if (r >= sq * a.g) return;
    auto row = [&](int s) { return (int64_t)(s == 0 ? 2 * w + 1 : 2 * (w + s)) * BM + rr; };
    float m = -INFINITY;
    bool some = false;  // a piece with a key for the row; one that is NaN has no part in the maximum
    for (int s = 0; s < c.pieces; ++s) {
        const float v = a.pf_lse[row(s)];
        m = fmaxf(m, v);
        some |= v != -INFINITY;
    }
    f32x4 acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
    float lse = INFINITY;
    if (some) {
        float sum = 0.f;
        for (int s = 0; s < c.pieces; ++s) {
            const float wgt = fast_exp2((a.pf_lse[row(s)] - m) * kLog2e);
            sum += wgt;
            acc0 += *reinterpret_cast<const f32x4*>(a.pf_o + row(s) * HD + d0) * wgt;
            acc1 += *reinterpret_cast<const f32x4*>(a.pf_o + row(s) * HD + d0 + 4) * wgt;
        }
        acc0 *= 1.f / sum;
        acc1 *= 1.f / sum;
        lse = m + fast_log2(sum) * kLn2;
    }
    const int i = r / a.g, h = c.hk * a.g + r % a.g;
    uint16_t* o = static_cast<uint16_t*>(a.out) + q_row(a, c.b, i, a.o_sb, a.o_si) + (int64_t)h * a.o_sh;
    if (d0 < a.hd)
        *reinterpret_cast<u32x4*>(o + d0) = u32x4{pack2<DT>(acc0[0], acc0[1]), pack2<DT>(acc0[2], acc0[3]),
                                                  pack2<DT>(acc1[0], acc1[1]), pack2<DT>(acc1[2], acc1[3])};
    if (d0 == 0) a.lse[lse_at(a, c.b, h, i)] = lse;
}

template <int DT, int HD, int BM>
void launch_items_merge(const QuantFwdArgs& a, int grid, hipStream_t stream) {
    if (!a.cut) return;
    constexpr int RPB = 256 / (HD / 8);
    hipLaunchKernelGGL((fa_quant_prefill_merge_kernel<DT, HD, BM>), dim3((unsigned)(grid * (BM / RPB))), dim3(256), 0, stream, a);
}

}  // namespace

}  // namespace fa
