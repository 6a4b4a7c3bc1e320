// fa_quant_items.h -- the work items of the prefill kernels over 8-bit codes: their
// list, their split over the keys, and the merge of the pieces.
#pragma once
#include "fa_quant.h"
#include "fa_pipe.h"

#include <type_traits>

namespace fa {

namespace {

constexpr int kQuantMaxB = 2048;  // sequences of a launch: their list lives in LDS

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

__device__ __forceinline__ void split_of(const QuantFwdArgs& a, int range, int chunk_auto, int& ns, int& chunk) {
    chunk = chunk_auto;
    ns = a.allow_split && range > 0 ? (range + chunk - 1) / chunk : 1;
}

// The list of work items: prefix over the sequences in LDS, made by every
// workgroup alike; workgroup 0 leaves it for the merge. Keys are cut into chunks so
// that there are about target_items pieces, none under min_chunk keys.
template <int BM, int BN, int NW>
__device__ void build_list(const QuantFwdArgs& a, int* s_pref, long long* s_red, int& total, int& chunk_auto) {
    constexpr int NT = NW * 64;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    chunk_auto = 0x3fffffff;
    if (a.allow_split) {
        long long work = 0;
        for (int b = tid; b < a.B; b += NT) {
            const Rows r = rows_of<BM>(a, b);
            work += (long long)a.Hk * r.mt * (r.q.hi - r.q.lo);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) work += __shfl_xor(work, o);
        if (lane == 0) s_red[wave] = work;
        __syncthreads();
        work = 0;
        for (int w = 0; w < NW; ++w) work += s_red[w];
        long long c = (work + a.target_items - 1) / a.target_items;
        c = c < a.min_chunk ? a.min_chunk : c;
        c = (c + BN - 1) / BN * BN;
        chunk_auto = (int)(c > 0x3fffffff ? 0x3fffffff : c);
    }
    for (int b = tid; b < a.B; b += NT) {
        const Rows r = rows_of<BM>(a, b);
        int ns, chunk;
        split_of(a, r.q.hi - r.q.lo, chunk_auto, ns, chunk);
        s_pref[b + 1] = a.Hk * r.mt * ns;
        if (blockIdx.x == 0 && a.allow_split) a.pf_sched[a.B + 1 + b] = ns;
    }
    __syncthreads();
    if (wave == 0) {
        const int seg = (a.B + 63) / 64, b0 = lane * seg;
        int local = 0;
        for (int k = 0; k < seg; ++k)
            if (b0 + k < a.B) local += s_pref[b0 + k + 1];
        int incl = local;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o);
            if (lane >= o) incl += v;
        }
        int run = incl - local;
        for (int k = 0; k < seg; ++k)
            if (b0 + k < a.B) {
                run += s_pref[b0 + k + 1];
                s_pref[b0 + k + 1] = run;
            }
        if (lane == 0) s_pref[0] = 0;
    }
    __syncthreads();
    total = s_pref[a.B];
    if (blockIdx.x == 0 && a.allow_split)
        for (int b = tid; b <= a.B; b += NT) a.pf_sched[b] = s_pref[b];
}

// Merge of split items: a thread for each row and 8 columns.
template <int DT, int HD, int BM>
__global__ void __launch_bounds__(256) fa_quant_prefill_merge_kernel(QuantFwdArgs a, int mt_max) {
    constexpr int DCH = HD / 8, RPB = 256 / DCH, BPT = BM / RPB;
    const int blk = blockIdx.x % BPT, item = blockIdx.x / BPT;
    const int hk = item % a.Hk, mt = item / a.Hk % mt_max, b = item / a.Hk / mt_max;
    const int ns = a.pf_sched[a.B + 1 + b];
    if (ns <= 1) return;
    int sq = a.cu_q ? a.cu_q[b + 1] - a.cu_q[b] : a.Sq;
    sq = min(max(sq, 0), a.Sq);
    const int rows = sq * a.g > a.dec_rows ? sq * a.g : 0, mt_b = (rows + BM - 1) / BM;
    const int rr = blk * RPB + threadIdx.x / DCH, d0 = threadIdx.x % DCH * 8, r = mt * BM + rr;
    if (mt >= mt_b || r >= rows) return;
    const int w0 = a.pf_sched[b] + (mt_b - 1 - mt) * ns * a.Hk + hk;
    float m = -INFINITY;
    for (int s = 0; s < ns; ++s) m = fmaxf(m, a.pf_lse[(int64_t)(w0 + s * a.Hk) * BM + rr]);
    f32x4 acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
    float lse = INFINITY;
    if (m != -INFINITY) {
        float sum = 0.f;
        for (int s = 0; s < ns; ++s) {
            const int64_t prow = (int64_t)(w0 + s * a.Hk) * BM + rr;
            const float wgt = fast_exp2((a.pf_lse[prow] - m) * kLog2e);
            sum += wgt;
            acc0 += *reinterpret_cast<const f32x4*>(a.pf_o + prow * HD + d0) * wgt;
            acc1 += *reinterpret_cast<const f32x4*>(a.pf_o + prow * HD + d0 + 4) * wgt;
        }
        acc0 *= 1.f / sum;
        acc1 *= 1.f / sum;
        lse = m + fast_log2(sum) * kLn2;
    }
    const int i = r / a.g, h = hk * a.g + r % a.g;
    uint16_t* o = static_cast<uint16_t*>(a.out) + q_row(a, b, i, a.o_sb, a.o_si) + (int64_t)h * a.o_sh;
    if (d0 < a.hd)
        *reinterpret_cast<u32x4*>(o + d0) = u32x4{pack2<DT>(acc0[0], acc0[1]), pack2<DT>(acc0[2], acc0[3]),
                                                  pack2<DT>(acc1[0], acc1[1]), pack2<DT>(acc1[2], acc1[3])};
    if (d0 == 0) a.lse[lse_at(a, b, h, i)] = lse;
}

template <int DT, int HD, int BM>
void launch_items_merge(const QuantFwdArgs& a, int mt_max, hipStream_t stream) {
    if (!a.allow_split) return;
    constexpr int RPB = 256 / (HD / 8);
    hipLaunchKernelGGL((fa_quant_prefill_merge_kernel<DT, HD, BM>), dim3((unsigned)(a.B * mt_max * a.Hk * (BM / RPB))), dim3(256), 0,
                       stream, a, mt_max);
}

}  // namespace

}  // namespace fa
