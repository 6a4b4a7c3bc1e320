// fa_quant_list.h -- what the decode kernels over 8-bit and 4-bit codes share: the list
// of tiles that their waves split (fa_quant_split.h), where a tile lies in it, and
// the merge of what the waves of a sequence left.
#pragma once
#include "fa_quant.h"
#include "fa_pipe.h"
#include "fa_quant_split.h"

namespace fa {

namespace {

// kv heads whose tiles neighbouring waves take: a key's rows of them lie side by side
__device__ __forceinline__ int heads_per_group(const QuantFwdArgs& a) { return a.Hk % 4 == 0 ? 4 : a.Hk % 2 == 0 ? 2 : 1; }

struct Seg {
    int S, n;      // first tile of the list, tiles
    int b, hk;
    int lo_tile;
    QuantSeq q;    // of a block of rows: lo and hi are the block's
    int row0, rows;  // packed rows
};

__device__ __forceinline__ Seg seg_of(const QuantFwdArgs& a, const int* s_pref, int t, int hs, int h, int KT) {
    int bl = 0, bh = a.B;
    while (bh - bl > 1) {
        const int mid = (bl + bh) >> 1;
        if (s_pref[mid] <= t) bl = mid;
        else bh = mid;
    }
    Seg s;
    s.b = bl;
    s.q = quant_seq(a, bl);
    s.lo_tile = s.q.lo / KT;
    s.n = (s.q.hi + KT - 1) / KT - s.lo_tile;
    const int hg = (int)((uint32_t)(t - s_pref[bl]) / (uint32_t)max(s.n, 1));
    s.hk = hg * hs + h;
    s.S = s_pref[bl] + hg * s.n;
    s.row0 = 0;
    s.rows = s.q.sq * a.g;
    return s;
}

// the last i of [0, n) with s[i] <= x
template <typename T>
__device__ __forceinline__ int place_of(const T* s, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Longer sequences, in blocks of kBlockRows packed rows that read their keys each for itself. A tile costs the
// decode kernel twice what its rows cost the prefill kernel, but that one begins 40 us later: it executes 2700
// instructions before its first product, and fetches each line of them for the first time. Prompts of 64, 128,
// 256 and 512 tokens of 32 heads onto 8 take 30, 30, 35 and 43 us in place of 53, 56, 59 and 68, one of 1024, if it were let,
// 96 in place of 85; 256 tokens that end 4000 keys 67 in place of 73, 16000 keys 163 in place of 110; 8
// prompts of 256 tokens, of which each wave has several blocks, 89 in place of 36. The number of blocks is the
// host's to bound (kBlockSegs); the keys every workgroup of both kernels counts, alike (kBlockUnits). A call
// whose blocks are not taken after all costs 3 to 10 us more. At head dims 64, 128 and 256, with 32, 64 and 8 heads
// onto 8 and 16 onto 1, 64 to 1024 tokens behind none to 16000 keys, calls with the rule take 0.69, 0.73 and 0.78 of what they
// take without on average, 1.11 at worst (D256, 64 heads onto 8, 128 tokens after 4000 keys: 125 for 113).
__device__ __forceinline__ int blocks_of(const QuantFwdArgs& a, const QuantSeq& q) {
    return (q.sq * a.g + kBlockRows - 1) / kBlockRows;
}

// by a whole workgroup of NT threads
template <int NT>
__device__ __forceinline__ bool blocks_take(const QuantFwdArgs& a, int64_t* s_sum) {
    int64_t units = 0;
    for (int b = threadIdx.x; b < a.B; b += NT) {
        const QuantSeq q = quant_seq(a, b);
        units += (int64_t)a.Hk * blocks_of(a, q) * max((q.hi - q.lo) / 64, 1);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) units += (int64_t)__shfl_xor((long long)units, o);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = units;
    __syncthreads();
    units = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) units += s_sum[w];
    __syncthreads();
    return units <= kBlockUnits;
}

// Block i of sequence b: q's keys become those that its rows see.
__device__ __forceinline__ void cut_to_block(const QuantFwdArgs& a, Seg& s, int i) {
    s.row0 = i * kBlockRows;
    s.rows = min(s.q.sq * a.g - s.row0, kBlockRows);
    const int diag = s.q.sk - s.q.sq;
    s.q.lo = max(0, key_lo(s.row0 / a.g + diag, a.wl, 0));
    s.q.hi = max(s.q.lo, min(s.q.sk, key_hi((s.row0 + s.rows - 1) / a.g + diag, a.wr, 0) + 1));
}

// Segment of tile t of the list of blocks: s_blk blocks before each sequence, s_pref tiles before each of n blocks
__device__ __forceinline__ Seg block_seg_of(const QuantFwdArgs& a, const int* s_blk, const int* s_pref, int n, int t, int hs, int h,
                                            int KT) {
    const int e = place_of(s_pref, n, t);
    Seg s;
    s.b = place_of(s_blk, a.B, e);
    s.q = quant_seq(a, s.b);
    cut_to_block(a, s, e - s_blk[s.b]);
    s.lo_tile = s.q.lo / KT;
    s.n = (s.q.hi + KT - 1) / KT - s.lo_tile;
    const int hg = (int)((uint32_t)(t - s_pref[e]) / (uint32_t)max(s.n, 1));
    s.hk = hg * hs + h;
    s.S = s_pref[e] + hg * s.n;
    return s;
}

// max over the lanes l, l ^ 16, l ^ 32, l ^ 48. A swap exchanges the odd rows of 16
// (32) lanes of one register with the even ones of the other. In assembly, since the
// compiler's builtin gives the first result for both; it wants two wait states after
// its operands' last write.
__device__ __forceinline__ float max4(float v) {
    float w = v;
    asm("s_nop 1\n\tv_permlane16_swap_b32 %0, %1" : "+v"(v), "+v"(w));
    v = w = fmaxf(v, w);
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %1" : "+v"(v), "+v"(w));
    return fmaxf(v, w);
}

// Merge of what a segment's workers left: 16 rows and 32 columns of a segment per
// workgroup; groups of threads fold a share of the partials each, with a running
// maximum, and meet in LDS. A row is empty where its weights sum to 0, which says so
// for NaN as well: such partials have no part in the maximum (fmaxf).
// KT: keys of a tile, NWAVE: waves of a workgroup of the kernel that left them, MT: threads of a workgroup, BLK: the list is of blocks.
template <int DT, int HD, int KT, int NWAVE, int MT, bool BLK>
__global__ void __launch_bounds__(MT) fa_quant_merge_kernel(QuantFwdArgs a, int grid, int nr) {
    __shared__ __attribute__((aligned(16))) float s_acc[MT][8];
    __shared__ float s_gm[MT], s_gs[MT];
    constexpr int COLS = HD / 32, CH = 4;  // 8-column chunks of a workgroup
    const int sig = blockIdx.x / COLS, part = blockIdx.x % COLS;
    const int e = (int)((uint32_t)sig / (uint32_t)a.Hk), hk = sig - e * a.Hk;  // sequence, or block
    const int hs = heads_per_group(a), hg = hk / hs, hsel = hk - hg * hs;
    int b = e, last = a.B, first = 0;  // first: the block's first row
    QuantSeq q;
    if constexpr (BLK) {
        last = min(a.block_pref[a.B], a.blocks);
        if (e >= last) return;
        Seg s;
        b = place_of(a.block_pref, a.B, e);
        s.q = quant_seq(a, b);
        cut_to_block(a, s, e - a.block_pref[b]);
        q = s.q;
        first = s.row0;
    } else {
        q = quant_seq(a, b);
    }
    const int T = a.sched[last], S0 = a.sched[e];
    const int row0 = blockIdx.y * 16, rows = min(q.sq * a.g - first - row0, 16);
    if (T < 0 || rows <= 0 || (!BLK && q.sq * a.g > a.dec_rows)) return;
    const int per = q.hi > q.lo ? (q.hi + KT - 1) / KT - q.lo / KT : 0, S = S0 + hg * per;
    const Split sp = split_list(T, grid * (NWAVE / hs));
    int wf = 0, n = 0;
    if (per > 0) {
        wf = sp.owner(S);
        n = sp.owner(S + per - 1) - wf + 1;
        if (n == 1) return;  // written by its one worker
    }
    const bool slot1 = per > 0 && sp.first(wf) < S;  // the first partial is its worker's last
    const int tid = threadIdx.x;
    int rp = 1;
    while (rp < rows) rp <<= 1;
    const int GS = CH * rp, NG = MT / GS;
    const int grp = tid / GS, rr = tid % GS / CH, d0 = part * 32 + tid % CH * 8;
    float m = -INFINITY, sum = 0.f;
    f32x4 acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
    if (rr < rows) {
#pragma unroll 4
        for (int j = grp; j < n; j += NG) {
            const int64_t pr = (((int64_t)(wf + j) * hs + hsel) * 2 + (j == 0 && slot1 ? 1 : 0)) * (16 * nr) + row0 + rr;
            const float v = a.part_lse[pr];
            const f32x4 o0 = *reinterpret_cast<const f32x4*>(a.part_o + pr * HD + d0);
            const f32x4 o1 = *reinterpret_cast<const f32x4*>(a.part_o + pr * HD + d0 + 4);
            if (v != -INFINITY) {
                const float mn = fmaxf(m, v);
                const float c = fast_exp2((m - mn) * kLog2e), wgt = fast_exp2((v - mn) * kLog2e);
                acc0 = acc0 * c + o0 * wgt;
                acc1 = acc1 * c + o1 * wgt;
                sum = sum * c + wgt;
                m = mn;
            }
        }
    }
    *reinterpret_cast<f32x4*>(&s_acc[tid][0]) = acc0;
    *reinterpret_cast<f32x4*>(&s_acc[tid][4]) = acc1;
    s_gm[tid] = m;
    s_gs[tid] = sum;
    // halve the groups until one is left
    for (int half = NG / 2; half > 0; half /= 2) {
        __syncthreads();
        if (grp < half) {
            const int o = tid + half * GS;
            const float mo = s_gm[o], M = fmaxf(m, mo);
            if (s_gs[o] != 0.f || sum != 0.f) {
                const float c = fast_exp2((m - M) * kLog2e), co = fast_exp2((mo - M) * kLog2e);
                acc0 = acc0 * c + *reinterpret_cast<const f32x4*>(&s_acc[o][0]) * co;
                acc1 = acc1 * c + *reinterpret_cast<const f32x4*>(&s_acc[o][4]) * co;
                sum = sum * c + s_gs[o] * co;
                m = M;
                *reinterpret_cast<f32x4*>(&s_acc[tid][0]) = acc0;
                *reinterpret_cast<f32x4*>(&s_acc[tid][4]) = acc1;
                s_gm[tid] = m;
                s_gs[tid] = sum;
            }
        }
    }
    if (grp != 0 || rr >= rows) return;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    acc0 *= inv;
    acc1 *= inv;
    const int r = first + row0 + rr, i = r / a.g, h = hk * a.g + r % a.g;
    uint16_t* o = static_cast<uint16_t*>(a.out) + q_row(a, b, i, a.o_sb, a.o_si) + (int64_t)h * a.o_sh;
    if (d0 < a.hd)
        *reinterpret_cast<u32x4*>(o + d0) = u32x4{pack2<DT>(acc0[0], acc0[1]), pack2<DT>(acc0[2], acc0[3]),
                                                  pack2<DT>(acc1[0], acc1[1]), pack2<DT>(acc1[2], acc1[3])};
    if (d0 == 0) a.lse[lse_at(a, b, h, i)] = sum == 0.f ? INFINITY : m + fast_log2(sum) * kLn2;
}

constexpr int kMergeThreads = 512;
template <int DT, int HD, int KT, int NWAVE, int MT = kMergeThreads, bool BLK = false>
void launch_list_merge(const QuantFwdArgs& a, int nr, int grid, hipStream_t stream) {
    hipLaunchKernelGGL((fa_quant_merge_kernel<DT, HD, KT, NWAVE, MT, BLK>), dim3((BLK ? a.blocks : a.B) * a.Hk * (HD / 32), nr), dim3(MT), 0, stream, a, grid, nr);
}

}  // namespace

}  // namespace fa
