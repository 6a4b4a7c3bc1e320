// fa_fp4_attend.hip -- attention over the 4-bit cache, one wave for a query row of a head:
// 64 keys at a time, a lane's score of one of them, then the lanes' channels over all 64.
#include "fa_fp4.h"

#include <algorithm>

namespace fa {

namespace {

template <int DT>
__device__ __forceinline__ float fp4_value(const uint8_t* row, const uint8_t* scale, int d) {
    const uint32_t code = row[d >> 1] >> (4 * (d & 1)) & 15u;
    return f16_to_32<DT>((uint16_t)fp4_widen8<DT>(code, fp4_scale(scale[d / kGroup]))[0]);
}

template <int DT>
__global__ void __launch_bounds__(256) fa_fp4_attend_kernel(QuantFwdArgs a, int64_t row0, int64_t rows, bool few) {
    __shared__ float s_q[4][256], s_p[4][64];
    __shared__ int64_t s_v[4][64], s_vs[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t id = row0 + (int64_t)blockIdx.x * 4 + wave;
    if (id >= rows) return;
    const int h = (int)(id % a.H);
    const int64_t t = id / a.H;
    int b, i;
    if (a.cu_q) {
        if (t < a.cu_q[0] || t >= a.cu_q[a.B]) return;
        b = seq_of(a.cu_q, a.B, (int)t);
        i = (int)t - a.cu_q[b];
    } else {
        b = (int)(t / a.Sq);
        i = (int)(t % a.Sq);
    }
    const QuantSeq q = quant_seq(a, b);
    if (i < 0 || i >= q.sq || (q.sq * a.g <= a.dec_rows) != few) return;
    const int hk = h / a.g, d = i + q.sk - q.sq;
    const int lo = max(0, key_lo(d, a.wl, 0)), hi = min(q.sk - 1, key_hi(d, a.wr, 0));
    const uint16_t* qp = static_cast<const uint16_t*>(a.q) + q_row(a, b, i, a.q_sb, a.q_si) + (int64_t)h * a.q_sh;
    for (int c = lane; c < a.hd; c += 64) s_q[wave][c] = f16_to_32<DT>(qp[c]);
    const uint8_t *ks = reinterpret_cast<const uint8_t*>(a.ks), *vs = reinterpret_cast<const uint8_t*>(a.vs);
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int j0 = lo; j0 <= hi; j0 += 64) {
        const int j = j0 + lane;
        float x = -INFINITY;
        int64_t v = -1, vsc = 0;
        if (j <= hi) {
            const int pi = a.table ? (int)udiv(a.page, (uint32_t)j) : 0;
            const int64_t r = j - pi * a.page_size, p = a.table ? a.table[(int64_t)q.crow * a.t_stride + pi] : q.crow;
            if (p >= 0 && p < a.num_pages) {
                const uint8_t* kr = a.k + p * a.k_sp + r * a.k_si + (int64_t)hk * a.k_sh;
                const uint8_t* sr = ks + p * a.ks_sp + r * a.ks_sb + (int64_t)hk * a.ks_sh;
                v = p * a.v_sp + r * a.v_si + (int64_t)hk * a.v_sh;
                vsc = p * a.vs_sp + r * a.vs_sb + (int64_t)hk * a.vs_sh;
                float s = 0.f;
                for (int c = 0; c < a.hd; ++c) s = __builtin_fmaf(s_q[wave][c], fp4_value<DT>(kr, sr, c), s);
                x = a.softcap > 0.f ? a.softcap * kLog2e * fast_tanh(s * (a.scale / a.softcap)) : s * (a.scale * kLog2e);
            }
        }
        s_v[wave][lane] = v;
        s_vs[wave][lane] = vsc;
        float top = x;
        for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
        const float mn = fmaxf(m, top), u = mn == -INFINITY ? 0.f : mn;
        const float p = v >= 0 ? fast_exp2(x - u) : 0.f;
        s_p[wave][lane] = p;
        float sum = p;
        for (int k = 1; k < 64; k <<= 1) sum += __shfl_xor(sum, k);
        const float alpha = fast_exp2(m - u);
        l = l * alpha + sum;
        m = mn;
        for (int e = 0; e < 4; ++e) {
            const int c = lane + 64 * e;
            o[e] *= alpha;
            if (c >= a.hd) continue;
            for (int k = 0; k < 64; ++k) {
                const int64_t at = s_v[wave][k];
                if (at >= 0) o[e] = __builtin_fmaf(s_p[wave][k], fp4_value<DT>(a.v + at, vs + s_vs[wave][k], c), o[e]);
            }
        }
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    uint16_t* op = static_cast<uint16_t*>(a.out) + q_row(a, b, i, a.o_sb, a.o_si) + (int64_t)h * a.o_sh;
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < a.hd) op[lane + 64 * e] = f32_to_16<DT>(o[e] * inv);
    if (lane == 0) a.lse[lse_at(a, b, h, i)] = l != 0.f ? (m + fast_log2(l)) * kLn2 : INFINITY;
}

}  // namespace

static hipError_t launch_fp4_attend(const QuantFwdArgs& a, bool few, hipStream_t stream) {
    const int64_t rows = (a.cu_q ? (int64_t)a.total_q : (int64_t)a.B * a.Sq) * a.H, most = 1 << 24;
    for (int64_t r = 0; r < rows; r += most) {
        const dim3 grid((unsigned)((std::min(rows - r, most) + 3) / 4)), nt(256);
        const int64_t end = std::min(rows, r + most);
        if (a.bf16) hipLaunchKernelGGL(fa_fp4_attend_kernel<DT_BF16>, grid, nt, 0, stream, a, r, end, few);
        else hipLaunchKernelGGL(fa_fp4_attend_kernel<DT_FP16>, grid, nt, 0, stream, a, r, end, few);
    }
    return hipGetLastError();
}

hipError_t launch_fp4_prefill(const QuantFwdArgs& a, int, int, int, int, hipStream_t stream) { return launch_fp4_attend(a, false, stream); }

}  // namespace fa
