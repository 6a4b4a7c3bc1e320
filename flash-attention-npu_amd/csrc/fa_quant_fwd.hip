// fa_quant_fwd.hip -- attention over a cache of 8-bit codes: fa_quant_fwd.
//
// With c the codes and s, t the scales of K and V,
//   x_j = softmax_scale * s_j (q . ck_j),  out = sum_j e^(x_j - m) t_j cv_j / sum_j e^(x_j - m),
// kept in fp32 with a running maximum m. One workgroup for each query row and head.
#include "fa_common.h"
#include "fa_quant_args.h"

namespace fa {

namespace {

constexpr int NT = 256;

template <int CT>
__device__ __forceinline__ float code_value(uint8_t c) {
    if constexpr (CT == CT_INT8) return (float)(int8_t)c;
    else return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
}

__device__ __forceinline__ float block_reduce(float v, bool is_max, float* s_r) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const float u = __shfl_xor(v, o);
        v = is_max ? fmaxf(v, u) : v + u;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_r[threadIdx.x >> 6] = v;
    __syncthreads();
    const float x = is_max ? fmaxf(s_r[0], s_r[1]) : s_r[0] + s_r[1], y = is_max ? fmaxf(s_r[2], s_r[3]) : s_r[2] + s_r[3];
    return is_max ? fmaxf(x, y) : x + y;
}

template <int DT, int CT>
__global__ void __launch_bounds__(NT) fa_quant_fwd_kernel(QuantFwdArgs a) {
    __shared__ float s_q[256], s_p[NT], s_r[4];
    __shared__ int64_t s_row[NT];
    const int tid = threadIdx.x, h = blockIdx.y, hk = h / a.g;
    int b, i, sq;
    int64_t T = blockIdx.x;
    if (a.cu_q) {
        b = seq_of(a.cu_q, a.B, (int)T);
        i = (int)T - a.cu_q[b];
        sq = min(a.cu_q[b + 1] - a.cu_q[b], a.Sq);
        if (i < 0 || i >= sq) return;
    } else {
        b = (int)(T / a.Sq);
        i = (int)(T % a.Sq);
        sq = a.Sq;
    }
    if (sq * a.g <= a.dec_rows) return;
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (a.cu_q ? T * a.q_si : (int64_t)b * a.q_sb + (int64_t)i * a.q_si) +
                        (int64_t)h * a.q_sh;
    if (tid < a.hd) s_q[tid] = f16_to_32<DT>(q[tid]);
    const int sk = min(max(a.seqlens[b], 0), a.capacity);
    const int row = a.batch_idx ? min(max(a.batch_idx[b], 0), a.rows - 1) : a.row0 + b;
    const int d = i + sk - sq;
    const int lo = max(0, key_lo(d, a.wl, 0)), hi = min(sk, key_hi(d, a.wr, 0) + 1);
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int j0 = lo; j0 < hi; j0 += NT) {
        __syncthreads();
        const int j = j0 + tid;
        float x = -INFINITY, t = 0.f;
        s_row[tid] = -1;
        if (j < hi) {
            const int pi = a.table ? (int)udiv(a.page, (uint32_t)j) : 0;
            const int id = a.table ? a.table[(int64_t)row * a.t_stride + pi] : row;
            if (id >= 0 && id < a.num_pages) {
                const int inp = j - pi * a.page_size, sb = (int)udiv(a.sblk, (uint32_t)inp);
                const uint8_t* k = a.k + (int64_t)id * a.k_sp + (int64_t)inp * a.k_si + (int64_t)hk * a.k_sh;
                float s = 0.f;
                for (int e = 0; e < a.hd; ++e) s += s_q[e] * code_value<CT>(k[e]);
                x = s * (a.scale * a.ks[(int64_t)id * a.ks_sp + (int64_t)sb * a.ks_sb + (int64_t)hk * a.ks_sh]);
                if (a.softcap > 0.f) x = a.softcap * tanhf(x / a.softcap);
                t = a.vs[(int64_t)id * a.vs_sp + (int64_t)sb * a.vs_sb + (int64_t)hk * a.vs_sh];
                s_row[tid] = (int64_t)id * a.v_sp + (int64_t)inp * a.v_si;
            }
        }
        const float mn = fmaxf(m, block_reduce(x, true, s_r));
        if (mn == -INFINITY) continue;
        const float p = expf(x - mn), c = expf(m - mn);
        l = l * c + block_reduce(p, false, s_r);
        acc *= c;
        m = mn;
        s_p[tid] = p * t;
        __syncthreads();
        if (tid < a.hd)
            for (int u = 0; u < NT; ++u)
                if (s_row[u] >= 0) acc += s_p[u] * code_value<CT>(a.v[s_row[u] + (int64_t)hk * a.v_sh + tid]);
    }
    uint16_t* o = static_cast<uint16_t*>(a.out) + (a.cu_q ? T * a.o_si : (int64_t)b * a.o_sb + (int64_t)i * a.o_si) +
                  (int64_t)h * a.o_sh;
    if (tid < a.hd) o[tid] = f32_to_16<DT>(l > 0.f ? acc / l : 0.f);
    if (tid == 0)
        a.lse[a.cu_q ? (int64_t)h * a.lse_sh + T : (int64_t)b * a.lse_sb + (int64_t)h * a.lse_sh + i] =
            l > 0.f ? m + logf(l) : INFINITY;
}

}  // namespace

hipError_t launch_quant_fwd(const QuantFwdArgs& a, int dtype, int ct, hipStream_t stream) {
    const dim3 grid(a.cu_q ? (unsigned)a.total_q : (unsigned)a.B * (unsigned)a.Sq, (unsigned)a.H);
    if (dtype == DT_BF16) {
        if (ct == CT_INT8) hipLaunchKernelGGL((fa_quant_fwd_kernel<DT_BF16, CT_INT8>), grid, dim3(NT), 0, stream, a);
        else hipLaunchKernelGGL((fa_quant_fwd_kernel<DT_BF16, CT_E4M3>), grid, dim3(NT), 0, stream, a);
    } else {
        if (ct == CT_INT8) hipLaunchKernelGGL((fa_quant_fwd_kernel<DT_FP16, CT_INT8>), grid, dim3(NT), 0, stream, a);
        else hipLaunchKernelGGL((fa_quant_fwd_kernel<DT_FP16, CT_E4M3>), grid, dim3(NT), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace fa
