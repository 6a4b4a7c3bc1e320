// fa_quant_read.hip -- rows of a quantised cache as values of 16 or 32 bits: fa_quant_read.
//
// One pass: codes and scales in, values out, which are most of what moves (2 bytes
// for 0.53 of a 4-bit cache), and the rate of writes is what bounds it: 41 000 rows of 8 heads x 128 from
// a 4-bit cache to bf16 take 36 us (5.9 TB/s), 64 rows 3.5; 13 contexts of 5 heads x 96, 128 MB in all, 25 us
// from the last cache level and 35 from memory. Values are rounded once, from 32 bits.
#include "fa_fp4.h"
#include "fa_quant_read_args.h"

#include <algorithm>

namespace fa {

namespace {

constexpr int kMostRows = 32;  // rows of a workgroup
enum : int { DT_F32 = 2 };

// Eight codes under their scale, in fp32 (0 of a row that is not there: the codes and the scale are 0)
template <int CT>
__device__ __forceinline__ f32x8 values8(u32x2 w, float s) {
    f32x8 y;
    if constexpr (CT == CT_FP4) {
        const auto p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s, 0), p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s, 1),
                   p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s, 2), p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[0], s, 3);
        y[0] = p0[0], y[1] = p0[1], y[2] = p1[0], y[3] = p1[1], y[4] = p2[0], y[5] = p2[1], y[6] = p3[0], y[7] = p3[1];
    } else {
        const u32x2 lo = widen4<CT>(w[0]), hi = widen4<CT>(w[1]);  // exact in fp16
        y = widen8<DT_FP16>(u32x4{lo[0], lo[1], hi[0], hi[1]}) * s;
    }
    return y;
}

// A thread makes 8 channels of a row and head, of k and of v.
template <int OT, int CT>
__global__ void __launch_bounds__(256) fa_quant_read_kernel(QuantReadArgs a, int rows_per_group) {
    __shared__ int64_t s_at[4][kMostRows];  // k, v, their scales; -1: the row has no place
    const int64_t r0 = a.row0 + (int64_t)blockIdx.x * rows_per_group;
    const int n = (int)min((int64_t)rows_per_group, a.total - r0);
    if ((int)threadIdx.x < n) {
        const int64_t row = r0 + threadIdx.x;
        int64_t page = -1, j = 0;
        if (a.slots) {
            const int64_t s = a.slots[row];
            if (s >= 0 && s < a.num_slots) {
                page = a.num_slots <= 0xffffffffll ? (int64_t)udiv(a.page, (uint32_t)s) : s / a.page_size;
                j = s - page * a.page_size;
            }
        } else if (row >= a.cu[0] && row < a.cu[a.B]) {
            const int b = seq_of(a.cu, a.B, (int)row);
            const int64_t key = row - a.cu[b];  // below 0 where cu is no prefix sum
            int64_t at = b;
            if (a.batch_idx) at = a.batch_idx[b];
            if (at >= 0 && at < a.rows && key >= 0 && key < a.capacity) {
                const int64_t pi = udiv(a.page, (uint32_t)key);
                j = key - pi * a.page_size;
                page = a.table ? (int64_t)a.table[at * a.t_stride + pi] : at;
                if (page >= a.num_pages) page = -1;
            }
        }
        const bool ok = page >= 0;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            s_at[kv][threadIdx.x] = ok ? page * a.c_sp[kv] + j * a.c_si[kv] : -1;
            s_at[2 + kv][threadIdx.x] = ok ? page * a.s_sp[kv] + (CT == CT_FP4 ? j : (int64_t)udiv(a.sblk, (uint32_t)j)) * a.s_sb[kv] : 0;
        }
    }
    __syncthreads();
    // Two of a lane's pieces at a time, k and v of each: eight loads are under way together.
    const uint32_t all = (uint32_t)n * a.per_row.d;
    for (uint32_t id0 = threadIdx.x; id0 < all; id0 += 512) {
        u32x2 w[2][2];
        float s[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t id = id0 + 256 * u;
            const int r = id < all ? (int)udiv(a.per_row, id) : 0;
            const uint32_t in = id < all ? id - (uint32_t)r * a.per_row.d : 0, h = udiv(a.chunks, in), c = in - h * a.chunks.d;
            const bool ok = id < all && s_at[0][r] != -1;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                w[u][kv] = u32x2{0u, 0u};
                s[u][kv] = 0.f;
                if (ok) {
                    const uint8_t* codes = a.c[kv] + s_at[kv][r] + (int64_t)h * a.c_sh[kv];
                    const int64_t sat = s_at[2 + kv][r] + (int64_t)h * a.s_sh[kv];
                    if constexpr (CT == CT_FP4) {
                        w[u][kv][0] = *reinterpret_cast<const uint32_t*>(codes + c * 4);
                        s[u][kv] = fp4_scale(static_cast<const uint8_t*>(a.s[kv])[sat + c / 4]);
                    } else {
                        w[u][kv] = *reinterpret_cast<const u32x2*>(codes + c * 8);
                        s[u][kv] = static_cast<const float*>(a.s[kv])[sat];
                    }
                }
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t id = id0 + 256 * u;
            if (id >= all) break;
            const int64_t to = (r0 * (int64_t)a.per_row.d + id) * 8;
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                if constexpr (OT == DT_F32) {
                    const f32x8 y = values8<CT>(w[u][kv], s[u][kv]);
                    float* t = static_cast<float*>(a.o[kv]) + to;
                    *reinterpret_cast<f32x4*>(t) = f32x4{y[0], y[1], y[2], y[3]};
                    *reinterpret_cast<f32x4*>(t + 4) = f32x4{y[4], y[5], y[6], y[7]};
                } else {
                    u32x4* t = reinterpret_cast<u32x4*>(static_cast<uint16_t*>(a.o[kv]) + to);
                    if constexpr (CT == CT_FP4) *t = fp4_widen8<OT>(w[u][kv][0], s[u][kv]);
                    else *t = pack8<OT>(values8<CT>(w[u][kv], s[u][kv]));
                }
            }
        }
    }
}

template <int OT>
void launch_read_t(const QuantReadArgs& a, int ct, int rows, dim3 grid, hipStream_t stream) {
    const dim3 nt(256);
    if (ct == CT_FP4) hipLaunchKernelGGL((fa_quant_read_kernel<OT, CT_FP4>), grid, nt, 0, stream, a, rows);
    else if (ct == CT_INT8) hipLaunchKernelGGL((fa_quant_read_kernel<OT, CT_INT8>), grid, nt, 0, stream, a, rows);
    else hipLaunchKernelGGL((fa_quant_read_kernel<OT, CT_E4M3>), grid, nt, 0, stream, a, rows);
}

}  // namespace

hipError_t launch_quant_read(QuantReadArgs a, int dtype, int ct, hipStream_t stream) {
    // as in fa_fp4_append.hip: 41 000 rows take 36.0 us, 40.8 at 1/1024, 38.2 at 1/2048, 35.0 at 1/8192; the
    // 13 contexts 24.8, 23.8, 26.1 and 26.2
    const int rows = (int)std::min<int64_t>(std::max<int64_t>(a.total / 4096, 1), kMostRows);
    const int64_t groups = (a.total + rows - 1) / rows, most = (1 << 24) - 1;  // less than 2^32 threads of a launch
    for (int64_t g = 0; g < groups; g += most) {
        a.row0 = g * rows;
        const dim3 grid((unsigned)std::min(groups - g, most));
        if (dtype == DT_F32) launch_read_t<DT_F32>(a, ct, rows, grid, stream);
        else if (dtype == DT_BF16) launch_read_t<DT_BF16>(a, ct, rows, grid, stream);
        else launch_read_t<DT_FP16>(a, ct, rows, grid, stream);
    }
    return hipGetLastError();
}

}  // namespace fa
