// fa_fp4_append.hip -- new k / v rows into the 4-bit cache: fa_fp4_append.
//
// A group of 32 channels of a row is quantised by itself: its scale is the smallest power of
// two s with max |x| <= 6 s, its codes are x / s (exact) rounded by the hardware's
// conversion, to the nearest with ties to the even code. Scales that are powers of two
// are what the format holds, and a token's own scales leave earlier tokens alone.
#include "fa_fp4.h"

#include <algorithm>

namespace fa {

namespace {

constexpr int kMostRows = 32;  // rows of a workgroup

// Four lanes hold a group, 8 channels each. Rows of a workgroup: their places first, then all
// their groups of k and v.
template <int DT>
__global__ void __launch_bounds__(256) fa_fp4_append_kernel(QuantAppendArgs a, int rows_per_group, UDiv per_row) {
    __shared__ int64_t s_at[4][kMostRows];  // k, v, their scales; -1: the row has no place
    constexpr uint32_t kInf = DT == DT_FP16 ? 0x7c00u : 0x7f80u;
    constexpr int kMost = DT == DT_FP16 ? 13 : 125;  // exponent of the largest scale
    const int64_t r0 = a.row0 + (int64_t)blockIdx.x * rows_per_group;
    const int n = (int)min((int64_t)rows_per_group, a.total_new - r0);
    if ((int)threadIdx.x < n) {
        const int64_t s = a.slots[r0 + threadIdx.x];
        const bool ok = s >= 0 && s < a.num_slots;
        const int64_t page = !ok ? 0 : a.num_slots <= 0xffffffffll ? (int64_t)udiv(a.page, (uint32_t)s) : s / a.page_size;
        const int64_t j = s - page * a.page_size;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            s_at[kv][threadIdx.x] = ok ? page * a.c_sp[kv] + j * a.c_si[kv] : -1;
            s_at[2 + kv][threadIdx.x] = page * a.s_sp[kv] + j * a.s_sb[kv];
        }
    }
    __syncthreads();
    for (uint32_t id = threadIdx.x; id < (uint32_t)n * per_row.d; id += 256) {
        const int r = (int)udiv(per_row, id);
        const uint32_t in = id - (uint32_t)r * per_row.d, h = udiv(a.chunks, in), c = in - h * a.chunks.d;
        if (s_at[0][r] == -1) continue;  // all four lanes
        u32x4 x[2];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
            x[kv] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.x[kv]) + (r0 + r) * a.x_si[kv] + (int64_t)h * a.x_sh[kv] + c * 8);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            // the largest |x| by its bits, which are in the order of the values, inf and NaN on top
            uint32_t most = 0;
            bool odd = false;
#pragma unroll
            for (int e = 0; e < 8; ++e) most = max(most, x[kv][e >> 1] >> (16 * (e & 1)) & 0x7fffu);
            most = max(most, (uint32_t)__shfl_xor((int)most, 1));
            most = max(most, (uint32_t)__shfl_xor((int)most, 2));
            odd = most >= kInf;
            const bool nan = most > kInf;
            most = min(most, kInf - 1);
            // most = m 2^e with 1 <= m < 2: s = 2^(e - 2), 2^(e - 1) where m > 1.5
            const uint32_t u = __builtin_bit_cast(uint32_t, f16_to_32<DT>((uint16_t)most));
            const int e = min(max((int)(u >> 23) - 127 - 2 + ((u & 0x7fffffu) > 0x400000u ? 1 : 0), -100), kMost);
            const float inv = exp2i(-e);
            uint32_t code = 0;
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                uint32_t b = x[kv][i >> 1] >> (16 * (i & 1)) & 0xffffu;
                if (odd && (b & 0x7fffu) >= kInf) b = (b & 0x8000u) | (kInf - 1);
                y[i] = f16_to_32<DT>((uint16_t)b) * inv;
            }
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[0], y[1], 1.f, 0);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[2], y[3], 1.f, 1);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[4], y[5], 1.f, 2);
            code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, y[6], y[7], 1.f, 3);
            *reinterpret_cast<uint32_t*>(a.c[kv] + s_at[kv][r] + (int64_t)h * a.c_sh[kv] + c * 4) = code;
            if (c % 4 == 0)
                reinterpret_cast<uint8_t*>(a.s[kv])[s_at[2 + kv][r] + (int64_t)h * a.s_sh[kv] + c / 4] = nan ? 255 : (uint8_t)(e + 127);
        }
    }
}

}  // namespace

hipError_t launch_fp4_append(QuantAppendArgs a, int dtype, hipStream_t stream) {
    a.page = udiv_make((uint32_t)a.page_size);
    a.chunks = udiv_make((uint32_t)a.hd / 8);
    const UDiv per_row = udiv_make((uint32_t)a.Hk * (uint32_t)(a.hd / 8));
    // several passes of a workgroup where there are workgroups enough for that
    const int rows = (int)std::min<int64_t>(std::max<int64_t>(a.total_new / 2048, 1), kMostRows);
    const int64_t groups = (a.total_new + rows - 1) / rows, most = 1 << 24;  // 2^32 threads of a launch
    for (int64_t g = 0; g < groups; g += most - 1) {
        a.row0 = g * rows;
        const dim3 grid((unsigned)std::min(groups - g, most - 1)), nt(256);
        if (dtype == DT_BF16) hipLaunchKernelGGL(fa_fp4_append_kernel<DT_BF16>, grid, nt, 0, stream, a, rows, per_row);
        else hipLaunchKernelGGL(fa_fp4_append_kernel<DT_FP16>, grid, nt, 0, stream, a, rows, per_row);
    }
    return hipGetLastError();
}

}  // namespace fa
