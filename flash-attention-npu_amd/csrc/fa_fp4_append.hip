// fa_fp4_append.hip -- new k / v rows into the 4-bit cache: fa_fp4_append.
//
// A group of 32 channels of a row is quantised by itself: its scale is the smallest power of
// two s with max |x| <= 6 s, its codes are x / s (exact) rounded by the hardware's
// conversion, to the nearest with ties to the even code. Scales that are powers of two
// are what the format holds, and a token's own scales leave earlier tokens alone.
//
// What bounds it: memory; a row is read once, a quarter of its bytes written. 41 000 rows of
// 8 heads x 128, bf16, take 55 us (3.9 TB/s; 42 at the rate of a copy); 64 rows 3.6, a launch.
// Two pieces of a row are in flight per thread, so that the second's loads lie under the first's maximum
// (one: 65 us for what 58 took, with fp32 conversions in place of the 16-bit pairs').
#include "fa_fp4.h"

#include <algorithm>

namespace fa {

namespace {

constexpr int kMostRows = 32;  // rows of a workgroup

// The largest |x| of a group, 8 values in each of four neighbouring lanes, by its bits: below the
// sign they are in the order of the values, inf and NaN on top.
__device__ __forceinline__ uint32_t group_most(u32x4 x) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    u16x2 m = {0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, x[e] & 0x7fff7fffu));
    uint32_t most = max((uint32_t)m[0], (uint32_t)m[1]);
    most = max(most, (uint32_t)__builtin_amdgcn_mov_dpp((int)most, 0xb1, 0xf, 0xf, true));  // lane ^ 1
    return max(most, (uint32_t)__builtin_amdgcn_mov_dpp((int)most, 0x4e, 0xf, 0xf, true));  // lane ^ 2
}

// Eight codes of x / s
template <int DT>
__device__ __forceinline__ uint32_t codes8(u32x4 x, float s) {
    const uint32_t x0 = x[0], x1 = x[1], x2 = x[2], x3 = x[3];  // (a bit cast of a vector's element takes the first)
    uint32_t r = 0;
    if constexpr (DT == DT_FP16) {
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, x0), s, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, x1), s, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, x2), s, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(r, __builtin_bit_cast(f16x2, x3), s, 3);
    } else {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, x0), s, 0);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, x1), s, 1);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, x2), s, 2);
        r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, x3), s, 3);
    }
    return r;
}

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
    // Two of a lane's pieces at a time, k and v of each: four loads are under way together.
    const uint32_t all = (uint32_t)n * per_row.d;
    for (uint32_t id0 = threadIdx.x; id0 < all; id0 += 512) {
        u32x4 x[2][2];
        int r[2], h[2], c[2];
        bool ok[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const uint32_t id = id0 + 256 * u;
            ok[u] = id < all;
            r[u] = ok[u] ? (int)udiv(per_row, id) : 0;
            const uint32_t in = ok[u] ? id - (uint32_t)r[u] * per_row.d : 0;
            h[u] = (int)udiv(a.chunks, in);
            c[u] = (int)(in - (uint32_t)h[u] * a.chunks.d);
            ok[u] = ok[u] && s_at[0][r[u]] != -1;  // alike in the four lanes of a group
#pragma unroll
            for (int kv = 0; kv < 2; ++kv)
                x[u][kv] = ok[u] ? *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.x[kv]) + (r0 + r[u]) * a.x_si[kv] +
                                                                   (int64_t)h[u] * a.x_sh[kv] + c[u] * 8)
                                 : u32x4{0u, 0u, 0u, 0u};
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int kv = 0; kv < 2; ++kv) {
                u32x4& y = x[u][kv];
                uint32_t most = group_most(y);
                const bool nan = most > kInf;
                if (__ballot(most >= kInf)) {
                    // inf, and NaN of whatever, as the largest finite value
                    if (most >= kInf) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if ((y[e >> 1] >> (16 * (e & 1)) & 0x7fffu) >= kInf)
                                y[e >> 1] = (y[e >> 1] & ~(0x7fffu << (16 * (e & 1)))) | (kInf - 1) << (16 * (e & 1));
                        most = kInf - 1;
                    }
                }
                // most = m 2^e with 1 <= m < 2: s = 2^(e - 2), 2^(e - 1) where m > 1.5
                const uint32_t b = __builtin_bit_cast(uint32_t, f16_to_32<DT>((uint16_t)most));
                const int e = min(max((int)(b >> 23) - 127 - 2 + ((b & 0x7fffffu) > 0x400000u ? 1 : 0), -100), kMost);
                const uint32_t code = codes8<DT>(y, exp2i(e));
                if (ok[u]) {
                    *reinterpret_cast<uint32_t*>(a.c[kv] + s_at[kv][r[u]] + (int64_t)h[u] * a.c_sh[kv] + c[u] * 4) = code;
                    if (c[u] % 4 == 0)
                        reinterpret_cast<uint8_t*>(a.s[kv])[s_at[2 + kv][r[u]] + (int64_t)h[u] * a.s_sh[kv] + c[u] / 4] = nan ? 255 : (uint8_t)(e + 127);
                }
            }
        }
    }
}

}  // namespace

hipError_t launch_fp4_append(QuantAppendArgs a, int dtype, hipStream_t stream) {
    a.page = udiv_make((uint32_t)a.page_size);
    a.chunks = udiv_make((uint32_t)a.hd / 8);
    const UDiv per_row = udiv_make((uint32_t)a.Hk * (uint32_t)(a.hd / 8));
    // Several rows to a workgroup, which looks up their places once, where there are workgroups enough for that:
    // 41 000 rows take 54.9 us at 1/4096 of them each, 58.1 at 1/1024, 57.5 at 1/2048, 53.9 at 1/8192
    const int rows = (int)std::min<int64_t>(std::max<int64_t>(a.total_new / 4096, 1), kMostRows);
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
