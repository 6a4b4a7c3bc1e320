// fa_quant_append.hip -- new k / v rows into a cache of 8-bit codes with a
// scale for each block of tokens and kv head: fa_quant_append.
//
// The scale of a block is a power of two: x / s and c * s are then exact, a block
// that is filled one token at a time keeps its codes until a value outgrows its
// range, and where it does, its codes move by whole bits, so the roundings of
// repeated growth add up to less than one step (with max |x| / m, every token
// that is a new largest would round the whole block again). It costs at most one
// bit of the range.
#include "fa_common.h"
#include "fa_quant_args.h"

namespace fa {

namespace {

constexpr float kFloorScale = 0x1p-100f;

template <int CT>
constexpr float code_max() { return CT == CT_INT8 ? 127.f : 448.f; }

// the smallest power of two s >= 2^-100 with most <= s * m, m = 127 or 448
template <int CT>
__device__ __forceinline__ float scale_for(float most) {
    // m = 1.984375 * 2^6 or 1.75 * 2^8: exponent of most less that of m, one more
    // where the mantissa of most is the larger
    constexpr int me = CT == CT_INT8 ? 6 : 8;
    constexpr uint32_t mm = CT == CT_INT8 ? 0x7e0000u : 0x600000u;
    const uint32_t u = __builtin_bit_cast(uint32_t, most);
    const int e = (int)(u >> 23) - me + ((u & 0x7fffffu) > mm ? 1 : 0);
    return __builtin_bit_cast(float, (uint32_t)max(e, 27) << 23);  // 27: 2^-100; a subnormal most has u >> 23 = 0
}

template <int CT>
__device__ __forceinline__ float clamp_code(float y) {
    return fminf(fmaxf(y, -code_max<CT>()), code_max<CT>());
}

// four codes of y, rounded to nearest even, in one word
template <int CT>
__device__ __forceinline__ uint32_t codes4(const float (&y)[4]) {
    if constexpr (CT == CT_INT8) {
        uint32_t r = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float c = __builtin_isnan(y[i]) ? 0.f : clamp_code<CT>(y[i]);
            r |= ((uint32_t)(int)__builtin_rintf(c) & 0xffu) << (8 * i);
        }
        return r;
    } else {
        float c[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] = __builtin_isnan(y[i]) ? y[i] : clamp_code<CT>(y[i]);
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(c[0], c[1], 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(c[2], c[3], r, true);
        return (uint32_t)r;
    }
}

template <int CT>
__device__ __forceinline__ void values4(uint32_t w, float (&y)[4]) {
    if constexpr (CT == CT_INT8) {
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (float)(int8_t)(w >> (8 * i));
    } else {
        y[0] = __builtin_amdgcn_cvt_f32_fp8((int)w, 0);
        y[1] = __builtin_amdgcn_cvt_f32_fp8((int)w, 1);
        y[2] = __builtin_amdgcn_cvt_f32_fp8((int)w, 2);
        y[3] = __builtin_amdgcn_cvt_f32_fp8((int)w, 3);
    }
}

// One wave for each (row, head, k or v); the waves of rows that begin no run end
// at once.
template <int DT, int CT>
__global__ void __launch_bounds__(64) fa_quant_append_kernel(QuantAppendArgs a) {
    const int lane = threadIdx.x;
    const int64_t i0 = blockIdx.x;
    const int h = blockIdx.y, kv = blockIdx.z;
    auto block_of = [&](int64_t i) -> int64_t {
        const int64_t s = a.slots[i];
        return s >= 0 && s < a.num_slots ? s / a.scale_block : -1;
    };
    const int64_t blk = block_of(i0);
    if (blk < 0 || (i0 > 0 && block_of(i0 - 1) == blk)) return;
    int64_t i1 = i0 + 1;
    while (i1 < a.total_new && block_of(i1) == blk) ++i1;

    const int64_t row0 = blk * a.scale_block;  // first row of the block
    const int64_t page = row0 / a.page_size;
    const int inp = (int)(row0 - page * a.page_size);
    uint8_t* cache = a.c[kv] + page * a.c_sp[kv] + (int64_t)inp * a.c_si[kv] + (int64_t)h * a.c_sh[kv];
    float* sp = a.s[kv] + page * a.s_sp[kv] + (int64_t)(inp / a.scale_block) * a.s_sb[kv] + (int64_t)h * a.s_sh[kv];
    const uint16_t* x = static_cast<const uint16_t*>(a.x[kv]) + i0 * a.x_si[kv] + (int64_t)h * a.x_sh[kv];
    const int ch = a.hd / 8, n = (int)(i1 - i0) * ch;

    constexpr float kBig = DT == DT_FP16 ? 65504.f : 0x1.fep127f;
    auto load8 = [&](int idx, float (&y)[8]) {
        const u32x4 r = *reinterpret_cast<const u32x4*>(x + (int64_t)(idx / ch) * a.x_si[kv] + (idx % ch) * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float f = f16_to_32<DT>((uint16_t)(r[e >> 1] >> (16 * (e & 1))));
            y[e] = __builtin_isinf(f) ? copysignf(kBig, f) : f;
        }
    };
    float most = 0.f;
    for (int idx = lane; idx < n; idx += 64) {
        float y[8];
        load8(idx, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(y[e]));  // NaN is left out
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o));

    const int first = (int)(a.slots[i0] - row0);
    float s = scale_for<CT>(most);
    if (first > 0) {
        const float old = *sp;
        if (old >= s) {
            s = old;
        } else {
            const int hc = a.hd / 4;
            for (int idx = lane; idx < first * hc; idx += 64) {
                uint32_t* w = reinterpret_cast<uint32_t*>(cache + (int64_t)(idx / hc) * a.c_si[kv] + (idx % hc) * 4);
                float y[4];
                values4<CT>(*w, y);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] *= old / s;
                *w = codes4<CT>(y);
            }
        }
    }
    if (lane == 0) *sp = s;
    for (int idx = lane; idx < n; idx += 64) {
        float y[8];
        load8(idx, y);
        float lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            lo[e] = y[e] / s;
            hi[e] = y[4 + e] / s;
        }
        const int64_t place = a.slots[i0 + idx / ch] - row0;
        *reinterpret_cast<u32x2*>(cache + place * a.c_si[kv] + (idx % ch) * 8) = u32x2{codes4<CT>(lo), codes4<CT>(hi)};
    }
}

}  // namespace

hipError_t launch_quant_append(const QuantAppendArgs& a, int dtype, int ct, hipStream_t stream) {
    const dim3 grid((unsigned)a.total_new, (unsigned)a.Hk, 2);
    if (dtype == DT_BF16) {
        if (ct == CT_INT8) hipLaunchKernelGGL((fa_quant_append_kernel<DT_BF16, CT_INT8>), grid, dim3(64), 0, stream, a);
        else hipLaunchKernelGGL((fa_quant_append_kernel<DT_BF16, CT_E4M3>), grid, dim3(64), 0, stream, a);
    } else {
        if (ct == CT_INT8) hipLaunchKernelGGL((fa_quant_append_kernel<DT_FP16, CT_INT8>), grid, dim3(64), 0, stream, a);
        else hipLaunchKernelGGL((fa_quant_append_kernel<DT_FP16, CT_E4M3>), grid, dim3(64), 0, stream, a);
    }
    return hipGetLastError();
}

}  // namespace fa
