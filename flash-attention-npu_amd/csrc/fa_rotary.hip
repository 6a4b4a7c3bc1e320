// fa_rotary.hip -- tables of cosines and sines (fa_rotary_table), and the rotation of
// rows of q and k by them (fa_rotary).
//
// Tables: the angle of position p and pair i is p f_i. In 32 bits an angle of 10^5
// keeps no more than 7 bits behind the point, so the product is taken in 64, in quarter
// turns, and only what is left of one (|r| <= 1/2) goes through a sine and cosine in 32
// bits. Whole quarters change places and signs, so that a value near 0 is the sine of a
// small rest, whose bits are all there (of whole turns, the cosine of 52174 would have 6).
// The f_i, whatever their scaling, are the host's and come as arguments.
// 131072 positions of 64 pairs in fp32, 67 MB, take 13.8 us (4.9 TB/s of writes), 64 positions
// 2.8. Four angles a thread make whole 16-byte stores.
//
// Rotation: (x1, x2) -> (x1 c - x2 s, x2 c + x1 s), products rounded to fp32 before the sum
// as in fa_rope.h, so that the rows equal bit for bit what flash_attn_with_kvcache makes of
// them with the same tables. The way back, which is also the gradient, has -s for s.
// Memory bounds it: q and k in and out once, a table's row read again by each head out of the caches.
// B4 S4096 H32/8 D128 bf16, 336 MB, takes 62 us (5.4 TB/s); q and k of 64 tokens 3.6. One launch for
// both, a thread for two pieces of eight values, whose loads do not wait for each other.
#include "fa_common.h"
#include "fa_rotary_args.h"

#include <algorithm>
#include <climits>

namespace fa {

namespace {

enum : int { DT_F32 = 2 };

template <int T>
__device__ __forceinline__ void store4(void* base, int64_t at, const float (&y)[4]) {
    if constexpr (T == DT_F32) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(base) + at) = f32x4{y[0], y[1], y[2], y[3]};
    } else {
        const uint32_t lo = f32_to_16<T>(y[0]) | (uint32_t)f32_to_16<T>(y[1]) << 16;
        const uint32_t hi = f32_to_16<T>(y[2]) | (uint32_t)f32_to_16<T>(y[3]) << 16;
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(base) + at) = u32x2{lo, hi};
    }
}

__device__ __forceinline__ int64_t position_at(const void* p, int wide, int64_t i) {
    return wide ? static_cast<const int64_t*>(p)[i] : (int64_t)static_cast<const int*>(p)[i];
}

// Sine and cosine of x quarter turns, |x| <= 1/2 (an eighth of a turn): their Taylor series, of which what is left out is less
// than 2^-28 of the value. Of pi / 2, which the sine of a small x is a multiple by, the rounding to fp32 is added back.
__device__ __forceinline__ void sincos_rest(float x, float& s, float& c) {
    constexpr double h = 1.57079632679489661923, h2 = h * h, h3 = h * h2, h4 = h2 * h2, h8 = h4 * h4;
    constexpr float kHigh = (float)h, kLow = (float)(h - (double)kHigh);
    const float z = x * x;
    float u = __builtin_fmaf(z, (float)(h * h8 / 362880), (float)(-h3 * h4 / 5040));
    u = __builtin_fmaf(z, u, (float)(h * h4 / 120));
    u = __builtin_fmaf(z, u, (float)(-h3 / 6));
    s = __builtin_fmaf(x, kHigh, x * __builtin_fmaf(z, u, kLow));
    float v = __builtin_fmaf(z, (float)(-h2 * h8 / 3628800), (float)(h8 / 40320));
    v = __builtin_fmaf(z, v, (float)(-h2 * h4 / 720));
    v = __builtin_fmaf(z, v, (float)(h4 / 24));
    v = __builtin_fmaf(z, v, (float)(-h2 / 2));
    c = __builtin_fmaf(z, v, 1.f);
}

// A thread makes 4 angles of a position.
template <int T>
__global__ void __launch_bounds__(256) fa_rotary_table_kernel(RotaryTableArgs a, UDiv quads, int64_t row0, uint32_t items) {
    const uint32_t id = blockIdx.x * 256 + threadIdx.x;
    if (id >= items) return;
    const uint32_t r = udiv(quads, id);
    const int i0 = (int)(id - r * quads.d) * 4;
    const int64_t row = row0 + r;
    const double p = (double)position_at(a.positions, a.wide, row);
    float c[4], s[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        // the nearest whole number of quarter turns: past 2^52 a number has no bits below 1
        const double w = __builtin_fma(p, a.turns[i0 + e], 0x1.8p52), q = w - 0x1.8p52;
        const int k = (int)__builtin_bit_cast(uint64_t, w) & 3;
        float sr, cr;
        const float rest = (float)__builtin_fma(p, a.turns[i0 + e], -q);
        sincos_rest(fminf(fmaxf(rest, -0.5f), 0.5f), sr, cr);  // (past 2^51 quarter turns nothing is left of an angle)
        const float x = k & 1 ? sr : cr, y = k & 1 ? cr : sr;  // a quarter turn takes (cos, sin) to (-sin, cos)
        c[e] = (k == 1 || k == 2 ? -x : x) * a.factor;
        s[e] = (k & 2 ? -y : y) * a.factor;
    }
    store4<T>(a.cos, row * a.half + i0, c);
    store4<T>(a.sin, row * a.half + i0, s);
}

// eight values of a table's row, in fp32
template <int T>
__device__ __forceinline__ f32x8 table8(const void* base, int64_t at) {
    f32x8 y;
    if constexpr (T == DT_F32) {
        const f32x4 lo = *reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + at);
        const f32x4 hi = *reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + at + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = lo[e], y[e + 4] = hi[e];
    } else {
        const u32x4 r = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + at);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = f16_to_32<T>((uint16_t)(r[e >> 1] >> (16 * (e & 1))));
    }
    return y;
}
template <int DT>
__device__ __forceinline__ f32x8 wide8(u32x4 r) {
    f32x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = f16_to_32<DT>((uint16_t)(r[e >> 1] >> (16 * (e & 1))));
    return y;
}

// A unit of a head row is 16 values that turn together: 8 pairs, chunks u and u + rd/16
// of 8 (halves) or chunks 2u and 2u + 1 (neighbours); past rd it is a chunk that is copied.
template <int DT, int T, bool INTER>
__global__ void __launch_bounds__(256) fa_rotary_kernel(RotaryArgs a) {
    const uint32_t id = blockIdx.x * 256 + threadIdx.x;
    if (id >= a.items) return;
    const uint32_t r = udiv(a.per_row, id), in = id - r * a.per_row.d;
    const uint32_t hh = udiv(a.units, in);
    const int u = (int)(in - hh * a.units.d);
    const int64_t row = a.row0 + r;
    const int which = (int)hh >= a.heads0, h = (int)hh - (which ? a.heads0 : 0);
    // the row's sequence and place in it
    int64_t b = 0, i = row;
    bool turned = true;  // rows of no sequence are not
    if (a.cu) {
        b = seq_of(a.cu, a.B, (int)row);
        i = row - a.cu[b];
        turned = row >= a.cu[0] && row < a.cu[a.B];
    } else {
        b = udiv(a.seqlen, (uint32_t)row);
        i = row - b * a.seqlen.d;
    }
    const int64_t xb = a.cu ? 0 : b, xi = a.cu ? row : i;
    const uint16_t* x = static_cast<const uint16_t*>(a.x[which]) + xb * a.x_sb[which] + xi * a.x_si[which] + (int64_t)h * a.x_sh[which];
    uint16_t* o = static_cast<uint16_t*>(a.o[which]) + xb * a.o_sb[which] + xi * a.o_si[which] + (int64_t)h * a.o_sh[which];
    const int nrot = a.rd / 16;
    if (u >= nrot) {
        const int d = a.rd + (u - nrot) * 8;
        *reinterpret_cast<u32x4*>(o + d) = *reinterpret_cast<const u32x4*>(x + d);
        return;
    }
    const int d0 = INTER ? u * 16 : u * 8, d1 = INTER ? d0 + 8 : d0 + a.rd / 2;
    const u32x4 x0 = *reinterpret_cast<const u32x4*>(x + d0), x1 = *reinterpret_cast<const u32x4*>(x + d1);
    if (!turned) {
        if (!a.in_place) {
            *reinterpret_cast<u32x4*>(o + d0) = x0;
            *reinterpret_cast<u32x4*>(o + d1) = x1;
        }
        return;
    }
    int64_t p;
    if (a.positions) p = position_at(a.positions, a.wide, xb * a.p_sb + xi * a.p_si);
    else p = (a.offsets ? (int64_t)a.offsets[b] : a.offset) + i;
    p = min(max(p, (int64_t)0), (int64_t)a.seqlen_ro - 1);
    const f32x8 c = table8<T>(a.cos, p * a.c_stride + u * 8), s = table8<T>(a.sin, p * a.s_stride + u * 8) * a.sign;
    const f32x8 y0 = wide8<DT>(x0), y1 = wide8<DT>(x1);
    f32x8 z0, z1;
    {
#pragma clang fp contract(off)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v0 = INTER ? (e < 4 ? y0[2 * e & 7] : y1[2 * e & 7]) : y0[e];
            const float v1 = INTER ? (e < 4 ? y0[(2 * e & 7) + 1] : y1[(2 * e & 7) + 1]) : y1[e];
            const float g = v0 * c[e] - v1 * s[e], k = v1 * c[e] + v0 * s[e];
            if (!INTER) {
                z0[e] = g;
                z1[e] = k;
            } else if (e < 4) {
                z0[2 * e & 7] = g;
                z0[(2 * e & 7) + 1] = k;
            } else {
                z1[2 * e & 7] = g;
                z1[(2 * e & 7) + 1] = k;
            }
        }
    }
    *reinterpret_cast<u32x4*>(o + d0) = pack8<DT>(z0);
    *reinterpret_cast<u32x4*>(o + d1) = pack8<DT>(z1);
}

template <int DT>
void launch_rotary_t(const RotaryArgs& a, bool inter, bool wide_table, hipStream_t stream) {
    const dim3 grid((a.items + 255) / 256), nt(256);
    if (inter && wide_table) hipLaunchKernelGGL((fa_rotary_kernel<DT, DT_F32, true>), grid, nt, 0, stream, a);
    else if (inter) hipLaunchKernelGGL((fa_rotary_kernel<DT, DT, true>), grid, nt, 0, stream, a);
    else if (wide_table) hipLaunchKernelGGL((fa_rotary_kernel<DT, DT_F32, false>), grid, nt, 0, stream, a);
    else hipLaunchKernelGGL((fa_rotary_kernel<DT, DT, false>), grid, nt, 0, stream, a);
}

constexpr int64_t kMostItems = 1ll << 30;  // of a launch

}  // namespace

hipError_t launch_rotary_table(const RotaryTableArgs& a, int dtype, hipStream_t stream) {
    const UDiv quads = udiv_make((uint32_t)a.half / 4);
    const int64_t most = kMostItems / quads.d;
    for (int64_t r = 0; r < a.n; r += most) {
        const uint32_t items = (uint32_t)(std::min(most, a.n - r) * quads.d);
        const dim3 grid((items + 255) / 256), nt(256);
        if (dtype == DT_F32) hipLaunchKernelGGL(fa_rotary_table_kernel<DT_F32>, grid, nt, 0, stream, a, quads, r, items);
        else if (dtype == DT_BF16) hipLaunchKernelGGL(fa_rotary_table_kernel<DT_BF16>, grid, nt, 0, stream, a, quads, r, items);
        else hipLaunchKernelGGL(fa_rotary_table_kernel<DT_FP16>, grid, nt, 0, stream, a, quads, r, items);
    }
    return hipGetLastError();
}

hipError_t launch_rotary(RotaryArgs a, int dtype, bool inter, bool wide_table, hipStream_t stream) {
    const uint32_t units = (uint32_t)(a.rd / 16 + (a.in_place ? 0 : (a.hd - a.rd) / 8));
    a.units = udiv_make(units);
    a.per_row = udiv_make(units * (uint32_t)a.heads);
    const int64_t most = std::max<int64_t>(kMostItems / a.per_row.d, 1);
    for (a.row0 = 0; a.row0 < a.rows; a.row0 += most) {
        a.items = (uint32_t)(std::min(most, a.rows - a.row0) * a.per_row.d);
        if (dtype == DT_BF16) launch_rotary_t<DT_BF16>(a, inter, wide_table, stream);
        else launch_rotary_t<DT_FP16>(a, inter, wide_table, stream);
    }
    return hipGetLastError();
}

}  // namespace fa
