// fa_quant.h -- device code that the attention kernels over 8-bit codes share:
// codes to fp16 operands, and the sequences of a call.
//
// Every code is an fp16 value (int8: |c| <= 128; e4m3: steps of 2^-9 up to 448), so
// both products run as fp16 MFMAs on the codes themselves and the scales meet the
// results: K's on the scores, V's on the weights.
#pragma once
#include "fa_common.h"
#include "fa_quant_args.h"

namespace fa {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t byte_perm(uint32_t hi, uint32_t lo, uint32_t sel) {
    return __builtin_amdgcn_perm(hi, lo, sel);  // sel bytes 0..3: of lo, 4..7: of hi
}

// Four codes (the bytes of w, lowest first) as four fp16 values, exactly.
// int8: the byte plus 128 under the exponent of 1024 is 1152 + c.
template <int CT>
__device__ __forceinline__ u32x2 widen4(uint32_t w) {
    if constexpr (CT == CT_INT8) {
        const uint32_t u = w ^ 0x80808080u;
        const f16x2 off = {(_Float16)1152.f, (_Float16)1152.f};
        const f16x2 a = __builtin_bit_cast(f16x2, byte_perm(0x64646464u, u, 0x04010400u)) - off;
        const f16x2 b = __builtin_bit_cast(f16x2, byte_perm(0x64646464u, u, 0x04030402u)) - off;
        return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
    } else {
        return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, false)),
                     __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.0f, true))};
    }
}

__device__ __forceinline__ f32x4 mfma_f16(u32x4 a, u32x4 b, f32x4 c) { return mfma16x16x32<DT_FP16>(a, b, c); }

// 2^k for k in [-126, 127]
__device__ __forceinline__ float exp2i(int k) { return __builtin_bit_cast(float, (uint32_t)(k + 127) << 23); }

// A query row enters its products as fp16, times the power of two that puts its
// largest value in [2^14, 2^15): a bf16 value keeps its 8 bits down to 2^-28 of
// the largest and what is lost below is less than 2^-38 of it, under the rounding of the
// fp32 sums. The exponent for a row whose largest |q| is `most`:
__device__ __forceinline__ int q_shift(float most) {
    const int e = (int)(__builtin_bit_cast(uint32_t, most) >> 23) - 127;
    return most > 0.f ? min(14 - e, 126) : 0;
}

// Keys and query rows of a sequence; [lo, hi) holds the keys that some row sees.
struct QuantSeq {
    int lo, hi, sk, sq, crow;
};

__device__ __forceinline__ QuantSeq quant_seq(const QuantFwdArgs& a, int b) {
    QuantSeq s;
    s.sk = min(max(a.seqlens[b], 0), a.capacity);
    s.crow = a.row0 + b;
    if (a.batch_idx) {  // a row that is not there has no keys
        s.crow = a.batch_idx[b];
        if ((unsigned)s.crow >= (unsigned)a.rows) s.crow = s.sk = 0;
    }
    s.sq = a.Sq;
    if (a.cu_q) {
        // rows past total_q are not there, nor are their keys, the sequence's last
        const int first = a.cu_q[b], end = max(a.cu_q[b + 1], first), upto = min(end, a.total_q);
        s.sk = max(s.sk - (end - max(upto, first)), 0);
        s.sq = first < 0 ? 0 : min(max(upto - first, 0), a.Sq);
    }
    s.lo = max(0, key_lo(s.sk - s.sq, a.wl, 0));
    s.hi = min(s.sk, key_hi(s.sk - 1, a.wr, 0) + 1);
    if (s.sq == 0) s.hi = s.lo;
    return s;
}

// Rows of q and out, and the lse, of query position i of sequence b
__device__ __forceinline__ int64_t q_row(const QuantFwdArgs& a, int b, int i, int64_t sb, int64_t si) {
    return a.cu_q ? ((int64_t)a.cu_q[b] + i) * si : (int64_t)b * sb + (int64_t)i * si;
}
__device__ __forceinline__ int64_t lse_at(const QuantFwdArgs& a, int b, int h, int i) {
    return a.cu_q ? (int64_t)h * a.lse_sh + a.cu_q[b] + i : (int64_t)b * a.lse_sb + (int64_t)h * a.lse_sh + i;
}

// Inclusive prefix sums in place over s[1 .. n], by one wave; s[0] = 0
template <typename T>
__device__ __forceinline__ void prefix_sums(T* s, int n) {
    const int lane = threadIdx.x & 63, seg = (n + 63) / 64, b0 = lane * seg;
    T local = 0;
    for (int k = 0; k < seg; ++k)
        if (b0 + k < n) local += s[b0 + k + 1];
    T incl = local;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T v = __shfl_up(incl, o);
        if (lane >= o) incl += v;
    }
    T run = incl - local;
    for (int k = 0; k < seg; ++k)
        if (b0 + k < n) {
            run += s[b0 + k + 1];
            s[b0 + k + 1] = run;
        }
    if (lane == 0) s[0] = 0;
}

// x y, and 0 where x is 0, whatever y: a hidden key's weight
__device__ __forceinline__ float mul_or_0(float x, float y) {
    float r;
    asm("v_mul_legacy_f32 %0, %1, %2" : "=v"(r) : "v"(x), "v"(y));
    return r;
}

// Weights. A code c of V with scale t enters its row's sum as p t c, x the score in log2
// units. A row keeps a running maximum u of x + log2 t, and with w = 2^(x + log2 t - u)
//   O = sum of w c,   l = sum of w / t,   out = O / l,   log2 of the sum of 2^x = u + log2 l,
// so that a weight is as precise as it is large in its row's sum, and keys that the row
// does not see have no part in that. w / t keeps its bits while a row's scales are
// within 2^100 of each other, so this is for plain ones. For others l has a running maximum
// of its own, m of x: l = sum of 2^(x - m), out = O / l 2^(u - m).
__device__ __forceinline__ bool plain_scale(float t) { return t > 0x1p-40f && t < 0x1p40f; }

// log2 |t|; -inf for 0 and for what is no number, whose weights are formed apart
__device__ __forceinline__ float scale_log2(float t) {
    const float a = fabsf(t);
    const bool small = a < 0x1p-100f;  // the logarithm takes no subnormal
    const float y = fast_log2(small ? a * 0x1p64f : a) - (small ? 64.f : 0.f);
    return a < INFINITY ? y : -INFINITY;
}

// u + log2 l, the exponent of l added first: l is far from 1 where t is
__device__ __forceinline__ float add_log2(float u, float l) {
    return u + (float)__builtin_amdgcn_frexp_expf(l) + fast_log2(__builtin_amdgcn_frexp_mantf(l));
}

// eight 16-bit values as fp32
template <int DT>
__device__ __forceinline__ f32x8 widen8(u32x4 r) {
    f32x8 y;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = f16_to_32<DT>((uint16_t)(r[e >> 1] >> (16 * (e & 1))));
    return y;
}
template <int DT>
__device__ __forceinline__ f32x8 load8(const void* base, int64_t off) {
    return widen8<DT>(*reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + off));
}

}  // namespace fa
