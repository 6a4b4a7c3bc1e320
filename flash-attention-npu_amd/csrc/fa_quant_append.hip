// fa_quant_append.hip -- new k / v rows into a cache of 8-bit codes with a
// scale for each block of tokens and kv head: fa_quant_append.
//
// The scale of a block is a power of two: x / s and c * s are then exact, a block
// that is filled one token at a time keeps its codes until a value outgrows its
// range, and where it does, its codes move by whole bits, so the roundings of
// repeated growth add up to less than one step (with max |x| / m, every token
// that is a new largest would round the whole block again). It costs at most one
// bit of the range.
//
// What bounds it: memory for prompts (41 000 rows of 8 heads, D128, bf16 to e4m3,
// 291 MB: 80-86 us, 3.4-3.6 TB/s; a row read twice, once for the maximum and once for
// its codes, took 485), the launch for decode steps (64 tokens: 7 us).
#include "fa_common.h"
#include "fa_quant_args.h"

#include <algorithm>
#include <type_traits>

namespace fa {

namespace {

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

// Four codes of y in one word, rounded to nearest even; |y| <= m by the choice of
// the scale. int8: the sum with 1.5 * 2^23 is rounded to whole numbers and ends in
// the code's byte.
template <int CT>
__device__ __forceinline__ uint32_t codes4(const float (&y)[4]) {
    if constexpr (CT == CT_INT8) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[i] = __builtin_bit_cast(uint32_t, y[i] + 0x1.8p23f);
        const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400u), b = __builtin_amdgcn_perm(u[3], u[2], 0x04000c0cu);
        return a | b;
    } else {
        int r = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
        r = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], r, true);
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

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

// x of lane l (uniform), as a uniform value
__device__ __forceinline__ int64_t lane_value(int64_t x, int l) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, l);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)x >> 32), l);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// A unit is a run (the rows of one block that stand together) and a head of k or v. WPU
// waves share one: 4 where a block's rows exceed what a wave holds in registers.
// A wave (or workgroup) looks for the runs that begin among rows_per_unit rows.
// hd / 8 lanes take a row, 16 bytes each, so a lane's columns stay the same.
// KEEP: passes of rows that stay in registers between the two readings.
template <int DT, int CT, int WPU, int KEEP>
__global__ void __launch_bounds__(256, KEEP > 4 ? 3 : 4) fa_quant_append_kernel(QuantAppendArgs a) {
    __shared__ uint32_t s_most[4];
    constexpr int UNITS = 4 / WPU, LANES = 64 * WPU;
    constexpr uint32_t kInf = DT == DT_FP16 ? 0x7c00u : 0x7f80u;
    const int lane = threadIdx.x & 63, ul = threadIdx.x % LANES;
    // launch_t: fewer than 2^26. What a wave has in common is told to be in scalar registers.
    const uint32_t unit = blockIdx.x * UNITS + __builtin_amdgcn_readfirstlane(threadIdx.x / LANES);
    const uint32_t chunk = unit / (uint32_t)(2 * a.Hk);
    const int64_t c0 = a.row0 + (int64_t)chunk * a.rows_per_unit;
    if (c0 >= a.total_new) return;  // WPU 4: the whole workgroup
    const int uh = (int)(unit - chunk * (uint32_t)(2 * a.Hk)), kv = uh >= a.Hk ? 1 : 0, h = uh - kv * a.Hk;
    const int ch = a.hd / 8, rp = LANES / ch;            // lanes of a row, rows of a pass
    const int lrow = (int)udiv(a.chunks, (uint32_t)ul), lcol = (ul - lrow * ch) * 8;
    const bool use = lrow < rp;

    const bool short_slots = a.num_slots <= 0xffffffffll;
    auto over = [&](const UDiv& d, int64_t s) -> int64_t {
        return short_slots ? (int64_t)udiv(d, (uint32_t)s) : (int64_t)((uint64_t)s / d.d);
    };
    auto slot_at = [&](int64_t i) -> int64_t {
        const int64_t s = i >= 0 && i < a.total_new ? a.slots[i] : -1;
        return s < a.num_slots ? s : -1;
    };
    auto block_of = [&](int64_t s) -> int64_t { return s >= 0 ? over(a.block, s) : -1; };
    // lane l: rows c0 - 1 + l and c0 + 63 + l; whether a run begins at the first
    const int64_t slot0 = slot_at(c0 - 1 + lane), slot1 = slot_at(c0 + 63 + lane);
    const int64_t blk0 = block_of(slot0), blk1 = block_of(slot1), blkp = (int64_t)__shfl_up((long long)blk0, 1);
    unsigned long long starts = __ballot(lane > 0 && lane <= a.rows_per_unit && blk0 >= 0 && blk0 != blkp);
    while (starts) {
        const int l0 = __builtin_ctzll(starts);
        starts &= starts - 1;
        const int64_t i0 = c0 - 1 + l0;
        const int64_t s0 = lane_value(slot0, l0), blk = lane_value(blk0, l0);
        const int64_t row0 = blk * a.scale_block;
        // the run ends at the first other block: in these rows, or further on
        const unsigned long long other0 = __ballot(blk0 != blk) >> l0 >> 1, other1 = __ballot(blk1 != blk);
        int64_t i1 = c0 + 127;
        if (other0) {
            i1 = i0 + 1 + __builtin_ctzll(other0);
        } else if (other1) {
            i1 = c0 + 63 + __builtin_ctzll(other1);
        } else {
            while (true) {
                const unsigned long long other = __ballot(block_of(slot_at(i1 + lane)) != blk);
                if (other) {
                    i1 += __builtin_ctzll(other);
                    break;
                }
                i1 += 64;
            }
        }
        const int n = (int)(i1 - i0), first = (int)(s0 - row0);
        const int64_t page = over(a.page, row0);
        const int inp = (int)(row0 - page * a.page_size);
        uint8_t* cache = a.c[kv] + page * a.c_sp[kv] + (int64_t)inp * a.c_si[kv] + (int64_t)h * a.c_sh[kv];
        float* sp = a.s[kv] + page * a.s_sp[kv] + (int64_t)(inp / a.scale_block) * a.s_sb[kv] + (int64_t)h * a.s_sh[kv];
        const uint16_t* x = static_cast<const uint16_t*>(a.x[kv]) + i0 * a.x_si[kv] + (int64_t)h * a.x_sh[kv];
        const float old = first > 0 ? *sp : 0.f;
        const uint32_t loff = (uint32_t)lrow * (uint32_t)a.x_si[kv] + lcol;  // 32 bits: the host checks the stride
        auto load = [&](int r) -> u32x4 {  // this lane's part of rows r .. r + rp - 1 of the run
            const bool ok = use && r + lrow < n;
            return ok ? *reinterpret_cast<const u32x4*>(x + (int64_t)r * a.x_si[kv] + loff) : u32x4{0u, 0u, 0u, 0u};
        };
        // the largest |x| by its bits: below the sign they are in the order of the
        // values, inf and NaN on top
        u32x4 keep[KEEP];
        u16x2 mb = {0, 0};
        auto larger = [&](u32x4 r) {
#pragma unroll
            for (int e = 0; e < 4; ++e) mb = __builtin_elementwise_max(mb, __builtin_bit_cast(u16x2, r[e] & 0x7fff7fffu));
        };
#pragma unroll
        for (int u = 0; u < KEEP; ++u) keep[u] = load(u * rp);
#pragma unroll
        for (int u = 0; u < KEEP; ++u) larger(keep[u]);
        for (int r = KEEP * rp; r < n; r += rp) larger(load(r));
        auto reduce = [&](uint32_t m) -> uint32_t {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o));
            if constexpr (WPU > 1) {
                __syncthreads();  // the run before is through with s_most
                if (lane == 0) s_most[threadIdx.x >> 6] = m;
                __syncthreads();
                m = max(max(s_most[0], s_most[1]), max(s_most[2], s_most[3]));
            }
            return m;
        };
        uint32_t most = reduce(max((uint32_t)mb[0], (uint32_t)mb[1]));
        const bool odd = most >= kInf;  // inf or NaN in the run
        if (odd) {
            // inf counts as the largest finite value, NaN not at all
            uint32_t m = 0;
            for (int r = 0; r < n; r += rp) {
                const u32x4 v = load(r);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint32_t b = v[e >> 1] >> (16 * (e & 1)) & 0x7fffu;
                    if (b <= kInf) m = max(m, b == kInf ? kInf - 1 : b);
                }
            }
            most = reduce(m);
        }
        float s = scale_for<CT>(f16_to_32<DT>((uint16_t)most));
        if (old >= s) {
            s = old;
        } else if (first > 0) {
            const int hc = a.hd / 4;
            const float f = old / s;
            for (int idx = ul; idx < first * hc; idx += LANES) {
                uint32_t* w = reinterpret_cast<uint32_t*>(cache + (int64_t)(idx / hc) * a.c_si[kv] + (idx % hc) * 4);
                float y[4];
                values4<CT>(*w, y);
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] *= f;
                *w = codes4<CT>(y);
            }
        }
        // a power of two is exact by its inverse; a scale of another value, kept, is divided by
        const bool exact = (__builtin_bit_cast(uint32_t, s) & 0x7fffffu) == 0;
        const float inv = 1.f / s;
        auto store = [&](int r, u32x4 v, auto plain_tag) {  // by all lanes: they exchange slots
            constexpr bool PLAIN = decltype(plain_tag)::value;
            float y[2][4];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                uint16_t b = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
                if constexpr (PLAIN) {
                    y[e >> 2][e & 3] = f16_to_32<DT>(b) * inv;
                } else {
                    const bool nan = (b & 0x7fffu) > kInf;
                    if ((b & 0x7fffu) == kInf) b = (uint16_t)(b - 1);
                    const float f = f16_to_32<DT>(b);
                    y[e >> 2][e & 3] = CT == CT_INT8 && nan ? 0.f : exact ? f * inv : f / s;
                }
            }
            const int l = l0 + r + lrow;  // where the row's slot is, above or in memory
            int at = __shfl((int)(slot0 - row0), l & 63);
            const int at1 = __shfl((int)(slot1 - row0), l & 63);
            if (l >= 64) at = at1;
            if (use && r + lrow < n) {
                if (l >= 128) at = (int)(a.slots[i0 + r + lrow] - row0);
                *reinterpret_cast<u32x2*>(cache + (int64_t)at * a.c_si[kv] + lcol) = u32x2{codes4<CT>(y[0]), codes4<CT>(y[1])};
            }
        };
        auto store_all = [&](auto plain_tag) {
#pragma unroll
            for (int u = 0; u < KEEP; ++u) {
                // one pass at a time, and nothing of it before the branch on the
                // kind: all of them widened at once would not fit in registers
                asm volatile("" : "+v"(keep[u]));
                if (u * rp < n) store(u * rp, keep[u], plain_tag);
            }
            for (int r = KEEP * rp; r < n; r += rp) store(r, load(r), plain_tag);
        };
        if (exact && !odd) store_all(std::integral_constant<bool, true>{});
        else store_all(std::integral_constant<bool, false>{});
        if constexpr (WPU > 1) __syncthreads();  // every wave has read the old scale
        if (ul == 0) *sp = s;
    }
}

template <int DT, int CT>
void launch_t(QuantAppendArgs& a, hipStream_t stream) {
    // Few tokens are single runs, each a unit's own, of which a wave keeps 4 passes.
    // Many come in whole blocks, one or two a unit: 16 passes, in 4 waves where one
    // would not hold a block.
    const bool few = a.total_new <= 1024, wide = (int64_t)a.scale_block * (a.hd / 8) > 16 * 64;
    a.rows_per_unit = few ? 1 : a.scale_block < 63 ? a.scale_block : 63;
    a.block = udiv_make((uint32_t)a.scale_block);
    a.page = udiv_make((uint32_t)a.page_size);
    a.chunks = udiv_make((uint32_t)a.hd / 8);
    const int64_t chunks = (a.total_new + a.rows_per_unit - 1) / a.rows_per_unit;
    // A launch has fewer than 2^32 threads; chunks past that many go into others, one after
    // another (an even number, so that they fill their workgroups of four units). A run belongs to
    // the chunk in which it begins.
    const int64_t most = ((1ll << 32) / 256 - 1) * (wide && !few ? 1 : 4) / (2 * a.Hk) & ~1ll;
    for (int64_t c = 0; c < chunks; c += most) {
        a.row0 = c * a.rows_per_unit;
        const int64_t units = std::min(chunks - c, most) * 2 * a.Hk;
        const dim3 one((unsigned)units), four((unsigned)((units + 3) / 4)), nt(256);
        if (few) hipLaunchKernelGGL((fa_quant_append_kernel<DT, CT, 1, 4>), four, nt, 0, stream, a);
        else if (wide) hipLaunchKernelGGL((fa_quant_append_kernel<DT, CT, 4, 16>), one, nt, 0, stream, a);
        else hipLaunchKernelGGL((fa_quant_append_kernel<DT, CT, 1, 16>), four, nt, 0, stream, a);
    }
}

}  // namespace

hipError_t launch_quant_append(QuantAppendArgs a, int dtype, int ct, hipStream_t stream) {
    if (dtype == DT_BF16) {
        if (ct == CT_INT8) launch_t<DT_BF16, CT_INT8>(a, stream);
        else launch_t<DT_BF16, CT_E4M3>(a, stream);
    } else {
        if (ct == CT_INT8) launch_t<DT_FP16, CT_INT8>(a, stream);
        else launch_t<DT_FP16, CT_E4M3>(a, stream);
    }
    return hipGetLastError();
}

}  // namespace fa
