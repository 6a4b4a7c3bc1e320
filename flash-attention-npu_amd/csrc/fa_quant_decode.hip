// fa_quant_decode.hip -- attention over 8-bit codes for few query rows (a kv
// head's g query heads x positions, at most 64 packed rows): the cache is
// streamed once, at the rate that HBM gives.
//
// Split: the 64-key tiles (32 at head dim 256) of all sequences and kv heads form
// one list, built in LDS by each workgroup from cache_seqlens and cut into equal
// contiguous ranges, one per wave (fa_decode_split.h); waves of a CU take
// adjacent kv heads of one range, so that a key row is requested by a CU at once. A
// range that ends inside a sequence leaves a partial, merged by the second launch.
//
// A tile: lane (li, G) of a wave loads a quarter of key row li, which is its operand
// of S^T = K.Q^T as it stands once widened, and columns li * D/16 .. of value rows
// 4G .. 4G + 3, which two byte permutations turn into its operand of O^T = V^T.P^T:
// no shared memory and no barrier on the way, and each wave keeps the next tiles
// (32 KB) in flight in registers. Page ids and scales come through a small table in
// LDS, filled 32 tiles at a time.
//
// Scales: the K scale of 16 keys multiplies their scores. The V scale t multiplies
// the weights p, which are then rounded to fp16, so they are kept relative to a
// running power of two R >= t that moves up like a maximum, w = p * t / R * 2^14: a
// weight keeps its 11 bits as long as p * t / R > 2^-28.
#include "fa_quant.h"
#include "fa_decode_split.h"

namespace fa {

namespace {

constexpr int NWAVE = 4;
constexpr int MAXB = 2048;
constexpr int TAB = 32;  // tiles of one half of a wave's table

template <int HD>
struct Cfg {
    static constexpr int KT = HD == 256 ? 32 : 64;     // keys of a tile
    static constexpr int NH = KT / 16;
    static constexpr int KL = HD / 64;                 // 16-byte loads of a lane for its quarter key row
    static constexpr int KSTEPS = HD / 32;
    static constexpr int VW = HD / 64;                 // words of a lane for its columns of a value row
    static constexpr int VB = HD / 16;                 // columns of a lane, PV products of a 16-row tile
    static constexpr int STAGES = HD == 64 ? 5 : 3;
};

__device__ __forceinline__ int heads_per_group(const QuantFwdArgs& a) { return a.Hk % 4 == 0 ? 4 : a.Hk % 2 == 0 ? 2 : 1; }

struct Seg {
    int S, n;      // first tile of the list, tiles
    int b, hk;
    int lo_tile;
    QuantSeq q;
};

__device__ __forceinline__ Seg seg_of(const QuantFwdArgs& a, const int* s_pref, const QuantSeq* s_seq, int t, int hs, int h,
                                      int KT) {
    int bl = 0, bh = a.B;
    while (bh - bl > 1) {
        const int mid = (bl + bh) >> 1;
        if (s_pref[mid] <= t) bl = mid;
        else bh = mid;
    }
    Seg s;
    s.b = bl;
    s.n = (s_pref[bl + 1] - s_pref[bl]) / (a.Hk / hs);
    const int hg = s.n > 0 ? (t - s_pref[bl]) / s.n : 0;
    s.hk = hg * hs + h;
    s.S = s_pref[bl] + hg * s.n;
    s.q = s_seq[bl];
    s.lo_tile = s.q.lo / KT;
    return s;
}

// CT: cache type; HD: kernel head dim (HDM: the cache's is smaller, columns past it
// are zero); NR: 16-row tiles of packed rows.
template <int CT, int HD, int NR, bool HDM>
__global__ void __launch_bounds__(256, 1) fa_quant_decode_kernel(QuantFwdArgs a) {
    using C = Cfg<HD>;
    constexpr int KT = C::KT, NH = C::NH, KL = C::KL, KSTEPS = C::KSTEPS, VW = C::VW, VB = C::VB, STAGES = C::STAGES;
    __shared__ int s_pref[MAXB + 1];
    __shared__ QuantSeq s_seq[MAXB];
    __shared__ int64_t s_koff[NWAVE][2 * TAB * NH], s_voff[NWAVE][2 * TAB * NH];
    __shared__ __attribute__((aligned(16))) float s_ks[NWAVE][2 * TAB * NH], s_vs[NWAVE][2 * TAB * NH];
    __shared__ int s_ok[NWAVE][2 * TAB];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int li = lane & 15, G = lane >> 4;
    const int hs = heads_per_group(a), hgs = a.Hk / hs;

    // ---- the list of tiles ----------------------------------------------------------
    for (int b = tid; b < a.B; b += 256) {
        const QuantSeq s = quant_seq(a, b);
        s_seq[b] = s;
        s_pref[b + 1] = s.hi > s.lo && s.sq * a.g <= a.dec_rows ? hgs * ((s.hi + KT - 1) / KT - s.lo / KT) : 0;
    }
    __syncthreads();
    if (wave == 0) {
        const int seg = (a.B + 63) / 64, b0 = lane * seg;
        int local = 0;
        for (int k = 0; k < seg; ++k)
            if (b0 + k < a.B) local += s_pref[b0 + k + 1];
        int incl = local;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o);
            if (lane >= o) incl += v;
        }
        int run = incl - local;
        for (int k = 0; k < seg; ++k)
            if (b0 + k < a.B) {
                run += s_pref[b0 + k + 1];
                s_pref[b0 + k + 1] = run;
            }
        if (lane == 0) s_pref[0] = 0;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int b = tid; b <= a.B; b += 256) a.sched[b] = s_pref[b];

    const long long T = s_pref[a.B];
    const int hsel = wave % hs;
    const long long W = (long long)gridDim.x * (NWAVE / hs);
    const long long gw = (long long)(wave / hs) * gridDim.x + blockIdx.x;  // wave-major, as in fa_decode.hip
    const long long wid = gw * hs + hsel;
    const long long ovh = dec::seg_ovh(T, W, (long long)a.B * hgs);
    const long long CT_ = dec::split_total(T, ovh, a.B, hgs);
    const int t0 = dec::split_tfirst(gw * CT_ / W, s_pref, a.B, hgs, ovh, T, CT_);
    const int t1 = dec::split_tfirst((gw + 1) * CT_ / W, s_pref, a.B, hgs, ovh, T, CT_);
    if (t0 >= t1) return;  // no barrier follows: the waves go on alone

    int64_t* koff = s_koff[wave];
    int64_t* voff = s_voff[wave];
    float* tks = s_ks[wave];
    float* tvs = s_vs[wave];
    int* tok = s_ok[wave];

    // Offsets, scales and visibility of the 16-key blocks of tiles base .. base + TAB
    // - 1, into their half of the table. A block without a visible key has offset 0
    // and scales 0.
    auto fill = [&](int base) {
        constexpr int PER = TAB * NH / 64;
        const int at0 = (((base - t0) / TAB) & 1) * TAB * NH;
        int id[PER], inp[PER], kvh[PER];
        bool ok[PER];
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int t = base + (u * 64 + lane) / NH;
            id[u] = -1;
            inp[u] = 0;
            kvh[u] = 0;
            if (t < t1) {
                const Seg s = seg_of(a, s_pref, s_seq, t, hs, hsel, KT);
                const int key = (s.lo_tile + (t - s.S)) * KT + (lane % NH) * 16;
                kvh[u] = s.hk;
                if (key < s.q.hi && key + 16 > s.q.lo) {
                    const int pi = a.table ? (int)udiv(a.page, (uint32_t)key) : 0;
                    inp[u] = key - pi * a.page_size;
                    id[u] = a.table ? a.table[(int64_t)s.q.crow * a.t_stride + pi] : s.q.crow;
                }
            }
        }
        float ks[PER], vs[PER];
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            ok[u] = id[u] >= 0 && id[u] < a.num_pages;
            const int64_t p = ok[u] ? id[u] : 0, r = ok[u] ? inp[u] : 0, h = kvh[u];
            const int64_t sb = udiv(a.sblk, (uint32_t)r);
            ks[u] = a.ks[p * a.ks_sp + sb * a.ks_sb + h * a.ks_sh];
            vs[u] = a.vs[p * a.vs_sp + sb * a.vs_sb + h * a.vs_sh];
            const int at = at0 + u * 64 + lane;
            koff[at] = p * a.k_sp + r * a.k_si + h * a.k_sh;
            voff[at] = p * a.v_sp + r * a.v_si + h * a.v_sh;
            const unsigned long long m = __ballot(ok[u]);
            if (lane % NH == 0) tok[at / NH] = (int)(m >> lane) & ((1 << NH) - 1);
        }
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int at = at0 + u * 64 + lane;
            tks[at] = ok[u] ? ks[u] : 0.f;
            tvs[at] = ok[u] ? vs[u] : 0.f;
        }
    };
    fill(t0);

    // ---- loads ------------------------------------------------------------------------
    u32x4 kr[STAGES][NH][KL];
    uint32_t vr[STAGES][NH][4][VW];
    const uint32_t kin = (uint32_t)li * (uint32_t)a.k_si + G * (HD / 4);
    uint32_t vin[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) vin[i] = (uint32_t)(4 * G + i) * (uint32_t)a.v_si + li * VB;
    auto uniform64 = [](int64_t x) -> int64_t {
        const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)x);
        const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)x >> 32));
        return (int64_t)((uint64_t)hi << 32 | lo);
    };
    auto issue = [&](int t, u32x4 (&kk)[NH][KL], uint32_t (&vv)[NH][4][VW]) {
        if (t >= t1) return;
        const int at = ((t - t0) % (2 * TAB)) * NH;
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            const uint8_t* kb = a.k + uniform64(koff[at + h]);
            const uint8_t* vb = a.v + uniform64(voff[at + h]);
#pragma unroll
            for (int s = 0; s < KL; ++s)
                kk[h][s] = !HDM || G * (HD / 4) + 16 * s < a.hd ? *reinterpret_cast<const u32x4*>(kb + kin + 16 * s)
                                                                : u32x4{0u, 0u, 0u, 0u};
            const bool in = !HDM || li * VB < a.hd;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (VW == 1) {
                    vv[h][i][0] = in ? *reinterpret_cast<const uint32_t*>(vb + vin[i]) : 0u;
                } else if constexpr (VW == 2) {
                    const u32x2 x = in ? *reinterpret_cast<const u32x2*>(vb + vin[i]) : u32x2{0u, 0u};
                    vv[h][i][0] = x[0];
                    vv[h][i][1] = x[1];
                } else {
                    const u32x4 x = in ? *reinterpret_cast<const u32x4*>(vb + vin[i]) : u32x4{0u, 0u, 0u, 0u};
#pragma unroll
                    for (int w = 0; w < 4; ++w) vv[h][i][w] = x[w];
                }
            }
        }
    };

    // ---- a segment: q, sums ----------------------------------------------------------------
    Seg cs = seg_of(a, s_pref, s_seq, t0, hs, hsel, KT);
    u32x4 qreg[NR][KSTEPS];
    float qs[NR];              // what the scores of a row are to be multiplied by for its q_shift
    int qi[NR];
    f32x4 oacc[NR][VB];
    float m_run[NR], l_run[NR];
    int rows = 0, eR = 30;     // R = 2^(eR - 127)
    int flo = 0, fhi = 0;      // keys that every row sees
    auto begin_seg = [&]() {
        rows = cs.q.sq * a.g;
        flo = key_lo(cs.q.sk - 1, a.wl, 0);
        fhi = key_hi(cs.q.sk - cs.q.sq, a.wr, 0);
        eR = 30;
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            const int r = rt * 16 + li;
            const bool ok = r < rows;
            qi[rt] = ok ? r / a.g : 0;
            const int h = cs.hk * a.g + (ok ? r % a.g : 0);
            const int64_t base = q_row(a, cs.b, qi[rt], a.q_sb, a.q_si) + (int64_t)h * a.q_sh;
            f32x8 x[KSTEPS];
            float most = 0.f;
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s) {
                const int d = G * (HD / 4) + 8 * s;
                x[s] = ok && (!HDM || d < a.hd) ? load8(a.q, base + d, a.bf16) : f32x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[s][e]));
            }
            const int sh = q_shift(wave_max16x4(most));
            const float up = exp2i(sh);
            qs[rt] = exp2i(-sh);
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s) qreg[rt][s] = pack8<DT_FP16>(x[s] * up);
            m_run[rt] = -INFINITY;
            l_run[rt] = 0.f;
#pragma unroll
            for (int j = 0; j < VB; ++j) oacc[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    auto end_seg = [&]() {
        const bool whole = cs.S >= t0 && cs.S + cs.n <= t1;
        const float back = exp2i(eR - 127 - 14);
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            const int r = rt * 16 + li;
            const float l = wave_sum16x4(l_run[rt]);
            const bool some = l != 0.f;  // NaN: some
            const float inv = some ? back / l : 0.f;
            const float lse = some ? (m_run[rt] + fast_log2(l)) * kLn2 : INFINITY;
            if (r >= rows) continue;
            if (whole) {
                const int h = cs.hk * a.g + r % a.g;
                uint16_t* o = static_cast<uint16_t*>(a.out) + q_row(a, cs.b, qi[rt], a.o_sb, a.o_si) + (int64_t)h * a.o_sh;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int d = (4 * G + i) * VB;
                    if (HDM && d >= a.hd) continue;
#pragma unroll
                    for (int j = 0; j < VB; j += 4)
                        *reinterpret_cast<u32x2*>(o + d + j) =
                            u32x2{pack2(oacc[rt][j][i] * inv, oacc[rt][j + 1][i] * inv, a.bf16),
                                  pack2(oacc[rt][j + 2][i] * inv, oacc[rt][j + 3][i] * inv, a.bf16)};
                }
                if (G == 0) a.lse[lse_at(a, cs.b, h, qi[rt])] = lse;
            } else {
                const int slot = cs.S <= t0 ? 0 : 1;  // this worker's first segment, else its last
                const int64_t row = (wid * 2 + slot) * (16 * NR) + r;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < VB; j += 4)
                        *reinterpret_cast<f32x4*>(a.part_o + row * HD + (4 * G + i) * VB + j) =
                            f32x4{oacc[rt][j][i], oacc[rt][j + 1][i], oacc[rt][j + 2][i], oacc[rt][j + 3][i]} * inv;
                if (G == 0) a.part_lse[row] = some ? lse : -INFINITY;
            }
        }
    };

    // ---- a tile ----------------------------------------------------------------------------
    const float scale2 = a.scale * kLog2e;
    auto compute = [&](int t, const u32x4 (&kk)[NH][KL], uint32_t (&vv)[NH][4][VW]) {
        const int key0 = (cs.lo_tile + (t - cs.S)) * KT;
        const int at = (t - t0) % (2 * TAB);
        float ks[NH], vs[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            ks[h] = tks[at * NH + h];
            vs[h] = tvs[at * NH + h];
        }
        const int ok = __builtin_amdgcn_readfirstlane(tok[at]);
        const bool full = ok == (1 << NH) - 1 && key0 + KT <= cs.q.sk && key0 >= flo && key0 + KT - 1 <= fhi;
        // S^T = K . Q^T on the codes
        f32x4 x[NR][NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) x[rt][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KL; ++s)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const u32x2 lo = widen4<CT>(kk[h][s][2 * u]), hi = widen4<CT>(kk[h][s][2 * u + 1]);
                    const u32x4 op = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                    for (int rt = 0; rt < NR; ++rt) x[rt][h] = mfma_f16(op, qreg[rt][2 * s + u], x[rt][h]);
                }
        }
        // scores in log2 units
#pragma unroll
        for (int rt = 0; rt < NR; ++rt)
#pragma unroll
            for (int h = 0; h < NH; ++h) {
                if (a.softcap > 0.f) {
                    const float c = qs[rt] * a.scale * ks[h];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[rt][h][e] = a.softcap * kLog2e * fast_tanh(x[rt][h][e] * c * (1.f / a.softcap));
                } else {
                    x[rt][h] *= qs[rt] * scale2 * ks[h];
                }
            }
        if (!full) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) {
                const int d = qi[rt] + cs.q.sk - cs.q.sq;
                const int rlo = key_lo(d, a.wl, 0), rhi = min(key_hi(d, a.wr, 0), cs.q.sk - 1);
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = key0 + h * 16 + G * 4 + e;
                        x[rt][h][e] = (ok >> h & 1) && j >= rlo && j <= rhi ? x[rt][h][e] : -INFINITY;
                    }
            }
            // values that no row sees must not meet the products, where 0 x NaN is NaN
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int j = key0 + h * 16 + G * 4 + i;
                    const bool seen = (ok >> h & 1) && j >= cs.q.lo && j < cs.q.hi;
#pragma unroll
                    for (int w = 0; w < VW; ++w) vv[h][i][w] = seen ? vv[h][i][w] : 0u;
                }
        }
        // R, and the weights' factor for each block
        float vmax = 0.f;
#pragma unroll
        for (int h = 0; h < NH; ++h) vmax = fmaxf(vmax, fabsf(vs[h]));
        const int e = (int)(__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, vmax)) >> 23) + 1;
        const int up = max(e - eR, 0);
        eR += up;
        const float shrink = up > 126 ? 0.f : exp2i(-up), toR = exp2i(127 + 14 - eR);
#pragma unroll
        for (int h = 0; h < NH; ++h) vs[h] *= toR;

        u32x4 pk[NR][NH / 2];
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            float mx = -INFINITY;
#pragma unroll
            for (int h = 0; h < NH; ++h) mx = fmaxf(mx, fmaxf(fmaxf(x[rt][h][0], x[rt][h][1]), fmaxf(x[rt][h][2], x[rt][h][3])));
            mx = fmaxf(m_run[rt], wave_max16x4(mx));
            const float m = mx == -INFINITY ? 0.f : mx;
            const float alpha = fast_exp2(m_run[rt] - m);
            m_run[rt] = mx;
            float sum = 0.f;
#pragma unroll
            for (int k2 = 0; k2 < NH / 2; ++k2) {
                f32x8 w;
#pragma unroll
                for (int e2 = 0; e2 < 8; ++e2) {
                    const int h = 2 * k2 + (e2 >> 2);
                    const float p = fast_exp2(x[rt][h][e2 & 3] - m);
                    sum += p;
                    w[e2] = p * vs[h];
                }
                pk[rt][k2] = pack8<DT_FP16>(w);
            }
            l_run[rt] = l_run[rt] * alpha + sum;
            const float c = alpha * shrink;
#pragma unroll
            for (int j = 0; j < VB; ++j) oacc[rt][j] *= c;
        }
        // O^T += V^T . P^T: columns 4w .. 4w + 3 of two blocks at a time
#pragma unroll
        for (int k2 = 0; k2 < NH / 2; ++k2)
#pragma unroll
            for (int w = 0; w < VW; ++w) {
                u32x4 op[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) {  // block c >> 1, keys 2 (c & 1) and the next
                    const uint32_t r0 = vv[2 * k2 + (c >> 1)][2 * (c & 1)][w], r1 = vv[2 * k2 + (c >> 1)][2 * (c & 1) + 1][w];
                    const u32x2 lo = widen4<CT>(byte_perm(r1, r0, 0x05010400u)), hi = widen4<CT>(byte_perm(r1, r0, 0x07030602u));
                    op[0][c] = lo[0];
                    op[1][c] = lo[1];
                    op[2][c] = hi[0];
                    op[3][c] = hi[1];
                }
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int rt = 0; rt < NR; ++rt) oacc[rt][4 * w + j] = mfma_f16(op[j], pk[rt][k2], oacc[rt][4 * w + j]);
            }
    };

    begin_seg();
#pragma unroll
    for (int st = 0; st < STAGES - 1; ++st) issue(t0 + st, kr[st], vr[st]);
    int filled = t0 + TAB;
    for (int tb = t0; tb < t1; tb += STAGES) {
        // the loads of this round reach tile tb + 2 STAGES - 2; the half that is
        // written over lies a half behind
        static_assert(2 * STAGES <= TAB, "");
        if (tb + 2 * STAGES > filled && filled < t1) {
            fill(filled);
            filled += TAB;
        }
#pragma unroll
        for (int st = 0; st < STAGES; ++st) {
            const int t = tb + st;
            if (t < t1) {
                issue(t + STAGES - 1, kr[(st + STAGES - 1) % STAGES], vr[(st + STAGES - 1) % STAGES]);
                if (t >= cs.S + cs.n) {
                    end_seg();
                    cs = seg_of(a, s_pref, s_seq, t, hs, hsel, KT);
                    begin_seg();
                }
                compute(t, kr[st], vr[st]);
            }
        }
    }
    end_seg();
}

// Merge of what a segment's workers left (fa_decode_merge_kernel's rules for which
// they are): 16 rows of a segment per workgroup and blockIdx.y; groups of threads
// fold a share of the partials each, with a running maximum, and meet in LDS.
template <int HD>
__global__ void __launch_bounds__(256) fa_quant_merge_kernel(QuantFwdArgs a, int workers, int nr) {
    __shared__ __attribute__((aligned(16))) float s_acc[256][8];
    __shared__ float s_gm[256], s_gs[256];
    constexpr int CH = HD / 2 / 8;  // 8-column chunks of a row, half of them in each workgroup
    const int sig = blockIdx.x >> 1, half = blockIdx.x & 1;
    const int b = sig / a.Hk, hk = sig % a.Hk;
    const int hs = heads_per_group(a), hgs = a.Hk / hs, hg = hk / hs, hsel = hk % hs;
    int sq = a.cu_q ? a.cu_q[b + 1] - a.cu_q[b] : a.Sq;
    sq = min(max(sq, 0), a.Sq);
    const int row0 = blockIdx.y * 16, rows = min(sq * a.g - row0, 16);
    if (rows <= 0 || sq * a.g > a.dec_rows) return;
    const long long T = a.sched[a.B], W = workers / hs;
    const int per = (a.sched[b + 1] - a.sched[b]) / hgs;
    const long long S = a.sched[b] + (long long)hg * per;
    const long long ovh = dec::seg_ovh(T, W, (long long)a.B * hgs);
    const long long CT_ = dec::split_total(T, ovh, a.B, hgs);
    auto owner = [&](long long t) { return dec::split_owner(t + ovh * ((long long)b * hgs + hg), W, CT_); };
    long long wf = 0;
    int n = 0;
    if (per > 0) {
        wf = owner(S);
        n = T >= W ? (int)(owner(S + per - 1) - wf + 1) : per;
        if (n == 1) return;  // written by its one worker
    }
    bool slot1 = false;  // the first partial is its worker's last
    if (per > 0 && S > 0) {
        const long long jp = ovh > 0 ? dec::split_prev_segment(b, hg, hgs, a.sched) : 0;
        slot1 = dec::split_owner(S - 1 + ovh * jp, W, CT_) == wf;
    }
    const int tid = threadIdx.x;
    int rp = 1;
    while (rp < rows) rp <<= 1;
    const int GS = CH * rp, NG = 256 / GS;
    const int grp = tid / GS, rr = tid % GS / CH, d0 = half * (HD / 2) + tid % CH * 8;
    float m = -INFINITY, sum = 0.f;
    f32x4 acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
    if (rr < rows) {
#pragma unroll 4
        for (int j = grp; j < n; j += NG) {
            const long long w = T >= W ? wf + j : owner(S + j);
            const int64_t pr = ((w * hs + hsel) * 2 + (j == 0 && slot1 ? 1 : 0)) * (16 * nr) + row0 + rr;
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
    if (NG > 1) {
        *reinterpret_cast<f32x4*>(&s_acc[tid][0]) = acc0;
        *reinterpret_cast<f32x4*>(&s_acc[tid][4]) = acc1;
        s_gm[tid] = m;
        s_gs[tid] = sum;
        __syncthreads();
        if (grp != 0) return;
        float M = m;
        for (int q = 1; q < NG; ++q) M = fmaxf(M, s_gm[tid + q * GS]);
        if (M != -INFINITY) {
            const float c = fast_exp2((m - M) * kLog2e);
            acc0 *= c;
            acc1 *= c;
            sum *= c;
            for (int q = 1; q < NG; ++q) {
                const int o = tid + q * GS;
                const float cg = fast_exp2((s_gm[o] - M) * kLog2e);
                acc0 += *reinterpret_cast<const f32x4*>(&s_acc[o][0]) * cg;
                acc1 += *reinterpret_cast<const f32x4*>(&s_acc[o][4]) * cg;
                sum += s_gs[o] * cg;
            }
        }
        m = M;
    }
    if (rr >= rows) return;
    const float inv = m == -INFINITY ? 0.f : 1.f / sum;
    acc0 *= inv;
    acc1 *= inv;
    const int r = row0 + rr, i = r / a.g, h = hk * a.g + r % a.g;
    uint16_t* o = static_cast<uint16_t*>(a.out) + q_row(a, b, i, a.o_sb, a.o_si) + (int64_t)h * a.o_sh;
    if (d0 < a.hd)
        *reinterpret_cast<u32x4*>(o + d0) = u32x4{pack2(acc0[0], acc0[1], a.bf16), pack2(acc0[2], acc0[3], a.bf16),
                                                  pack2(acc1[0], acc1[1], a.bf16), pack2(acc1[2], acc1[3], a.bf16)};
    if (d0 == 0) a.lse[lse_at(a, b, h, i)] = m == -INFINITY ? INFINITY : m + fast_log2(sum) * kLn2;
}

template <int CT, int HD, int NR>
void launch_h(const QuantFwdArgs& a, int grid, hipStream_t stream) {
    if (a.hd < HD) hipLaunchKernelGGL((fa_quant_decode_kernel<CT, HD, NR, true>), dim3(grid), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((fa_quant_decode_kernel<CT, HD, NR, false>), dim3(grid), dim3(256), 0, stream, a);
}

template <int CT, int HD>
void launch_n(const QuantFwdArgs& a, int nr, int grid, hipStream_t stream) {
    if (nr == 1) launch_h<CT, HD, 1>(a, grid, stream);
    else if (nr == 2) launch_h<CT, HD, 2>(a, grid, stream);
    else launch_h<CT, HD, 4>(a, grid, stream);
    hipLaunchKernelGGL((fa_quant_merge_kernel<HD>), dim3(a.B * a.Hk * 2, nr), dim3(256), 0, stream, a, grid * NWAVE, nr);
}

template <int HD>
void launch_d(const QuantFwdArgs& a, int ct, int nr, int grid, hipStream_t stream) {
    if (ct == CT_INT8) launch_n<CT_INT8, HD>(a, nr, grid, stream);
    else launch_n<CT_E4M3, HD>(a, nr, grid, stream);
}

}  // namespace

int quant_decode_workers(int grid) { return grid * NWAVE; }

// kd: kernel head dim; nr: 16-row tiles (1, 2 or 4)
hipError_t launch_quant_decode(const QuantFwdArgs& a, int ct, int kd, int nr, int grid, hipStream_t stream) {
    if (kd == 64) launch_d<64>(a, ct, nr, grid, stream);
    else if (kd == 128) launch_d<128>(a, ct, nr, grid, stream);
    else launch_d<256>(a, ct, nr, grid, stream);
    return hipGetLastError();
}

}  // namespace fa
