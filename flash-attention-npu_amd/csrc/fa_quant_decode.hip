// fa_quant_decode.hip -- attention over 8-bit codes for few query rows (a kv
// head's g query heads x positions, at most 32 packed rows): the cache is
// streamed once, at the rate that HBM gives.
//
// Split: the 32-key tiles (64 at head dim 64) of all sequences and kv heads form
// one list, built in LDS by each workgroup from cache_seqlens and cut into equal
// contiguous ranges, one per wave; waves of a CU take adjacent kv heads of one
// range, so that a key row is requested by a CU at once. A range that ends inside a
// sequence leaves a partial, merged by the second launch.
//
// Loads go straight into LDS: each wave has two tiles of keys and two of values there
// and asks for tile t + 2 of either as soon as it is through with tile t's, so no
// barrier is needed and 8 waves (4 at head dim 256) keep about 96 KB in flight. Two
// waves per SIMD, since the chain of one tile (reads, products, maximum over lanes,
// exponentials, products) takes 2500 clocks, as long as HBM takes for two. Rows are
// swizzled by the order in which the lanes load. A lane reads the quarter of a key row
// that is its operand of S^T = K.Q^T once widened, and V^T for O^T = V^T.P^T by byte
// transpose reads of the key rows that its weights belong to. Page ids and scales
// come through a small table in LDS, filled 32 blocks of 16 keys at a time, in steps
// some tiles apart: a wait for the table would be one for every row asked for before.
//
// Scales: the K scale of 16 keys multiplies their scores, the V scale t goes into the
// weights' exponent (fa_quant.h), 2^14 w rounded to fp16: a weight keeps its 11 bits as
// long as it is more than 2^-28 of its row's largest.
//
// Measured (D128, g 4 and 8): 64 paged e4m3 sequences, 966 MB: 188-194 us, 5.0-5.2 TB/s; 32
// contiguous int8 ones, 194 MB: 53 us; 4 tokens over a window of 4096, 8 sequences:
// 32 us; one sequence of 777 keys: 15.3 us, 12 here, of which the start before the first
// tile (list, ids, rows, scales: each waits for the one before) is most, and 4 in the merge.
// Tiles in registers instead of LDS, with one wave per SIMD: 190, 55, 36 and 15 us.
#include "fa_quant_list.h"

#include <algorithm>

namespace fa {

namespace {

template <int HD>
struct Cfg {
    static constexpr int NWAVE = HD == 256 ? 4 : 8;    // waves of a workgroup
    static constexpr int KT = HD == 64 ? 64 : 32;      // keys of a tile
    static constexpr int NH = KT / 16;                 // blocks of 16
    static constexpr int TAB = 32 / NH;                // tiles of one half of a wave's table
    static constexpr int KL = HD / 64;                 // 16-byte reads of a lane for its quarter key row
    static constexpr int KSTEPS = HD / 32;
    static constexpr int DBLK = HD / 16;
    static constexpr int LPB = HD / 64;                // 1 KB loads of a block
    static constexpr int TILE = KT * HD;               // bytes of a tile of keys or of values
    static constexpr int LOADS = NH * LPB;             // loads of it
    // swizzle of the 16-byte chunks of row r
    static __device__ __forceinline__ int f(int r) { return HD == 64 ? (r >> 1) & 3 : HD == 128 ? r & 7 : r & 15; }
};

// One 16-key block of K or V into LDS: LPB loads of 1 KB, as dma16x4 (fa_pipe.h).
template <int LPB>
__device__ __forceinline__ void dma_block(unsigned lds, const char* base, const unsigned (&off)[LPB]) {
    if constexpr (LPB == 4) {
        dma16x4(lds, base, off);
    } else {
        base = uniform(base);
        lds = __builtin_amdgcn_readfirstlane(lds);
        if constexpr (LPB == 2)
            asm volatile(
                "s_mov_b32 m0, %0\n\ts_nop 3\n\t"
                "global_load_lds_dwordx4 %2, %1\n\t"
                "global_load_lds_dwordx4 %3, %1 offset:1024" ::"s"(lds), "s"(base), "v"(off[0]), "v"(off[1])
                : "memory", "m0");
        else
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %2, %1" ::"s"(lds), "s"(base), "v"(off[0])
                         : "memory", "m0");
    }
}

// DT: type of q and out; CT: cache type; HD: kernel head dim (the cache's may be smaller: columns past it
// repeat the row's first and meet zeros of q); NR: 16-row tiles of packed rows.
template <int DT, int CT, int HD, int NR>
__global__ void __launch_bounds__(Cfg<HD>::NWAVE * 64, 1) fa_quant_decode_kernel(QuantFwdArgs a) {
    using C = Cfg<HD>;
    constexpr int NWAVE = C::NWAVE, NT = NWAVE * 64, KT = C::KT, NH = C::NH, TAB = C::TAB, KL = C::KL, KSTEPS = C::KSTEPS,
                  DBLK = C::DBLK, LPB = C::LPB;
    __shared__ __attribute__((aligned(1024))) uint8_t s_ring[NWAVE][4 * C::TILE];
    __shared__ int s_pref[kQuantMaxB + 1];
    __shared__ int64_t s_koff[NWAVE][64], s_voff[NWAVE][64];
    __shared__ float s_ks[NWAVE][64], s_vs[NWAVE][64], s_lv[NWAVE][64], s_iv[NWAVE][64];
    __shared__ int s_ok[NWAVE][64 / NH];

    // The arguments read anew where they are used once in many tiles (the assembly hides
    // that they stay the same): held all along they would not fit in scalar registers.
    auto anew = []() -> const QuantFwdArgs& {
        auto p = __builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(p));
        return *(const QuantFwdArgs*)p;
    };
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, G = lane >> 4;
    const int hs = heads_per_group(a), hgs = a.Hk / hs;

    // ---- the list of tiles ----------------------------------------------------------
    for (int b = tid; b < a.B; b += NT) {
        const QuantSeq s = quant_seq(a, b);
        s_pref[b + 1] = s.hi > s.lo && s.sq * a.g <= a.dec_rows ? hgs * ((s.hi + KT - 1) / KT - s.lo / KT) : 0;
    }
    __syncthreads();
    if (wave == 0) prefix_sums(s_pref, a.B);
    __syncthreads();
    if (blockIdx.x == 0)
        for (int b = tid; b <= a.B; b += NT) a.sched[b] = s_pref[b];

    const int hsel = wave % hs;
    const int gw = (wave / hs) * gridDim.x + blockIdx.x;  // wave-major, as in fa_decode.hip
    const int64_t wid = (int64_t)gw * hs + hsel;
    const Split sp = split_list(s_pref[a.B], gridDim.x * (NWAVE / hs));
    const int t0 = __builtin_amdgcn_readfirstlane(sp.first(gw)), t1 = __builtin_amdgcn_readfirstlane(sp.first(gw + 1));
    if (t0 >= t1) return;  // no barrier follows: the waves go on alone

    // ---- the table: offsets, scales and visibility of the 16-key blocks ------------------
    // Tiles base .. base + TAB - 1, a block for each of 32 lanes. A block without a visible
    // key has the offset of a row that is there and plain scales. In
    // steps: page ids asked for; offsets, scales asked for; scales. tlv, tiv: log2 and
    // inverse (times 2^-14) of V's scale; tok: the tile's visible blocks, and bit 8 where V's scales are plain.
    int64_t* koff = s_koff[wave];
    int64_t* voff = s_voff[wave];
    float *tks = s_ks[wave], *tvs = s_vs[wave], *tlv = s_lv[wave], *tiv = s_iv[wave];
    int* tok = s_ok[wave];
    int id, inp, kvh;
    float ksv, vsv;
    auto fill_ids = [&](int base) {
        const QuantFwdArgs& A = anew();
        const int t = base + lane / NH;
        id = -1;
        inp = kvh = 0;
        if (lane < 32 && t < t1) {
            const Seg s = seg_of(A, s_pref, t, hs, hsel, KT);
            const int key = (s.lo_tile + (t - s.S)) * KT + (lane % NH) * 16;
            kvh = s.hk;
            if (key < s.q.hi && key + 16 > s.q.lo) {
                const int pi = A.table ? (int)udiv(A.page, (uint32_t)key) : 0;
                inp = key - pi * A.page_size;
                id = A.table ? A.table[(int64_t)s.q.crow * A.t_stride + pi] : s.q.crow;
            }
        }
    };
    auto slot_of = [&](int base) { return (((base - t0) / TAB) & 1) * 32 + (lane & 31); };
    auto fill_rows = [&](int base) {
        const QuantFwdArgs& A = anew();
        const bool ok = id >= 0 && id < A.num_pages;
        const int64_t p = ok ? id : 0, r = ok ? inp : 0, h = kvh;
        const int64_t sb = udiv(A.sblk, (uint32_t)r);
        ksv = A.ks[p * A.ks_sp + sb * A.ks_sb + h * A.ks_sh];
        vsv = A.vs[p * A.vs_sp + sb * A.vs_sb + h * A.vs_sh];
        const int at = slot_of(base);
        if (lane < 32) {
            koff[at] = p * A.k_sp + r * A.k_si + h * A.k_sh;
            voff[at] = p * A.v_sp + r * A.v_si + h * A.v_sh;
        }
    };
    auto fill_scales = [&](int base) {
        const bool ok = id >= 0 && id < a.num_pages;
        const int at = slot_of(base);
        const float v = ok ? vsv : 1.f, lv = scale_log2(v);
        const unsigned long long mo = __ballot(ok), mp = __ballot(plain_scale(v));
        if (lane < 32) {
            constexpr int kAll = (1 << NH) - 1;
            tks[at] = ok ? ksv : 1.f;
            tvs[at] = v;
            tlv[at] = lv;
            tiv[at] = fast_exp2(-14.f - lv);
            if (lane % NH == 0) tok[at / NH] = ((int)(mo >> lane) & kAll) | ((((int)(mp >> lane) & kAll) == kAll) << 8);
        }
    };

    // ---- loads ------------------------------------------------------------------------
    const unsigned ring = lds_addr(s_ring[wave]);
    unsigned kin[LPB], vin[LPB];  // what a lane loads of a block: chunk c ^ f(r) of row r to chunk c
#pragma unroll
    for (int u = 0; u < LPB; ++u) {
        const int at = u * 64 + lane, r = at / DBLK, c = (at % DBLK) ^ C::f(r), col = c * 16 < a.hd ? c * 16 : 0;
        kin[u] = (unsigned)r * (unsigned)a.k_si + col + (LPB - 1 - u) * 1024;
        vin[u] = (unsigned)r * (unsigned)a.v_si + col + (LPB - 1 - u) * 1024;
    }
    auto issue_k = [&](int t) {
        if (t >= t1) return;
        const int at = (t - t0) % (2 * TAB) * NH;
        const unsigned to = ring + ((t - t0) & 1) * C::TILE;
        int64_t off[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) off[h] = koff[at + h];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // also: the reads of the tile that is written over are done
#pragma unroll
        for (int h = 0; h < NH; ++h)
            dma_block<LPB>(to + h * (16 * HD), reinterpret_cast<const char*>(a.k + off[h]) - (LPB - 1) * 1024, kin);
    };
    auto issue_v = [&](int t) {
        if (t >= t1) return;
        const int at = (t - t0) % (2 * TAB) * NH;
        const unsigned to = ring + (2 + ((t - t0) & 1)) * C::TILE;
        int64_t off[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) off[h] = voff[at + h];
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int h = 0; h < NH; ++h)
            dma_block<LPB>(to + h * (16 * HD), reinterpret_cast<const char*>(a.v + off[h]) - (LPB - 1) * 1024, vin);
    };

    // ---- a segment: q, sums ----------------------------------------------------------------
    Seg cs;
    u32x4 qreg[NR][KSTEPS];
    float qs[NR];              // what the scores of a row are to be multiplied by for its q_shift
    int qi[NR];
    f32x4 oacc[NR][DBLK];
    float u_run[NR], l_run[NR], m_run[NR];
    bool apart = false;        // l is relative to m, else to u
    int rows = 0;
    int flo = 0, fhi = 0;      // keys that every row sees
    auto load_q = [&](int t) {
        const QuantFwdArgs& A = anew();
        cs = seg_of(A, s_pref, t, hs, hsel, KT);
        rows = cs.q.sq * A.g;
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            const int r = rt * 16 + li;
            const bool ok = r < rows;
            qi[rt] = ok ? r / A.g : 0;
            const int h = cs.hk * A.g + (ok ? r % A.g : 0);
            const uint16_t* q = static_cast<const uint16_t*>(A.q) + q_row(A, cs.b, qi[rt], A.q_sb, A.q_si) + (int64_t)h * A.q_sh;
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s) {
                const int d = G * (HD / 4) + 8 * s;
                qreg[rt][s] = ok && d < A.hd ? *reinterpret_cast<const u32x4*>(q + d) : u32x4{0u, 0u, 0u, 0u};
            }
        }
    };
    const float scale2 = a.softcap > 0.f ? a.scale / a.softcap : a.scale * kLog2e;
    auto begin_seg = [&]() {
        flo = key_lo(cs.q.sk - 1, a.wl, 0);
        fhi = min(key_hi(cs.q.sk - cs.q.sq, a.wr, 0), cs.q.sk - 1);
        apart = false;
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            float most = 0.f;
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s) {
                const f32x8 x = widen8<DT>(qreg[rt][s]);
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[e]));
            }
            const int sh = q_shift(max4(most));
            const float up = exp2i(sh);
            qs[rt] = exp2i(-sh) * scale2;
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s) qreg[rt][s] = pack8<DT_FP16>(widen8<DT>(qreg[rt][s]) * up);
            u_run[rt] = m_run[rt] = -INFINITY;
            l_run[rt] = 0.f;
#pragma unroll
            for (int db = 0; db < DBLK; ++db) oacc[rt][db] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    };
    auto end_seg = [&]() {
        const QuantFwdArgs& A = anew();
        const bool whole = cs.S >= t0 && cs.S + cs.n <= t1;
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            const int r = rt * 16 + li;
            const float l = wave_sum16x4(l_run[rt]);
            const bool some = l != 0.f;  // NaN: some
            // 2^(u - m) may be out of range where the quotient is not: half of it on either side
            const float up = apart && some ? fast_exp2(0.5f * (u_run[rt] - m_run[rt])) : 1.f;
            if (apart) {
#pragma unroll
                for (int db = 0; db < DBLK; ++db) oacc[rt][db] *= up;
            }
            const float inv = some ? up * 0x1p-14f / l : 0.f;
            const float lse = some ? add_log2(apart ? m_run[rt] : u_run[rt], l) * kLn2 : INFINITY;
            if (r >= rows) continue;
            if (whole) {
                const int h = cs.hk * A.g + r % A.g;
                uint16_t* o = static_cast<uint16_t*>(A.out) + q_row(A, cs.b, qi[rt], A.o_sb, A.o_si) + (int64_t)h * A.o_sh;
#pragma unroll
                for (int db = 0; db < DBLK; ++db) {
                    if (16 * db >= A.hd) continue;
                    const f32x4 y = oacc[rt][db] * inv;
                    *reinterpret_cast<u32x2*>(o + 16 * db + 4 * G) = u32x2{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
                }
                if (G == 0) A.lse[lse_at(A, cs.b, h, qi[rt])] = lse;
            } else {
                const int slot = cs.S <= t0 ? 0 : 1;  // this worker's first segment, else its last
                const int64_t row = (wid * 2 + slot) * (16 * NR) + r;
#pragma unroll
                for (int db = 0; db < DBLK; ++db)
                    *reinterpret_cast<f32x4*>(A.part_o + row * HD + 16 * db + 4 * G) = oacc[rt][db] * inv;
                if (G == 0) A.part_lse[row] = some ? lse : -INFINITY;
            }
        }
    };

    // ---- a tile ----------------------------------------------------------------------------
    const int kx = C::f(li) << 4;
    // the key row of the transpose reads, in the first of two blocks for lanes 0-7 of
    // a group of 16 and in the second for the others
    const int vrow = (li >> 3) * 16 + 4 * G + ((li >> 1) & 3), vx = C::f(vrow) << 4;
    auto compute = [&](int t) {
        const int key0 = (cs.lo_tile + (t - cs.S)) * KT;
        const int at = (t - t0) % (2 * TAB);
        const unsigned kt = ring + ((t - t0) & 1) * C::TILE, vt = kt + 2 * C::TILE;
        // behind tile t's keys: its values, the next tile's keys and values
        if (t + 1 < t1) wait_loads<3 * C::LOADS>();
        else wait_loads<C::LOADS>();
        float ks[NH], lv[NH], iv[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            ks[h] = tks[at * NH + h];
            lv[h] = tlv[at * NH + h];
            iv[h] = tiv[at * NH + h];
        }
        const int bits = __builtin_amdgcn_readfirstlane(tok[at]), ok = bits & ((1 << NH) - 1);
        const bool plain = bits >> 8 & 1;
        const bool full = ok == (1 << NH) - 1 && key0 >= flo && key0 + KT - 1 <= fhi;
        // S^T = K . Q^T on the codes
        f32x4 x[NR][NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) x[rt][h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KL; ++s) {
                const u32x4 k = row_read(kt + (h * 16 + li) * HD + (((G * KL + s) << 4) ^ kx));
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const u32x2 lo = widen4<CT>(k[2 * u]), hi = widen4<CT>(k[2 * u + 1]);
                    const u32x4 op = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                    for (int rt = 0; rt < NR; ++rt) x[rt][h] = mfma_f16(op, qreg[rt][2 * s + u], x[rt][h]);
                }
            }
        }
        issue_k(t + 2);
        // one reference again where the two are close
        if (plain && apart) {
            float d[NR];
            bool far = false;
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) {
                d[rt] = m_run[rt] == u_run[rt] ? 0.f : m_run[rt] - u_run[rt];
                far |= !(fabsf(d[rt]) <= 60.f);
            }
            if (!__ballot(far)) {
                apart = false;
#pragma unroll
                for (int rt = 0; rt < NR; ++rt) l_run[rt] *= fast_exp2(d[rt]);
            }
        }
        if (!plain && !apart) {
            apart = true;
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) m_run[rt] = u_run[rt];
        }
        // scores in log2 units, the log2 of V's scale added where there is one reference
        float add[NH];
#pragma unroll
        for (int h = 0; h < NH; ++h) add[h] = apart ? 0.f : lv[h];
        if (a.softcap > 0.f) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt)
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        x[rt][h][e] = __builtin_fmaf(a.softcap * kLog2e, fast_tanh(x[rt][h][e] * (qs[rt] * ks[h])), add[h]);
        } else {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt)
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[rt][h][e] = __builtin_fmaf(x[rt][h][e], qs[rt] * ks[h], add[h]);
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
        }
        u32x4 pk[NR][NH / 2];
        auto top = [&](const f32x4& y) { return fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3])); };
        if (!apart) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) {
                float mx = -INFINITY;
#pragma unroll
                for (int h = 0; h < NH; ++h) mx = fmaxf(mx, top(x[rt][h]));
                mx = fmaxf(u_run[rt], max4(mx));
                const float u = mx == -INFINITY ? 0.f : mx;
                const float alpha = fast_exp2(u_run[rt] - u);
                u_run[rt] = mx;
                l_run[rt] *= alpha;
#pragma unroll
                for (int k2 = 0; k2 < NH / 2; ++k2) {
                    f32x8 w;
#pragma unroll
                    for (int e2 = 0; e2 < 8; ++e2) w[e2] = fast_exp2(x[rt][2 * k2 + (e2 >> 2)][e2 & 3] - (u - 14.f));
                    l_run[rt] = __builtin_fmaf((w[0] + w[1]) + (w[2] + w[3]), iv[2 * k2], l_run[rt]);
                    l_run[rt] = __builtin_fmaf((w[4] + w[5]) + (w[6] + w[7]), iv[2 * k2 + 1], l_run[rt]);
                    pk[rt][k2] = pack8<DT_FP16>(w);
                }
#pragma unroll
                for (int db = 0; db < DBLK; ++db) oacc[rt][db] *= alpha;
            }
        } else {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) {
                float mx = -INFINITY, ux = -INFINITY;
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    mx = fmaxf(mx, top(x[rt][h]));
                    ux = fmaxf(ux, top(x[rt][h]) + lv[h]);
                }
                mx = fmaxf(m_run[rt], max4(mx));
                ux = fmaxf(u_run[rt], max4(ux));
                const float m = mx == -INFINITY ? 0.f : mx, u = ux == -INFINITY ? 0.f : ux;
                const float alpha = fast_exp2(u_run[rt] - u);
                l_run[rt] *= fast_exp2(m_run[rt] - m);
                m_run[rt] = mx;
                u_run[rt] = ux;
#pragma unroll
                for (int k2 = 0; k2 < NH / 2; ++k2) {
                    f32x8 w;
#pragma unroll
                    for (int e2 = 0; e2 < 8; ++e2) {
                        const int h = 2 * k2 + (e2 >> 2);
                        const float t = tvs[at * NH + h], y = x[rt][h][e2 & 3], p = fast_exp2(y - m);
                        l_run[rt] += p;
                        // a scale that is no number multiplies what is visible
                        w[e2] = copysignf(fast_exp2(y + lv[h] - (u - 14.f)), t) + mul_or_0(p, fabsf(t) < INFINITY ? 0.f : t);
                    }
                    pk[rt][k2] = pack8<DT_FP16>(w);
                }
#pragma unroll
                for (int db = 0; db < DBLK; ++db) oacc[rt][db] *= alpha;
            }
        }
        // behind tile t's values: the next tile's keys and values, the keys after that
        if (t + 2 < t1) wait_loads<3 * C::LOADS>();
        else if (t + 1 < t1) wait_loads<2 * C::LOADS>();
        else wait_loads<0>();
        if (!full) {
            // values that no row sees must not meet the products, where 0 x NaN is NaN
#pragma unroll 1
            for (int c = lane; c < KT * DBLK; c += 64) {
                const int r = c / DBLK, j = key0 + r;
                if (!(ok >> (r >> 4) & 1) || j < cs.q.lo || j >= cs.q.hi) row_write(vt + c * 16, u32x4{0u, 0u, 0u, 0u});
            }
        }
        // O^T += V^T . P^T
#pragma unroll
        for (int k2 = 0; k2 < NH / 2; ++k2)
#pragma unroll
            for (int db = 0; db < DBLK; ++db) {
                const u32x2 v = tr8_read(vt + (32 * k2 + vrow) * HD + ((db << 4) ^ vx) + (li & 1) * 8);
                const u32x2 lo = widen4<CT>(v[0]), hi = widen4<CT>(v[1]);
                const u32x4 op = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                for (int rt = 0; rt < NR; ++rt) oacc[rt][db] = mfma_f16(op, pk[rt][k2], oacc[rt][db]);
            }
        issue_v(t + 2);
    };

    // q and the first page ids are asked for together, then key rows and scales.
    fill_ids(t0);
    load_q(t0);
    fill_rows(t0);
#pragma unroll 1
    for (int t = t0; t < t0 + 2; ++t) {
        issue_k(t);
        issue_v(t);
    }
    fill_scales(t0);
    int qat = t0, send = min(cs.S + cs.n, t1);
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
        // the other half of the table, whose tiles are done
        static_assert(TAB >= 8, "");
        const int step = (t - t0) % TAB, next = t - step + TAB;
        if (next < t1) {
            if (step == 0) fill_ids(next);
            else if (step == 2) fill_rows(next);
            else if (step == 4) fill_scales(next);
        }
        if (t == qat) {
            if (t > t0) {
                load_q(t);
                send = min(cs.S + cs.n, t1);
            }
            begin_seg();
        }
        compute(t);
        if (t + 1 == send) {
            end_seg();
            qat = send;
        }
    }
}

template <int DT, int CT, int HD>
void launch_n(const QuantFwdArgs& a, int nr, int grid, hipStream_t stream) {
    const dim3 nt(Cfg<HD>::NWAVE * 64);
    if (nr == 1) hipLaunchKernelGGL((fa_quant_decode_kernel<DT, CT, HD, 1>), dim3(grid), nt, 0, stream, a);
    else hipLaunchKernelGGL((fa_quant_decode_kernel<DT, CT, HD, 2>), dim3(grid), nt, 0, stream, a);
    launch_list_merge<DT, HD, Cfg<HD>::KT, Cfg<HD>::NWAVE>(a, nr, grid, stream);
}

template <int HD>
void launch_d(const QuantFwdArgs& a, int ct, int nr, int grid, hipStream_t stream) {
    if (a.bf16) {
        if (ct == CT_INT8) launch_n<DT_BF16, CT_INT8, HD>(a, nr, grid, stream);
        else launch_n<DT_BF16, CT_E4M3, HD>(a, nr, grid, stream);
    } else {
        if (ct == CT_INT8) launch_n<DT_FP16, CT_INT8, HD>(a, nr, grid, stream);
        else launch_n<DT_FP16, CT_E4M3, HD>(a, nr, grid, stream);
    }
}

}  // namespace

// Sequences of `capacity` keys that one launch takes: its list of tiles counts in 32 bits, and the
// merge has fewer than 2^32 threads (kd: kernel head dim)
int64_t quant_decode_batch(int kd, int Hk, int64_t capacity) {
    const int64_t hgs = Hk % 4 == 0 ? Hk / 4 : Hk % 2 == 0 ? Hk / 2 : Hk, kt = kd == 64 ? Cfg<64>::KT : Cfg<128>::KT;
    return std::min(0x7fffffffll / (hgs * (capacity / kt + 2)), 0xffffffffll / kMergeThreads / ((int64_t)Hk * (kd / 32)));
}

int quant_decode_workers(int kd, int grid) { return grid * (kd == 256 ? Cfg<256>::NWAVE : Cfg<128>::NWAVE); }

// kd: kernel head dim; nr: 16-row tiles (1 or 2)
hipError_t launch_quant_decode(const QuantFwdArgs& a, int ct, int kd, int nr, int grid, hipStream_t stream) {
    if (kd == 64) launch_d<64>(a, ct, nr, grid, stream);
    else if (kd == 128) launch_d<128>(a, ct, nr, grid, stream);
    else launch_d<256>(a, ct, nr, grid, stream);
    return hipGetLastError();
}

}  // namespace fa
