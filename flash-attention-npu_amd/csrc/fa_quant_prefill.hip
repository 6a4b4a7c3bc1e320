// fa_quant_prefill.hip -- attention over 8-bit codes for many query rows (prompts
// and their chunks, speculated tokens of many heads).
//
// Rows of a work item are (query position, q head) pairs of one kv head; items with
// few rows and long keys are cut over the keys and merged by a second launch. Eight
// waves (two per SIMD) of 16-row blocks share tiles of keys in LDS, double buffered,
// one barrier a tile. The codes are widened to fp16 once, on their way into LDS, so the
// products meet what 16-bit rows would give them: S^T = K.Q^T, whose accumulator
// holds the P^T operand of O^T = V^T.P^T, V^T by transpose reads. Page ids are read a
// tile ahead of the rows that they lead to.
//
// K's scale multiplies the scores of its 16 keys; V's the weights, kept relative to a
// running power of two (fa_quant_decode.hip). The running maximum is lazy: it moves
// only where a new score exceeds it by 2^4, and the weights' unit leaves room for that
// (2^10 in place of 2^14: a weight keeps its 11 bits as long as p t / R > 2^-24).
#include "fa_pipe.h"
#include "fa_quant.h"

#include <type_traits>

namespace fa {

namespace {

constexpr int MAXB = 2048;
constexpr int NW = 8, NT = NW * 64;
constexpr float kLazy = 4.f;
constexpr int kUnit = 10;  // w = p t / R 2^kUnit, p <= 2^kLazy

template <int HD>
struct Cfg {
    static constexpr int RB = HD == 64 ? 4 : HD == 128 ? 2 : 1;   // 16-row blocks of a wave
    static constexpr int BM = NW * RB * 16;                        // rows of a work item
    static constexpr int BN = 8192 / HD;                           // keys of a tile: 16 codes per thread
    static constexpr int NB = BN / 16;
    static constexpr int DCH = HD / 16;                            // 16-code chunks of a row
    static constexpr int KSTEPS = HD / 32;
    static constexpr int DBLK = HD / 16;
    static constexpr int VPRE = HD == 64 ? 4 : 8;                  // V^T operands read ahead of the softmax
};

struct Rows {
    int rows, mt;
    QuantSeq q;
};

template <int BM>
__device__ __forceinline__ Rows rows_of(const QuantFwdArgs& a, int b) {
    Rows r;
    r.q = quant_seq(a, b);
    if (r.q.hi < r.q.lo) r.q.hi = r.q.lo;
    r.rows = r.q.sq * a.g > a.dec_rows ? r.q.sq * a.g : 0;
    r.mt = (r.rows + BM - 1) / BM;
    return r;
}

__device__ __forceinline__ void split_of(const QuantFwdArgs& a, int range, int chunk_auto, int& ns, int& chunk) {
    chunk = chunk_auto;
    ns = a.allow_split && range > 0 ? (range + chunk - 1) / chunk : 1;
}

// The list of work items: prefix over the sequences in LDS, made by every
// workgroup alike; workgroup 0 leaves it for the merge. Keys are cut into chunks so
// that there are about target_items pieces, none under min_chunk keys.
template <int BM, int BN>
__device__ void build_list(const QuantFwdArgs& a, int* s_pref, long long* s_red, int& total, int& chunk_auto) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    chunk_auto = 0x3fffffff;
    if (a.allow_split) {
        long long work = 0, base = 0;
        for (int b = tid; b < a.B; b += NT) {
            const Rows r = rows_of<BM>(a, b);
            base += (long long)a.Hk * r.mt;
            work += (long long)a.Hk * r.mt * (r.q.hi - r.q.lo);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            work += __shfl_xor(work, o);
            base += __shfl_xor(base, o);
        }
        if (lane == 0) {
            s_red[wave * 2] = work;
            s_red[wave * 2 + 1] = base;
        }
        __syncthreads();
        work = 0;
        base = 0;
        for (int w = 0; w < NW; ++w) {
            work += s_red[w * 2];
            base += s_red[w * 2 + 1];
        }
        if (base < a.target_items) {
            long long c = (work + a.target_items - 1) / a.target_items;
            c = c < a.min_chunk ? a.min_chunk : c;
            c = (c + BN - 1) / BN * BN;
            chunk_auto = (int)(c > 0x3fffffff ? 0x3fffffff : c);
        }
    }
    for (int b = tid; b < a.B; b += NT) {
        const Rows r = rows_of<BM>(a, b);
        int ns, chunk;
        split_of(a, r.q.hi - r.q.lo, chunk_auto, ns, chunk);
        s_pref[b + 1] = a.Hk * r.mt * ns;
        if (blockIdx.x == 0 && a.allow_split) a.pf_sched[a.B + 1 + b] = ns;
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
    total = s_pref[a.B];
    if (blockIdx.x == 0 && a.allow_split)
        for (int b = tid; b <= a.B; b += NT) a.pf_sched[b] = s_pref[b];
}

// CAP: soft cap
template <int DT, int CT, int HD, bool CAP>
__global__ void __launch_bounds__(NT, 1) fa_quant_prefill_kernel(QuantFwdArgs a) {
    using C = Cfg<HD>;
    constexpr int RB = C::RB, BM = C::BM, BN = C::BN, NB = C::NB, DCH = C::DCH, KSTEPS = C::KSTEPS, DBLK = C::DBLK,
                  VPRE = C::VPRE;
    __shared__ __attribute__((aligned(16))) uint16_t s_k[2][BN * HD];
    __shared__ __attribute__((aligned(16))) uint16_t s_v[2][BN * HD];
    __shared__ float s_ks[2][NB], s_vs[2][NB];
    __shared__ int s_ok[2][NB];
    __shared__ int s_pref[MAXB + 1];
    __shared__ long long s_red[2 * NW];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int li = lane & 15, G = lane >> 4;
    int total, chunk_auto;
    build_list<BM, BN>(a, s_pref, s_red, total, chunk_auto);

    auto swzk = [](int r, int c) { return HD == 64 ? swz_k64(r, c) : swz_k(r, c); };
    auto swzv = [](int r, int c) { return HD == 64 ? swz_v64(r, c) : swz_v(r, c); };
    int offk[KSTEPS], offv[DBLK];
#pragma unroll
    for (int s = 0; s < KSTEPS; ++s) offk[s] = li * HD + (swzk(li, 4 * s + G) << 3);
    const int r4 = li >> 2, c4 = li & 3;
#pragma unroll
    for (int db = 0; db < DBLK; ++db)
        offv[db] = (4 * G + r4) * HD + (swzv(4 * G + r4, 2 * db + (c4 >> 1)) << 3) + (c4 & 1) * 4;
    // this thread's part of a tile: 16 codes of one row of K and of V
    const int kk = tid / DCH, dch = tid % DCH;
    const bool in = dch * 16 < a.hd;
    const int sblk = tid % NB, swhich = tid / NB;  // threads below 2 NB carry the scales

    for (int k = 0; k * (int)gridDim.x < total; ++k) {
        // items are numbered heaviest first within a sequence; odd passes run the other way
        const int w = k * (int)gridDim.x + ((k & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x);
        if (w >= total) continue;
        int bl = 0, bh = a.B;
        while (bh - bl > 1) {
            const int mid = (bl + bh) >> 1;
            if (s_pref[mid] <= w) bl = mid;
            else bh = mid;
        }
        const int b = bl, g = a.g;
        const Rows R = rows_of<BM>(a, b);
        int ns, chunk;
        split_of(a, R.q.hi - R.q.lo, chunk_auto, ns, chunk);
        const int local = w - s_pref[b];
        const int hk = local % a.Hk, split = local / a.Hk % ns, mt = R.mt - 1 - local / a.Hk / ns;
        const int diag0 = R.q.sk - R.q.sq;
        const int row0 = mt * BM, item_rows = min(BM, R.rows - row0);
        int k_lo = max(0, key_lo(row0 / g + diag0, a.wl, 0));
        int k_hi = min(R.q.sk, key_hi((row0 + item_rows - 1) / g + diag0, a.wr, 0) + 1);
        if (ns > 1) {
            k_lo = max(k_lo, R.q.lo + split * chunk);
            k_hi = min(k_hi, R.q.lo + (split + 1) * chunk);
        }
        k_hi = max(k_hi, k_lo);
        const int base = k_lo & ~15;  // tiles start at a block of 16 keys
        const int ntiles = (k_hi - base + BN - 1) / BN;

        const int wrow0 = row0 + wave * RB * 16, wrows = min(RB * 16, R.rows - wrow0);
        const bool live = wrows > 0;
        const int i_lo = live ? wrow0 / g : 0, i_hi = live ? (wrow0 + wrows - 1) / g : 0;
        const int w_lo = max(k_lo, key_lo(i_lo + diag0, a.wl, 0)), w_hi = min(k_hi - 1, key_hi(i_hi + diag0, a.wr, 0));
        const int f_lo = max(k_lo, key_lo(i_hi + diag0, a.wl, 0)), f_hi = min(k_hi - 1, key_hi(i_lo + diag0, a.wr, 0));

        // ---- tiles: registers -> widened -> LDS ---------------------------------------------
        const int* trow = a.table ? a.table + (int64_t)R.q.crow * a.t_stride : nullptr;
        auto page_of = [&](int j, int& inp) -> int {  // -1: no key of this item
            inp = 0;
            if (j >= k_hi || j + 16 <= k_lo) return -1;
            const int pi = trow ? (int)udiv(a.page, (uint32_t)j) : 0;
            inp = j - pi * a.page_size;
            return trow ? trow[pi] : R.q.crow;
        };
        u32x4 kr, vr;
        float sc = 0.f;
        int sok = 0;
        int id, inp, sid = -1, sinp = 0;
        auto ids = [&](int t0) {
            id = page_of(t0 + kk, inp);
            if (t0 + kk < k_lo) id = -1;
            if (tid < 2 * NB) sid = page_of(t0 + sblk * 16, sinp);
        };
        auto load_tile = [&]() {  // the rows that `ids` found
            const bool ok = id >= 0 && id < a.num_pages && in;
            kr = u32x4{0u, 0u, 0u, 0u};
            vr = kr;
            if (ok) {
                kr = *reinterpret_cast<const u32x4*>(a.k + (int64_t)id * a.k_sp + (int64_t)inp * a.k_si + (int64_t)hk * a.k_sh + dch * 16);
                vr = *reinterpret_cast<const u32x4*>(a.v + (int64_t)id * a.v_sp + (int64_t)inp * a.v_si + (int64_t)hk * a.v_sh + dch * 16);
            }
            if (tid < 2 * NB) {
                sok = sid >= 0 && sid < a.num_pages;
                sc = 0.f;
                if (sok) {
                    const int64_t sb = udiv(a.sblk, (uint32_t)sinp);
                    sc = swhich ? a.vs[(int64_t)sid * a.vs_sp + sb * a.vs_sb + (int64_t)hk * a.vs_sh]
                                : a.ks[(int64_t)sid * a.ks_sp + sb * a.ks_sb + (int64_t)hk * a.ks_sh];
                }
            }
        };
        auto store_tile = [&](int buf) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const u32x2 k0 = widen4<CT>(kr[2 * u]), k1 = widen4<CT>(kr[2 * u + 1]);
                const u32x2 v0 = widen4<CT>(vr[2 * u]), v1 = widen4<CT>(vr[2 * u + 1]);
                *reinterpret_cast<u32x4*>(&s_k[buf][kk * HD + (swzk(kk & 15, 2 * dch + u) << 3)]) = u32x4{k0[0], k0[1], k1[0], k1[1]};
                *reinterpret_cast<u32x4*>(&s_v[buf][kk * HD + (swzv(kk & 15, 2 * dch + u) << 3)]) = u32x4{v0[0], v0[1], v1[0], v1[1]};
            }
            if (tid < NB) {
                s_ks[buf][sblk] = sc;
                s_ok[buf][sblk] = sok;
            } else if (tid < 2 * NB) {
                s_vs[buf][sblk] = sc;
            }
        };
        // a page outside the cache anywhere in the item: its tiles all test each key
        int bad = 0;
        if (trow && ntiles > 0) {
            const int p0 = (int)udiv(a.page, (uint32_t)k_lo), p1 = (int)udiv(a.page, (uint32_t)(k_hi - 1));
            for (int p = p0 + tid; p <= p1; p += NT) bad |= trow[p] < 0 || trow[p] >= a.num_pages;
        }
        if (ntiles > 0) {
            ids(base);
            load_tile();
            ids(base + BN);
        }
        bad = __syncthreads_or(bad);  // also: the tiles of the item before are read

        // ---- Q --------------------------------------------------------------------------------
        u32x4 qreg[RB][KSTEPS];
        float qs[RB];
        int rlo[RB], rhi[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = wrow0 + rb * 16 + li;
            const bool ok = r < R.rows;
            const int i = ok ? r / g : 0, h = hk * g + (ok ? r % g : 0);
            rlo[rb] = max(k_lo, key_lo(i + diag0, a.wl, 0));
            rhi[rb] = min(k_hi - 1, key_hi(i + diag0, a.wr, 0));
            const int64_t at = q_row(a, b, i, a.q_sb, a.q_si) + (int64_t)h * a.q_sh;
            f32x8 x[KSTEPS];
            float most = 0.f;
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s) {
                const int d = (4 * s + G) * 8;
                x[s] = ok && d < a.hd ? load8<DT>(a.q, at + d) : f32x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf(x[s][e]));
            }
            const int sh = q_shift(wave_max16x4(most));
            const float up = exp2i(sh);
            qs[rb] = exp2i(-sh) * a.scale * (CAP ? 1.f / a.softcap : kLog2e);
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s) qreg[rb][s] = pack8<DT_FP16>(x[s] * up);
        }
        f32x4 oacc[RB][DBLK];
        float m_run[RB], l_run[RB];
        int eR = 30;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            m_run[rb] = -1e30f;  // finite: exp2(x - m) never forms inf - inf
            l_run[rb] = 0.f;
#pragma unroll
            for (int db = 0; db < DBLK; ++db) oacc[rb][db] = f32x4{0.f, 0.f, 0.f, 0.f};
        }

        // 32 keys of the tile in buf, those at 32 hh
        auto tile = [&](int buf, int hh, int s0, auto mask_tag) {
            constexpr bool MASK = decltype(mask_tag)::value;
            f32x4 x[RB][2];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) x[rb][0] = x[rb][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KSTEPS; ++s)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const u32x4 av = *reinterpret_cast<const u32x4*>(&s_k[buf][offk[s] + (hh * 32 + kb * 16) * HD]);
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) x[rb][kb] = mfma_f16(av, qreg[rb][s], x[rb][kb]);
                }
            auto read_vt = [&](int db) {
                const s16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)&s_v[buf][offv[db] + 32 * hh * HD]);
                const s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)&s_v[buf][offv[db] + (32 * hh + 16) * HD]);
                const u32x2 l2 = __builtin_bit_cast(u32x2, lo4), h2 = __builtin_bit_cast(u32x2, hi4);
                return u32x4{l2[0], l2[1], h2[0], h2[1]};
            };
            u32x4 vt[VPRE];
#pragma unroll
            for (int db = 0; db < VPRE; ++db) vt[db] = read_vt(db);
            const float ks[2] = {s_ks[buf][2 * hh], s_ks[buf][2 * hh + 1]};
            float vs[2] = {s_vs[buf][2 * hh], s_vs[buf][2 * hh + 1]};
            const float vmax = fmaxf(fabsf(vs[0]), fabsf(vs[1]));
            const int up = max((int)(__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, vmax)) >> 23) + 1 - eR, 0);
            bool need = up > 0;
            float xmax[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float mx = -INFINITY;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const float c = qs[rb] * ks[kb];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float y = x[rb][kb][e] * c;
                        if constexpr (CAP) y = a.softcap * kLog2e * fast_tanh(y);
                        if constexpr (MASK) {
                            const int j = s0 + kb * 16 + G * 4 + e;
                            y = s_ok[buf][2 * hh + kb] && j >= rlo[rb] && j <= rhi[rb] ? y : -INFINITY;
                        }
                        x[rb][kb][e] = y;
                        mx = fmaxf(mx, y);
                    }
                }
                xmax[rb] = mx;
                need |= mx > m_run[rb] + kLazy;
            }
            if (__ballot(need)) {
                eR += up;
                const float shrink = up > 126 ? 0.f : exp2i(-up);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const float mn = fmaxf(m_run[rb], wave_max16x4(xmax[rb]));
                    const float alpha = fast_exp2(m_run[rb] - mn);
                    m_run[rb] = mn;
                    l_run[rb] *= alpha;
#pragma unroll
                    for (int db = 0; db < DBLK; ++db) {
                        f32x4 o = oacc[rb][db];
                        asm volatile("" : "+v"(o));  // pins the multiply inside this branch
                        oacc[rb][db] = o * (alpha * shrink);
                    }
                }
            }
            const float toR = exp2i(127 + kUnit - eR);
            vs[0] *= toR;
            vs[1] *= toR;
            u32x4 pk[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                f32x8 wt;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float p = fast_exp2(x[rb][e >> 2][e & 3] - m_run[rb]);
                    sum += p;
                    wt[e] = p * vs[e >> 2];
                }
                l_run[rb] += sum;
                pk[rb] = pack8<DT_FP16>(wt);
            }
            __builtin_amdgcn_s_setprio(1);  // the SIMD's other wave fills the slots between these products
#pragma unroll
            for (int db = 0; db < DBLK; ++db) {
                const u32x4 cur = vt[db % VPRE];
                if (db + VPRE < DBLK) vt[db % VPRE] = read_vt(db + VPRE);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) oacc[rb][db] = mfma_f16(cur, pk[rb], oacc[rb][db]);
            }
            __builtin_amdgcn_s_setprio(0);
        };

        if (ntiles > 0) {
            store_tile(0);
            if (ntiles > 1) load_tile();
            ids(base + 2 * BN);
        }
        __syncthreads();
        for (int t = 0; t < ntiles; ++t) {
            const int buf = t & 1, s0 = base + t * BN;
            if (live && s0 <= w_hi && s0 + BN > w_lo) {
#pragma unroll
                for (int hh = 0; hh < BN / 32; ++hh) {
                    const int h0 = s0 + 32 * hh;
                    if (h0 > w_hi || h0 + 32 <= w_lo) continue;
                    if (!bad && h0 >= f_lo && h0 + 31 <= f_hi) tile(buf, hh, h0, std::integral_constant<bool, false>{});
                    else tile(buf, hh, h0, std::integral_constant<bool, true>{});
                }
            }
            if (t + 1 < ntiles) store_tile(buf ^ 1);
            if (t + 2 < ntiles) load_tile();
            ids(base + (t + 3) * BN);
            __syncthreads();
        }

        // ---- results --------------------------------------------------------------------------
        const float back = exp2i(eR - 127 - kUnit);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = wrow0 + rb * 16 + li;
            const float l = wave_sum16x4(l_run[rb]);
            const bool some = l != 0.f;
            const float inv = some ? back / l : 0.f;
            const float lse = some ? (m_run[rb] + fast_log2(l)) * kLn2 : INFINITY;
            if (r >= R.rows) continue;
            if (ns == 1) {
                const int i = r / g, h = hk * g + r % g;
                uint16_t* o = static_cast<uint16_t*>(a.out) + q_row(a, b, i, a.o_sb, a.o_si) + (int64_t)h * a.o_sh;
#pragma unroll
                for (int db = 0; db < DBLK; ++db) {
                    if (16 * db >= a.hd) continue;
                    const f32x4 y = oacc[rb][db] * inv;
                    *reinterpret_cast<u32x2*>(o + 16 * db + 4 * G) = u32x2{pack2<DT>(y[0], y[1]), pack2<DT>(y[2], y[3])};
                }
                if (G == 0) a.lse[lse_at(a, b, h, i)] = lse;
            } else {
                const int64_t prow = (int64_t)w * BM + (r - row0);
#pragma unroll
                for (int db = 0; db < DBLK; ++db)
                    *reinterpret_cast<f32x4*>(a.pf_o + prow * HD + 16 * db + 4 * G) = oacc[rb][db] * inv;
                if (G == 0) a.pf_lse[prow] = some ? lse : -INFINITY;
            }
        }
    }
}

// Merge of split items: a thread for each row and 8 columns.
template <int DT, int HD>
__global__ void __launch_bounds__(256) fa_quant_prefill_merge_kernel(QuantFwdArgs a, int mt_max) {
    constexpr int BM = Cfg<HD>::BM, DCH = HD / 8, RPB = 256 / DCH, BPT = BM / RPB;
    const int blk = blockIdx.x % BPT, item = blockIdx.x / BPT;
    const int hk = item % a.Hk, mt = item / a.Hk % mt_max, b = item / a.Hk / mt_max;
    const int ns = a.pf_sched[a.B + 1 + b];
    if (ns <= 1) return;
    int sq = a.cu_q ? a.cu_q[b + 1] - a.cu_q[b] : a.Sq;
    sq = min(max(sq, 0), a.Sq);
    const int rows = sq * a.g > a.dec_rows ? sq * a.g : 0, mt_b = (rows + BM - 1) / BM;
    const int rr = blk * RPB + threadIdx.x / DCH, d0 = threadIdx.x % DCH * 8, r = mt * BM + rr;
    if (mt >= mt_b || r >= rows) return;
    const int w0 = a.pf_sched[b] + (mt_b - 1 - mt) * ns * a.Hk + hk;
    float m = -INFINITY;
    for (int s = 0; s < ns; ++s) m = fmaxf(m, a.pf_lse[(int64_t)(w0 + s * a.Hk) * BM + rr]);
    f32x4 acc0 = {0.f, 0.f, 0.f, 0.f}, acc1 = acc0;
    float lse = INFINITY;
    if (m != -INFINITY) {
        float sum = 0.f;
        for (int s = 0; s < ns; ++s) {
            const int64_t prow = (int64_t)(w0 + s * a.Hk) * BM + rr;
            const float wgt = fast_exp2((a.pf_lse[prow] - m) * kLog2e);
            sum += wgt;
            acc0 += *reinterpret_cast<const f32x4*>(a.pf_o + prow * HD + d0) * wgt;
            acc1 += *reinterpret_cast<const f32x4*>(a.pf_o + prow * HD + d0 + 4) * wgt;
        }
        acc0 *= 1.f / sum;
        acc1 *= 1.f / sum;
        lse = m + fast_log2(sum) * kLn2;
    }
    const int i = r / a.g, h = hk * a.g + r % a.g;
    uint16_t* o = static_cast<uint16_t*>(a.out) + q_row(a, b, i, a.o_sb, a.o_si) + (int64_t)h * a.o_sh;
    if (d0 < a.hd)
        *reinterpret_cast<u32x4*>(o + d0) = u32x4{pack2<DT>(acc0[0], acc0[1]), pack2<DT>(acc0[2], acc0[3]),
                                                  pack2<DT>(acc1[0], acc1[1]), pack2<DT>(acc1[2], acc1[3])};
    if (d0 == 0) a.lse[lse_at(a, b, h, i)] = lse;
}

template <int DT, int CT, int HD>
void launch_c(const QuantFwdArgs& a, int grid, int mt_max, hipStream_t stream) {
    if (a.softcap > 0.f) hipLaunchKernelGGL((fa_quant_prefill_kernel<DT, CT, HD, true>), dim3(grid), dim3(NT), 0, stream, a);
    else hipLaunchKernelGGL((fa_quant_prefill_kernel<DT, CT, HD, false>), dim3(grid), dim3(NT), 0, stream, a);
    if (!a.allow_split) return;
    constexpr int RPB = 256 / (HD / 8);
    hipLaunchKernelGGL((fa_quant_prefill_merge_kernel<DT, HD>), dim3((unsigned)(a.B * mt_max * a.Hk * (Cfg<HD>::BM / RPB))), dim3(256),
                       0, stream, a, mt_max);
}

template <int HD>
void launch_d(const QuantFwdArgs& a, int ct, int grid, int mt_max, hipStream_t stream) {
    if (a.bf16) {
        if (ct == CT_INT8) launch_c<DT_BF16, CT_INT8, HD>(a, grid, mt_max, stream);
        else launch_c<DT_BF16, CT_E4M3, HD>(a, grid, mt_max, stream);
    } else {
        if (ct == CT_INT8) launch_c<DT_FP16, CT_INT8, HD>(a, grid, mt_max, stream);
        else launch_c<DT_FP16, CT_E4M3, HD>(a, grid, mt_max, stream);
    }
}

}  // namespace

int quant_prefill_rows(int kd) { return kd == 64 ? Cfg<64>::BM : kd == 128 ? Cfg<128>::BM : Cfg<256>::BM; }
int quant_prefill_keys(int kd) { return kd == 64 ? Cfg<64>::BN : kd == 128 ? Cfg<128>::BN : Cfg<256>::BN; }

hipError_t launch_quant_prefill(const QuantFwdArgs& a, int ct, int kd, int grid, int mt_max, hipStream_t stream) {
    if (kd == 64) launch_d<64>(a, ct, grid, mt_max, stream);
    else if (kd == 128) launch_d<128>(a, ct, grid, mt_max, stream);
    else launch_d<256>(a, ct, grid, mt_max, stream);
    return hipGetLastError();
}

}  // namespace fa
