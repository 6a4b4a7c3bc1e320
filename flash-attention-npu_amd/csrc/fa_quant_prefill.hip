// fa_quant_prefill.hip -- attention over 8-bit codes for many query rows (prompts
// and their chunks, speculated tokens of many heads).
//
// Rows of a work item are (query position, q head) pairs of one kv head; few or
// ragged items are cut over the keys (fa_quant_items.h), the pieces merged by a second launch. Eight
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
#include "fa_quant_items.h"

#include <type_traits>

namespace fa {

namespace {

constexpr int NW = 8, NT = NW * 64;
constexpr float kLazy = 4.f;
constexpr int kUnit = 10;  // w = p t / R 2^kUnit, p <= 2^kLazy

template <int HD, int RB_>
struct Cfg {
    static constexpr int RB = RB_;                                 // 16-row blocks of a wave
    static constexpr int BM = NW * RB * 16;                        // rows of a work item
    static constexpr int BN = 8192 / HD;                           // keys of a tile: 16 codes per thread
    static constexpr int NB = BN / 16;
    static constexpr int DCH = HD / 16;                            // 16-code chunks of a row
    static constexpr int KSTEPS = HD / 32;
    static constexpr int DBLK = HD / 16;
    static constexpr int VPRE = HD == 64 ? 4 : 8;                  // V^T operands read ahead of the softmax
};

// CAP: soft cap
template <int DT, int CT, int HD, int RB_, bool CAP>
__global__ void __launch_bounds__(NT, 1) fa_quant_prefill_kernel(QuantFwdArgs a) {
    using C = Cfg<HD, RB_>;
    constexpr int RB = C::RB, BM = C::BM, BN = C::BN, NB = C::NB, DCH = C::DCH, KSTEPS = C::KSTEPS, DBLK = C::DBLK,
                  VPRE = C::VPRE;
    __shared__ __attribute__((aligned(16))) uint16_t s_k[2][BN * HD];
    __shared__ __attribute__((aligned(16))) uint16_t s_v[2][BN * HD];
    // of the blocks of 16 keys: K scale; V scale, its log2 and inverse; whether the page
    // is in the cache; of the tile: whether the softmax scale and all of these are positive
    __shared__ float s_ks[2][NB], s_vs[2][NB], s_lv[2][NB], s_iv[2][NB];
    __shared__ int s_ok[2][NB], s_plain[2];
    __shared__ int64_t s_koff[2][NB], s_voff[2][NB];  // where its rows are; below 0: nowhere
    __shared__ int s_pref[kQuantMaxB + 1];
    __shared__ int64_t s_line[kQuantMaxB + 1];

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int li = lane & 15, G = lane >> 4;
    build_list<BM, BN, NW>(a, s_pref, s_line);

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
    const uint32_t kin = (uint32_t)(kk & 15) * (uint32_t)a.k_si + (in ? dch * 16 : 0);
    const uint32_t vin = (uint32_t)(kk & 15) * (uint32_t)a.v_si + (in ? dch * 16 : 0);
    auto anew = []() -> const QuantFwdArgs& {  // as in fa_quant_decode.hip
        auto p = __builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(p));
        return *(const QuantFwdArgs*)p;
    };

    const int entries = s_pref[a.B], grid = (int)gridDim.x;
    Line line{};
    int worker = blockIdx.x;
    int64_t at = 0, end;  // places on the line, or numbers of whole items
    if (a.cut) {
        line.len = s_line[min(entries, kQuantMaxB)];
        line.total = line.len * a.Hk;
        line.workers = (int)min((int64_t)grid, max((int64_t)1, line.total / kLeast));
        // all at work: neighbours on the line, who read the same keys, share an XCD's L2
        if (line.workers == grid && grid % 8 == 0) worker = worker % 8 * (grid / 8) + worker / 8;
        if (tid == 0) reinterpret_cast<CutItem*>(a.pf_cut)[worker] = CutItem{0, 0, 0, 0};
        end = 0;
        if (line.total > 0 && worker < line.workers) {
            at = line.cut(worker);
            end = line.cut(worker + 1);
        }
    } else {
        end = (entries * (int64_t)a.Hk + grid - 1) / grid;
    }

    while (at < end) {
        int e, hk, t_lo = 0, t_hi = 0x7fffffff, slot = -1;  // tiles and slot of a piece
        const int g = a.g;
        if (a.cut) {
            hk = (int)(at / line.len);
            const int64_t p0 = hk * line.len;
            e = find_in(s_line, min(entries, kQuantMaxB), at - p0);
        } else {
            // items are numbered heaviest first within a sequence; odd passes run the other way
            const int64_t w = at * grid + ((at & 1) ? grid - 1 - (int)blockIdx.x : (int)blockIdx.x);
            ++at;
            if (w >= entries * (int64_t)a.Hk) continue;
            hk = (int)(w % a.Hk);
            e = (int)(w / a.Hk);
        }
        const int b = find_in(s_pref, a.B, e);
        const Rows R = rows_of<BM>(a, b);
        const int mt = a.cut ? e - s_pref[b] : s_pref[b + 1] - 1 - e;
        const int diag0 = R.q.sk - R.q.sq;
        const int row0 = mt * BM;
        const Keys K = keys_of(a, R.q, row0, min(BM, R.rows - row0));
        int k_lo = K.lo, k_hi = K.hi;
        if (a.cut) {
            const int64_t p0 = hk * line.len + s_line[e], p1 = hk * line.len + s_line[e + 1], upto = min(end, p1);
            const int cost = tile_cost<BM, BM / NW>(R.rows, mt);
            if (at > p0) t_lo = max(0, (int)((at - p0 - kStart) / cost));
            if (upto < p1) t_hi = max(0, (int)((upto - p0 - kStart) / cost));
            if (at > p0 || upto < p1) {
                slot = at > p0 ? 2 * worker : 2 * worker + 1;
                if (at == p0 && tid == 0)
                    reinterpret_cast<CutItem*>(a.pf_cut)[worker] = CutItem{line.holder(p1 - 1) - worker + 1, b, mt, hk};
                const int base = k_lo & ~15;
                if (t_hi < tiles_of<BN>(K)) k_hi = min(k_hi, base + t_hi * BN);
                k_lo = max(k_lo, base + t_lo * BN);
                k_hi = max(k_hi, k_lo);
            }
            at = upto;
        }
        const int base = k_lo & ~15;
        const int ntiles = (k_hi - base + BN - 1) / BN;

        const int wrow0 = row0 + wave * RB * 16, wrows = min(RB * 16, R.rows - wrow0);
        const bool live = wrows > 0;
        const int i_lo = live ? wrow0 / g : 0, i_hi = live ? (wrow0 + wrows - 1) / g : 0;
        const int w_lo = max(k_lo, key_lo(i_lo + diag0, a.wl, 0)), w_hi = min(k_hi - 1, key_hi(i_hi + diag0, a.wr, 0));
        const int f_lo = max(k_lo, key_lo(i_hi + diag0, a.wl, 0)), f_hi = min(k_hi - 1, key_hi(i_lo + diag0, a.wr, 0));

        // ---- tiles: registers -> widened -> LDS ---------------------------------------------
        // The blocks of 16 keys of a tile are looked after by the first NB lanes of the
        // last wave, which causal items leave idle soonest: page id, three tiles ahead
        // of the products; rows' place and scales, two tiles; all others read the place.
        const int* trow = a.table ? a.table + (int64_t)R.q.crow * a.t_stride : nullptr;
        const bool keeper = tid >= NT - 64 && tid < NT - 64 + NB;
        int bid = -1, binp = 0;
        float bks = 0.f, bvs = 0.f;
        bool bok = false;
        auto block_id = [&](int t) {
            const QuantFwdArgs& A = anew();
            const int j = base + t * BN + lane * 16;
            bid = -1;
            binp = 0;
            if (j < k_hi && j + 16 > k_lo) {
                const int pi = trow ? (int)udiv(A.page, (uint32_t)j) : 0;
                binp = j - pi * A.page_size;
                bid = trow ? trow[pi] : R.q.crow;
            }
        };
        auto block_place = [&](int t) {
            const QuantFwdArgs& A = anew();
            bok = bid >= 0 && bid < A.num_pages;
            const int64_t p = bok ? bid : 0, r = bok ? binp : 0;
            s_koff[t & 1][lane] = bok ? p * A.k_sp + r * A.k_si : -1;
            s_voff[t & 1][lane] = p * A.v_sp + r * A.v_si;
            const int64_t sb = udiv(A.sblk, (uint32_t)r);
            bks = A.ks[p * A.ks_sp + sb * A.ks_sb + (int64_t)hk * A.ks_sh];
            bvs = A.vs[p * A.vs_sp + sb * A.vs_sb + (int64_t)hk * A.vs_sh];
        };
        const uint8_t* kbase = a.k + (int64_t)hk * a.k_sh;
        const uint8_t* vbase = a.v + (int64_t)hk * a.v_sh;
        u32x4 kr, vr;
        auto load_tile = [&](int t) {
            const int64_t ko = s_koff[t & 1][kk >> 4], vo = s_voff[t & 1][kk >> 4];
            const int j = base + t * BN + kk;
            const bool ok = ko >= 0 && j >= k_lo && j < k_hi && in;
            kr = u32x4{0u, 0u, 0u, 0u};
            vr = kr;
            if (ok) {
                kr = *reinterpret_cast<const u32x4*>(kbase + ko + kin);
                vr = *reinterpret_cast<const u32x4*>(vbase + vo + vin);
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
            if (keeper) {
                s_ks[buf][lane] = bok ? bks : 0.f;
                s_vs[buf][lane] = bok ? bvs : 0.f;
                s_lv[buf][lane] = fast_log2(bvs);
                s_iv[buf][lane] = 1.f / bvs;
                s_ok[buf][lane] = bok;
                const unsigned long long odd = __ballot(!bok || !(anew().scale > 0.f && bks > 0.f && bks < INFINITY && bvs > 0x1p-100f && bvs < 0x1p100f));
                if (lane == 0) s_plain[buf] = odd == 0;
            }
        };
        // the tiles of the item before are read by all when the first barrier is passed
        __syncthreads();
        if (ntiles > 0 && keeper) {
            block_id(0);
            block_place(0);
            block_id(1);
        }
        __syncthreads();
        if (ntiles > 0) load_tile(0);

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

        // 32 keys of the tile in buf, those at 32 hh. PLAIN: all rows see all of them and
        // the scales are positive. Scores then stay as the products give them until
        // the exponential's argument, and the V scale goes there too, as its log2, so
        // that the weight comes out whole; the sum of p takes it back, once for a block.
        auto tile = [&](int buf, int hh, int s0, auto plain_tag) {
            constexpr bool PLAIN = decltype(plain_tag)::value;
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
            constexpr bool RAW = PLAIN && !CAP;  // x stays raw
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                float mx = -INFINITY;
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    const float c = qs[rb] * ks[kb];
                    if constexpr (RAW) {
                        mx = fmaxf(mx, c * fmaxf(fmaxf(x[rb][kb][0], x[rb][kb][1]), fmaxf(x[rb][kb][2], x[rb][kb][3])));
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float y = x[rb][kb][e] * c;
                            if constexpr (CAP) y = a.softcap * kLog2e * fast_tanh(y);
                            if constexpr (!PLAIN) {
                                const int j = s0 + kb * 16 + G * 4 + e;
                                y = s_ok[buf][2 * hh + kb] && j >= rlo[rb] && j <= rhi[rb] ? y : -INFINITY;
                            }
                            x[rb][kb][e] = y;
                            mx = fmaxf(mx, y);
                        }
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
            u32x4 pk[RB];
            if constexpr (PLAIN) {
                const float unit = (float)(127 + kUnit - eR), back = exp2i(eR - 127 - kUnit);
                const float lv[2] = {s_lv[buf][2 * hh] + unit, s_lv[buf][2 * hh + 1] + unit};
                const float iv[2] = {s_iv[buf][2 * hh] * back, s_iv[buf][2 * hh + 1] * back};
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    f32x8 wt;
#pragma unroll
                    for (int kb = 0; kb < 2; ++kb) {
                        const float c = RAW ? qs[rb] * ks[kb] : 1.f, d = lv[kb] - m_run[rb];
#pragma unroll
                        for (int e = 0; e < 4; ++e) wt[4 * kb + e] = fast_exp2(__builtin_fmaf(x[rb][kb][e], c, d));
                        l_run[rb] += ((wt[4 * kb] + wt[4 * kb + 1]) + (wt[4 * kb + 2] + wt[4 * kb + 3])) * iv[kb];
                    }
                    pk[rb] = pack8<DT_FP16>(wt);
                }
            } else {
                const float toR = exp2i(127 + kUnit - eR);
                vs[0] *= toR;
                vs[1] *= toR;
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

        // Turn t: tile t's products, tile t + 1 from registers to LDS, tile t + 2 asked
        // for at the place left in turn t - 1, and tile t + 3's left in this one. The
        // keeper's scales of tile t + 1 go down before it asks for tile t + 2's.
        if (ntiles > 0) {
            store_tile(0);
            if (keeper) {
                block_place(1);
                block_id(2);
            }
        }
        __syncthreads();
        if (ntiles > 1) load_tile(1);
        for (int t = 0; t < ntiles; ++t) {
            const int buf = t & 1, s0 = base + t * BN;
            if (live && s0 <= w_hi && s0 + BN > w_lo) {
                const bool plain = __builtin_amdgcn_readfirstlane(s_plain[buf]);
#pragma unroll
                for (int hh = 0; hh < BN / 32; ++hh) {
                    const int h0 = s0 + 32 * hh;
                    if (h0 > w_hi || h0 + 32 <= w_lo) continue;
                    if (plain && h0 >= f_lo && h0 + 31 <= f_hi) tile(buf, hh, h0, std::integral_constant<bool, true>{});
                    else tile(buf, hh, h0, std::integral_constant<bool, false>{});
                }
            }
            if (t + 1 < ntiles) {
                store_tile(buf ^ 1);
                if (keeper) {
                    block_place(t + 2);
                    block_id(t + 3);
                }
            }
            __syncthreads();
            if (t + 2 < ntiles) load_tile(t + 2);
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
            if (slot < 0) {
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
                const int64_t prow = (int64_t)slot * BM + (r - row0);
#pragma unroll
                for (int db = 0; db < DBLK; ++db)
                    *reinterpret_cast<f32x4*>(a.pf_o + prow * HD + 16 * db + 4 * G) = oacc[rb][db] * inv;
                if (G == 0) a.pf_lse[prow] = some ? lse : -INFINITY;
            }
        }
    }
}

template <int DT, int CT, int HD, int RB>
void launch_r(const QuantFwdArgs& a, int grid, hipStream_t stream) {
    if (a.softcap > 0.f) hipLaunchKernelGGL((fa_quant_prefill_kernel<DT, CT, HD, RB, true>), dim3(grid), dim3(NT), 0, stream, a);
    else hipLaunchKernelGGL((fa_quant_prefill_kernel<DT, CT, HD, RB, false>), dim3(grid), dim3(NT), 0, stream, a);
    launch_items_merge<DT, HD, Cfg<HD, RB>::BM>(a, grid, stream);
}

template <int HD, int RB>
void launch_c(const QuantFwdArgs& a, int ct, int grid, hipStream_t stream) {
    if (a.bf16) {
        if (ct == CT_INT8) launch_r<DT_BF16, CT_INT8, HD, RB>(a, grid, stream);
        else launch_r<DT_BF16, CT_E4M3, HD, RB>(a, grid, stream);
    } else {
        if (ct == CT_INT8) launch_r<DT_FP16, CT_INT8, HD, RB>(a, grid, stream);
        else launch_r<DT_FP16, CT_E4M3, HD, RB>(a, grid, stream);
    }
}

}  // namespace

// Rows of an item: 128, or as many as the registers take where sequences have them.
int quant_prefill_rows(int kd, bool many) { return many && kd < 256 ? 256 : 128; }

hipError_t launch_quant_prefill(const QuantFwdArgs& a, int ct, int kd, int rows, int grid, hipStream_t stream) {
    if (kd == 64 && rows == 256) launch_c<64, 2>(a, ct, grid, stream);
    else if (kd == 64) launch_c<64, 1>(a, ct, grid, stream);
    else if (kd == 128 && rows == 256) launch_c<128, 2>(a, ct, grid, stream);
    else if (kd == 128) launch_c<128, 1>(a, ct, grid, stream);
    else launch_c<256, 1>(a, ct, grid, stream);
    return hipGetLastError();
}

}  // namespace fa
