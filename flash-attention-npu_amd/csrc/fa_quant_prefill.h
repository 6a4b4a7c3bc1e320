// fa_quant_prefill.h -- attention over 8-bit or 4-bit codes for many query rows (prompts
// and their chunks, speculated tokens of many heads): the kernel, which two sources
// instantiate.
//
// Rows of a work item are (query position, q head) pairs of one kv head; few or
// ragged items are cut over the keys (fa_quant_items.h), the pieces merged by a
// second launch. Four waves, one per SIMD, of RB x 32 rows.
//   * A tile's codes go from memory straight into LDS, two tiles before they are
//     widened to fp16 there, once for all rows, so the products meet what 16-bit rows
//     would give them.
//   * Per 32 keys a wave forms S^T = K.Q^T and O^T += V^T.P^T with 32x32x16 MFMA: a
//     lane holds one row and 16 keys, which is the packed P^T operand; V^T by transpose
//     reads. While the softmax of 32 keys runs, the scores of the next 32 are formed,
//     and their maximum is taken under the P.V products, in slots of one MFMA and a
//     share of the vector work (unit()).
//   * 4-bit codes meet their scales there: a value has no more than the 2 bits of its code, so
//     rows of q's type hold it with its scale, and nothing below is left of scales. A thread's 32 codes
//     of a row are one group, whose scale byte comes beside them. Weights are then of q's type too: in bf16
//     each is off by up to half a step of 2^-8, as in the 16-bit kernels (the result's error is 1.35
//     times that of exact weights; a second part of them would be half of all products again, and fp16 weights,
//     which the decode kernel has while V's scales lie in fp16's range, a second copy of each unit for those that do not).
//   * K's scale multiplies the scores of its 16 keys. V's goes into the weights'
//     exponent (fa_quant.h), so that the weight comes out whole; the row's sum takes it
//     back once for a block. The running maximum is lazy: it moves only where a
//     new one exceeds it by 2^4, and the weights' unit leaves room for that (the largest
//     is 2^10 to 2^14: a weight keeps its 11 bits as long as it is more than 2^-24 of that).
//   * Tiles with masked keys, pages outside the cache or K scales that are not plain
//     go through a second copy of the unit, which scales the scores as they are formed,
//     and tiles with V scales that are not plain through a third, with two references a row.
//
// What bounds it: the instructions of one wave. 32 keys of 64 rows take about 2640 clocks,
// 1024 of them products; beside them go 32 exponentials (16 clocks each), about 200 other vector
// instructions and the reads. Measured: chunk of 2048 onto 4096 keys, B4 H32/8 D128 e4m3:
// 742-757 us, 910-930 TFLOP/s (two waves per SIMD of 32 rows each, which do products and softmax
// mostly one after the other: 921; page ids and scales of each tile looked up
// in that tile instead of for 64 blocks at once: 927); 40 ragged sequences, H24/8 D64
// int8: 185 us, 150 of them here, where waves wait 27 % of the time, for the 800 starts of items (ids,
// rows, q one after another) above all. The same chunk over 4-bit codes, bf16: 698 us, 984 TFLOP/s (707 with the
// tiles' addresses in vector registers).
#pragma once
#include "fa_fp4.h"
#include "fa_pipe.h"
#include "fa_quant_items.h"
#include "fa_quant_list.h"

#include <type_traits>

namespace fa {

namespace {

constexpr int NW = 4, NT = NW * 64, NBUF = 3;
constexpr float kLazy = 4.f;
enum : int { FAST, MASKED, WILD };  // copies of a unit

template <int HD, int RB_>
struct Cfg {
    static constexpr int RB = RB_;             // 32-row blocks of a wave
    static constexpr int BM = NW * RB * 32;    // rows of a work item
    static constexpr int ROW = 2 * HD;         // bytes of a widened row
    static constexpr int NH = 512 / ROW;       // 32-key units of a tile
    static constexpr int BN = 32 * NH;         // keys of a tile: 32 codes of K and of V per thread
    static constexpr int NB = BN / 16;         // blocks of 16 keys of a tile
    static constexpr int TPG = 64 / NB;        // tiles of a group: its blocks are a wave's lanes
    static constexpr int KS = HD / 16;         // K operands of a unit
    static constexpr int DB = HD / 32;         // 32-dim blocks of O
    static constexpr int DCH = HD / 16;        // 16-code chunks of a row
    static constexpr int KT = BN * ROW;        // bytes of a tile of K (or V) in LDS
    static constexpr int TILE = 2 * KT;
};

// Codes CT as rows of DT meet them: the type of the operands, the log2 of the largest weight less
// kLazy (references are this much below their row's maximum), and a wave's bytes of a tile's codes.
template <int DT, int CT>
struct Operands {
    static constexpr bool FOUR = CT == CT_FP4;
    static constexpr int OT = FOUR ? DT : DT_FP16;
    static constexpr float kUnit = OT == DT_FP16 ? 10.f : -24.f;
    static constexpr int RAW = FOUR ? 2560 : 4096;
};

// 16 bytes per lane from each of four bases (k, k, v, v) + off to LDS address lds + 1024 u
// + 16 lane; the wait states are fa_pipe.h's. b<u> is 1024 u less than the base.
__device__ __forceinline__ void dma16_kkvv(unsigned lds, uint64_t b0, uint64_t b1, uint64_t b2, uint64_t b3, unsigned koff,
                                           unsigned voff) {
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\t"
        "global_load_lds_dwordx4 %5, %1\n\t"
        "global_load_lds_dwordx4 %5, %2 offset:1024\n\t"
        "global_load_lds_dwordx4 %6, %3 offset:2048\n\t"
        "global_load_lds_dwordx4 %6, %4 offset:0xc00" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "s"(b0), "s"(b1), "s"(b2), "s"(b3),
        "v"(koff), "v"(voff)
        : "memory", "m0");
}

// 4-bit codes: 16 bytes per lane of K and of V to lds + 16 lane and 1024 more, a byte of their scales
// each to the dwords at lds + 2048 + 4 lane and 256 more. The addresses are as much less.
__device__ __forceinline__ void dma_fp4(unsigned lds, uint64_t k, uint64_t v, uint64_t ks, uint64_t vs) {
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\t"
        "global_load_lds_dwordx4 %1, off\n\t"
        "global_load_lds_dwordx4 %2, off offset:1024\n\t"
        "global_load_lds_ubyte %3, off offset:2048\n\t"
        "global_load_lds_ubyte %4, off offset:2304" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "v"(k), "v"(v), "v"(ks), "v"(vs)
        : "memory", "m0");
}
// The same from scalar bases and offsets of 32 bits
__device__ __forceinline__ void dma_fp4(unsigned lds, uint64_t k, uint64_t v, uint64_t ks, uint64_t vs, unsigned kin, unsigned vin, unsigned ksin,
                                        unsigned vsin) {
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 3\n\t"
        "global_load_lds_dwordx4 %5, %1\n\t"
        "global_load_lds_dwordx4 %6, %2 offset:1024\n\t"
        "global_load_lds_ubyte %7, %3 offset:2048\n\t"
        "global_load_lds_ubyte %8, %4 offset:2304" ::"s"(__builtin_amdgcn_readfirstlane(lds)), "s"(k), "s"(v), "s"(ks), "s"(vs), "v"(kin),
        "v"(vin), "v"(ksin), "v"(vsin)
        : "memory", "m0");
}
// the dword at an LDS address
__device__ __forceinline__ uint32_t word_read(unsigned a) {
    return *(const __attribute__((address_space(3))) uint32_t*)(size_t)a;
}

// CAP: soft cap
template <int DT, int CT, int HD, int RB_, bool CAP>
__global__ void __launch_bounds__(NT, 1) fa_quant_prefill_kernel(QuantFwdArgs a) {
    using C = Cfg<HD, RB_>;
    constexpr int RB = C::RB, BM = C::BM, BN = C::BN, NB = C::NB, TPG = C::TPG, NH = C::NH, KS = C::KS, DB = C::DB, DCH = C::DCH, ROW = C::ROW,
                  KT = C::KT, TILE = C::TILE, NE = 16 * RB;
    using O = Operands<DT, CT>;
    constexpr bool FOUR = O::FOUR;
    constexpr int OT = O::OT;
    constexpr float kUnit = O::kUnit;
    // slots: S products, then the P.V products of the first and the last 16 keys
    constexpr int SS = KS * RB, SP = DB * RB;
    __shared__ __attribute__((aligned(256))) char s_t[NBUF * TILE];
    __shared__ __attribute__((aligned(256))) char s_raw[2 * NW * O::RAW];  // codes of two tiles, each thread's own
    __shared__ int s_pref[kQuantMaxB + 1];
    __shared__ int64_t s_line[kQuantMaxB + 1];
    __shared__ float s_m[RB][NT];  // each thread's m of its rows (fa_quant.h), used where V's scales are not plain

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hi = lane >> 5;
    if constexpr (FOUR) {
        if (a.blocks && blocks_take<NT>(a, s_line)) {  // the decode kernel has them all
            if (a.cut && tid == 0) reinterpret_cast<CutItem*>(a.pf_cut)[blockIdx.x] = CutItem{0, 0, 0, 0};
            return;
        }
    }
    build_list<BM, BN, NW>(a, s_pref, s_line);

    const unsigned lds0 = lds_addr(s_t);
    const unsigned rowa = lds0 + col * ROW + (slot_of<ROW>(col, hi) << 4);  // chunk 2s + hi: ^ (s << 5)
    const int tr_r = 4 * hi + ((lane & 15) >> 2), tr_c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    const unsigned tra = lds0 + KT + (lane & 1) * 8 + tr_r * ROW + (slot_of<ROW>(tr_r, tr_c) << 4);  // dim block db: ^ (db << 6)
    // This thread's part of a tile: of K and of V the 16 codes of chunk dch of rows kk
    // and kk + NT / DCH. A wave's rows of either lie in one block of 16 keys.
    // Of a 4-bit tile: the group dch of row kk, which is 32 codes and their scale.
    const int kk = FOUR ? tid / (HD / 32) : tid / DCH, dch = FOUR ? tid % (HD / 32) : tid % DCH;
    const bool in = dch * (FOUR ? 32 : 16) < a.hd, full = a.hd == HD;
    const uint32_t kin = (uint32_t)(kk & 15) * (uint32_t)a.k_si + (in ? dch * 16 : 0);
    const uint32_t vin = (uint32_t)(kk & 15) * (uint32_t)a.v_si + (in ? dch * 16 : 0);
    [[maybe_unused]] const uint32_t ksin = FOUR ? (uint32_t)(kk & 15) * (uint32_t)a.ks_sb + (in ? dch : 0) : 0;
    [[maybe_unused]] const uint32_t vsin = FOUR ? (uint32_t)(kk & 15) * (uint32_t)a.vs_sb + (in ? dch : 0) : 0;
    // of a 4-bit tile: chunk 4 dch; chunks 4 dch + 2, and one more, differ in bits 5 and 4
    const unsigned put0 = lds0 + kk * ROW + (slot_of<ROW>(kk, (FOUR ? 4 : 2) * dch) << 4), put1 = lds0 + kk * ROW + (slot_of<ROW>(kk, (FOUR ? 4 : 2) * dch + 1) << 4);
    const unsigned raw = __builtin_amdgcn_readfirstlane(lds_addr(s_raw)) + wave * O::RAW;
    auto block_of = [&](int u) { return (u * (NT / DCH) + wave * (64 / DCH)) >> 4; };
    auto anew = []() -> const QuantFwdArgs& {  // as in fa_quant_decode.hip
        auto p = __builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(p));
        return *(const QuantFwdArgs*)p;
    };

    [[maybe_unused]] const float cap = a.softcap * kLog2e;
    const int entries = s_pref[a.B], grid = (int)gridDim.x;
    Line line{};
    int worker = blockIdx.x;
    int64_t at = 0, end;  // places on the line, or numbers of whole items
    if (a.cut) {
        line = make_line(s_line[min(entries, kQuantMaxB)], a.Hk, grid);
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
            e = find_in(s_line, min(entries, kQuantMaxB), at - hk * line.len);
        } else {
            // items are numbered heaviest first within a sequence; odd passes run the other way
            const int64_t w = at * grid + ((at & 1) ? grid - 1 - (int)blockIdx.x : (int)blockIdx.x);
            ++at;
            if (w >= entries * (int64_t)a.Hk) continue;
            hk = (int)(w % a.Hk);
            e = (int)(w / a.Hk);
        }
        hk = __builtin_amdgcn_readfirstlane(hk);
        e = __builtin_amdgcn_readfirstlane(e);
        const int b = __builtin_amdgcn_readfirstlane(find_in(s_pref, a.B, e));
        const Rows R = rows_of<BM>(a, b);
        const int mt = __builtin_amdgcn_readfirstlane(a.cut ? e - s_pref[b] : s_pref[b + 1] - 1 - e);
        const int diag0 = R.q.sk - R.q.sq;
        const int row0 = mt * BM, item_rows = min(BM, R.rows - row0);
        const Keys K = keys_of(a, R.q, row0, item_rows);
        int k_lo = K.lo, k_hi = K.hi;
        if (a.cut) {
            const int64_t p0 = hk * line.len + s_line[e], p1 = hk * line.len + s_line[e + 1], upto = min(end, p1);
            if (at > p0) t_lo = tile_at(at - p0, NH);
            if (upto < p1) t_hi = tile_at(upto - p0, NH);
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
        k_lo = __builtin_amdgcn_readfirstlane(k_lo);
        k_hi = __builtin_amdgcn_readfirstlane(k_hi);
        slot = __builtin_amdgcn_readfirstlane(slot);
        const int base = k_lo & ~15;  // tiles start at a block of 16 keys
        const int ntiles = (k_hi - base + BN - 1) / BN;
        // tiles all of whose keys are visible to all rows: [t1, t2)
        const int i_lo = row0 / g, i_hi = (row0 + item_rows - 1) / g;
        const int f_lo = max(k_lo, key_lo(i_hi + diag0, a.wl, 0)), f_hi = min(k_hi, key_hi(i_lo + diag0, a.wr, 0) + 1);
        const int t1 = min(ntiles, (f_lo - base + BN - 1) / BN), t2 = max(t1, (f_hi - base) / BN);

        // ---- tiles: registers -> widened -> LDS ---------------------------------------------
        // The lanes of every wave look after a group of 64 blocks of 16 keys: where their
        // rows are and their scales. Page ids are read a group ahead.
        const int* trow = a.table ? a.table + (int64_t)R.q.crow * a.t_stride : nullptr;
        constexpr int kNoKeys = -0x7fffffff - 1;  // page of a block past the item's keys
        struct Scales {
            float k, v;
            uint64_t ok;        // blocks whose page is in the cache
        };
        Scales sc, sc_new;      // of the group at hand, and of the next once asked for
        sc_new = Scales{1.f, 1.f, 0};
        float lv = 0.f, iv_ = 1.f;     // log2 and inverse of sc.v, which for 0 is 0 and for no number itself
        uint64_t hard = 0, wild = 0;   // blocks that are not in the cache or whose scales are not plain; whose V scales are not
        int64_t ko = 0, vo = 0;  // where the blocks of the group asked for are
        [[maybe_unused]] int64_t kso = 0, vso = 0;  // and their scales of 4-bit codes
        uint64_t have = 0;       // its sc.ok
        int id_page, id_row;
        auto group_ids = [&](int gr) {
            const QuantFwdArgs& A = anew();
            const int64_t j = base + ((int64_t)gr * 64 + lane) * 16;
            id_page = kNoKeys;
            id_row = 0;
            if (j < k_hi) {
                const int pi = trow ? (int)udiv(A.page, (uint32_t)j) : 0;
                id_row = (int)j - pi * A.page_size;
                id_page = trow ? trow[pi] : R.q.crow;
            }
        };
        auto group_places = [&](Scales& s) {
            const QuantFwdArgs& A = anew();
            const bool ok = id_page >= 0 && id_page < A.num_pages;
            const int64_t p = ok ? id_page : 0, r = ok ? id_row : 0;
            // less what load u (K) and 2 + u (V) of the block add
            const int u = FOUR ? 0 : lane % NB / (NB / 2);
            ko = (int64_t)(A.k + ((int64_t)hk * A.k_sh + p * A.k_sp + r * A.k_si)) - 1024 * u;
            vo = (int64_t)(A.v + ((int64_t)hk * A.v_sh + p * A.v_sp + r * A.v_si)) - 1024 * (FOUR ? 1 : 2 + u);
            s.k = s.v = 1.f;
            if constexpr (FOUR) {
                kso = (int64_t)(reinterpret_cast<const uint8_t*>(A.ks) + ((int64_t)hk * A.ks_sh + p * A.ks_sp + r * A.ks_sb)) - 2048;
                vso = (int64_t)(reinterpret_cast<const uint8_t*>(A.vs) + ((int64_t)hk * A.vs_sh + p * A.vs_sp + r * A.vs_sb)) - 2304;
            } else if (ok) {
                const int64_t sb = udiv(A.sblk, (uint32_t)r);
                s.k = A.ks[p * A.ks_sp + sb * A.ks_sb + (int64_t)hk * A.ks_sh];
                s.v = A.vs[p * A.vs_sp + sb * A.vs_sb + (int64_t)hk * A.vs_sh];
            }
            have = s.ok = __ballot(ok);
        };
        auto wild_of = [&](const Scales& s) { return FOUR ? 0 : __ballot(!plain_scale(s.v)); };
        auto hard_of = [&](const Scales& s) {
            if constexpr (FOUR) return ~s.ok | __ballot(!(anew().scale > 0.f));
            return ~s.ok | __ballot(!(anew().scale > 0.f && s.k > 0.f && s.k < INFINITY && plain_scale(s.v)));
        };
        auto begin_group = [&]() {
            if constexpr (FOUR) {
                hard = hard_of(sc);
                return;
            }
            lv = scale_log2(sc.v);
            iv_ = copysignf(fminf(fast_exp2(-lv), 0x1p127f), sc.v);
            iv_ = lv == -INFINITY ? sc.v : iv_;
            hard = hard_of(sc);
            wild = wild_of(sc);
        };
        // Rows outside the item, blocks of pages outside the cache and columns past the
        // head dim are read where there is memory, and put down as 0.
        constexpr uint64_t kTileBlocks = ((uint64_t)1 << NB) - 1;
        bool part_a = false, part_b = false;  // the two tiles asked for: whether they have such
        uint64_t have_a = 0, have_b = 0;
        auto ask = [&](int t, int tg) {  // tg: the tile's number in its group
            auto from = [&](int64_t o, int u) {
                const int bl = tg * NB + (FOUR ? wave * (64 / (HD / 32)) / 16 + u : block_of(u));
                return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(o >> 32), bl) << 32 |
                       (uint32_t)__builtin_amdgcn_readlane((int)o, bl);
            };
            part_a = part_b;
            have_a = have_b;
            have_b = have >> (tg * NB);
            part_b = base + t * BN < k_lo || base + (t + 1) * BN > k_hi || !full || (have_b & kTileBlocks) != kTileBlocks;
            if constexpr (FOUR && HD > 64) {
                dma_fp4(raw + (t & 1) * (NW * O::RAW), from(ko, 0), from(vo, 0), from(kso, 0), from(vso, 0), kin, vin, ksin, vsin);
            } else if constexpr (FOUR) {
                // at head dim 64 a wave's rows lie in two blocks
                auto mine = [&](int64_t o) { return lane >= 32 ? from(o, 1) : from(o, 0); };
                dma_fp4(raw + (t & 1) * (NW * O::RAW), mine(ko) + kin, mine(vo) + vin, mine(kso) + ksin, mine(vso) + vsin);
            } else {
                dma16_kkvv(raw + (t & 1) * (NW * O::RAW), from(ko, 0), from(ko, 1), from(vo, 0), from(vo, 1), kin, vin);
            }
        };
        u32x4 got[2];
        [[maybe_unused]] uint32_t got_scale;
        auto get_part = [&](int t, int part) {  // part 0 .. 3: K of u = 0, 1, then V
            if constexpr (FOUR) {
                if (part & 1) return;  // the second half of the codes that part - 1 got
                const unsigned at = raw + (t & 1) * (NW * O::RAW);
                got[0] = row_read(at + (part >> 1) * 1024 + lane * 16);
                got_scale = word_read(at + 2048 + (part >> 1) * 256 + lane * 4);
                return;
            }
            got[part & 1] = row_read(raw + (t & 1) * (NW * O::RAW) + part * 1024 + lane * 16);
        };
        auto put_part = [&](int t, int part, unsigned tile) {
            if constexpr (FOUR) {
                uint32_t w0 = got[0][2 * (part & 1)], w1 = got[0][2 * (part & 1) + 1], s = got_scale;
                if (part_a) {
                    const int j = base + t * BN + kk;
                    if (!(in && j >= k_lo && j < k_hi && (have_a >> (kk >> 4) & 1))) w0 = w1 = s = 0;
                }
                const unsigned at = put0 ^ (part & 1) << 5, to = tile + (part >> 1) * KT;
                row_write(at + to, fp4_widen8<DT>(w0, fp4_scale(s)));
                row_write((at ^ 16) + to, fp4_widen8<DT>(w1, fp4_scale(s)));
                return;
            }
            u32x4 x = got[part & 1];
            const int u = part & 1;
            if (part_a) {
                const int j = base + t * BN + u * (NT / DCH) + kk;
                if (!(in && j >= k_lo && j < k_hi && (have_a >> block_of(u) & 1))) x = u32x4{0u, 0u, 0u, 0u};
            }
            const unsigned to = tile + u * (NT / DCH) * ROW + (part >> 1) * KT;
            const u32x2 c0 = widen4<CT>(x[0]), c1 = widen4<CT>(x[1]), c2 = widen4<CT>(x[2]), c3 = widen4<CT>(x[3]);
            row_write(put0 + to, u32x4{c0[0], c0[1], c1[0], c1[1]});
            row_write(put1 + to, u32x4{c2[0], c2[1], c3[0], c3[1]});
        };
        // the loads of an item's start in the order in which they are waited for
        group_ids(0);
        // ---- q as B operands: lane holds row col, chunks 2s + hi -------------------------------
        const int wrow0 = row0 + wave * RB * 32;
        u32x4 qreg[RB][KS];
        int rlo[RB];       // the row's visible keys: the first, as offset from the item's first tile, and
        unsigned rsee[RB]; // their number
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = wrow0 + rb * 32 + col;
            const bool ok = r < R.rows;
            const int i = ok ? r / g : 0, h = hk * g + (ok ? r % g : 0);
            const int first = max(k_lo, key_lo(i + diag0, a.wl, 0));
            rlo[rb] = first - base - 4 * hi;
            rsee[rb] = (unsigned)max(min(k_hi - 1, key_hi(i + diag0, a.wr, 0)) + 1 - first, 0);
            const int64_t qat = q_row(a, b, i, a.q_sb, a.q_si) + (int64_t)h * a.q_sh;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const int d = (2 * s + hi) * 8;
                qreg[rb][s] = ok && d < a.hd ? *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + qat + d)
                                             : u32x4{0u, 0u, 0u, 0u};
            }
        }
        if (ntiles > 0) {
            group_places(sc);
            group_ids(1);
            ask(0, 0);
            ask(1, 1);
        }
        float qs[RB];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float most = 0.f;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const f32x8 x = widen8<DT>(qreg[rb][s]);
#pragma unroll
                for (int e2 = 0; e2 < 8; ++e2) most = fmaxf(most, fabsf(x[e2]));
            }
            const int sh = FOUR ? 0 : q_shift(fmaxf(most, __shfl_xor(most, 32)));
            const float up = exp2i(sh);
            qs[rb] = exp2i(-sh) * a.scale * (CAP ? 1.f / a.softcap : kLog2e);
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                if constexpr (!FOUR) qreg[rb][s] = pack8<DT_FP16>(widen8<DT>(qreg[rb][s]) * up);
                asm volatile("" : "+a"(qreg[rb][s]));  // one tuple per operand, in accumulation registers
            }
        }

        if (ntiles > 0) {
            wait_loads<0>();
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    get_part(t, x);
                    put_part(t, x, t * TILE);
                }
                ask(t + 2, t + 2);
            }
        }

        f32x16 o[RB][DB];
        float u[RB], l[RB];  // references (fa_quant.h; less kUnit) and sums of the rows
        bool apart = false;  // l is relative to m, else to u
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            u[rb] = -1e30f;  // finite floor: exp2(x - u) never forms inf - inf
            l[rb] = 0.f;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[rb][db][i] = 0.f;
        }

        // LDS addresses of this lane's operands in the tile read next, moved on
        // with the tile; opaque, so that the rest goes into the instructions' offsets
        unsigned ra[KS], ta[DB], tb[DB];
#pragma unroll
        for (int s = 0; s < KS; ++s) ra[s] = rowa ^ (s << 5);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            ta[db] = tra ^ (db << 6);
            tb[db] = (tra ^ (db << 6) ^ 32) + 8 * ROW;
        }
        auto move_on = [&](unsigned& x, unsigned by) {
            x += by;
            asm volatile("" : "+v"(x));
        };
        u32x4 kop[KS], vop[2 * DB];
        auto read_rows = [&](int h, int s) {  // operands s and s + 1
            kop[s] = row_read(ra[s] + h * 32 * ROW);
            kop[s + 1] = row_read(ra[s + 1] + h * 32 * ROW);
        };
        auto read_tr = [&](int h, int x) {  // x, x + 1: step of 16 keys, then dim block
#pragma unroll
            for (int i = x; i < x + 2; ++i) {
                const int o_ = (h * 32 + i / DB * 16) * ROW;
                vop[i] = tr_read(ta[i % DB] + o_, tb[i % DB] + o_);
            }
        };
        auto lane_of = [](float x, int i) {
            return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), i));
        };

        // Scores of the unit at hand are raw products times cc, or scores themselves (cc =
        // 1); peak: the largest of them with log2 of V's scale added, peakx: of the scores alone.
        float cc[RB][2], peak[RB], peakx[RB];
        auto scored = [&](f32x16 (&n)[RB], int el, int s0, float c, unsigned ok) {  // s0: key offset of the unit
            const int rb = el / 16, i = el % 16;
            float y = n[rb][i] * c;
            if constexpr (CAP) y = cap * fast_tanh(y);
            const unsigned seen = ok >> (i / 8) & 1 ? rsee[rb] : 0;
            n[rb][i] = (unsigned)(s0 - rlo[rb] + 8 * (i / 4) + i % 4) < seen ? y : -INFINITY;
        };
        // moves the running maxima to those of the scores where they exceed them by 2^4
        auto raise = [&](bool live, auto kind) {
            constexpr bool TWO = decltype(kind)::value == WILD;
            bool need = false;
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                need |= peak[rb] > u[rb] + (kUnit + kLazy);
                if constexpr (TWO) need |= peakx[rb] > s_m[rb][tid] + kLazy;
            }
            if (live && __ballot(need)) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    const float un = fmaxf(u[rb], fmaxf(peak[rb], __shfl_xor(peak[rb], 32)) - kUnit);
                    const float alpha = fast_exp2(u[rb] - un);
                    u[rb] = un;
                    if constexpr (TWO) {
                        const float m = s_m[rb][tid], mn = fmaxf(m, fmaxf(peakx[rb], __shfl_xor(peakx[rb], 32)));
                        l[rb] *= fast_exp2(m - mn);
                        s_m[rb][tid] = mn;
                    } else {
                        l[rb] *= alpha;
                    }
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[rb][db][i] *= alpha;
                    }
                }
            }
        };
        const f32x16 zero = {};

        // One unit: its softmax and P.V while the scores of the next are formed (n_), one
        // MFMA to a slot. Each score takes three slots: scaled, its exponential,
        // summed and packed; they are spread evenly up to the last keys' P.V products.
        // H: the unit at hand in its tile; its successor's K is read from place A of a tile.
        u32x4 pk[RB][2];
        float px[NE], lk[2];  // lk: log2 of V's scales of the unit at hand
        auto unit = [&](f32x16 (&c_)[RB], f32x16 (&n_)[RB], auto hh, int tg, int s0n, auto kind, auto more, auto ahead) {
            constexpr int H = decltype(hh)::value, A = (H + 1) % NH, KIND = decltype(kind)::value;
            constexpr bool RAW = KIND == FAST && !CAP, TWO = KIND == WILD;
            float dd[RB][2], nn[RB][2], iv[2], ln[2];
            [[maybe_unused]] float sg[2], no[2], m[RB], pw[NE];  // TWO: V's sign, its scale where that is no number, m, weights
            const int bl = tg * NB + 2 * H;  // the unit's blocks; the next unit's follow
            [[maybe_unused]] const unsigned ok = (unsigned)(sc.ok >> ((bl + 2) & 63));
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const float ks = FOUR ? 1.f : lane_of(sc.k, (bl + 2 + kb) & 63);
                ln[kb] = FOUR ? 0.f : lane_of(lv, (bl + 2 + kb) & 63);
                iv[kb] = TWO || FOUR ? 1.f : lane_of(iv_, bl + kb);
                if constexpr (TWO) {
                    const float t = lane_of(iv_, bl + kb);
                    sg[kb] = copysignf(1.f, t);
                    no[kb] = fabsf(t) < INFINITY ? 0.f : t;
                }
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    dd[rb][kb] = lk[kb] - u[rb];
                    nn[rb][kb] = qs[rb] * ks;
                }
            }
            if constexpr (TWO) {
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) m[rb] = s_m[rb][tid];
            }
            float part[RB], top[RB][2];
            int slot = 0;
            auto next = [&]() {
#pragma unroll
                for (int q = 0; q < NE; ++q) {
                    // q-th score: the first 16 keys of every row block, then the others
                    const int ks = q / (8 * RB), rb = q / 8 % RB, i = 8 * ks + q % 8;
                    const int when = q * (SS + SP - 2) / NE;
                    if (slot == when) {
                        if constexpr (TWO) {
                            pw[q] = __builtin_fmaf(c_[rb][i], cc[rb][ks], dd[rb][ks]);
                            px[q] = __builtin_fmaf(c_[rb][i], cc[rb][ks], -m[rb]);
                        } else {
                            px[q] = __builtin_fmaf(c_[rb][i], cc[rb][ks], dd[rb][ks]);
                        }
                    }
                    if (slot == when + 1) {
                        px[q] = fast_exp2(px[q]);
                        if constexpr (TWO) pw[q] = fast_exp2(pw[q]);
                    }
                    if (slot == when + 2) {
                        part[rb] = q % 8 == 0 ? px[q] : part[rb] + px[q];
                        if (q % 8 == 7) l[rb] = TWO ? l[rb] + part[rb] : __builtin_fmaf(part[rb], iv[ks], l[rb]);
                        if constexpr (TWO) px[q] = __builtin_fmaf(pw[q], sg[ks], mul_or_0(px[q], no[ks]));
                        if (q & 1) pk[rb][ks][q / 2 % 4] = pack2<OT>(px[q - 1], px[q]);
                    }
                }
#pragma unroll
                for (int e = 0; e < NE; ++e) {
                    if (slot != SS + 2 + e * (2 * SP - 4) / NE) continue;
                    const int rb = e / 16, kb = e / 8 % 2;
                    if constexpr (KIND != FAST) {
                        scored(n_, e, s0n, nn[rb][kb], ok);
                    } else if constexpr (CAP) {
                        n_[rb][e % 16] = cap * fast_tanh(n_[rb][e % 16] * nn[rb][kb]);
                    }
                    top[rb][kb] = e % 8 == 0 ? n_[rb][e % 16] : fmaxf(top[rb][kb], n_[rb][e % 16]);
                }
                ++slot;
                fence();
            };
            // operands are read two steps ahead, the last one read is used first
#pragma unroll
            for (int s = 0; s < KS; s += 2) {
#pragma unroll
                for (int d = 1; d >= 0; --d) {
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        n_[rb] = mfma32<OT>(kop[s + d], qreg[rb][s + d], s == 0 && d == 1 ? zero : n_[rb]);
                        if (d == 1 && rb == 0) {
                            if (s + 2 < KS) read_rows(A, s + 2);
                            else read_tr(H, 0);
                        }
                        next();
                    }
                }
            }
#pragma unroll
            for (int x = 0; x < 2 * DB; x += 2) {
#pragma unroll
                for (int d = 1; d >= 0; --d) {
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        o[rb][(x + d) % DB] = mfma32<OT>(vop[x + d], pk[rb][(x + d) / DB], o[rb][(x + d) % DB]);
                        if (d == 1 && rb == 0) {
                            if (x + 2 < 2 * DB) read_tr(H, x + 2);
                            else ahead();
                        }
                        more(x * RB + (1 - d) * RB + rb);
                        next();
                    }
                }
            }
            more(2 * SP);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                if constexpr (RAW) peak[rb] = fmaxf(__builtin_fmaf(top[rb][0], nn[rb][0], ln[0]), __builtin_fmaf(top[rb][1], nn[rb][1], ln[1]));
                else peak[rb] = fmaxf(top[rb][0] + ln[0], top[rb][1] + ln[1]);
                if constexpr (TWO) peakx[rb] = fmaxf(top[rb][0], top[rb][1]);
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) cc[rb][kb] = RAW ? nn[rb][kb] : 1.f;
            }
            lk[0] = ln[0];
            lk[1] = ln[1];
        };

        if (ntiles > 0) {
            begin_group();
            __syncthreads();
            f32x16 s0[RB], s1[RB];
#pragma unroll
            for (int s = 0; s < KS; s += 2) read_rows(0, s);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                s0[rb] = zero;
#pragma unroll
                for (int s = 0; s < KS; ++s) s0[rb] = mfma32<OT>(kop[s], qreg[rb][s], s0[rb]);
            }
            lk[0] = lane_of(lv, 0);
            lk[1] = lane_of(lv, 1);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {  // (the sums are 0)
                float top[2];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    scored(s0, rb * 16 + i, 0, qs[rb] * lane_of(sc.k, i / 8), (unsigned)sc.ok);
                    top[i / 8] = i % 8 == 0 ? s0[rb][i] : fmaxf(top[i / 8], s0[rb][i]);
                }
                const float mx = fmaxf(top[0], top[1]), ux = fmaxf(top[0] + lk[0], top[1] + lk[1]);
                u[rb] = fmaxf(u[rb], fmaxf(ux, __shfl_xor(ux, 32)) - kUnit);
                s_m[rb][tid] = fmaxf(-1e30f, fmaxf(mx, __shfl_xor(mx, 32)));
                cc[rb][0] = cc[rb][1] = 1.f;
            }
            if constexpr (NH == 1) {
#pragma unroll
                for (int s = 0; s < KS; ++s) move_on(ra[s], TILE);
            }
            read_rows(NH > 1 ? 1 : 0, 0);
            int t = 0, tg = 0, nb = 1, fb = 2;  // buffers of tiles t + 1 and t + 2
            auto next_buf = [](int x) { return x == NBUF - 1 ? 0 : x + 1; };
            auto step_to = [](int x) { return x == 0 ? 0u - (NBUF - 1) * (unsigned)TILE : (unsigned)TILE; };
            constexpr int LAST = (2 * DB - 2) * RB;  // first product of the last operand pair: `ahead` runs there
            // Tile t + 2 goes down, in four parts, in tile t's last unit, past its barrier
            // (a tile of one unit: before it); then tile t + 4 is asked for in its place.
            auto stage = [&](int x) {
#pragma unroll
                for (int part = 0; part < 4; ++part) {
                    if (x == part * 2 * SP / 4) {
                        if (part == 0) wait_loads<4>();  // all but tile t + 3's
                        get_part(t, part);
                    }
                    if (x == part * 2 * SP / 4 + 1) put_part(t + 2, part, fb * TILE);
                }
                if (x == 2 * SP) {
                    const int ag = (tg + 4) % TPG;
                    if (ag == 0) {
                        group_places(sc_new);
                        group_ids((t + 4) / TPG + 1);
                    }
                    ask(t + 4, ag);
                }
            };
            auto tile = [&](auto kind) {
                const unsigned by = step_to(nb);  // from tile t's buffer to the next
                const int s0k = t * BN;
                if constexpr (NH > 1) {
                    auto half = [&](auto hh) {
                        constexpr int H = decltype(hh)::value;
                        unit(H % 2 ? s1 : s0, H % 2 ? s0 : s1, hh, tg, s0k + 32 * (H + 1), kind,
                             [&](int x) {
                                 if (H == NH - 2 && x == SP / 2) {
#pragma unroll
                                     for (int s = 0; s < KS; ++s) move_on(ra[s], by);
                                 }
                                 if (H == NH - 2 && x == LAST - 1) __syncthreads();
                                 if (H == NH - 1) stage(x);
                                 if (H == NH - 1 && x == LAST) {
#pragma unroll
                                     for (int db = 0; db < DB; ++db) {
                                         move_on(ta[db], by);
                                         move_on(tb[db], by);
                                     }
                                 }
                             },
                             [&]() { read_rows((H + 2) % NH, 0); });
                        if constexpr (H < NH - 1) raise(true, kind);
                    };
                    half(std::integral_constant<int, 0>{});
                    half(std::integral_constant<int, 1>{});
                    if constexpr (NH == 4) {
                        half(std::integral_constant<int, 2>{});
                        half(std::integral_constant<int, 3>{});
                    }
                } else {
                    const unsigned by2 = step_to(next_buf(nb));  // from tile t + 1's buffer to the next
                    unit(s0, s1, std::integral_constant<int, 0>{}, tg, s0k + 32, kind,
                         [&](int x) {
                             if (x == SP / 2) {
#pragma unroll
                                 for (int s = 0; s < KS; ++s) move_on(ra[s], by2);
                             }
                             stage(x);
                             if (x == LAST - 1) __syncthreads();
                             if (x == LAST) {
#pragma unroll
                                 for (int db = 0; db < DB; ++db) {
                                     move_on(ta[db], by);
                                     move_on(tb[db], by);
                                 }
                             }
                         },
                         [&]() { read_rows(0, 0); });
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) s0[rb] = s1[rb];
                }
                nb = next_buf(nb);
                fb = next_buf(fb);
                ++t;
                if (++tg == TPG) {
                    tg = 0;
                    sc = sc_new;
                    begin_group();
                } else if (tg + 1 == TPG) {
                    // the next tile's scores take scales of the next group: they go where those of
                    // this group's first tile were
                    if constexpr (!FOUR) {
                        sc.k = lane < NB ? sc_new.k : sc.k;
                        lv = lane < NB ? scale_log2(sc_new.v) : lv;
                    }
                    sc.ok = (sc.ok & ~kTileBlocks) | (sc_new.ok & kTileBlocks);
                    hard = (hard & ~kTileBlocks) | (hard_of(sc_new) & kTileBlocks);
                    wild = (wild & ~kTileBlocks) | (wild_of(sc_new) & kTileBlocks);
                }
                raise(t < ntiles, kind);
            };
            // a tile's copy of the unit covers the weights of it and the scores formed in
            // it: those of its later units and of the next tile's first
            auto among = [&](uint64_t x) { return ((x >> (tg * NB) | x >> ((tg + 1) % TPG * NB)) & kTileBlocks) != 0; };
            auto odd = [&]() { return t < t1 || t + 1 >= t2 || among(hard); };
            apart = !FOUR && among(wild);
            while (t < ntiles) {
                while (!FOUR && t < ntiles && (apart || among(wild))) {
                    if (!apart) {
                        apart = true;
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) s_m[rb][tid] = u[rb];
                    }
                    if constexpr (!FOUR) tile(std::integral_constant<int, WILD>{});
                    if (among(wild)) continue;
                    // one reference again where the two are close
                    bool far = false;
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) far |= !(fabsf(s_m[rb][tid] - u[rb]) <= 60.f);
                    if (__ballot(far) == 0) {
                        apart = false;
#pragma unroll
                        for (int rb = 0; rb < RB; ++rb) l[rb] *= fast_exp2(s_m[rb][tid] - u[rb]);
                    }
                }
                while (t < ntiles && odd() && !among(wild)) tile(std::integral_constant<int, MASKED>{});
                while (t < ntiles && !odd()) tile(std::integral_constant<int, FAST>{});
            }
        }
        wait_loads<0>();  // asked for past the end
        __syncthreads();  // the next item's tiles go where other waves may still read

        // ---- results: lane holds O^T [dims 32db + 8q + 4hi + i][row col] --------------------------
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = wrow0 + rb * 32 + col;
            const float lrow = l[rb] + __shfl_xor(l[rb], 32);
            const bool some = lrow != 0.f;
            // 2^(u - m) may be out of range where the quotient is not: half of it on either side
            float m = u[rb], up = 1.f;
            if (apart) {
                m = s_m[rb][tid];
                up = fast_exp2(0.5f * (u[rb] - m));
#pragma unroll
                for (int db = 0; db < DB; ++db) {
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[rb][db][i] *= up;
                }
            }
            const float inv = some ? up / lrow : 0.f;
            const float lse = some ? add_log2(m, lrow) * kLn2 : INFINITY;
            if (r >= R.rows) continue;
            if (slot < 0) {
                const int i = r / g, h = hk * g + r % g;
                uint16_t* orow = static_cast<uint16_t*>(a.out) + q_row(a, b, i, a.o_sb, a.o_si) + (int64_t)h * a.o_sh;
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int d = 32 * db + 8 * q + 4 * hi;
                        if (d >= a.hd) continue;
                        *reinterpret_cast<u32x2*>(orow + d) =
                            u32x2{pack2<DT>(o[rb][db][4 * q] * inv, o[rb][db][4 * q + 1] * inv),
                                  pack2<DT>(o[rb][db][4 * q + 2] * inv, o[rb][db][4 * q + 3] * inv)};
                    }
                if (hi == 0) a.lse[lse_at(a, b, h, i)] = lse;
            } else {
                const int64_t prow = (int64_t)slot * BM + (r - row0);
#pragma unroll
                for (int db = 0; db < DB; ++db)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        *reinterpret_cast<f32x4*>(a.pf_o + prow * HD + 32 * db + 8 * q + 4 * hi) =
                            f32x4{o[rb][db][4 * q] * inv, o[rb][db][4 * q + 1] * inv, o[rb][db][4 * q + 2] * inv,
                                  o[rb][db][4 * q + 3] * inv};
                if (hi == 0) a.pf_lse[prow] = some ? lse : -INFINITY;
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

}  // namespace

}  // namespace fa
