// fa_fp4_decode.hip -- attention over the 4-bit cache for few query rows (a kv head's g
// query heads x positions, at most 32 packed rows): the cache is streamed once.
//
// Split: as in fa_quant_decode.hip, 64-key tiles of all sequences and kv heads in one
// list, cut into equal ranges, one per wave; what a range leaves of a sequence is merged by a
// second launch.
//
// Four neighbouring lanes load a key's row, 32 channels each at head dim 128, which have one scale, so a
// value is one conversion with its scale (fa_fp4.h). A tile's registers are asked for again as
// soon as they are used, so that one tile is always in flight. Keys change lanes through LDS as codes, since the
// products want a row's quarters 16 lanes apart, and values once they are 16 bits wide, 32 keys at a
// time, since O^T = V^T.P^T wants the keys of a channel side by side: written by rows, read by transpose
// reads. Nothing waits for another wave.
//
// Weights and values meet as fp16, in bf16 calls too, whose 8 bits for a weight would be most of the
// result's error: fp16 holds the values of scales from 2^-23 to 2^13 exactly. Weights are kept in units
// that make a row's largest 2^14, so that one has all its bits down to 2^-28 of that. A bf16 call whose
// values leave that range goes on in bf16, a weight as the sum of two numbers, in units that make the
// largest 2^-20: the sum of 2^20 values of 2^127 stays in fp32. (bf16 weights of one part took the same time, at
// 1.35 times the error.) What decides is the scale bytes of the values that some row sees, so groups of zeros, whose byte is 27 or,
// in a cleared cache, 0, take this path too: with 32 channels of every head dead 64 paged sequences take 107.5 us in place
// of 104.7. Two row tiles at head dims 128 and 256 have it alone: both copies of the products do not fit their registers.
//
// What bounds it: reads, and for short calls the start. 64 paged sequences of 512 to 32768 keys, H64/8
// D128 bf16, 427 MB: 95 us (4.5 TB/s; of 64 x 32768 keys 5.0), and 9 for the merge; the data path of the loads is busy 74 % of
// the time, vector instructions take a third, products 11 %, and waves wait for a third of it. One sequence of 777 keys: 12
// and 4.6 us, of which the list, page ids, first keys and q, one after another, have 8; 4 tokens over a window of
// 4096, 8 sequences, fp16: 21 and 7. Long sequences of D64 3.85, D256 4.4 TB/s,
// of 32 packed rows 3.25 (fp16 3.7), where registers hold fewer loads in flight.
// Lanes that load 16 apart, as the products want them, keep the data path of the loads busy 83 % of the time and
// cost more than the exchange through LDS; loads marked non-temporal made 127 us of 106, as
// a 128-byte line holds two heads' rows.
#include "fa_fp4.h"
#include "fa_quant_list.h"

#include <type_traits>

namespace fa {

namespace {

template <int HD>
struct Cfg4 {
    static constexpr int NWAVE = 4;                  // waves of a workgroup
    static constexpr int KT = 64, NB = KT / 16;      // keys of a tile, blocks of 16
    static constexpr int W = HD / 32;                // words of 8 codes that a lane has of a row
    static constexpr int NL = HD == 256 ? 2 : 1;     // loads of them, each under one scale
    static constexpr int DBLK = HD / 16;
    static constexpr int ROW = 2 * HD;               // bytes of a widened row
    static constexpr int TILES = 64 / NB;            // tiles whose places a wave's lanes hold
    // first channel of word w of quarter G
    static __device__ __forceinline__ int channel(int G, int w) {
        return HD == 64 ? 16 * G + 8 * w : HD == 128 ? 32 * G + 8 * w : 128 * (w >> 2) + 32 * G + 8 * (w & 3);
    }
    // slot of 16-byte chunk c of row r: conflict free for the writes of one chunk of 16 rows and for the
    // transpose reads of two chunks of 8 rows
    static __device__ __forceinline__ int slot(int r, int c) {
        return HD == 64 ? swz_b64(r, c) : c ^ (((r & 7) << 1) | ((r >> 3) & 1));
    }
};

// Workgroups of a compute unit, a wave of each on a SIMD: as many as the registers hold. (Three at
// head dim 128, with a third fewer registers each: 126 us where two took 123.)
__host__ __device__ constexpr int groups_of_cu(int hd, int nr) { return hd == 256 ? 1 : 2; }

// A tile's codes and scales, as a lane loads them
template <int HD>
struct Tile {
    uint32_t k[4][Cfg4<HD>::W], v[4][Cfg4<HD>::W];
    uint32_t ks[4][Cfg4<HD>::NL], vs[4][Cfg4<HD>::NL];
};

template <int N>
__device__ __forceinline__ void load_words(uint32_t* to, const uint8_t* p) {
    if constexpr (N == 4) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(p);
        to[0] = x[0], to[1] = x[1], to[2] = x[2], to[3] = x[3];
    } else {
        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
        to[0] = x[0], to[1] = x[1];
    }
}

template <int N>
__device__ __forceinline__ void words_write(unsigned a, const uint32_t* x) {
    if constexpr (N == 4) row_write(a, u32x4{x[0], x[1], x[2], x[3]});
    else *(__attribute__((address_space(3))) u32x2*)(size_t)a = u32x2{x[0], x[1]};
}
template <int N>
__device__ __forceinline__ void words_read(uint32_t* to, unsigned a) {
    if constexpr (N == 4) {
        const u32x4 x = row_read(a);
        to[0] = x[0], to[1] = x[1], to[2] = x[2], to[3] = x[3];
    } else {
        const u32x2 x = lds_load_u32x2(a);
        to[0] = x[0], to[1] = x[1];
    }
}

// DT: type of q and out; HD: kernel head dim (the cache's may be smaller: lanes past it
// hold the row's first codes and meet zeros of q); NR: 16-row tiles of packed rows; BLK: sequences of
// more rows are there in blocks (fa_quant_list.h).
template <int DT, int HD, int NR, bool BLK>
__global__ void __launch_bounds__(Cfg4<HD>::NWAVE * 64, groups_of_cu(HD, NR)) fa_fp4_decode_kernel(QuantFwdArgs a) {
    using C = Cfg4<HD>;
    constexpr int NWAVE = C::NWAVE, NT = NWAVE * 64, KT = C::KT, NB = C::NB, W = C::W, NL = C::NL, DBLK = C::DBLK, ROW = C::ROW, TILES = C::TILES;
    constexpr float kTop = 14.f, kTopWide = -20.f;  // log2 of the largest weight
    // bf16 calls go by fp16 while they can, but for those whose registers hold the products' code once only
    constexpr bool WIDE = DT == DT_BF16, BOTH = WIDE && (NR == 1 || HD == 64);
    __shared__ __attribute__((aligned(1024))) char s_v[NWAVE][32 * ROW];
    __shared__ int s_pref[kQuantMaxB + 1], s_blk[BLK ? kQuantMaxB + 1 : 1];

    auto anew = []() -> const QuantFwdArgs& {  // as in fa_quant_decode.hip
        auto p = __builtin_amdgcn_kernarg_segment_ptr();
        asm volatile("" : "+s"(p));
        return *(const QuantFwdArgs*)p;
    };
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, G = lane >> 4;   // row (column) and quarter of a product's operand
    const int lr = lane >> 2, lq = lane & 3;   // row and quarter that a lane loads of 16 keys: four lanes a row
    const int hs = heads_per_group(a), hgs = a.Hk / hs;

    // ---- the list of tiles ----------------------------------------------------------
    const int hsel = wave % hs;
    int n = a.B;  // its entries
    if constexpr (BLK) {
        static_assert(NR * 16 == kBlockRows, "");
        __shared__ int64_t s_sum[NWAVE];
        const bool all = blocks_take<NT>(a, s_sum);  // or none
        for (int b = tid; b < a.B; b += NT) s_blk[b + 1] = all ? blocks_of(a, quant_seq(a, b)) : 0;
        __syncthreads();
        if (wave == 0) prefix_sums(s_blk, a.B);
        __syncthreads();
        n = min(s_blk[a.B], a.blocks);  // (a.blocks is enough for prefixes of rows)
        for (int e = tid; e < n; e += NT) {
            Seg s;
            s.b = place_of(s_blk, a.B, e);
            s.q = quant_seq(a, s.b);
            cut_to_block(a, s, e - s_blk[s.b]);
            s_pref[e + 1] = s.q.hi > s.q.lo ? hgs * ((s.q.hi + KT - 1) / KT - s.q.lo / KT) : 0;
        }
        if (blockIdx.x == 0)
            for (int b = tid; b <= a.B; b += NT) a.block_pref[b] = s_blk[b];
    } else {
        __shared__ int64_t s_sum[NWAVE];
        if (a.blocks && blocks_take<NT>(a, s_sum)) {  // nothing is left, nor for the merge
            if (blockIdx.x == 0 && tid == 0) a.sched[a.B] = -1;
            return;
        }
        for (int b = tid; b < a.B; b += NT) {
            const QuantSeq s = quant_seq(a, b);
            s_pref[b + 1] = s.hi > s.lo && s.sq * a.g <= a.dec_rows ? hgs * ((s.hi + KT - 1) / KT - s.lo / KT) : 0;
        }
    }
    __syncthreads();
    if (wave == 0) prefix_sums(s_pref, n);
    __syncthreads();
    if (blockIdx.x == 0)
        for (int b = tid; b <= n; b += NT) a.sched[b] = s_pref[b];
    auto seg_at = [&](const QuantFwdArgs& A, int t) {
        if constexpr (BLK) return block_seg_of(A, s_blk, s_pref, n, t, hs, hsel, KT);
        else return seg_of(A, s_pref, t, hs, hsel, KT);
    };

    const int gw = (wave / hs) * gridDim.x + blockIdx.x;  // wave-major, as in fa_decode.hip
    const int64_t wid = (int64_t)gw * hs + hsel;
    const Split sp = split_list(s_pref[n], gridDim.x * (NWAVE / hs));
    const int t0 = __builtin_amdgcn_readfirstlane(sp.first(gw)), t1 = __builtin_amdgcn_readfirstlane(sp.first(gw + 1));
    if (t0 >= t1) return;  // no barrier follows: the waves go on alone

    // ---- places: lane l looks after block l % 4 of tile l / 4 of 16 tiles ------------------
    // A block without a visible key has the place of a row that is there.
    int id, inp, kvh;
    int64_t koff, voff, ksoff, vsoff;
    uint64_t have = 0;  // the blocks of the 16 tiles whose page is in the cache
    auto ask_ids = [&](int base) {
        const QuantFwdArgs& A = anew();
        const int t = base + lane / NB;
        id = -1;
        inp = kvh = 0;
        if (t < t1) {
            const Seg s = seg_at(A, t);
            const int key = (s.lo_tile + (t - s.S)) * KT + (lane % NB) * 16;
            kvh = s.hk;
            if (key < s.q.hi && key + 16 > s.q.lo) {
                const int pi = A.table ? (int)udiv(A.page, (uint32_t)key) : 0;
                inp = key - pi * A.page_size;
                id = A.table ? A.table[(int64_t)s.q.crow * A.t_stride + pi] : s.q.crow;
            }
        }
    };
    auto places = [&]() {
        const QuantFwdArgs& A = anew();
        const bool ok = id >= 0 && id < A.num_pages;
        const int64_t p = ok ? id : 0, r = ok ? inp : 0, h = kvh;
        koff = p * A.k_sp + r * A.k_si + h * A.k_sh;
        voff = p * A.v_sp + r * A.v_si + h * A.v_sh;
        ksoff = p * A.ks_sp + r * A.ks_sb + h * A.ks_sh;
        vsoff = p * A.vs_sp + r * A.vs_sb + h * A.vs_sh;
        have = __ballot(ok);
    };

    // ---- loads ------------------------------------------------------------------------
    const int groups = a.hd / kGroup;
    uint32_t kin[NL], vin[NL], ksin[NL], vsin[NL];  // where a lane's codes and scales are in a block
    uint32_t mine[NL];  // the bits of codes that are the lane's own
#pragma unroll
    for (int u = 0; u < NL; ++u) {
        const int grp = HD == 64 ? lq >> 1 : 4 * u + lq, at = HD == 64 ? 8 * lq : 64 * u + 16 * lq;
        const bool in = grp < groups;
        mine[u] = in ? ~0u : 0u;
        kin[u] = (uint32_t)lr * (uint32_t)a.k_si + (in ? at : 0);
        vin[u] = (uint32_t)lr * (uint32_t)a.v_si + (in ? at : 0);
        ksin[u] = (uint32_t)lr * (uint32_t)a.ks_sb + (in ? grp : 0);
        vsin[u] = (uint32_t)lr * (uint32_t)a.vs_sb + (in ? grp : 0);
    }
    const uint8_t* ksb = reinterpret_cast<const uint8_t*>(a.ks);
    const uint8_t* vsb = reinterpret_cast<const uint8_t*>(a.vs);
    auto of_lane = [](int64_t x, int l) {
        return (int64_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l) << 32 |
                         (uint32_t)__builtin_amdgcn_readlane((int)x, l));
    };
    // Past the range the last tile is asked for again, so that every wait counts the same loads. The
    // places are those of asked tile's 16 until `places` moves on.
    int asked = t0;
    unsigned bits = 0;  // visible blocks of the tile at hand
    auto ask_k = [&](Tile<HD>& T) {
        const int i = asked - t0;
        if (asked < t1 && i % TILES == 0) {
            places();
            ask_ids(asked + TILES);
        }
        const int at = (min(asked, t1 - 1) - t0) % TILES * NB;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint8_t *p = a.k + of_lane(koff, at + b), *s = ksb + of_lane(ksoff, at + b);
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                load_words<W / NL>(T.k[b] + u * (W / NL), p + kin[u]);
                T.ks[b][u] = s[ksin[u]];
            }
        }
    };
    auto ask_v = [&](Tile<HD>& T) {
        const int at = (min(asked, t1 - 1) - t0) % TILES * NB;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const uint8_t *p = a.v + of_lane(voff, at + b), *s = vsb + of_lane(vsoff, at + b);
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                load_words<W / NL>(T.v[b] + u * (W / NL), p + vin[u]);
                T.vs[b][u] = s[vsin[u]];
            }
        }
        ++asked;
    };
    auto bits_of = [&]() { return (unsigned)(have >> ((min(asked, t1 - 1) - t0) % TILES * NB)) & 15u; };

    // ---- a segment: q, sums ----------------------------------------------------------------
    Seg cs;
    u32x4 qreg[NR][W];
    int qi[NR];
    f32x4 oacc[NR][DBLK];
    float m_run[NR], l_run[NR];
    bool wide = WIDE && !BOTH;  // values out of the range of fp16 have come up
    int rows = 0;
    int flo = 0, fhi = 0;      // keys that every row sees
    const float scale2 = a.softcap > 0.f ? a.scale / a.softcap : a.scale * kLog2e;
    // what scores are multiplied by in the exponent, where that leaves their order
    const float late = a.softcap > 0.f || !(scale2 > 0.f) ? 1.f : scale2;
    auto begin_seg = [&](int t) {
        const QuantFwdArgs& A = anew();
        cs = seg_at(A, t);
        rows = cs.rows;
        wide = WIDE && !BOTH;
        const int diag = cs.q.sk - cs.q.sq;
        flo = key_lo(BLK ? (cs.row0 + rows - 1) / A.g + diag : cs.q.sk - 1, A.wl, 0);
        fhi = min(key_hi(BLK ? cs.row0 / A.g + diag : diag, A.wr, 0), cs.q.sk - 1);
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            const int r = rt * 16 + li;
            const bool ok = r < rows;
            qi[rt] = ok ? (cs.row0 + r) / A.g : 0;
            const int h = cs.hk * A.g + (ok ? (cs.row0 + r) % A.g : 0);
            const uint16_t* q = static_cast<const uint16_t*>(A.q) + q_row(A, cs.b, qi[rt], A.q_sb, A.q_si) + (int64_t)h * A.q_sh;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const int d = C::channel(G, w);
                qreg[rt][w] = ok && d < A.hd ? *reinterpret_cast<const u32x4*>(q + d) : u32x4{0u, 0u, 0u, 0u};
            }
            m_run[rt] = -INFINITY;
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
            const float inv = some ? 1.f / l : 0.f;
            const float lse = some ? (m_run[rt] - (wide ? kTopWide : kTop) + fast_log2(l)) * kLn2 : INFINITY;
            if (r >= rows) continue;
            if (whole) {
                const int h = cs.hk * A.g + (cs.row0 + r) % A.g;
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
    const unsigned vt = lds_addr(s_v[wave]);
    const int tr_row = 4 * G + (li >> 2);
    // Keys' codes use the values' place: 16 rows of KB / 16 bytes, a lane's piece in a slot that sets the rows of
    // eight lanes' reads on different banks
    constexpr int KB = 16 * 4 * (W / NL) * 4, PIECE = 4 * (W / NL);
    const auto piece = [](int r, int q) { return (r * 4 + (q ^ ((HD == 64 ? r >> 3 : r >> 2) & 3))) * PIECE; };
    const unsigned kt_put = vt + piece(lr, lq), kt_get = vt + piece(li, G);
    auto compute = [&](int t, Tile<HD>& T) {
        const int key0 = (cs.lo_tile + (t - cs.S)) * KT;
        const unsigned ok = bits;
        const bool full = ok == 15u && key0 >= flo && key0 + KT - 1 <= fhi;
        // codes past the head dim are 0, since inf x 0 is NaN
        if (groups * kGroup != HD) {
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int w = 0; w < W; ++w) T.k[b][w] &= mine[w * NL / W];
        }
        // Keys to the lanes that want them, the codes by LDS and the scales from lane to lane
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < NL; ++u) words_write<W / NL>(kt_put + (b * NL + u) * KB, T.k[b] + u * (W / NL));
        uint32_t kw[NB][W], ks[NB][NL];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int u = 0; u < NL; ++u) {
                words_read<W / NL>(kw[b] + u * (W / NL), kt_get + (b * NL + u) * KB);
                ks[b][u] = (uint32_t)__builtin_amdgcn_ds_bpermute((4 * li + G) * 4, (int)T.ks[b][u]);
            }
        // S^T = K . Q^T
        f32x4 x[NR][NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) x[rt][b] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < W; ++w) {
                const u32x4 op = fp4_widen8<DT>(kw[b][w], fp4_scale(ks[b][w * NL / W]));
#pragma unroll
                for (int rt = 0; rt < NR; ++rt) x[rt][b] = mfma16x16x32<DT>(op, qreg[rt][w], x[rt][b]);
            }
        }
        ask_k(T);
        bits = bits_of();
        if (a.softcap > 0.f) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt)
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[rt][b][e] = a.softcap * kLog2e * fast_tanh(x[rt][b][e] * scale2);
        } else if (!(scale2 > 0.f)) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt)
#pragma unroll
                for (int b = 0; b < NB; ++b) x[rt][b] *= scale2;
        }
        if (!full) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) {
                const int d = qi[rt] + cs.q.sk - cs.q.sq;
                const int rlo = key_lo(d, a.wl, 0), rhi = min(key_hi(d, a.wr, 0), cs.q.sk - 1);
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = key0 + b * 16 + G * 4 + e;
                        x[rt][b][e] = (ok >> b & 1) && j >= rlo && j <= rhi ? x[rt][b][e] : -INFINITY;
                    }
            }
        }
        // values that no row sees must not meet the products, where 0 x NaN is NaN
        if (!full) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int j = key0 + 16 * b + lr;
                const bool seen = (ok >> b & 1) && j >= cs.q.lo && j < cs.q.hi;
#pragma unroll
                for (int w = 0; w < W; ++w) T.v[b][w] = seen ? T.v[b][w] : 0u;
#pragma unroll
                for (int u = 0; u < NL; ++u) T.vs[b][u] = seen ? T.vs[b][u] : 127u;
            }
        }
        if constexpr (BOTH) {
            uint32_t out = 0;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int u = 0; u < NL; ++u) out = max(out, T.vs[b][u] - 104u);
            if (!wide && __ballot(out > 140u - 104u)) {
                wide = true;
#pragma unroll
                for (int rt = 0; rt < NR; ++rt) {
                    l_run[rt] *= 0x1p-34f;  // 2^(kTopWide - kTop)
#pragma unroll
                    for (int db = 0; db < DBLK; ++db) oacc[rt][db] *= 0x1p-34f;
                }
            }
        }
        // the running maximum
        float up[NR], base[NR];
        bool moved = false;
#pragma unroll
        for (int rt = 0; rt < NR; ++rt) {
            float mx = -INFINITY;
#pragma unroll
            for (int b = 0; b < NB; ++b) mx = fmaxf(mx, fmaxf(fmaxf(x[rt][b][0], x[rt][b][1]), fmaxf(x[rt][b][2], x[rt][b][3])));
            mx = fmaxf(m_run[rt], max4(mx) * late);
            moved |= mx > m_run[rt];
            const float u = mx == -INFINITY ? 0.f : mx;
            up[rt] = fast_exp2(m_run[rt] - u);
            base[rt] = u - (wide ? kTopWide : kTop);
            m_run[rt] = mx;
        }
        if (__ballot(moved)) {
#pragma unroll
            for (int rt = 0; rt < NR; ++rt) {
                l_run[rt] *= up[rt];
#pragma unroll
                for (int db = 0; db < DBLK; ++db) oacc[rt][db] *= up[rt];
            }
        }
        // weights, and O^T += V^T . P^T, 32 keys at a time, on operands of type OT
        auto values = [&](auto tag) {
            constexpr int OT = decltype(tag)::value;
            constexpr bool TWO = OT == DT_BF16;
#pragma unroll
            for (int k2 = 0; k2 < NB / 2; ++k2) {
                u32x4 pk[NR], pl[NR];
#pragma unroll
                for (int rt = 0; rt < NR; ++rt) {
                    f32x8 w;
#pragma unroll
                    for (int e = 0; e < 8; ++e) w[e] = fast_exp2(__builtin_fmaf(x[rt][2 * k2 + (e >> 2)][e & 3], late, -base[rt]));
                    l_run[rt] += ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                    pk[rt] = pack8<OT>(w);
                    if constexpr (TWO) {
                        pl[rt] = pack8<OT>(w - widen8<OT>(pk[rt]));
                        if constexpr (BOTH) fence();  // the rare path is not to take registers of the other
                    }
                }
#pragma unroll
                for (int bb = 0; bb < 2; ++bb) {
                    const int b = 2 * k2 + bb, r = 16 * bb + lr;
#pragma unroll
                    for (int w = 0; w < W; ++w)
                        row_write(vt + r * ROW + (C::slot(lr, C::channel(lq, w) / 8) << 4), fp4_widen8<OT>(T.v[b][w], fp4_scale(T.vs[b][w * NL / W])));
                    if constexpr (TWO && BOTH) fence();
                }
                if (k2 == NB / 2 - 1) ask_v(T);
#pragma unroll
                for (int db = 0; db < DBLK; ++db) {
                    const unsigned p = vt + tr_row * ROW + (C::slot(tr_row, 2 * db + ((li & 3) >> 1)) << 4) + (li & 1) * 8;
                    const u32x4 op = tr_read(p, p + 16 * ROW);
#pragma unroll
                    for (int rt = 0; rt < NR; ++rt) {
                        oacc[rt][db] = mfma16x16x32<OT>(op, pk[rt], oacc[rt][db]);
                        if constexpr (TWO) oacc[rt][db] = mfma16x16x32<OT>(op, pl[rt], oacc[rt][db]);
                    }
                    if constexpr (TWO && BOTH) fence();
                }
            }
        };
        if constexpr (!WIDE) {
            values(std::integral_constant<int, DT_FP16>{});
        } else if constexpr (!BOTH) {
            values(std::integral_constant<int, DT_BF16>{});
        } else {
            if (wide) values(std::integral_constant<int, DT_BF16>{});
            else values(std::integral_constant<int, DT_FP16>{});
        }
    };

    Tile<HD> T;
    ask_ids(t0);
    ask_k(T);
    bits = bits_of();
    ask_v(T);
    int qat = t0, send = t0;
#pragma unroll 1
    for (int t = t0; t < t1; ++t) {
        if (t == qat) {
            begin_seg(t);
            send = min(cs.S + cs.n, t1);
        }
        compute(t, T);
        if (t + 1 == send) {
            end_seg();
            qat = send;
        }
    }
}

template <int DT, int HD>
void launch_n(const QuantFwdArgs& a, int nr, int cus, hipStream_t stream) {
    const dim3 nt(Cfg4<HD>::NWAVE * 64);
    const int grid = cus * groups_of_cu(HD, nr);
    if (a.blocks) {
        hipLaunchKernelGGL((fa_fp4_decode_kernel<DT, HD, 2, true>), dim3(grid), nt, 0, stream, a);
        launch_list_merge<DT, HD, Cfg4<HD>::KT, Cfg4<HD>::NWAVE, 256, true>(a, 2, grid, stream);
        if (a.dec_rows == 0) return;
        nr = 1;  // short sequences of a call whose blocks are not taken
    }
    if (nr == 1) hipLaunchKernelGGL((fa_fp4_decode_kernel<DT, HD, 1, false>), dim3(grid), nt, 0, stream, a);
    else hipLaunchKernelGGL((fa_fp4_decode_kernel<DT, HD, 2, false>), dim3(grid), nt, 0, stream, a);
    // Many segments fill the chip with small workgroups, few want more threads for the pieces of each:
    // 64 sequences of 8 heads of D128 take 9.0 us with 256 threads and 12.8 with 512, 8 sequences 7.2 with 512 and
    // 9.6 with 256. Blocks have few pieces each: 512 tokens of 32 heads 54 us in all with 256, 61 with 512.
    if ((int64_t)a.B * a.Hk * (HD / 32) >= 4 * cus) launch_list_merge<DT, HD, Cfg4<HD>::KT, Cfg4<HD>::NWAVE, 256>(a, nr, grid, stream);
    else launch_list_merge<DT, HD, Cfg4<HD>::KT, Cfg4<HD>::NWAVE>(a, nr, grid, stream);
}

template <int HD>
void launch_d(const QuantFwdArgs& a, int nr, int cus, hipStream_t stream) {
    if (a.bf16) launch_n<DT_BF16, HD>(a, nr, cus, stream);
    else launch_n<DT_FP16, HD>(a, nr, cus, stream);
}

}  // namespace

int fp4_decode_workers(int kd, int nr, int cus) { return cus * groups_of_cu(kd, nr) * Cfg4<128>::NWAVE; }

// kd: kernel head dim; nr: 16-row tiles (1 or 2); cus: compute units
hipError_t launch_fp4_decode(const QuantFwdArgs& a, int, int kd, int nr, int cus, hipStream_t stream) {
    if (kd == 64) launch_d<64>(a, nr, cus, stream);
    else if (kd == 128) launch_d<128>(a, nr, cus, stream);
    else launch_d<256>(a, nr, cus, stream);
    return hipGetLastError();
}

}  // namespace fa
