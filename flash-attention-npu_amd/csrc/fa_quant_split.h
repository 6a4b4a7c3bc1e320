// fa_quant_split.h -- how the attention kernels over 8-bit codes share their work:
// the decode kernel's list of tiles over its workers, and the prefill kernel's line
// of item costs over its workgroups. The kernels and their merges compute them
// apart, so both have to be exact inverses; tests/host/fa_quant_split_check.cpp
// holds them against brute force. Integer code only, host and device.
#pragma once
#include <stdint.h>

#if defined(__HIPCC__) || defined(__HIP__)
#define FA_QSPLIT_FN __host__ __device__ inline
#else
#define FA_QSPLIT_FN inline
#endif

namespace fa {

// Decode. The list holds T tiles, sequence by sequence and head group by head group; the
// first We of W workers share it, T = q We + r: r of them take q + 1 tiles. Workers
// have kMinTiles at least, since a partial costs its merge about what a tile costs here.
constexpr int kMinTiles = 2;
struct Split {
    int We, q, r;
    FA_QSPLIT_FN int first(int w) const { return w < We ? w * q + (w < r ? w : r) : We * q + r; }
    FA_QSPLIT_FN int owner(int t) const {
        const uint32_t u = (uint32_t)t, big = (uint32_t)r * ((uint32_t)q + 1u);
        return (int)(u < big ? u / ((uint32_t)q + 1u) : (uint32_t)r + (u - big) / (uint32_t)q);
    }
};
FA_QSPLIT_FN Split split_list(int T, int W) {
    Split s;
    const int most = W < T / kMinTiles ? W : T / kMinTiles;
    s.We = most > 1 ? most : 1;
    s.q = (int)((uint32_t)T / (uint32_t)s.We);
    s.r = T - s.q * s.We;
    return s;
}

// Prefill. Ragged items, or few, are cut: laid end to end, head after head, their costs
// make a line that the workgroups share evenly, so one piece begins and one ends
// inside an item at most. Costs are in units of 32 keys: an item takes kStart more than
// its tiles of keys, and a workgroup takes at least kLeast. Ragged batch of 40 sequences
// of 64 to 8192 keys: 281 us with whole items in turn, 194 cut; kStart of 8, 16, 24: 207,
// 185, 183 us.
constexpr int kStart = 16, kLeast = 48;

struct Line {
    int64_t len;   // of one head
    int64_t total;
    int workers;
    FA_QSPLIT_FN int64_t cut(int w) const { return w * total / workers; }
    // the worker that holds place x: the last w with cut(w) <= x
    FA_QSPLIT_FN int holder(int64_t x) const { return (int)(((x + 1) * workers - 1) / total); }
};
FA_QSPLIT_FN Line make_line(int64_t len, int heads, int grid) {
    Line l;
    l.len = len;
    l.total = len * heads;
    const int64_t most = l.total / kLeast > 1 ? l.total / kLeast : 1;
    l.workers = (int)(grid < most ? grid : most);
    return l;
}
// The tile of an item at which a piece ends, or the next begins: `at` units past the
// item's start, tiles of nh units. Within the first kStart units: tile 0.
FA_QSPLIT_FN int tile_at(int64_t at, int nh) { return at > kStart ? (int)((at - kStart) / nh) : 0; }

}  // namespace fa
