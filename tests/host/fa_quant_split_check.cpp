// Host check of the work split of the attention kernels over 8-bit codes
// (flash-attention-npu_amd/csrc/fa_quant_split.h) against brute force: every tile of
// the decode list has one worker, owner() names it, and workers' ranges are
// equal up to a tile; every place of the prefill's line has one workgroup, holder()
// names it, and the pieces of each item, followed as the kernel follows them, cover its
// tiles once and in order and lie with as many workgroups as the merge is told.
#include <cstdio>
#include <random>
#include <vector>

#include "fa_quant_split.h"

using namespace fa;

static int failures = 0;
#define CHECK(cond, ...)                                  \
    do {                                                  \
        if (!(cond)) {                                    \
            if (++failures <= 20) {                       \
                std::printf("FAIL %s:%d: ", __FILE__, __LINE__); \
                std::printf(__VA_ARGS__);                 \
                std::printf("\n");                        \
            }                                             \
        }                                                 \
    } while (0)

static void check_list(int T, int W) {
    const Split s = split_list(T, W);
    CHECK(s.We >= 1 && s.We <= (W > 1 ? W : 1), "T %d W %d: We %d", T, W, s.We);
    CHECK(s.first(0) == 0 && s.first(W) == T, "T %d W %d", T, W);
    if (s.We > 1) CHECK(s.q >= kMinTiles, "T %d W %d: q %d", T, W, s.q);
    for (int w = 0; w < W; ++w) {
        const int a = s.first(w), b = s.first(w + 1);
        CHECK(a <= b && b - a - 1 <= s.q, "T %d W %d w %d: %d %d", T, W, w, a, b);
        if (w < s.We) CHECK(b - a >= s.q, "T %d W %d w %d: %d %d", T, W, w, a, b);
        else CHECK(a == b, "T %d W %d w %d: %d %d", T, W, w, a, b);
        const int step = b - a > 64 ? (b - a) / 16 : 1;
        for (long long t = a; t < b; t += step) CHECK(s.owner((int)t) == w, "T %d W %d t %lld: %d not %d", T, W, t, s.owner((int)t), w);
        if (a < b) CHECK(s.owner(b - 1) == w, "T %d W %d t %d", T, W, b - 1);
    }
}

static void check_line(const std::vector<int>& tiles, int heads, int grid, int nh) {
    std::vector<int64_t> at0(tiles.size() + 1, 0);
    for (size_t e = 0; e < tiles.size(); ++e) at0[e + 1] = at0[e] + kStart + (int64_t)tiles[e] * nh;
    const Line l = make_line(at0.back(), heads, grid);
    CHECK(l.workers >= 1 && l.workers <= grid, "workers %d of %d", l.workers, grid);
    CHECK(l.cut(0) == 0 && l.cut(l.workers) == l.total, "ends");
    std::vector<int> done(tiles.size() * heads, 0), pieces(tiles.size() * heads, 0), told(tiles.size() * heads, 0);
    for (int w = 0; w < l.workers; ++w) {
        int64_t at = l.cut(w);
        const int64_t end = l.cut(w + 1);
        CHECK(at < end, "worker %d has nothing", w);
        if (at < end) {
            CHECK(l.holder(at) == w && l.holder(end - 1) == w, "worker %d: holders %d %d", w, l.holder(at), l.holder(end - 1));
            CHECK(w == 0 || l.holder(at - 1) == w - 1, "worker %d", w);
        }
        int begun = 0, ended = 0;  // pieces that do not begin, or end, with their item
        while (at < end) {
            const int hk = (int)(at / l.len);
            size_t e = 0;
            while (e + 1 < tiles.size() && at0[e + 1] <= at - hk * l.len) ++e;
            const int64_t p0 = hk * l.len + at0[e], p1 = hk * l.len + at0[e + 1], upto = end < p1 ? end : p1;
            const size_t item = hk * tiles.size() + e;
            const int lo = at > p0 ? tile_at(at - p0, nh) : 0, hi = upto < p1 ? tile_at(upto - p0, nh) : tiles[e];
            CHECK(lo == done[item] && hi >= lo && hi <= tiles[e], "item %zu: tiles %d to %d after %d of %d", item, lo, hi, done[item], tiles[e]);
            done[item] = hi;
            ++pieces[item];
            begun += at > p0;
            ended += at == p0 && upto < p1;  // one that does both has the slot of the former
            if (at == p0) told[item] = l.holder(p1 - 1) - w + 1;
            at = upto;
        }
        CHECK(begun <= 1 && ended <= 1, "worker %d: %d and %d pieces", w, begun, ended);
    }
    for (size_t i = 0; i < done.size(); ++i)
        CHECK(done[i] == tiles[i % tiles.size()] && pieces[i] == told[i], "item %zu: %d of %d tiles, %d pieces, %d told", i, done[i],
              tiles[i % tiles.size()], pieces[i], told[i]);
}

int main() {
    std::mt19937 g(1);
    auto rnd = [&](int lo, int hi) { return lo + (int)(g() % (unsigned)(hi - lo + 1)); };
    long long cases = 0;
    for (int T = 0; T <= 300; ++T)
        for (int W : {1, 2, 3, 7, 64, 256, 512}) check_list(T, W), ++cases;
    for (int k = 0; k < 300; ++k) check_list(rnd(1, 1 << rnd(1, 30)), rnd(1, 2048)), ++cases;
    check_list(0x7fffffff, 2048);
    check_list(0x7fffffff, 1);
    for (int k = 0; k < 4000; ++k) {
        std::vector<int> tiles(rnd(1, k % 10 ? 12 : 300));
        const int most = 1 << rnd(0, 10);
        for (int& t : tiles) t = rnd(0, 4) ? rnd(0, most) : 0;
        check_line(tiles, rnd(1, 9), rnd(1, 300), 1 << rnd(0, 2));
        ++cases;
    }
    // as long as they come: 2048 entries of 2^30 keys, 65535 heads
    Line l = make_line(2048ll * (kStart + (1 << 25)), 65535, 256);
    CHECK(l.cut(256) == l.total && l.holder(l.total - 1) == 255 && l.holder(0) == 0, "the longest line");
    std::printf("%lld cases, %d failures\n", cases, failures);
    return failures != 0;
}
