// Host check of which rows the rotation may turn in place (flash-attention-npu_amd/csrc/fa_rotary_rows.h)
// against brute force: layouts that it lets pass hold no address twice, and those that users have pass.
#include <cstdio>
#include <random>
#include <set>

#include "fa_rotary_rows.h"

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

static std::multiset<int64_t> places(const RotaryRows& x, int64_t at) {
    std::multiset<int64_t> p;
    for (int64_t b = 0; b < x.size[0]; ++b)
        for (int64_t i = 0; i < x.size[1]; ++i)
            for (int64_t h = 0; h < x.size[2]; ++h)
                for (int64_t d = 0; d < x.hd; ++d) p.insert(at + b * x.stride[0] + i * x.stride[1] + h * x.stride[2] + d);
    return p;
}

static bool repeats(const std::multiset<int64_t>& p) {
    for (auto it = p.begin(); it != p.end(); ++it)
        if (p.count(*it) > 1) return true;
    return false;
}

int main() {
    std::mt19937 rng(7);
    auto up_to = [&](int lo, int hi) { return (int64_t)std::uniform_int_distribution<int>(lo, hi)(rng); };
    int once = 0, apart = 0, meet = 0;
    for (int n = 0; n < 60000; ++n) {
        RotaryRows q{}, k{};
        q.hd = k.hd = up_to(1, 4);
        // strides of a few nested layouts, and any
        const int64_t row = up_to(1, 6) * q.hd, most = up_to(0, 2) ? 24 : 4;
        for (int i = 0; i < 3; ++i) {
            q.size[i] = up_to(n % 50 == 0 ? 0 : 1, 3);
            k.size[i] = i < 2 ? q.size[i] : up_to(1, 3);
            q.stride[i] = up_to(0, 1) ? row * up_to(0, 4) : up_to(0, (int)most);
            k.stride[i] = up_to(0, 2) ? q.stride[i] : up_to(0, 1) ? row * up_to(0, 4) : up_to(0, (int)most);
        }
        const int64_t delta = up_to(-40, 40);
        const auto pq = places(q, 0), pk = places(k, delta);
        const bool alone = rows_once(q), clear = rows_apart(q, k, delta);
        CHECK(!alone || !repeats(pq), "case %d: q holds an address twice", n);
        bool both = false;
        for (int64_t x : pq) both |= pk.count(x) > 0;
        CHECK(!clear || !both, "case %d: q and k meet", n);
        once += alone;
        apart += clear;
        meet += both;
    }
    CHECK(once > 5000 && apart > 5000 && meet > 5000, "too few of a kind: %d %d %d", once, apart, meet);

    const int64_t B = 2, S = 5, H = 4, Hk = 2, D = 8, all = H + 2 * Hk;
    const RotaryRows q{{B, S, H}, {S * all * D, all * D, D}, D}, k{{B, S, Hk}, {S * all * D, all * D, D}, D};
    CHECK(rows_once(q) && rows_apart(q, k, H * D), "heads of a projection");
    CHECK(rows_apart(k, q, -H * D), "heads of a projection, k first");
    CHECK(!rows_apart(q, k, (H - 1) * D), "a head of both");
    CHECK(!rows_apart(q, k, 0), "one beginning");
    CHECK(!rows_apart(q, q, 0), "one tensor");
    const RotaryRows qt{{B, S, H}, {all * S * D, D, S * D}, D}, kt{{B, S, Hk}, {all * S * D, D, S * D}, D};
    CHECK(rows_once(qt) && rows_apart(qt, kt, H * S * D) && !rows_apart(qt, kt, (H - 1) * S * D), "heads first");
    const RotaryRows q3{{B, S, H}, {S * H * 3 * D, H * 3 * D, 3 * D}, D};
    CHECK(rows_apart(q3, q3, D) && rows_apart(q3, q3, 2 * D) && !rows_apart(q3, q3, 3 * D) && !rows_apart(q3, q3, D - 1), "q, k, v of each head");
    CHECK(!rows_apart(q3, RotaryRows{{B, S, 1}, {S * H * 3 * D, H * 3 * D, 0}, D}, 3 * D) &&
              rows_apart(q3, RotaryRows{{B, S, 1}, {S * H * 3 * D, H * 3 * D, 0}, D}, D), "one head of k");
    const RotaryRows qc{{B, S, H}, {S * H * D, H * D, D}, D}, kc{{B, S, Hk}, {S * Hk * D, Hk * D, D}, D};
    CHECK(rows_apart(qc, kc, B * S * H * D) && rows_apart(qc, kc, -B * S * Hk * D) && !rows_apart(qc, kc, B * S * H * D - 1), "two tensors");
    const RotaryRows one{{1, 1, H}, {0, 0, D}, D}, onek{{1, 1, Hk}, {7, 9, D}, D};
    CHECK(rows_apart(one, onek, H * D) && !rows_apart(one, onek, (H - 1) * D), "one row");
    const RotaryRows odd{{B, S, H}, {2 * S * H * D, 2 * H * D, D}, D};
    CHECK(rows_apart(odd, odd, H * D) && rows_apart(odd, odd, -H * D), "every other row");
    CHECK(rows_apart(RotaryRows{{0, S, H}, {0, 0, 0}, D}, k, 0), "no rows");
    std::printf("rotary rows: %d once, %d apart, %d meet, %d failures\n", once, apart, meet, failures);
    return failures != 0;
}
