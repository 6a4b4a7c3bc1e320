// fa_rotary_rows.h -- whether rows that are turned in place lie apart: a row that is there
// twice, or one of q's that is one of k's too, would be turned by two threads at once.
// Integer code on the host; tests/host/fa_rotary_rows_check.cpp holds it against brute force.
#pragma once
#include <stdint.h>

#include <algorithm>

namespace fa {

// Batch, rows and heads, and the channels of a head, which lie side by side. In elements.
struct RotaryRows {
    int64_t size[3], stride[3], hd;
    bool empty() const { return size[0] == 0 || size[1] == 0 || size[2] == 0 || hd == 0; }
};

// Up to three (stride, size)
struct RotarySteps {
    int64_t stride[3], size[3];
    int n = 0;
    void add(int64_t st, int64_t si) {
        if (si <= 1) return;
        int at = n++;
        for (; at > 0 && stride[at - 1] > st; --at) stride[at] = stride[at - 1], size[at] = size[at - 1];
        stride[at] = st;
        size[at] = si;
    }
    // Places are different addresses where each stride passes what the smaller ones reach, from `reach` on.
    bool apart(int64_t reach) const {
        for (int i = 0; i < n; ++i) {
            if (stride[i] <= reach) return false;
            reach += stride[i] * (size[i] - 1);
        }
        return true;
    }
};

inline bool rows_once(const RotaryRows& x) {
    if (x.empty()) return true;
    RotarySteps steps;
    for (int i = 0; i < 3; ++i) steps.add(x.stride[i], x.size[i]);
    return steps.apart(x.hd - 1);
}

// k begins `delta` elements behind q. They lie apart where some of the dimensions step alike in both, in steps that pass
// what the others reach, and what those others hold of q and of k, at one place of the first, are two ranges that do
// not meet: with none stepping alike, two tensors; rows, parts of one projection; heads, a projection whose q and k
// alternate. Others count as meeting.
inline bool rows_apart(const RotaryRows& q, const RotaryRows& k, int64_t delta) {
    if (q.empty() || k.empty()) return true;
    for (unsigned alike = 0; alike < 8; ++alike) {
        RotarySteps steps;
        int64_t rq = q.hd - 1, rk = k.hd - 1;
        bool ok = true;
        for (int i = 0; i < 3; ++i) {
            if (alike >> i & 1) {
                if (q.size[i] > 1 && k.size[i] > 1 && q.stride[i] != k.stride[i]) ok = false;
                steps.add(q.size[i] > 1 ? q.stride[i] : k.stride[i], std::max(q.size[i], k.size[i]));
            } else {
                rq += q.size[i] > 1 ? q.stride[i] * (q.size[i] - 1) : 0;
                rk += k.size[i] > 1 ? k.stride[i] * (k.size[i] - 1) : 0;
            }
        }
        if (!ok || (delta <= rq && delta + rk >= 0)) continue;
        if (steps.apart(std::max(rq, delta + rk) - std::min<int64_t>(0, delta))) return true;
    }
    return false;
}

}  // namespace fa
