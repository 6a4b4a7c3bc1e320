// fa_checks.h -- what the C entries' argument checks share: the message of a refusal,
// alignment, multiples.
#pragma once
#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "../../include/fa_mi355x.h"

namespace fa {
fa_status_t report_error(fa_status_t st, const char* msg);
}  // namespace fa

namespace {

inline fa_status_t fail(fa_status_t st, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return fa::report_error(st, buf);
}

#define FA_CHECK(cond, ...)                              \
    do {                                                 \
        if (!(cond)) return fail(FA_EINVAL, __VA_ARGS__); \
    } while (0)

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline bool multiples(int64_t n, int64_t a, int64_t b, int64_t c) { return a % n == 0 && b % n == 0 && c % n == 0; }

}  // namespace
