// capi_checks.h — what the C entry points' argument checks share.
#pragma once

#include "qimg_internal.h"

#define QIMG_REQUIRE(cond, ...)                                                     \
    do {                                                                            \
        if (!(cond)) return qimg::api_fail(QIMG_ERR_INVALID_ARG, __VA_ARGS__);      \
    } while (0)

namespace {

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
[[maybe_unused]] int64_t align256(int64_t n) { return (n + 255) / 256 * 256; }

// strides of a tensor [T, H, D], in elements
bool good_strides(int64_t t, int64_t h) {
    return t >= 0 && t <= (int64_t{1} << 24) && h >= 0 && t % 8 == 0 && h % 8 == 0;
}

// no two heads of an output [T, H, D] share memory: the rows of one dimension lie
// behind all that the other spans
bool apart(int T, int64_t t, int H, int64_t h, int D) {
    if (T == 1) return H == 1 || h >= D;
    if (H == 1) return t >= D;
    return (h >= D && t >= D && h <= (t - D) / (H - 1)) || (t >= D && h >= D && t <= (h - D) / (T - 1));
}

}  // namespace
