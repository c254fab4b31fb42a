// Host rules on buffers that share memory.  The serving kernels read their inputs in some CTAs while others write, so an
// output must be apart from everything else that a call touches, or lie exactly over the input that it replaces.
#pragma once

#include <stdint.h>

namespace deca {

// Runs of `bytes` bytes at every combination of up to four strides (bytes) and counts.
struct Region {
    const void *at;
    int64_t bytes;
    int64_t count[4], stride[4];
};

inline Region region(const void *at, int64_t bytes, int64_t n0 = 1, int64_t s0 = 0, int64_t n1 = 1, int64_t s1 = 0, int64_t n2 = 1,
                     int64_t s2 = 0) {
    return {at, bytes, {n0, n1, n2, 1}, {s0, s1, s2, 0}};
}

inline bool region_empty(const Region &r) {
    for (int i = 0; i < 4; ++i)
        if (r.count[i] <= 0) return true;
    return r.bytes <= 0 || !r.at;
}

// Whether the same elements lie at the same places.
inline bool regions_equal(const Region &a, const Region &b) {
    if (a.at != b.at || a.bytes != b.bytes) return false;
    for (int i = 0; i < 4; ++i)
        if (a.count[i] != b.count[i] || (a.count[i] > 1 && a.stride[i] != b.stride[i])) return false;
    return true;
}

// The first byte of a region and its length, without the dimensions whose stride is a multiple of `pitch` (0: with all).
inline void region_span(const Region &r, int64_t pitch, __int128 *first, __int128 *length) {
    *first = (__int128) reinterpret_cast<uintptr_t>(r.at);
    *length = r.bytes;
    for (int i = 0; i < 4; ++i) {
        if (r.count[i] <= 1 || (pitch != 0 && r.stride[i] % pitch == 0)) continue;
        const __int128 reach = (__int128)(r.count[i] - 1) * r.stride[i];
        if (reach < 0) *first += reach;
        *length += reach < 0 ? -reach : reach;
    }
}

// Whether no byte belongs to both, shown by spans that do not meet (pitch = 0), by spans of at most one pitch that do
// not meet on a circle of that length (column blocks of one projection, keys and values that alternate in one cache), or
// block by block where both repeat with one stride that is longer than both together.  False where none shows it.
inline bool regions_apart(const Region &a, const Region &b) {
    if (region_empty(a) || region_empty(b)) return true;
    auto apart_at = [&](int64_t pitch) {
        __int128 a0, an, b0, bn;
        region_span(a, pitch, &a0, &an);
        region_span(b, pitch, &b0, &bn);
        if (pitch == 0) return a0 + an <= b0 || b0 + bn <= a0;
        if (an > pitch || bn > pitch) return false;
        int64_t d = (int64_t)(b0 - a0) % pitch;
        if (d < 0) d += pitch;
        return d >= an && d + bn <= pitch;
    };
    if (apart_at(0)) return true;
    for (const Region *r : {&a, &b})
        for (int i = 0; i < 4; ++i) {
            const int64_t pitch = r->stride[i] < 0 ? -r->stride[i] : r->stride[i];
            if (r->count[i] > 1 && pitch > 0 && apart_at(pitch)) return true;
        }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            if (a.count[i] <= 1 || b.count[j] <= 1 || a.stride[i] != b.stride[j] || a.stride[i] <= 0) continue;
            Region x = a, y = b;
            x.count[i] = y.count[j] = 1;
            __int128 x0, xn, y0, yn;
            region_span(x, 0, &x0, &xn);
            region_span(y, 0, &y0, &yn);
            const __int128 from = x0 < y0 ? x0 : y0, to = x0 + xn > y0 + yn ? x0 + xn : y0 + yn;
            if (to - from <= a.stride[i] && regions_apart(x, y)) return true;
        }
    return false;
}

}  // namespace deca
