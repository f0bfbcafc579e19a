// Where the rows of two tensors of a call lie in memory: plain C++, so that it can be checked against brute force on the host.
#pragma once
#include <cstdint>

namespace ttsamd {

// Rows of `bytes` bytes, [tokens][heads] of them, `t` and `h` bytes apart (any sign).
struct RowSet {
    const void *at;
    int64_t t, h, tokens, heads, bytes;
};

inline int64_t floor_div(int64_t x, int64_t y) { return x / y - (x % y != 0 && (x < 0) != (y < 0)); }

// Whether -below < d + i t + j h < above for some i in [i0, i1] and j in [j0, j1]; `apart`: other than i = j = 0.
inline bool lands(int64_t d, int64_t t, int64_t h, int64_t i0, int64_t i1, int64_t j0, int64_t j1, int64_t below, int64_t above, bool apart)
{
    if (i1 - i0 < j1 - j0) return lands(d, h, t, j0, j1, i0, i1, below, above, apart);
    if (t < 0) return lands(d, -t, h, -i1, -i0, j0, j1, below, above, apart);
    for (int64_t j = j0; j <= j1; ++j) {                      // the shorter range
        const int64_t x = d + j * h;
        int64_t i = t == 0 ? i0 : floor_div(-below - x, t) + 1;        // the first that is not too low
        if (i < i0) i = i0;
        if (apart && j == 0 && i == 0) ++i;
        if (i <= i1 && x + i * t > -below && x + i * t < above) return true;
    }
    return false;
}

// Whether two rows of a set share a byte.
inline bool rows_meet(const RowSet &a)
{
    const int64_t t = a.t < 0 ? -a.t : a.t, h = a.h < 0 ? -a.h : a.h;
    if (a.tokens < 2 ? a.heads < 2 || h >= a.bytes : a.heads < 2 ? t >= a.bytes : (h >= a.bytes && t >= (a.heads - 1) * h + a.bytes) ||
                                                                                  (t >= a.bytes && h >= (a.tokens - 1) * t + a.bytes))
        return false;
    return lands(0, a.t, a.h, -(a.tokens - 1), a.tokens - 1, -(a.heads - 1), a.heads - 1, a.bytes, a.bytes, true);
}

// Whether a and b are the same rows in the same places.
inline bool same_rows(const RowSet &a, const RowSet &b)
{
    return a.at == b.at && a.tokens == b.tokens && a.heads == b.heads && a.bytes == b.bytes && (a.tokens <= 1 || a.t == b.t) && (a.heads <= 1 || a.h == b.h);
}

// Whether a row of a and a row of b share a byte; also true where that is not easily told (other strides, and ranges that cross).
inline bool sets_meet(RowSet a, RowSet b)
{
    if (a.tokens < 1 || a.heads < 1 || b.tokens < 1 || b.heads < 1 || a.bytes < 1 || b.bytes < 1) return false;
    if (a.tokens == 1) a.t = b.t;
    if (b.tokens == 1) b.t = a.t;
    if (a.heads == 1) a.h = b.h;
    if (b.heads == 1) b.h = a.h;
    auto low = [](const RowSet &s) { return (s.t < 0 ? (s.tokens - 1) * s.t : 0) + (s.h < 0 ? (s.heads - 1) * s.h : 0); };
    auto high = [](const RowSet &s) { return (s.t > 0 ? (s.tokens - 1) * s.t : 0) + (s.h > 0 ? (s.heads - 1) * s.h : 0) + s.bytes; };
    const int64_t d = (int64_t)((uintptr_t)b.at - (uintptr_t)a.at);
    if (d + low(b) >= high(a) || d + high(b) <= low(a)) return false;
    if (a.t == b.t && a.h == b.h)
        return lands(d, a.t, a.h, -(a.tokens - 1), b.tokens - 1, -(a.heads - 1), b.heads - 1, b.bytes, a.bytes, false);
    if (a.t == b.t) {                                          // a token's heads as one run
        RowSet x = a, y = b;
        x.tokens = y.tokens = 1;
        const int64_t xl = low(x), xb = high(x) - xl, yl = low(y), yb = high(y) - yl;
        return lands(d + yl - xl, a.t, 0, -(a.tokens - 1), b.tokens - 1, 0, 0, yb, xb, false);
    }
    return true;
}

}  // namespace ttsamd
