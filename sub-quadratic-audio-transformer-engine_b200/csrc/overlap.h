// Do two strided tensors share memory? Host-side checks of the C ABI's outputs (internal to libsubq_b200).
#pragma once

#include <stdint.h>

#include <algorithm>
#include <utility>

namespace subq {

// Rows of `bytes` bytes at `at` + sum of x_i stride_i, 0 <= x_i < count_i (strides in bytes, at least 0); no rows where a
// count is 0 or `at` is null.
struct MemRows {
    uintptr_t at = 0;
    int64_t bytes = 0;
    int64_t count[3] = {1, 1, 1};
    __int128 stride[3] = {0, 0, 0};

    bool none() const { return !at || bytes <= 0 || count[0] <= 0 || count[1] <= 0 || count[2] <= 0; }
    __int128 end() const {  // one past the last byte
        __int128 x = (__int128)at + bytes;
        for (int i = 0; i < 3; ++i) x += (count[i] - 1) * stride[i];
        return x;
    }
};

// Is there a z with lo_i <= z_i <= hi_i and L <= D + sum of stride_i z_i <= U? Strides descending and above 0, so that for
// nested strides (every ordinary layout) only a value or two of each z_i comes into question. `steps` bounds the search
// of layouts that are nothing of the kind, which are then taken to be apart.
struct Term {
    __int128 stride, lo, hi;
};
inline bool reaches(const Term* t, int n, __int128 D, __int128 L, __int128 U, int& steps) {
    if (n == 0) return L <= D && D <= U;
    if (--steps < 0) return false;
    __int128 least = 0, most = 0;  // what the terms after the first can add
    for (int i = 1; i < n; ++i) least += t[i].stride * t[i].lo, most += t[i].stride * t[i].hi;
    auto floor_div = [](__int128 a, __int128 b) { return a / b - (a % b < 0); };
    const __int128 s = t[0].stride;
    const __int128 from = std::max(t[0].lo, -floor_div(D + most - L, s)), to = std::min(t[0].hi, floor_div(U - D - least, s));
    for (__int128 z = from; z <= to; ++z)
        if (reaches(t + 1, n - 1, D + s * z, L, U, steps)) return true;
    return false;
}

// Terms of equal stride as one, descending.
inline int merge_terms(Term* t, int n) {
    std::sort(t, t + n, [](const Term& a, const Term& b) { return a.stride > b.stride; });
    int m = 0;
    for (int i = 0; i < n; ++i) {
        if (t[i].stride == 0 || (t[i].lo == 0 && t[i].hi == 0)) continue;
        if (m && t[m - 1].stride == t[i].stride) t[m - 1].lo += t[i].lo, t[m - 1].hi += t[i].hi;
        else t[m++] = t[i];
    }
    return m;
}

inline bool rows_overlap(const MemRows& a, const MemRows& b) {
    if (a.none() || b.none() || a.end() <= (__int128)b.at || b.end() <= (__int128)a.at) return false;
    Term t[6];
    for (int i = 0; i < 3; ++i) {
        t[i] = {a.stride[i], 0, a.count[i] - 1};
        t[3 + i] = {b.stride[i], -(__int128)(b.count[i] - 1), 0};
    }
    int steps = 1 << 16;
    // rows [A, A + a.bytes) and [B, B + b.bytes) meet where -a.bytes < A - B < b.bytes
    return reaches(t, merge_terms(t, 6), (__int128)a.at - (__int128)b.at, 1 - a.bytes, b.bytes - 1, steps);
}

// Do two different rows of one tensor share memory? (Of the two rows' indices, the first that differs is larger in one.)
inline bool rows_overlap_themselves(const MemRows& a) {
    if (a.none()) return false;
    for (int i = 0; i < 3; ++i) {
        if (a.count[i] == 1) continue;
        if (a.stride[i] < a.bytes) return true;
        Term t[3];
        int n = 0;
        t[n++] = {a.stride[i], 1, a.count[i] - 1};
        for (int j = i + 1; j < 3; ++j) t[n++] = {a.stride[j], -(__int128)(a.count[j] - 1), a.count[j] - 1};
        int steps = 1 << 16;
        if (reaches(t, merge_terms(t, n), 0, 1 - a.bytes, a.bytes - 1, steps)) return true;
    }
    return false;
}

}  // namespace subq
