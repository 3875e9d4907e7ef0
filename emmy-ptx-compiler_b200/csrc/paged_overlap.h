// Whether two areas of memory, each of equal runs of bytes at up to three strides, have a byte in common. An operator may not
// write where it reads, or twice, in an order that nobody has chosen; but views of one buffer whose runs lie between one
// another's (queries, keys and values of one projection, keys and values side by side in a page) are apart.
#pragma once

#include <stdint.h>

#include <algorithm>

namespace emb {
namespace paged {

using wide = __int128;  // a 31-bit count times a 34-bit stride

struct Area {
    const char* name;
    uint64_t at;
    int64_t run;  // bytes of one
    wide end;     // behind the last byte
    int n = 0;
    int64_t count[3], stride[3];  // runs, and bytes from one to the next (the first n)

    Area(const char* name_, const void* p, int64_t run_) : name(name_), at(reinterpret_cast<uintptr_t>(p)), run(p ? run_ : 0), end(wide(at) + run) {}
    // (a stride of 0 repeats a run; no runs at all are no area)
    Area& by(int64_t c, int64_t s) {
        if (c < 1) run = 0;
        if (c > 1 && s > 0) count[n] = c, stride[n] = s, ++n, end += wide(c - 1) * s;
        return *this;
    }
    bool same(const Area& b) const {
        if (at != b.at || run != b.run || n != b.n) return false;
        for (int i = 0; i < n; ++i)
            if (count[i] != b.count[i] || stride[i] != b.stride[i]) return false;
        return true;
    }
};

struct Steps {  // how far two areas' runs may lie apart by one stride
    wide stride, back, ahead;
};

// is a sum of d_k stride_k, -back_k <= d_k <= ahead_k, between lo and hi? Strides descend, so that few d of each are left; where
// strides of two areas hardly differ there may be many, and the answer is yes when `looks` run out.
inline bool reaches(const Steps* s, int n, wide lo, wide hi, int& looks) {
    if (--looks < 0) return true;
    if (n == 0) return lo < 0 && 0 < hi;
    wide least = 0, most = 0;  // of the smaller strides' sum
    for (int k = 1; k < n; ++k) least -= s[k].back * s[k].stride, most += s[k].ahead * s[k].stride;
    const auto floor_of = [&](wide x) { return x >= 0 ? x / s[0].stride : -((-x + s[0].stride - 1) / s[0].stride); };
    const wide first = std::max(-s[0].back, floor_of(lo - most) + 1), end = std::min(s[0].ahead, floor_of(hi - least - 1));
    for (wide d = first; d <= end; ++d)
        if (reaches(s + 1, n - 1, lo - d * s[0].stride, hi - d * s[0].stride, looks)) return true;
    return false;
}

inline bool runs_touch(const Area& a, const Area& b) {
    Steps s[6] = {};
    int n = 0;
    const auto add = [&](wide stride, wide back, wide ahead) {
        int i = 0;
        while (i < n && s[i].stride > stride) ++i;
        if (i < n && s[i].stride == stride) {
            s[i].back += back, s[i].ahead += ahead;
            return;
        }
        for (int k = n++; k > i; --k) s[k] = s[k - 1];
        s[i] = {stride, back, ahead};
    };
    for (int i = 0; i < a.n; ++i) add(a.stride[i], 0, a.count[i] - 1);
    for (int i = 0; i < b.n; ++i) add(b.stride[i], b.count[i] - 1, 0);
    // run i of a is at a.at + x, run j of b at b.at + y, and x - y is such a sum: they meet where
    // b.at - a.at - a.run < x - y < b.at - a.at + b.run
    int looks = 4096;
    const wide ahead = wide(b.at) - wide(a.at);
    return reaches(s, n, ahead - a.run, ahead + b.run, looks);
}

inline bool touch(const Area& a, const Area& b) { return a.end > b.at && b.end > a.at && a.run > 0 && b.run > 0 && runs_touch(a, b); }

// the first of `written` that touches another of them or one of `read` (which: the names), but for a pair that is `allowed` where
// it is the same area
template <int W, int R> inline bool touches(const Area (&written)[W], const Area (&read)[R], const Area* allowed, const char* (&which)[2]) {
    for (int i = 0; i < W; ++i) {
        for (int k = i + 1; k < W; ++k)
            if (touch(written[i], written[k])) return which[0] = written[i].name, which[1] = written[k].name, true;
        for (int k = 0; k < R; ++k)
            if (touch(written[i], read[k]) && !(&read[k] == allowed && i == 0 && written[i].same(read[k]))) return which[0] = written[i].name, which[1] = read[k].name, true;
    }
    return false;
}

}  // namespace paged
}  // namespace emb
