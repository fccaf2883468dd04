// Whether two strided pieces of memory share a byte.
#pragma once
#include <cstdint>

namespace wt {

struct Strided3 {   // rows of `row` bytes at p + i0 * stride[0] + i1 * stride[1] + i2 * stride[2], i < size; strides >= 0
    const char *p;
    int64_t row;
    int n;                        // dimensions kept: more than one index, strides above zero, those that reach furthest first
    int64_t size[3], stride[3];

    Strided3() : p(nullptr), row(0), n(0) {}
    Strided3(const void *at, int64_t row_bytes, int dims, const int64_t *sizes, const int64_t *strides) : p(static_cast<const char *>(at)), row(row_bytes), n(0) {
        for (int i = 0; i < dims; ++i) {
            if (sizes[i] == 0) row = 0;
            if (sizes[i] <= 1 || strides[i] == 0) continue;
            int j = n++;
            for (; j > 0 && stride[j - 1] * (size[j - 1] - 1) < strides[i] * (sizes[i] - 1); --j) size[j] = size[j - 1], stride[j] = stride[j - 1];
            size[j] = sizes[i], stride[j] = strides[i];
        }
        if (row == 0) n = 0;
    }
    int64_t extent(int from) const {
        int64_t e = row;
        for (int i = from; i < n; ++i) e += stride[i] * (size[i] - 1);
        return e;
    }
};

// dimensions from ka on of a at 0, those from kb on of b at `delta`.  Dimensions of one stride are taken as one difference of indexes,
// others index by index where the pieces meet; steps run out only for pieces woven into each other in many different ways,
// which then count as overlapping.
inline bool overlap(const Strided3 &a, int ka, const Strided3 &b, int kb, int64_t delta, int *steps) {
    const int64_t ea = a.extent(ka), eb = b.extent(kb);
    if (delta >= ea || -delta >= eb) return false;
    if ((ka == a.n && kb == b.n) || --*steps < 0) return true;
    const auto first_above = [](int64_t x, int64_t s) { return x >= 0 ? x / s + 1 : -((-x + s - 1) / s) + 1; };   // least i with i * s > x
    if (ka < a.n && kb < b.n && a.stride[ka] == b.stride[kb]) {
        const int64_t s = a.stride[ka], ia = a.extent(ka + 1), ib = b.extent(kb + 1);
        int64_t d = first_above(-ib - delta, s);
        if (d < 1 - a.size[ka]) d = 1 - a.size[ka];
        for (; d < b.size[kb] && delta + d * s < ia; ++d)
            if (overlap(a, ka + 1, b, kb + 1, delta + d * s, steps)) return true;
        return false;
    }
    if (kb == b.n || (ka < a.n && ea >= eb)) {
        const int64_t s = a.stride[ka], ia = a.extent(ka + 1);
        int64_t i = first_above(delta - ia, s);
        if (i < 0) i = 0;
        for (; i < a.size[ka] && i * s < delta + eb; ++i)
            if (overlap(a, ka + 1, b, kb, delta - i * s, steps)) return true;
        return false;
    }
    const int64_t s = b.stride[kb], ib = b.extent(kb + 1);
    int64_t i = first_above(-ib - delta, s);
    if (i < 0) i = 0;
    for (; i < b.size[kb] && delta + i * s < ea; ++i)
        if (overlap(a, ka, b, kb + 1, delta + i * s, steps)) return true;
    return false;
}
inline bool overlap(const Strided3 &a, const Strided3 &b) {
    if (a.row == 0 || b.row == 0) return false;
    int steps = 1 << 20;
    return overlap(a, 0, b, 0, static_cast<int64_t>(reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p)), &steps);
}

}  // namespace wt
