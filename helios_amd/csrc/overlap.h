// Whether two arrays of a call share a byte, for arrays of strides: exact, so that arrays that lie
// between each other in one allocation pass.  Host only; what is known to be apart costs a comparison.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <initializer_list>
#include <utility>

namespace rt {

struct Axis {
    uint64_t count, stride;  // count 1 at least; stride in bytes
};

namespace overlap_detail {

typedef __int128 Wide;  // counts to 2^30 times strides to 2^41

inline Wide floor_div(Wide a, Wide b) { return a >= 0 ? a / b : -((-a + b - 1) / b); }

// Whether -b_len < delta + sum of k_i stride_i < a_len for some |k_i| < count_i, axes from `axis` on, the largest
// stride first.  Where one axis' stride spans all those after it there are two k to try; `steps` bounds
// the others, and an array that needs more is taken to overlap.
inline bool meet(Wide delta, Wide a_len, Wide b_len, const Axis* axis, const Axis* end, int* steps) {
    if (axis == end) return delta > -b_len && delta < a_len;
    Wide reach = 0;
    for (const Axis* i = axis + 1; i != end; ++i) reach += (Wide)(i->count - 1) * (Wide)i->stride;
    const Wide stride = (Wide)axis->stride, most = (Wide)axis->count - 1;
    if (stride == 0 || most == 0) return meet(delta, a_len, b_len, axis + 1, end, steps);
    const Wide low = -b_len - reach - delta, high = a_len + reach - delta;  // low < k stride < high
    const Wide first = std::max(-most, floor_div(low, stride) + 1), last = std::min(most, -floor_div(-high, stride) - 1);
    for (Wide k = first; k <= last; ++k) {
        if (--*steps < 0) return true;
        if (meet(delta + k * stride, a_len, b_len, axis + 1, end, steps)) return true;
    }
    return false;
}

}  // namespace overlap_detail

// Two arrays of the same axes, whose innermost runs are a_len and b_len bytes.
inline bool overlap(const void* a, uint64_t a_len, const void* b, uint64_t b_len, std::initializer_list<Axis> axes) {
    Axis sorted[4];
    size_t n = 0;
    for (const Axis& x : axes) sorted[n++] = x;
    std::sort(sorted, sorted + n, [](const Axis& x, const Axis& y) { return x.stride > y.stride; });
    const overlap_detail::Wide delta =
        (overlap_detail::Wide)reinterpret_cast<uintptr_t>(b) - (overlap_detail::Wide)reinterpret_cast<uintptr_t>(a);
    int steps = 1 << 14;
    return overlap_detail::meet(delta, (overlap_detail::Wide)a_len, (overlap_detail::Wide)b_len, sorted, sorted + n, &steps);
}

// `rows` rows (1 at least, under 2^24) of a and of b, each with a stride of its own under 2^34 bytes.
struct Rows {
    const void* at;
    uint64_t stride, bytes;
};
inline bool overlap(const Rows& a, const Rows& b, uint64_t rows) {
    if (rows == 1 || a.stride == b.stride) return overlap(a.at, a.bytes, b.at, b.bytes, {Axis{rows, a.stride}});
    const int64_t pa = (int64_t)reinterpret_cast<uintptr_t>(a.at), pb = (int64_t)reinterpret_cast<uintptr_t>(b.at);
    const int64_t sa = (int64_t)a.stride, sb = (int64_t)b.stride, last = (int64_t)rows - 1, la = (int64_t)a.bytes, lb = (int64_t)b.bytes;
    if (pa >= pb + last * sb + lb || pb >= pa + last * sa + la) return false;
    for (int64_t i = 0; i <= last; ++i) {
        // the last row of b that begins before this one of a ends
        const int64_t begin = pa + i * sa, before = begin + la - 1 - pb;
        if (before < 0) continue;
        const int64_t j = sb == 0 || before / sb > last ? last : before / sb;
        if (pb + j * sb + lb > begin) return true;
    }
    return false;
}

}  // namespace rt
