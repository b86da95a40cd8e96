// The overlap of strided arrays (overlap.h) on the host, for tests.
#include "overlap.h"

extern "C" {
int rt_overlap(uint64_t a, uint64_t a_len, uint64_t b, uint64_t b_len, const uint64_t* count, const uint64_t* stride) {
    return rt::overlap(reinterpret_cast<const void*>(a), a_len, reinterpret_cast<const void*>(b), b_len,
                       {{count[0], stride[0]}, {count[1], stride[1]}, {count[2], stride[2]}});
}
int rt_rows_overlap(uint64_t a, uint64_t a_stride, uint64_t a_len, uint64_t b, uint64_t b_stride, uint64_t b_len, uint64_t rows) {
    return rt::overlap(rt::Rows{reinterpret_cast<const void*>(a), a_stride, a_len}, rt::Rows{reinterpret_cast<const void*>(b), b_stride, b_len}, rows);
}
}
