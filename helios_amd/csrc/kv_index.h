// Index arithmetic of the paged-cache kernels, usable on the host: which tokens a query
// tile holds, which keys it can see, how a key range is split, where a key lies.
//
// A batch is `requests` runs of consecutive rows of q (run r: rows starts[r] up to
// starts[r + 1]); run r's last row is position kv_lens[r] - 1 of its request.  Rows past
// starts[requests] belong to no request; they are handled as one more run with no keys,
// so that their outputs are zeros.  Everything read from device memory is clamped before
// it is used as an index: rows to [0, tokens], a length to what its table row can hold,
// a page outside [0, num_pages) counts as absent.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kv {

constexpr int kGroupKeys = 16;  // keys of one MFMA tile; pages are multiples of it

__host__ __device__ inline int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }
__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// Keys [lo, hi) that at least one of the `n` query rows from position `pos0` on sees;
// empty as lo >= hi.  window 0: no lower bound.
struct KeyRange {
    int lo, hi;
};
__host__ __device__ inline KeyRange visible_keys(int pos0, int n, int kv_len, int window) {
    KeyRange r;
    r.hi = pos0 + n < kv_len ? pos0 + n : kv_len;
    r.lo = window > 0 && pos0 - window + 1 > 0 ? pos0 - window + 1 : 0;
    return r;
}

// The key tiles [first, last) of split `s` of `splits`, of `tiles` tiles.  At most
// ceil(tiles / least) of the splits get any, so short ranges are not spread thin.
struct TileRange {
    int first, last;
};
__host__ __device__ inline TileRange split_tiles(int tiles, int s, int splits, int least) {
    const int most = ceil_div(tiles, least);
    const int used = most < splits ? most : splits;
    TileRange r{0, 0};
    if (s >= used) return r;
    const int per = ceil_div(tiles, used);
    r.first = s * per < tiles ? s * per : tiles;
    r.last = r.first + per < tiles ? r.first + per : tiles;
    return r;
}

// Whether all 16 keys from `key` on are seen by every one of `n` rows from `pos0` on.
__host__ __device__ inline bool all_visible(int key, int keys, int pos0, int n, int window) {
    return key + keys - 1 <= pos0 && (window <= 0 || key > pos0 + n - 1 - window);
}

// Entry `at` of a request's table: its page, or -1 if there is none (past the table, or not
// a page of the cache).
__host__ __device__ inline int page_at(const int* table, int at, int width, int num_pages) {
    if (at < 0 || at >= width) return -1;
    const int page = table[at];
    return page >= 0 && page < num_pages ? page : -1;
}

// The rows of run r (r = requests: the rows past the last start), clamped to the batch.
__host__ __device__ inline int run_bound(const int* starts, int r, int requests, int tokens) {
    return r > requests ? tokens : clampi(starts[r], 0, tokens);
}

}  // namespace kv
