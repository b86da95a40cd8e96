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
#include <math.h>
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

// How a launch's tiles are cut into items (find_item in kv_device.h): tiles of a run of `rows`
// rows, `tokens` to a tile; the units of `unit` keys that one of them sees at most (1 for a
// tile without keys: it is an item too); the items of a tile of so many units, `per` to an item.
__host__ __device__ inline int tiles_of(int rows, int tokens) { return (int)((uint32_t)(rows + tokens - 1) / (uint32_t)tokens); }
__host__ __device__ inline int units_of(int rows, int len, int table_keys, int tokens, int unit, int window) {
    int keys = clampi(len, 0, table_keys);
    const int reach = window + (rows < tokens ? rows : tokens);
    if (window > 0 && keys > reach) keys = reach;
    const int units = rows > 0 ? (int)((uint32_t)(keys + unit - 1) / (uint32_t)unit) : 0;
    return units < 1 ? 1 : units;
}
__host__ __device__ inline int parts_of(int units, int per) { return (int)((uint32_t)(units + per - 1) / (uint32_t)per); }

// Units of an item, two ways.  All requests alike: as many parts of each tile as there are slots
// for (at most `slots` items, or one to a tile); `most` is 1 at least.  Else an even share of all units, `sum` over
// the tiles (rounded up past the sum's error: at most `slots` items and one more to a tile).
__host__ __device__ inline int alike_units(int most, int tiles, int slots) {
    return parts_of(most, tiles > 0 && tiles < slots ? slots / tiles : 1);
}
__host__ __device__ inline int even_units(float sum, int slots) { return (int)fminf(sum * 1.0001f / (float)slots, 1.0e9f) + 1; }
// The one whose items, `slots` at a time, end sooner; but `least` at least.
__host__ __device__ inline int item_units(int alike, int items_alike, int even, int items_even, int slots, int least) {
    const float cost_alike = (float)parts_of(items_alike, slots) * (float)alike;
    const int per = (float)parts_of(items_even, slots) * (float)even < cost_alike ? even : alike;
    return per < least ? least : per;
}

// The most tiles of `tokens` rows that `runs` runs of least..most rows, `rows` in all, can make.
__host__ __device__ inline int most_tiles(int64_t rows, int64_t runs, int tokens, int least, int most) {
    const int64_t fit = rows / least;
    const int64_t by_rows = rows / tokens + (fit < runs ? fit : runs);
    const int64_t by_runs = runs * ((most < rows ? most : rows) / tokens + 1);
    return (int)(by_rows < by_runs ? by_rows : by_runs);
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
