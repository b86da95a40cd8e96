// Device pieces shared by the paged attention kernels (kv_attention.hip, kv_tile.hip).
#pragma once

#include "kv_index.h"
#include "kv_kernels.h"
#include "q4_common.h"

namespace kv {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));


constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;
constexpr float kNegInf = -__builtin_huge_valf();

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// Maximum and sum over the four lanes l % 16, + 16, + 32, + 48.
__device__ __forceinline__ float col_max(float v) {
    u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
    p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
}
__device__ __forceinline__ float col_sum(float v) {
    u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(p.x) + __uint_as_float(p.y);
    p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p.x) + __uint_as_float(p.y);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), bf16x2));  // one conversion of two
}

// Two e4m3 of a word as two bf16 (exact).
template <bool HI>
__device__ __forceinline__ uint32_t e4m3_to_bf16(uint32_t w) {
    return __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
}

// Zeros the bf16 (or e4m3) values of a word that are infinite or NaN.
template <bool FP8>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {
    uint32_t keep = 0;
    if (FP8) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (((w >> (8 * i)) & 0x7Fu) != 0x7Fu) keep |= 0xFFu << (8 * i);
    } else {
        if ((w & 0x7F80u) != 0x7F80u) keep |= 0xFFFFu;
        if ((w & 0x7F800000u) != 0x7F800000u) keep |= 0xFFFF0000u;
    }
    return w & keep;
}
template <bool FP8>
__device__ __forceinline__ bool any_nonfinite(uint32_t w) {
    if (FP8) {
        // a byte is NaN as its low seven bits are all ones: adding one then carries into bit 7
        return (((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u) != 0;
    }
    return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
}

// Inclusive sum over the lanes of a wave (row shifts of 1, 2, 4, 8, then the rows' last
// lanes to the rows after them).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_scan(v), 63); }
template <int DPP, int ROWS>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), DPP, ROWS, 0xf, ROWS == 0xf));
}
__device__ __forceinline__ float wave_total(float v) {
    v = dpp_add<0x118, 0xf>(dpp_add<0x114, 0xf>(dpp_add<0x112, 0xf>(dpp_add<0x111, 0xf>(v))));
    v = dpp_add<0x143, 0xc>(dpp_add<0x142, 0xa>(v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ int wave_max(int v) {
    const auto at_least = [](int a, int b) { return a > b ? a : b; };
    v = at_least(v, __builtin_amdgcn_update_dpp(v, v, 0x111, 0xf, 0xf, false));
    v = at_least(v, __builtin_amdgcn_update_dpp(v, v, 0x112, 0xf, 0xf, false));
    v = at_least(v, __builtin_amdgcn_update_dpp(v, v, 0x114, 0xf, 0xf, false));
    v = at_least(v, __builtin_amdgcn_update_dpp(v, v, 0x118, 0xf, 0xf, false));
    v = at_least(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xa, 0xf, false));
    v = at_least(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(v, 63);
}

template <int DPP, int ROWS>
__device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(v), __float_as_int(v), DPP, ROWS, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float v) {
    v = dpp_max<0x118, 0xf>(dpp_max<0x114, 0xf>(dpp_max<0x112, 0xf>(dpp_max<0x111, 0xf>(v))));
    v = dpp_max<0x143, 0xc>(dpp_max<0x142, 0xa>(v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// A query tile: `n` consecutive rows of q from `row0`, at positions pos0.. of `request`; its
// keys are cut into `splits` parts, of which this is `split`; part s is item first_item + s.
struct Tile {
    int request, row0, n, pos0, kv_len;
    int split, splits, first_item;
};

// What the tiles of a launch are: the requests that have from `least` to `most` rows, cut
// into runs of `tokens`; their key ranges counted in units of `unit` keys, and cut so that
// there are about `slots` items (at most slots + the number of tiles; 0: no cuts).
struct Cuts {
    int tokens, least, most, unit, slots, window;
    int min_units, few_units;  // the least units of an item; where all units are fewer than the slots
};

// Item number `index` of the launch, or (BY_TILE) its tile number `index` as split 0; n = 0
// past the last.  The lengths are on the device only, so every workgroup finds the cuts
// anew: C units to an item, from the sum and the maximum of the requests' units.  All lanes
// of a wave take part; the result is the same in all.
template <bool BY_TILE>
__device__ __forceinline__ Tile find_item(const Batch& b, int page_shift, const Cuts& cuts, int index, int lane) {
    struct Run {
        int start, rows, len, tiles, units;
    };
    const auto load = [&](int base) {
        const int r = base + lane;
        Run run{0, 0, 0, 0, 0};
        if (r <= b.requests) {
            run.start = run_bound(b.starts, r, b.requests, b.tokens);
            const int end = run_bound(b.starts, r + 1, b.requests, b.tokens);
            run.len = r < b.requests ? b.kv_lens[r] : 0;
            run.rows = end - run.start >= cuts.least && end - run.start <= cuts.most ? end - run.start : 0;
        }
        run.tiles = tiles_of(run.rows, cuts.tokens);
        run.units = units_of(run.rows, run.len, b.width << page_shift, cuts.tokens, cuts.unit, cuts.window);
        return run;
    };
    const Run head = load(0);
    int per = 0x7fffffff >> 1;  // units of an item
    if (cuts.slots > 0) {
        float sum = 0.0f;
        int tiles = 0, most = 1;  // where the launch has no tile, too
        for (int base = 0; base <= b.requests; base += 64) {
            const Run r = base == 0 ? head : load(base);
            sum += wave_total((float)r.tiles * (float)r.units);
            tiles += wave_total(r.tiles);
            const int u = wave_max(r.tiles > 0 ? r.units : 0);
            most = most > u ? most : u;
        }
        const int alike = alike_units(most, tiles, cuts.slots), even = even_units(sum, cuts.slots);
        int items_alike = 0, items_even = 0;
        for (int base = 0; base <= b.requests; base += 64) {
            const Run r = base == 0 ? head : load(base);
            items_alike += wave_total(r.tiles * parts_of(r.units, alike));
            items_even += wave_total(r.tiles * parts_of(r.units, even));
        }
        per = item_units(alike, items_alike, even, items_even, cuts.slots, sum <= (float)cuts.slots ? cuts.few_units : cuts.min_units);
    }
    int before = 0, before_items = 0;
    for (int base = 0; base <= b.requests; base += 64) {
        const Run r = base == 0 ? head : load(base);
        const int splits = parts_of(r.units, per);
        const int sum = wave_scan(BY_TILE ? r.tiles : r.tiles * splits);
        const unsigned long long past = __ballot(before + sum > index);
        const int items = BY_TILE ? wave_scan(r.tiles * splits) : sum;
        if (past != 0) {
            const int at = __ffsll(past) - 1;
            Tile t;
            t.request = base + at;
            const int tiles = __builtin_amdgcn_readlane(r.tiles, at);
            t.splits = __builtin_amdgcn_readlane(splits, at);
            const int own = BY_TILE ? tiles : tiles * t.splits;
            const int nth = index - (before + __builtin_amdgcn_readlane(sum, at) - own);
            const int tile = BY_TILE ? nth : (int)((uint32_t)nth / (uint32_t)t.splits);
            t.split = BY_TILE ? 0 : nth - tile * t.splits;
            t.first_item = before_items + __builtin_amdgcn_readlane(items, at) - tiles * t.splits + tile * t.splits;
            if (tile < 0 || tile >= tiles) break;  // starts that are no starts: the sums have overflowed
            const int start = __builtin_amdgcn_readlane(r.start, at), count = __builtin_amdgcn_readlane(r.rows, at);
            const int skip = tile * cuts.tokens;
            t.row0 = start + skip;
            t.n = count - skip < cuts.tokens ? count - skip : cuts.tokens;
            t.kv_len = __builtin_amdgcn_readlane(r.len, at);
            t.pos0 = t.kv_len - count + skip;
            return t;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
        before_items += __builtin_amdgcn_readlane(items, 63);
    }
    return Tile{0, 0, 0, 0, 0, 0, 1, 0};
}

// Tokens x heads of a query tile of ROWS rows: all of a KV head's query heads if they fit
// (row = token * heads + head), else runs of ROWS of them.
struct Shape {
    int heads, chunks, tokens;
};
__host__ __device__ inline Shape tile_shape(int rows, int group) {
    Shape s;
    s.heads = group < rows ? group : rows;
    s.chunks = ceil_div(group, s.heads);
    s.tokens = rows / s.heads;
    return s;
}

// Units are what a workgroup takes in one step; an item is of 256 keys at least, of 128 where
// the call's units of 64 are no more than the slots, so that items of 128 fill half of them at
// most (four single tokens over 246 to 3316 keys of 512 dims: 17.8 us in place of 23; one over
// 32768, where the items are many, 21 either way and its join 8 for 6).  One unit past that
// border halves the items: of requests with 8 tokens over 1032 keys and 8 KV heads three (51
// units, 64 slots) make 216 workgroups, four (68) make 160.
constexpr int kRowsUnit = 64, kTileUnit = 32;
constexpr int kRowsLeast = 256, kRowsFew = 128, kTileLeast = 256;
__host__ __device__ inline Cuts rows_cuts(const AttnArgs& a, const Items& it, const Shape& sh) {
    return Cuts{sh.tokens, 1, a.tile_from - 1, kRowsUnit, it.slots, a.window, kRowsLeast / kRowsUnit, kRowsFew / kRowsUnit};
}
__host__ __device__ inline Cuts tile_cuts(const AttnArgs& a, const Items& it, const Shape& sh) {
    return Cuts{sh.tokens, a.tile_from, kNoTiles, kTileUnit, it.slots, a.window, kTileLeast / kTileUnit, kTileLeast / kTileUnit};
}

// Adds the infinities and NaN of groups that some row does not see to the outputs of the
// rows that do see them.  `put(row, head, dim, v)` adds v to that output.  Keys [lo, hi),
// masked in aligned groups of `granule`.
template <int D, bool FP8, class Put>
__device__ void fix_nonfinite(const AttnArgs& a, const Tile& t, const Shape& sh, int kv_head, int lo, int hi, int granule,
                              int threads, Put put) {
    const int* table = a.batch.tables + (int64_t)t.request * a.batch.stride;
    const Pages& pg = a.pages;
    for (int key = lo; key < hi; ++key) {
        const int base = key & ~(granule - 1);
        if (all_visible(base, granule, t.pos0, t.n, a.window)) {
            key = base + granule - 1;  // none of the group's
            continue;
        }
        const int page = page_at(table, key >> pg.page_shift, a.batch.width, pg.num_pages);
        if (page < 0) continue;
        const int64_t off = (int64_t)page * pg.page_stride + (int64_t)kv_head * pg.head_stride +
                            (int64_t)(key & ((1 << pg.page_shift) - 1)) * pg.token_stride;
        for (int d = (int)threadIdx.x; d < D; d += threads) {
            float v;
            if (FP8) {
                const uint32_t b = (uint8_t)pg.v[off + d];
                if ((b & 0x7Fu) != 0x7Fu) continue;
                v = __uint_as_float(0x7FC00000u);
            } else {
                const uint32_t b = reinterpret_cast<const uint16_t*>(pg.v)[off + d];
                if ((b & 0x7F80u) != 0x7F80u) continue;
                v = __uint_as_float(b << 16);
            }
            for (int i = 0; i < t.n; ++i) {
                const int pos = t.pos0 + i;
                if (key > pos || (a.window > 0 && key <= pos - a.window)) continue;
                for (int h = 0; h < sh.heads; ++h) put(i, h, d, v);
            }
        }
    }
}

}  // namespace
}  // namespace kv
