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
    return (uint32_t)q4::f32_to_bf16(a) | ((uint32_t)q4::f32_to_bf16(b) << 16);
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

// A query tile: `n` consecutive rows of q from `row0`, at positions pos0.. of `request`.
struct Tile {
    int request, row0, n, pos0, kv_len;
};

// Tile number `tile` of the batch when the rows of every request that has from `least` to
// `most` of them are cut into runs of `tokens`; n = 0 past the last.  All lanes of a wave
// take part; the result is the same in all.
__device__ __forceinline__ Tile find_tile(const Batch& b, int tile, int tokens, int least, int most, int lane) {
    int before = 0;
    for (int base = 0; base <= b.requests; base += 64) {
        const int r = base + lane;
        int s = 0, e = 0, len = 0;
        if (r <= b.requests) {
            s = run_bound(b.starts, r, b.requests, b.tokens);
            e = run_bound(b.starts, r + 1, b.requests, b.tokens);
            len = r < b.requests ? b.kv_lens[r] : 0;
        }
        const int rows = e - s >= least && e - s <= most ? e - s : 0;
        const int tiles = (rows + tokens - 1) / tokens;
        int sum = tiles;  // inclusive sum over the lanes
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(sum, d);
            sum += lane >= d ? o : 0;
        }
        const unsigned long long past = __ballot(before + sum > tile);
        if (past != 0) {
            const int at = __ffsll(past) - 1;
            Tile t;
            t.request = base + at;
            const int first = before + __builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(tiles, at);
            const int start = __builtin_amdgcn_readlane(s, at), count = __builtin_amdgcn_readlane(rows, at);
            const int skip = (tile - first) * tokens;
            t.row0 = start + skip;
            t.n = count - skip < tokens ? count - skip : tokens;
            const int kv = __builtin_amdgcn_readlane(len, at);
            t.pos0 = kv - count + skip;
            t.kv_len = kv;
            return t;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return Tile{0, 0, 0, 0, 0};
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
        if (all_visible(base, granule, t.pos0, t.n, a.window)) continue;
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
