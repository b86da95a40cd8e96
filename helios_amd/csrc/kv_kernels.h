// Launch interface of the paged-cache kernels (kv_heads.hip, kv_scaled_append.hip, kv_attention.hip,
// kv_tile.hip, kv_scaled.hip, kv_pool.hip); arguments are checked by kv_runtime.cpp.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kv {

// The pages of a cache that are free (the first free_count of free_pages, the last one next), the
// requests' tokens and their tables.
struct Pool {
    int* free_pages;
    int* free_count;
    int* lens;
    int* tables;
    int64_t stride;
    int num_pages, page_shift, requests, width;
};
struct Reserve {
    const int* new_tokens;
    int* starts;
    int* kv_lens;
    int* granted;      // may be null, as the next two
    int* positions;
    int64_t* slots;
};
size_t reserve_scratch(const Pool& p, int rows);  // bytes of launch_reserve's needs; 0: null
hipError_t launch_reserve(const Pool& p, const Reserve& a, int rows, int* needs, hipStream_t stream);  // kv_pool.hip
size_t release_scratch(const Pool& p);  // bytes of launch_release's counts; 0: null
hipError_t launch_release(const Pool& p, const int* lens, int window, int* counts, hipStream_t stream);

// Strides in elements.
struct Pages {
    char* k;
    char* v;
    int64_t page_stride, token_stride, head_stride;
    int num_pages, page_shift, kv_heads, head_dim;
    int fp8;  // pages hold e4m3, else bf16
    float k_scale, v_scale;
};

// A scale for each block of 2^block_shift tokens of a page and KV head, 2^(byte - 127): those of
// page p and head h at p * page_stride + h * head_stride, a page's blocks side by side.
struct BlockScales {
    uint8_t* k;
    uint8_t* v;
    int64_t page_stride, head_stride;
    int block_shift;
};

struct Batch {
    const int* starts;
    const int* kv_lens;
    const int* tables;
    int requests, tokens, width, stride;
};

struct Rope {
    const float* inv_freq;
    int pairs, distance;
};

// One set of heads of every row: x[row * x_stride + head * D + d].
struct Heads {
    const uint16_t* x;
    uint16_t* out;  // q and k of the plain call; null: into the pages
    const uint16_t* weight;
    int64_t x_stride, out_stride;
    int count, norm;
    float eps;
};

struct HeadArgs {
    Heads part[3];  // q, k, v; count 0 where absent
    Rope rope;
    const int* positions;  // null: from the batch
    Batch batch;
    Pages pages;
    int rows, head_dim;
    int append;
};

hipError_t launch_heads(const HeadArgs& a, hipStream_t stream);
bool scaled_append_fits(const HeadArgs& a, const BlockScales& sc);  // whether the launch can count its threads
hipError_t launch_scaled_append(const HeadArgs& a, const BlockScales& sc, hipStream_t stream);  // kv_scaled_append.hip

struct AttnArgs {
    const uint16_t* q;
    uint16_t* out;
    float* lse;  // may be null
    int64_t q_stride, out_stride;
    Pages pages;
    Batch batch;
    int q_heads, window;
    float scale;
    int kernel;     // gemma4_kv_set_attention_kernel's setting
    int tile_from;  // requests of this many rows or more go to the 128-row tiles, the rest to rows16
};

// How the rows of one kernel are cut into items (kv_device.h Cuts): `slots` items fill the
// card (0: no cuts), `items` is the most there can be, each of `parts` KV heads' workgroups
// (or runs of heads).  A tile of one item is stored by the kernel itself; the others leave
// their rows' sums of e^(s - m) v in part_o [items][parts][rows][head_dim] and (m, sum of
// e^(s - m)) in part_ml, to be joined by a second launch.
struct Items {
    int slots, items, parts;
    float* part_o;
    float2* part_ml;
};

// How a call is run: which kernels, and their items.
constexpr int kNoTiles = 0x40000000;  // more rows than any request has
struct AttnPlan {
    bool use_tiles, use_rows;  // 128-row tiles; 16-row tiles
    int tile_from;             // AttnArgs::tile_from
    Items tiles, rows;
    size_t o_bytes(const Items& it, int rows_of, int head_dim) const {
        return it.slots > 0 ? (((size_t)it.items * it.parts * rows_of * head_dim * 4 + 255) & ~(size_t)255) : 0;
    }
    size_t ml_bytes(const Items& it, int rows_of) const {
        return it.slots > 0 ? (((size_t)it.items * it.parts * rows_of * sizeof(float2) + 255) & ~(size_t)255) : 0;
    }
};
constexpr int kThinRows = 16, kWideRows = 128;
AttnPlan plan_attention(const AttnArgs& a, bool scaled);  // scaled: the pages have block scales
hipError_t launch_tiles(const AttnArgs& a, const Items& it, hipStream_t stream);  // kv_tile.hip
hipError_t launch_scaled_tiles(const AttnArgs& a, const Items& it, const BlockScales& sc, hipStream_t stream);  // kv_scaled.hip
hipError_t launch_scaled_rows16(const AttnArgs& a, const Items& it, const BlockScales& sc, hipStream_t stream);
// scales: null, or those of e4m3 pages
hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, const BlockScales* scales, hipStream_t stream);

}  // namespace kv
