// Launch interface of the paged-cache kernels (kv_heads.hip, kv_attention.hip, kv_tile.hip);
// arguments are checked by kv_runtime.cpp.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace kv {

// Strides in elements.
struct Pages {
    char* k;
    char* v;
    int64_t page_stride, token_stride, head_stride;
    int num_pages, page_shift, kv_heads, head_dim;
    int fp8;  // pages hold e4m3, else bf16
    float k_scale, v_scale;
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
AttnPlan plan_attention(const AttnArgs& a);
hipError_t launch_tiles(const AttnArgs& a, const Items& it, hipStream_t stream);  // kv_tile.hip
hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, hipStream_t stream);

}  // namespace kv
