// Launch interface of the paged-cache kernels (kv_heads.hip, kv_attention.hip); arguments
// are checked by kv_runtime.cpp.
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
    int tile_from;  // requests of this many rows or more go to the 128-row tiles, the rest to rows16
    // scratch of a split launch: [splits][tokens][q_heads] rows of head_dim, and their
    // running maximum and sum
    float* part_o;
    float2* part_ml;
    int splits;
};

// How a call is run: which kernels, and splits of the key range.
constexpr int kNoTiles = 0x40000000;  // more rows than any request has
struct AttnPlan {
    bool tiles, rows;  // 128-row tiles; 16-row tiles
    int tile_from;     // AttnArgs::tile_from
    int splits;
    size_t o_bytes, ml_bytes;
};
AttnPlan plan_attention(const AttnArgs& a);
hipError_t launch_tiles(const AttnArgs& a, hipStream_t stream);  // kv_tile.hip
hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, hipStream_t stream);

}  // namespace kv
