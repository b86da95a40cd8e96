// Device pieces of the head norms, the rotation and the appends (kv_heads.hip, kv_scaled_append.hip):
// a head of D elements lies in D/8 neighbouring lanes, eight to a lane.  heads_kernel has the norm and
// the turn written out: by these functions its code is ordered otherwise, and 2048 tokens of 17 heads
// of 512 took 22.4 us in place of 21.7.
#pragma once

#include "kv_device.h"

namespace kv {
namespace {

template <int DPP>
__device__ __forceinline__ float dpp_sum(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), DPP, 0xf, 0xf, true));
}
// Sum over a head's lanes, in each of them; all in registers.
template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
    v = dpp_sum<0xB1>(v);                      // lane ^ 1
    v = dpp_sum<0x4E>(v);                      // lane ^ 2
    v = dpp_sum<0x141>(v);                     // the other four of eight
    if (LANES > 8) v = dpp_sum<0x140>(v);      // the other eight of sixteen
    if (LANES > 16) {
        const u32x2 p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(p.x) + __uint_as_float(p.y);
    }
    if (LANES > 32) {
        const u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = __uint_as_float(p.x) + __uint_as_float(p.y);
    }
    return v;
}

__device__ __forceinline__ float clamp_e4m3(float v) {
    // NaN passes, as in a conversion
    return v != v ? v : fminf(fmaxf(v, -448.0f), 448.0f);
}

// Eight bf16 of a head as floats.
__device__ __forceinline__ void unpack_head(const uint32_t (&w)[4], float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = q4::bf16_lo(w[i]);
        x[2 * i + 1] = q4::bf16_hi(w[i]);
    }
}

// x / sqrt(mean of squares + eps) * weight, of a sum of squares over the head.
template <int D>
__device__ __forceinline__ void norm_head(float (&x)[8], float squares, float eps, const uint4& weight) {
    const float inv = rsqrtf(squares * (1.0f / D) + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= inv;
    const uint32_t w[4] = {weight.x, weight.y, weight.z, weight.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] *= q4::bf16_lo(w[i]);
        x[2 * i + 1] *= q4::bf16_hi(w[i]);
    }
}

// Cosine and sine of position * inv_freq, the angle formed and reduced in fp64.
__device__ __forceinline__ float2 turn_by(int pos, float inv_freq) {
    const double turns = (double)pos * (double)inv_freq * 0.15915494309189533577;
    const float f = (float)(turns - rint(turns));
    float s, cs;
    sincospif(2.0f * f, &s, &cs);
    return make_float2(cs, s);
}

// Turns the pairs of a head (`rot`; else it passes) by the cosines and sines in `turn`; c: the
// lane's place among the head's.  Every lane of the wave takes part.
__device__ __forceinline__ void turn_head(float (&x)[8], const float2* turn, int pairs, int dist, bool rot, int c, int lane) {
    if (dist == 1) {
        // a lane's four pairs turn or pass together (pairs is a multiple of 8); those that pass
        // are selected, as a turn by zero would spread an infinity to its neighbour (as a
        // branch it cost the other distances: 2048 tokens of 17 heads of 512 20.4 -> 20.9 us)
        const bool turns = rot && 4 * c < pairs;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 cs = turns ? turn[4 * c + i] : make_float2(1.0f, 0.0f);
            const float u0 = x[2 * i], u1 = x[2 * i + 1];
            x[2 * i] = turns ? u0 * cs.x - u1 * cs.y : u0;
            x[2 * i + 1] = turns ? u1 * cs.x + u0 * cs.y : u1;
        }
    } else {
        const int dl = dist / 8;
        const bool first = 8 * c < pairs, second = 8 * c >= dist && 8 * c < dist + pairs;
        const int src = lane + (first ? dl : (second ? -dl : 0));
        const int i0 = first ? 8 * c : 8 * c - dist;
        // the pair's other half, dl lanes up or down
        float other[8];
        if (dl == 32) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x[i]), __float_as_uint(x[i]), false, false);
                other[i] = __uint_as_float(first ? p.y : p.x);
            }
        } else if (dl == 16) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const u32x2 p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x[i]), __float_as_uint(x[i]), false, false);
                other[i] = __uint_as_float(first ? p.y : p.x);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) other[i] = __shfl(x[i], src);
        }
        if (rot && (first || second)) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 cs = turn[i0 + i];
                x[i] = first ? x[i] * cs.x - other[i] * cs.y : x[i] * cs.x + other[i] * cs.y;
            }
        }
    }
}

struct Row {
    int pos, page, slot;  // page -1: nothing to store
    bool in_batch;
};

// The request of row t and its place in the cache.  Every lane of the wave takes part.
__device__ __forceinline__ Row find_row(const Batch& b, const Pages& pg, int t, int lane) {
    Row r{0, -1, 0, false};
    // starts are nondecreasing: the request is the number of starts[1..] that are <= t
    int request = 0;
    for (int base = 0; base < b.requests; base += 64) {
        const int i = base + lane;
        const int end = i < b.requests ? b.starts[i + 1] : 0x7fffffff;
        const unsigned long long past = __ballot(end <= t);
        request += __popcll(past);
        if (past != ~0ull) break;
    }
    if (request >= b.requests || t < b.starts[0]) return r;
    const int first = b.starts[request], last = b.starts[request + 1];
    const int kv = b.kv_lens[request];
    r.in_batch = t >= first && t < last;
    r.pos = kv - (last - t);
    if (r.in_batch && r.pos >= 0)
        r.page = page_at(b.tables + (int64_t)request * b.stride, r.pos >> pg.page_shift, b.width, pg.num_pages);
    r.slot = r.pos & ((1 << pg.page_shift) - 1);
    return r;
}

}  // namespace
}  // namespace kv
