// Head norms, position rotation and the append to a paged cache, in one pass.
//
//   n_d = x_d rsqrt(mean(x^2) + eps) w_d       (per head of D elements; w optional)
//   y_i = n_i cos - n_{i+s} sin,  y_{i+s} = n_{i+s} cos + n_i sin   (pairs i < P, distance s)
//
// Everything is computed in fp32 from the bf16 inputs and rounded once, when it is stored
// as bf16 or e4m3: no rounding between the norm and the rotation.  The angle
// position * inv_freq is formed and reduced to a turn in fp64 (its integer part reaches
// 2^31, where an fp32 product would be off by whole radians), its sine and cosine in fp32.
//
// Bound by memory (2 B read and 2 or 1 B written per element) for many rows and by the
// launch and its chain of loads for few.  A workgroup takes one row: the row's sines and
// cosines are computed once, into LDS, for all its heads.  A head is D/8 lanes of 16
// bytes each; the pair's other half lies s/8 lanes away (or, for adjacent pairs, in the
// lane itself), and the head's sum is taken over its lanes, in registers.  Up to five heads'
// loads per thread go out before anything that waits; fewer than 512 rows give every 256
// threads of heads a workgroup of their own.
// One token's 24 heads of 256: 3.5 us (4.2 with the loads after the row's position and with
// LDS permutes); 32 tokens into a cache of 64-token pages 4.7 (5.3); 2048 tokens of 17 heads
// of 512, 71 MB: 20 us, 3.5 TB/s, where a large copy moves 4.9.
#include "kv_device.h"

namespace kv {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 5;  // heads whose loads are on their way at once, per thread

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

// of q, k and v's, selected rather than indexed: the arguments stay in scalar registers
template <class T>
__device__ __forceinline__ T pick(int which, T q, T k, T v) {
    return which == 0 ? q : (which == 1 ? k : v);
}
template <>
__device__ __forceinline__ uint4 pick(int which, uint4 q, uint4 k, uint4 v) {
    return make_uint4(pick(which, q.x, k.x, v.x), pick(which, q.y, k.y, v.y), pick(which, q.z, k.z, v.z), pick(which, q.w, k.w, v.w));
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

template <int D>
__global__ __launch_bounds__(kThreads, 6) void heads_kernel(HeadArgs a) {
    constexpr int LANES = D / 8;
    constexpr int kUnits = kThreads / LANES;  // heads a workgroup handles at once
    __shared__ float2 turn[D / 2];
    const int tid = (int)threadIdx.x, lane = tid & 63;
    const int row = (int)blockIdx.x;
    const int c = tid & (LANES - 1);

    // A batch of heads at a time: all its loads go out first, the first batch's before anything
    // that waits (the row's request and page, the angles).
    const int nq = a.part[0].count, nk = a.part[1].count, nv = a.part[2].count;
    const int total = nq + nk + nv;
    const int stride = kUnits * (int)gridDim.y;
    const int rounds = ceil_div(total, stride);
    const auto unit_of = [&](int it) { return it * stride + (int)blockIdx.y * kUnits + tid / LANES; };
    const auto which_of = [&](int u) { return u < nq || u >= total ? 0 : (u < nq + nk ? 1 : 2); };
    const auto head_of = [&](int u, int which) { return u - (which == 0 ? 0 : (which == 1 ? nq : nq + nk)); };
    uint4 raw[kBatch];
    const auto load = [&](int it0) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            const int u = unit_of(it0 + b), which = which_of(u);
            const uint16_t* x = pick(which, a.part[0].x, a.part[1].x, a.part[2].x);
            const int64_t x_stride = pick(which, a.part[0].x_stride, a.part[1].x_stride, a.part[2].x_stride);
            raw[b] = make_uint4(0, 0, 0, 0);
            if (u < total) raw[b] = *reinterpret_cast<const uint4*>(x + row * x_stride + (int64_t)head_of(u, which) * D + 8 * c);
        }
    };
    load(0);
    const auto weight_of = [&](const Heads& p) {
        return p.weight != nullptr ? *reinterpret_cast<const uint4*>(p.weight + 8 * c)
                                   : make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);  // ones
    };
    const uint4 q_weight = weight_of(a.part[0]), k_weight = weight_of(a.part[1]), v_weight = weight_of(a.part[2]);

    Row r{0, -1, 0, true};
    if (a.append)
        r = find_row(a.batch, a.pages, row, lane);
    if (a.positions != nullptr) r.pos = a.positions[row];

    const int pairs = a.rope.pairs, dist = a.rope.distance;
    for (int i = tid; i < pairs; i += kThreads) {
        const double turns = (double)r.pos * (double)a.rope.inv_freq[i] * 0.15915494309189533577;
        const float f = (float)(turns - rint(turns));
        float s, cs;
        sincospif(2.0f * f, &s, &cs);
        turn[i] = make_float2(cs, s);
    }
    __syncthreads();

    for (int it0 = 0; it0 < rounds; it0 += kBatch) {
        if (it0 > 0) load(it0);
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (it0 + b >= rounds) break;
            const int u = unit_of(it0 + b);
            const bool live = u < total;
            const int which = which_of(u), head = head_of(u, which);
            const uint32_t w4[4] = {raw[b].x, raw[b].y, raw[b].z, raw[b].w};
            float x[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = q4::bf16_lo(w4[i]);
                x[2 * i + 1] = q4::bf16_hi(w4[i]);
            }
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
            ss = head_sum<LANES>(ss);
            if (pick(which, a.part[0].norm, a.part[1].norm, a.part[2].norm)) {
                const float inv = rsqrtf(ss * (1.0f / D) + pick(which, a.part[0].eps, a.part[1].eps, a.part[2].eps));
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= inv;
                const uint4 wr = pick(which, q_weight, k_weight, v_weight);
                const uint32_t ww[4] = {wr.x, wr.y, wr.z, wr.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[2 * i] *= q4::bf16_lo(ww[i]);
                    x[2 * i + 1] *= q4::bf16_hi(ww[i]);
                }
            }
            if (pairs > 0) {
                const bool rot = which != 2;
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
            if (!live) continue;
            uint16_t* const out = pick(which, a.part[0].out, a.part[1].out, a.part[2].out);
            if (out != nullptr) {
                const int64_t out_stride = pick(which, a.part[0].out_stride, a.part[1].out_stride, a.part[2].out_stride);
                uint32_t o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    o[i] = r.in_batch ? pack_bf16(x[2 * i], x[2 * i + 1]) : 0u;
                *reinterpret_cast<uint4*>(out + row * out_stride + (int64_t)head * D + 8 * c) =
                    make_uint4(o[0], o[1], o[2], o[3]);
            } else if (r.page >= 0) {
                const Pages& pg = a.pages;
                const int64_t at = (int64_t)r.page * pg.page_stride + (int64_t)head * pg.head_stride +
                                   (int64_t)r.slot * pg.token_stride + 8 * c;
                char* base = which == 1 ? pg.k : pg.v;
                if (pg.fp8) {
                    const float sc = which == 1 ? pg.k_scale : pg.v_scale;
                    float z[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) z[i] = clamp_e4m3(x[i] / sc);
                    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
                    lo = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], lo, true);
                    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(z[4], z[5], 0, false);
                    hi = __builtin_amdgcn_cvt_pk_fp8_f32(z[6], z[7], hi, true);
                    *reinterpret_cast<uint2*>(base + at) = make_uint2((uint32_t)lo, (uint32_t)hi);
                } else {
                    uint32_t o[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        o[i] = pack_bf16(x[2 * i], x[2 * i + 1]);
                    *reinterpret_cast<uint4*>(base + 2 * at) = make_uint4(o[0], o[1], o[2], o[3]);
                }
            }
        }
    }
}

template <int D>
hipError_t launch(const HeadArgs& a, hipStream_t stream) {
    const int units = kThreads / (D / 8);
    const int total = a.part[0].count + a.part[1].count + a.part[2].count;
    const dim3 grid((unsigned)a.rows, (unsigned)(a.rows < 512 ? ceil_div(total, units) : 1));
    heads_kernel<D><<<grid, kThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_heads(const HeadArgs& a, hipStream_t stream) {
    switch (a.head_dim) {
        case 64: return launch<64>(a, stream);
        case 128: return launch<128>(a, stream);
        case 256: return launch<256>(a, stream);
        case 512: return launch<512>(a, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace kv
