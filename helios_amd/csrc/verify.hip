// Drafted tokens checked against the target's probabilities, and tokens sampled from logits.
//
//   z_i = cap tanh(x_i / cap) / T,  p_i = e^(z_i) / sum_j e^(z_j)   (q likewise of the drafter's)
//   draft d, the token of the next row, stands while u q_d < p_d
//   the first that does not: a token from max(p - q, 0); all stand: one from the last row's p
//   from weights w: the first i with w_0 + .. + w_i > u (w_0 + .. + w_(n-1))
//   T = 0: p and q are 1 at the first largest logit, 0 elsewhere
//   a logit of -inf or NaN has weight 0 whatever cap and T; a drafter that gives no logits is sure (q_d = 1)
//
// Sums and weights are fp64: a token is a place in a sum of some 2^18 terms, and an fp32 sum
// (2^-24 of it off) would miss by one wherever the terms are smaller than that.
//
// Bound by reading the logits once.  A row is cut into chunks, a workgroup each, that stay in
// registers between the search for the chunk's maximum and the sum of weights relative to it
// (stats_kernel).  Each request's own workgroups then join its rows' chunks, find the first draft
// that falls and sum max(p - q, 0) over their chunk of that one row (rest_kernel); a workgroup
// per request finds the chunk and the place in it (pick_kernel).  Orders are fixed: no atomics.
#include "q4_common.h"
#include "verify_kernels.h"

namespace verify {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kSweep = 8 * kThreads;  // places that a workgroup reads at once

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// A chunk's largest logit (as it is), the first place that has it, and the sum of its weights
// relative to it.
struct alignas(16) Part {
    double sum;
    float top;
    int at;
};

// What a request's row to sample from is: written by rest_kernel, read by pick_kernel.
struct alignas(16) Spot {
    double p_scale, q_scale;  // weights e^(..) times these are p and q
    float p_top, q_top;
    int row, token;           // token: the draft that fell where the drafter is sure; -1: none
    int kind;                 // 0: nothing to sample, 1: from p, 2: from max(p - q, 0)
    int pad;
};

struct Work {
    Part* parts;   // [target rows, then drafter's rows][chunks]
    double* rest;  // [requests][chunks], of requests whose spot is of kind 2
    Spot* spots;   // [requests]
};

__device__ __forceinline__ int clampi(int v, int lo, int hi) { return v < lo ? lo : (v > hi ? hi : v); }

__device__ __forceinline__ float value_of(const Logits& l, int64_t at) {
    return l.f32 ? static_cast<const float*>(l.x)[at] : __uint_as_float((uint32_t) static_cast<const uint16_t*>(l.x)[at] << 16);
}

__device__ __forceinline__ double capped(float x, double cap) {
    return cap > 0.0 ? cap * tanh((double)x / cap) : (double)x;
}

// e^(z(x) - z(top)); 0 for -inf and NaN.
__device__ __forceinline__ double weight(float x, float top, double z_top, double cap, double inv_heat) {
    if (x == top) return x == -__builtin_huge_valf() ? 0.0 : 1.0;
    if (!(x > -__builtin_huge_valf())) return 0.0;
    return exp((capped(x, cap) - z_top) * inv_heat);
}

// Eight values from place i0 on; -inf from `end` on.
template <bool F32>
__device__ __forceinline__ void load8(const Logits& l, int64_t row, int i0, int end, float (&x)[8]) {
    if constexpr (F32) {
        const float* at = static_cast<const float*>(l.x) + row * l.stride + i0;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i0 + i < end ? at[i] : -__builtin_huge_valf();
    } else {
        const uint16_t* at = static_cast<const uint16_t*>(l.x) + row * l.stride + i0;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = i0 + i < end ? __uint_as_float((uint32_t)at[i] << 16) : -__builtin_huge_valf();
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) v += __shfl_xor(v, d);
    return v;
}
// The larger logit, the earlier place of equals.
__device__ __forceinline__ void better(float& top, int& at, float other, int other_at) {
    const bool take = other > top || (other == top && other_at < at);
    top = take ? other : top;
    at = take ? other_at : at;
}
__device__ __forceinline__ void wave_best(float& top, int& at) {
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
        const float t = __shfl_xor(top, d);
        const int i = __shfl_xor(at, d);
        better(top, at, t, i);
    }
}
__device__ __forceinline__ double group_sum(double v, double* sums) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    double all = 0.0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all += sums[w];
    return all;
}

// The request of a row; `requests` for none.  Every lane of the wave takes part.
__device__ __forceinline__ int request_of(const Args& a, int row) {
    if (a.starts == nullptr) return row;
    const int lane = (int)threadIdx.x & 63;
    int request = 0;
    for (int base = 0; base < a.requests; base += 64) {
        const int i = base + lane;
        const int end = i < a.requests ? a.starts[i + 1] : 0x7fffffff;
        const unsigned long long past = __ballot(end <= row);
        request += __popcll(past);
        if (past != ~0ull) break;
    }
    return row < a.starts[0] ? a.requests : request;
}
__device__ __forceinline__ int start_of(const Args& a, int r) { return a.starts == nullptr ? r : clampi(a.starts[r], 0, a.rows); }
// 0 where the request is greedy
__device__ __forceinline__ double inv_heat_of(const Args& a, int r) {
    const float t = a.heats != nullptr ? a.heats[r] : a.heat;
    return t > 0.0f ? 1.0 / (double)t : 0.0;
}

template <bool F32, int SWEEPS>
__global__ __launch_bounds__(kThreads) void stats_kernel(Args a, Work w, Chunks c) {
    __shared__ double sums[kWaves];
    __shared__ float tops[kWaves];
    __shared__ int ats[kWaves];
    const int tid = (int)threadIdx.x;
    const int index = (int)blockIdx.x / c.count, chunk = (int)blockIdx.x - index * c.count;
    const bool of_draft = index >= a.rows;
    const int row = of_draft ? index - a.rows : index;
    const Logits& l = of_draft ? a.draft : a.target;
    const int begin = chunk * c.size, end = begin + c.size < a.vocab ? begin + c.size : a.vocab;
    float x[SWEEPS][8];
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s) load8<F32>(l, row, begin + s * kSweep + 8 * tid, end, x[s]);
    const int r = request_of(a, row);
    if (r >= a.requests) return;  // padding
    float top = -__builtin_huge_valf();
    int at = 0x7fffffff;
#pragma unroll
    for (int s = 0; s < SWEEPS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (x[s][i] > top) {
                top = x[s][i];
                at = begin + s * kSweep + 8 * tid + i;
            }
    wave_best(top, at);
    if ((tid & 63) == 0) {
        tops[tid >> 6] = top;
        ats[tid >> 6] = at;
    }
    __syncthreads();
    top = tops[0];
    at = ats[0];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) better(top, at, tops[i], ats[i]);
    const double inv_heat = inv_heat_of(a, r);
    double sum = 0.0;
    if (inv_heat > 0.0) {
        const double cap = l.cap, z_top = capped(top, cap);
#pragma unroll
        for (int s = 0; s < SWEEPS; ++s)
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += weight(x[s][i], top, z_top, cap, inv_heat);
        sum = group_sum(sum, sums);
    }
    if (tid == 0) w.parts[(int64_t)index * c.count + chunk] = Part{sum, top, at};
}

struct Total {
    double sum;
    float top;
    int at;
};
// A row's chunks joined, by the lanes of a wave.
__device__ __forceinline__ Total join(const Part* parts, int count, double cap, double inv_heat) {
    const int lane = (int)threadIdx.x & 63;
    Total t{0.0, -__builtin_huge_valf(), 0x7fffffff};
    for (int i = lane; i < count; i += 64) better(t.top, t.at, parts[i].top, parts[i].at);
    wave_best(t.top, t.at);
    if (inv_heat > 0.0) {
        const double z_top = capped(t.top, cap);
        for (int i = lane; i < count; i += 64) t.sum += parts[i].sum * weight(parts[i].top, t.top, z_top, cap, inv_heat);
        t.sum = wave_sum(t.sum);
    }
    return t;
}

// The probability of place `at`, as of its row's total.
__device__ __forceinline__ double chance(const Logits& l, int64_t row, int at, int vocab, const Total& t, double inv_heat) {
    if (at < 0 || at >= vocab) return 0.0;
    if (!(inv_heat > 0.0)) return at == t.at ? 1.0 : 0.0;
    const double w = weight(value_of(l, row * l.stride + at), t.top, capped(t.top, l.cap), l.cap, inv_heat);
    return t.sum > 0.0 ? w / t.sum : 0.0;
}

// The weight of place `at` of a request's row to sample from.
__device__ __forceinline__ double rest_weight(const Args& a, const Spot& s, int at, float x, float y, double p_z, double q_z, double inv_heat) {
    double v = weight(x, s.p_top, p_z, a.target.cap, inv_heat) * s.p_scale;
    if (s.kind == 2) {
        if (a.draft.x != nullptr) {
            v -= weight(y, s.q_top, q_z, a.draft.cap, inv_heat) * s.q_scale;
            v = v > 0.0 ? v : 0.0;
        } else if (at == s.token) {
            v = 0.0;
        }
    }
    return v;
}

template <bool F32>
__global__ __launch_bounds__(kThreads) void rest_kernel(Args a, Work w, Chunks c) {
    __shared__ double sums[kWaves];
    __shared__ int firsts[kWaves];
    __shared__ Spot spot;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = (int)blockIdx.x / c.count, chunk = (int)blockIdx.x - r * c.count;
    const int start = start_of(a, r);
    const int n = a.starts == nullptr ? 1 : start_of(a, r + 1) - start;
    if (chunk == 0) {
        // rows of no request
        if (a.starts != nullptr && r == a.requests - 1)
            for (int i = clampi(a.starts[a.requests], 0, a.rows) + tid; i < a.rows; i += kThreads) a.out[i] = -1;
        if (a.starts != nullptr && r == 0)
            for (int i = tid; i < start; i += kThreads) a.out[i] = -1;
    }
    if (n <= 0) {
        if (chunk == 0 && tid == 0) {
            if (a.accepted != nullptr) a.accepted[r] = 0;
            w.spots[r].kind = 0;
        }
        return;
    }
    const double inv_heat = inv_heat_of(a, r);
    const Part* const parts = w.parts + (int64_t)start * c.count;
    const Part* const draft_parts = w.parts + ((int64_t)a.rows + start) * c.count;

    // the first draft that falls: a wave to a row
    int first = n - 1;
    for (int i = wave; i < n - 1 && i < first; i += kWaves) {
        const int token = a.tokens[start + i + 1];
        const Total p = join(parts + (int64_t)i * c.count, c.count, a.target.cap, inv_heat);
        const double p_at = chance(a.target, start + i, token, a.vocab, p, inv_heat);
        double q_at = 1.0;
        if (a.draft.x != nullptr) {
            const Total q = join(draft_parts + (int64_t)i * c.count, c.count, a.draft.cap, inv_heat);
            q_at = chance(a.draft, start + i, token, a.vocab, q, inv_heat);
        }
        if (!((double)a.uniforms[2 * (start + i)] * q_at < p_at)) first = i;
    }
    if (lane == 0) firsts[wave] = first;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) first = firsts[i] < first ? firsts[i] : first;

    if (wave == 0) {
        Spot s{};
        s.row = start + first;
        const Total p = join(parts + (int64_t)first * c.count, c.count, a.target.cap, inv_heat);
        s.kind = inv_heat > 0.0 && p.sum > 0.0 ? (first < n - 1 ? 2 : 1) : 0;
        s.p_top = p.top;
        s.p_scale = p.sum > 0.0 ? 1.0 / p.sum : 0.0;
        s.token = -1;
        if (s.kind == 2) {
            if (a.draft.x != nullptr) {
                const Total q = join(draft_parts + (int64_t)first * c.count, c.count, a.draft.cap, inv_heat);
                s.q_top = q.top;
                s.q_scale = q.sum > 0.0 ? 1.0 / q.sum : 0.0;
            } else {
                s.token = a.tokens[s.row + 1];
            }
        }
        if (lane == 0) {
            spot = s;
            if (chunk == 0) {
                w.spots[r] = s;
                if (a.accepted != nullptr) a.accepted[r] = first;
                // greedy, or nothing has a weight: the first largest logit, or none
                if (s.kind == 0) a.out[s.row] = !(inv_heat > 0.0) && p.at < a.vocab ? p.at : -1;
            }
        }
    }
    __syncthreads();
    if (chunk == 0)
        for (int i = tid; i < n; i += kThreads)
            if (i != first) a.out[start + i] = i < first ? a.tokens[start + i + 1] : -1;
    const Spot s = spot;
    if (s.kind != 2) return;  // p's sums are those of its chunks

    const double p_z = capped(s.p_top, a.target.cap), q_z = capped(s.q_top, a.draft.cap);
    const int begin = chunk * c.size, end = begin + c.size < a.vocab ? begin + c.size : a.vocab;
    double sum = 0.0;
    for (int i0 = begin + 8 * tid; i0 < end; i0 += kSweep) {
        float x[8], y[8] = {};
        load8<F32>(a.target, s.row, i0, end, x);
        if (a.draft.x != nullptr) load8<F32>(a.draft, s.row, i0, end, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) sum += rest_weight(a, s, i0 + i, x[i], y[i], p_z, q_z, inv_heat);
    }
    sum = group_sum(sum, sums);
    if (tid == 0) w.rest[(int64_t)r * c.count + chunk] = sum;
}

// Inclusive sums over the workgroup's threads; `total` of all of them.
__device__ __forceinline__ double group_scan(double v, double* sums, double* total) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double up = __shfl_up(v, d);
        v += lane >= d ? up : 0.0;
    }
    __syncthreads();
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    double before = 0.0, all = 0.0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        before += i < wave ? sums[i] : 0.0;
        all += sums[i];
    }
    *total = all;
    return v + before;
}

template <bool F32>
__global__ __launch_bounds__(kThreads) void pick_kernel(Args a, Work w, Chunks c) {
    __shared__ double sums[kWaves];
    __shared__ int found, last;
    __shared__ double found_before;
    const int tid = (int)threadIdx.x, r = (int)blockIdx.x;
    Spot s = w.spots[r];
    if (s.kind == 0) return;
    const double inv_heat = inv_heat_of(a, r);
    const double u = (double)(a.starts == nullptr ? a.uniforms[s.row] : a.uniforms[2 * s.row + 1]);
    const double* const rest = w.rest + (int64_t)r * c.count;
    const Part* const parts = w.parts + (int64_t)s.row * c.count;
    const double p_z = capped(s.p_top, a.target.cap), q_z = s.kind == 2 ? capped(s.q_top, a.draft.cap) : 0.0;
    const auto chunk_weight = [&](int i) {
        if (i >= c.count) return 0.0;
        return s.kind == 2 ? rest[i] : parts[i].sum * weight(parts[i].top, s.p_top, p_z, a.target.cap, inv_heat) * s.p_scale;
    };
    double total = 0.0;
    const auto sum_all = [&]() {
        total = 0.0;
        for (int base = 0; base < c.count; base += kThreads) total += group_sum(chunk_weight(base + tid), sums);
    };
    sum_all();
    if (s.kind == 2 && !(total > 0.0)) {
        s.kind = 1;  // p and q are equal to the last bit
        sum_all();
    }
    const double goal = u * total;
    // the chunk: the first whose sum with those before it exceeds the goal, else the last with any weight
    if (tid == 0) {
        found = 0x7fffffff;
        last = -1;
        found_before = 0.0;
    }
    __syncthreads();
    double before = 0.0;
    for (int base = 0; base < c.count; base += kThreads) {
        const double v = chunk_weight(base + tid);
        double here;
        const double upto = before + group_scan(v, sums, &here);
        if (v > 0.0) atomicMax(&last, base + tid);
        if (v > 0.0 && upto > goal) atomicMin(&found, base + tid);
        __syncthreads();
        if (found == base + tid) found_before = upto - v;
        __syncthreads();
        if (found != 0x7fffffff) break;
        before += here;
    }
    const bool past = found == 0x7fffffff;  // rounding, or u >= 1: the last place with any weight
    const int chunk = past ? last : found;
    if (chunk < 0) {  // no weight at all: logits that are no numbers
        if (tid == 0) a.out[s.row] = -1;
        return;
    }
    const double before_chunk = found_before;
    __syncthreads();
    if (tid == 0) {
        found = 0x7fffffff;
        last = -1;
    }
    __syncthreads();
    const int begin = chunk * c.size, end = begin + c.size < a.vocab ? begin + c.size : a.vocab;
    before = past ? 0.0 : before_chunk;
    for (int base = begin; base < end; base += kSweep) {
        const int i0 = base + 8 * tid;
        float x[8], y[8] = {};
        double v[8], sum = 0.0;
        load8<F32>(a.target, s.row, i0, end, x);
        if (s.kind == 2 && a.draft.x != nullptr) load8<F32>(a.draft, s.row, i0, end, y);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = i0 + i < end ? rest_weight(a, s, i0 + i, x[i], y[i], p_z, q_z, inv_heat) : 0.0;
            sum += v[i];
        }
        double here;
        double upto = before + group_scan(sum, sums, &here) - sum;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            upto += v[i];
            if (v[i] > 0.0) {
                atomicMax(&last, i0 + i);
                if (!past && upto > goal) atomicMin(&found, i0 + i);
            }
        }
        __syncthreads();
        if (found != 0x7fffffff) break;
        before += here;
    }
    if (tid == 0) a.out[s.row] = found != 0x7fffffff ? found : last;
}

// Chunks of whole sweeps: about as many as fill the card twice, of 2048 to 8192 places.
Chunks chunks_of(const Args& a) {
    const int rows = a.rows * (a.draft.x != nullptr ? 2 : 1);
    const int sweeps = ceil_div(a.vocab, kSweep);
    int per = 1;
    while (per < 4 && (int64_t)ceil_div(sweeps, 2 * per) * rows >= 1024) per *= 2;
    return Chunks{per * kSweep, ceil_div(sweeps, per)};
}

// Workgroups of a launch, which counts its threads in 32 bits.
constexpr int64_t kMostGroups = 0xFFFFFFFFll / kThreads;

size_t part_bytes(const Args& a, const Chunks& c) { return (size_t)a.rows * (a.draft.x != nullptr ? 2 : 1) * c.count * sizeof(Part); }
size_t rest_bytes(const Args& a, const Chunks& c) { return (((size_t)a.requests * c.count * sizeof(double)) + 15) & ~(size_t)15; }

template <bool F32>
hipError_t launch_of(const Args& a, const Work& w, const Chunks& c, hipStream_t stream) {
    const unsigned rows = (unsigned)(a.rows * (a.draft.x != nullptr ? 2 : 1)) * (unsigned)c.count;
    switch (c.size / kSweep) {
        case 1: stats_kernel<F32, 1><<<rows, kThreads, 0, stream>>>(a, w, c); break;
        case 2: stats_kernel<F32, 2><<<rows, kThreads, 0, stream>>>(a, w, c); break;
        case 4: stats_kernel<F32, 4><<<rows, kThreads, 0, stream>>>(a, w, c); break;
        default: return hipErrorInvalidValue;
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    rest_kernel<F32><<<(unsigned)a.requests * (unsigned)c.count, kThreads, 0, stream>>>(a, w, c);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    pick_kernel<F32><<<(unsigned)a.requests, kThreads, 0, stream>>>(a, w, c);
    return hipGetLastError();
}

}  // namespace

bool fits(const Args& a) {
    const Chunks c = chunks_of(a);
    const int64_t rows = (int64_t)a.rows * (a.draft.x != nullptr ? 2 : 1);
    return rows * c.count <= kMostGroups && (int64_t)a.requests * c.count <= kMostGroups;
}

size_t scratch_bytes(const Args& a) {
    const Chunks c = chunks_of(a);
    return part_bytes(a, c) + rest_bytes(a, c) + (size_t)a.requests * sizeof(Spot);
}

hipError_t launch(const Args& a, void* scratch, hipStream_t stream) {
    const Chunks c = chunks_of(a);
    char* at = static_cast<char*>(scratch);
    Work w;
    w.parts = reinterpret_cast<Part*>(at);
    w.rest = reinterpret_cast<double*>(at + part_bytes(a, c));
    w.spots = reinterpret_cast<Spot*>(at + part_bytes(a, c) + rest_bytes(a, c));
    return a.target.f32 ? launch_of<true>(a, w, c, stream) : launch_of<false>(a, w, c, stream);
}

}  // namespace verify
