// Head norms, position rotation and the append to pages of e4m3 with a scale for each block of
// tokens and KV head.
//
// The norm and the rotation are those of kv_heads.hip.  For the new tokens of a block:
//
//   a  = max |y| over the block's new tokens and the head's dims
//   e  = the least exponent with a <= 448 * 2^e, in [-100, 80]
//   e' = e where the block's first slot is among them, else max(e, the block's exponent)
//   code = e4m3(y 2^-e');  tokens before them: code' = e4m3(code 2^(e_old - e'))
//
// The scales are powers of two: the scaling itself is exact, so a code has e4m3's one rounding,
// and when a later token raises the scale, the codes held lose only what falls under e4m3's
// least step (2^-9 of the scale).
//
// Every (block, KV head) of k and of v is a workgroup's, so the maximum needs no other; the
// block's codes are rewritten only where its scale rises.  q's rows have workgroups of their own
// in the same launch.
#include "kv_heads_device.h"

namespace kv {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 16;  // tokens held in registers at once; blocks are multiples of it

// The new tokens of one block: rows row0.. of the batch, `n` of them, the first at slot `at` of
// `page` (slots of the page), `before` tokens of the block before it.
struct Run {
    int row0, n, pos0, page, at, before;
};

// Blocks [first, last) that positions [lo, hi) touch.
__device__ __forceinline__ int blocks_of(int lo, int hi, int shift) { return hi > lo ? ((hi - 1) >> shift) - (lo >> shift) + 1 : 0; }

// Number `index` of the batch's blocks; n = 0 past the last.  Every lane of the wave takes part.
__device__ __forceinline__ Run find_run(const Batch& b, const Pages& pg, int block_shift, int index, int lane) {
    Run run{0, 0, 0, -1, 0, 0};
    const int table_keys = b.width << pg.page_shift;
    int before = 0;
    for (int base = 0; base < b.requests; base += 64) {
        const int r = base + lane;
        int start = 0, lo = 0, hi = 0, pos = 0;
        if (r < b.requests) {
            start = run_bound(b.starts, r, b.requests, b.tokens);
            const int rows = run_bound(b.starts, r + 1, b.requests, b.tokens) - start;
            const int len = clampi(b.kv_lens[r], 0, 0x40000000);
            if (rows > 0) {
                pos = len - rows;  // of the first row; rows before position 0 or past the table go nowhere
                lo = pos < 0 ? 0 : pos;
                hi = len < table_keys ? len : table_keys;
            }
        }
        const int blocks = blocks_of(lo, hi, block_shift);
        const int sum = wave_scan(blocks);
        const unsigned long long past = __ballot(before + sum > index);
        if (past != 0) {
            const int at = __ffsll(past) - 1;
            const int nth = index - (before + __builtin_amdgcn_readlane(sum, at) - __builtin_amdgcn_readlane(blocks, at));
            const int l = __builtin_amdgcn_readlane(lo, at), h = __builtin_amdgcn_readlane(hi, at);
            const int block = (l >> block_shift) + nth, begin = block << block_shift;
            const int first = l > begin ? l : begin, end = h < begin + (1 << block_shift) ? h : begin + (1 << block_shift);
            run.pos0 = first;
            run.n = end - first;
            run.before = first - begin;
            run.row0 = __builtin_amdgcn_readlane(start, at) + first - __builtin_amdgcn_readlane(pos, at);
            run.page = page_at(b.tables + (int64_t)(base + at) * b.stride, begin >> pg.page_shift, b.width, pg.num_pages);
            run.at = first & ((1 << pg.page_shift) - 1);
            return run;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return run;
}

__device__ __forceinline__ uint4 weight_of(const Heads& p, int c) {
    return p.weight != nullptr ? *reinterpret_cast<const uint4*>(p.weight + 8 * c)
                               : make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);  // ones
}

template <int D>
__device__ __forceinline__ void norm_of(float (&x)[8], const Heads& p, const uint4& weight) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
    ss = head_sum<D / 8>(ss);
    if (p.norm) norm_head<D>(x, ss, p.eps, weight);
}

__device__ __forceinline__ void load_head(const uint16_t* at, float (&x)[8]) {
    const uint4 raw = *reinterpret_cast<const uint4*>(at);
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    unpack_head(w, x);
}

__device__ __forceinline__ uint2 codes_of(const float (&x)[8], float by) {
    float z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) z[i] = clamp_e4m3(x[i] * by);
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(z[0], z[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(z[2], z[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(z[4], z[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(z[6], z[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// Codes by a power of two, rounded to codes again.
__device__ __forceinline__ uint32_t lowered(uint32_t w, float by) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    int out = __builtin_amdgcn_cvt_pk_fp8_f32(lo[0] * by, lo[1] * by, 0, false);
    out = __builtin_amdgcn_cvt_pk_fp8_f32(hi[0] * by, hi[1] * by, out, true);
    return (uint32_t)out;
}

// One (block, head) of k or v, or some heads of a row of q.
template <int D>
__global__ __launch_bounds__(kThreads) void scaled_append_kernel(HeadArgs a, BlockScales sc, int runs) {
    constexpr int LANES = D / 8, kUnits = kThreads / LANES;
    constexpr int kRounds = kChunk > kUnits ? kChunk / kUnits : 1;  // of a chunk's tokens
    __shared__ float2 turn[kChunk][D / 2];
    __shared__ float tops[kThreads / 64];
    const int tid = (int)threadIdx.x, lane = tid & 63, c = tid & (LANES - 1), unit = tid / LANES;
    const int pairs = a.rope.pairs, dist = a.rope.distance;
    const int heads = a.pages.kv_heads, parts = 2 * heads;

    if ((int)blockIdx.x >= runs * parts) {
        // q
        const int per_row = ceil_div(a.part[0].count, kUnits);
        const int index = (int)blockIdx.x - runs * parts;
        const int row = index / per_row, head = (index - row * per_row) * kUnits + unit;
        const bool live = head < a.part[0].count;
        float x[8] = {};
        if (live) load_head(a.part[0].x + row * a.part[0].x_stride + (int64_t)head * D + 8 * c, x);
        const uint4 weight = weight_of(a.part[0], c);
        const Row r = find_row(a.batch, a.pages, row, lane);
        for (int i = tid; i < pairs; i += kThreads) turn[0][i] = turn_by(r.pos, a.rope.inv_freq[i]);
        __syncthreads();
        norm_of<D>(x, a.part[0], weight);
        if (pairs > 0) turn_head(x, turn[0], pairs, dist, true, c, lane);
        if (!live) return;
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = r.in_batch ? pack_bf16(x[2 * i], x[2 * i + 1]) : 0u;
        *reinterpret_cast<uint4*>(a.part[0].out + row * a.part[0].out_stride + (int64_t)head * D + 8 * c) = make_uint4(o[0], o[1], o[2], o[3]);
        return;
    }

    const int index = (int)blockIdx.x / parts, part = (int)blockIdx.x - index * parts;
    const bool is_v = part >= heads;
    const int head = is_v ? part - heads : part;
    const Heads& from = is_v ? a.part[2] : a.part[1];
    const Run run = find_run(a.batch, a.pages, sc.block_shift, index, lane);
    if (run.n <= 0 || run.page < 0) return;
    const uint4 weight = weight_of(from, c);
    const bool rot = !is_v && pairs > 0;
    char* const codes = (is_v ? a.pages.v : a.pages.k) + (int64_t)run.page * a.pages.page_stride + (int64_t)head * a.pages.head_stride;
    uint8_t* const scale = (is_v ? sc.v : sc.k) + (int64_t)run.page * sc.page_stride + (int64_t)head * sc.head_stride + (run.at >> sc.block_shift);
    const int held = run.before > 0 ? clamp_scale(*scale) : kScaleBias + kScaleLow;

    // this thread's heads of the chunk from token `t0` on, normed and turned
    float x[kRounds][8];
    const auto take = [&](int t0) {
        if (rot) {
            __syncthreads();  // the chunk before is done with the angles
            for (int i = tid; i < kChunk * pairs; i += kThreads) {
                const int t = i / pairs;
                if (t0 + t < run.n) turn[t][i - t * pairs] = turn_by(run.pos0 + t0 + t, a.rope.inv_freq[i - t * pairs]);
            }
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int t = r * kUnits + unit;
            const bool live = t < kChunk && t0 + t < run.n;
#pragma unroll
            for (int i = 0; i < 8; ++i) x[r][i] = 0.0f;
            if (live) load_head(from.x + (int64_t)(run.row0 + t0 + t) * from.x_stride + (int64_t)head * D + 8 * c, x[r]);
            norm_of<D>(x[r], from, weight);
            if (rot) turn_head(x[r], turn[t < kChunk ? t : 0], pairs, dist, true, c, lane);
        }
    };

    float top = 0.0f;
    const auto raise = [&](int t0) {
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int t = r * kUnits + unit;
            if (t < kChunk && t0 + t < run.n)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = fabsf(x[r][i]);
                    top = v > top && v < __builtin_huge_valf() ? v : top;  // infinities and NaN have no say
                }
        }
    };
    for (int t0 = 0; t0 < run.n; t0 += kChunk) {
        take(t0);
        raise(t0);
    }
    top = wave_max(top);
    if (lane == 0) tops[tid / 64] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) top = fmaxf(top, tops[w]);
    const int least = least_scale(top);
    const int now = least > held ? least : held;

    if (run.before > 0 && now > held) {
        // the tokens before, by the new scale
        const float by = scale_value(kScaleBias - (now - held < kScaleBias ? now - held : kScaleBias - 1));  // 2^-126 leaves nothing either
        for (int t = unit; t < run.before; t += kUnits) {
            uint2* const at = reinterpret_cast<uint2*>(codes + (int64_t)(run.at - run.before + t) * a.pages.token_stride + 8 * c);
            const uint2 w = *at;
            *at = make_uint2(lowered(w.x, by), lowered(w.y, by));
        }
    }
    const float by = scale_value(2 * kScaleBias - now);
    for (int t0 = 0; t0 < run.n; t0 += kChunk) {
        if (run.n > kChunk) take(t0);
#pragma unroll
        for (int r = 0; r < kRounds; ++r) {
            const int t = r * kUnits + unit;
            if (t >= kChunk || t0 + t >= run.n) continue;
            *reinterpret_cast<uint2*>(codes + (int64_t)(run.at + t0 + t) * a.pages.token_stride + 8 * c) = codes_of(x[r], by);
        }
    }
    if (tid == 0) *scale = (uint8_t)now;
}

// The most blocks that the batch's rows touch: n rows, n / block + 2 at most, and n.
int most_runs(const HeadArgs& a, const BlockScales& sc) {
    const int64_t touched = ((int64_t)a.rows >> sc.block_shift) + 2 * (int64_t)a.batch.requests;
    return (int)(touched < a.rows ? touched : a.rows);
}

template <int D>
hipError_t launch(const HeadArgs& a, const BlockScales& sc, hipStream_t stream) {
    const int64_t groups = scaled_append_groups(a, sc);
    if (groups > (int64_t)kMostGroups) return hipErrorInvalidValue;
    scaled_append_kernel<D><<<(unsigned)groups, kThreads, 0, stream>>>(a, sc, most_runs(a, sc));
    return hipGetLastError();
}

}  // namespace

int64_t scaled_append_groups(const HeadArgs& a, const BlockScales& sc) {
    const int units = kThreads / (a.head_dim / 8);
    return (int64_t)most_runs(a, sc) * 2 * a.pages.kv_heads + (int64_t)a.rows * ceil_div(a.part[0].count, units);
}

hipError_t launch_scaled_append(const HeadArgs& a, const BlockScales& sc, hipStream_t stream) {
    switch (a.head_dim) {
        case 64: return launch<64>(a, sc, stream);
        case 128: return launch<128>(a, sc, stream);
        case 256: return launch<256>(a, sc, stream);
        case 512: return launch<512>(a, sc, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace kv
