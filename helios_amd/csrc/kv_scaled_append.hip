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
// in the same launch.  Bound by the chain of loads for few tokens (32 of one token, 16 query and 8
// KV heads of 256: 6.4 us) and by memory and the angles for many: five prompts of up to 777 tokens, 16
// and one of 512, 39 MB, 14.2 us, 2.7 TB/s, where a large copy moves 4.9 (26.6 with 256 threads, two
// passes over a block's tokens and a row of q to four workgroups).
#include "kv_heads_device.h"

namespace kv {
namespace {

// The new tokens of one block: rows row0.. of the batch, `n` of them, the first at position pos0 and
// slot `at` of the page in `entry` of `table`, `before` tokens of the block before it.
struct Run {
    int row0, n, pos0, at, before, entry;
    const int* table;
};

// Blocks [first, last) that positions [lo, hi) touch.
__device__ __forceinline__ int blocks_of(int lo, int hi, int shift) { return hi > lo ? ((hi - 1) >> shift) - (lo >> shift) + 1 : 0; }

// Number `index` of the batch's blocks; n = 0 past the last.  Every lane of the wave takes part.
__device__ __forceinline__ Run find_run(const Batch& b, const Pages& pg, int block_shift, int index, int lane) {
    Run run{0, 0, 0, 0, 0, 0, nullptr};
    const int table_keys = b.width << pg.page_shift;
    int before = 0;
    for (int base = 0; base < b.requests; base += 64) {
        const int r = base + lane;
        int start = 0, lo = 0, hi = 0, pos = 0;
        if (r < b.requests) {
            start = run_bound(b.starts, r, b.requests, b.tokens);
            const int rows = run_bound(b.starts, r + 1, b.requests, b.tokens) - start;
            const int len = b.kv_lens[r] > 0 ? b.kv_lens[r] : 0;  // may be past the table: positions count from it
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
            run.entry = begin >> pg.page_shift;
            run.table = b.tables + (int64_t)(base + at) * b.stride;
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

// Rows of q's `count` heads to a workgroup of `units`: a wave finds each.
__host__ __device__ inline int q_rows(int count, int units, int threads) {
    const int fit = units / count, waves = threads / 64;
    return fit < 1 ? 1 : (fit < waves ? fit : waves);
}

// One (block, head) of k or v, or some heads or rows of q.
template <int D, int THREADS>
__global__ __launch_bounds__(THREADS, 8) void scaled_append_kernel(HeadArgs a, BlockScales sc, int runs) {
    constexpr int LANES = D / 8, kUnits = THREADS / LANES;  // tokens at once
    constexpr int kHeld = 2;                                // rounds of them that stay in registers
    __shared__ float2 turn[kUnits][D / 2];
    __shared__ float tops[THREADS / 64];
    const int tid = (int)threadIdx.x, lane = tid & 63, c = tid & (LANES - 1), unit = tid / LANES;
    const int pairs = a.rope.pairs, dist = a.rope.distance;
    const int heads = a.pages.kv_heads, parts = 2 * heads;

    if ((int)blockIdx.x >= runs * parts) {
        // q: some heads of a row, or some whole rows
        __shared__ int positions[THREADS / 64], inside[THREADS / 64];
        const int count = a.part[0].count, rows_here = q_rows(count, kUnits, THREADS);
        const int per_row = ceil_div(count, kUnits);  // 1 where there are several rows
        const int index = (int)blockIdx.x - runs * parts;
        const int row0 = index / per_row * rows_here, nth = rows_here > 1 ? unit / count : 0;
        const int row = row0 + nth, head = (rows_here > 1 ? unit - nth * count : unit) + (index % per_row) * kUnits;
        const bool live = nth < rows_here && row < a.rows && head < count;
        float x[8] = {};
        if (live) load_head(a.part[0].x + row * a.part[0].x_stride + (int64_t)head * D + 8 * c, x);
        const uint4 weight = weight_of(a.part[0], c);
        const int wave = tid / 64;
        if (wave < rows_here) {
            const int at = __builtin_amdgcn_readfirstlane(row0 + wave < a.rows ? row0 + wave : a.rows - 1);
            const Row r = find_row(a.batch, a.pages, at, lane);
            if (lane == 0) {
                positions[wave] = r.pos;
                inside[wave] = r.in_batch;
            }
        }
        __syncthreads();
        for (int i = tid; i < rows_here * pairs; i += THREADS) {
            const int t = i / pairs;
            turn[t][i - t * pairs] = turn_by(positions[t], a.rope.inv_freq[i - t * pairs]);
        }
        __syncthreads();
        norm_of<D>(x, a.part[0], weight);
        if (pairs > 0) turn_head(x, turn[nth < rows_here ? nth : 0], pairs, dist, true, c, lane);
        if (!live) return;
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = inside[nth] ? pack_bf16(x[2 * i], x[2 * i + 1]) : 0u;
        *reinterpret_cast<uint4*>(a.part[0].out + row * a.part[0].out_stride + (int64_t)head * D + 8 * c) = make_uint4(o[0], o[1], o[2], o[3]);
        return;
    }

    const int index = (int)blockIdx.x / parts, part = (int)blockIdx.x - index * parts;
    const bool is_v = part >= heads;
    const int head = is_v ? part - heads : part;
    const Heads& from = is_v ? a.part[2] : a.part[1];
    const Run run = find_run(a.batch, a.pages, sc.block_shift, index, lane);
    if (run.n <= 0) return;
    const bool rot = !is_v && pairs > 0;
    const int rounds = ceil_div(run.n, kUnits);
    const uint16_t* const x0 = from.x + (int64_t)run.row0 * from.x_stride + (int64_t)head * D + 8 * c;

    // this thread's heads, normed and turned: of the first rounds in registers (all of them, but for
    // the longest blocks of the largest heads, whose others are made twice)
    float x[kHeld][8];
    const auto load = [&](int r, float (&v)[8]) {
        const int t = r * kUnits + unit;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
        if (t < run.n) load_head(x0 + (int64_t)t * from.x_stride, v);
    };
    const auto make = [&](int r, float (&v)[8]) {
        const int t0 = r * kUnits;
        if (rot) {
            __syncthreads();  // the round before is done with the angles
            for (int i = tid; i < kUnits * pairs; i += THREADS) {
                const int t = i / pairs;
                if (t0 + t < run.n) turn[t][i - t * pairs] = turn_by(run.pos0 + t0 + t, a.rope.inv_freq[i - t * pairs]);
            }
            __syncthreads();
        }
        norm_of<D>(v, from, weight_of(from, c));
        if (rot) turn_head(v, turn[unit], pairs, dist, true, c, lane);
    };
    float top = 0.0f;
    const auto raise = [&](int r, const float (&v)[8]) {
        if (r * kUnits + unit < run.n)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float size = fabsf(v[i]);
                top = size > top && size < __builtin_huge_valf() ? size : top;  // infinities and NaN have no say
            }
    };
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
        if (r < rounds) load(r, x[r]);
    const int page = page_at(run.table, run.entry, a.batch.width, a.pages.num_pages);
    if (page < 0) return;
    char* const codes = (is_v ? a.pages.v : a.pages.k) + (int64_t)page * a.pages.page_stride + (int64_t)head * a.pages.head_stride;
    uint8_t* const scale = (is_v ? sc.v : sc.k) + (int64_t)page * sc.page_stride + (int64_t)head * sc.head_stride + (run.at >> sc.block_shift);
    const int held = run.before > 0 ? clamp_scale(*scale) : kScaleBias + kScaleLow;
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
        if (r < rounds) {
            make(r, x[r]);
            raise(r, x[r]);
        }
    for (int r = kHeld; r < rounds; ++r) {
        float v[8];
        load(r, v);
        make(r, v);
        raise(r, v);
    }
    top = wave_max(top);
    if (lane == 0) tops[tid / 64] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) top = fmaxf(top, tops[w]);
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
    const auto store = [&](int r, const float (&v)[8]) {
        const int t = r * kUnits + unit;
        if (t < run.n) *reinterpret_cast<uint2*>(codes + (int64_t)(run.at + t) * a.pages.token_stride + 8 * c) = codes_of(v, by);
    };
#pragma unroll
    for (int r = 0; r < kHeld; ++r)
        if (r < rounds) store(r, x[r]);
    for (int r = kHeld; r < rounds; ++r) {
        float v[8];
        load(r, v);
        make(r, v);
        store(r, v);
    }
    if (tid == 0) *scale = (uint8_t)now;
}

// The most blocks that the batch's rows touch: n rows, n / block + 2 at most, and n.
int most_runs(const HeadArgs& a, const BlockScales& sc) {
    const int64_t touched = ((int64_t)a.rows >> sc.block_shift) + 2 * (int64_t)a.batch.requests;
    return (int)(touched < a.rows ? touched : a.rows);
}

// Threads of a workgroup: 256 for few tokens to a request (32 of one token, 8 KV heads of 256: 6.5 us, by
// 1024 12.2), else as many as hold a block's tokens in two rounds of them, in registers: 512 tokens
// of one KV head of 512, blocks of 16, 13.8 us by 256 and 9.0 by 512; 2048 tokens of 8 of 256, blocks
// of 16, 29 by 256 and 46 by 1024; 4 requests of 500, blocks of 64, 50 by 256 and 36 by 1024.
int threads_of(const HeadArgs& a, const BlockScales& sc) {
    if (a.rows < 8 * a.batch.requests) return 256;
    const int lanes = (a.head_dim / 8) << sc.block_shift;
    return lanes <= 2 * 256 ? 256 : (lanes <= 2 * 512 ? 512 : 1024);
}

int64_t groups_of(const HeadArgs& a, const BlockScales& sc) {
    const int threads = threads_of(a, sc), units = threads / (a.head_dim / 8), count = a.part[0].count;
    const int64_t q = count == 0 ? 0 : (int64_t)ceil_div(a.rows, q_rows(count, units, threads)) * ceil_div(count, units);
    return (int64_t)most_runs(a, sc) * 2 * a.pages.kv_heads + q;
}

template <int D>
hipError_t launch(const HeadArgs& a, const BlockScales& sc, hipStream_t stream) {
    const unsigned groups = (unsigned)groups_of(a, sc);
    const int runs = most_runs(a, sc);
    switch (threads_of(a, sc)) {
        case 256: scaled_append_kernel<D, 256><<<groups, 256, 0, stream>>>(a, sc, runs); break;
        case 512: scaled_append_kernel<D, 512><<<groups, 512, 0, stream>>>(a, sc, runs); break;
        default: scaled_append_kernel<D, 1024><<<groups, 1024, 0, stream>>>(a, sc, runs); break;
    }
    return hipGetLastError();
}

}  // namespace

bool scaled_append_fits(const HeadArgs& a, const BlockScales& sc) {
    return groups_of(a, sc) * threads_of(a, sc) <= 0xFFFFFFFFll;  // a launch counts its threads in 32 bits
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
