// Attention of new tokens over a paged cache.
//
//   s_ij = scale q_i . k_j,  out_i = sum_j softmax_j(s_i) v_j,  lse_i = log sum_j exp s_ij
//
// over the keys j that row i sees (kv_index.h).  One pass over the keys with the running
// maximum m and sum l of the softmax, all in fp32; the weights exp(s - m) <= 1 are rounded
// to bf16 for their product with V (matrix cores), which moves an output by about 2^-9 of
// its size over the square root of the keys that carry it, less than the output's own
// rounding to bf16.  l sums the weights before that rounding.  e4m3 keys and values are
// exact in bf16; their scales are applied to s and to the output.
//
// rows16_kernel: 16 query rows (tokens x heads sharing a KV head) at a time; each wave of
// a workgroup takes key tiles of its own and the waves' sums meet at the end.  Bound by
// the bytes of K and V: both go from memory straight into registers in the layout of the
// matrix instructions, with no LDS.
//   S^T = K Q^T (16x16x32, A = K): lane (n = l % 16, g = l / 16) of a 16-key group reads
//   16 bytes of key n; it gets back s of query n and keys 4g..4g+3.
//   O^T += V^T P^T (16x16x16, A = V^T): those four weights are just the lane's B operand.
//   For A the lane reads EPL consecutive values of each of its keys 4g..4g+3 and
//   transposes them among its own registers (byte permutes): product e of a block covers
//   the dims EPL m + e.  Query n's output then lies in lanes (n, g) as runs of 4 EPL dims.
//
// Masked places: a group of 16 keys that is not seen by all rows is masked by selects
// after the product, so nothing in a hidden key counts.  A weight of zero times an
// infinity or NaN in a hidden value would still be NaN: values of such groups that are
// not finite are taken as zero in the product, and what of them is visible is added to
// the outputs at the end (fix_nonfinite; only workgroups that met one run it).
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

constexpr int kWaves = 4;
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

// Tile number `tile` of the batch when every request's rows are cut into runs of `tokens`;
// n = 0 past the last.  All lanes of a wave take part; the result is the same in all.
__device__ __forceinline__ Tile find_tile(const Batch& b, int tile, int tokens, int lane) {
    int before = 0;
    for (int base = 0; base <= b.requests; base += 64) {
        const int r = base + lane;
        int s = 0, e = 0, len = 0;
        if (r <= b.requests) {
            s = run_bound(b.starts, r, b.requests, b.tokens);
            e = run_bound(b.starts, r + 1, b.requests, b.tokens);
            len = r < b.requests ? b.kv_lens[r] : 0;
        }
        const int rows = e > s ? e - s : 0;
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
// rows that do see them.  `put(row, dim, v)` adds v to that output.  Keys [lo, hi), from
// a multiple of 16.
template <int D, bool FP8, class Put>
__device__ void fix_nonfinite(const AttnArgs& a, const Tile& t, const Shape& sh, int kv_head, int lo, int hi, int threads,
                              Put put) {
    const int* table = a.batch.tables + (int64_t)t.request * a.batch.stride;
    const Pages& pg = a.pages;
    for (int key = lo; key < hi; ++key) {
        const int base = key & ~(kGroupKeys - 1);
        if (all_visible(base, kGroupKeys, t.pos0, t.n, a.window)) continue;
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

template <int D, bool FP8>
struct Rows16 {
    static constexpr int kElt = FP8 ? 1 : 2;
    static constexpr int kChunks = D * kElt / 64;              // 16-byte K loads per lane and 16-key group
    static constexpr int kEpl = (D / 16) < (16 / kElt) ? D / 16 : 16 / kElt;  // V values per lane and key
    static constexpr int kBlocks = D / (16 * kEpl);
    static constexpr int kVWords = kEpl * kElt / 4;            // words of those
    // 16-key groups per tile: K and V of a tile are about 32 KiB per workgroup step
    static constexpr int kGroups = D * kElt >= 512 ? 1 : 2;
};

template <int D, bool FP8>
__global__ __launch_bounds__(64 * kWaves, D == 512 ? 1 : 2) void rows16_kernel(AttnArgs a) {
    using C = Rows16<D, FP8>;
    constexpr int NG = C::kGroups;
    constexpr int kTileKeys = NG * kGroupKeys;
    __shared__ float2 ml[kWaves][16];
    __shared__ f32x4 obuf[2][D / 16 * 64];
    __shared__ int found[kWaves];

    const int lane = (int)threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int group = a.q_heads / a.pages.kv_heads;
    const Shape sh = tile_shape(16, group);
    const int per_tile = a.pages.kv_heads * sh.chunks;
    const int split = (int)blockIdx.y;
    const int tile_no = (int)blockIdx.x / per_tile;
    const int part = (int)blockIdx.x - tile_no * per_tile;
    const int kv_head = part / sh.chunks, chunk = part - kv_head * sh.chunks;

    const Tile t = find_tile(a.batch, tile_no, sh.tokens, lane);
    if (t.n <= 0) return;
    const int kv_len = clampi(t.kv_len, 0, a.batch.width << a.pages.page_shift);

    // this lane's query row
    const int tok = n / sh.heads, hh = n - tok * sh.heads;
    const int in_group = chunk * sh.heads + hh;
    const bool live = tok < t.n && in_group < group;
    const int row = t.row0 + (live ? tok : 0);
    const int q_head = kv_head * group + (live ? in_group : 0);
    const int pos = live ? t.pos0 + tok : t.pos0;
    const int above = a.window > 0 ? pos - a.window : -0x7fffffff;  // keys in (above, pos]

    u32x4 q[D / 32];
    {
        const uint16_t* qp = a.q + (int64_t)row * a.q_stride + (int64_t)q_head * D;
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            // the dims of step s in lane group g: those of K's 16-byte loads
            const int d = FP8 ? 64 * (s / 2) + 16 * g + 8 * (s & 1) : 32 * s + 8 * g;
            const u32x4 zero = {0, 0, 0, 0};
            q[s] = live ? *reinterpret_cast<const u32x4*>(qp + d) : zero;
        }
    }

    f32x4 o[C::kBlocks][C::kEpl];
#pragma unroll
    for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
        for (int e = 0; e < C::kEpl; ++e) o[b][e] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kNegInf, l = 0.0f;
    bool nonfinite = false;

    const KeyRange keys = visible_keys(t.pos0, t.n, kv_len, a.window);
    const int lo = keys.lo & ~(kGroupKeys - 1);
    const int tiles = keys.hi > lo ? ceil_div(keys.hi - lo, kTileKeys) : 0;
    const TileRange range = split_tiles(tiles, split, a.splits, kWaves);
    const int* table = a.batch.tables + (int64_t)t.request * a.batch.stride;
    const float c = a.scale * (FP8 ? a.pages.k_scale : 1.0f) * kLog2e;
    const uint32_t row_bytes = (uint32_t)a.pages.token_stride * C::kElt;
    const uint32_t k_lane = (uint32_t)n * row_bytes + 16u * g;
    const uint32_t v_lane = 4u * g * row_bytes + (uint32_t)(n * C::kEpl * C::kElt);

    int pages[NG];
    for (int i = 0, ti = range.first + wave; ti < range.last; ++i, ti += kWaves) {
        if ((i & 63) == 0) {
            // the table entries of this wave's next 64 tiles, one per lane
            const int tl = ti + lane * kWaves;
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                const int at = (lo + tl * kTileKeys + j * kGroupKeys) >> a.pages.page_shift;
                pages[j] = tl < range.last ? page_at(table, at, a.batch.width, a.pages.num_pages) : -1;
            }
        }
        u32x4 kf[NG][C::kChunks];
        uint32_t vf[NG][4][C::kBlocks][C::kVWords];
        int first_key[NG];
        bool there[NG];
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const int key = lo + ti * kTileKeys + j * kGroupKeys;
            const int page = __builtin_amdgcn_readlane(pages[j], i & 63);
            first_key[j] = key;
            there[j] = page >= 0;
            const int64_t off = ((int64_t)(there[j] ? page : 0) * a.pages.page_stride +
                                 (int64_t)kv_head * a.pages.head_stride +
                                 (int64_t)(key & ((1 << a.pages.page_shift) - 1)) * a.pages.token_stride) * C::kElt;
            const char* kp = a.pages.k + off;
            const char* vp = a.pages.v + off;
#pragma unroll
            for (int s = 0; s < C::kChunks; ++s)
                kf[j][s] = *reinterpret_cast<const u32x4*>(kp + k_lane + 64u * s);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
                    for (int w = 0; w < C::kVWords; ++w)
                        vf[j][k][b][w] = reinterpret_cast<const uint32_t*>(
                            vp + v_lane + (uint32_t)k * row_bytes + (uint32_t)(b * 16 * C::kEpl * C::kElt))[w];
        }

        float x[NG][4];
        float top = kNegInf;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int st = 0; st < D / 32; ++st) {
                u32x4 kk;
                if (FP8) {
                    const u32x4 raw = kf[j][st / 2];
                    const uint32_t w0 = (st & 1) ? raw.z : raw.x, w1 = (st & 1) ? raw.w : raw.y;
                    kk = u32x4{e4m3_to_bf16<false>(w0), e4m3_to_bf16<true>(w0), e4m3_to_bf16<false>(w1), e4m3_to_bf16<true>(w1)};
                } else {
                    kk = kf[j][st];
                }
                s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kk), __builtin_bit_cast(bf16x8, q[st]), s, 0, 0, 0);
            }
            const bool masked = !there[j] || !all_visible(first_key[j], kGroupKeys, t.pos0, t.n, a.window);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[j][r] = s[r] * c;
            if (masked) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = first_key[j] + 4 * g + r;
                    x[j][r] = there[j] && key <= pos && key > above ? x[j][r] : kNegInf;
                }
                bool bad = false;
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
                        for (int w = 0; w < C::kVWords; ++w) bad |= any_nonfinite<FP8>(vf[j][k][b][w]);
                if (__any(bad)) {
                    nonfinite = true;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
#pragma unroll
                        for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
                            for (int w = 0; w < C::kVWords; ++w) vf[j][k][b][w] = finite_only<FP8>(vf[j][k][b][w]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, x[j][r]);
        }
        top = col_max(top);
        if (__any(top > m)) {
            const float next = fmaxf(m, top);
            const float alpha = exp2_hw(m - (next == kNegInf ? 0.0f : next));
            m = next;
            l *= alpha;
#pragma unroll
            for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
                for (int e = 0; e < C::kEpl; ++e) o[b][e] *= alpha;
        }
        const float base = m == kNegInf ? 0.0f : m;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            float p[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[r] = exp2_hw(x[j][r] - base);
                l += p[r];
            }
            const u32x2 pb = {pack_bf16(p[0], p[1]), pack_bf16(p[2], p[3])};
            const s16x4 bop = __builtin_bit_cast(s16x4, pb);
#pragma unroll
            for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
                for (int w = 0; w < C::kVWords; ++w) {
                    const uint32_t k0 = vf[j][0][b][w], k1 = vf[j][1][b][w], k2 = vf[j][2][b][w], k3 = vf[j][3][b][w];
                    if (FP8) {
                        const uint32_t lo01 = __builtin_amdgcn_perm(k1, k0, 0x05010400u), hi01 = __builtin_amdgcn_perm(k1, k0, 0x07030602u);
                        const uint32_t lo23 = __builtin_amdgcn_perm(k3, k2, 0x05010400u), hi23 = __builtin_amdgcn_perm(k3, k2, 0x07030602u);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t sel = (e & 1) ? 0x07060302u : 0x05040100u;
                            const uint32_t four = e < 2 ? __builtin_amdgcn_perm(lo23, lo01, sel) : __builtin_amdgcn_perm(hi23, hi01, sel);
                            const u32x2 av = {e4m3_to_bf16<false>(four), e4m3_to_bf16<true>(four)};
                            o[b][4 * w + e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, av), bop, o[b][4 * w + e], 0, 0, 0);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const uint32_t sel = e ? 0x07060302u : 0x05040100u;
                            const u32x2 av = {__builtin_amdgcn_perm(k1, k0, sel), __builtin_amdgcn_perm(k3, k2, sel)};
                            o[b][2 * w + e] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, av), bop, o[b][2 * w + e], 0, 0, 0);
                        }
                    }
                }
        }
    }

    // the waves' sums, on a common maximum
    l = col_sum(l);
    if (g == 0) ml[wave][n] = make_float2(m, l);
    if (lane == 0) found[wave] = nonfinite;
    __syncthreads();
    float top = kNegInf;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, ml[w][n].x);
    const float base = top == kNegInf ? 0.0f : top;
    float total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) total += ml[w][n].y * exp2_hw(ml[w][n].x - base);
    const float mine = exp2_hw(m - base);
#pragma unroll
    for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
        for (int e = 0; e < C::kEpl; ++e) o[b][e] *= mine;
    const auto put = [&](int slot) {
#pragma unroll
        for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < C::kEpl; ++e) obuf[slot][(b * C::kEpl + e) * 64 + lane] = o[b][e];
    };
    const auto add = [&](int slot) {
#pragma unroll
        for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
            for (int e = 0; e < C::kEpl; ++e) o[b][e] += obuf[slot][(b * C::kEpl + e) * 64 + lane];
    };
    if (wave >= 2) put(wave - 2);
    __syncthreads();
    if (wave < 2) add(wave);
    __syncthreads();
    if (wave == 1) put(0);
    __syncthreads();
    const int64_t out_row = (int64_t)row * a.q_heads + q_head;
    const int64_t part_row = (int64_t)split * a.batch.tokens * a.q_heads;
    if (wave == 0) {
        add(0);
        if (live) {
            if (a.splits == 1) {
                const float norm = total > 0.0f || total != total ? (FP8 ? a.pages.v_scale : 1.0f) / total : 0.0f;
                uint16_t* op = a.out + (int64_t)row * a.out_stride + (int64_t)q_head * D;
#pragma unroll
                for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int e = 0; e < C::kEpl; e += 4) {
                            u32x2 w;
                            w.x = pack_bf16(o[b][e][r] * norm, o[b][e + 1][r] * norm);
                            w.y = pack_bf16(o[b][e + 2][r] * norm, o[b][e + 3][r] * norm);
                            *reinterpret_cast<u32x2*>(op + b * 16 * C::kEpl + C::kEpl * (4 * g + r) + e) = w;
                        }
                if (a.lse != nullptr && g == 0) a.lse[out_row] = (top + __builtin_amdgcn_logf(total)) * kLn2;
            } else {
                if (g == 0) a.part_ml[part_row + out_row] = make_float2(top, total);
                if (top != kNegInf || total != 0.0f) {
                    float* op = a.part_o + (part_row + out_row) * D;
#pragma unroll
                    for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int e = 0; e < C::kEpl; e += 4) {
                                const f32x4 w = {o[b][e][r], o[b][e + 1][r], o[b][e + 2][r], o[b][e + 3][r]};
                                *reinterpret_cast<f32x4*>(op + b * 16 * C::kEpl + C::kEpl * (4 * g + r) + e) = w;
                            }
                }
            }
        }
    }
    __syncthreads();
    bool fix = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) fix |= found[w] != 0;
    if (fix) {
        const int from = lo + range.first * kTileKeys;
        const int upto = lo + range.last * kTileKeys < keys.hi ? lo + range.last * kTileKeys : keys.hi;
        fix_nonfinite<D, FP8>(a, t, sh, kv_head, from, upto, 64 * kWaves, [&](int i, int h, int d, float v) {
            const int ig = chunk * sh.heads + h;
            if (ig >= group) return;
            const int64_t rr = t.row0 + i;
            const int qh = kv_head * group + ig;
            if (a.splits == 1) {
                uint16_t* op = a.out + rr * a.out_stride + (int64_t)qh * D + d;
                *op = q4::f32_to_bf16(__uint_as_float((uint32_t)*op << 16) + v);
            } else {
                float* op = a.part_o + (part_row + rr * a.q_heads + qh) * D + d;
                *op += v;
            }
        });
    }
}

// Joins the splits of each output row, in split order: one wave per row and 64 D/64 lanes.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a, float v_scale) {
    constexpr int kLanes = D / 4;  // four values each
    const int64_t rows = (int64_t)a.batch.tokens * a.q_heads;
    const int64_t row = (int64_t)blockIdx.x * (256 / kLanes) + (int)threadIdx.x / kLanes;
    const int d = 4 * ((int)threadIdx.x % kLanes);
    if (row >= rows) return;
    float top = kNegInf;
    for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.part_ml[s * rows + row].x);
    const float base = top == kNegInf ? 0.0f : top;
    float total = 0.0f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const float2 ml = a.part_ml[s * rows + row];
        if (ml.x == kNegInf && ml.y == 0.0f) continue;
        const float w = exp2_hw(ml.x - base);
        total += ml.y * w;
        o += *reinterpret_cast<const f32x4*>(a.part_o + (s * rows + row) * D + d) * w;
    }
    const float norm = total > 0.0f || total != total ? v_scale / total : 0.0f;
    const int64_t tok = row / a.q_heads;
    const int head = (int)(row - tok * a.q_heads);
    u32x2 w;
    w.x = pack_bf16(o[0] * norm, o[1] * norm);
    w.y = pack_bf16(o[2] * norm, o[3] * norm);
    *reinterpret_cast<u32x2*>(a.out + tok * a.out_stride + (int64_t)head * D + d) = w;
    if (a.lse != nullptr && d == 0) a.lse[row] = (top + __builtin_amdgcn_logf(total)) * kLn2;
}

template <int D, bool FP8>
hipError_t launch(const AttnArgs& a, hipStream_t stream) {
    const Shape sh = tile_shape(16, a.q_heads / a.pages.kv_heads);
    const unsigned tiles = (unsigned)(a.batch.tokens / sh.tokens + a.batch.requests + 1);
    rows16_kernel<D, FP8><<<dim3(tiles * (unsigned)(a.pages.kv_heads * sh.chunks), (unsigned)a.splits), 64 * kWaves, 0, stream>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.splits == 1) return e;
    const int64_t rows = (int64_t)a.batch.tokens * a.q_heads;
    constexpr int per = 256 / (D / 4);
    join_kernel<D><<<(unsigned)((rows + per - 1) / per), 256, 0, stream>>>(a, FP8 ? a.pages.v_scale : 1.0f);
    return hipGetLastError();
}

}  // namespace

AttnPlan plan_attention(const AttnArgs& a) {
    AttnPlan p{16, 1, 0, 0};
    const Shape sh = tile_shape(16, a.q_heads / a.pages.kv_heads);
    const int64_t wgs = ((int64_t)a.batch.tokens / sh.tokens + a.batch.requests) * a.pages.kv_heads * sh.chunks;
    int64_t keys = (int64_t)a.batch.width << a.pages.page_shift;
    if (a.window > 0 && keys > a.window + sh.tokens) keys = a.window + sh.tokens;
    // splits until the card has two workgroups per CU, each with 256 keys or more
    int64_t splits = wgs > 0 ? 512 / wgs : 1;
    if (splits > keys / 256) splits = keys / 256;
    if (splits > 128) splits = 128;
    if (splits < 1) splits = 1;
    p.splits = (int)splits;
    if (p.splits > 1) {
        const size_t rows = (size_t)p.splits * a.batch.tokens * a.q_heads;
        p.o_bytes = rows * a.pages.head_dim * 4;
        p.ml_bytes = rows * sizeof(float2);
    }
    return p;
}

hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, hipStream_t stream) {
    (void)plan;
    switch (a.pages.head_dim * 2 + a.pages.fp8) {
        case 128: return launch<64, false>(a, stream);
        case 129: return launch<64, true>(a, stream);
        case 256: return launch<128, false>(a, stream);
        case 257: return launch<128, true>(a, stream);
        case 512: return launch<256, false>(a, stream);
        case 513: return launch<256, true>(a, stream);
        case 1024: return launch<512, false>(a, stream);
        case 1025: return launch<512, true>(a, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace kv
