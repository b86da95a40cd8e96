// Attention of new tokens over a paged cache.
//
//   s_ij = scale q_i . k_j,  out_i = sum_j softmax_j(s_i) v_j,  lse_i = log sum_j exp s_ij
//
// over the keys j that row i sees (kv_index.h).  One pass over the keys with the running
// maximum m and sum l of the softmax, all in fp32; the weights exp(s - m) are rounded to
// bf16 for their product with V (matrix cores), 2^-8 of each at most: the outputs of 4096
// random keys are then 1.8e-3 off in the 2-norm (2.2e-3 from the 128-row tiles), 1.7e-3 of it
// their own rounding.  A row's largest weight is exactly 1 here, so that a row that one key
// dominates loses little; in the 128-row tiles it need not be (kv_tile.hip).  l sums the
// weights before that rounding.  e4m3 keys and values are
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
#include "kv_device.h"

namespace kv {
namespace {

constexpr int kWaves = 4;

// Workgroups of rows16 that cuts are made for: one per CU at head_dim 512, where the registers
// hold one wave per SIMD, else two.  (At 64 and 128 dims the registers would hold three or more;
// what more and shorter items do there has not been measured.)
int rows_fill(const AttnArgs& a) { return a.pages.head_dim == 512 ? 256 : 512; }
// Those of the 128-row tiles: one per CU, two of the smaller heads (registers and LDS).
int tiles_fill(const AttnArgs& a) { return a.pages.head_dim >= 256 ? 256 : 512; }

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
__global__ __launch_bounds__(64 * kWaves, D == 512 ? 1 : 2) void rows16_kernel(AttnArgs a, Items it) {
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
    const Shape sh = tile_shape(kThinRows, group);
    const int item = (int)blockIdx.x / it.parts;
    const int part = (int)blockIdx.x - item * it.parts;
    const int kv_head = part / sh.chunks, chunk = part - kv_head * sh.chunks;

    const Tile t = find_item<false>(a.batch, a.pages.page_shift, rows_cuts(a, it, sh), item, lane);
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
    const TileRange range = split_tiles(tiles, t.split, t.splits, 1);
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
    const int64_t slot = (int64_t)blockIdx.x * kThinRows;  // rows of this item's partial sums
    if (wave == 0) {
        add(0);
        if (live) {
            if (t.splits == 1) {
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
                if (g == 0) it.part_ml[slot + n] = make_float2(top, total);
                if (top != kNegInf || total != 0.0f) {
                    float* op = it.part_o + (slot + n) * D;
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
        fix_nonfinite<D, FP8>(a, t, sh, kv_head, from, upto, kGroupKeys, 64 * kWaves, [&](int i, int h, int d, float v) {
            const int ig = chunk * sh.heads + h;
            if (ig >= group) return;
            const int64_t rr = t.row0 + i;
            const int qh = kv_head * group + ig;
            if (t.splits == 1) {
                uint16_t* op = a.out + rr * a.out_stride + (int64_t)qh * D + d;
                *op = q4::f32_to_bf16(__uint_as_float((uint32_t)*op << 16) + v);
            } else {
                float* op = it.part_o + (slot + i * sh.heads + h) * D + d;
                *op += v;
            }
        });
    }
}

// Joins the items of each tile that has several; bound by the latency of its loads for few
// rows and by their bytes for many.  Sixteen lanes of four dims take a slice of 64 dims of a
// row.  Where rows fill the card (`many`) or a tile has eight items at most, one such group
// sums a slice's items; else they are dealt to the workgroup's sixteen groups, whose sums
// meet in LDS.  Either way always in the same order.
template <int D>
__global__ __launch_bounds__(256) void join_kernel(AttnArgs a, Items it, Cuts cuts, int rows, int many) {
    constexpr int kSets = 16, kSlices = D / 64;
    __shared__ f32x4 sums[kSets][16];
    __shared__ float totals[kSets];
    const int lane = (int)threadIdx.x & 63;
    const int set = (int)threadIdx.x / 16, d4 = 4 * ((int)threadIdx.x % 16);
    const int group = a.q_heads / a.pages.kv_heads;
    const Shape sh = tile_shape(rows, group);
    const int tile_no = (int)blockIdx.x / it.parts;
    const int part = (int)blockIdx.x - tile_no * it.parts;
    const int kv_head = part / sh.chunks, chunk = part - kv_head * sh.chunks;
    const Tile t = find_item<true>(a.batch, a.pages.page_shift, cuts, tile_no, lane);
    if (t.n <= 0 || t.splits < 2 || t.first_item < 0 || t.first_item + t.splits > it.items) return;
    const float v_scale = a.pages.fp8 ? a.pages.v_scale : 1.0f;
    const int64_t step = (int64_t)it.parts * rows;  // partial rows from one item to the next
    const int work = t.n * sh.heads * kSlices;
    const int heads_here = group - chunk * sh.heads < sh.heads ? group - chunk * sh.heads : sh.heads;
    const auto first_of = [&](int r) { return ((int64_t)t.first_item * it.parts + part) * rows + r; };
    const auto store = [&](int r, int d, f32x4 o, float top, float total) {
        const float norm = total > 0.0f || total != total ? v_scale / total : 0.0f;
        const int tok = r / sh.heads;
        const int64_t row = t.row0 + tok;
        const int head = kv_head * group + chunk * sh.heads + r - tok * sh.heads;
        *reinterpret_cast<u32x2*>(a.out + row * a.out_stride + (int64_t)head * D + d) =
            u32x2{pack_bf16(o[0] * norm, o[1] * norm), pack_bf16(o[2] * norm, o[3] * norm)};
        if (a.lse != nullptr && d == 0) a.lse[row * a.q_heads + head] = (top + __builtin_amdgcn_logf(total)) * kLn2;
    };

    if (many || t.splits <= 8) {
        for (int w = (int)blockIdx.y * kSets + set; w < work; w += (int)gridDim.y * kSets) {
            const int r = w / kSlices, d = 64 * (w % kSlices) + d4;
            if (r % sh.heads >= heads_here) continue;
            const int64_t first = first_of(r);
            float top = kNegInf, total = 0.0f;
            f32x4 o = {0.f, 0.f, 0.f, 0.f};
            for (int s0 = 0; s0 < t.splits; s0 += 8) {
                float2 ml[8];
                f32x4 v[8];
                float next = top;
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    const int64_t at = first + (s0 + s < t.splits ? s0 + s : s0) * step;
                    ml[s] = it.part_ml[at];
                    v[s] = *reinterpret_cast<const f32x4*>(it.part_o + at * D + d);
                    next = fmaxf(next, ml[s].x);
                }
                const float base = next == kNegInf ? 0.0f : next, scale = __builtin_amdgcn_exp2f(top - base);
                total *= scale;
                o *= scale;
#pragma unroll
                for (int s = 0; s < 8; ++s) {
                    const bool any = s0 + s < t.splits && (ml[s].x != kNegInf || ml[s].y != 0.0f);  // else the item left nothing there
                    const float e = __builtin_amdgcn_exp2f(ml[s].x - base);
                    total += any ? ml[s].y * e : 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[i] += any ? v[s][i] * e : 0.0f;
                }
                top = next;
            }
            store(r, d, o, top, total);
        }
        return;
    }
    for (int w = (int)blockIdx.y; w < work; w += (int)gridDim.y) {
        const int r = w / kSlices, d = 64 * (w % kSlices) + d4;
        if (r % sh.heads >= heads_here) continue;
        const int64_t first = first_of(r);
        float top = kNegInf;
        for (int s = lane; s < t.splits; s += 64) top = fmaxf(top, it.part_ml[first + s * step].x);
        top = wave_max(top);
        const float base = top == kNegInf ? 0.0f : top;
        float total = 0.0f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
        for (int s = set; s < t.splits; s += kSets) {
            const float2 ml = it.part_ml[first + s * step];
            const f32x4 v = *reinterpret_cast<const f32x4*>(it.part_o + (first + s * step) * D + d);
            const bool any = ml.x != kNegInf || ml.y != 0.0f;
            const float e = __builtin_amdgcn_exp2f(ml.x - base);
            total += any ? ml.y * e : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] += any ? v[i] * e : 0.0f;
        }
        __syncthreads();  // the sums of the row before are read
        sums[set][d4 / 4] = o;
        if (d4 == 0) totals[set] = total;
        __syncthreads();
        if (set == 0) {
            for (int s = 1; s < kSets; ++s) {
                o += sums[s][d4 / 4];
                total += totals[s];
            }
            store(r, d, o, top, total);
        }
    }
}

template <int D, bool FP8>
hipError_t launch_rows(const AttnArgs& a, const Items& it, hipStream_t stream) {
    rows16_kernel<D, FP8><<<(unsigned)it.items * (unsigned)it.parts, 64 * kWaves, 0, stream>>>(a, it);
    return hipGetLastError();
}

hipError_t launch_rows16(const AttnArgs& a, const Items& it, hipStream_t stream) {
    switch (a.pages.head_dim * 2 + a.pages.fp8) {
        case 128: return launch_rows<64, false>(a, it, stream);
        case 129: return launch_rows<64, true>(a, it, stream);
        case 256: return launch_rows<128, false>(a, it, stream);
        case 257: return launch_rows<128, true>(a, it, stream);
        case 512: return launch_rows<256, false>(a, it, stream);
        case 513: return launch_rows<256, true>(a, it, stream);
        case 1024: return launch_rows<512, false>(a, it, stream);
        case 1025: return launch_rows<512, true>(a, it, stream);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_join(const AttnArgs& a, const Items& it, const Cuts& cuts, int rows, hipStream_t stream) {
    if (it.slots == 0) return hipSuccess;
    const int tiles = (it.items - it.slots) * it.parts;
    // slices of 64 dims, of a tile and in all: sixteen a workgroup if they are many
    const int group = a.q_heads / a.pages.kv_heads, heads = group < rows ? group : rows, slices = a.pages.head_dim / 64;
    const int64_t live = (int64_t)a.batch.tokens * heads;
    const int work = (int)(live < rows ? live : rows) * slices;
    const bool many = (int64_t)a.batch.tokens * a.q_heads * slices >= 2048;
    const int most = many ? ceil_div(work, 16) : work, fill = ceil_div(2048, tiles);
    const int y = most < fill ? most : fill;
    const dim3 grid((unsigned)tiles, (unsigned)y);
    switch (a.pages.head_dim) {
        case 64: join_kernel<64><<<grid, 256, 0, stream>>>(a, it, cuts, rows, many); break;
        case 128: join_kernel<128><<<grid, 256, 0, stream>>>(a, it, cuts, rows, many); break;
        case 256: join_kernel<256><<<grid, 256, 0, stream>>>(a, it, cuts, rows, many); break;
        case 512: join_kernel<512><<<grid, 256, 0, stream>>>(a, it, cuts, rows, many); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

// The most tiles that runs of least..most rows can make (the padding is a run too).
int most_tiles(const AttnArgs& a, int tokens, int least, int most) {
    return kv::most_tiles(a.batch.tokens, (int64_t)a.batch.requests + 1, tokens, least, most);
}

// The most keys a tile of `tokens` can see.
int64_t most_keys(const AttnArgs& a, int tokens) {
    const int64_t keys = (int64_t)a.batch.width << a.pages.page_shift;
    return a.window > 0 && keys > a.window + tokens ? a.window + tokens : keys;
}

// Items of a kernel's rows: `fill` workgroups fill the card.  No cuts where the tiles alone
// fill it, or where no tile has keys for two items of `least_keys`.
Items plan_items(const AttnArgs& a, const Shape& sh, int tiles, int fill, int least_keys) {
    Items it{};
    it.parts = a.pages.kv_heads * sh.chunks;
    const int64_t keys = most_keys(a, sh.tokens);
    const int slots = fill / it.parts;
    it.slots = tiles < slots && keys >= 2 * least_keys ? slots : 0;
    it.items = it.slots + tiles;
    return it;
}

}  // namespace

AttnPlan plan_attention(const AttnArgs& a) {
    AttnPlan p{};
    const int group = a.q_heads / a.pages.kv_heads;
    const int64_t tokens = a.batch.tokens, requests = a.batch.requests;
    const Shape wide = tile_shape(kWideRows, group), thin = tile_shape(kThinRows, group);
    // A request goes to the 128-row tiles if it has 64 rows (96 of 64 dims): us of 16-row and of
    // 128-row tiles, four requests of 32768 keys, 512 dims: 65 / 82 at 32 rows, 101 / 84 at 64;
    // 256 dims: 222 / 223 and 363 / 227; 128 dims: 86 / 102 at 48, 154 / 101 at 96; 64 dims:
    // 54 / 71 at 64, 95 / 70 at 128.  In a call of little work (rows x keys x dims under 8e8) the
    // wide tiles' start costs more than they save: one request of 4096 keys, 512 dims, 256 rows
    // (5e8) 33 / 39, eight of 128 rows (2e9) 60 / 48; 256 dims, window 1024, one of 128 tokens
    // (6e8) 26.8 / 27.5; 64 dims, eight of 64 rows (5e8) 22 / 27, of 128 (1.1e9) 32 / 28.
    const int from = ceil_div(a.pages.head_dim == 64 ? 96 : 64, wide.heads);
    const double work = (double)tokens * a.q_heads * (double)most_keys(a, wide.tokens) * a.pages.head_dim;
    // One request: its kernel is known.  Several with a row each at least: none reaches
    // `from` rows if the sum stays under this (were some of them empty, the 16-row kernel
    // would still be right).
    if (a.kernel == 2 || (a.kernel == 0 && work < 8e8))
        p.tile_from = kNoTiles;
    else if (requests == 1)
        p.tile_from = tokens >= from ? 1 : kNoTiles;
    else
        p.tile_from = tokens >= from + requests - 1 ? from : kNoTiles;
    p.use_rows = p.tile_from > 1;
    p.use_tiles = p.tile_from != kNoTiles;
    if (p.use_tiles) p.tiles = plan_items(a, wide, most_tiles(a, wide.tokens, p.tile_from, kNoTiles), tiles_fill(a), kTileLeast);
    if (p.use_rows) p.rows = plan_items(a, thin, most_tiles(a, thin.tokens, 1, p.tile_from - 1), rows_fill(a), kRowsLeast);
    return p;
}

hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, hipStream_t stream) {
    const int group = a.q_heads / a.pages.kv_heads;
    hipError_t e = hipSuccess;
    if (plan.use_tiles) e = launch_tiles(a, plan.tiles, stream);
    if (plan.use_rows && e == hipSuccess) e = launch_rows16(a, plan.rows, stream);
    if (plan.use_tiles && e == hipSuccess)
        e = launch_join(a, plan.tiles, tile_cuts(a, plan.tiles, tile_shape(kWideRows, group)), kWideRows, stream);
    if (plan.use_rows && e == hipSuccess)
        e = launch_join(a, plan.rows, rows_cuts(a, plan.rows, tile_shape(kThinRows, group)), kThinRows, stream);
    return e;
}

}  // namespace kv
