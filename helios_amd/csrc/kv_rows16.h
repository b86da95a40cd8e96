// The 16-row attention tiles' device code; the formulas and the layout are in kv_attention.hip.
#pragma once

#include "kv_device.h"

namespace kv {
namespace {

constexpr int kWaves = 4;

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

// `from`: nothing, or where the pages' values have their scales (BlockScales; FP8 only).
template <int D, bool FP8, class... From>
__global__ __launch_bounds__(64 * kWaves, D == 512 ? 1 : 2) void rows16_kernel(AttnArgs a, Items it, From... from) {
    using C = Rows16<D, FP8>;
    constexpr bool kScaled = sizeof...(From) > 0;
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

    // A tile of this wave's: its groups' first keys, whether they have pages, their scales (kScaled)
    // and where they lie.
    struct Groups {
        int first_key[NG];
        bool there[NG];
        float k_by[NG], v_by[NG];
        int64_t off[NG];
    };
    int pages[NG];
    uint32_t scales[NG];
    const auto fetch_pages = [&](int ti) {
        // the table entries of this wave's next 64 tiles, one per lane
        const int tl = ti + lane * kWaves;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const int at = (lo + tl * kTileKeys + j * kGroupKeys) >> a.pages.page_shift;
            pages[j] = tl < range.last ? page_at(table, at, a.batch.width, a.pages.num_pages) : -1;
        }
        if constexpr (kScaled)
#pragma unroll
            for (int j = 0; j < NG; ++j)
                scales[j] = scale_bytes(scales_of(from...), pages[j], kv_head,
                                        (uint32_t)(lo + tl * kTileKeys + j * kGroupKeys) & ((1u << a.pages.page_shift) - 1u));
    };
    const auto find = [&](int i, int ti, Groups& at) {
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const int key = lo + ti * kTileKeys + j * kGroupKeys;
            const int page = __builtin_amdgcn_readlane(pages[j], i & 63);
            at.first_key[j] = key;
            at.there[j] = page >= 0;
            at.off[j] = ((int64_t)(at.there[j] ? page : 0) * a.pages.page_stride + (int64_t)kv_head * a.pages.head_stride +
                         (int64_t)(key & ((1 << a.pages.page_shift) - 1)) * a.pages.token_stride) * C::kElt;
        }
    };
    const auto find_scales = [&](int i, Groups& at) {
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const int both = kScaled ? __builtin_amdgcn_readlane((int)scales[j], i & 63) : 0;
            at.k_by[j] = kScaled ? scale_value(both & 0xFF) : 1.0f;
            at.v_by[j] = kScaled ? scale_value(both >> 8) : 1.0f;
        }
    };
    u32x4 kf[NG][C::kChunks];
    uint32_t vf[NG][4][C::kBlocks][C::kVWords];
    const auto load_k = [&](const Groups& at, int j) {
        const char* kp = a.pages.k + at.off[j];
#pragma unroll
        for (int s = 0; s < C::kChunks; ++s)
            kf[j][s] = *reinterpret_cast<const u32x4*>(kp + k_lane + 64u * s);
    };
    const auto load_v = [&](const Groups& at, int j) {
        const char* vp = a.pages.v + at.off[j];
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int b = 0; b < C::kBlocks; ++b)
#pragma unroll
                for (int w = 0; w < C::kVWords; ++w)
                    vf[j][k][b][w] = reinterpret_cast<const uint32_t*>(
                        vp + v_lane + (uint32_t)k * row_bytes + (uint32_t)(b * 16 * C::kEpl * C::kElt))[w];
    };
    // Infinities and NaN of group j's V, where some row does not see all of it.
    const auto clear_v = [&](int j) {
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
    };

    Groups cur, nxt;
    if (kScaled && range.first + wave < range.last) {
        // The next tile's K loads go out when this one's have been used, its V loads likewise, so that
        // a wave always has some on their way (32 single tokens over up to 16000 keys of 512 dims: 49.5
        // us -> 45.8; 64 over 1024 keys of 256, where a workgroup has 8 tiles a wave, 49 either way).
        // Two groups a tile at 512 dims: 47.8.
        fetch_pages(range.first + wave);
        find(0, range.first + wave, cur);
#pragma unroll
        for (int j = 0; j < NG; ++j) load_k(cur, j);
#pragma unroll
        for (int j = 0; j < NG; ++j) load_v(cur, j);
        find_scales(0, cur);
    }
    for (int i = 0, ti = range.first + wave; ti < range.last; ++i, ti += kWaves) {
        const bool more = ti + kWaves < range.last;
        if constexpr (!kScaled) {
            if ((i & 63) == 0) fetch_pages(ti);
            find(i, ti, cur);
#pragma unroll
            for (int j = 0; j < NG; ++j) {
                load_k(cur, j);
                load_v(cur, j);
            }
            find_scales(i, cur);
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
                    kk = u32x4{e4m3_to_bf16<false>(w0, cur.k_by[j]), e4m3_to_bf16<true>(w0, cur.k_by[j]), e4m3_to_bf16<false>(w1, cur.k_by[j]),
                               e4m3_to_bf16<true>(w1, cur.k_by[j])};
                } else {
                    kk = kf[j][st];
                }
                s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kk), __builtin_bit_cast(bf16x8, q[st]), s, 0, 0, 0);
            }
            const bool masked = !cur.there[j] || !all_visible(cur.first_key[j], kGroupKeys, t.pos0, t.n, a.window);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[j][r] = s[r] * c;
            if (masked) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = cur.first_key[j] + 4 * g + r;
                    x[j][r] = cur.there[j] && key <= pos && key > above ? x[j][r] : kNegInf;
                }
                if (!kScaled) clear_v(j);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) top = fmaxf(top, x[j][r]);
        }
        if (kScaled && more) {
            if ((i & 63) == 63) fetch_pages(ti + kWaves);
            find(i + 1, ti + kWaves, nxt);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < NG; ++j) load_k(nxt, j);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (kScaled)
#pragma unroll
            for (int j = 0; j < NG; ++j)
                if (!cur.there[j] || !all_visible(cur.first_key[j], kGroupKeys, t.pos0, t.n, a.window)) clear_v(j);
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
                            const u32x2 av = {e4m3_to_bf16<false>(four, cur.v_by[j]), e4m3_to_bf16<true>(four, cur.v_by[j])};
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
        if (kScaled && more) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < NG; ++j) load_v(nxt, j);
            find_scales(i + 1, nxt);
            cur = nxt;
            __builtin_amdgcn_sched_barrier(0);
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

}  // namespace
}  // namespace kv
