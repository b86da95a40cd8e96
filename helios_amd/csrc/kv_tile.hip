// Attention of many new tokens over a paged cache: 128 query rows (tokens x heads that
// share a KV head) per workgroup.
//
// The formulas, the softmax and the masked places are those of kv_attention.hip.  With 128
// rows per key the work is bound by the matrix cores (a key's 2 D bytes of K and V feed
// 4 x 128 x D operations), so the layout is chosen to keep them fed from one wave per SIMD:
//
//   S^T = K Q^T (32x32x16, A = K): wave w holds rows 32w..32w+31 of Q in registers and
//   reads each 32-key tile of K from LDS.  Lane (n = l % 32, h = l / 32) gets s of row n
//   and keys 8b + 4h + r (b, r < 4), so a row's maximum needs one exchange of two lanes.
//   O^T += V^T P^T (32x32x16, A = V^T): the waves divide the dims of V, not the rows: the
//   softmax weights go to the other waves through LDS (8 KiB a tile, in the B operand's own
//   order), and each wave reads only its slice of V, straight from memory into registers,
//   once for all the rows.  The order of keys within a product is free, so A's lane (dim,
//   h) takes the keys whose weights lane (row, h) has, in that order; a lane loads E
//   consecutive dims of each of its keys and transposes them by byte permutes.
//
// Each wave holding all dims of its own 32 rows instead would read K and V from LDS for
// every 32 rows: 156 B a cycle at the matrix cores' full rate (head_dim 512), where LDS
// gives 128; this split asks for 98.
//
// One barrier per tile: before it tile i's weights are written and tile i + 1's scores are
// computed from LDS (the softmax of tile i between their products); after it the DMA of
// K tile i + 3 starts in the buffer just read, and the waves multiply tile i's weights by V.
// The running maximum of a row is raised only when a score exceeds it by 2^8: weights up to
// 2^8 lose nothing in bf16 or in the fp32 sums, and the outputs (256 registers at head_dim
// 512) are seldom rescaled.
#include "kv_device.h"

namespace kv {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kTileKeys = 32;
constexpr int kTileWaves = 4;
constexpr float kSlack = 8.0f;  // how far a score may exceed the running maximum (log2)

template <int D, bool FP8>
struct TileConf {
    static constexpr int kElt = FP8 ? 1 : 2;
    static constexpr int kSlices = D == 512 ? 4 : (D == 64 ? 1 : 2);  // dim slices
    static constexpr int kGroups = kSlices;                           // 32-row groups of a wave's outputs
    static constexpr int kSliceDims = D / kSlices;
    static constexpr int kE = kSliceDims / 32;                        // consecutive dims of a lane
    static constexpr int kRowBytes = D * kElt;
    static constexpr int kCpr = kRowBytes / 16;                       // 16-byte chunks of a K row
    static constexpr int kSteps = D / 16;
    static constexpr int kDmaKeys = 1024 / kRowBytes;                 // keys of one DMA
    static constexpr int kDmas = kTileKeys / kDmaKeys;                // DMAs of a tile
    static constexpr int kTileBytes = kTileKeys * kRowBytes;
};

// K rows lie in LDS as they do in memory, their 16-byte chunks permuted by xor with
// swizzle(key): 32 lanes reading the same chunk of 32 keys then spread over the banks.
template <int CPR>
__device__ __forceinline__ int swizzle(int key) {
    constexpr int per = CPR >= 16 ? 1 : 16 / CPR;
    constexpr int mask = CPR >= 16 ? 15 : CPR - 1;
    return (key / per) & mask;
}

__device__ __forceinline__ f32x16 mfma32(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// o[e] += av[e] x p for the E products of a row group, accumulators in AGPRs: with the builtin
// the compiler keeps accumulators either all in VGPRs or, S among them, all in AGPRs, and
// neither holds 256 of O beside the rest.  It sees no hazards in asm: the leading wait states
// cover operands the VALU has just written, and mfma_settled() goes between these products
// and the next VALU access to o.
template <int E>
__device__ __forceinline__ void mfma_acc(f32x16 (&o)[E], const u32x4 (&av)[E], u32x4 p) {
    static_assert(E == 2 || E == 4, "two or four products");
    if constexpr (E == 4) {
        asm("s_nop 1\n\t"
            "v_mfma_f32_32x32x16_bf16 %0, %4, %8, %0\n\t"
            "v_mfma_f32_32x32x16_bf16 %1, %5, %8, %1\n\t"
            "v_mfma_f32_32x32x16_bf16 %2, %6, %8, %2\n\t"
            "v_mfma_f32_32x32x16_bf16 %3, %7, %8, %3"
            : "+a"(o[0]), "+a"(o[1]), "+a"(o[2]), "+a"(o[3])
            : "v"(av[0]), "v"(av[1]), "v"(av[2]), "v"(av[3]), "v"(p));
    } else {
        asm("s_nop 1\n\t"
            "v_mfma_f32_32x32x16_bf16 %0, %2, %4, %0\n\t"
            "v_mfma_f32_32x32x16_bf16 %1, %3, %4, %1\n\t"
            "s_nop 1"
            : "+a"(o[0]), "+a"(o[1])
            : "v"(av[0]), "v"(av[1]), "v"(p));
    }
}
__device__ __forceinline__ void mfma_settled(f32x16& o) { asm volatile("s_nop 15\n\ts_nop 15" : "+a"(o)); }

__device__ __forceinline__ float half_max(float v) {
    const u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
}
__device__ __forceinline__ float half_sum(float v) {
    const u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p.x) + __uint_as_float(p.y);
}

// The E values of one key a lane holds, as words (E * kElt = 2, 4 or 8 bytes).
template <int BYTES>
struct VWords {
    static constexpr int kCount = BYTES == 8 ? 2 : 1;
    uint32_t w[kCount];
};
template <int BYTES>
__device__ __forceinline__ VWords<BYTES> load_v(__amdgpu_buffer_rsrc_t r, uint32_t lane_off, uint32_t off) {
    VWords<BYTES> v;
    if constexpr (BYTES == 2) {
        v.w[0] = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(r, (int)lane_off, (int)off, 0);
    } else if constexpr (BYTES == 4) {
        v.w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)lane_off, (int)off, 0);
    } else {
        const u32x2 t = __builtin_amdgcn_raw_buffer_load_b64(r, (int)lane_off, (int)off, 0);
        v.w[0] = t.x;
        v.w[1] = t.y;
    }
    return v;
}

// bf16 pair (dim E of key a, dim E of key b)
template <bool FP8, int BYTES, int E>
__device__ __forceinline__ uint32_t pair_of(const VWords<BYTES>& a, const VWords<BYTES>& b) {
    if constexpr (FP8) {
        const uint32_t both = __builtin_amdgcn_perm(b.w[0], a.w[0], E < 2 ? 0x05010400u : 0x07030602u);
        return e4m3_to_bf16<(E & 1) != 0>(both);
    } else {
        return __builtin_amdgcn_perm(b.w[E / 2], a.w[E / 2], (E & 1) ? 0x07060302u : 0x05040100u);
    }
}

struct TileShared {
    float alpha[2][128];
    uint32_t raised[2][kTileWaves];
    float m[128], l[128];
    uint32_t found[kTileWaves];
};

template <int D, bool FP8>
__global__ __launch_bounds__(64 * kTileWaves, 1) void tile_kernel(AttnArgs a, Items it) {
    using C = TileConf<D, FP8>;
    constexpr int E = C::kE, RG = C::kGroups;
    constexpr int kVBytes = E * C::kElt;
    __shared__ alignas(1024) uint4 kbuf[2][C::kTileBytes / 16];
    __shared__ u32x4 pbuf[2][kTileWaves][2][64];
    __shared__ TileShared sm;

    const int lane = (int)threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int n = lane & 31, h = lane >> 5;
    const int group = a.q_heads / a.pages.kv_heads;
    const Shape sh = tile_shape(kWideRows, group);
    const int item = (int)blockIdx.x / it.parts;
    const int part = (int)blockIdx.x - item * it.parts;
    const int kv_head = part / sh.chunks, chunk = part - kv_head * sh.chunks;

    const Tile t = find_item<false>(a.batch, a.pages.page_shift, tile_cuts(a, it, sh), item, lane);
    if (t.n <= 0) return;
    const int kv_len = clampi(t.kv_len, 0, a.batch.width << a.pages.page_shift);

    // this lane's query row
    const int tile_row = 32 * wave + n;
    const int tok = tile_row / sh.heads, hh = tile_row - tok * sh.heads;
    const int in_group = chunk * sh.heads + hh;
    const bool live = tok < t.n && in_group < group;
    const int row = t.row0 + (live ? tok : 0);
    const int q_head = kv_head * group + (live ? in_group : 0);
    const int pos = live ? t.pos0 + tok : t.pos0;
    const int above = a.window > 0 ? pos - a.window : -0x7fffffff;  // keys in (above, pos]

    // The scale's sign goes into Q, so that the largest product is the largest score.  A scale
    // of zero makes every score zero (or NaN) in Q already.
    const float c = a.scale == 0.0f ? 1.0f : fabsf(a.scale) * (FP8 ? a.pages.k_scale : 1.0f) * kLog2e;
    u32x4 q[C::kSteps];
    {
        const uint16_t* qp = a.q + (int64_t)row * a.q_stride + (int64_t)q_head * D;
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
        const uint32_t keep = live && a.scale != 0.0f ? ~0u : 0u;
#pragma unroll
        for (int s = 0; s < C::kSteps; ++s) {
            // the dims of the K chunk that step s uses in lane half h
            const int d = FP8 ? 32 * (s / 2) + 16 * h + 8 * (s & 1) : 16 * s + 8 * h;
            q[s] = (*reinterpret_cast<const u32x4*>(qp + d) ^ flip) & keep;
        }
    }

    const KeyRange keys = visible_keys(t.pos0, t.n, kv_len, a.window);
    const int lo = keys.lo & ~(kTileKeys - 1);
    const int tiles = keys.hi > lo ? ceil_div(keys.hi - lo, kTileKeys) : 0;
    const TileRange range = split_tiles(tiles, t.split, t.splits, 1);
    const int count = range.last - range.first;
    const int key0 = lo + range.first * kTileKeys;
    const int* table = a.batch.tables + (int64_t)t.request * a.batch.stride;
    const uint32_t row_bytes = (uint32_t)a.pages.token_stride * C::kElt;

    // Pages of the 16-key groups of 32 tiles, one per lane: chunk j of 64 groups in page_at_[j & 1].
    const auto fetch_pages = [&](int ch) {
        const int g = 64 * ch + lane;
        const int at = (key0 + g * kGroupKeys) >> a.pages.page_shift;
        return g < 2 * count ? page_at(table, at, a.batch.width, a.pages.num_pages) : -1;
    };
    int pages_even = fetch_pages(0), pages_odd = fetch_pages(1);
    const auto page_of = [&](int g) {
        const int v = ((g >> 6) & 1) ? pages_odd : pages_even;
        return __builtin_amdgcn_readlane(v, g & 63);
    };
    // bytes from this head's first page to the first of the 16 keys of group g
    const uint64_t page_bytes = (uint64_t)a.pages.page_stride * C::kElt;
    const int64_t head_bytes = (int64_t)kv_head * a.pages.head_stride * C::kElt;
    const char* const k_head = a.pages.k + head_bytes;
    const char* const v_head = a.pages.v + head_bytes;
    const uint32_t slot_mask = (1u << a.pages.page_shift) - 1u;
    const auto group_offset = [&](int g) {
        const int page = page_of(g);
        return (uint32_t)(page < 0 ? 0 : page) * page_bytes + (uint64_t)((uint32_t)(key0 + g * kGroupKeys) & slot_mask) * row_bytes;
    };

    const uint32_t group_bytes = 15u * row_bytes + (uint32_t)C::kRowBytes;
    // K tile `tl` into buffer tl & 1; each DMA brings kDmaKeys whole rows
    const auto dma_k = [&](int tl) {
        int ln = lane;
        asm volatile("" : "+v"(ln));  // offsets are cheap to make again and dear to keep
        const int dma_key = ln / C::kCpr, dma_chunk = ln & (C::kCpr - 1);
#pragma unroll
        for (int j = 0; j < (C::kDmas + kTileWaves - 1) / kTileWaves; ++j) {
            const int d = wave * ((C::kDmas + kTileWaves - 1) / kTileWaves) + j;
            if (C::kDmas >= kTileWaves || d < C::kDmas) {
                const int first = d * C::kDmaKeys;  // key within the tile
                const int g = 2 * tl + first / kGroupKeys;
                const __amdgpu_buffer_rsrc_t r = q4::make_rsrc(k_head + group_offset(g), group_bytes);
                const uint32_t voff = (uint32_t)dma_key * row_bytes + 16u * (uint32_t)(dma_chunk ^ swizzle<C::kCpr>(first + dma_key));
                q4::dma16(r, &kbuf[tl & 1][d * 64], voff, (uint32_t)(first % kGroupKeys) * row_bytes);
            }
        }
    };

    // This lane's reads of K: key n's chunk 2u + h, at its row + 16 ((2u + h) ^ swizzle(n)).  The
    // low four bits of 2u go in by xor, the rest as an offset; steps that share those bits
    // follow each other, so that few addresses are alive.
    constexpr int kUnits = C::kCpr / 2, kFar = C::kCpr > 16 ? C::kCpr / 16 : 1, kPer = FP8 ? 2 : 1;
    typedef const __attribute__((address_space(3))) u32x4* LdsPtr;
    const uint32_t k_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)(const void*)&kbuf[0][0] +
                            (uint32_t)n * C::kRowBytes + 16u * (uint32_t)(h ^ swizzle<C::kCpr>(n));
    const auto unit_of = [](int i) { return i / kFar + 8 * (i % kFar); };
    const auto read_k = [&](uint32_t base, int u) {
        return *((LdsPtr)(uintptr_t)(base ^ (16u * (uint32_t)((2 * u) & 15))) + (2 * u) / 16 * 16);
    };
    // s += the products of unit u
    const auto product = [&](f32x16 s, int u, u32x4 raw) {
        if constexpr (FP8) {
            const u32x4 k0 = {e4m3_to_bf16<false>(raw.x), e4m3_to_bf16<true>(raw.x), e4m3_to_bf16<false>(raw.y), e4m3_to_bf16<true>(raw.y)};
            const u32x4 k1 = {e4m3_to_bf16<false>(raw.z), e4m3_to_bf16<true>(raw.z), e4m3_to_bf16<false>(raw.w), e4m3_to_bf16<true>(raw.w)};
            return mfma32(k1, q[kPer * u + kPer - 1], mfma32(k0, q[kPer * u], s));
        } else {
            return mfma32(raw, q[u], s);
        }
    };

    const int slice = wave % C::kSlices;
    const int rg0 = wave / C::kSlices * RG;  // first row group of this wave's outputs
    const uint32_t v_lane = 4u * h * row_bytes + (uint32_t)((slice * C::kSliceDims + n * E) * C::kElt);

    f32x16 o[RG][E];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
        for (int e = 0; e < E; ++e) o[rg][e] = f32x16{};
    float m = kNegInf, l = 0.0f;
    bool nonfinite = false;

    // The tile's scores in `s`: masks them, if some row does not see all of its keys, and
    // raises the running maximum, if a score exceeds it by more than kSlack (the wave's sums
    // here, the outputs when the weights are used).
    struct Seen {
        bool visible, there[2];
    };
    const auto seen_of = [&](int tl) {
        Seen v;
        v.visible = all_visible(key0 + tl * kTileKeys, kTileKeys, t.pos0, t.n, a.window);
        v.there[0] = page_of(2 * tl) >= 0;
        v.there[1] = page_of(2 * tl + 1) >= 0;
        return v;
    };
    const auto top_of = [&](const f32x16& s) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        return half_max(top) * c;
    };
    const auto settle = [&](int tl, f32x16& s, float top, const Seen& seen) {
        if (!seen.visible || !seen.there[0] || !seen.there[1]) {
            int first = key0 + tl * kTileKeys + 4 * h;
            asm volatile("" : "+v"(first));
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = first + 8 * (i / 4) + i % 4;
                s[i] = seen.there[i / 8] && key <= pos && key > above ? s[i] : kNegInf;
            }
            top = top_of(s);
        }
        uint32_t raised = 0;
        if (__any(top > m + kSlack)) {
            const float next = fmaxf(m, top);
            const float alpha = __builtin_amdgcn_exp2f(m - (next == kNegInf ? 0.0f : next));
            m = next;
            l *= alpha;
            if (h == 0) sm.alpha[tl & 1][tile_row] = alpha;
            raised = 1;
        }
        if (lane == 0) sm.raised[tl & 1][wave] = raised;
    };

    f32x16 s_cur = {};
    Seen seen = {};
    if (count > 0) {
        dma_k(0);
        if (count > 1) dma_k(1);
        q4::wait_vm_lds<0>();
        q4::lds_barrier();
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // or all reads move ahead, into registers Q needs
            s_cur = product(s_cur, unit_of(i), read_k(k_base, unit_of(i)));
        }
        seen = seen_of(0);
        settle(0, s_cur, top_of(s_cur), seen);
        q4::wait_lds();
        q4::lds_barrier();
        if (count > 2) dma_k(2);
    }

    for (int tl = 0; tl < count; ++tl) {
        if ((tl & 31) == 0 && tl > 0) {
            if ((tl >> 5) & 1)
                pages_even = fetch_pages((tl >> 5) + 1);
            else
                pages_odd = fetch_pages((tl >> 5) + 1);
        }
        const int par = tl & 1;
        // The next tile's scores; between their products the loads of this tile's V and this
        // tile's weights (the order is the source's: slices end in scheduling barriers).
        VWords<kVBytes> v[2][8];
        const __amdgpu_buffer_rsrc_t vr[2] = {q4::make_rsrc(v_head + group_offset(2 * tl), group_bytes),
                                              q4::make_rsrc(v_head + group_offset(2 * tl + 1), group_bytes)};
        f32x16 s_next = {};
        const float base = m == kNegInf ? 0.0f : m;
        float last = 0.0f;
        u32x4 pk = {};
        uint32_t kb = k_base + (uint32_t)((tl + 1) & 1) * (uint32_t)C::kTileBytes;
        asm volatile("" : "+v"(kb));
        constexpr int kAhead = kUnits < 4 ? kUnits : 4;
        u32x4 kf[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) kf[i] = read_k(kb, unit_of(i));
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            s_next = product(s_next, unit_of(i), kf[i % kAhead]);
            if (i + kAhead < kUnits) kf[i % kAhead] = read_k(kb, unit_of(i + kAhead));
#pragma unroll
            for (int j = 16 * i / kUnits; j < 16 * (i + 1) / kUnits; ++j)
                v[j / 8][j % 8] = load_v<kVBytes>(vr[j / 8], v_lane, (uint32_t)(8 * (j % 8 / 4) + j % 4) * row_bytes);
#pragma unroll
            for (int e = 16 * i / kUnits; e < 16 * (i + 1) / kUnits; ++e) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s_cur[e], c, -base));
                l += w;
                if (e & 1)
                    pk[e / 2 % 4] = pack_bf16(last, w);
                last = w;
                if (e % 8 == 7) pbuf[par][wave][e / 8][lane] = pk;
            }
        }
        __builtin_amdgcn_sched_barrier(0);

        // K of tile tl + 2 has landed (its DMAs are older than the 16 loads of V) and the
        // weights are written
        q4::wait_vm_lds<16>();
        q4::lds_barrier();

        if (!seen.visible || !seen.there[0] || !seen.there[1]) {
#pragma unroll
            for (int st = 0; st < 2; ++st) {
                if (seen.visible && seen.there[st]) continue;
                bool bad = false;
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int w = 0; w < VWords<kVBytes>::kCount; ++w) bad |= any_nonfinite<FP8>(v[st][j].w[w]);
                if (__any(bad)) {
                    nonfinite = true;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int w = 0; w < VWords<kVBytes>::kCount; ++w) v[st][j].w[w] = finite_only<FP8>(v[st][j].w[w]);
                }
            }
        }

        const uint32_t up = sm.raised[par][lane & (kTileWaves - 1)];
        if (__any(up != 0)) {
#pragma unroll
            for (int rg = 0; rg < RG; ++rg) {
                if (__builtin_amdgcn_readlane(up, rg0 + rg) != 0) {
                    const float f = sm.alpha[par][32 * (rg0 + rg) + n];
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        mfma_settled(o[rg][e]);
                        o[rg][e] *= f;
                        mfma_settled(o[rg][e]);
                        __builtin_amdgcn_sched_barrier(0);  // one at a time: they pass through VGPRs
                    }
                }
            }
        }

        // this tile's products, the next one's maximum between them
        const auto transposed = [&](int st, int j, u32x4 (&av)[E]) {
            av[0][j] = pair_of<FP8, kVBytes, 0>(v[st][2 * j], v[st][2 * j + 1]);
            av[1][j] = pair_of<FP8, kVBytes, 1>(v[st][2 * j], v[st][2 * j + 1]);
            if constexpr (E == 4) {
                av[2][j] = pair_of<FP8, kVBytes, 2>(v[st][2 * j], v[st][2 * j + 1]);
                av[3][j] = pair_of<FP8, kVBytes, 3>(v[st][2 * j], v[st][2 * j + 1]);
            }
        };
        u32x4 pw[2 * RG];
        constexpr int kPAhead = 2 * RG < 3 ? 2 * RG : 3;
#pragma unroll
        for (int i = 0; i < kPAhead; ++i) pw[i] = pbuf[par][rg0 + i % RG][i / RG][lane];
        u32x4 av0[E], av1[E];
#pragma unroll
        for (int j = 0; j < 4; ++j) transposed(0, j, av0);
        float top = s_next[0];
#pragma unroll
        for (int i = 0; i < 2 * RG; ++i) {
            __builtin_amdgcn_sched_barrier(0);
            mfma_acc<E>(o[i % RG], i < RG ? av0 : av1, pw[i]);
            if (i == (2 * RG + 1) / 2 && tl + 3 < count) dma_k(tl + 3);  // into the buffer read before the barrier
            if (i + kPAhead < 2 * RG) pw[i + kPAhead] = pbuf[par][rg0 + (i + kPAhead) % RG][(i + kPAhead) / RG][lane];
            if (i < RG) {
#pragma unroll
                for (int j = 4 * i / RG; j < 4 * (i + 1) / RG; ++j) transposed(1, j, av1);
            } else {
#pragma unroll
                for (int j = 16 * (i - RG) / RG; j < 16 * (i - RG + 1) / RG; ++j) top = fmaxf(top, s_next[j]);
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        top = half_max(top) * c;

        if (tl + 1 < count) {
            seen = seen_of(tl + 1);
            settle(tl + 1, s_next, top, seen);
        }
        s_cur = s_next;
    }

#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
        for (int e = 0; e < E; ++e) mfma_settled(o[rg][e]);

    const int64_t slot = (int64_t)blockIdx.x * kWideRows;  // rows of this item's partial sums
    // every row's maximum and sum, for the waves that hold its outputs
    l = half_sum(l);
    if (h == 0) {
        sm.m[tile_row] = m;
        sm.l[tile_row] = l;
        if (live) {
            const int64_t out_row = (int64_t)row * a.q_heads + q_head;
            if (t.splits > 1)
                it.part_ml[slot + tile_row] = make_float2(m, l);
            else if (a.lse != nullptr)
                a.lse[out_row] = (m + __builtin_amdgcn_logf(l)) * kLn2;
        }
    }
    if (lane == 0) sm.found[wave] = nonfinite;
    __syncthreads();

#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        const int r = 32 * (rg0 + rg) + n;
        const int rtok = r / sh.heads, rig = chunk * sh.heads + r - rtok * sh.heads;
        if (rtok >= t.n || rig >= group) continue;
        const float total = sm.l[r];
        const int64_t orow = t.row0 + rtok;
        const int ohead = kv_head * group + rig;
        const int d0 = slice * C::kSliceDims + 4 * h * E;
        if (t.splits == 1) {
            const float norm = total > 0.0f || total != total ? (FP8 ? a.pages.v_scale : 1.0f) / total : 0.0f;
            uint16_t* op = a.out + orow * a.out_stride + (int64_t)ohead * D + d0;
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                // rows 8b + 4h + i of the product are dims E (8b + 4h + i) + e: 4 E of them in a run
                uint32_t w[2 * E];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < E; e += 2)
                        w[(i * E + e) / 2] = pack_bf16(o[rg][e][4 * b + i] * norm, o[rg][e + 1][4 * b + i] * norm);
#pragma unroll
                for (int i = 0; i < 2 * E; i += 4)
                    *reinterpret_cast<u32x4*>(op + 8 * b * E + 2 * i) = u32x4{w[i], w[i + 1], w[i + 2], w[i + 3]};
            }
        } else if (sm.m[r] != kNegInf || total != 0.0f) {
            float* op = it.part_o + (slot + r) * D + d0;
#pragma unroll
            for (int b = 0; b < 4; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (E == 4) {
                        *reinterpret_cast<f32x4*>(op + 8 * b * E + i * E) =
                            f32x4{o[rg][0][4 * b + i], o[rg][1][4 * b + i], o[rg][2][4 * b + i], o[rg][3][4 * b + i]};
                    } else if ((i & 1) == 0) {
                        *reinterpret_cast<f32x4*>(op + 8 * b * E + i * E) =
                            f32x4{o[rg][0][4 * b + i], o[rg][1][4 * b + i], o[rg][0][4 * b + i + 1], o[rg][1][4 * b + i + 1]};
                    }
                }
        }
    }
    bool fix = false;
#pragma unroll
    for (int w = 0; w < kTileWaves; ++w) fix |= sm.found[w] != 0;
    if (fix) {
        __syncthreads();  // the outputs are in memory
        const int from = key0;
        const int upto = key0 + count * kTileKeys < keys.hi ? key0 + count * kTileKeys : keys.hi;
        fix_nonfinite<D, FP8>(a, t, sh, kv_head, from, upto, kTileKeys, 64 * kTileWaves, [&](int i, int hd, int d, float v) {
            const int ig = chunk * sh.heads + hd;
            if (ig >= group) return;
            const int64_t rr = t.row0 + i;
            const int qh = kv_head * group + ig;
            if (t.splits == 1) {
                uint16_t* op = a.out + rr * a.out_stride + (int64_t)qh * D + d;
                *op = q4::f32_to_bf16(__uint_as_float((uint32_t)*op << 16) + v);
            } else {
                float* op = it.part_o + (slot + i * sh.heads + hd) * D + d;
                *op += v;
            }
        });
    }
}

template <int D, bool FP8>
hipError_t launch(const AttnArgs& a, const Items& it, hipStream_t stream) {
    tile_kernel<D, FP8><<<(unsigned)it.items * (unsigned)it.parts, 64 * kTileWaves, 0, stream>>>(a, it);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_tiles(const AttnArgs& a, const Items& it, hipStream_t stream) {
    if (it.items == 0) return hipSuccess;
    switch (a.pages.head_dim * 2 + a.pages.fp8) {
        case 128: return launch<64, false>(a, it, stream);
        case 129: return launch<64, true>(a, it, stream);
        case 256: return launch<128, false>(a, it, stream);
        case 257: return launch<128, true>(a, it, stream);
        case 512: return launch<256, false>(a, it, stream);
        case 513: return launch<256, true>(a, it, stream);
        case 1024: return launch<512, false>(a, it, stream);
        case 1025: return launch<512, true>(a, it, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace kv
