// Attention of many new tokens over a paged cache: 128 query rows (tokens x heads that
// share a KV head) per workgroup.
//
// The formulas, the softmax and the masked places are those of kv_attention.hip.  With 128
// rows per key the work is bound by the matrix cores (a key's 2 D bytes of K and V feed
// 4 x 128 x D operations), so the layout is chosen to keep them fed from one wave per SIMD:
//
//   S^T = K Q^T (32x32x16, A = K): a wave holds 32 rows of Q in registers and
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
// One wave per SIMD has nobody to fill its waits, so a step mixes three tiles' work, one
// barrier each: the products of tile i's V, those of tile i + 2's scores, and between every two
// of them a share of tile i + 1's softmax, of the transposes, of the DMAs of K tile i + 3 and of
// the loads of V tile i + 1.  (Scores first and V after them, in two blocks: 1095 us at 2048
// tokens over 16384 keys, 16 heads of 512 over one; in turns of four products 1070; in turns of
// one 971, 1.06 PFLOP/s.)  A wave issues an instruction every 6 cycles at best, five beside a
// product of 32, and a step has 316 beside its 64 products: that, and the time at its barrier,
// is what keeps it from the library product's 1.24 PFLOP/s.  Loads of V take 16 bytes a lane, two keys at once:
// the vector memory path moves 64 B a cycle, and a wave that waits for it issues no products.
//
// head_dim 256 has the registers for two waves per SIMD: eight waves, tiles of 64 keys; wave w
// and w + 4 hold the same rows of Q and score a half of the keys each, exchanging the rows'
// maxima through LDS; V's dims are in four slices, each for two waves of 64 rows.  2048 tokens
// of 16 heads over 8, window 1024: 68 us with four waves, 53.4 with eight (644 TFLOP/s; some
// 19 us of it are a workgroup's start and end, which a longer range pays once).
//
// The running maximum of a row is raised only when a score exceeds it by 2^8: weights up to
// 2^8 are rounded by as much relative to themselves as smaller ones, the fp32 sums hold them,
// and the outputs (256 registers at head_dim 512) are seldom rescaled.  Its price: a row's
// largest weight is no longer exactly 1 and is rounded like the others.  Over 4096 random keys
// the weights' rounding is then 1.5e-3 to 1.8e-3 of the outputs in the 2-norm (a model on the
// host), where with the exact maximum it is 0.8e-3 to 1.0e-3; beside the outputs' own 1.7e-3
// that makes 2.2e-3 in all, not 1.8e-3.
#include "kv_device.h"

namespace kv {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kSlack = 8.0f;  // how far a score may exceed the running maximum (log2)

template <int D>
constexpr int tile_waves = D == 256 ? 8 : 4;

template <int D, bool FP8>
struct TileConf {
    static constexpr int kElt = FP8 ? 1 : 2;
    static constexpr int kWaves = tile_waves<D>;
    static constexpr int kHalves = kWaves / 4;                        // waves that share 32 rows' scores, by keys
    static constexpr int kKeys = 32 * kHalves;                        // keys of a tile
    static constexpr int kSteps16 = kKeys / 16;                       // groups of 16 keys, steps of V's products
    static constexpr int kSlices = D >= 256 ? 4 : (D == 64 ? 1 : 2);  // dim slices
    static constexpr int kGroups = 4 * kSlices / kWaves;              // 32-row groups of a wave's outputs
    static constexpr int kSliceDims = D / kSlices;
    static constexpr int kE = kSliceDims / 32;                        // consecutive dims of a lane
    static constexpr int kRowBytes = D * kElt;
    static constexpr int kCpr = kRowBytes / 16;                       // 16-byte chunks of a K row
    static constexpr int kSteps = D / 16;
    static constexpr int kDmaKeys = 1024 / kRowBytes;                 // keys of one DMA
    static constexpr int kDmas = kKeys / kDmaKeys;                    // DMAs of a tile
    static constexpr int kTileBytes = kKeys * kRowBytes;
    // LDS that holds two tiles of K, and before and after them passes on each wave's rows of Q
    // and of the outputs (32 rows of a slice, in fp32 if they are partial)
    static constexpr int kQBytes = 32 * 2 * D, kOutBytes = 32 * 4 * kSliceDims;
    static constexpr int kPassBytes = 4 * kQBytes > kWaves * kOutBytes ? 4 * kQBytes : kWaves * kOutBytes;
    static constexpr int kStageBytes = 2 * kTileBytes > kPassBytes ? 2 * kTileBytes : kPassBytes;
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

// o += a x p.  AGPRS: with the accumulators in AGPRs, for head_dim 512: with the builtin the
// compiler keeps accumulators either all in VGPRs or, S among them, all in AGPRs, and neither
// holds 256 of O beside the rest.  It sees no hazards in asm.  An operand that the VALU writes
// needs two wait states before the product (operands_settled() after the transposes; a test
// reads the compiled code for any other write), and mfma_settled() goes between the products
// and the next VALU access to o.  (The wait states in each product's own asm cost an issue
// slot of the five a product has.)
template <bool AGPRS>
__device__ __forceinline__ void mfma_acc(f32x16& o, u32x4 a, u32x4 p) {
    if constexpr (AGPRS)
        asm("v_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(o) : "v"(a), "v"(p));
    else
        o = mfma32(a, p, o);
}
template <bool AGPRS>
__device__ __forceinline__ void operands_settled() {
    if constexpr (AGPRS) {
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_nop 1");
    }
}
template <bool AGPRS>
__device__ __forceinline__ void mfma_settled(f32x16& o) {
    if constexpr (AGPRS) asm volatile("s_nop 15\n\ts_nop 15" : "+a"(o));
}

// The two bf16 of a word times zero: zeros, and NaN for what is infinite or NaN.
__device__ __forceinline__ uint32_t times_zero(uint32_t w) {
    return ((w & 0x7F80u) == 0x7F80u ? 0x7FC0u : 0u) | ((w & 0x7F800000u) == 0x7F800000u ? 0x7FC00000u : 0u);
}

__device__ __forceinline__ float half_max(float v) {
    const u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p.x), __uint_as_float(p.y));
}
__device__ __forceinline__ float half_sum(float v) {
    const u32x2 p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p.x) + __uint_as_float(p.y);
}

// The E values of one key a lane holds (E * kElt = 2, 4 or 8 bytes).
template <int BYTES>
struct VWords {
    static constexpr int kCount = BYTES == 8 ? 2 : 1;
    uint32_t w[kCount];
};
// A load of 2 BYTES a lane: 16 lanes take all dims of a slice of one key, the next 16 those of
// another (the address unit takes as long for 8 bytes a lane as for 16).
template <int BYTES>
struct VRaw {
    static constexpr int kCount = BYTES == 8 ? 4 : (BYTES == 4 ? 2 : 1);
    uint32_t w[kCount];
};
template <int BYTES>
__device__ __forceinline__ VRaw<BYTES> load_v(__amdgpu_buffer_rsrc_t r, uint32_t lane_off, uint32_t off) {
    VRaw<BYTES> v;
    if constexpr (BYTES == 2) {
        v.w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)lane_off, (int)off, 0);
    } else if constexpr (BYTES == 4) {
        const u32x2 t = __builtin_amdgcn_raw_buffer_load_b64(r, (int)lane_off, (int)off, 0);
        v.w[0] = t.x;
        v.w[1] = t.y;
    } else {
        const u32x4 t = __builtin_amdgcn_raw_buffer_load_b128(r, (int)lane_off, (int)off, 0);
#pragma unroll
        for (int i = 0; i < 4; ++i) v.w[i] = t[i];
    }
    return v;
}
// The two keys of such a load: even rows of 16 lanes keep the first half of the dims of both,
// odd rows the second.
template <int BYTES>
__device__ __forceinline__ void both_keys(const VRaw<BYTES>& raw, VWords<BYTES>& first, VWords<BYTES>& second) {
    if constexpr (BYTES == 2) {
        const u32x2 p = __builtin_amdgcn_permlane16_swap(raw.w[0] & 0xFFFFu, raw.w[0] >> 16, false, false);
        first.w[0] = p.x;
        second.w[0] = p.y;
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 4; ++i) {
            const u32x2 p = __builtin_amdgcn_permlane16_swap(raw.w[i], raw.w[BYTES / 4 + i], false, false);
            first.w[i] = p.x;
            second.w[i] = p.y;
        }
    }
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

template <int WAVES>
struct TileShared {
    float alpha[4][128];
    float top[4][WAVES / 4][128];  // used where two waves share rows
    uint32_t raised[4][4];         // by 32-row group
    int pos[128];
    int64_t q_at[128], out_at[128];  // elements from q's and out's start; out -1: no such row
    float m[128], l[WAVES / 4][128];
    uint32_t found[WAVES];
};

template <int D, bool FP8>
__global__ __launch_bounds__(64 * tile_waves<D>, tile_waves<D> / 4) void tile_kernel(AttnArgs a, Items it) {
    using C = TileConf<D, FP8>;
    constexpr int E = C::kE, RG = C::kGroups;
    constexpr bool kAgprs = D == 512;
    constexpr int kVBytes = E * C::kElt, kWaves = C::kWaves, kTileKeys = C::kKeys, kSt = C::kSteps16;
    __shared__ alignas(1024) char stage[C::kStageBytes];
    __shared__ u32x4 pbuf[2][4][kSt][64];
    __shared__ TileShared<kWaves> sm;

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

    // this lane's query row; where two waves have the same rows, each has its half of a tile's keys
    const int own = C::kHalves == 1 ? wave : wave & 3, half = C::kHalves == 1 ? 0 : wave >> 2;  // 32-row group, half of the keys
    const int tile_row = 32 * own + n;
    const int tok = tile_row / sh.heads, hh = tile_row - tok * sh.heads;
    const int in_group = chunk * sh.heads + hh;
    const bool live = tok < t.n && in_group < group;
    const int row = t.row0 + (live ? tok : 0);
    const int q_head = kv_head * group + (live ? in_group : 0);
    const int pos = live ? t.pos0 + tok : t.pos0;
    if (h == 0 && half == 0) {
        sm.pos[tile_row] = pos;
        sm.q_at[tile_row] = (int64_t)row * a.q_stride + (int64_t)q_head * D;
        sm.out_at[tile_row] = live ? (int64_t)row * a.out_stride + (int64_t)q_head * D : -1;
    }

    // Q: whole rows by DMA into the wave's part of the stage (a lane's own 16 bytes of 32 rows
    // would take the vector memory path twice as long), then into registers in B's layout.
    // The scale's sign goes into Q, so that the largest product is the largest score.  A scale
    // of zero (or one that vanishes with the keys') makes every score zero or NaN in Q already:
    // as a factor it would make NaN of the hidden keys' -inf.
    const float factor = fabsf(a.scale) * (FP8 ? a.pages.k_scale : 1.0f) * kLog2e;
    const bool no_scale = factor == 0.0f;
    const float c = no_scale ? 1.0f : factor;
    u32x4 q[C::kSteps];
    {
        constexpr int kCpr = D / 8, kRows = 64 / kCpr;  // chunks of a row, rows of a DMA
        typedef const __attribute__((address_space(1))) void* GlobalPtr;
        typedef __attribute__((address_space(3))) void* LdsPtr;
        char* const mine = stage + own * C::kQBytes;
        if (half == 0)
#pragma unroll
        for (int j = 0; j < 32 / kRows; ++j) {
            const int r = j * kRows + lane / kCpr, ch = (lane & (kCpr - 1)) ^ swizzle<kCpr>(r);
            __builtin_amdgcn_global_load_lds((GlobalPtr)(a.q + sm.q_at[32 * own + r] + 8 * ch), (LdsPtr)(mine + j * 1024), 16, 0, 0);
        }
        q4::wait_vm_lds<0>();
        if (no_scale && half == 0) {
            // in LDS: beside Q's registers it cost every call (a mixed batch of 12 requests 186 -> 189 us)
#pragma nounroll
            for (int i = lane; i < C::kQBytes / 16; i += 64) {
                u32x4* const at = reinterpret_cast<u32x4*>(mine) + i;
                const u32x4 w = *at;
                *at = u32x4{times_zero(w.x), times_zero(w.y), times_zero(w.z), times_zero(w.w)};
            }
            q4::wait_lds();
        }
        if (C::kHalves > 1) q4::lds_barrier();
        const uint32_t flip = a.scale < 0.0f ? 0x80008000u : 0u;
        const uint32_t keep = live ? ~0u : 0u;
#pragma unroll
        for (int s = 0; s < C::kSteps; ++s) {
            // the dims of the K chunk that step s uses in lane half h
            const int ch = FP8 ? 4 * (s / 2) + 2 * h + (s & 1) : 2 * s + h;
            q[s] = (*reinterpret_cast<const u32x4*>(mine + n * 2 * D + 16 * (ch ^ swizzle<kCpr>(n))) ^ flip) & keep;
        }
        q4::wait_lds();
        q4::lds_barrier();  // K takes the stage
    }

    const KeyRange keys = visible_keys(t.pos0, t.n, kv_len, a.window);
    const int lo = keys.lo & ~(kTileKeys - 1);
    const int tiles = keys.hi > lo ? ceil_div(keys.hi - lo, kTileKeys) : 0;
    const TileRange range = split_tiles(tiles, t.split, t.splits, 1);
    const int count = range.last - range.first;
    const int key0 = lo + range.first * kTileKeys;
    const int* table = a.batch.tables + (int64_t)t.request * a.batch.stride;
    const uint32_t row_bytes = (uint32_t)a.pages.token_stride * C::kElt;

    // Where the 16-key groups lie: lane i has group `window` + i's bytes from this head's first
    // page, and its bit of `present` whether there is a page.  The window moves by 32
    // groups; the pages of the next one are read that far ahead.
    const uint64_t page_bytes = (uint64_t)a.pages.page_stride * C::kElt;
    const int64_t head_bytes = (int64_t)kv_head * a.pages.head_stride * C::kElt;
    const char* const k_head = a.pages.k + head_bytes;
    const char* const v_head = a.pages.v + head_bytes;
    const auto fetch_pages = [&](int first) {
        const int g = first + lane;
        return g < kSt * count ? page_at(table, (key0 + g * kGroupKeys) >> a.pages.page_shift, a.batch.width, a.pages.num_pages) : -1;
    };
    int window = 0, pages_next = 0;
    uint64_t offsets = 0;
    unsigned long long present = 0;
    const auto move_window = [&](int first, int pages) {
        window = first;
        present = __ballot(pages >= 0);
        const uint32_t slot = (uint32_t)(key0 + (first + lane) * kGroupKeys) & ((1u << a.pages.page_shift) - 1u);
        offsets = (uint32_t)(pages < 0 ? 0 : pages) * page_bytes + (uint64_t)slot * row_bytes;
    };
    const auto group_offset = [&](int g) {
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)offsets, g - window);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(offsets >> 32), g - window);
        return ((uint64_t)hi << 32) | lo;
    };

    const uint32_t group_bytes = 15u * row_bytes + (uint32_t)C::kRowBytes;
    // K tile `tl` into a buffer: each DMA brings kDmaKeys whole rows, a wave's lie in one group of
    // 16 keys.  Past the last tile the resource is empty (the DMAs bring zeros).
    constexpr int kWaveDmas = (C::kDmas + kWaves - 1) / kWaves;
    const int first_dma = wave * kWaveDmas % C::kDmas, first_key = first_dma * C::kDmaKeys;
    const auto k_source = [&](int tl) {
        return q4::make_rsrc(k_head + group_offset(kSt * tl + first_key / kGroupKeys), tl < count ? group_bytes : 0u);
    };
    const uint32_t k_lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)(const void*)stage;
    // this lane's row among a DMA's and its chunk there; the DMA's first key adds its own bits
    // (swizzle(key + i) = swizzle(key) ^ swizzle(i) for i < kDmaKeys)
    struct DmaBase {
        uint32_t to, swz;
    };
    const auto dma_base = [&]() {
        DmaBase d{k_lds + (uint32_t)first_dma * 1024u, 16u * (uint32_t)swizzle<C::kCpr>(first_key)};
        asm volatile("" : "+s"(d.to), "+s"(d.swz));  // sums with it are cheap to make again and dear to keep
        return d;
    };
    const auto dma_k = [&](__amdgpu_buffer_rsrc_t r, uint32_t buffer, int j, int ln, const DmaBase& d) {
        const uint32_t dma_row = C::kDmaKeys == 1 ? 0u : ((uint32_t)ln / C::kCpr) * row_bytes;
        const uint32_t dma_chunk = 16u * (((uint32_t)ln & (C::kCpr - 1)) ^ (C::kDmaKeys == 1 ? 0u : (uint32_t)swizzle<C::kCpr>(ln / C::kCpr)));
        const int key = first_key + j * C::kDmaKeys;
        const uint32_t swz = 16u * (uint32_t)swizzle<C::kCpr>(j * C::kDmaKeys) ^ d.swz;
        q4::dma16_at(r, d.to + buffer * (uint32_t)C::kTileBytes + (uint32_t)j * 1024u, dma_row + (dma_chunk ^ swz),
                     (uint32_t)(key % kGroupKeys) * row_bytes);
    };

    // This lane's reads of K: key n's chunk 2u + h, at its row + 16 ((2u + h) ^ swizzle(n)).  The
    // low four bits of 2u go in by xor, the rest as an offset; steps that share those bits
    // follow each other, so that few addresses are alive.
    constexpr int kUnits = C::kCpr / 2, kFar = C::kCpr > 16 ? C::kCpr / 16 : 1, kPer = FP8 ? 2 : 1;
    typedef const __attribute__((address_space(3))) u32x4* LdsPtr;
    const auto k_base = [&](int ln) {
        return k_lds + (uint32_t)(32 * half + (ln & 31)) * C::kRowBytes + 16u * (uint32_t)((ln >> 5) ^ swizzle<C::kCpr>(ln & 31));
    };
    const auto unit_of = [](int i) { return i / kFar + 8 * (i % kFar); };
    const auto read_k = [&](uint32_t base, int buffer, int u) {
        return *((LdsPtr)(uintptr_t)(base ^ (16u * (uint32_t)((2 * u) & 15))) + (2 * u) / 16 * 16 + buffer * (C::kTileBytes / 16));
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
    // lane (h, r = l / 16 % 2, m = l % 16) reads dims 2 E m .. of key 4h + r of a load's
    const uint32_t v_lane = (uint32_t)(4 * h + ((lane >> 4) & 1)) * row_bytes + (uint32_t)((slice * C::kSliceDims + (lane & 15) * 2 * E) * C::kElt);

    f32x16 o[RG][E];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
        for (int e = 0; e < E; ++e) o[rg][e] = f32x16{};
    float m = kNegInf, l = 0.0f;
    bool nonfinite = false;

    constexpr uint32_t kAllPages = (1u << kSt) - 1u;
    // whether every row of the tile sees all of tile tl's keys, and which groups have pages
    const auto all_seen = [&](int tl) { return all_visible(key0 + tl * kTileKeys, kTileKeys, t.pos0, t.n, a.window); };
    const auto pages_of = [&](int tl) { return (uint32_t)(present >> (kSt * tl - window)) & kAllPages; };
    const auto top_of = [&](const f32x16& s) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[i]);
        return half_max(top) * c;
    };
    // Raises the running maximum, if a score of tile tl exceeds it by more than kSlack: the
    // wave's sums here, the outputs when the weights are used.
    const auto raise = [&](int tl, float top) {
        uint32_t raised = 0;
        if (__any(top > m + kSlack)) {
            const float next = fmaxf(m, top);
            const float alpha = __builtin_amdgcn_exp2f(m - (next == kNegInf ? 0.0f : next));
            m = next;
            l *= alpha;
            int ln = lane;
            asm volatile("" : "+v"(ln));
            if (ln < 32 && half == 0) sm.alpha[tl & 3][32 * own + ln] = alpha;
            raised = 1;
        }
        if (lane == 0 && half == 0) sm.raised[tl & 3][own] = raised;
    };
    // Tile tl's scores in `s`: masks them, if some row does not see all of its keys (or there is
    // no such tile).  Their maximum raises the running one at once where a wave has all of a
    // row's keys; where two share them it goes to LDS, and both raise (`raise_shared`) after
    // the next barrier, before the tile's weights.
    const auto settle = [&](int tl, f32x16& s, float top) {
        if (tl >= count) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = kNegInf;
            return;
        }
        const uint32_t there = pages_of(tl);
        if (!all_seen(tl) || there != kAllPages) {
            int ln = lane;
            asm volatile("" : "+v"(ln));
            const int pos = sm.pos[32 * own + (ln & 31)];
            const int above = a.window > 0 ? pos - a.window : -0x7fffffff;  // keys in (above, pos]
            const int first = key0 + tl * kTileKeys + 32 * half + 4 * (ln >> 5);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int key = first + 8 * (i / 4) + i % 4;
                s[i] = (there >> (2 * half + i / 8) & 1) && key <= pos && key > above ? s[i] : kNegInf;
            }
            top = top_of(s);
        }
        if constexpr (C::kHalves == 1) {
            raise(tl, top);
        } else {
            int ln = lane;
            asm volatile("" : "+v"(ln));
            if (ln < 32) sm.top[tl & 3][half][32 * own + ln] = top;
        }
    };
    const auto raise_shared = [&](int tl) {
        if (C::kHalves == 1 || tl >= count) return;
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int r = 32 * own + (ln & 31);
        raise(tl, fmaxf(sm.top[tl & 3][0][r], sm.top[tl & 3][C::kHalves - 1][r]));
    };

    VRaw<kVBytes> v[kSt][4];  // a tile's V: this lane's dims of its keys in each group of 16
    const auto v_source = [&](int g) { return q4::make_rsrc(v_head + group_offset(g), group_bytes); };
    const auto fetch_v = [&](__amdgpu_buffer_rsrc_t r, int j) { return load_v<kVBytes>(r, v_lane, (uint32_t)(8 * (j / 2) + 2 * (j % 2)) * row_bytes); };

    // Weight e of a tile's 16 (scores in `s`) is made when weight e - 1 is summed and packed.
    float before = 0.0f, last = 0.0f;
    uint32_t pk[4];
    const auto weight_done = [&](int e, int par, int ln) {
        if (e < 0) return;
        l += last;
        asm volatile("" : "+v"(l));  // here, between the products
        if (e & 1) pk[e / 2 % 4] = pack_bf16(before, last);
        if (e % 8 == 7) pbuf[par][own][2 * half + e / 8][ln] = u32x4{pk[0], pk[1], pk[2], pk[3]};
    };
    const auto weight = [&](int e, const f32x16& s, float base, int par, int ln) {
        const float w = __builtin_amdgcn_exp2f(fmaf(s[e], c, -base));
        weight_done(e - 1, par, ln);
        before = last;
        last = w;
    };

    f32x16 s2[2] = {};  // scores of an even and an odd tile
    if (count > 0) {
        const int pages = fetch_pages(0);
        pages_next = fetch_pages(32);
        move_window(0, pages);
        const __amdgpu_buffer_rsrc_t k0 = k_source(0), k1 = k_source(1), k2 = k_source(2);
#pragma unroll
        for (int j = 0; j < kWaveDmas; ++j) dma_k(k0, 0, j, lane, dma_base());
#pragma unroll
        for (int j = 0; j < kWaveDmas; ++j) dma_k(k1, 1, j, lane, dma_base());
        q4::wait_vm_lds<0>();
        q4::lds_barrier();
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < kUnits; ++i) {
                if (i % 4 == 0) __builtin_amdgcn_sched_barrier(0);  // or all reads move ahead, into registers Q needs
                s2[b] = product(s2[b], unit_of(i), read_k(k_base(lane), b, unit_of(i)));
            }
        settle(0, s2[0], top_of(s2[0]));
        if constexpr (C::kHalves > 1) {
            settle(1, s2[1], top_of(s2[1]));
            q4::wait_lds();
            q4::lds_barrier();
            raise_shared(0);
        }
        const float base = m == kNegInf ? 0.0f : m;
#pragma unroll
        for (int e = 0; e < 16; ++e) weight(e, s2[0], base, 0, lane);
        weight_done(15, 0, lane);
        if constexpr (C::kHalves == 1) {
            settle(1, s2[1], top_of(s2[1]));
            q4::wait_lds();
            q4::lds_barrier();
        }
#pragma unroll
        for (int j = 0; j < kWaveDmas; ++j) dma_k(k2, 0, j, lane, dma_base());
#pragma unroll
        for (int st = 0; st < kSt; ++st) {
            const __amdgpu_buffer_rsrc_t r = v_source(st);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[st][j] = fetch_v(r, j);
        }
    }

    // Per tile tl: its weights are in LDS and its V is on the way, and the next tile's scores
    // are in s2.  The products of its V, those of the scores of tile tl + 2, and the weights of
    // tile tl + 1 take turns, so that neither the matrix cores nor LDS nor the VALU wait for
    // the others for long.  The order is the source's: slices end in scheduling barriers.
    constexpr int kSlices = kSt * RG, kPerSlice = kUnits / kSlices;
    for (int pair = 0; pair < count; pair += 2) {
#pragma unroll
        for (int par = 0; par < 2; ++par) {
            const int tl = pair + par;
            if (tl >= count) break;
            // K of tile tl + 2 has landed (its DMAs are older than the loads of V) and the
            // weights are written
            q4::wait_vm_lds<4 * kSt>();
            q4::lds_barrier();
            int ln = lane;
            asm volatile("" : "+v"(ln));  // addresses made from it are made here, not kept
            const uint32_t kb = k_base(ln);

            const uint32_t up = sm.raised[tl & 3][ln & 3];
            raise_shared(tl + 1);
            const uint32_t there = pages_of(tl);
            if (!all_seen(tl) || there != kAllPages) {
                const bool visible = all_seen(tl);
#pragma unroll
                for (int st = 0; st < kSt; ++st) {
                    if (visible && (there >> st & 1)) continue;
                    bool bad = false;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int w = 0; w < VRaw<kVBytes>::kCount; ++w) bad |= any_nonfinite<FP8>(v[st][j].w[w]);
                    if (__any(bad)) {
                        nonfinite = true;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int w = 0; w < VRaw<kVBytes>::kCount; ++w) v[st][j].w[w] = finite_only<FP8>(v[st][j].w[w]);
                    }
                }
            }
            if (tl > 0 && __any(up != 0)) {  // before the first products there is nothing to rescale
#pragma unroll
                for (int rg = 0; rg < RG; ++rg) {
                    if (__builtin_amdgcn_readlane(up, rg0 + rg) != 0) {
                        const float f = sm.alpha[tl & 3][32 * (rg0 + rg) + (ln & 31)];
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            mfma_settled<kAgprs>(o[rg][e]);
                            o[rg][e] *= f;
                            mfma_settled<kAgprs>(o[rg][e]);
                            __builtin_amdgcn_sched_barrier(0);  // one at a time: they pass through VGPRs
                        }
                    }
                }
            }

            // keys 2j and 2j + 1 of a lane's eight in group st, into A's register j
            const auto transposed = [&](int st, int j, u32x4 (&av)[E]) {
                VWords<kVBytes> k0, k1;
                both_keys<kVBytes>(v[st][j], k0, k1);
                av[0][j] = pair_of<FP8, kVBytes, 0>(k0, k1);
                av[1][j] = pair_of<FP8, kVBytes, 1>(k0, k1);
                if constexpr (E == 4) {
                    av[2][j] = pair_of<FP8, kVBytes, 2>(k0, k1);
                    av[3][j] = pair_of<FP8, kVBytes, 3>(k0, k1);
                }
            };
            u32x4 kf[kPerSlice], pw[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) pw[i] = pbuf[par][rg0 + i % RG][i / RG][ln];
#pragma unroll
            for (int i = 0; i < kPerSlice; ++i) kf[i] = read_k(kb, par, unit_of(i));
            u32x4 av[E];
#pragma unroll
            for (int j = 0; j < 4; ++j) transposed(0, j, av);
            __amdgpu_buffer_rsrc_t kr, vr[kSt];
            constexpr bool kManyDmas = kWaveDmas >= 8;  // enough to keep their base in registers
            const DmaBase kd = kManyDmas ? dma_base() : DmaBase{};
            f32x16 s_new = {};
            const float base = m == kNegInf ? 0.0f : m;
            constexpr int kTurns = kSlices * E;  // one product of each kind, and a share of the rest
            const auto score = [&](int i, int turn) {
                // the unit's product; the next slice's read follows
#pragma unroll
                for (int k = kPerSlice * turn / E; k < kPerSlice * (turn + 1) / E; ++k) {
                    const int u = i * kPerSlice + k;
                    s_new = product(s_new, unit_of(u), kf[k]);
                    if (u + kPerSlice < kUnits) kf[k] = read_k(kb, par, unit_of(u + kPerSlice));
                }
            };
            const auto share = [&](int i, int turn) {
                const int at = i * E + turn;
#pragma unroll
                for (int e = 16 * at / kTurns; e < 16 * (at + 1) / kTurns; ++e) weight(e, s2[par ^ 1], base, par ^ 1, ln);
                // DMAs of K tile tl + 3 into the buffer of the block before, then V's loads into
                // the registers whose values have been transposed
                if (at == 0) kr = k_source(tl + 3);
#pragma unroll
                for (int st = 0; st < kSt; ++st)
                    if (at == st + 1) vr[st] = v_source(kSt * (tl + 1) + st);
                constexpr int kMid = kTurns / 2;
                const int late = at - kMid;
                if (late < 0) {
#pragma unroll
                    for (int j = kWaveDmas * at / kMid; j < kWaveDmas * (at + 1) / kMid; ++j)
                        dma_k(kr, (uint32_t)(par ^ 1), j, kManyDmas ? ln : lane, kManyDmas ? kd : dma_base());
                } else {
#pragma unroll
                    for (int j = 4 * kSt * late / kMid; j < 4 * kSt * (late + 1) / kMid; ++j) v[j / 4][j % 4] = fetch_v(vr[j / 4], j % 4);
                }
            };
            float top = kNegInf;
#pragma unroll
            for (int i = 0; i < kSlices; ++i) {
                // at the change of groups the scores' products cover the transposes, at the end
                // V's cover the new scores' maximum
                const bool next_group = i > 0 && i % RG == 0, scores_first = next_group || i == kSlices - 1;
                if (scores_first) {
#pragma unroll
                    for (int turn = 0; turn < E; ++turn) {
                        __builtin_amdgcn_sched_barrier(0);
                        score(i, turn);
                        if (next_group)
#pragma unroll
                            for (int j = 4 * turn / E; j < 4 * (turn + 1) / E; ++j) transposed(i / RG, j, av);
                        if (i == kSlices - 1) share(i, turn);
                    }
                }
                if (i % RG == 0) operands_settled<kAgprs>();
#pragma unroll
                for (int turn = 0; turn < E; ++turn) {
                    __builtin_amdgcn_sched_barrier(0);
                    mfma_acc<kAgprs>(o[i % RG][turn], av[turn], pw[i % 2]);
                    if (!scores_first) score(i, turn);
                    if (i < kSlices - 1) share(i, turn);
                    if (i == kSlices - 1) {
                        if (turn == 0) weight_done(15, par ^ 1, ln);
#pragma unroll
                        for (int j = 16 * turn / E; j < 16 * (turn + 1) / E; ++j) top = fmaxf(top, s_new[j]);
                    }
                }
                if (i + 2 < kSlices) pw[i % 2] = pbuf[par][rg0 + (i + 2) % RG][(i + 2) / RG][ln];
            }
            __builtin_amdgcn_sched_barrier(0);
            s2[par] = s_new;
            settle(tl + 2, s2[par], half_max(top) * c);
            if (tl % (32 / kSt) == 32 / kSt - 1) {
                move_window(kSt * (tl + 1), pages_next);
                pages_next = fetch_pages(kSt * (tl + 1) + 32);
            }
        }
    }
    q4::wait_vm<0>();  // no DMA is on its way as the workgroup ends

#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
        for (int e = 0; e < E; ++e) mfma_settled<kAgprs>(o[rg][e]);

    const int64_t slot = (int64_t)blockIdx.x * kWideRows;  // rows of this item's partial sums
    // every row's maximum and sum, for the waves that hold its outputs
    l = half_sum(l);
    if (h == 0) {
        if (half == 0) sm.m[tile_row] = m;
        sm.l[half][tile_row] = l;
    }
    if (lane == 0) sm.found[wave] = nonfinite;
    __syncthreads();
    const auto sum_of = [&](int r) { return C::kHalves == 1 ? sm.l[0][r] : sm.l[0][r] + sm.l[C::kHalves - 1][r]; };
    if (h == 0 && half == 0 && live) {
        const float total = sum_of(tile_row);
        if (t.splits > 1)
            it.part_ml[slot + tile_row] = make_float2(m, total);
        else if (a.lse != nullptr)
            a.lse[(int64_t)row * a.q_heads + q_head] = (m + __builtin_amdgcn_logf(total)) * kLn2;
    }

    // Outputs pass through the wave's part of the stage, so that stores take whole runs of a
    // row's slice (16 bytes of 64 rows each took 64 requests an instruction).  Product e's row
    // 16 x + 8 b + 4 h + i is dim 2 E (8 b + 4 h + i) + E x + e.
    char* const mine = stage + wave * C::kOutBytes;
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        const int r0 = 32 * (rg0 + rg);
        if (t.splits == 1) {
            constexpr int kCpr = C::kSliceDims / 8, kRows = 64 / kCpr;
            const float total = sum_of(r0 + n);
            const float norm = total > 0.0f || total != total ? (FP8 ? a.pages.v_scale : 1.0f) / total : 0.0f;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                uint32_t w[4 * E];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < 2; ++x)
#pragma unroll
                        for (int e = 0; e < E; e += 2)
                            w[(2 * E * i + E * x + e) / 2] = pack_bf16(o[rg][e][8 * x + 4 * b + i] * norm, o[rg][e + 1][8 * x + 4 * b + i] * norm);
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    const int ch = (2 * b + h) * E + i;
                    *reinterpret_cast<u32x4*>(mine + n * 2 * C::kSliceDims + 16 * (ch ^ swizzle<kCpr>(n))) =
                        u32x4{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
                }
            }
#pragma unroll
            for (int j = 0; j < 32 / kRows; ++j) {
                const int r = j * kRows + lane / kCpr, ch = lane & (kCpr - 1);
                const u32x4 w = *reinterpret_cast<const u32x4*>(mine + r * 2 * C::kSliceDims + 16 * (ch ^ swizzle<kCpr>(r)));
                const int64_t at = sm.out_at[r0 + r];
                if (at >= 0) *reinterpret_cast<u32x4*>(a.out + at + slice * C::kSliceDims + 8 * ch) = w;
            }
        } else {
            constexpr int kCpr = C::kSliceDims / 4, kRows = 64 / kCpr;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int x = 0; x < E / 2; ++x) {
                        const int k0 = 4 * b + i, k1 = 8 + 4 * b + i;
                        f32x4 w;
                        if constexpr (E == 4)
                            w = f32x4{o[rg][0][x ? k1 : k0], o[rg][1][x ? k1 : k0], o[rg][2][x ? k1 : k0], o[rg][3][x ? k1 : k0]};
                        else
                            w = f32x4{o[rg][0][k0], o[rg][1][k0], o[rg][0][k1], o[rg][1][k1]};
                        const int ch = (8 * b + 4 * h + i) * (E / 2) + x;
                        *reinterpret_cast<f32x4*>(mine + n * 4 * C::kSliceDims + 16 * (ch ^ swizzle<kCpr>(n))) = w;
                    }
#pragma unroll
            for (int j = 0; j < 32 / kRows; ++j) {
                const int r = j * kRows + lane / kCpr, ch = lane & (kCpr - 1);
                *reinterpret_cast<f32x4*>(it.part_o + (slot + r0 + r) * D + slice * C::kSliceDims + 4 * ch) =
                    *reinterpret_cast<const f32x4*>(mine + r * 4 * C::kSliceDims + 16 * (ch ^ swizzle<kCpr>(r)));
            }
        }
    }
    bool fix = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) fix |= sm.found[w] != 0;
    if (fix) {
        __syncthreads();  // the outputs are in memory
        const int from = key0;
        const int upto = key0 + count * kTileKeys < keys.hi ? key0 + count * kTileKeys : keys.hi;
        fix_nonfinite<D, FP8>(a, t, sh, kv_head, from, upto, kTileKeys, 64 * kWaves, [&](int i, int hd, int d, float v) {
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
    tile_kernel<D, FP8><<<(unsigned)it.items * (unsigned)it.parts, 64 * tile_waves<D>, 0, stream>>>(a, it);
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
