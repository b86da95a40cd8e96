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
#include "kv_rows16.h"

namespace kv {
namespace {

// Workgroups of rows16 that cuts are made for: one per CU at head_dim 512, where the registers
// hold one wave per SIMD, else two.  (At 64 and 128 dims the registers would hold three or more;
// what more and shorter items do there has not been measured.)
int rows_fill(const AttnArgs& a) { return a.pages.head_dim == 512 ? 256 : 512; }
// Those of the 128-row tiles: one per CU, two of the smaller heads (registers and LDS).
int tiles_fill(const AttnArgs& a) { return a.pages.head_dim >= 256 ? 256 : 512; }

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

AttnPlan plan_attention(const AttnArgs& a, bool scaled) {
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
    // Over pages of e4m3 with block scales, half the bytes for the 16-row tiles, further on (us, 16-row
    // / 128-row): 512 dims, one of 64 tokens over 4096 keys (2e9) 41 / 52, sixteen of 8 (4.3e9) 64 / 75,
    // twenty (5.4e9) 104 / 82; 256 dims, window 1024, one of 512 tokens (2.3e9) 28 / 41, of 1024 (4.6e9)
    // 53 / 56, of 1400 (6.2e9) 75 / 63; 128 dims, one of 128 over 16384 (2.1e9) 35 / 39, of 200 (3.4e9)
    // 55 / 45; 64 dims, one of 64 over 16384 (2.1e9) 38 / 39, of 128 (4.3e9) 64 / 56.
    const double work = (double)tokens * a.q_heads * (double)most_keys(a, wide.tokens) * a.pages.head_dim;
    const double little = !scaled ? 8e8 : (a.pages.head_dim >= 256 ? 4.6e9 : 2.2e9);
    // One request: its kernel is known.  Several with a row each at least: none reaches
    // `from` rows if the sum stays under this (were some of them empty, the 16-row kernel
    // would still be right).
    if (a.kernel == 2 || (a.kernel == 0 && work < little))
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

hipError_t launch_attention(const AttnArgs& a, const AttnPlan& plan, const BlockScales* scales, hipStream_t stream) {
    const int group = a.q_heads / a.pages.kv_heads;
    hipError_t e = hipSuccess;
    if (plan.use_tiles) e = scales != nullptr ? launch_scaled_tiles(a, plan.tiles, *scales, stream) : launch_tiles(a, plan.tiles, stream);
    if (plan.use_rows && e == hipSuccess)
        e = scales != nullptr ? launch_scaled_rows16(a, plan.rows, *scales, stream) : launch_rows16(a, plan.rows, stream);
    if (plan.use_tiles && e == hipSuccess)
        e = launch_join(a, plan.tiles, tile_cuts(a, plan.tiles, tile_shape(kWideRows, group)), kWideRows, stream);
    if (plan.use_rows && e == hipSuccess)
        e = launch_join(a, plan.rows, rows_cuts(a, plan.rows, tile_shape(kThinRows, group)), kThinRows, stream);
    return e;
}

}  // namespace kv
