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
#include "kv_tile_kernel.h"

namespace kv {
namespace {

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
