// Attention over pages of e4m3 with a scale for each block of tokens and KV head: the kernels of
// kv_attention.hip and kv_tile.hip, whose conversion of two codes to bf16 takes the scale as its
// operand.  The scales are powers of two, so the bf16 values are exact and nothing else differs.
//
// A block is a multiple of the 16 keys of a group, so a group has one scale for K and one for V.
// They are read where a wave reads its groups' pages, a lane a group (64 tiles at a time in the
// 16-row tiles, 32 groups ahead in the 128-row ones), and cost two lane reads a group.
//
// 64 single tokens over 1024 keys, 8 KV heads of 256, 230 MB: 49 us, 4.7 TB/s; 32 over up to 16000
// keys, one of 512, 201 MB: 46 us and a join of 7; 2048 tokens over 16384 keys, 16 heads of 512 over
// one: 951-983 us, 1.05-1.08 PFLOP/s.  By one scale for all pages the same calls take 54.5, 45 + 7 and
// (bf16) 959-1047.
#include "kv_rows16.h"
#include "kv_tile_kernel.h"

namespace kv {
namespace {

template <int D>
hipError_t launch_rows(const AttnArgs& a, const Items& it, const BlockScales& sc, hipStream_t stream) {
    rows16_kernel<D, true, BlockScales><<<(unsigned)it.items * (unsigned)it.parts, 64 * kWaves, 0, stream>>>(a, it, sc);
    return hipGetLastError();
}

template <int D>
hipError_t launch_wide(const AttnArgs& a, const Items& it, const BlockScales& sc, hipStream_t stream) {
    tile_kernel<D, true, BlockScales><<<(unsigned)it.items * (unsigned)it.parts, 64 * tile_waves<D>, 0, stream>>>(a, it, sc);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_scaled_rows16(const AttnArgs& a, const Items& it, const BlockScales& sc, hipStream_t stream) {
    switch (a.pages.head_dim) {
        case 64: return launch_rows<64>(a, it, sc, stream);
        case 128: return launch_rows<128>(a, it, sc, stream);
        case 256: return launch_rows<256>(a, it, sc, stream);
        case 512: return launch_rows<512>(a, it, sc, stream);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_scaled_tiles(const AttnArgs& a, const Items& it, const BlockScales& sc, hipStream_t stream) {
    if (it.items == 0) return hipSuccess;
    switch (a.pages.head_dim) {
        case 64: return launch_wide<64>(a, it, sc, stream);
        case 128: return launch_wide<128>(a, it, sc, stream);
        case 256: return launch_wide<256>(a, it, sc, stream);
        case 512: return launch_wide<512>(a, it, sc, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace kv
