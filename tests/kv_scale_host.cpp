// The scales of blocks of e4m3 (kv_index.h) on the host, for tests.
#include "kv_index.h"

extern "C" {
int kv_least_scale(uint32_t bits) { return kv::least_scale_of(bits); }
int kv_clamp_scale(int byte) { return kv::clamp_scale(byte); }
}
