// The index arithmetic of the paged-cache kernels (kv_index.h) on the host, for tests.
#include "kv_index.h"

extern "C" {
int kv_page_at(const int* table, int at, int width, int num_pages) { return kv::page_at(table, at, width, num_pages); }
int kv_run_bound(const int* starts, int r, int requests, int tokens) { return kv::run_bound(starts, r, requests, tokens); }
void kv_visible(int pos0, int n, int kv_len, int window, int* out) {
    const kv::KeyRange r = kv::visible_keys(pos0, n, kv_len, window);
    out[0] = r.lo;
    out[1] = r.hi;
}
int kv_all_visible(int key, int keys, int pos0, int n, int window) { return kv::all_visible(key, keys, pos0, n, window); }
void kv_split(int tiles, int s, int splits, int least, int* out) {
    const kv::TileRange r = kv::split_tiles(tiles, s, splits, least);
    out[0] = r.first;
    out[1] = r.last;
}
}
