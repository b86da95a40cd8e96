// The cuts of a launch into items (kv_index.h, as find_item puts them together) on the host.
#include "kv_index.h"

extern "C" {

int kv_most_tiles(int64_t rows, int64_t runs, int tokens, int least, int most) { return kv::most_tiles(rows, runs, tokens, least, most); }

// The tiles of each run (runs of rows[r] rows and len[r] keys; those of least..most rows
// count) and the items of each of its tiles.
void kv_items(const int* rows, const int* len, int runs, int table_keys, int tokens, int least, int most, int unit, int slots,
              int window, int min_units, int few_units, int* tiles, int* splits) {
    float sum = 0.0f;
    int all = 0, longest = 1, items_alike = 0, items_even = 0;
    for (int r = 0; r < runs; ++r) {
        const int n = rows[r] >= least && rows[r] <= most ? rows[r] : 0;
        tiles[r] = kv::tiles_of(n, tokens);
        splits[r] = kv::units_of(n, len[r], table_keys, tokens, unit, window);
        sum += (float)tiles[r] * (float)splits[r];
        all += tiles[r];
        if (tiles[r] > 0 && splits[r] > longest) longest = splits[r];
    }
    const int alike = kv::alike_units(longest, all, slots), even = kv::even_units(sum, slots);
    for (int r = 0; r < runs; ++r) {
        items_alike += tiles[r] * kv::parts_of(splits[r], alike);
        items_even += tiles[r] * kv::parts_of(splits[r], even);
    }
    const int per = kv::item_units(alike, items_alike, even, items_even, slots, sum <= (float)slots ? few_units : min_units);
    for (int r = 0; r < runs; ++r) splits[r] = kv::parts_of(splits[r], per);
}

}  // extern "C"
