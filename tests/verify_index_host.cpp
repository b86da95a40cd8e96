// The sampling kernels' index arithmetic (verify_index.h) on the host, for tests: counts how
// often each (row, part) is taken; -1 for one out of range.
#include "verify_index.h"

extern "C" {
// seen [rows][parts]; returns parts, or -1
int verify_stats(int rows, int vocab, int* seen) {
    const verify::Plan p = verify::plan_of(rows, vocab);
    if (seen == nullptr) return p.parts;
    const int64_t waves = p.groups() * (verify::kStatsThreads / 64);
    for (int64_t wave = 0; wave < waves; ++wave) {
        const verify::Place w = verify::place_of(p, (int)wave);
        if (w.part == -1) continue;
        if (w.row < 0 || w.row >= rows || w.part < 0 || w.part >= p.parts || (int64_t)w.part * p.size() >= vocab) return -1;
        ++seen[(int64_t)w.row * p.parts + w.part];
    }
    return p.parts;
}
// seen [requests][parts]; returns the workgroups of a request, or -1
int verify_rest(int requests, int parts, int* seen) {
    const int groups = verify::rest_groups(requests, parts);
    for (int r = 0; r < requests; ++r)
        for (int g = 0; g < groups; ++g)
            for (int wave = 0; wave < verify::kWide / 64; ++wave)
                for (int part = verify::first_part(g, wave); part < parts; part += verify::part_step(groups)) {
                    if (part < 0) return -1;
                    ++seen[(int64_t)r * parts + part];
                }
    return groups;
}
}
