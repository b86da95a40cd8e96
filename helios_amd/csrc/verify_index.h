// Index arithmetic of the sampling kernels, usable on the host: how a launch's waves and
// workgroups share rows and parts.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace verify {

constexpr int kStatsThreads = 256, kWide = 1024;  // of a workgroup of stats_kernel, and of the others

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

// A row is cut into parts of 512 `sweeps` places (8 a lane and sweep), a wave's each in stats_kernel
// and rest_kernel.  `rows` of them: the target's, then the drafter's if there is one.
struct Plan {
    int rows, parts, sweeps;
    __host__ __device__ int size() const { return 512 * sweeps; }
    __host__ __device__ int64_t groups() const {
        return ((int64_t)rows * parts + kStatsThreads / 64 - 1) / (kStatsThreads / 64);
    }
};
// Parts of 2048 where that leaves two waves to a SIMD at least, else of 512.  stats_kernel in us (under a
// profiler), by 512 and by 2048, rows of 262144 bf16: 3.3 / 4.1 for one, 4.4 / 4.4 for 8, 6.1 / 5.3 for 16,
// 11.3 / 8.7 for 32, 56 / 39 for 256; with a softcap 3.7 / 6.3, 6.2 / 7.1, 9.6 / 9.0, 16.4 / 15.5, 109 / 97.
__host__ __device__ inline Plan plan_of(int rows, int vocab) {
    const int64_t large = (int64_t)rows * ceil_div(vocab, 2048);
    const int sweeps = large >= 2 * 4 * 256 ? 4 : 1;
    return Plan{rows, ceil_div(vocab, 512 * sweeps), sweeps};
}
// The row and part of a wave of stats_kernel; part -1 for the last workgroup's waves past the last row.
struct Place {
    int row, part;
};
__host__ __device__ inline Place place_of(const Plan& p, int wave) {
    const int row = wave / p.parts;
    return row < p.rows ? Place{row, wave - row * p.parts} : Place{0, -1};
}

// rest_kernel: workgroups to a request, one to a CU in all, as each finds the request's first draft
// that falls; workgroup g's wave takes parts first_part(g, wave), + groups * waves, ...
__host__ __device__ inline int rest_groups(int requests, int parts) {
    const int most = ceil_div(parts, kWide / 64), fill = ceil_div(256, requests);
    return most < fill ? most : fill;
}
__host__ __device__ inline int first_part(int group, int wave) { return group * (kWide / 64) + wave; }
__host__ __device__ inline int part_step(int groups) { return groups * (kWide / 64); }

}  // namespace verify
