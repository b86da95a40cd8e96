// Pages of a paged cache given out and taken back on the GPU, and the slots of a batch's rows.
//
//   reserve: n_r new tokens for request r, which holds len_r:
//     starts = exclusive sums of n;  kv_r = len_r + n_r
//     need_r = absent entries of table r in [ceil(len_r / page), ceil(kv_r / page))
//     granted in order of the requests while the sums of need stay within the free pages, each
//     request whole or not at all; page i of those is free[count - 1 - i]
//     row i of request r: position len_r + i, slot page * page_size + position % page_size
//   release: len_r tokens are kept; entries before the page of position len_r - window + 1 (with
//     a window) and from ceil(len_r / page) on go back, the first of F freed ones on top:
//     freed page i to free[count + F - 1 - i]
//
// So a release right after a reserve restores the free pages in their order, and nothing
// depends on timing: there are no atomics, orders are those of prefix sums.
//
// A few hundred bytes for a decoding batch and a megabyte for prompts: what counts is the chain
// of dependent loads and the launches.  One workgroup does a call of few entries and rows;
// longer ones spread the rows (reserve) or the requests' tables (release) over the card in a
// second launch.
#include "kv_device.h"

namespace kv {
namespace {

constexpr int kThreads = 1024, kPoolWaves = kThreads / 64;
constexpr int kMostNew = 1 << 24;  // tokens of a batch

// Inclusive sum over the workgroup; `sums` is scratch of a value per wave, `total` the sum.
__device__ __forceinline__ int64_t group_scan(int64_t v, int64_t* sums, int64_t* total) {
    const int lane = (int)threadIdx.x & 63, wave = (int)threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t up = __shfl_up(v, d);
        v += lane >= d ? up : 0;
    }
    __syncthreads();  // the scan before is read
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int w = 0; w < (int)blockDim.x / 64; ++w) {
        before += w < wave ? sums[w] : 0;
        all += sums[w];
    }
    *total = all;
    return v + before;
}

__device__ __forceinline__ int pages_for(int len, int shift) { return (int)(((int64_t)len + (1 << shift) - 1) >> shift); }
__device__ __forceinline__ bool is_page(const Pool& p, int entry) { return entry >= 0 && entry < p.num_pages; }

struct Request {
    int len, rows, first, end;  // tokens held, new ones, the pages that these need
    bool fits;
};
__device__ __forceinline__ Request request_of(const Pool& p, const int* new_tokens, int r) {
    Request q;
    q.len = clampi(p.lens[r], 0, p.width << p.page_shift);
    q.rows = clampi(new_tokens[r], 0, kMostNew);
    q.first = pages_for(q.len, p.page_shift);
    q.end = pages_for(q.len + q.rows, p.page_shift);
    q.fits = q.end <= p.width;
    return q;
}

__device__ __forceinline__ void slots_of(const Pool& p, const Reserve& a, int row) {
    // the request is the number of starts[1..] that are <= row
    int lo = 0, hi = p.requests;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.starts[mid + 1] <= row)
            lo = mid + 1;
        else
            hi = mid;
    }
    int pos = 0;
    int64_t slot = -1;
    if (lo < p.requests) {
        pos = clampi(p.lens[lo], 0, p.width << p.page_shift) + row - a.starts[lo];
        const int page = page_at(p.tables + (int64_t)lo * p.stride, pos >> p.page_shift, p.width, p.num_pages);
        if (page >= 0) slot = ((int64_t)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
    }
    if (a.positions != nullptr) a.positions[row] = pos;
    if (a.slots != nullptr) a.slots[row] = slot;
}

__global__ __launch_bounds__(kThreads) void reserve_kernel(Pool p, Reserve a, int rows_here) {
    __shared__ int64_t sums[kPoolWaves];
    __shared__ int needs[kThreads], taken[kThreads];
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int free_count = clampi(*p.free_count, 0, p.num_pages);
    int64_t row_sum = 0, need_sum = 0, given = 0;
    if (tid == 0) a.starts[0] = 0;
    for (int base = 0; base < p.requests; base += kThreads) {
        const int r = base + tid, here = p.requests - base < kThreads ? p.requests - base : kThreads;
        Request q{0, 0, 0, 0, true};
        if (r < p.requests) q = request_of(p, a.new_tokens, r);
        // absent entries: a wave to a request
        for (int i = wave; i < here; i += kPoolWaves) {
            const Request w = request_of(p, a.new_tokens, base + i);
            const int* table = p.tables + (int64_t)(base + i) * p.stride;
            int count = 0;
            if (w.fits)
                for (int j = w.first; j < w.end; j += 64)
                    count += __popcll(__ballot(j + lane < w.end && !is_page(p, table[j + lane < w.end ? j + lane : j])));
            if (lane == 0) needs[i] = count;
        }
        __syncthreads();
        const int need = r < p.requests ? needs[tid] : 0;
        int64_t rows, all_rows, all_needs;
        rows = group_scan(q.rows, sums, &all_rows) + row_sum;
        const int64_t upto = group_scan(need, sums, &all_needs) + need_sum;
        const bool granted = q.fits && (need == 0 || upto <= free_count);
        taken[tid] = granted && r < p.requests ? (int)(upto - need) : -1;
        int64_t now;
        (void)group_scan(granted ? need : 0, sums, &now);
        given += now;
        if (r < p.requests) {
            a.starts[r + 1] = (int)(rows < 0x7FFFFFFF ? rows : 0x7FFFFFFF);
            a.kv_lens[r] = q.len + q.rows;
            if (a.granted != nullptr) a.granted[r] = granted;
        }
        row_sum += all_rows;
        need_sum += all_needs;
        for (int i = wave; i < here; i += kPoolWaves) {
            if (taken[i] < 0 || needs[i] == 0) continue;
            const Request w = request_of(p, a.new_tokens, base + i);
            int* table = p.tables + (int64_t)(base + i) * p.stride;
            int nth = taken[i];
            for (int j = w.first; j < w.end; j += 64) {
                const bool absent = j + lane < w.end && !is_page(p, table[j + lane < w.end ? j + lane : j]);
                const unsigned long long which = __ballot(absent);
                const int mine = nth + __popcll(which & ((1ull << lane) - 1));
                if (absent) table[j + lane] = p.free_pages[free_count - 1 - mine];
                nth += __popcll(which);
            }
        }
        __syncthreads();
    }
    if (tid == 0) *p.free_count = free_count - (int)given;
    for (int row = tid; row < rows_here; row += kThreads) slots_of(p, a, row);
}

__global__ __launch_bounds__(256) void slots_kernel(Pool p, Reserve a, int rows) {
    const int row = (int)(blockIdx.x * 256 + threadIdx.x);
    if (row < rows) slots_of(p, a, row);
}

// Whether entry j of request r's table goes back, where `len` tokens are kept.
__device__ __forceinline__ bool goes(const Pool& p, int entry, int j, int len, int window) {
    if (!is_page(p, entry)) return false;
    const int reach = window > 0 && len - window + 1 > 0 ? len - window + 1 : 0;
    return j < (reach >> p.page_shift) || j >= pages_for(len, p.page_shift);
}

__device__ __forceinline__ void put_back(const Pool& p, int64_t at, int page) {
    if (at >= 0 && at < p.num_pages) p.free_pages[at] = page;
}

// All of it in one workgroup.
__global__ __launch_bounds__(kThreads) void release_kernel(Pool p, const int* lens, int window) {
    __shared__ int64_t sums[kPoolWaves];
    const int tid = (int)threadIdx.x;
    const int free_count = clampi(*p.free_count, 0, p.num_pages);
    const int entries = p.requests * p.width;
    int64_t freed = 0, total = 0;
    for (int base = 0; base < entries; base += kThreads) {
        const int i = base + tid, r = i / p.width, j = i - r * p.width;
        const bool gone = i < entries && goes(p, p.tables[(int64_t)r * p.stride + j], j, clampi(lens[r], 0, p.width << p.page_shift), window);
        int64_t here;
        (void)group_scan(gone, sums, &here);
        total += here;
    }
    for (int base = 0; base < entries; base += kThreads) {
        const int i = base + tid, r = i / p.width, j = i - r * p.width;
        bool gone = false;
        int* const at = p.tables + (int64_t)r * p.stride + j;
        if (i < entries) gone = goes(p, *at, j, clampi(lens[r], 0, p.width << p.page_shift), window);
        int64_t here;
        const int64_t nth = freed + group_scan(gone, sums, &here) - 1;
        if (gone) {
            put_back(p, free_count + total - 1 - nth, *at);
            *at = -1;
        }
        freed += here;
    }
    __syncthreads();
    for (int r = tid; r < p.requests; r += kThreads) p.lens[r] = clampi(lens[r], 0, p.width << p.page_shift);
    if (tid == 0) *p.free_count = (int)(free_count + total < p.num_pages ? free_count + total : p.num_pages);
}

// counts[r]: the pages of request r that go back; counts[requests]: the free pages before.
__global__ __launch_bounds__(256) void count_kernel(Pool p, const int* lens, int window, int* counts) {
    __shared__ int64_t sums[4];
    const int r = (int)blockIdx.x, len = clampi(lens[r], 0, p.width << p.page_shift);
    int64_t n = 0, all;
    for (int j = (int)threadIdx.x; j < p.width; j += 256) n += goes(p, p.tables[(int64_t)r * p.stride + j], j, len, window);
    (void)group_scan(n, sums, &all);
    if (threadIdx.x == 0) {
        counts[r] = (int)all;
        if (r == 0) counts[p.requests] = clampi(*p.free_count, 0, p.num_pages);
    }
}

__global__ __launch_bounds__(256) void return_kernel(Pool p, const int* lens, int window, const int* counts) {
    __shared__ int64_t sums[4];
    const int tid = (int)threadIdx.x, r = (int)blockIdx.x;
    const int len = clampi(lens[r], 0, p.width << p.page_shift);
    int64_t before = 0, after = 0, freed, rest;
    for (int i = tid; i < p.requests; i += 256) {
        before += i < r ? counts[i] : 0;
        after += i >= r ? counts[i] : 0;
    }
    (void)group_scan(before, sums, &freed);
    (void)group_scan(after, sums, &rest);
    const int64_t total = freed + rest, base = counts[p.requests];
    if (counts[r] > 0)
        for (int j0 = 0; j0 < p.width; j0 += 256) {
            const int j = j0 + tid;
            int* const at = p.tables + (int64_t)r * p.stride + j;
            const bool gone = j < p.width && goes(p, *at, j, len, window);
            int64_t here;
            const int64_t nth = freed + group_scan(gone, sums, &here) - 1;
            if (gone) {
                put_back(p, base + total - 1 - nth, *at);
                *at = -1;
            }
            freed += here;
        }
    if (tid == 0) {
        p.lens[r] = len;
        if (r == 0) *p.free_count = (int)(base + total < p.num_pages ? base + total : p.num_pages);
    }
}

// Rows and table entries that one workgroup takes.
constexpr int kFewRows = 4096, kFewEntries = 16384;

}  // namespace

hipError_t launch_reserve(const Pool& p, const Reserve& a, int rows, hipStream_t stream) {
    const bool mapped = a.positions != nullptr || a.slots != nullptr;
    const int here = mapped && rows <= kFewRows ? rows : 0;
    reserve_kernel<<<1, kThreads, 0, stream>>>(p, a, here);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !mapped || rows <= kFewRows) return e;
    slots_kernel<<<(unsigned)ceil_div(rows, 256), 256, 0, stream>>>(p, a, rows);
    return hipGetLastError();
}

size_t release_scratch(const Pool& p) {
    return (int64_t)p.requests * p.width <= kFewEntries ? 0 : ((size_t)p.requests + 1) * sizeof(int);
}

hipError_t launch_release(const Pool& p, const int* lens, int window, int* counts, hipStream_t stream) {
    if (counts == nullptr) {
        release_kernel<<<1, kThreads, 0, stream>>>(p, lens, window);
        return hipGetLastError();
    }
    count_kernel<<<(unsigned)p.requests, 256, 0, stream>>>(p, lens, window, counts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return_kernel<<<(unsigned)p.requests, 256, 0, stream>>>(p, lens, window, counts);
    return hipGetLastError();
}

}  // namespace kv
