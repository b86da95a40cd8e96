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
// depends on timing: orders are those of prefix sums, and there are no atomics on the pool.
//
// A few hundred bytes for a decoding batch and a megabyte for prompts: what counts is the chain
// of dependent loads, and the launches.  A batch of few rows is one workgroup's, a thread to a
// request (what a decoding step needs) and a wave to each that needs many pages; larger ones take
// two launches: what each request needs, then a workgroup to a request.  release likewise.
// us: a token for each of 8 requests, reserve 3.1 and release 3.0 (6.2 and 7.4 with scans through LDS and
// entries one after another); 96 requests' mixed prompts in tables of 2048, 84000 rows, 2.6 + 3.7 + 4.1 (the
// map) and 2.8 + 4.5.
#include "kv_device.h"

namespace kv {
namespace {

constexpr int kThreads = 1024, kGroup = 256;
constexpr int kMostNew = 1 << 24;  // tokens of a batch

// Inclusive sums over the workgroup of two values, of a wave's lanes each within 32 bits; `all` their
// totals.  sums: scratch of two a wave.
struct Two {
    int64_t a, b;
};
template <int THREADS>
__device__ __forceinline__ Two group_scan(int a, int b, Two* sums, Two* all) {
    const int wave = (int)threadIdx.x >> 6;
    a = wave_scan(a);
    b = wave_scan(b);
    __syncthreads();  // the scan before is read
    if ((threadIdx.x & 63) == 63) sums[wave] = Two{a, b};
    __syncthreads();
    Two before{0, 0};
    *all = Two{0, 0};
#pragma unroll
    for (int w = 0; w < THREADS / 64; ++w) {
        before.a += w < wave ? sums[w].a : 0;
        before.b += w < wave ? sums[w].b : 0;
        all->a += sums[w].a;
        all->b += sums[w].b;
    }
    return Two{a + before.a, b + before.b};
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

// Absent entries among [first, end) of a table, by a wave.
__device__ __forceinline__ int count_absent(const Pool& p, const int* table, int first, int end, int lane) {
    int count = 0;
    for (int j0 = first; j0 < end; j0 += 256) {
        int entry[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) entry[k] = j0 + 64 * k + lane < end ? table[j0 + 64 * k + lane] : 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) count += __popcll(__ballot(j0 + 64 * k + lane < end && !is_page(p, entry[k])));
    }
    return count;
}
// Fills them from the free pages, the first from free_pages[top - 1] on down.
__device__ __forceinline__ void fill_absent(const Pool& p, int* table, int first, int end, int top, int lane) {
    for (int j0 = first; j0 < end; j0 += 256) {
        int entry[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) entry[k] = j0 + 64 * k + lane < end ? table[j0 + 64 * k + lane] : 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const bool absent = j0 + 64 * k + lane < end && !is_page(p, entry[k]);
            const unsigned long long which = __ballot(absent);
            if (absent) table[j0 + 64 * k + lane] = p.free_pages[top - 1 - __popcll(which & ((1ull << lane) - 1))];
            top -= __popcll(which);
        }
    }
}

__device__ __forceinline__ int saturated(int64_t v) { return (int)(v < 0x7FFFFFFF ? v : 0x7FFFFFFF); }

// Row `row` of the batch: row `nth` of request r, which holds `len` (nth < 0: of none).
__device__ __forceinline__ void map_row(const Pool& p, const Reserve& a, int row, int r, int len, int nth) {
    int pos = 0;
    int64_t slot = -1;
    if (nth >= 0) {
        pos = len + nth;
        const int page = page_at(p.tables + (int64_t)r * p.stride, pos >> p.page_shift, p.width, p.num_pages);
        if (page >= 0) slot = ((int64_t)page << p.page_shift) + (pos & ((1 << p.page_shift) - 1));
    }
    if (a.positions != nullptr) a.positions[row] = pos;
    if (a.slots != nullptr) a.slots[row] = slot;
}

// All of it in one workgroup, up to kThreads requests: a thread to a request.
constexpr int kShort = 4;  // entries that a thread looks at itself
__global__ __launch_bounds__(kThreads) void reserve_kernel(Pool p, Reserve a, int rows) {
    __shared__ Two sums[kThreads / 64];
    __shared__ int starts[kThreads + 1], lens[kThreads], work[kThreads], tops[kThreads], listed[kThreads];
    __shared__ int list_size, given;
    const int tid = (int)threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid == 0) {
        list_size = 0;
        given = 0;
        starts[0] = 0;
        a.starts[0] = 0;
    }
    Request q{0, 0, 0, 0, true};
    if (tid < p.requests) q = request_of(p, a.new_tokens, tid);
    const int free_count = clampi(*p.free_count, 0, p.num_pages);
    int* const table = p.tables + (int64_t)(tid < p.requests ? tid : 0) * p.stride;
    const int entries = q.fits ? q.end - q.first : 0;
    const bool many = entries > kShort;
    int need = 0, absent = 0;
    if (!many) {
        int entry[kShort];
#pragma unroll
        for (int k = 0; k < kShort; ++k) entry[k] = k < entries ? table[q.first + k] : 0;
#pragma unroll
        for (int k = 0; k < kShort; ++k)
            if (k < entries && !is_page(p, entry[k])) {
                absent |= 1 << k;
                ++need;
            }
    }
    __syncthreads();
    if (many) listed[atomicAdd(&list_size, 1)] = tid;  // in any order: each is a request of its own
    __syncthreads();
    const int long_ones = list_size;
    for (int i = wave; i < long_ones; i += kThreads / 64) {
        const int r = listed[i];
        const Request w = request_of(p, a.new_tokens, r);
        const int n = count_absent(p, p.tables + (int64_t)r * p.stride, w.first, w.end, lane);
        if (lane == 0) work[r] = n;
    }
    if (long_ones > 0) __syncthreads();
    if (many) need = work[tid];
    Two all;
    const Two upto = group_scan<kThreads>(q.rows, need, sums, &all);
    const bool granted = q.fits && (need == 0 || upto.b <= free_count);
    const int top = free_count - (int)(upto.b - need);
    if (tid < p.requests) {
        starts[tid + 1] = a.starts[tid + 1] = saturated(upto.a);
        lens[tid] = q.len;
        tops[tid] = granted ? top : -1;
        a.kv_lens[tid] = q.len + q.rows;
        if (a.granted != nullptr) a.granted[tid] = granted;
        if (granted && need > 0) atomicMax(&given, (int)upto.b);  // sums rise: the last one granted
        if (granted && !many) {
            int nth = 0;
#pragma unroll
            for (int k = 0; k < kShort; ++k)
                if (absent >> k & 1) table[q.first + k] = p.free_pages[top - 1 - nth++];
        }
    }
    __syncthreads();
    for (int i = wave; i < long_ones; i += kThreads / 64) {
        const int r = listed[i];
        if (tops[r] < 0) continue;
        const Request w = request_of(p, a.new_tokens, r);
        fill_absent(p, p.tables + (int64_t)r * p.stride, w.first, w.end, tops[r], lane);
    }
    if (long_ones > 0) __syncthreads();
    if (tid == 0) *p.free_count = free_count - given;
    for (int row = tid; row < rows; row += kThreads) {
        // the request is the number of starts[1..] that are <= row
        int lo = 0, hi = p.requests;
        while (lo < hi) {
            const int mid = (lo + hi) / 2;
            if (starts[mid + 1] <= row)
                lo = mid + 1;
            else
                hi = mid;
        }
        map_row(p, a, row, lo, lo < p.requests ? lens[lo] : 0, lo < p.requests ? row - starts[lo] : -1);
    }
}

// needs[r]: the pages that request r needs; needs[requests]: the free pages before.
__global__ __launch_bounds__(kGroup) void need_kernel(Pool p, Reserve a, int* needs) {
    const int lane = (int)threadIdx.x & 63, r = (int)blockIdx.x * (kGroup / 64) + ((int)threadIdx.x >> 6);
    if (r >= p.requests) return;
    const Request q = request_of(p, a.new_tokens, r);
    const int n = q.fits ? count_absent(p, p.tables + (int64_t)r * p.stride, q.first, q.end, lane) : 0;
    if (lane == 0) {
        needs[r] = n;
        if (r == 0) needs[p.requests] = clampi(*p.free_count, 0, p.num_pages);
    }
}

// A workgroup to a request; the sums before it are taken anew by each.
__global__ __launch_bounds__(kGroup) void fill_kernel(Pool p, Reserve a, const int* needs, int rows) {
    __shared__ Two sums[kGroup / 64];
    const int tid = (int)threadIdx.x, lane = tid & 63, r = (int)blockIdx.x;
    const int free_count = needs[p.requests];
    const Request q = request_of(p, a.new_tokens, r);
    Two before{0, 0}, all;
    int64_t given = 0;
    for (int base = 0; base < (r == 0 ? p.requests : r); base += kGroup) {
        const int i = base + tid;
        const bool in = i < (r == 0 ? p.requests : r);
        const int n = in ? clampi(a.new_tokens[i], 0, kMostNew) : 0, need = in ? needs[i] : 0;
        const Two upto = group_scan<kGroup>(n, need, sums, &all);
        if (r == 0) {
            // the first workgroup finds what is given out in all: sums rise, so the last one granted
            const int mine = before.b + upto.b <= free_count ? (int)(before.b + upto.b) : 0;
            const int most = wave_max(mine);
            __syncthreads();
            if (lane == 0) sums[tid >> 6].a = most;
            __syncthreads();
            for (int w = 0; w < kGroup / 64; ++w) given = sums[w].a > given ? sums[w].a : given;
        }
        before.a += all.a;
        before.b += all.b;
    }
    if (r == 0) before = Two{0, 0};
    const int need = needs[r];
    const bool granted = q.fits && (need == 0 || before.b + need <= free_count);
    const int start = saturated(before.a);
    if (tid == 0) {
        if (r == 0) {
            a.starts[0] = 0;
            *p.free_count = free_count - (int)given;
        }
        a.starts[r + 1] = saturated(before.a + q.rows);
        a.kv_lens[r] = q.len + q.rows;
        if (a.granted != nullptr) a.granted[r] = granted;
    }
    if (granted && need > 0 && tid < 64) fill_absent(p, p.tables + (int64_t)r * p.stride, q.first, q.end, free_count - (int)before.b, lane);
    if (rows == 0) return;
    __syncthreads();
    for (int i = tid; i < q.rows && start + (int64_t)i < rows; i += kGroup) map_row(p, a, start + i, r, q.len, i);
    if (r == p.requests - 1)
        for (int64_t row = before.a + q.rows + tid; row < rows; row += kGroup) map_row(p, a, (int)row, r, 0, -1);
}

// Rows of batches too long for fill_kernel's workgroups to map.
__global__ __launch_bounds__(kGroup) void slots_kernel(Pool p, Reserve a, int rows) {
    const int row = (int)(blockIdx.x * kGroup + threadIdx.x);
    if (row >= rows) return;
    int lo = 0, hi = p.requests;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (a.starts[mid + 1] <= row)
            lo = mid + 1;
        else
            hi = mid;
    }
    const bool in = lo < p.requests;
    map_row(p, a, row, lo, in ? clampi(p.lens[lo], 0, p.width << p.page_shift) : 0, in ? row - a.starts[lo] : -1);
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

// All of it in one workgroup, a thread to PER neighbouring entries.
constexpr int kHeld = 16;  // the most
template <int PER>
__global__ __launch_bounds__(kThreads) void release_kernel(Pool p, const int* lens, int window) {
    __shared__ Two sums[kThreads / 64];
    const int tid = (int)threadIdx.x, entries = p.requests * p.width;
    const int free_count = clampi(*p.free_count, 0, p.num_pages);
    const int first = tid * PER;
    int r = first / p.width, j = first - r * p.width;
    int* at[PER];
    int entry[PER], len[PER], place[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const bool in = first + k < entries;  // the others look at entry 0, and keep it
        at[k] = p.tables + (in ? (int64_t)r * p.stride + j : 0);
        place[k] = j;
        entry[k] = *at[k];
        len[k] = lens[in ? r : 0];
        if (++j == p.width) {
            j = 0;
            ++r;
        }
    }
    int gone = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k)
        if (first + k < entries && goes(p, entry[k], place[k], clampi(len[k], 0, p.width << p.page_shift), window)) gone |= 1 << k;
    Two all;
    const int64_t upto = group_scan<kThreads>(__popc(gone), 0, sums, &all).a;
    const int64_t top = free_count + all.a;
    int64_t to = top - 1 - (upto - __popc(gone));
#pragma unroll
    for (int k = 0; k < PER; ++k)
        if (gone >> k & 1) {
            put_back(p, to--, entry[k]);
            *at[k] = -1;
        }
    // every length has been read: they may be the pool's own
    for (int i = tid; i < p.requests; i += kThreads) p.lens[i] = clampi(lens[i], 0, p.width << p.page_shift);
    if (tid == 0) *p.free_count = (int)(top < p.num_pages ? top : p.num_pages);
}

// Entries of a request's table that a thread of the next two kernels holds at once.
constexpr int kRun = 8;
// counts[r]: the pages of request r that go back; counts[requests]: the free pages before.
__global__ __launch_bounds__(kGroup) void count_kernel(Pool p, const int* lens, int window, int* counts) {
    __shared__ Two sums[kGroup / 64];
    const int r = (int)blockIdx.x, len = clampi(lens[r], 0, p.width << p.page_shift);
    const int* const table = p.tables + (int64_t)r * p.stride;
    int n = 0;
    for (int j0 = (int)threadIdx.x; j0 < p.width; j0 += kGroup * kRun) {
        int entry[kRun];
#pragma unroll
        for (int k = 0; k < kRun; ++k) entry[k] = j0 + k * kGroup < p.width ? table[j0 + k * kGroup] : -1;
#pragma unroll
        for (int k = 0; k < kRun; ++k) n += goes(p, entry[k], j0 + k * kGroup, len, window);
    }
    Two all;
    (void)group_scan<kGroup>(n, 0, sums, &all);
    if (threadIdx.x == 0) {
        counts[r] = (int)all.a;
        if (r == 0) counts[p.requests] = clampi(*p.free_count, 0, p.num_pages);
    }
}

__global__ __launch_bounds__(kGroup) void return_kernel(Pool p, const int* lens, int window, const int* counts) {
    __shared__ Two sums[kGroup / 64];
    const int tid = (int)threadIdx.x, r = (int)blockIdx.x;
    const int len = clampi(lens[r], 0, p.width << p.page_shift), base = counts[p.requests];
    Two all{0, 0};
    int64_t freed = 0, total = 0;
    for (int i0 = 0; i0 < p.requests; i0 += kGroup) {
        const int i = i0 + tid, n = i < p.requests ? counts[i] : 0;
        (void)group_scan<kGroup>(i < r ? n : 0, n, sums, &all);
        freed += all.a;
        total += all.b;
    }
    if (counts[r] > 0)
        for (int j0 = 0; j0 < p.width; j0 += kGroup * kRun) {
            int* const at = p.tables + (int64_t)r * p.stride + j0 + tid * kRun;
            int entry[kRun], gone = 0;
#pragma unroll
            for (int k = 0; k < kRun; ++k) entry[k] = j0 + tid * kRun + k < p.width ? at[k] : -1;
#pragma unroll
            for (int k = 0; k < kRun; ++k)
                if (goes(p, entry[k], j0 + tid * kRun + k, len, window)) gone |= 1 << k;
            const int64_t upto = group_scan<kGroup>(__popc(gone), 0, sums, &all).a;
            int64_t to = base + total - 1 - (freed + upto - __popc(gone));
#pragma unroll
            for (int k = 0; k < kRun; ++k)
                if (gone >> k & 1) {
                    put_back(p, to--, entry[k]);
                    at[k] = -1;
                }
            freed += all.a;
        }
    if (tid == 0) {
        p.lens[r] = len;
        if (r == 0) *p.free_count = (int)(base + total < p.num_pages ? base + total : p.num_pages);
    }
}

// One workgroup takes so many rows and requests (reserve), so many table entries (release).
constexpr int kFewRows = 4096, kFewRequests = kThreads, kFewEntries = kThreads * kHeld;
// From so many rows on, in all or to a request, the map is a launch of its own (4 us): one request of
// 16000 rows takes its workgroup 17 us, four of 8000 12, four of 2000 5, 96 of 200 3.7.
constexpr int kManyRows = 32768, kManyRowsEach = 4096;

}  // namespace

size_t reserve_scratch(const Pool& p, int rows) {
    return rows <= kFewRows && p.requests <= kFewRequests ? 0 : ((size_t)p.requests + 1) * sizeof(int);
}

hipError_t launch_reserve(const Pool& p, const Reserve& a, int rows, int* needs, hipStream_t stream) {
    if (a.positions == nullptr && a.slots == nullptr) rows = 0;
    if (needs == nullptr) {
        reserve_kernel<<<1, kThreads, 0, stream>>>(p, a, rows);
        return hipGetLastError();
    }
    need_kernel<<<(unsigned)ceil_div(p.requests, kGroup / 64), kGroup, 0, stream>>>(p, a, needs);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const bool apart = rows >= kManyRows || rows / p.requests >= kManyRowsEach;
    fill_kernel<<<(unsigned)p.requests, kGroup, 0, stream>>>(p, a, needs, apart ? 0 : rows);
    e = hipGetLastError();
    if (e != hipSuccess || !apart) return e;
    slots_kernel<<<(unsigned)ceil_div(rows, kGroup), kGroup, 0, stream>>>(p, a, rows);
    return hipGetLastError();
}

size_t release_scratch(const Pool& p) {
    return (int64_t)p.requests * p.width <= kFewEntries ? 0 : ((size_t)p.requests + 1) * sizeof(int);
}

hipError_t launch_release(const Pool& p, const int* lens, int window, int* counts, hipStream_t stream) {
    if (counts == nullptr) {
        const int per = ceil_div(p.requests * p.width, kThreads);
        if (per <= 1)
            release_kernel<1><<<1, kThreads, 0, stream>>>(p, lens, window);
        else if (per <= 4)
            release_kernel<4><<<1, kThreads, 0, stream>>>(p, lens, window);
        else
            release_kernel<kHeld><<<1, kThreads, 0, stream>>>(p, lens, window);
        return hipGetLastError();
    }
    count_kernel<<<(unsigned)p.requests, kGroup, 0, stream>>>(p, lens, window, counts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    return_kernel<<<(unsigned)p.requests, kGroup, 0, stream>>>(p, lens, window, counts);
    return hipGetLastError();
}

}  // namespace kv
