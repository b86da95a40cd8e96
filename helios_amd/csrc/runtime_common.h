// What the C ABI's entry points share (qmm_runtime.cpp, kv_runtime.cpp): the last
// error, the scratch memory kept per (device, stream) and the device guard.
//
// Conventions of the reference runtime (native/gemma4_mlx/src/runtime.cc): status
// codes and a thread-local last-error buffer (runtime.cc:46, :116-133).
#pragma once

#include "gemma4_qmm.h"

#include <hip/hip_runtime.h>

#include <cstdio>
#include <memory>
#include <mutex>
#include <string>
#include <thread>
#include <vector>

// hidden: two builds of the library loaded into one process keep their own
namespace rt __attribute__((visibility("hidden"))) {

inline thread_local char g_last_error[512] = "";

// Records the message (truncated to the buffer) and returns status.  The const char*
// forms build no std::string, so they cannot throw: catch blocks use them.
inline Gemma4Status fail_nothrow(Gemma4Status status, const char* message) noexcept {
    std::snprintf(g_last_error, sizeof(g_last_error), "%s", message);
    return status;
}

inline Gemma4Status fail(Gemma4Status status, const char* message) noexcept { return fail_nothrow(status, message); }

inline Gemma4Status fail(Gemma4Status status, const std::string& message) noexcept {
    return fail_nothrow(status, message.c_str());
}

inline Gemma4Status ok() {
    g_last_error[0] = '\0';
    return GEMMA4_OK;
}

inline Gemma4Status hip_fail(const char* where, hipError_t e) {
    return fail(GEMMA4_ERR_RUNTIME, std::string(where) + ": " + hipGetErrorName(e) + " (" +
                                        hipGetErrorString(e) + ")");
}

// Per-device stream-ordered memory pool for per-call scratch (the GEMM's group sums
// of x).  Its release threshold is unlimited, so after the first calls allocations
// are served from memory the pool keeps; it is separate from the device's default
// pool, so callers' own allocators are untouched.  Allocations are stream-ordered,
// which keeps forward reentrant across streams.
inline std::mutex g_pool_mu;
inline hipMemPool_t g_pools[64] = {};

inline hipError_t scratch_pool(int device, hipMemPool_t* out) {
    if (device < 0 || device >= 64) return hipErrorInvalidDevice;
    std::lock_guard<std::mutex> lock(g_pool_mu);
    if (g_pools[device] == nullptr) {
        hipMemPoolProps props{};
        props.allocType = hipMemAllocationTypePinned;
        props.handleTypes = hipMemHandleTypeNone;
        props.location.type = hipMemLocationTypeDevice;
        props.location.id = device;
        hipMemPool_t pool = nullptr;
        hipError_t e = hipMemPoolCreate(&pool, &props);
        if (e != hipSuccess) return e;
        uint64_t keep = UINT64_MAX;
        e = hipMemPoolSetAttribute(pool, hipMemPoolAttrReleaseThreshold, &keep);
        if (e != hipSuccess) {
            (void)hipMemPoolDestroy(pool);
            return e;
        }
        g_pools[device] = pool;
    }
    *out = g_pools[device];
    return hipSuccess;
}

// Device memory kept per (device, stream) for the scratch of the calls on that stream.
// Work on one stream runs in order, so consecutive calls can reuse it; `mu` is held
// for a whole call (its scratch and its launches), so calls from several host threads
// on one stream cannot interleave their launches.  It grows by allocating a larger
// buffer when a call is not being captured into a graph.  An outgrown buffer that a
// capture took pieces of is kept (a graph captured earlier may still use it) until
// gemma4_qmm_release_scratch; one no capture used is freed once the stream is idle.  A
// stream-ordered pool allocation per call (and, under capture, an allocation node per
// call in the graph) cost 5-10 us per forward on the GPU: k_proj 2048x3840 at 512 rows,
// split four ways, 31 us per forward in a graph against 22 us with the workspace.
struct StreamWorkspace {
    int device = -1;
    hipStream_t stream = nullptr;
    std::thread::id thread;  // hipStreamPerThread: a different stream in every thread
    char* buf = nullptr;
    size_t cap = 0;
    bool buf_captured = false;    // a graph capture took pieces of buf
    std::vector<char*> retired;  // outgrown buffers that captures used
    std::mutex mu;
};
inline std::mutex g_ws_mu;
inline std::vector<std::unique_ptr<StreamWorkspace>> g_ws;

inline StreamWorkspace* stream_workspace(int device, hipStream_t stream) {
    const std::thread::id thread = stream == hipStreamPerThread ? std::this_thread::get_id() : std::thread::id();
    std::lock_guard<std::mutex> lock(g_ws_mu);
    for (auto& w : g_ws)
        if (w->device == device && w->stream == stream && w->thread == thread) return w.get();
    g_ws.push_back(std::make_unique<StreamWorkspace>());
    g_ws.back()->device = device;
    g_ws.back()->stream = stream;
    g_ws.back()->thread = thread;
    return g_ws.back().get();
}

// Device memory one call borrows for its kernels' scratch (the GEMM's group sums and
// split-K partials, the greedy head's keys, LoRA's x.A^T, attention's partial sums):
// consecutive 256-byte-aligned pieces of the stream's workspace, or, for the
// allocation-free entry point, of `scratch`.  A call captured into a graph whose stream
// workspace is too small takes stream-ordered allocations from the private pool
// instead, released on the same stream after the launches (allocation nodes of the
// graph).
struct Scratch {
    hipStream_t stream = nullptr;
    int device = 0;
    bool fixed = false;  // pieces of `scratch`: no allocation and nothing to release
    char* base = nullptr;
    size_t cap = 0, used = 0;
    StreamWorkspace* ws = nullptr;  // the stream's workspace (not fixed)
    std::unique_lock<std::mutex> ws_lock;
    void* owned[2] = {};
    int n_owned = 0;

    // bytes still available (fixed mode; unlimited otherwise)
    size_t room() const { return fixed ? cap - used : ~(size_t)0; }

    hipError_t take(size_t bytes, void** out) {
        *out = nullptr;
        if (bytes == 0) return hipSuccess;
        const size_t need = (bytes + 255) & ~(size_t)255;
        if (fixed) {
            if (need > cap - used) return hipErrorOutOfMemory;
            *out = base + used;
            used += need;
            return hipSuccess;
        }
        if (ws == nullptr) {
            ws = stream_workspace(device, stream);
            ws_lock = std::unique_lock<std::mutex>(ws->mu);
            base = ws->buf;
            cap = ws->cap;
            used = 0;
        }
        hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
        const bool capturing =
            hipStreamIsCapturing(stream, &capture) != hipSuccess || capture != hipStreamCaptureStatusNone;
        if (need <= cap - used) {
            *out = base + used;
            used += need;
            if (capturing) ws->buf_captured = true;
            return hipSuccess;
        }
        if (!capturing) {
            // grow: a new buffer for this and later calls.  Pieces this call took from
            // the old one stay valid (it is released only after this call's launches,
            // see `release`), as does every graph that used it.  (The pool for the
            // fallback below is made here too, outside any capture.)
            hipMemPool_t pool = nullptr;
            (void)scratch_pool(device, &pool);
            size_t ncap = ws->cap * 2 > need ? ws->cap * 2 : need;
            ncap = (ncap + ((size_t)1 << 20) - 1) & ~(((size_t)1 << 20) - 1);
            char* nb = nullptr;
            if (hipMalloc(&nb, ncap) == hipSuccess) {
                if (ws->buf != nullptr) {
                    if (ws->buf_captured)
                        ws->retired.push_back(ws->buf);
                    else
                        outgrown = ws->buf;
                }
                ws->buf = base = nb;
                ws->cap = cap = ncap;
                ws->buf_captured = false;
                *out = base;
                used = need;
                return hipSuccess;
            }
            (void)hipGetLastError();  // out of memory: fall back to the pool
        }
        if (n_owned == 2) return hipErrorInvalidValue;
        hipMemPool_t pool = nullptr;
        hipError_t e = scratch_pool(device, &pool);
        if (e == hipSuccess) e = hipMallocFromPoolAsync(out, bytes, pool, stream);
        if (e == hipSuccess) owned[n_owned++] = *out;
        return e;
    }

    // queues the release of every pool allocation after the work on the stream
    hipError_t release() {
        hipError_t first = hipSuccess;
        for (int i = 0; i < n_owned; ++i) {
            const hipError_t e = hipFreeAsync(owned[i], stream);
            if (first == hipSuccess) first = e;
        }
        n_owned = 0;
        if (outgrown != nullptr) {
            // an outgrown buffer no capture used: freed once the stream's work (this
            // call's launches included) is done
            hipError_t e = hipStreamSynchronize(stream);
            if (e == hipSuccess) e = hipFree(outgrown);
            outgrown = nullptr;
            if (first == hipSuccess) first = e;
        }
        return first;
    }

    char* outgrown = nullptr;  // the stream's previous buffer, freed by release()
};

// Restores the caller's current device on scope exit.
struct DeviceGuard {
    int saved = -1;
    bool changed = false;
    hipError_t enter(int device) {
        hipError_t e = hipGetDevice(&saved);
        if (e != hipSuccess) return e;
        if (saved != device) {
            e = hipSetDevice(device);
            changed = (e == hipSuccess);
        }
        return e;
    }
    ~DeviceGuard() {
        if (changed) (void)hipSetDevice(saved);
    }
};

}  // namespace rt
