// Launch interface of the sampling kernels (verify.hip); arguments are checked by
// verify_runtime.cpp.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace verify {

// Rows of logits: row r at x + r * stride elements.
struct Logits {
    const void* x;  // null: none (the drafter's)
    int64_t stride;
    int f32;        // else bf16
    float cap;      // 0: none
};

struct Args {
    Logits target, draft;
    const int* tokens;       // the rows' own tokens; null: no drafts, a request a row
    const int* starts;       // [requests + 1]; null likewise
    const float* uniforms;   // [rows, 2], or [rows] without drafts
    const float* heats;      // temperatures [requests]; null: `heat` for all
    float heat;
    int requests, rows, vocab;
    int* out;                // [rows]
    int* accepted;           // [requests]; may be null
};

bool fits(const Args& a);  // whether the launches can count their threads
size_t scratch_bytes(const Args& a);
hipError_t launch(const Args& a, void* scratch, hipStream_t stream);

}  // namespace verify
