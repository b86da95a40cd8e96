// C ABI of the sampling calls (include/gemma4_qmm.h): argument checks and dispatch.
#include "gemma4_qmm.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "runtime_common.h"
#include "verify_kernels.h"

namespace {

using namespace rt;

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

Gemma4Status bad(const char* name, const std::string& what) { return fail(GEMMA4_ERR_INVALID_ARGUMENT, std::string(name) + ": " + what); }
Gemma4Status unsupported(const char* name, const char* what) {
    return fail(GEMMA4_ERR_UNSUPPORTED_CONFIG, std::string(name) + ": " + what);
}

Gemma4Status check_logits(const Gemma4Logits* l, uint32_t rows, uint32_t vocab, const char* which, const char* name, verify::Logits* out) {
    if (l == nullptr || (l->x_dev == nullptr && rows > 0)) return bad(name, std::string("requires non-null ") + which + "logits");
    if (l->dtype != GEMMA4_QMM_BF16 && l->dtype != GEMMA4_QMM_F32) return bad(name, std::string(which) + "logits must be BF16 or F32");
    if (!aligned(l->x_dev, l->dtype == GEMMA4_QMM_F32 ? 4 : 2)) return bad(name, std::string(which) + "logits must be aligned to their type");
    if (l->stride < vocab || l->stride > ((uint64_t)1 << 40))
        return bad(name, std::string(which) + "logits' stride must hold vocab values (and at most 2^40)");
    if (!(std::isfinite(l->softcap) && l->softcap >= 0)) return bad(name, std::string(which) + "softcap must be finite and >= 0 (0: none)");
    *out = verify::Logits{l->x_dev, (int64_t)l->stride, l->dtype == GEMMA4_QMM_F32, l->softcap};
    return GEMMA4_OK;
}

Gemma4Status check_common(uint32_t rows, uint32_t vocab, const float* uniforms, float heat, const float* heats, const int32_t* out,
                          const char* name) {
    if (vocab == 0 || vocab > (1u << 24)) return unsupported(name, "vocab must be 1 to 2^24");
    if (rows > (1u << 20)) return unsupported(name, "rows must be at most 2^20");
    if (heats == nullptr && !(std::isfinite(heat) && heat >= 0)) return bad(name, "temperature must be finite and >= 0 (0: greedy)");
    if (rows == 0) return GEMMA4_OK;
    if (uniforms == nullptr || out == nullptr) return bad(name, "requires non-null uniforms and out_tokens");
    if (!aligned(uniforms, 4) || !aligned(out, 4) || !aligned(heats, 4))
        return bad(name, "uniforms, temperatures and out_tokens must be 4-byte aligned");
    return GEMMA4_OK;
}

Span logits_span(const verify::Logits& l, const verify::Args& a) {
    return Span{l.x, ((uint64_t)(a.rows - 1) * (uint64_t)l.stride + (uint64_t)a.vocab) * (l.f32 ? 4 : 2), false};
}

Gemma4Status run(const verify::Args& a, const char* name, void* stream) {
    if (!verify::fits(a)) return unsupported(name, "rows * vocab is too large for one launch");
    const uint64_t rows = 4 * (uint64_t)a.rows, requests = 4 * (uint64_t)a.requests;
    if (clash({logits_span(a.target, a), logits_span(a.draft, a), {a.tokens, rows, false}, {a.starts, requests + 4, false},
               {a.uniforms, a.starts != nullptr ? 2 * rows : rows, false}, {a.heats, requests, false}, {a.out, rows, true},
               {a.accepted, requests, true}}))
        return bad(name, "an array that is written must not overlap another");
    Scratch sc;
    sc.stream = static_cast<hipStream_t>(stream);
    hipError_t e = hipGetDevice(&sc.device);
    if (e != hipSuccess) return hip_fail((std::string(name) + ": hipGetDevice").c_str(), e);
    void* ws = nullptr;
    e = sc.take(verify::scratch_bytes(a), &ws);
    if (e != hipSuccess)
        return fail(GEMMA4_ERR_MEMORY_GUARD, std::string(name) + ": workspace allocation failed: " + hipGetErrorString(e));
    e = verify::launch(a, ws, sc.stream);
    const hipError_t er = sc.release();
    if (e != hipSuccess) return hip_fail((std::string(name) + ": launch").c_str(), e);
    if (er != hipSuccess) return hip_fail((std::string(name) + ": workspace release").c_str(), er);
    return ok();
}

}  // namespace

extern "C" {

Gemma4Status gemma4_sample(const Gemma4Logits* logits, uint32_t rows, uint32_t vocab, const float* uniforms_dev, float temperature,
                           const float* temperatures_dev, int32_t* out_tokens_dev, void* stream) {
    try {
        const char* const name = "gemma4_sample";
        verify::Args a{};
        Gemma4Status st = check_common(rows, vocab, uniforms_dev, temperature, temperatures_dev, out_tokens_dev, name);
        if (st == GEMMA4_OK) st = check_logits(logits, rows, vocab, "", name, &a.target);
        if (st != GEMMA4_OK) return st;
        if (rows == 0) return ok();
        a.uniforms = uniforms_dev;
        a.heats = temperatures_dev;
        a.heat = temperature;
        a.requests = a.rows = (int)rows;
        a.vocab = (int)vocab;
        a.out = out_tokens_dev;
        return run(a, name, stream);
    } catch (...) {
        return fail_nothrow(GEMMA4_ERR_RUNTIME, "gemma4_sample: unexpected native exception");
    }
}

Gemma4Status gemma4_verify_drafts(const Gemma4Logits* logits, const Gemma4Logits* draft_logits, const int32_t* tokens_dev,
                                  const int32_t* query_starts_dev, uint32_t requests, uint32_t rows, uint32_t vocab,
                                  const float* uniforms_dev, float temperature, const float* temperatures_dev, int32_t* out_tokens_dev,
                                  int32_t* accepted_dev, void* stream) {
    try {
        const char* const name = "gemma4_verify_drafts";
        verify::Args a{};
        Gemma4Status st = check_common(rows, vocab, uniforms_dev, temperature, temperatures_dev, out_tokens_dev, name);
        if (st == GEMMA4_OK) st = check_logits(logits, rows, vocab, "", name, &a.target);
        if (st == GEMMA4_OK && draft_logits != nullptr) st = check_logits(draft_logits, rows, vocab, "draft ", name, &a.draft);
        if (st != GEMMA4_OK) return st;
        if (draft_logits != nullptr && draft_logits->dtype != logits->dtype) return bad(name, "logits and draft logits must be of one type");
        if (requests == 0 || requests > (1u << 20)) return bad(name, "requests must be 1 to 2^20");
        if (rows == 0) return ok();
        if (tokens_dev == nullptr || query_starts_dev == nullptr || accepted_dev == nullptr)
            return bad(name, "requires non-null tokens, query_starts and accepted");
        if (!aligned(tokens_dev, 4) || !aligned(query_starts_dev, 4) || !aligned(accepted_dev, 4))
            return bad(name, "tokens, query_starts and accepted must be 4-byte aligned");
        a.tokens = tokens_dev;
        a.starts = query_starts_dev;
        a.uniforms = uniforms_dev;
        a.heats = temperatures_dev;
        a.heat = temperature;
        a.requests = (int)requests;
        a.rows = (int)rows;
        a.vocab = (int)vocab;
        a.out = out_tokens_dev;
        a.accepted = accepted_dev;
        return run(a, name, stream);
    } catch (...) {
        return fail_nothrow(GEMMA4_ERR_RUNTIME, "gemma4_verify_drafts: unexpected native exception");
    }
}

}  // extern "C"
