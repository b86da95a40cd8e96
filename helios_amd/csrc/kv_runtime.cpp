// C ABI of the paged-cache calls (include/gemma4_qmm.h): argument checks and dispatch.
#include "gemma4_qmm.h"

#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <string>

#include "kv_index.h"
#include "kv_kernels.h"
#include "overlap.h"
#include "runtime_common.h"

namespace {

using namespace rt;

std::atomic<uint32_t> g_attention_kernel{0};

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

Gemma4Status bad(const char* name, const char* what) { return fail(GEMMA4_ERR_INVALID_ARGUMENT, std::string(name) + ": " + what); }
Gemma4Status unsupported(const char* name, const char* what) {
    return fail(GEMMA4_ERR_UNSUPPORTED_CONFIG, std::string(name) + ": " + what);
}

bool head_dim_ok(uint32_t d) { return d == 64 || d == 128 || d == 256 || d == 512; }

Gemma4Status check_pages(const Gemma4KvPages* p, const char* name, kv::Pages* out) {
    if (p == nullptr) return bad(name, "requires non-null pages");
    if (p->k_dev == nullptr || p->v_dev == nullptr) return bad(name, "requires non-null k and v pages");
    if (!head_dim_ok(p->head_dim)) return unsupported(name, "head_dim must be 64, 128, 256 or 512");
    if (p->page_size < 16 || p->page_size > 65536 || (p->page_size & (p->page_size - 1)) != 0)
        return unsupported(name, "page_size must be a power of two from 16 to 65536");
    if (p->dtype != GEMMA4_KV_BF16 && p->dtype != GEMMA4_KV_E4M3)
        return bad(name, "the cache dtype must be BF16 or E4M3");
    if (p->num_pages == 0 || p->num_pages > (1u << 30) || p->kv_heads == 0 || p->kv_heads > 4096)
        return bad(name, "num_pages and kv_heads must be > 0 (and at most 2^30 and 4096)");
    const uint64_t elt = p->dtype == GEMMA4_KV_E4M3 ? 1 : 2, most = (uint64_t)1 << 40;
    if (p->page_stride > most || p->token_stride > most || p->head_stride > most)
        return unsupported(name, "a stride exceeds 2^40 elements");
    if (!aligned(p->k_dev, 16) || !aligned(p->v_dev, 16) || p->page_stride * elt % 16 != 0 ||
        p->token_stride * elt % 16 != 0 || p->head_stride * elt % 16 != 0)
        return bad(name, "pages and their strides must be multiples of 16 bytes");
    if (p->token_stride < p->head_dim || (p->kv_heads > 1 && p->head_stride < p->head_dim) ||
        (p->num_pages > 1 && p->page_stride < p->head_dim))
        return bad(name, "a stride is shorter than head_dim");
    // the kernels' offsets within 64 tokens are 32 bits wide
    if (p->token_stride * elt > ((uint64_t)1 << 24)) return unsupported(name, "token_stride exceeds 16 MiB");
    const bool fp8 = p->dtype == GEMMA4_KV_E4M3;
    if (fp8 && !(std::isfinite(p->k_scale) && std::isfinite(p->v_scale) && p->k_scale > 0 && p->v_scale > 0))
        return bad(name, "k_scale and v_scale must be finite and > 0");
    out->k = static_cast<char*>(p->k_dev);
    out->v = static_cast<char*>(p->v_dev);
    out->page_stride = (int64_t)p->page_stride;
    out->token_stride = (int64_t)p->token_stride;
    out->head_stride = (int64_t)p->head_stride;
    out->num_pages = (int)p->num_pages;
    out->page_shift = __builtin_ctz(p->page_size);
    out->kv_heads = (int)p->kv_heads;
    out->head_dim = (int)p->head_dim;
    out->fp8 = fp8;
    out->k_scale = fp8 ? p->k_scale : 1.0f;
    out->v_scale = fp8 ? p->v_scale : 1.0f;
    return GEMMA4_OK;
}

// Block scales: pages as those of e4m3 whose own scales are 1.
Gemma4Status check_scaled(const Gemma4KvPages* p, const Gemma4KvScales* sc, const char* name, kv::Pages* pages, kv::BlockScales* out) {
    if (p == nullptr) return bad(name, "requires non-null pages");
    if (sc == nullptr || sc->k_dev == nullptr || sc->v_dev == nullptr) return bad(name, "requires non-null k and v scales");
    if (p->dtype != GEMMA4_KV_E4M3) return bad(name, "block scales belong to E4M3 pages");
    Gemma4KvPages own = *p;
    own.k_scale = own.v_scale = 1.0f;
    const Gemma4Status st = check_pages(&own, name, pages);
    if (st != GEMMA4_OK) return st;
    if (sc->block < 16 || sc->block > 256 || (sc->block & (sc->block - 1)) != 0 || sc->block > p->page_size)
        return unsupported(name, "a scale's block must be a power of two from 16 to 256, at most page_size");
    const uint64_t per = p->page_size / sc->block, most = (uint64_t)1 << 40;
    if (sc->page_stride > most || sc->head_stride > most) return unsupported(name, "a scale stride exceeds 2^40 bytes");
    if ((p->kv_heads > 1 && sc->head_stride < per) || (p->num_pages > 1 && sc->page_stride < per))
        return bad(name, "a scale stride is shorter than a page's blocks");
    *out = kv::BlockScales{sc->k_dev, sc->v_dev, (int64_t)sc->page_stride, (int64_t)sc->head_stride, __builtin_ctz(sc->block)};
    return GEMMA4_OK;
}

Gemma4Status check_batch(const Gemma4KvBatch* b, const kv::Pages& pages, const char* name, kv::Batch* out) {
    if (b == nullptr) return bad(name, "requires a non-null batch");
    if (b->requests == 0 || b->requests > (1u << 20)) return bad(name, "requests must be 1 to 2^20");
    if (b->tokens >= (1u << 24)) return unsupported(name, "tokens must be under 2^24");
    if (b->query_starts_dev == nullptr || b->kv_lens_dev == nullptr || b->block_tables_dev == nullptr)
        return bad(name, "requires non-null query_starts, kv_lens and block_tables");
    if (!aligned(b->query_starts_dev, 4) || !aligned(b->kv_lens_dev, 4) || !aligned(b->block_tables_dev, 4))
        return bad(name, "the batch's arrays must be 4-byte aligned");
    if (b->pages_per_request == 0 || b->table_stride < b->pages_per_request)
        return bad(name, "pages_per_request must be > 0 and at most table_stride");
    if (b->table_stride > 0x7FFFFFFFu) return unsupported(name, "table_stride must be under 2^31");  // an int in the kernels
    if (((uint64_t)b->pages_per_request << pages.page_shift) > ((uint64_t)1 << 30))
        return unsupported(name, "a request's pages exceed 2^30 tokens");
    out->starts = b->query_starts_dev;
    out->kv_lens = b->kv_lens_dev;
    out->tables = b->block_tables_dev;
    out->requests = (int)b->requests;
    out->tokens = (int)b->tokens;
    out->width = (int)b->pages_per_request;
    out->stride = (int)b->table_stride;
    return GEMMA4_OK;
}

Gemma4Status check_rope(const Gemma4Rope* r, uint32_t head_dim, const char* name, kv::Rope* out) {
    *out = kv::Rope{nullptr, 0, 8};
    if (r == nullptr || r->pairs == 0) return GEMMA4_OK;
    if (r->inv_freq_dev == nullptr || !aligned(r->inv_freq_dev, 4)) return bad(name, "rope needs inv_freq, 4-byte aligned");
    if (r->pairs % 8 != 0 || r->pairs > head_dim / 2) return bad(name, "rope pairs must be a multiple of 8, at most head_dim / 2");
    if (r->distance != 1 && (r->distance % 8 != 0 || r->distance < r->pairs || r->distance > head_dim ||
                             r->distance + r->pairs > head_dim))
        return bad(name, "rope distance must be 1, or a multiple of 8 from pairs to head_dim - pairs");
    *out = kv::Rope{r->inv_freq_dev, (int)r->pairs, (int)r->distance};
    return GEMMA4_OK;
}

Gemma4Status check_heads(const Gemma4Heads* h, uint32_t head_dim, bool has_out, const char* which, const char* name,
                         kv::Heads* out) {
    const auto at = [&](const char* what) { return std::string(name) + ": " + which + what; };
    if (h->x_dev == nullptr || (has_out && h->out_dev == nullptr))
        return fail(GEMMA4_ERR_INVALID_ARGUMENT, at(" requires non-null pointers"));
    if (!has_out && h->out_dev != nullptr)
        return fail(GEMMA4_ERR_INVALID_ARGUMENT, at(" goes to the cache: out_dev must be NULL"));
    if (h->count == 0 || h->count > 65536) return fail(GEMMA4_ERR_INVALID_ARGUMENT, at(" count must be 1 to 65536"));
    if (!aligned(h->x_dev, 16) || !aligned(h->out_dev, 16) || !aligned(h->weight_dev, 16) || h->x_stride % 8 != 0 ||
        h->out_stride % 8 != 0)
        return fail(GEMMA4_ERR_INVALID_ARGUMENT, at(" pointers and strides must be multiples of 16 bytes"));
    const uint64_t least = (uint64_t)h->count * head_dim, most = (uint64_t)1 << 32;
    if (h->x_stride < least || (has_out && h->out_stride < least) || h->x_stride > most || h->out_stride > most)
        return fail(GEMMA4_ERR_INVALID_ARGUMENT, at(" stride must hold count * head_dim elements (and at most 2^32)"));
    if (h->norm > 1) return fail(GEMMA4_ERR_INVALID_ARGUMENT, at(" norm must be 0 or 1"));
    if (h->norm == 1 && !(std::isfinite(h->eps) && h->eps >= 0))
        return fail(GEMMA4_ERR_INVALID_ARGUMENT, at(" eps must be finite and >= 0"));
    out->x = h->x_dev;
    out->out = has_out ? h->out_dev : nullptr;
    out->weight = h->norm ? h->weight_dev : nullptr;
    out->x_stride = (int64_t)h->x_stride;
    out->out_stride = (int64_t)h->out_stride;
    out->count = (int)h->count;
    out->norm = (int)h->norm;
    out->eps = h->eps;
    return GEMMA4_OK;
}

Gemma4Status check_pool(const Gemma4KvPool* p, const char* name, kv::Pool* out) {
    if (p == nullptr) return bad(name, "requires a non-null pool");
    if (p->free_pages_dev == nullptr || p->free_count_dev == nullptr || p->lens_dev == nullptr || p->block_tables_dev == nullptr)
        return bad(name, "requires non-null free_pages, free_count, lens and block_tables");
    if (!aligned(p->free_pages_dev, 4) || !aligned(p->free_count_dev, 4) || !aligned(p->lens_dev, 4) || !aligned(p->block_tables_dev, 4))
        return bad(name, "the pool's arrays must be 4-byte aligned");
    if (p->page_size < 16 || p->page_size > 65536 || (p->page_size & (p->page_size - 1)) != 0)
        return unsupported(name, "page_size must be a power of two from 16 to 65536");
    if (p->num_pages == 0 || p->num_pages > (1u << 30)) return bad(name, "num_pages must be 1 to 2^30");
    if (p->requests == 0 || p->requests > (1u << 20)) return bad(name, "requests must be 1 to 2^20");
    if (p->pages_per_request == 0 || p->table_stride < p->pages_per_request)
        return bad(name, "pages_per_request must be > 0 and at most table_stride");
    if (p->table_stride > 0x7FFFFFFFu) return unsupported(name, "table_stride must be under 2^31");
    if ((uint64_t)p->pages_per_request * p->page_size > ((uint64_t)1 << 30))
        return unsupported(name, "a request's pages exceed 2^30 tokens");
    *out = kv::Pool{p->free_pages_dev, p->free_count_dev, p->lens_dev, p->block_tables_dev, (int64_t)p->table_stride, (int)p->num_pages,
                    __builtin_ctz(p->page_size), (int)p->requests, (int)p->pages_per_request};
    return GEMMA4_OK;
}

uint64_t table_bytes(const kv::Pool& p) { return 4 * ((uint64_t)(p.requests - 1) * (uint64_t)p.stride + (uint64_t)p.width); }

// The scaled append's K and V, and its q, k and v, are workgroups of one launch in any order: null, or which of
// the arrays written would take from another.
const char* mixed(const kv::HeadArgs& a, const kv::BlockScales& sc) {
    const kv::Pages& p = a.pages;
    const uint64_t pages = (uint64_t)p.num_pages, heads = (uint64_t)p.kv_heads, slots = 1ull << p.page_shift, dim = (uint64_t)p.head_dim;
    if (overlap(p.k, dim, p.v, dim, {{pages, (uint64_t)p.page_stride}, {slots, (uint64_t)p.token_stride}, {heads, (uint64_t)p.head_stride}}))
        return "the k and v pages must not overlap";
    const uint64_t per = slots >> sc.block_shift;
    if (overlap(sc.k, per, sc.v, per, {{pages, (uint64_t)sc.page_stride}, {heads, (uint64_t)sc.head_stride}}))
        return "the k and v scales must not overlap";
    const kv::Heads& q = a.part[0];
    if (q.count == 0) return nullptr;
    const uint64_t rows = (uint64_t)a.rows;
    const auto in = [&](const kv::Heads& h) { return Rows{h.x, 2 * (uint64_t)h.x_stride, 2 * (uint64_t)h.count * dim}; };
    const Rows out{q.out, 2 * (uint64_t)q.out_stride, 2 * (uint64_t)q.count * dim};
    if (overlap(out, in(a.part[1]), rows) || overlap(out, in(a.part[2]), rows)) return "q's out must not overlap k's or v's rows";
    const bool in_place = q.out == q.x && (q.out_stride == q.x_stride || rows == 1);
    return !in_place && overlap(out, in(q), rows) ? "q's out must be its x or not overlap it" : nullptr;
}

// scales: null, or those of the pages' blocks
Gemma4Status append(const char* name, const Gemma4KvPages* pages, const Gemma4KvScales* scales, bool scaled, const Gemma4KvBatch* batch,
                    const Gemma4Heads* q, const Gemma4Heads* k, const Gemma4Heads* v, const Gemma4Rope* rope, void* stream) {
    kv::HeadArgs a{};
    kv::BlockScales sc{};
    Gemma4Status st = scaled ? check_scaled(pages, scales, name, &a.pages, &sc) : check_pages(pages, name, &a.pages);
    if (st == GEMMA4_OK) st = check_batch(batch, a.pages, name, &a.batch);
    if (st == GEMMA4_OK) st = check_rope(rope, pages->head_dim, name, &a.rope);
    if (st != GEMMA4_OK) return st;
    if (k == nullptr || v == nullptr) return bad(name, "requires non-null k and v");
    if (k->count != pages->kv_heads || v->count != pages->kv_heads)
        return bad(name, "k and v must have the cache's kv_heads");
    if (batch->tokens == 0) return ok();
    if (q != nullptr) st = check_heads(q, pages->head_dim, true, "q", name, &a.part[0]);
    if (st == GEMMA4_OK) st = check_heads(k, pages->head_dim, false, "k", name, &a.part[1]);
    if (st == GEMMA4_OK) st = check_heads(v, pages->head_dim, false, "v", name, &a.part[2]);
    if (st != GEMMA4_OK) return st;
    a.rows = (int)batch->tokens;
    a.head_dim = (int)pages->head_dim;
    a.append = 1;
    if (scaled && !kv::scaled_append_fits(a, sc))
        return unsupported(name, "tokens * heads is too large for one launch");
    if (scaled)
        if (const char* const what = mixed(a, sc)) return bad(name, what);
    const hipError_t e = scaled ? kv::launch_scaled_append(a, sc, static_cast<hipStream_t>(stream))
                                : kv::launch_heads(a, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail((std::string(name) + ": launch").c_str(), e);
    return ok();
}

Gemma4Status attend(const char* name, const Gemma4KvPages* pages, const Gemma4KvScales* scales, bool scaled, const Gemma4KvBatch* batch,
                    const uint16_t* q_dev, uint64_t q_stride, uint32_t q_heads, float scale, uint32_t window, uint16_t* out_dev,
                    uint64_t out_stride, float* lse_dev, void* stream) {
    kv::AttnArgs a{};
    kv::BlockScales sc{};
    Gemma4Status st = scaled ? check_scaled(pages, scales, name, &a.pages, &sc) : check_pages(pages, name, &a.pages);
    if (st == GEMMA4_OK) st = check_batch(batch, a.pages, name, &a.batch);
    if (st != GEMMA4_OK) return st;
    if (q_heads == 0 || q_heads > 65536 || q_heads % pages->kv_heads != 0)
        return bad(name, "q_heads must be a multiple of kv_heads (and at most 65536)");
    if (!std::isfinite(scale)) return bad(name, "scale must be finite");
    if (window > (1u << 30)) return unsupported(name, "window exceeds 2^30 (0: none)");
    if (batch->tokens == 0) return ok();
    if (q_dev == nullptr || out_dev == nullptr) return bad(name, "requires non-null q and out");
    if (!aligned(q_dev, 16) || !aligned(out_dev, 16) || q_stride % 8 != 0 || out_stride % 8 != 0 || !aligned(lse_dev, 4))
        return bad(name, "q, out and their strides must be multiples of 16 bytes, lse of 4");
    const uint64_t least = (uint64_t)q_heads * pages->head_dim, most = (uint64_t)1 << 32;
    if (q_stride < least || out_stride < least || q_stride > most || out_stride > most)
        return bad(name, "q_stride and out_stride must hold q_heads * head_dim elements (and at most 2^32)");
    a.q = q_dev;
    a.out = out_dev;
    a.lse = lse_dev;
    a.q_stride = (int64_t)q_stride;
    a.out_stride = (int64_t)out_stride;
    a.q_heads = (int)q_heads;
    a.window = (int)window;
    a.scale = scale;
    a.kernel = (int)g_attention_kernel.load(std::memory_order_relaxed);
    // a launch's workgroups are counted in 31 bits
    if (((uint64_t)batch->tokens + batch->requests + 1) * q_heads > 0x7FFFFFFFull)
        return unsupported(name, "tokens * q_heads exceeds 2^31");
    kv::AttnPlan plan = kv::plan_attention(a, scaled);
    a.tile_from = plan.tile_from;
    // a launch's threads are counted in 32 bits, 512 to a workgroup at most
    for (const kv::Items* it : {&plan.tiles, &plan.rows})
        if ((uint64_t)it->items * (uint64_t)it->parts >= (1u << 23))
            return unsupported(name, "tokens * q_heads is too large for one launch");
    Scratch scratch;
    scratch.stream = static_cast<hipStream_t>(stream);
    hipError_t e = hipGetDevice(&scratch.device);
    if (e != hipSuccess) return hip_fail((std::string(name) + ": hipGetDevice").c_str(), e);
    const int d = a.pages.head_dim;
    const size_t wide_o = plan.o_bytes(plan.tiles, kv::kWideRows, d), wide_ml = plan.ml_bytes(plan.tiles, kv::kWideRows);
    const size_t thin_o = plan.o_bytes(plan.rows, kv::kThinRows, d), thin_ml = plan.ml_bytes(plan.rows, kv::kThinRows);
    void* ws = nullptr;
    e = scratch.take(wide_o + wide_ml + thin_o + thin_ml, &ws);
    if (e != hipSuccess)
        return fail(GEMMA4_ERR_MEMORY_GUARD, std::string(name) + ": workspace allocation failed: " + hipGetErrorString(e));
    char* at = static_cast<char*>(ws);
    plan.tiles.part_o = reinterpret_cast<float*>(at);
    plan.tiles.part_ml = reinterpret_cast<float2*>(at + wide_o);
    plan.rows.part_o = reinterpret_cast<float*>(at + wide_o + wide_ml);
    plan.rows.part_ml = reinterpret_cast<float2*>(at + wide_o + wide_ml + thin_o);
    e = kv::launch_attention(a, plan, scaled ? &sc : nullptr, scratch.stream);
    const hipError_t er = scratch.release();
    if (e != hipSuccess) return hip_fail((std::string(name) + ": launch").c_str(), e);
    if (er != hipSuccess) return hip_fail((std::string(name) + ": workspace release").c_str(), er);
    return ok();
}

}  // namespace

extern "C" {

uint32_t gemma4_kv_set_attention_kernel(uint32_t kernel) { return g_attention_kernel.exchange(kernel > 2u ? 0u : kernel); }

Gemma4Status gemma4_qk_norm_rope(const Gemma4Heads* q, const Gemma4Heads* k, const Gemma4Rope* rope,
                                 const int32_t* positions_dev, uint32_t rows, uint32_t head_dim, void* stream) {
    try {
        const char* const name = "gemma4_qk_norm_rope";
        kv::HeadArgs a{};
        if (q == nullptr) return bad(name, "requires non-null q");
        if (!head_dim_ok(head_dim)) return unsupported(name, "head_dim must be 64, 128, 256 or 512");
        Gemma4Status st = check_rope(rope, head_dim, name, &a.rope);
        if (st != GEMMA4_OK) return st;
        if (rows >= (1u << 24)) return unsupported(name, "rows must be under 2^24");
        if (rows == 0) return ok();
        st = check_heads(q, head_dim, true, "q", name, &a.part[0]);
        if (st == GEMMA4_OK && k != nullptr) st = check_heads(k, head_dim, true, "k", name, &a.part[1]);
        if (st != GEMMA4_OK) return st;
        if (a.rope.pairs > 0 && (positions_dev == nullptr || !aligned(positions_dev, 4)))
            return bad(name, "a rotation requires positions, 4-byte aligned");
        a.positions = a.rope.pairs > 0 ? positions_dev : nullptr;
        a.rows = (int)rows;
        a.head_dim = (int)head_dim;
        const hipError_t e = kv::launch_heads(a, static_cast<hipStream_t>(stream));
        if (e != hipSuccess) return hip_fail("gemma4_qk_norm_rope: launch", e);
        return ok();
    } catch (...) {
        return fail_nothrow(GEMMA4_ERR_RUNTIME, "gemma4_qk_norm_rope: unexpected native exception");
    }
}

Gemma4Status gemma4_kv_append(const Gemma4KvPages* pages, const Gemma4KvBatch* batch, const Gemma4Heads* q,
                              const Gemma4Heads* k, const Gemma4Heads* v, const Gemma4Rope* rope, void* stream) {
    try {
        return append("gemma4_kv_append", pages, nullptr, false, batch, q, k, v, rope, stream);
    } catch (...) {
        return fail_nothrow(GEMMA4_ERR_RUNTIME, "gemma4_kv_append: unexpected native exception");
    }
}

Gemma4Status gemma4_kv_append_scaled(const Gemma4KvPages* pages, const Gemma4KvScales* scales, const Gemma4KvBatch* batch,
                                     const Gemma4Heads* q, const Gemma4Heads* k, const Gemma4Heads* v, const Gemma4Rope* rope,
                                     void* stream) {
    try {
        return append("gemma4_kv_append_scaled", pages, scales, true, batch, q, k, v, rope, stream);
    } catch (...) {
        return fail_nothrow(GEMMA4_ERR_RUNTIME, "gemma4_kv_append_scaled: unexpected native exception");
    }
}

Gemma4Status gemma4_kv_attention(const Gemma4KvPages* pages, const Gemma4KvBatch* batch, const uint16_t* q_dev,
                                 uint64_t q_stride, uint32_t q_heads, float scale, uint32_t window, uint16_t* out_dev,
                                 uint64_t out_stride, float* lse_dev, void* stream) {
    try {
        return attend("gemma4_kv_attention", pages, nullptr, false, batch, q_dev, q_stride, q_heads, scale, window, out_dev, out_stride,
                      lse_dev, stream);
    } catch (...) {
        return fail_nothrow(GEMMA4_ERR_RUNTIME, "gemma4_kv_attention: unexpected native exception");
    }
}

Gemma4Status gemma4_kv_attention_scaled(const Gemma4KvPages* pages, const Gemma4KvScales* scales, const Gemma4KvBatch* batch,
                                        const uint16_t* q_dev, uint64_t q_stride, uint32_t q_heads, float scale, uint32_t window,
                                        uint16_t* out_dev, uint64_t out_stride, float* lse_dev, void* stream) {
    try {
        return attend("gemma4_kv_attention_scaled", pages, scales, true, batch, q_dev, q_stride, q_heads, scale, window, out_dev,
                      out_stride, lse_dev, stream);
    } catch (...) {
        return fail_nothrow(GEMMA4_ERR_RUNTIME, "gemma4_kv_attention_scaled: unexpected native exception");
    }
}

Gemma4Status gemma4_kv_reserve(const Gemma4KvPool* pool, const int32_t* new_tokens_dev, int32_t* query_starts_dev, int32_t* kv_lens_dev,
                               int32_t* granted_dev, uint32_t rows, int32_t* positions_dev, int64_t* slots_dev, void* stream) {
    try {
        const char* const name = "gemma4_kv_reserve";
        kv::Pool p{};
        const Gemma4Status st = check_pool(pool, name, &p);
        if (st != GEMMA4_OK) return st;
        if (new_tokens_dev == nullptr || query_starts_dev == nullptr || kv_lens_dev == nullptr)
            return bad(name, "requires non-null new_tokens, query_starts and kv_lens");
        if (kv_lens_dev == pool->lens_dev) return bad(name, "kv_lens must not be the pool's lens");
        if (!aligned(new_tokens_dev, 4) || !aligned(query_starts_dev, 4) || !aligned(kv_lens_dev, 4) || !aligned(granted_dev, 4) ||
            !aligned(positions_dev, 4) || !aligned(slots_dev, 8))
            return bad(name, "arrays must be aligned to their type");
        if (rows >= (1u << 24)) return unsupported(name, "rows must be under 2^24");
        const uint64_t of_requests = 4ull * p.requests;
        if (clash({{p.free_pages, 4ull * p.num_pages, false}, {p.free_count, 4, true}, {p.lens, of_requests, false},
                   {p.tables, table_bytes(p), true}, {new_tokens_dev, of_requests, false}, {query_starts_dev, of_requests + 4, true},
                   {kv_lens_dev, of_requests, true}, {granted_dev, of_requests, true}, {positions_dev, 4ull * rows, true},
                   {slots_dev, 8ull * rows, true}}))
            return bad(name, "an array that is written must not overlap another");
        const kv::Reserve a{new_tokens_dev, query_starts_dev, kv_lens_dev, granted_dev, positions_dev, slots_dev};
        Scratch sc;
        sc.stream = static_cast<hipStream_t>(stream);
        hipError_t e = hipGetDevice(&sc.device);
        if (e != hipSuccess) return hip_fail("gemma4_kv_reserve: hipGetDevice", e);
        void* needs = nullptr;
        e = sc.take(kv::reserve_scratch(p, (int)rows), &needs);
        if (e != hipSuccess)
            return fail(GEMMA4_ERR_MEMORY_GUARD, std::string(name) + ": workspace allocation failed: " + hipGetErrorString(e));
        e = kv::launch_reserve(p, a, (int)rows, static_cast<int*>(needs), sc.stream);
        const hipError_t er = sc.release();
        if (e != hipSuccess) return hip_fail("gemma4_kv_reserve: launch", e);
        if (er != hipSuccess) return hip_fail("gemma4_kv_reserve: workspace release", er);
        return ok();
    } catch (...) {
        return fail_nothrow(GEMMA4_ERR_RUNTIME, "gemma4_kv_reserve: unexpected native exception");
    }
}

Gemma4Status gemma4_kv_release(const Gemma4KvPool* pool, const int32_t* lens_dev, uint32_t window, void* stream) {
    try {
        const char* const name = "gemma4_kv_release";
        kv::Pool p{};
        const Gemma4Status st = check_pool(pool, name, &p);
        if (st != GEMMA4_OK) return st;
        if (lens_dev == nullptr || !aligned(lens_dev, 4)) return bad(name, "requires non-null lens, 4-byte aligned");
        if (window > (1u << 30)) return unsupported(name, "window exceeds 2^30 (0: none)");
        const uint64_t of_requests = 4ull * p.requests;
        if (clash({{p.free_pages, 4ull * p.num_pages, true}, {p.free_count, 4, true}, {p.lens, of_requests, true},
                   {p.tables, table_bytes(p), true}, {lens_dev == p.lens ? nullptr : lens_dev, of_requests, false}}))
            return bad(name, "the pool's arrays must not overlap, nor lens any of them (it may be the pool's own)");
        Scratch sc;
        sc.stream = static_cast<hipStream_t>(stream);
        hipError_t e = hipGetDevice(&sc.device);
        if (e != hipSuccess) return hip_fail("gemma4_kv_release: hipGetDevice", e);
        void* counts = nullptr;
        e = sc.take(kv::release_scratch(p), &counts);
        if (e != hipSuccess)
            return fail(GEMMA4_ERR_MEMORY_GUARD, std::string(name) + ": workspace allocation failed: " + hipGetErrorString(e));
        e = kv::launch_release(p, lens_dev, (int)window, static_cast<int*>(counts), sc.stream);
        const hipError_t er = sc.release();
        if (e != hipSuccess) return hip_fail("gemma4_kv_release: launch", e);
        if (er != hipSuccess) return hip_fail("gemma4_kv_release: workspace release", er);
        return ok();
    } catch (...) {
        return fail_nothrow(GEMMA4_ERR_RUNTIME, "gemma4_kv_release: unexpected native exception");
    }
}

}  // extern "C"
