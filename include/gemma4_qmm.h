/*
 * gemma4_qmm — MI355X (gfx950) affine 4-bit quantized linear layers behind a C ABI.
 *
 * Drop-in for the reference's quantized-linear call sites.  The reference issues
 * every projection as
 *     mlx::core::quantized_matmul(x, W, scales, biases, transpose=true,
 *                                 group_size, bits, "affine")
 * at native/gemma4_mlx/src/native_model.cc:349-362 (q/k/v/o and gate/up/down,
 * call sites :802,813,821,892,934,939,949 prefill, :993,1005,1009,1128,1318-1321
 * decode, :1158,1167,1171,1281,1366-1369 block/verify) and the lm_head at
 * native_model.cc:1782-1795.  Those weights are loaded once and stay resident
 * (native_model.cc:3550-3566), so the boundary here is a handle that owns the
 * device copy of one projection's weight triple, plus a forward call per step.
 *
 * Conventions follow the reference C ABI (native/gemma4_mlx/include/gemma4_mlx.h,
 * native/gemma4_mlx/src/runtime.cc):
 *   - every entry point returns a Gemma4Status (gemma4_mlx.h:12-21);
 *   - failures store a message in a thread-local buffer read back with
 *     gemma4_qmm_get_last_error (runtime.cc:46, :116-133, :816-823);
 *   - handles are opaque, carry a magic number checked on entry (runtime.cc:41-45),
 *     and have an explicit free (runtime.cc:900-912);
 *   - no C++ exception crosses the ABI (native_model.cc:3582-3588);
 *   - pointers are null-checked and sizes validated before use
 *     (spec/03-rust-mlx-ffi-contract.md "Safety checklist").
 *
 * Data formats (the MLX affine format, model_manifest.cc:101-162,
 * native_model.cc:281-287):
 *   weight  uint32 [N, K/8]  element k of a row is nibble k%8 of word k/8, lowest nibble first
 *   scales  bf16   [N, K/64] (raw bit patterns as uint16)
 *   biases  bf16   [N, K/64]
 *   w[n,k] = scales[n,k/64] * q[n,k] + biases[n,k/64]
 *   x       bf16   [M, K] row-major, device memory, 16-byte aligned
 *   y       bf16 or fp32 [M, N] row-major, device memory;  y = x . W^T
 * bits = 4 or 8 with group_size = 64 is accepted: the default of the reference's
 * Gemma 4 12B artifact and the only overrides its loader allows (model_manifest.cc:148).
 * With bits = 8 the weight is uint32 [N, K/4], code k in byte k%4 of word k/4, lowest
 * byte first; it is held as two 4-bit planes (q = 16*qh + ql) and runs on the same
 * kernels over 2K, which read x in place as [x | x].
 *
 * Streams are hipStream_t values passed as void* (NULL = the null stream).  All
 * device work is asynchronous on that stream.  A handle is immutable after
 * create, so forward/dequantize may run concurrently on several streams and
 * threads; create and free must not overlap use.  Scratch (split-K partial sums,
 * the 256-row GEMM tile's group sums, the greedy head's keys, LoRA's x.A^T, the
 * partial sums of attention whose key ranges are cut) comes from device memory the
 * library keeps per (device, stream) and reuses call after call in stream order.  A
 * HIP graph that captured a call uses its capture stream's memory, so replays of
 * graphs captured on one stream must not overlap one another or calls on that stream
 * (replay them on one stream, or serialize).  When a call needs more, the stream's
 * memory grows; the outgrown buffer is freed unless a capture used it.  The memory is
 * held until gemma4_qmm_release_scratch or the end of the process.
 */
#ifndef GEMMA4_QMM_H
#define GEMMA4_QMM_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define GEMMA4_QMM_ABI_VERSION 2u

/* Same codes as the reference status enum (gemma4_mlx.h:12-21); defined here only
 * when that header has not been included first. */
#ifndef GEMMA4_MLX_H
typedef enum Gemma4Status {
    GEMMA4_OK = 0,
    GEMMA4_ERR_INVALID_ARGUMENT = 1,
    GEMMA4_ERR_UNSUPPORTED_CONFIG = 2,
    GEMMA4_ERR_MODEL_LOAD = 3,
    GEMMA4_ERR_RUNTIME = 4,
    GEMMA4_ERR_MEMORY_GUARD = 5,
    GEMMA4_ERR_CACHE = 6,
    GEMMA4_ERR_ADAPTER = 7
} Gemma4Status;
#endif

typedef struct Gemma4QLinear Gemma4QLinear;

typedef enum Gemma4QmmDtype {
    GEMMA4_QMM_BF16 = 0,
    GEMMA4_QMM_F32 = 1
} Gemma4QmmDtype;

typedef struct Gemma4QmmVersionInfo {
    uint32_t abi_version;
    const char* backend_name;
    const char* backend_version;
} Gemma4QmmVersionInfo;

/* Shape and quantization of one projection (the reference's QuantizationSpec,
 * model_manifest.h:10-13, plus the weight's logical shape). */
typedef struct Gemma4QLinearDesc {
    uint32_t out_features; /* N */
    uint32_t in_features;  /* K, a multiple of group_size */
    uint32_t bits;         /* 4 or 8 */
    uint32_t group_size;   /* 64 */
} Gemma4QLinearDesc;

typedef struct Gemma4QLinearInfo {
    uint32_t out_features;
    uint32_t in_features;
    uint32_t bits;
    uint32_t group_size;
    uint64_t device_bytes; /* resident bytes of the tiled weight triple */
    int32_t device;        /* HIP device ordinal that holds it */
    uint32_t flags;        /* GEMMA4_QLINEAR_GEGLU_PAIR for a gate|up pair */
} Gemma4QLinearInfo;

#define GEMMA4_QLINEAR_GEGLU_PAIR 1u

/* Replaces gemma4_runtime_version (runtime.cc:805-814) for this library. */
Gemma4Status gemma4_qmm_runtime_version(Gemma4QmmVersionInfo* out);

/* Replaces gemma4_get_last_error (runtime.cc:816-823): copies this thread's last
 * error message (empty after a success) into buffer, NUL-terminated. */
Gemma4Status gemma4_qmm_get_last_error(char* buffer, size_t buffer_len);

/* Path choice of the forward calls in this process.  No counterpart in the
 * reference (MLX picks its own kernels); for tests and benchmarks that pin a path.
 *   0 (the default): automatic.  Calls of up to 31 rows, and of up to 1024 while
 *     ceil(rows / 16) * N * K' <= 5.5e7 (K' = 2K for 8-bit handles), take no scratch:
 *     they run on the decode kernels (16-row slabs, one pass over the weights per
 *     slab) or, on wide outputs, on the GEMM with K unsplit (from 17 rows with
 *     ceil(rows / 16) * N >= 4.5e4; 8-bit handles from 9 rows with 6e4 and from 12
 *     with 3e4; never while the slabs' work is at most 3.5e7).  For the Gemma 4
 *     shapes: the decode kernels up to 48 rows for 4096x3840, 96 for 2048x3840, 432
 *     for 512x3840 and 31 for 8192x3840, gate and down; up to 16 for the gate|up
 *     pair.  The GEMM with any plan otherwise.
 *   r > 0: the GEMM from r rows on, the decode kernels below.
 * Both paths meet the same accuracy contract; they sum in different orders, so the
 * last bits of some outputs differ between them.  Returns the previous setting.
 * Takes effect for calls issued after it returns (a process-wide atomic). */
uint32_t gemma4_qmm_set_gemm_min_rows(uint32_t rows);

/* Decode kernel family of the forward calls in this process.  No counterpart in the
 * reference; for tests and benchmarks that pin a kernel.
 *   0 (the default): automatic, chosen per shape.
 *   1: the int8 matrix-core kernels (x split exactly into three int8 limbs per
 *      64-column group) for every call of 1-8 rows they can run (x's limbs and the
 *      kernel's sums within a CU's LDS).
 *   2: the bf16 matrix-core kernels only.
 * All meet the same accuracy contract and sum in different orders.  Values above 2
 * are taken as 0.  Returns the previous setting; takes effect for calls issued after
 * it returns. */
uint32_t gemma4_qmm_set_decode_kernel(uint32_t variant);

/* GEMM (prefill) form of the forward calls in this process.  No counterpart in the
 * reference; for tests and benchmarks that compare the two.
 *   0 (the default): the plan may take the pre-pass forms, which scale x per row by
 *      a power of two into fp16: the fp16 form for 256-row tiles of handles whose
 *      scales allow it (every nonzero scale within 2^26 of the largest, none inf or
 *      NaN; weights expanded as s 2^p (q - 8), exact fp16 products with no per-group
 *      scale step), and for 8-bit handles the one-pass form (weights as 1024 + q from
 *      both planes, one pass over K instead of two 4-bit planes over 2K); the bf16
 *      form elsewhere.
 *   1: the bf16 form only (x as given, weights as 1 + q/16, scaled per group).
 * Both meet the same accuracy contract and sum in different orders.  Values above 1
 * are taken as 0.  Returns the previous setting; takes effect for calls issued after
 * it returns. */
uint32_t gemma4_qmm_set_gemm_form(uint32_t form);

/* Releases the device memory the library keeps for the scratch of calls on `stream`
 * on the current device (for hipStreamPerThread, the calling thread's), after waiting
 * for the stream's work.  No counterpart in the reference (MLX frees per call); for
 * long-running hosts that retire streams.  Graphs captured on that stream that used
 * the memory must not be replayed afterwards; later calls on the stream allocate
 * again.  A stream the library never used is a no-op. */
Gemma4Status gemma4_qmm_release_scratch(void* stream);

/* Load one projection's weight triple from HOST memory in MLX layout onto the
 * current HIP device (the per-prefix tensors the reference keeps in Impl::tensors,
 * native_model.cc:84-104, :3550-3566).  The host arrays may be freed on return. */
Gemma4Status gemma4_qlinear_create(const Gemma4QLinearDesc* desc, const uint32_t* weight,
                                   const uint16_t* scales, const uint16_t* biases,
                                   Gemma4QLinear** out);

/* Same, from DEVICE memory in MLX layout on the current device (weights already
 * uploaded by the caller).  The caller's buffers are read by a repack kernel on
 * `stream`; the call waits for that stream, so they may be freed on return and
 * the handle is usable on any stream. */
Gemma4Status gemma4_qlinear_create_device(const Gemma4QLinearDesc* desc, const uint32_t* weight_dev,
                                          const uint16_t* scales_dev, const uint16_t* biases_dev,
                                          void* stream, Gemma4QLinear** out);

/* Releases the device copy.  NULL is accepted (no-op), as for the reference frees. */
Gemma4Status gemma4_qlinear_free(Gemma4QLinear* linear);

Gemma4Status gemma4_qlinear_info(const Gemma4QLinear* linear, Gemma4QLinearInfo* out);

/* y[M,N] = x[M,K] . W^T — replaces quantized_linear (native_model.cc:349-362) and the
 * lm_head product (native_model.cc:1782-1795).  y_dtype BF16 is the model dtype;
 * F32 is the GEMMA4D_NATIVE_FORCE_FLOAT32 output (model_dtype, native_model.cc:330-340).
 * Accumulation is fp32.  rows == 0 is a no-op. */
Gemma4Status gemma4_qlinear_forward(const Gemma4QLinear* linear, void* stream, const uint16_t* x_dev,
                                    uint32_t rows, void* y_dev, Gemma4QmmDtype y_dtype);

/* Scratch bytes gemma4_qlinear_forward (or gemma4_qgeglu_forward, for a pair) takes
 * for `rows` rows under the current path choice: 0 on the decode path, else the GEMM
 * plan's group sums, its pre-pass forms' fp16 copy of x and row exponents, and its
 * split-K partial sums.  No counterpart in the reference.  When
 * it is at most 64 MiB, gemma4_qlinear_forward_noalloc runs the same plan, so the two
 * calls give identical bits. */
Gemma4Status gemma4_qlinear_scratch_bytes(const Gemma4QLinear* linear, uint32_t rows, uint64_t* out);

/* gemma4_qlinear_forward for callers that cannot allocate device memory (code under
 * HIP graph capture, tight serving loops, hosts that forbid allocation): the same
 * arguments, results and kernels, with every scratch buffer taken from a static
 * 64 MiB device array that the library holds on each GPU it runs on until the
 * process ends.  No counterpart in the reference (its MLX ops allocate per call).
 * It calls no hipMalloc, hipFree or allocating library routine.  Scratch needs:
 * none on the decode path (gemma4_qmm_set_gemm_min_rows); on the GEMM path the table
 * of x's group sums that the 256-row tile and the pre-pass forms (fp16, one-pass
 * 8-bit) read (1 KiB per 16 rows, rounded up to the tile, and per 512 columns of K),
 * the pre-pass forms' fp16 copy of x (2 bytes per element) and row exponents (4 bytes
 * per row), and split-K partial
 * sums, only as far as the array has room (a cheaper tile, another form or fewer
 * splits than gemma4_qlinear_forward may choose, so the fp32 summation order, and with
 * it the last bits of some outputs, can differ from that call's; unsplit bf16-form
 * plans on tiles of 32 to 128 rows need none), so no call is refused for want of
 * scratch.  Every call
 * on a GPU shares that GPU's array: calls that overlap in time on one GPU (other
 * streams, other threads) race and must be serialized by the caller. */
Gemma4Status gemma4_qlinear_forward_noalloc(const Gemma4QLinear* linear, void* stream, const uint16_t* x_dev,
                                            uint32_t rows, void* y_dev, Gemma4QmmDtype y_dtype);

/* The MLP block in one call — replaces the decode MLP's gate and up quantized_linear,
 * geglu and down quantized_linear (native_model.cc:1318-1321; prefill :934-949):
 *     h = geglu(x . Wg^T, x . Wu^T)   (bf16 [rows, F], written to h_dev)
 *     y = h . Wd^T                    (bf16 [rows, N_down])
 * gate_up is a pair from gemma4_qgeglu_create, down a projection whose in_features is
 * the pair's F, on the same device.  It queues the pair's launch and then down's (the
 * kernels of gemma4_qgeglu_forward and gemma4_qlinear_forward, so the same bits).
 * y_dtype must be BF16 (the bf16 model dtype; under the float32 override h is fp32,
 * which these kernels do not take as x): GEMMA4_ERR_UNSUPPORTED_CONFIG otherwise.
 * h_dev is 16-byte aligned. */
Gemma4Status gemma4_qmlp_forward(const Gemma4QLinear* gate_up, const Gemma4QLinear* down, void* stream,
                                 const uint16_t* x_dev, uint32_t rows, uint16_t* h_dev, void* y_dev,
                                 Gemma4QmmDtype y_dtype);

/* Writes the fp32 dequantized weight W[N,K] = s*q + b (row-major) to w_dev —
 * mlx::core::dequantize (native_model.cc:364-376) with a float32 result.  Bit-exact:
 * the product s*q is exact in fp32, so the value is unique.  For a gate|up pair the
 * output is [2, F, K]: the gate rows, then the up rows. */
Gemma4Status gemma4_qlinear_dequantize(const Gemma4QLinear* linear, void* stream, float* w_dev);

/* ---- LoRA adapters on a quantized projection ----
 * Replaces quantized_linear's add_lora_delta_if_active (native_model.cc:316-328):
 *     y = model_dtype(base + model_dtype((float32(x) . A^T) . B^T * scale))
 * with the adapter module's A [rank, K] (lora_A.weight) and B [N, rank]
 * (lora_B.weight) as float32 and scale = alpha / rank (native_model.cc:3376-3426).
 * With y_dtype BF16 the base output and the delta are each rounded to bf16 and added
 * in bf16 (the scale is bf16, model_scalar); F32 keeps everything fp32. */
typedef struct Gemma4QLora Gemma4QLora;

/* Copies A and B (host fp32, row-major) to the current device. */
Gemma4Status gemma4_qlora_create(const float* a, const float* b, uint32_t rank, uint32_t in_features,
                                 uint32_t out_features, float scale, Gemma4QLora** out);
Gemma4Status gemma4_qlora_free(Gemma4QLora* lora);

/* gemma4_qlinear_forward plus the adapter's delta; lora NULL is the plain forward.
 * The adapter must match the projection's K and N and live on its device.  Up to 4
 * rows with rank up to 64: one fused launch and no scratch; otherwise scratch of at
 * most 8 * rows * rank * 4 bytes (x . A^T summed over up to eight slices of K).  Where
 * the forward runs on an unsplit GEMM plan and the rank is a multiple of 4 up to 32,
 * x . A^T is formed first and the GEMM's epilogue adds the delta (t . B^T in fp32, then
 * the same roundings); otherwise the delta is added after the forward. */
Gemma4Status gemma4_qlinear_forward_lora(const Gemma4QLinear* linear, const Gemma4QLora* lora, void* stream,
                                         const uint16_t* x_dev, uint32_t rows, void* y_dev, Gemma4QmmDtype y_dtype);

/* Quantized embedding gather — replaces quantized_embedding (native_model.cc:364-376:
 * take of the embed_tokens triple's rows, then dequantize; the same tied triple the
 * lm_head uses).  out[t, :] = s * q + b of row ids[t], for t < count:
 *   ids_dev int32 [count] on the device; ids outside [0, N) give rows of zeros
 *   out_dev [count, K] of dtype, 16-byte aligned: F32 is bit-exact (as
 *   gemma4_qlinear_dequantize); BF16 is that fp32 value rounded once (to nearest even). */
Gemma4Status gemma4_qlinear_embed(const Gemma4QLinear* linear, void* stream, const int32_t* ids_dev, uint32_t count,
                                  void* out_dev, Gemma4QmmDtype dtype);

/* Greedy lm_head: the product, the final-logit softcap and argmax in one call —
 * replaces target_logits_for_hidden (native_model.cc:1782-1795: quantized_matmul, then
 * tanh(logits / 30) * 30) followed by argmax over the vocabulary (native_model.cc:3734,
 * :3825, :3934; per row at :4114, :4242) and the max logit (greedy_logit_for_vector_logits).
 *   token_dev [rows] int32   index of the first maximum of row m's softcapped logits
 *   value_dev [rows] float   that maximum (optional, NULL to skip)
 *   logits_dev [rows, N]     the softcapped logits in dtype (optional, NULL to skip)
 * softcap 0 skips the softcap.  With dtype BF16 the logits and every softcap op are
 * rounded to bf16 as the reference's bf16 array ops are; F32 keeps fp32.  rows <= 16
 * (a decode step or a verify block, gemma4_mlx.h:77-79).  Deterministic: ties go to
 * the lowest index whatever the execution order.  Uses a stream-ordered scratch of
 * rows * ceil(N/16) * 8 bytes. */
Gemma4Status gemma4_qlinear_forward_greedy(const Gemma4QLinear* linear, void* stream, const uint16_t* x_dev,
                                           uint32_t rows, float softcap, void* logits_dev, Gemma4QmmDtype dtype,
                                           int32_t* token_dev, float* value_dev);

/* ---- Fused gate|up projection with the GeGLU epilogue ----
 * Replaces the reference's MLP front half, two quantized_linear calls on the same
 * input followed by geglu (native_model.cc:934-949 prefill, :1318-1321 decode, and
 * geglu itself at native_model.cc:378-386):
 *     h[M,F] = geglu(x . Wg^T, x . Wu^T),  geglu(g, u) = 0.5*g*(1+tanh(c1*(g+c2*g^3)))*u
 * in one pass over both weight matrices, without writing gate and up to memory.
 * With h_dtype BF16 the qmm outputs and every GeGLU op are rounded to bf16 as the
 * reference's bf16 array ops are (constants bf16(0.7978845608), bf16(0.044715));
 * with F32 everything stays fp32 (the GEMMA4D_NATIVE_FORCE_FLOAT32 path).  The pair
 * is one Gemma4QLinear handle (freed with gemma4_qlinear_free; info reports
 * out_features = F and flags = GEMMA4_QLINEAR_GEGLU_PAIR); desc describes one of
 * the two projections (out_features = F, the same K, bits and group size for both). */
Gemma4Status gemma4_qgeglu_create(const Gemma4QLinearDesc* desc, const uint32_t* gate_weight,
                                  const uint16_t* gate_scales, const uint16_t* gate_biases, const uint32_t* up_weight,
                                  const uint16_t* up_scales, const uint16_t* up_biases, Gemma4QLinear** out);

/* Same, from device memory in MLX layout (as gemma4_qlinear_create_device). */
Gemma4Status gemma4_qgeglu_create_device(const Gemma4QLinearDesc* desc, const uint32_t* gate_weight_dev,
                                         const uint16_t* gate_scales_dev, const uint16_t* gate_biases_dev,
                                         const uint32_t* up_weight_dev, const uint16_t* up_scales_dev,
                                         const uint16_t* up_biases_dev, void* stream, Gemma4QLinear** out);

/* h[M,F] = geglu(x . Wg^T, x . Wu^T) on a handle from gemma4_qgeglu_create*.  x as for
 * gemma4_qlinear_forward; h is [rows, F] of h_dtype in device memory.  A plain
 * projection handle is rejected here, and a pair is rejected by gemma4_qlinear_forward. */
Gemma4Status gemma4_qgeglu_forward(const Gemma4QLinear* pair, void* stream, const uint16_t* x_dev, uint32_t rows,
                                   void* h_dev, Gemma4QmmDtype h_dtype);

/* ---- Attention over a paged cache ----
 * What a layer does between its q|k|v projection and its o projection, for a batch of
 * requests that each have one new token (decode), a few (a verify block) or many (a
 * prompt or a chunk of one): the per-head norms and the rotation of queries and keys,
 * the append of keys and values to the cache, and the attention that reads it.  In the
 * reference these are MLX's fast::rms_norm, fast::rope and
 * fast::scaled_dot_product_attention around a cache per request
 * (native_model.cc:808-881); here the cache is paged and shared by the requests.
 *
 * All memory is the caller's; the structs below only describe it and may be built per
 * call.  Strides are in elements.  Device arrays (positions, starts, lengths, tables) are
 * read when the call's kernels run, so a captured graph follows their contents.
 * q, k, v, weights and outputs are bf16; sums, norms, angles and softmax statistics are
 * 32 bits or more, and results are rounded once, when they are stored. */

typedef enum Gemma4KvDtype {
    GEMMA4_KV_BF16 = 0,
    GEMMA4_KV_E4M3 = 1 /* 8-bit floats (4 exponent bits, largest 448) times k_scale or v_scale */
} Gemma4KvDtype;

/* Page p of KV head h holds its token s at k_dev + p * page_stride + h * head_stride +
 * s * token_stride, head_dim consecutive elements; v_dev likewise.  Any order of the
 * three strides works ([pages, heads, page_size, head_dim] reads whole pages in runs).
 *   page_size   a power of two, 16 to 65536
 *   head_dim    64, 128, 256 or 512
 *   k_dev, v_dev, and every stride in bytes: multiples of 16 */
typedef struct Gemma4KvPages {
    void* k_dev;
    void* v_dev;
    uint64_t page_stride, token_stride, head_stride;
    uint32_t num_pages, page_size, kv_heads, head_dim;
    uint32_t dtype; /* Gemma4KvDtype */
    float k_scale, v_scale; /* finite, > 0; bf16 pages ignore them */
} Gemma4KvPages;

/* The new tokens of a batch: request r's are rows query_starts[r] .. query_starts[r+1] - 1
 * of q (k, v, out), its last one at position kv_lens[r] - 1.  Position p of request r lies
 * in page block_tables[r * table_stride + p / page_size], slot p % page_size.
 *   query_starts_dev  int32 [requests + 1], nondecreasing from 0; rows past the last are
 *                     padding: nothing is stored for them and their outputs are zeros
 *   kv_lens_dev       int32 [requests], the new tokens included
 *   block_tables_dev  int32 [requests, table_stride < 2^31], pages_per_request entries used.  An
 *                     entry outside [0, num_pages) is an absent page: append stores
 *                     nothing there, attention sees no keys there */
typedef struct Gemma4KvBatch {
    const int32_t* query_starts_dev;
    const int32_t* kv_lens_dev;
    const int32_t* block_tables_dev;
    uint32_t requests, tokens, pages_per_request, table_stride;
} Gemma4KvBatch;

/* Rotation by angle position * inv_freq[i] of elements (i, i + distance) for i < pairs;
 * distance 1 means adjacent pairs (2i, 2i + 1).  Other elements pass unrotated.  pairs is
 * a multiple of 8, pairs <= distance, distance a multiple of 8 (or 1) and
 * distance + pairs <= head_dim (2 * pairs for adjacent ones).  pairs 0: no rotation. */
typedef struct Gemma4Rope {
    const float* inv_freq_dev; /* [pairs] */
    uint32_t pairs, distance;
} Gemma4Rope;

/* `count` heads of every row: head h of row t at x_dev + t * x_stride + h * head_dim, e.g.
 * a run of columns of a fused q|k|v output.  norm 1 divides each head by
 * sqrt(mean of squares + eps) and multiplies by weight_dev (head_dim values; NULL: ones);
 * norm 0 leaves it.  out_dev/out_stride: where the result goes (it may be x_dev itself
 * with the same stride); NULL where it goes to the cache. */
typedef struct Gemma4Heads {
    const uint16_t* x_dev;
    uint16_t* out_dev;
    const uint16_t* weight_dev;
    uint64_t x_stride, out_stride;
    uint32_t count;
    uint32_t norm;
    float eps;
} Gemma4Heads;

/* Norm and rotation of q's and k's heads (k may be NULL) in one launch; positions_dev is
 * int32 [rows].  rope NULL: norms only. */
Gemma4Status gemma4_qk_norm_rope(const Gemma4Heads* q, const Gemma4Heads* k, const Gemma4Rope* rope,
                                 const int32_t* positions_dev, uint32_t rows, uint32_t head_dim, void* stream);

/* Stores the batch's k (normed, rotated) and v (normed if v->norm, never rotated) into its
 * pages, and, with q not NULL, norms and rotates q into q->out_dev in the same launch.
 * k and v may read the same columns.  E4M3 pages hold value / scale, saturated at 448. */
Gemma4Status gemma4_kv_append(const Gemma4KvPages* pages, const Gemma4KvBatch* batch, const Gemma4Heads* q,
                              const Gemma4Heads* k, const Gemma4Heads* v, const Gemma4Rope* rope, void* stream);

/* out[t, h] = softmax(scale * q[t, h] . K) V over the keys that row t's position p sees:
 * positions 0..p, or with window > 0 the last `window` of those, in present pages.  Query
 * heads share KV heads in equal consecutive groups (q_heads a multiple of kv_heads).  The
 * batch's own tokens must be in the cache (gemma4_kv_append).  A row that sees no key
 * gives zeros and lse -inf.  Whatever lies in hidden places (a page's unused slots
 * included) is never part of a result, infinities and NaN included.
 *   q_dev [tokens, q_heads, head_dim] with q_stride between rows, 16-byte aligned
 *   out_dev the same shape with out_stride
 *   lse_dev float [tokens, q_heads], log of the softmax's sum; NULL to skip
 * Pages that no row's window reaches never count, and their table entries may be absent (a
 * tile of up to 64 keys at the window's edge may load what a present entry there names).
 * Long key ranges of small batches are split over the card and joined by further launches,
 * in the stream's scratch memory. */
Gemma4Status gemma4_kv_attention(const Gemma4KvPages* pages, const Gemma4KvBatch* batch, const uint16_t* q_dev,
                                 uint64_t q_stride, uint32_t q_heads, float scale, uint32_t window, uint16_t* out_dev,
                                 uint64_t out_stride, float* lse_dev, void* stream);

/* ---- Pages of e4m3 with a scale for each block of tokens ----
 * The two calls above on E4M3 pages whose values are code * 2^(byte - 127), a byte for each
 * `block` consecutive tokens of a page and KV head, for K and for V (the pages' own k_scale and
 * v_scale are ignored).  No scale has to be known beforehand: the append sets a block's byte
 * from the values it stores. No counterpart in the reference.
 *   k_dev, v_dev  uint8: page p and head h's bytes at p * page_stride + h * head_stride, one for
 *                 each block of the page, side by side.  Bytes are taken as at least 27 and at
 *                 most 207 (2^-100 to 2^80)
 *   block         a power of two from 16 to 256, at most page_size */
typedef struct Gemma4KvScales {
    uint8_t* k_dev;
    uint8_t* v_dev;
    uint64_t page_stride, head_stride; /* bytes */
    uint32_t block;
} Gemma4KvScales;

/* gemma4_kv_append.  For the batch's new tokens of a block, of one KV head, the byte becomes the
 * least whose scale times 448 holds the largest finite value among them (0 to 2^-100 take 27);
 * where the block holds tokens before them (its first slot is not among the new ones) it never
 * falls, and where it rises the codes held are brought to the new scale and rounded again.
 * So a token that is dropped again (a draft that fell, one of a request that got no pages, stored
 * behind its last ones) has a lasting effect on the tokens before it in its block: once it has raised
 * the scale they are rounded once more, by at most half a step of a code at the raised scale (2^-4
 * of the value, or 2^-10 of the scale), and the scale stays until the block's first slot is stored anew.
 * Infinities are stored as +-448 times the scale, NaN as NaN.  Slots after the new tokens are
 * left as they are.  A block must be stored to for one request only in a call.  The k and v pages,
 * and the k and v scales, must not overlap, nor q's out k's or v's rows, nor other places of its own
 * x (it may be x itself): refused.  No other array of the call may lie in what it writes. */
Gemma4Status gemma4_kv_append_scaled(const Gemma4KvPages* pages, const Gemma4KvScales* scales, const Gemma4KvBatch* batch,
                                     const Gemma4Heads* q, const Gemma4Heads* k, const Gemma4Heads* v, const Gemma4Rope* rope,
                                     void* stream);

/* gemma4_kv_attention over such pages. */
Gemma4Status gemma4_kv_attention_scaled(const Gemma4KvPages* pages, const Gemma4KvScales* scales, const Gemma4KvBatch* batch,
                                        const uint16_t* q_dev, uint64_t q_stride, uint32_t q_heads, float scale, uint32_t window,
                                        uint16_t* out_dev, uint64_t out_stride, float* lse_dev, void* stream);

/* ---- Pages given out and taken back on the GPU ----
 * What a scheduler does to a batch's tables between two steps, from lengths on the device, so
 * that a captured step needs no host: pages for new tokens (gemma4_kv_reserve), which also
 * makes the arrays of the step's Gemma4KvBatch, and pages no longer needed back to the free
 * ones (gemma4_kv_release).  No counterpart in the reference (MLX grows an array per request).
 *   free_pages_dev   int32 [num_pages]: the first free_count of them are the free pages, the last
 *                    of those given out next
 *   free_count_dev   int32 [1]
 *   lens_dev         int32 [requests]: tokens that each request holds (0: an empty slot)
 *   block_tables_dev int32 [requests, table_stride], pages_per_request entries used; entries
 *                    outside [0, num_pages) are absent.  A page is in one table, or free
 * The calls on a pool must follow each other (one stream, or waits). */
typedef struct Gemma4KvPool {
    int32_t* free_pages_dev;
    int32_t* free_count_dev;
    int32_t* lens_dev;
    int32_t* block_tables_dev;
    uint32_t num_pages, page_size, requests, pages_per_request, table_stride;
} Gemma4KvPool;

/* Pages for new_tokens[r] tokens (negative: none) after the lens[r] that request r holds: absent
 * entries up to that of its last new token are filled, in the order of requests and entries,
 * from the end of the free pages.  A request gets all of its pages or none: none where the sum
 * of what it and those before it need exceeds the free pages, or its table is too short.
 *   query_starts_dev int32 [requests + 1], kv_lens_dev int32 [requests]: those of the batch
 *                    (exclusive sums of the new tokens; lens + new_tokens, also where pages were
 *                    not granted: the tokens then have absent pages, and nothing is stored for them
 *                    beyond the request's last page; in block-scaled pages what is stored there may
 *                    raise the scale of the tokens held.  A second call with new_tokens * granted makes
 *                    the same step without those requests)
 *   granted_dev      int32 [requests], 1 or 0; NULL to skip
 *   positions_dev    int32 [rows], slots_dev int64 [rows]; each NULL to skip: position of each of
 *                    the batch's rows in its request, and page * page_size + slot (-1 where there
 *                    is no page); rows past the last start get 0 and -1
 * lens are not changed: gemma4_kv_release sets them once it is known what is kept.  No array that is
 * written may overlap another.  More than 4096 rows or 1024 requests take scratch of 4 bytes a request. */
Gemma4Status gemma4_kv_reserve(const Gemma4KvPool* pool, const int32_t* new_tokens_dev, int32_t* query_starts_dev, int32_t* kv_lens_dev,
                               int32_t* granted_dev, uint32_t rows, int32_t* positions_dev, int64_t* slots_dev, void* stream);

/* Keeps lens[r] tokens of request r (0: the request is done) and gives back the pages behind
 * them and, with window > 0, those before what the next token sees (positions under
 * lens - window + 1).  Freed pages go to the end of the free ones, the last freed first, so
 * that a release of what was just reserved leaves them as they were.  lens_dev may be the
 * pool's own.  Tables of more than 16384 entries in all take scratch of 4 bytes a request. */
Gemma4Status gemma4_kv_release(const Gemma4KvPool* pool, const int32_t* lens_dev, uint32_t window, void* stream);

/* ---- Sampling, and drafted tokens ----
 * Rows of logits [rows, vocab], row r at x_dev + r * stride elements, BF16 or F32, aligned to their
 * type.  softcap > 0: cap * tanh(x / cap) in their place (native_model.cc:1794, unrounded).
 * Logits of -inf and NaN have no probability, whatever the softcap, nor have those whose weight is
 * under e^-700 of the largest's.  A weight is good to 4e-13 of itself; under a softcap to 2e-13 *
 * softcap / temperature more, 3e-9 at most. */
typedef struct Gemma4Logits {
    const void* x_dev;
    uint64_t stride;
    uint32_t dtype; /* Gemma4QmmDtype */
    float softcap;
} Gemma4Logits;

/* A token from each row's p = softmax(logits / temperature): the first i with
 * p_0 + .. + p_i > uniforms[row]; the first largest logit where the temperature is 0.
 *   uniforms_dev     float [rows] in [0, 1)
 *   temperatures_dev float [rows] (0 or less, or NaN: greedy; infinity: all alike), or NULL: `temperature` for all
 *   out_tokens_dev   int32 [rows]; -1 where no logit has a probability
 * Weights and sums are fp64.  Scratch: 16 bytes a row and 2048 logits (512 of few rows). */
Gemma4Status gemma4_sample(const Gemma4Logits* logits, uint32_t rows, uint32_t vocab, const float* uniforms_dev, float temperature,
                           const float* temperatures_dev, int32_t* out_tokens_dev, void* stream);

/* Drafted tokens against the target's probabilities.  Request r's rows are query_starts[r] ..
 * query_starts[r + 1] - 1: the first was fed its last known token, the others its drafts, so row
 * i's logits answer for the token of row i + 1.  Draft tokens[i + 1] stands while
 *     uniforms[i][0] * q(token) < p(token),
 * p and q the softmax of row i's logits and draft logits over the request's temperature (q = 1
 * where draft_logits is NULL: drafts that were not drawn at random).  At the first that falls a
 * token is drawn from max(p - q, 0) by uniforms[i][1]; where all stand, from the last row's p.
 * Temperature 0: p and q are 1 at the first largest logit.
 *   tokens_dev       int32 [rows], those fed; one outside [0, vocab) never stands
 *   query_starts_dev int32 [requests + 1], nondecreasing from 0; rows past the last are padding
 *   uniforms_dev     float [rows, 2] in [0, 1)
 *   temperatures_dev float [requests], or NULL
 *   out_tokens_dev   int32 [rows]: the accepted drafts from the request's first row on, then the
 *                    drawn token, then -1 (padding -1)
 *   accepted_dev     int32 [requests]: accepted drafts; accepted + 1 tokens are new (none where a
 *                    request has no rows)
 * draft_logits has the rows of logits; its last row of each request is not read for a result.
 * out_tokens and accepted overlap nothing.  Without rows nothing is written.  Scratch: that of
 * gemma4_sample for the rows of both, 8 bytes a request and part of a row, and 48 a request. */
Gemma4Status gemma4_verify_drafts(const Gemma4Logits* logits, const Gemma4Logits* draft_logits, const int32_t* tokens_dev,
                                  const int32_t* query_starts_dev, uint32_t requests, uint32_t rows, uint32_t vocab,
                                  const float* uniforms_dev, float temperature, const float* temperatures_dev, int32_t* out_tokens_dev,
                                  int32_t* accepted_dev, void* stream);

/* Attention kernels of this process.  No counterpart in the reference; for tests and
 * benchmarks that pin a kernel.
 *   0 (the default): by the rows of each request and the work of the call.
 *   1: 128-row tiles for every request that has rows enough, however small the call.
 *   2: 16-row tiles only.
 * Both meet the same accuracy contract and sum in different orders.  Values above 2 are
 * taken as 0.  Returns the previous setting; takes effect for calls issued after it returns. */
uint32_t gemma4_kv_set_attention_kernel(uint32_t kernel);

#ifdef __cplusplus
}
#endif

#endif /* GEMMA4_QMM_H */
