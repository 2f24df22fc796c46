/*
 * nne_cuda.h - C ABI of the B200 (sm_100a) backend for the int8 quantized-linear path of
 * elvin-mark/neural-network-engine.
 *
 * This is the whole boundary a host language binds: plain pointers and sizes, no C++ or torch
 * types.  The reference has no FFI for this path today; every entry point below names the
 * reference item (path within the reference project : line) whose work it takes over, which
 * is what the Rust side `src/gpu/cuda/ffi.rs` declares in an `extern "C"` block.
 *
 * Conventions
 *  - Every function returns an nne_status (0 = OK).  No C++ exception crosses the boundary.
 *  - `*_host` buffers are ordinary host memory owned by the caller; the call returns after the
 *    result is in place.  `*_dev` buffers are device pointers on the context's device; the call
 *    is asynchronous on `stream` (a cudaStream_t passed as void*, NULL = the legacy default
 *    stream) and never synchronises.
 *  - Weights are [N, K] row-major (N = out_features, K = in_features, K contiguous), exactly
 *    the layout of `QLinear.qweight` (src/nn/quantized.rs:80-81).
 *  - A layer handle is immutable after creation, so concurrent forwards on one handle are
 *    safe as long as each call uses its own stream and its own x/y buffers.  `_host` forwards
 *    serialise on a per-context mutex.
 *  - There is no CPU fallback: without a usable sm_100 device every call fails with
 *    NNE_ERR_CUDA or NNE_ERR_UNSUPPORTED.
 */
#ifndef NNE_CUDA_H_
#define NNE_CUDA_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#define NNE_API __attribute__((visibility("default")))
#else
#define NNE_API
#endif

/* Status codes.  The Rust side maps 1 -> EngineError::InvalidArgument (src/error.rs:41-42),
 * 2 -> EngineError::ShapeMismatch (src/error.rs:11-15), everything else ->
 * EngineError::GpuError(String) (src/error.rs:47-48) carrying nne_last_error's text. */
typedef enum nne_status {
    NNE_OK = 0,
    NNE_ERR_INVALID_ARGUMENT = 1,
    NNE_ERR_SHAPE_MISMATCH = 2,
    NNE_ERR_CUDA = 3,
    NNE_ERR_NCCL = 4,
    NNE_ERR_TIMEOUT = 5,
    NNE_ERR_OUT_OF_MEMORY = 6,
    NNE_ERR_UNSUPPORTED = 7
} nne_status;

typedef struct nne_ctx nne_ctx;         /* one per device: streams, staging, SM count   */
typedef struct nne_qlinear nne_qlinear; /* one device-resident int8 layer               */
typedef struct nne_qlinear4 nne_qlinear4; /* one device-resident 4-bit layer            */
typedef struct nne_kv_cache nne_kv_cache; /* a paged cache of keys and values           */
typedef struct nne_plan nne_plan;       /* a fixed list of forwards run as one launch   */
typedef struct nne_shard_group nne_shard_group; /* one rank's end of a column-shard exchange */

/* ---- status text -------------------------------------------------------------------------- */

/* Static description of a status code. */
NNE_API const char *nne_status_string(int status);
/* Copies the calling thread's last error message (NUL-terminated, truncated to n) into buf.
 * Takes the place of the String inside EngineError::GpuError (src/error.rs:47-48). */
NNE_API int nne_last_error(char *buf, size_t n);

/* ---- context ------------------------------------------------------------------------------
 * Plays the role of Arc<GpuContext> of the existing device backend (src/gpu/context.rs:20-59,
 * src/gpu/layers.rs:12-16): created once, shared by every layer placed on that device.       */
/* Side effect on the process: creation raises the release threshold of the device's DEFAULT
 * stream-ordered memory pool to "keep everything" (cudaMemPoolAttrReleaseThreshold), so that the
 * forwards' stream-ordered workspaces are reused instead of returned to the driver at every
 * synchronisation.  A host application that shares that pool inherits the setting. */
NNE_API int nne_cuda_ctx_create(int device, nne_ctx **out);
NNE_API int nne_cuda_ctx_destroy(nne_ctx *ctx);
/* Synchronises the device and reads the context's device error word.  Kernels here never spin
 * without a limit: a wait that runs out (about 2 s) sets this word and the kernel returns.  Returns
 * NNE_ERR_TIMEOUT (and clears the word) if that happened since the last check, else NNE_OK.  The
 * `_host` entry points perform this check themselves. */
NNE_API int nne_cuda_ctx_check(nne_ctx *ctx);
/* Exercises the path from a wait that runs out to NNE_ERR_TIMEOUT without breaking anything: runs a
 * one-CTA kernel that waits, with a limit of `limit_us` microseconds, for an event that never
 * comes (which = 0: a shared-memory barrier nobody arrives at; which = 1: an arrival word of the
 * column-shard exchange that nothing raises).  The kernel gives up, sets the error word and
 * returns; the call returns NNE_OK, and the next nne_cuda_ctx_check reports NNE_ERR_TIMEOUT once.
 * The context stays usable.  No counterpart in the reference. */
NNE_API int nne_cuda_ctx_selftest_wait(nne_ctx *ctx, int which, unsigned int limit_us);
/* The streaming GEMV (m <= 2, and every plan it runs) is a persistent kernel with one CTA per SM;
 * a kernel of another library launched beside it (an NCCL collective on a second stream) finds no
 * SM with room for its CTAs and waits for it to end.  This leaves `count` SMs out of that kernel's
 * grid, so that the two overlap.  0 (the default) uses every SM.  No counterpart in the reference. */
NNE_API int nne_cuda_ctx_reserve_sms(nne_ctx *ctx, int count);
/* Device facts the host side sizes its work with.  Any out pointer may be NULL. */
NNE_API int nne_cuda_ctx_info(const nne_ctx *ctx, int *device, int *sm_count, int *cc_major,
                              int *cc_minor, size_t *total_mem_bytes);

/* ---- device buffers -------------------------------------------------------------------------
 * What a device tensor type on the host side needs, so that a stack of QLinears keeps its
 * activations on the GPU between layers: the counterparts of GpuTensor::from_slice's buffer and
 * queue.write_buffer (src/gpu/tensor.rs:19-44) and of GpuTensor::to_cpu (src/gpu/tensor.rs:53-95).
 * upload returns when the bytes are on the device; download first waits for ALL work issued on the
 * device (like to_cpu's device.poll(Wait)) and reports a timed-out kernel as NNE_ERR_TIMEOUT. */
NNE_API int nne_device_alloc(nne_ctx *ctx, size_t bytes, void **out_dev);
NNE_API int nne_device_free(nne_ctx *ctx, void *ptr_dev);
NNE_API int nne_device_upload(nne_ctx *ctx, void *dst_dev, const void *src_host, size_t bytes);
NNE_API int nne_device_download(nne_ctx *ctx, void *dst_host, const void *src_dev, size_t bytes);
/* The context's own stream (a cudaStream_t as void*), the one the *_host entry points use: device
 * forwards issued on it are ordered with them and with each other. */
NNE_API void *nne_cuda_ctx_stream(nne_ctx *ctx);

/* ---- quantize / dequantize ----------------------------------------------------------------
 * nne_quantize_rows replaces the row loop of QLinear::from_linear (src/nn/quantized.rs:107-127):
 * per row absmax, scale = max>0 ? max/127 : 1, inv = 1/scale, q = round_half_away(v*inv)
 * clamped to [-128,127], NaN -> 0.  Codes and scales are bit-identical to the reference.      */
NNE_API int nne_quantize_rows(nne_ctx *ctx, const float *w_host, size_t rows, size_t cols,
                              int8_t *q_host, float *scales_host);
NNE_API int nne_quantize_rows_dev(nne_ctx *ctx, const float *w_dev, size_t rows, size_t cols,
                                  int8_t *q_dev, float *scales_dev, void *stream);

/* nne_quantize_tensor replaces Int8Tensor::from_raw (src/nn/quantized.rs:32-57): ONE scale for
 * all n elements.  The _dev form needs a 4-byte device scratch word for the grid-wide absmax;
 * it is part of the context.  *scale_dev receives the f32 scale.                              */
NNE_API int nne_quantize_tensor(nne_ctx *ctx, const float *v_host, size_t n, int8_t *q_host,
                                float *scale_out);
NNE_API int nne_quantize_tensor_dev(nne_ctx *ctx, const float *v_dev, size_t n, int8_t *q_dev,
                                    float *scale_dev, void *stream);

/* nne_dequantize_rows replaces Int8Tensor::dequantize (src/nn/quantized.rs:60-67; rows = 1,
 * cols = n, one scale) and the weight loop of QLinear::to_linear (src/nn/quantized.rs:200-209;
 * one scale per row): out = (f32)q * scale[row].                                              */
NNE_API int nne_dequantize_rows(nne_ctx *ctx, const int8_t *q_host, const float *scales_host,
                                size_t rows, size_t cols, float *out_host);
NNE_API int nne_dequantize_rows_dev(nne_ctx *ctx, const int8_t *q_dev, const float *scales_dev,
                                    size_t rows, size_t cols, float *out_dev, void *stream);

/* ---- layer --------------------------------------------------------------------------------
 * nne_qlinear_create_from_f32 replaces QLinear::from_linear (src/nn/quantized.rs:92-141):
 * uploads the f32 weight [N,K] (and bias [N] or NULL), quantizes ON DEVICE and keeps codes,
 * scales and bias resident.  The _dev form takes device pointers (the f32 weight is not kept).
 * nne_qlinear_create_from_i8 builds the same handle from the public fields of an existing
 * QLinear (src/nn/quantized.rs:79-88), e.g. after Clone or a load from disk.                   */
NNE_API int nne_qlinear_create_from_f32(nne_ctx *ctx, const float *w_host,
                                        const float *bias_host_or_null, size_t n, size_t k,
                                        nne_qlinear **out);
NNE_API int nne_qlinear_create_from_f32_dev(nne_ctx *ctx, const float *w_dev,
                                            const float *bias_dev_or_null, size_t n, size_t k,
                                            void *stream, nne_qlinear **out);
NNE_API int nne_qlinear_create_from_i8(nne_ctx *ctx, const int8_t *q_host,
                                       const float *scales_host, const float *bias_host_or_null,
                                       size_t n, size_t k, nne_qlinear **out);
NNE_API int nne_qlinear_destroy(nne_qlinear *ql);

/* Fills the host copies the reference keeps as pub fields `qweight` and `scales`
 * (src/nn/quantized.rs:80-83; read by tests/nn/quantization_tests.rs:38-39).  Either pointer
 * may be NULL. */
NNE_API int nne_qlinear_download(const nne_qlinear *ql, int8_t *q_host, float *scales_host);
/* in_features / out_features / has_bias and the device pointers of the resident tensors. */
NNE_API int nne_qlinear_info(const nne_qlinear *ql, size_t *n, size_t *k, int *has_bias,
                             const int8_t **q_dev, const float **scales_dev,
                             const float **bias_dev);
/* QLinear::memory_bytes (src/nn/quantized.rs:230-237): N*K + 4N (+4N with bias). */
NNE_API size_t nne_qlinear_memory_bytes(const nne_qlinear *ql);

/* nne_qlinear_forward_host replaces the compute of QLinear::forward_quantized
 * (src/nn/quantized.rs:164-193) for an input already flattened to [m, k]:
 * y[r,j] = (sum_i x[r,i] * q[j,i]) * scales[j] (+ bias[j]).  `k` is the caller's last input
 * dimension and is checked against in_features as the reference does (:156-162), returning
 * NNE_ERR_SHAPE_MISMATCH.  m = 0 is valid and does nothing.  Copies x up, runs, copies y back.
 * Accuracy of every forward entry point below (unless it says otherwise): within
 *     1e-3 * ||x_r||inf * scale_j * sum_i |q[j,i]|
 * of the exact value, per element.  What the kernels actually do: each activation row is rounded to
 * a 16-bit grid (2^-15 of the row's largest |x|: at most 3 % of that tolerance, about 0.1-0.4 % of it
 * on random data); all products and sums are exact integers after that.  For m <= 16 a row's result
 * does not depend on which other rows are in the batch. */
NNE_API int nne_qlinear_forward_host(nne_qlinear *ql, const float *x_host, size_t m, size_t k,
                                     float *y_host);
/* Same contraction on device-resident x [m,k] and y [m,n], asynchronous on `stream`. */
NNE_API int nne_qlinear_forward_dev(nne_qlinear *ql, const float *x_dev, size_t m, size_t k,
                                    float *y_dev, void *stream);
/* Same, but writes y with a row stride of `ldy` floats (ldy >= n): used by a column shard to
 * write its slice straight into the gathered [m, N_total] layout. */
NNE_API int nne_qlinear_forward_dev_strided(nne_qlinear *ql, const float *x_dev, size_t m,
                                            size_t k, float *y_dev, size_t ldy, void *stream);

/* Forward that never allocates.  It has no counterpart in the reference.  Meant for callers that
 * may not allocate device memory while they run - a serving loop whose memory budget was handed
 * out in full at start-up, or a thread that issues work while a collective is in flight and
 * cannot risk the device-wide synchronisation an allocation can bring.  Same contraction as
 * nne_qlinear_forward_dev, but with a LOOSER error bound: it always runs the bf16 tensor-core
 * kernel (codes dequantized to bf16 in shared memory - exact - and activations rounded to bf16,
 * fp32 accumulation), so per output channel j
 *     |y - exact| <= 2^-8 * ||x||inf * scale_j * sum_k |q_jk|   (+ fp32 summation error),
 * i.e. up to 3.9 times the 1e-3 tolerance nne_qlinear_forward_dev keeps; on N(0,1)
 * activations the rounding errors average out to a few percent of that tolerance, and on
 * activations that are exact in bf16 the result equals nne_qlinear_forward_dev's bit for bit.
 * The bf16 copy of the activations lives in a fixed 8 MiB array in the library's device image
 * (every GPU that loads the library holds it until the process exits) instead of a stream-ordered
 * allocation.  Limits: in_features % 16 == 0, x_dev 16-byte aligned, and m * in_features <=
 * 4 194 304 (4 Mi elements); anything larger is refused with NNE_ERR_INVALID_ARGUMENT and a
 * message naming the limit.  The first call on a device looks the array's address up
 * (cudaGetSymbolAddress); make that first call before any stream capture begins.  All calls on
 * a device share the one array and it keeps the last call's contents, so two calls whose kernels
 * can overlap on the GPU (different streams, no dependency) race: keep them on one stream or order
 * them with events.  Calls no cudaMalloc/cudaFree or other allocating routine.                   */
NNE_API int nne_qlinear_forward_dev_static(nne_qlinear *ql, const float *x_dev, size_t m, size_t k,
                                           float *y_dev, void *stream);

/* ---- plan: several forwards as one launch ----------------------------------------------------
 * A plan fixes a list of `count` forwards y_i[m, n_i] = QLinear_i.forward(x_i[m, k_i]) on device
 * buffers that stay in place, and nne_qlinear_plan_run issues all of them on `stream`.  It takes
 * the place of the back-to-back QLinear::forward calls a caller makes on projections that do
 * not depend on each other - q/k/v (src/models/llama.rs:226-228), gate/up
 * (src/models/llama.rs:344-346), or the per-layer timing loop of the decode benchmark - each
 * of which is the contraction of src/nn/quantized.rs:164-193.  For m = 1 and streaming-capable
 * shapes the whole list is ONE kernel launch whose weight stream never drains between layers;
 * for 2 <= m <= 16 it is one pre-pass and one launch of the small-batch tensor-core kernel over
 * all layers (layers given the same x pointer share one set of digit planes; the work areas are
 * allocated at creation, so a run allocates nothing; a plan must not run concurrently with
 * itself); otherwise the plan runs its layers one after the other.  Results are identical to
 * `count` calls of nne_qlinear_forward_dev.  Layers must outlive the plan.
 *
 * Items may also depend on one another: where an item reads a buffer an earlier item of the list
 * writes (or writes one an earlier item reads or writes), the plan orders them - the list behaves
 * like `count` forwards issued one after another on a stream.  The dependencies are found from the
 * pointers when the plan is created.  For m = 1 on streaming shapes the whole list is still ONE
 * launch: the grid meets between dependent layers (an arrival counter in device memory, bounded
 * wait, cooperative launch) while the weight stream runs on into the next layer's rows; the
 * counter carries over from run to run, so such a plan may be captured in a CUDA graph and
 * replayed, but must not run concurrently with itself.  Other sizes run the independent groups one
 * after another.  An item whose output overlaps one of its own inputs is refused
 * (NNE_ERR_INVALID_ARGUMENT), except a residual that is the output buffer itself.  After
 * NNE_ERR_TIMEOUT a plan with dependent items must be destroyed (its counter is left mid-count). */
NNE_API int nne_qlinear_plan_create(nne_ctx *ctx, size_t count, nne_qlinear *const *layers,
                                    const float *const *x_dev, float *const *y_dev, size_t m,
                                    nne_plan **out);
NNE_API int nne_qlinear_plan_run(nne_plan *plan, void *stream);
/* The same run with HOST activations and outputs: x_all_host holds the x_i one after another
 * (m * k_i floats each, list order), y_all_host receives the y_i one after another (m * n_i
 * floats each).  Copies them to and from the plan's device buffers (one copy per run of buffers
 * that continue one another in device memory, so a plan built over one x slab and one y slab
 * costs one copy each way), runs the plan on the context's stream and returns when y_all_host is
 * complete.  When both slabs are pinned host memory (cudaHostAlloc / cudaHostRegister), hold at most
 * 1 MiB together and the runs are 16-byte aligned multiples of four floats (nne_qlinear_forward_host
 * does the same for its x and y), the copies are done by two small kernels instead of
 * the copy engines: they chain with the forward kernels by programmatic dependent launch, so the
 * weight stream starts while x is still crossing PCIe (about a tenth off the round trip of a
 * 12-layer decode step).  In a list with dependent items (above) the part of x_all_host that belongs
 * to an item fed by an earlier item is uploaded like the rest and then overwritten on the device by
 * that item's result: its contents do not matter.  Serialised per context like the other *_host
 * entry points.  The reference has no
 * counterpart; it is what a caller of QLinear::forward on several independent projections
 * (q/k/v: src/models/llama.rs:226-228) gets instead of one host round trip per projection. */
NNE_API int nne_qlinear_plan_run_host(nne_plan *plan, const float *x_all_host, float *y_all_host);
NNE_API int nne_qlinear_plan_destroy(nne_plan *plan);
/* 1 when the whole list runs as one streaming launch, 2 when it runs as pre-pass + small-batch
 * kernel, else the number of layers (each then runs its own forward, of one or two launches). */
NNE_API int nne_qlinear_plan_launches(const nne_plan *plan);

/* ---- the steps either side of a QLinear in a decoder block ------------------------------------
 * RMSNorm over the last dimension, y = (x * rrms) * gamma with rrms = 1 / sqrt(mean(x^2) + eps)
 * (src/nn/norm.rs:141-165, row function :517-577); SwiGLU's element-wise step
 * out = silu(gate) * up, silu(v) = v / (1 + exp(-v)) (src/models/llama.rs:343-346,
 * src/tensor/ops.rs:177-179); the residual add out = a + b (src/models/llama.rs:377-392).
 * Device pointers, asynchronous on `stream`.  fp32, within 1e-5 relative of the reference's
 * results (the sum of squares is taken in another order).  out may alias an input. */
NNE_API int nne_rmsnorm_dev(nne_ctx *ctx, const float *x_dev, const float *gamma_dev, float eps,
                            size_t rows, size_t cols, float *y_dev, void *stream);
NNE_API int nne_silu_mul_dev(nne_ctx *ctx, const float *gate_dev, const float *up_dev, size_t n,
                             float *out_dev, void *stream);
NNE_API int nne_add_dev(nne_ctx *ctx, const float *a_dev, const float *b_dev, size_t n, float *out_dev,
                        void *stream);

/* A plan whose forwards take those steps in their stride.  Item i computes
 *     y = layer.forward(x') (+ residual),   x' = x | RMSNorm(x; gamma, eps) | silu(x) * x2,
 * which is how the QLinears of a LLaMA block meet their neighbours: q/k/v and gate/up read
 * RMSNorm(h) (src/models/llama.rs:377-392), down reads silu(gate) * up (:343-346), o and down add
 * the residual stream.  For m <= 2 on streaming shapes the decode kernel applies the transform while
 * it prepares the activations and adds the residual as it stores, so a chain of such plans never
 * leaves the device and launches nothing but the forwards; for other shapes the plan runs the
 * standalone kernels above around its forwards (into buffers it owns).  Results equal the
 * standalone kernels followed by nne_qlinear_forward_dev bit for bit in the second case and within
 * 1e-5 relative in the first (rrms is summed in another order).  Items may consume earlier items'
 * outputs (see above): a whole decoder block - or a whole stack of them - can be one plan, and at
 * m = 1 one launch. */
enum { NNE_INPUT_PLAIN = 0, NNE_INPUT_RMSNORM = 1, NNE_INPUT_SILU_MUL = 2 };
typedef struct nne_plan_item {
    nne_qlinear *layer;
    const float *x;        /* [m, in_features] */
    float *y;              /* [m, out_features] */
    int input_op;          /* NNE_INPUT_* */
    float eps;             /* RMSNORM */
    const float *gamma;    /* RMSNORM: [in_features] */
    const float *x2;       /* SILU_MUL: [m, in_features] (the "up" half; x is the "gate" half) */
    const float *residual; /* NULL, or [m, out_features] added to the forward's result */
} nne_plan_item;
NNE_API int nne_qlinear_plan_create_fused(nne_ctx *ctx, size_t count, const nne_plan_item *items,
                                          size_t m, nne_plan **out);

/* ---- 4-bit layer ----------------------------------------------------------------------------
 * QLinear with half the weight bytes: codes of 4 bits, one f32 scale for each `group` (32, 64 or 128)
 * consecutive inputs of a row; the last group of a row may be shorter.  The rounding rule is the one
 * of the int8 layer (src/nn/quantized.rs:107-127) with 7 in the place of 127 and a group in the place
 * of a row: scale = max|w_g| > 0 ? max|w_g| / 7 : 1, inv = 1 / scale, q = round_half_away(w * inv)
 * clamped to [-8, 7], NaN -> 0.  Public layout of the codes: [n, (k + 1) / 2] bytes, two's complement,
 * the even column in the low four bits (an odd k leaves the last high half 0); of the scales:
 * [n, ceil(k / group)].  No counterpart in the reference.
 *
 * A forward computes y[r,j] = sum_g scale[j,g] * sum_{i in g} q[j,i] * x[r,i] (+ bias[j]) with the
 * accuracy of f32: an activation is put on a grid of its group (off by 2^-23 of the group's largest |x| at
 * most), products and sums within a group are exact integers, sums over groups are f32.  A row's result does not depend on which other rows are in
 * the batch as long as the batch stays in one of the ranges 1..4, 5..8, 9..16, 17..32.  A row of x that
 * holds Inf or NaN gives NaN or Inf in every channel whose codes meet it; other rows are untouched.
 * Up to four rows are one launch; more are two, with a stream-ordered workspace of about 4 * m * k bytes.  Weights are read once for up to 32 rows, once more for each further 32.
 * The handle is immutable and forwards may run concurrently, as with nne_qlinear.  Limits: 2^22 rows,
 * 2^30 columns, 2^18 activation rows a call. */
NNE_API int nne_quantize_rows4_dev(nne_ctx *ctx, const float *w_dev, size_t rows, size_t cols, size_t group,
                                   uint8_t *q_dev, float *scales_dev, void *stream);
NNE_API int nne_qlinear4_create_from_f32(nne_ctx *ctx, const float *w_host, const float *bias_host_or_null,
                                         size_t n, size_t k, size_t group, nne_qlinear4 **out);
NNE_API int nne_qlinear4_create_from_f32_dev(nne_ctx *ctx, const float *w_dev, const float *bias_dev_or_null,
                                             size_t n, size_t k, size_t group, void *stream, nne_qlinear4 **out);
/* From codes and scales in the public layout; the buffers are not kept.  The _dev forms of creation
 * wait for `stream`: the layer is complete when they return. */
NNE_API int nne_qlinear4_create_from_i4(nne_ctx *ctx, const uint8_t *q_host, const float *scales_host,
                                        const float *bias_host_or_null, size_t n, size_t k, size_t group,
                                        nne_qlinear4 **out);
NNE_API int nne_qlinear4_create_from_i4_dev(nne_ctx *ctx, const uint8_t *q_dev, const float *scales_dev,
                                            const float *bias_dev_or_null, size_t n, size_t k, size_t group,
                                            void *stream, nne_qlinear4 **out);
NNE_API int nne_qlinear4_destroy(nne_qlinear4 *ql);
/* Codes and scales in the public layout, and the bias [n] (untouched where the layer has none); any pointer
 * may be NULL. */
NNE_API int nne_qlinear4_download(const nne_qlinear4 *ql, uint8_t *q_host, float *scales_host, float *bias_host);
/* The f32 weights [n, k] the layer stands for, q * scale (as QLinear::to_linear, src/nn/quantized.rs:200-209). */
NNE_API int nne_qlinear4_dequantize(const nne_qlinear4 *ql, float *w_host);
NNE_API int nne_qlinear4_info(const nne_qlinear4 *ql, size_t *n, size_t *k, size_t *group, int *has_bias);
/* Device bytes of the layer: codes and scales padded to 16 rows and 64 columns, and the bias. */
NNE_API size_t nne_qlinear4_memory_bytes(const nne_qlinear4 *ql);
/* The three forwards of nne_qlinear, with the same checks. */
NNE_API int nne_qlinear4_forward_host(nne_qlinear4 *ql, const float *x_host, size_t m, size_t k, float *y_host);
NNE_API int nne_qlinear4_forward_dev(nne_qlinear4 *ql, const float *x_dev, size_t m, size_t k, float *y_dev,
                                     void *stream);
NNE_API int nne_qlinear4_forward_dev_strided(nne_qlinear4 *ql, const float *x_dev, size_t m, size_t k,
                                             float *y_dev, size_t ldy, void *stream);

/* ---- paged key/value cache ----------------------------------------------------------------------
 * What a decoder block does between its q/k/v projections (src/models/llama.rs:226-228) and its output
 * projection, with keys and values in pages.  A pool is [pages][kv_heads][page_size][head_dim] of 16-bit
 * numbers; place i of a sequence lies in page page_table[sequence][i / page_size], at i % page_size.
 * head_dim is 64, 96, 128 or 256, page_size a power of two from 8 to 1024, pages * kv_heads * page_size
 * below 2^31.  rope_dims (a multiple of 8; 0: no rotation) is how many of a head's dimensions are rotated
 * by position, as pairs (i, i + rope_dims/2) or, interleaved, (2i, 2i + 1), pair i by position *
 * rope_base^(-2i / rope_dims), or by position * rope_freq[i] where rope_freq (host, rope_dims/2 numbers,
 * copied) is given.  The pools are the caller's (16-byte aligned device pointers that outlive the handle)
 * or, both NULL, the handle's own, zero-filled.  The handle is immutable; what the pools hold is ordered by
 * the streams of the calls that write and read them. */
enum { NNE_F16 = 1, NNE_BF16 = 2 };
typedef struct nne_kv_cache_desc {
    void *k_pages;
    void *v_pages;
    size_t pages;
    int page_size;
    int kv_heads;
    int head_dim;
    int dtype;             /* NNE_F16 or NNE_BF16 */
    int rope_dims;
    int rope_interleaved;
    double rope_base;
    const double *rope_freq;
} nne_kv_cache_desc;
NNE_API int nne_kv_cache_create(nne_ctx *ctx, const nne_kv_cache_desc *desc, nne_kv_cache **out);
NNE_API int nne_kv_cache_destroy(nne_kv_cache *cache);
/* The pools and the bytes of each; any out pointer may be NULL. */
NNE_API int nne_kv_cache_info(const nne_kv_cache *cache, void **k_pages, void **v_pages, size_t *bytes_each);

/* One pass over the q, k and v of `tokens` tokens: RMSNorm of each query and key head over head_dim (where a
 * gamma [head_dim] is given; the arithmetic of nne_rmsnorm_dev), rotation of queries and keys, queries to
 * q_out in f32, keys and values to their pages, rounded once.  f32 inputs [tokens][heads][head_dim] with a
 * stride in floats from token to token, so that the three may lie in one row of a fused projection.  q (with
 * q_out, q_heads) or k and v may be left out.  q_out is [tokens][q_heads][head_dim] without gaps and may be q
 * itself where q_stride is q_heads * head_dim; otherwise it overlaps no input.  sequence[t] is the row of
 * page_table [sequences][table_stride], index[t] the place in the sequence, position[t] what the rotation goes by
 * (NULL: index; drafted nodes of a tree share positions but not places).  A token with index[t] < 0 is padding:
 * nothing of it is read beyond that or written.  Where the sequence, the place or the page that the table names does not
 * exist, the token's key and value are not stored (its query is).  A place given twice in one call holds
 * one of the two tokens' values, element by element, afterwards.  index may be NULL when only queries are
 * given.  One launch, no workspace, asynchronous on `stream`. */
typedef struct nne_kv_append {
    const float *q;
    const float *k;
    const float *v;
    float *q_out;
    size_t q_stride;
    size_t k_stride;
    size_t v_stride;
    size_t tokens;
    int q_heads;
    float eps;
    const float *q_gamma;
    const float *k_gamma;
    const int32_t *page_table;
    size_t table_stride;
    int sequences;
    const int32_t *sequence;
    const int32_t *index;
    const int32_t *position;
} nne_kv_append;
NNE_API int nne_kv_append_dev(nne_kv_cache *cache, const nne_kv_append *args, void *stream);

/* Attention of the cache's newest tokens, drafted as a tree (or, one node a sequence, ordinary decoding): the
 * attention call of src/models/llama.rs between the projections, over pages.  Sequence b has the rows
 * node_start[b] .. node_start[b+1]-1 of q and out (node_start: [sequences + 1], ascending; rows outside are not
 * touched), context[b] earlier tokens in places 0 .. context[b]-1 of the cache, which every node sees, and
 * node j's key in place context[b] + j.  Node i sees node j where bit j of visible[row of i] is set - its ancestors
 * and itself, as a rule - or, visible NULL, where j <= i (a chain); bits of nodes that are not there mean nothing.
 *     out[row, h] = softmax(scale * q[row, h] . k) v      over what the node sees, head h / (q_heads / kv_heads)
 * A row that sees nothing is 0.  What a row does not see does not reach it, Inf and NaN included; Inf or NaN in a
 * key that it sees makes it NaN, in a value Inf or NaN.  Keys whose place the table does not name, or in a page
 * outside the pool, are seen by nobody.  q and out are f32, [row][q_heads][head_dim] with a stride in floats from row to row, and do not overlap.  The products are of f32 accuracy (q
 * and the probabilities keep 22 bits or more).  max_nodes (at most 64) bounds the nodes of a sequence: rows
 * of a sequence beyond it are not written; longer chains go through in pieces of 64, appended piece by piece.
 * At most 65535 sequences a call.  max_context only guides how far the work is split; contexts may be longer.  One
 * launch without workspace, or, few rows over long contexts, two with a stream-ordered workspace of some megabytes; asynchronous on `stream`.  Results
 * do not change from run to run. */
typedef struct nne_tree_attention {
    const float *q;
    float *out;
    size_t q_stride;
    size_t out_stride;
    size_t tokens;               /* rows of q and out */
    int q_heads;
    int sequences;
    int max_nodes;
    int max_context;
    float scale;
    const int32_t *node_start;
    const int32_t *context;
    const uint64_t *visible;
    const int32_t *page_table;   /* [sequences][table_stride] */
    size_t table_stride;
} nne_tree_attention;
NNE_API int nne_tree_attention_dev(nne_kv_cache *cache, const nne_tree_attention *args, void *stream);

/* ---- the next token --------------------------------------------------------------------------------
 * One token a row from logits [rows][vocab] f32 (a stride in floats from row to row; what the output projection
 * leaves, src/models/llama.rs), by settings of each row's own; every settings pointer is to [rows] device numbers
 * or NULL for "off":
 *     w_i = exp((l_i - max l) / temperature)      NULL: 1; a temperature that is not above 0 takes the argmax
 *     top_k > 0: only the first k in the order "larger logit first, of equal ones the lower index"
 *     top_p < 1: of those only the shortest prefix of that order whose mass reaches top_p * (their mass); at
 *                least one
 *     min_p > 0: of those only w_i >= min_p (the largest w is 1; above 1 counts as 1)
 *     token   = the first index, in index order, at which the mass kept so far exceeds uniform * (mass kept)
 * uniform[row] is in [0, 1).  NaN logits count as -inf, which is never drawn; -0 equals 0; a row without any other
 * logit gives -1.  Masses are held in units of 2^-40 of the largest weight: the draw is that of exact arithmetic but where
 * uniform lies within about 1e-7 of a border.  The same inputs give the same tokens.  vocab is at most 2^22.
 * One launch, no workspace, asynchronous on `stream`. */
typedef struct nne_sample {
    const float *logits;
    size_t row_stride;
    size_t rows;
    size_t vocab;
    const float *temperature;
    const int32_t *top_k;
    const float *top_p;
    const float *min_p;
    const float *uniform;
    int32_t *tokens;
} nne_sample;
NNE_API int nne_sample_dev(nne_ctx *ctx, const nne_sample *args, void *stream);

/* ---- column shards over the GPUs of one node -------------------------------------------------
 * The reference has no multi-device code.  Its forward computes output channel j from row j of
 * qweight, scales[j] and bias[j] alone (src/nn/quantized.rs:184-192) and quantizes per row
 * (:107-127), so rank g of G can own the rows [b_g, e_g) of a layer as an ordinary nne_qlinear
 * (bit-identical codes) and compute columns [b_g, e_g) of y [m, n_total]; every rank then needs all
 * columns - an all-gather of the output slices.
 *
 * A shard group is one rank's end of that exchange: one process per GPU (handles exchanged by any
 * transport) or one process driving several devices.  It owns a WINDOW of device memory which every
 * peer maps.  Gathered outputs live at the same offset in every rank's window.  Two routes:
 *   route 0, peer stores: a split-phase exchange.  nne_qlinear_plan_run only produces: the decode
 *            kernel (m <= 2 on streaming shapes) stores each result into all G windows itself; for
 *            other shapes a copy kernel pushes the slice out after the local forward.  Ordinary
 *            stores to peer-mapped memory; the run neither announces itself nor waits for anybody.
 *            nne_shard_group_wait completes it: it enqueues a one-warp kernel that announces this
 *            rank's runs issued so far in every window and returns once every rank has announced as
 *            many, i.e. once this rank's window holds every slice (bounded: about 2 s, then
 *            NNE_ERR_TIMEOUT through nne_cuda_ctx_check).  EVERY rank must call it for its runs - a
 *            rank that does not is never heard of.  Put it on a stream ordered after the runs:
 *            the run's own stream, before the reader of the gathered output; or a second stream
 *            (after an event), where it overlaps the next run.  nne_qlinear_plan_run_host does run,
 *            wait and copy-back itself.
 *   route 1, NCCL:  ncclAllGather on a communicator the host created (nne_shard_group_set_nccl),
 *            on the run's stream; needs equal slices in rank order.  m = 1 gathers in place; m > 1
 *            gathers [m, width] blocks into a staging area and interleaves them into row-major
 *            [m, n_total].  nne_shard_group_wait is not needed (and harmless).
 * Rules, as for collectives: all ranks issue the same sequence of sharded runs and waits on a
 * group, and a rank issues them on ONE stream (or orders them with events): a run announces the
 * rank's previous run as complete.  A rank
 * may overwrite an output area only when every peer has finished reading what it held: with run,
 * wait and the reads in ONE stream two alternating areas are enough ("a peer has signalled run e+1"
 * implies "it has read run e"); a caller that keeps d runs in flight before it waits needs 2 d areas.
 * A group holds at most 8 ranks.  No multicast object and no TMA access to peer memory is used. */
#define NNE_SHARD_HANDLE_BYTES 64
/* Allocates this rank's window of `window_bytes` (zero-filled; cudaMalloc, so it can be exported). */
NNE_API int nne_shard_group_create(nne_ctx *ctx, int rank, int world, size_t window_bytes,
                                   nne_shard_group **out);
/* Writes the NNE_SHARD_HANDLE_BYTES-byte handle other PROCESSES need to map this window. */
NNE_API int nne_shard_group_handle(const nne_shard_group *group, void *handle_out);
/* all_handles: world x NNE_SHARD_HANDLE_BYTES bytes in rank order (the own entry is ignored). */
NNE_API int nne_shard_group_connect(nne_shard_group *group, const void *all_handles);
/* One process driving all devices: all_groups[p] is rank p's group (peer access is enabled). */
NNE_API int nne_shard_group_connect_local(nne_shard_group *group, nne_shard_group *const *all_groups);
/* The window: device pointer and usable size. */
NNE_API int nne_shard_group_window(const nne_shard_group *group, void **base, size_t *bytes);
/* Completes every sharded run issued on this group so far (route 0): announce, then wait. */
NNE_API int nne_shard_group_wait(nne_shard_group *group, void *stream);
/* ncclComm_t (as void*) of this rank, created by the host, for route 1.  The library calls the
 * NCCL copy the process has loaded (or the one NNE_NCCL_LIB names); it does not link NCCL. */
NNE_API int nne_shard_group_set_nccl(nne_shard_group *group, void *nccl_comm);
/* Unmaps the peers' windows and frees this rank's.  Call it when no rank can still store into this
 * window or read a mapping of it (after a barrier of the host's own making). */
NNE_API int nne_shard_group_destroy(nne_shard_group *group);
/* A plan over column shards: shards[i] holds rows [row_begin[i], row_begin[i] + shards[i].n) of a
 * layer with n_total[i] output channels; x_dev[i] is [m, k_i] (replicated on every rank, anywhere
 * in device memory); y_full_dev[i] is the gathered output [m, n_total[i]] INSIDE this rank's window,
 * at the same window offset on every rank.  nne_qlinear_plan_run runs the forwards and the
 * exchange; nne_qlinear_plan_run_host returns the gathered outputs (m * n_total[i] floats each).
 * A group of one rank runs like an ordinary plan.  Destroy with nne_qlinear_plan_destroy. */
NNE_API int nne_qlinear_plan_create_sharded(nne_shard_group *group, size_t count,
                                            nne_qlinear *const *shards, const size_t *row_begin,
                                            const size_t *n_total, const float *const *x_dev,
                                            float *const *y_full_dev, size_t m, int route,
                                            nne_plan **out);

/* Which kernel a forward of m rows on this layer dispatches to: 1 = streaming GEMV (small m),
 * 2 = tcgen05/TMEM tensor-core kernel (integer form; NNE_PREFILL=bf16 in the environment selects
 * the bf16 form), 3 = generic kernel for shapes the others do not take, 4 = small-batch
 * tensor-core kernel (3 <= m <= 16: int8 weights as the MMA's M side, read once; bit-identical per
 * row to kernel 1; NNE_SKINNY=0 in the environment sends these sizes to kernel 1 instead). */
NNE_API int nne_qlinear_kernel_for(const nne_qlinear *ql, size_t m);
/* Number of kernels this library has launched in the calling process (all contexts). */
NNE_API uint64_t nne_launch_count(void);

#ifdef __cplusplus
}
#endif
#endif /* NNE_CUDA_H_ */
