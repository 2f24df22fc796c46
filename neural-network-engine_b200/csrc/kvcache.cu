// A paged key/value cache, and the step between the q/k/v projections and the attention call: per-head RMSNorm of
// queries and keys, rotation by position, keys and values into their pages - one pass over q, k and v.
//
//   x' = x / sqrt(mean(x^2) + eps) * gamma                                   (where a gamma is given; per head)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t),   t = position * freq_i  (pair i of the first rope_dims)
//
// pairs being (x_i, x_{i + dims/2}) or, interleaved, (x_{2i}, x_{2i+1}); freq_i = base^(-2i/dims) unless given.
// HBM bound: 4 bytes in per element, 4 out for a query's, 2 out for a key's or value's.
//
// The angle is formed in 64 bits and reduced to a quarter turn there: at position 120000 its f32 rounding alone would
// be 0.004 of a radian.  sin and cos of the rest are f32's.  They are computed once a CTA, i.e. once for all the heads
// of a token that the CTA takes, while the loads of its first heads are on their way.
#include <math.h>

#include <new>
#include <vector>

#include "kvcache.cuh"
#include "ptx.cuh"

namespace nne {

int check_cache(const nne_kv_cache *c) {
    if (!c || !c->ctx) return fail(NNE_ERR_INVALID_ARGUMENT, "null cache handle");
    return NNE_OK;
}

namespace {

constexpr int AP_WARPS = 8;  // heads a CTA works on at a time
// Of those, how many a warp has loads for on their way.  (Six, with the registers they take, leave fewer CTAs an SM to
// cover the chain index -> table -> store: 6001 tokens 71 us instead of 55.)
constexpr int AP_BATCH = 2;
// CTAs an SM: eight, at 32 registers a thread, where the compiler's own choice of 46 held five: 6001 tokens 55 -> 47 us.
template <int D>
constexpr int AP_PER_SM = D <= 128 ? 8 : 4;

struct AppendArgs {
    const float *q, *k, *v;
    float *q_out;
    size_t q_stride, k_stride, v_stride, table_stride;
    const float *q_gamma, *k_gamma;
    float eps;
    int q_heads, kv_heads, heads;  // heads: all that a token has here, queries, keys, values in that order
    int per_cta;                   // of them a CTA takes
    const int32_t *page_table, *sequence, *index, *position;
    int sequences;
    int page_shift, rope_dims, interleaved;
    size_t pages;
    const double *freq;
    void *k_pages, *v_pages;
};

// A warp holds a head as float4s: lane l elements 4l .. 4l+3 (+ 128 for d = 256).
template <typename T, int D, bool VEC>
__global__ void __launch_bounds__(AP_WARPS * 32, AP_PER_SM<D>) kv_append_kernel(const AppendArgs p) {
    constexpr int NV = (D + 127) / 128;        // float4s of a lane
    constexpr int LANES = D >= 128 ? 32 : D / 4;
    __shared__ float2 turn[D / 2];             // cos, sin
    __shared__ __align__(16) float head[AP_WARPS][D];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    grid_dependency_wait();
    grid_launch_dependents();
    const size_t token = blockIdx.x;
    const int index = p.index ? p.index[token] : 0;
    if (index < 0) return;  // a padded token: nothing of it is written
    const int h_end = min(p.heads, ((int)blockIdx.y + 1) * p.per_cta);

    auto load = [&](int h, float4 (&x)[NV]) {
        const float *src = h < p.q_heads                ? p.q + token * p.q_stride + (size_t)h * D
                           : h < p.q_heads + p.kv_heads ? p.k + token * p.k_stride + (size_t)(h - p.q_heads) * D
                                                        : p.v + token * p.v_stride + (size_t)(h - p.q_heads - p.kv_heads) * D;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (lane >= LANES) {
                x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            } else if (VEC) {
                x[i] = *reinterpret_cast<const float4 *>(src + lane * 4 + i * 128);
            } else {
                const float *s = src + lane * 4 + i * 128;
                x[i] = make_float4(s[0], s[1], s[2], s[3]);
            }
        }
    };
    int h0 = (int)blockIdx.y * p.per_cta + warp;
    float4 x[AP_BATCH][NV];
#pragma unroll
    for (int u = 0; u < AP_BATCH; ++u)
        if (h0 + u * AP_WARPS < h_end) load(h0 + u * AP_WARPS, x[u]);

    if (p.rope_dims) {
        const int pos = p.position ? p.position[token] : index;
        for (int i = threadIdx.x; i < p.rope_dims / 2; i += AP_WARPS * 32) {
            const double a = (double)pos * p.freq[i];
            const double quarters = rint(a * 0.63661977236758134308);             // 2 / pi
            const float r = (float)fma(quarters, -1.57079632679489661923, a);      // within a quarter of a half turn
            float s, c;
            sincosf(r, &s, &c);
            const int quad = (int)((long long)quarters & 3);
            turn[i] = quad == 0 ? make_float2(c, s) : quad == 1 ? make_float2(-s, c) : quad == 2 ? make_float2(-c, -s) : make_float2(s, -c);
        }
    }
    __syncthreads();
    int row0 = -1;
    if (p.k) {
        const int seq = p.sequence[token];
        if (seq >= 0 && seq < p.sequences)
            row0 = kv_row(p.page_table + (size_t)seq * p.table_stride, p.table_stride, index, p.page_shift, p.pages, p.kv_heads, 0);
    }

    for (; h0 < h_end; h0 += AP_BATCH * AP_WARPS) {
#pragma unroll
        for (int u = 0; u < AP_BATCH; ++u) {
            const int h = h0 + u * AP_WARPS;
            if (h >= h_end) break;
            const bool is_q = h < p.q_heads, is_v = h >= p.q_heads + p.kv_heads;
            float4 y[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) y[i] = x[u][i];
            if (h + AP_BATCH * AP_WARPS < h_end) load(h + AP_BATCH * AP_WARPS, x[u]);
            const float *gamma = is_q ? p.q_gamma : (is_v ? nullptr : p.k_gamma);
            if (gamma) {
                float ss = 0.0f;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    ss = fmaf(y[i].x, y[i].x, ss), ss = fmaf(y[i].y, y[i].y, ss);
                    ss = fmaf(y[i].z, y[i].z, ss), ss = fmaf(y[i].w, y[i].w, ss);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float rrms = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(ss, (float)D), p.eps)));
                if (lane < LANES) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const float *g = gamma + lane * 4 + i * 128;
                        y[i].x = y[i].x * rrms * g[0], y[i].y = y[i].y * rrms * g[1];
                        y[i].z = y[i].z * rrms * g[2], y[i].w = y[i].w * rrms * g[3];
                    }
                }
            }
            if (!is_v && p.rope_dims) {
                const int half = p.rope_dims / 2;
                if (!p.interleaved) {  // the other half of a pair is another lane's
                    __syncwarp();
                    if (lane < LANES) {
#pragma unroll
                        for (int i = 0; i < NV; ++i) *reinterpret_cast<float4 *>(&head[warp][lane * 4 + i * 128]) = y[i];
                    }
                    __syncwarp();
                }
                if (lane < LANES) {
#pragma unroll
                    for (int i = 0; i < NV; ++i) {
                        const int e = lane * 4 + i * 128;
                        if (e >= p.rope_dims) continue;  // rope_dims is a multiple of 8
                        if (p.interleaved) {
                            const float2 t0 = turn[e / 2], t1 = turn[e / 2 + 1];
                            y[i] = make_float4(y[i].x * t0.x - y[i].y * t0.y, y[i].y * t0.x + y[i].x * t0.y,
                                               y[i].z * t1.x - y[i].w * t1.y, y[i].w * t1.x + y[i].z * t1.y);
                        } else {
                            const bool low = e < half;
                            const int at = low ? e : e - half;
                            const float4 o = *reinterpret_cast<const float4 *>(&head[warp][low ? e + half : at]);
                            const float sign = low ? -1.0f : 1.0f;
                            const float2 t0 = turn[at], t1 = turn[at + 1], t2 = turn[at + 2], t3 = turn[at + 3];
                            y[i] = make_float4(y[i].x * t0.x + sign * o.x * t0.y, y[i].y * t1.x + sign * o.y * t1.y,
                                               y[i].z * t2.x + sign * o.z * t2.y, y[i].w * t3.x + sign * o.w * t3.y);
                        }
                    }
                }
            }
            if (lane >= LANES) continue;
            if (is_q) {
                float *dst = p.q_out + (token * p.q_heads + h) * D + lane * 4;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    if (VEC) {
                        *reinterpret_cast<float4 *>(dst + i * 128) = y[i];
                    } else {
                        dst[i * 128] = y[i].x, dst[i * 128 + 1] = y[i].y, dst[i * 128 + 2] = y[i].z, dst[i * 128 + 3] = y[i].w;
                    }
                }
            } else if (row0 >= 0) {
                const int kvh = h - p.q_heads - (is_v ? p.kv_heads : 0);
                T *dst = static_cast<T *>(is_v ? p.v_pages : p.k_pages) + (size_t)(row0 + (kvh << p.page_shift)) * D + lane * 4;
#pragma unroll
                for (int i = 0; i < NV; ++i)
                    *reinterpret_cast<uint2 *>(dst + i * 128) = make_uint2(pack_pair<T>(y[i].x, y[i].y), pack_pair<T>(y[i].z, y[i].w));
            }
        }
    }
}

template <typename T, int D>
int launch_append(nne_ctx *ctx, const AppendArgs &a, size_t tokens, bool vec, unsigned groups, cudaStream_t s) {
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)tokens, groups);
    cfg.blockDim = dim3(AP_WARPS * 32);
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = vec ? cudaLaunchKernelEx(&cfg, kv_append_kernel<T, D, true>, a)
                              : cudaLaunchKernelEx(&cfg, kv_append_kernel<T, D, false>, a);
    count_launch();
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NNE_ERR_CUDA, "cache append launch failed: %s", cudaGetErrorString(e));
    }
    return NNE_OK;
}

template <typename T>
int launch_append_d(nne_ctx *ctx, int d, const AppendArgs &a, size_t tokens, bool vec, unsigned groups, cudaStream_t s) {
    switch (d) {
        case 64: return launch_append<T, 64>(ctx, a, tokens, vec, groups, s);
        case 96: return launch_append<T, 96>(ctx, a, tokens, vec, groups, s);
        case 128: return launch_append<T, 128>(ctx, a, tokens, vec, groups, s);
        default: return launch_append<T, 256>(ctx, a, tokens, vec, groups, s);
    }
}

bool is_aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

}  // namespace
}  // namespace nne

using namespace nne;

extern "C" {

int nne_kv_cache_create(nne_ctx *ctx, const nne_kv_cache_desc *desc, nne_kv_cache **out) {
    NNE_GUARD_BEGIN
    if (!out) return fail(NNE_ERR_INVALID_ARGUMENT, "null out pointer");
    *out = nullptr;
    if (!desc) return fail(NNE_ERR_INVALID_ARGUMENT, "null descriptor");
    const int d = desc->head_dim, page = desc->page_size;
    if (d != 64 && d != 96 && d != 128 && d != 256)
        return fail(NNE_ERR_INVALID_ARGUMENT, "head_dim must be 64, 96, 128 or 256, got %d", d);
    if (page < 8 || page > 1024 || (page & (page - 1)))
        return fail(NNE_ERR_INVALID_ARGUMENT, "page_size must be a power of two from 8 to 1024, got %d", page);
    if (desc->dtype != NNE_F16 && desc->dtype != NNE_BF16)
        return fail(NNE_ERR_INVALID_ARGUMENT, "dtype must be NNE_F16 or NNE_BF16, got %d", desc->dtype);
    if (desc->kv_heads < 1 || desc->kv_heads > (1 << 16))
        return fail(NNE_ERR_INVALID_ARGUMENT, "kv_heads must be from 1 to 65536, got %d", desc->kv_heads);
    size_t rows;
    if (__builtin_mul_overflow(desc->pages, (size_t)desc->kv_heads * page, &rows) || rows > 0x7fffffffu)
        return fail(NNE_ERR_INVALID_ARGUMENT, "a cache holds at most 2^31 - 1 rows (pages * kv_heads * page_size)");
    if (desc->rope_dims < 0 || desc->rope_dims > d || desc->rope_dims % 8)
        return fail(NNE_ERR_INVALID_ARGUMENT, "rope_dims must be a multiple of 8 up to head_dim, got %d", desc->rope_dims);
    if (desc->rope_dims && !desc->rope_freq && !(desc->rope_base > 0.0 && isfinite(desc->rope_base)))
        return fail(NNE_ERR_INVALID_ARGUMENT, "rope_base must be positive and finite");
    if ((desc->k_pages == nullptr) != (desc->v_pages == nullptr))
        return fail(NNE_ERR_INVALID_ARGUMENT, "k_pages and v_pages are given together or not at all");
    if (!is_aligned(desc->k_pages, 16) || !is_aligned(desc->v_pages, 16))
        return fail(NNE_ERR_INVALID_ARGUMENT, "page pools must be 16-byte aligned");
    NNE_TRY(use_ctx(ctx));
    nne_kv_cache *c = new (std::nothrow) nne_kv_cache();
    if (!c) return fail(NNE_ERR_OUT_OF_MEMORY, "host allocation failed");
    c->ctx = ctx;
    c->device = ctx->device;
    c->pages = desc->pages;
    c->page = page;
    c->page_shift = __builtin_ctz((unsigned)page);
    c->kv_heads = desc->kv_heads;
    c->d = d;
    c->dtype = desc->dtype;
    c->rope_dims = desc->rope_dims;
    c->rope_interleaved = desc->rope_interleaved != 0;
    cudaError_t e = cudaSuccess;
    if (desc->k_pages) {
        c->k = desc->k_pages;
        c->v = desc->v_pages;
    } else {
        const size_t bytes = rows * d * 2;
        c->own = true;
        e = cudaMalloc(&c->k, bytes ? bytes : 16);
        if (e == cudaSuccess) e = cudaMalloc(&c->v, bytes ? bytes : 16);
        if (e == cudaSuccess) e = cudaMemset(c->k, 0, bytes);
        if (e == cudaSuccess) e = cudaMemset(c->v, 0, bytes);
    }
    if (e == cudaSuccess && c->rope_dims) {
        std::vector<double> f(c->rope_dims / 2);
        for (int i = 0; i < c->rope_dims / 2; ++i)
            f[i] = desc->rope_freq ? desc->rope_freq[i] : pow(desc->rope_base, -2.0 * i / c->rope_dims);
        e = cudaMalloc(&c->freq, f.size() * sizeof(double));
        if (e == cudaSuccess) e = cudaMemcpy(c->freq, f.data(), f.size() * sizeof(double), cudaMemcpyHostToDevice);
    }
    // a memset returns before it has run: the pools are zero when the handle is handed out
    if (e == cudaSuccess && c->own) e = cudaStreamSynchronize(nullptr);
    if (e != cudaSuccess) {
        cudaGetLastError();
        const int st = fail(e == cudaErrorMemoryAllocation ? NNE_ERR_OUT_OF_MEMORY : NNE_ERR_CUDA, "cache set-up failed: %s",
                            cudaGetErrorString(e));
        nne_kv_cache_destroy(c);
        return st;
    }
    *out = c;
    return NNE_OK;
    NNE_GUARD_END
}

int nne_kv_cache_destroy(nne_kv_cache *c) {
    NNE_GUARD_BEGIN
    if (!c) return NNE_OK;
    cudaSetDevice(c->device);
    if (c->own && c->k) cudaFree(c->k);
    if (c->own && c->v) cudaFree(c->v);
    if (c->freq) cudaFree(c->freq);
    delete c;
    return NNE_OK;
    NNE_GUARD_END
}

int nne_kv_cache_info(const nne_kv_cache *c, void **k_pages, void **v_pages, size_t *bytes_each) {
    NNE_TRY(check_cache(c));
    if (k_pages) *k_pages = c->k;
    if (v_pages) *v_pages = c->v;
    if (bytes_each) *bytes_each = c->pages * c->kv_heads * c->page * c->d * 2;
    return NNE_OK;
}

int nne_kv_append_dev(nne_kv_cache *c, const nne_kv_append *a, void *stream) {
    NNE_GUARD_BEGIN
    NNE_TRY(check_cache(c));
    if (!a) return fail(NNE_ERR_INVALID_ARGUMENT, "null arguments");
    if ((a->k == nullptr) != (a->v == nullptr)) return fail(NNE_ERR_INVALID_ARGUMENT, "k and v are given together or not at all");
    const size_t d = (size_t)c->d;
    if (a->q_heads < 0 || (a->q_heads > 0) != (a->q != nullptr) || (a->q != nullptr) != (a->q_out != nullptr))
        return fail(NNE_ERR_INVALID_ARGUMENT, "q, q_out and q_heads go together");
    if (a->q_heads > (1 << 16)) return fail(NNE_ERR_INVALID_ARGUMENT, "q_heads %d too large", a->q_heads);
    if (a->tokens > 0x7fffffffu) return fail(NNE_ERR_INVALID_ARGUMENT, "at most 2^31 - 1 tokens a call, got %zu", a->tokens);
    if (a->q && a->q_stride < a->q_heads * d) return fail(NNE_ERR_INVALID_ARGUMENT, "q_stride %zu below q_heads * head_dim", a->q_stride);
    if (a->k && (a->k_stride < c->kv_heads * d || a->v_stride < c->kv_heads * d))
        return fail(NNE_ERR_INVALID_ARGUMENT, "k_stride or v_stride below kv_heads * head_dim");
    if (a->k && (!a->page_table || !a->sequence || !a->index || a->table_stride == 0 || a->sequences < 0))
        return fail(NNE_ERR_INVALID_ARGUMENT, "storing keys needs page_table, table_stride, sequence and index");
    if (c->rope_dims && !a->position && !a->index) return fail(NNE_ERR_INVALID_ARGUMENT, "a rotation needs position or index");
    for (const void *ptr : {(const void *)a->q, (const void *)a->k, (const void *)a->v, (const void *)a->q_out, (const void *)a->q_gamma,
                            (const void *)a->k_gamma, (const void *)a->page_table, (const void *)a->sequence, (const void *)a->index,
                            (const void *)a->position})
        if (!is_aligned(ptr, 4)) return fail(NNE_ERR_INVALID_ARGUMENT, "device pointers must be 4-byte aligned");
    if (a->tokens == 0 || (!a->q && !a->k)) return NNE_OK;
    NNE_TRY(use_ctx(c->ctx));
    AppendArgs p = {};
    p.q = a->q, p.k = a->k, p.v = a->v, p.q_out = a->q_out;
    p.q_stride = a->q_stride, p.k_stride = a->k_stride, p.v_stride = a->v_stride, p.table_stride = a->table_stride;
    p.q_gamma = a->q_gamma, p.k_gamma = a->k_gamma, p.eps = a->eps;
    p.q_heads = a->q_heads;
    p.kv_heads = a->k ? c->kv_heads : 0;
    p.heads = p.q_heads + 2 * p.kv_heads;
    p.page_table = a->page_table, p.sequence = a->sequence, p.index = a->index, p.position = a->position;
    p.sequences = a->sequences;
    p.page_shift = c->page_shift, p.rope_dims = c->rope_dims, p.interleaved = c->rope_interleaved;
    p.pages = c->pages;
    p.freq = c->freq;
    p.k_pages = c->k, p.v_pages = c->v;
    // A CTA takes all heads of a token, so that its angles are computed once, unless there are so few tokens that
    // most SMs would have none: then the heads are spread, down to one round of the CTA's warps.
    const size_t rounds = ((size_t)p.heads + AP_WARPS - 1) / AP_WARPS;
    size_t groups = (2 * (size_t)c->ctx->sm_count + a->tokens - 1) / a->tokens;
    if (groups > rounds) groups = rounds;
    p.per_cta = (int)((rounds + groups - 1) / groups) * AP_WARPS;
    groups = ((size_t)p.heads + p.per_cta - 1) / p.per_cta;
    const bool vec = is_aligned(a->q, 16) && is_aligned(a->k, 16) && is_aligned(a->v, 16) && is_aligned(a->q_out, 16) &&
                     a->q_stride % 4 == 0 && a->k_stride % 4 == 0 && a->v_stride % 4 == 0;
    if (c->dtype == NNE_F16) return launch_append_d<__half>(c->ctx, c->d, p, a->tokens, vec, (unsigned)groups, (cudaStream_t)stream);
    return launch_append_d<__nv_bfloat16>(c->ctx, c->d, p, a->tokens, vec, (unsigned)groups, (cudaStream_t)stream);
    NNE_GUARD_END
}

}  // extern "C"
