// The paged key/value cache handle, shared by the kernels that fill it (kvcache.cu) and read it
// (tree_attention.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

struct nne_kv_cache {
    nne_ctx *ctx = nullptr;
    int device = 0;
    void *k = nullptr, *v = nullptr;  // [pages][kv_heads][page][d] of 16-bit numbers
    bool own = false;
    size_t pages = 0;
    int page = 0, page_shift = 0, kv_heads = 0, d = 0, dtype = 0;
    int rope_dims = 0, rope_interleaved = 0;
    double *freq = nullptr;  // [rope_dims / 2] on the device
};

namespace nne {

int check_cache(const nne_kv_cache *c);

// Row of the pool that holds place `index` of a sequence, or -1 where the table has no page of the pool for it.
__device__ __forceinline__ int kv_row(const int32_t *pages_of, size_t stride, int index, int shift, size_t pages, int kv_heads, int head) {
    const int slot = index >> shift;
    if (index < 0 || (size_t)slot >= stride) return -1;
    const int id = pages_of[slot];  // a plain load: the table may be an earlier kernel's work
    if (id < 0 || (size_t)id >= pages) return -1;
    return ((id * kv_heads + head) << shift) + (index & ((1 << shift) - 1));  // the host checks that rows fit 31 bits
}

// Two f32 numbers as a pair of the cache's type, each rounded once.
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack_pair<__half>(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <>
__device__ __forceinline__ uint32_t pack_pair<__nv_bfloat16>(float a, float b) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t v);
template <>
__device__ __forceinline__ float2 unpack_pair<__half>(uint32_t v) {
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}
template <>
__device__ __forceinline__ float2 unpack_pair<__nv_bfloat16>(uint32_t v) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&v));
}

}  // namespace nne
