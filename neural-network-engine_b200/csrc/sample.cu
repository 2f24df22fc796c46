// Drawing the next token of each row of logits: temperature, top-k, top-p, min-p, from given uniform numbers.
//
//   w_i = exp((l_i - max l) / T)
//   top-k: the first k in the order "larger logit first, of equal ones the lower index"
//   top-p: of those the shortest prefix with mass >= p * (their mass)
//   min-p: of those w_i >= min_p (the largest w is 1)
//   token: the first index, in index order, at which the mass kept up to there exceeds u * (mass kept)
//
// HBM has 4 bytes a logit to deliver once; what bounds the kernel at the usual sizes is the chain of passes over a row,
// each ending in a meeting.  So a row is the work of a cluster of up to 8 CTAs, which meet in hardware and read each
// other's shared memory: the row's later passes come from L1, and nothing of it goes through global memory or a
// second launch.
//
// Nothing is sorted.  A logit's bits, made monotone, are its key; top-k and top-p are each a search for the key at which a
// count or a mass reaches its target, 256 buckets a pass, first by distance from the maximum in units of T / 8 and
// then by the key's bits, until a bucket is one key; equal keys are cut off by index.  Masses are integers in units
// of 2^-40 of the largest weight, 64 bits wide: sums of them do not depend on order, so atomics leave results the same from run to run,
// and every pass sees the same totals.
#include <math.h>

#include "common.cuh"
#include "ptx.cuh"

namespace nne {
namespace {

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32;
constexpr int SM_BUCKETS = 256;
constexpr uint32_t KEY_NONE = 0x007fffffu;  // the key of -inf (and of NaN, which counts as -inf)

struct SampleArgs {
    const float *logits;
    size_t row_stride;
    unsigned vocab;
    const float *temperature, *top_p, *min_p, *uniform;
    const int32_t *top_k;
    int32_t *tokens;
};

__device__ __forceinline__ uint32_t key_of(float l) {
    if (!(l == l)) return KEY_NONE;
    const uint32_t b = __float_as_uint(l + 0.0f);  // -0 is 0
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float logit_of(uint32_t key) { return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key); }

struct Shared {
    unsigned long long mass[2][SM_BUCKETS];  // a round's buckets; the other set is zeroed meanwhile
    unsigned long long all[SM_BUCKETS];      // the cluster's buckets
    unsigned long long warp[SM_WARPS];
    unsigned long long word[2];              // what this CTA tells the others, alternating from meeting to meeting
    uint32_t bound[SM_BUCKETS + 1];          // first round: bucket j holds bound[j] > key >= bound[j + 1]
    unsigned found;
    int bucket;
    unsigned long long above;
};

__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned long long ld_cluster_u64(const void *p, unsigned rank) {
    uint32_t peer;
    unsigned long long v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer) : "memory");
    return v;
}
__device__ __forceinline__ unsigned ld_cluster_u32(const void *p, unsigned rank) {
    uint32_t peer;
    unsigned v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer) : "memory");
    return v;
}

struct Row {
    Shared *s;
    const float *l;          // this row
    unsigned begin, end;     // this warp's indices
    unsigned rank, ranks;
    int meeting, round;      // which of the alternating words and bucket sets is next
    float top, temperature;

    // A token's mass in units of 2^-40 of the largest.
    __device__ __forceinline__ float weight(float x) const { return x == top ? 1.0f : expf(__fdiv_rn(x - top, temperature)); }
    __device__ __forceinline__ static unsigned long long units(float w) { return __float2ull_rn(w * 0x1p40f); }

    template <typename F>
    __device__ __forceinline__ void each(F &&f) const {
        unsigned i = begin + (threadIdx.x & 31);
        for (; i + 224 < end; i += 256) {
            float x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) x[u] = l[i + u * 32];
#pragma unroll
            for (int u = 0; u < 8; ++u) f(i + u * 32, x[u]);
        }
        for (; i < end; i += 32) f(i, l[i]);
    }

    // Every CTA's word to every CTA; `mine` is the same in all threads.
    __device__ __forceinline__ const void *tell(unsigned long long mine) {
        unsigned long long *w = &s->word[meeting & 1];
        ++meeting;
        if (threadIdx.x == 0) *w = mine;
        cluster_meet();
        return w;
    }

    __device__ __forceinline__ unsigned long long block_max(unsigned long long v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
            v = u > v ? u : v;
        }
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s->warp[threadIdx.x >> 5] = v;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < SM_WARPS; ++w) v = s->warp[w] > v ? s->warp[w] : v;
        return v;
    }
    // The block's sum; s->warp holds the warps' sums until the next call.
    __device__ __forceinline__ unsigned long long block_sum(unsigned long long v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) s->warp[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0;
#pragma unroll
        for (int w = 0; w < SM_WARPS; ++w) v += s->warp[w];
        return v;
    }
    template <typename F>
    __device__ __forceinline__ unsigned long long total(F &&f) {
        unsigned long long v = 0;
        each([&](unsigned i, float x) { v += f(i, x); });
        const void *w = tell(block_sum(v));
        v = 0;
        for (unsigned r = 0; r < ranks; ++r) v += ld_cluster_u64(w, r);
        return v;
    }

    // The first index at which the running sum of f, in index order, exceeds goal(sum of all f); all CTAs learn it.
    template <typename F, typename G>
    __device__ __forceinline__ unsigned locate(F &&f, G &&goal) {
        unsigned long long v = 0;
        each([&](unsigned i, float x) { v += f(i, x); });
        const unsigned long long mine = block_sum(v);
        const void *w = tell(mine);
        unsigned long long sum = 0, before = 0;
        for (unsigned r = 0; r < ranks; ++r) sum += ld_cluster_u64(w, r);
        const unsigned long long want = goal(sum);
        unsigned owner = 0;
        for (unsigned r = 0; r < ranks; ++r) {
            const unsigned long long part = ld_cluster_u64(w, r);
            owner = r;
            if (before + part > want) break;
            before += part;
        }
        if (owner == rank) {
            const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
            for (int k = 0; k < warp; ++k) before += s->warp[k];
            if (before <= want && before + s->warp[warp] > want) {  // one warp
                unsigned at = end;
                for (unsigned i0 = begin; i0 < end; i0 += 32) {
                    const unsigned i = i0 + lane;
                    unsigned long long up = i < end ? f(i, l[i]) : 0;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long u = __shfl_up_sync(0xffffffffu, up, o);
                        if (lane >= o) up += u;
                    }
                    const unsigned hit = __ballot_sync(0xffffffffu, before + up > want);
                    if (hit) {
                        at = i0 + __ffs(hit) - 1;
                        break;
                    }
                    before += __shfl_sync(0xffffffffu, up, 31);
                }
                if (lane == 0) s->found = at;
            }
        }
        cluster_meet();
        return ld_cluster_u32(&s->found, owner);
    }

    // The largest key t with sum of f over keys >= t reaching `target` (>= 1), where the sum over all keys in
    // (KEY_NONE, first] does.  `above`: the sum over keys > t; `at`: that over the key itself.
    template <typename F>
    __device__ __forceinline__ uint32_t search(F &&f, uint32_t first, unsigned long long target, unsigned long long *above, unsigned long long *at) {
        uint32_t hi = first, lo = KEY_NONE;  // t lies in (lo, hi]
        unsigned long long over = 0;         // sum over keys > hi
        // bucket j of the first round: max - j T / 8 >= l > max - (j + 1) T / 8, the last one all the rest
        const float step = temperature * 0.125f, inv = 1.0f / step;
        for (int i = threadIdx.x; i <= SM_BUCKETS; i += SM_THREADS) {
            const float x = fmaf(-(float)i, step, top);
            s->bound[i] = i == 0 ? 0xffffffffu : (i == SM_BUCKETS ? 0u : key_of(x));
        }
        for (bool by_distance = true;; by_distance = false) {
            unsigned long long *set = s->mass[round & 1];
            const int shift = max(0, 32 - __clz(hi - lo - 1) - 8);  // 256 buckets of 2^shift keys cover (lo, hi]
            __syncthreads();  // bounds, and the zeroed set
            each([&](unsigned i, float x) {
                const uint32_t key = key_of(x);
                if (key > hi || key <= lo) return;
                int j;
                if (by_distance) {
                    const float d = (top - x) * inv;
                    j = d < (float)(SM_BUCKETS - 1) ? (int)d : SM_BUCKETS - 1;
                    while (j > 0 && key >= s->bound[j]) --j;
                    while (j < SM_BUCKETS - 1 && key < s->bound[j + 1]) ++j;
                    if (j == SM_BUCKETS - 1) return;  // what the others leave
                } else {
                    j = (int)((hi - key) >> shift);
                }
                const unsigned long long v = f(i, x);
                if (v) atomicAdd(&set[j], v);
            });
            cluster_meet();
            if (threadIdx.x < SM_BUCKETS) {
                unsigned long long v = 0;
                for (unsigned r = 0; r < ranks; ++r) v += ld_cluster_u64(&set[threadIdx.x], r);
                s->all[threadIdx.x] = v;
                s->mass[(round + 1) & 1][threadIdx.x] = 0;  // its readers passed the meeting
            }
            ++round;
            __syncthreads();
            if (threadIdx.x < 32) {  // the first bucket at which the sum reaches the target
                unsigned long long v[SM_BUCKETS / 32], up = 0;
#pragma unroll
                for (int k = 0; k < SM_BUCKETS / 32; ++k) up += v[k] = s->all[threadIdx.x * (SM_BUCKETS / 32) + k];
                unsigned long long sum = up;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const unsigned long long u = __shfl_up_sync(0xffffffffu, sum, o);
                    if ((int)threadIdx.x >= o) sum += u;
                }
                unsigned long long before = over + sum - up;
                const unsigned hit = __ballot_sync(0xffffffffu, over + sum >= target);
                const int lane = hit ? __ffs(hit) - 1 : 31;
                if ((int)threadIdx.x == lane) {
                    int k = 0;
#pragma unroll
                    for (; k < SM_BUCKETS / 32 - 1; ++k) {
                        if (before + v[k] >= target) break;
                        before += v[k];
                    }
                    s->bucket = lane * (SM_BUCKETS / 32) + k;
                    s->above = before;
                }
            }
            __syncthreads();
            const int j = s->bucket;
            over = s->above;
            if (by_distance) {
                if (j > 0) hi = s->bound[j] - 1;
                const uint32_t below = s->bound[j + 1];
                if (j < SM_BUCKETS - 1 && below > lo + 1) lo = below - 1;
            } else {
                const uint32_t width = 1u << shift, from = hi - (uint32_t)j * width;
                if (shift == 0) {
                    *above = over;
                    *at = s->all[j];
                    __syncthreads();
                    return from;
                }
                lo = from - lo > width ? from - width : lo;
                hi = from;
            }
            __syncthreads();  // bucket and bounds are read before they are written again
        }
    }
};

__global__ void __launch_bounds__(SM_THREADS) sample_kernel(const SampleArgs p) {
    __shared__ Shared sh;
    grid_dependency_wait();
    grid_launch_dependents();
    Row r;
    r.s = &sh;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r.rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r.ranks));
    const size_t row = blockIdx.x / r.ranks;
    r.l = p.logits + row * p.row_stride;
    r.meeting = r.round = 0;
    // indices of a CTA, and of a warp in it: contiguous, in whole 128-byte lines
    const unsigned span = ((p.vocab + r.ranks - 1) / r.ranks + 31) & ~31u, warp_span = ((span + SM_WARPS - 1) / SM_WARPS + 31) & ~31u;
    const unsigned cta_begin = min(r.rank * span, p.vocab), cta_end = min(cta_begin + span, p.vocab);
    r.begin = min(cta_begin + (threadIdx.x >> 5) * warp_span, cta_end);
    r.end = min(r.begin + warp_span, cta_end);
    for (int i = threadIdx.x; i < 2 * SM_BUCKETS; i += SM_THREADS) sh.mass[0][i] = 0;

    // The largest logit and where it is first.
    unsigned long long best = 0;
    r.each([&](unsigned i, float x) {
        const unsigned long long v = (unsigned long long)key_of(x) << 32 | (0xffffffffu - i);
        best = v > best ? v : best;
    });
    const void *w = r.tell(r.block_max(best));
    for (unsigned q = 0; q < r.ranks; ++q) {
        const unsigned long long v = ld_cluster_u64(w, q);
        best = v > best || q == 0 ? v : best;
    }
    const uint32_t top_key = (uint32_t)(best >> 32);
    const float t = p.temperature ? p.temperature[row] : 1.0f;
    int token;
    if (top_key <= KEY_NONE) {
        token = -1;  // no logit to choose
    } else if (!(t > 0.0f)) {
        token = (int)(0xffffffffu - (uint32_t)best);
    } else {
        r.top = logit_of(top_key);
        r.temperature = t;
        uint32_t cut = KEY_NONE + 1;  // kept: key > cut, or key == cut and index <= cut_index
        unsigned cut_index = 0xffffffffu;
        auto kept = [&](unsigned i, float x) {
            const uint32_t key = key_of(x);
            return key > cut || (key == cut && i <= cut_index);
        };
        const int k = p.top_k ? p.top_k[row] : 0;
        if (k > 0 && (unsigned)k < p.vocab) {
            auto one = [&](unsigned, float x) { return (unsigned long long)(key_of(x) > KEY_NONE); };
            if (r.total(one) > (unsigned long long)k) {
                unsigned long long above, at;
                const uint32_t key = r.search(one, top_key, (unsigned long long)k, &above, &at);
                if (above + at > (unsigned long long)k)
                    cut_index = r.locate([&](unsigned, float x) { return (unsigned long long)(key_of(x) == key); },
                                         [&](unsigned long long) { return (unsigned long long)k - above - 1; });
                cut = key;
            }
        }
        const float top_p = p.top_p ? p.top_p[row] : 1.0f;
        if (top_p < 1.0f) {
            auto mass = [&](unsigned i, float x) { return kept(i, x) ? Row::units(r.weight(x)) : 0ull; };
            const unsigned long long sum = r.total(mass);
            unsigned long long target = top_p > 0.0f ? (unsigned long long)ceil((double)top_p * (double)sum) : 1ull;
            target = target < 1 ? 1 : (target > sum ? sum : target);
            unsigned long long above, at;
            const uint32_t key = r.search(mass, top_key, target, &above, &at);
            const unsigned long long each = Row::units(r.weight(logit_of(key)));
            const unsigned long long have = at / each, need = (target - above + each - 1) / each;
            if (need < have) {
                const unsigned index = r.locate([&](unsigned i, float x) { return (unsigned long long)(key_of(x) == key && kept(i, x)); },
                                                [&](unsigned long long) { return need - 1; });
                cut_index = index;
            } else if (key != cut) {
                cut_index = 0xffffffffu;
            }
            cut = key;
        }
        float min_p = p.min_p ? p.min_p[row] : 0.0f;
        min_p = min_p > 1.0f ? 1.0f : min_p;
        float u = p.uniform[row];
        u = u > 0.0f ? u : 0.0f;
        token = (int)r.locate(
            [&](unsigned i, float x) {
                if (!kept(i, x)) return 0ull;
                const float w = r.weight(x);
                return w < min_p ? 0ull : Row::units(w);
            },
            [&](unsigned long long sum) {
                const double at = (double)u * (double)sum;
                return at < (double)sum ? min((unsigned long long)at, sum - 1) : sum - 1;
            });
    }
    if (r.rank == 0 && threadIdx.x == 0) p.tokens[row] = token;
    cluster_meet();  // nobody leaves while a peer may still read its shared memory
}

}  // namespace
}  // namespace nne

using namespace nne;

extern "C" int nne_sample_dev(nne_ctx *ctx, const nne_sample *a, void *stream) {
    NNE_GUARD_BEGIN
    NNE_TRY(use_ctx(ctx));
    if (!a) return fail(NNE_ERR_INVALID_ARGUMENT, "null arguments");
    if (a->vocab < 1 || a->vocab > ((size_t)1 << 22))
        return fail(NNE_ERR_INVALID_ARGUMENT, "vocab must be from 1 to 2^22, got %zu", a->vocab);
    if (a->row_stride < a->vocab) return fail(NNE_ERR_INVALID_ARGUMENT, "row_stride %zu below vocab", a->row_stride);
    if (a->rows > ((size_t)1 << 27)) return fail(NNE_ERR_INVALID_ARGUMENT, "at most 2^27 rows a call, got %zu", a->rows);
    if (a->rows == 0) return NNE_OK;
    if (!a->logits || !a->uniform || !a->tokens) return fail(NNE_ERR_INVALID_ARGUMENT, "null device pointer");
    if (reinterpret_cast<uintptr_t>(a->logits) & 3) return fail(NNE_ERR_INVALID_ARGUMENT, "logits are not 4-byte aligned");
    // CTAs a row: as many as leave each at least 2048 logits (four a thread), up to the 8 of a portable cluster.
    unsigned ranks = 1;
    while (ranks < 8 && a->vocab >= (size_t)ranks * 2 * 2048) ranks *= 2;
    SampleArgs p = {a->logits, a->row_stride, (unsigned)a->vocab, a->temperature, a->top_p, a->min_p, a->uniform, a->top_k, a->tokens};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = ranks;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a->rows * ranks));
    cfg.blockDim = dim3(SM_THREADS);
    cfg.stream = (cudaStream_t)stream;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel, p);
    count_launch();
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NNE_ERR_CUDA, "sampling launch failed: %s", cudaGetErrorString(e));
    }
    return NNE_OK;
    NNE_GUARD_END
}
