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
// Two or three passes where the settings leave few tokens, as they nearly always do: the maximum; for top-p, counts and masses by
// distance from it, in 256 buckets of T / 16 and T / 4, which show up to which bucket the settings can reach (top-k's reach is
// bounded by the threads' own maxima, min-p's is known); and the tokens up to there, at most 1024, into a list in the first CTA's
// shared memory.  That CTA orders them, cuts the list and draws.
// Where more are left and one setting cuts them, the list holds the bucket of the cut (or, a pass more, a 256th of it), and two passes
// draw from what is above it.
// Else nothing is sorted: a logit's bits, made monotone, are its key; top-k and top-p are each a
// search for the key at which a count or a mass reaches its target, 256 buckets a pass, first by distance from the maximum and
// then by the key's bits, until a bucket is one key; equal keys are cut off by index.
// Masses are integers in units of 2^-40 of the largest weight, 64 bits wide: sums of them do not depend on order, so atomics
// leave results the same from run to run, and every pass sees the same totals.
#include <math.h>

#include "common.cuh"
#include "ptx.cuh"

namespace nne {
namespace {

constexpr int SM_THREADS = 512, SM_WARPS = SM_THREADS / 32;
constexpr int SM_BUCKETS = 256;
constexpr float SM_PER_T = 16.0f;  // buckets of a temperature's width
constexpr int SM_FINE = 192;       // of them, that many; the others are four times as wide
constexpr int SM_LIST = 1024;      // tokens of the list: two a thread
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
    // Sets of levels 0 and 1; count's third is that of the threads' maxima.  Each its own: no meeting lies between the looks into
    // one and the first atomics on the next.
    unsigned count[3][SM_BUCKETS], low[2][SM_BUCKETS], high[2][SM_BUCKETS], all_count[SM_BUCKETS];
    unsigned long long list[SM_LIST];        // rank 0's: the cluster's
    unsigned long long aside[SM_LIST];       // this CTA's tokens for it
    unsigned listed;
    unsigned kept;
};

__device__ __forceinline__ unsigned long long ld_cluster_u64(const void *p, unsigned rank) {
    uint32_t peer;
    unsigned long long v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(peer));
    return v;
}
__device__ __forceinline__ unsigned ld_cluster_u32(const void *p, unsigned rank) {
    uint32_t peer;
    unsigned v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(peer));
    return v;
}

// One thread a warp looks, all have the value - and have waited for it - when this returns.
__device__ __forceinline__ unsigned ask_cluster_u32(const void *p, unsigned rank) {
    const unsigned v = (threadIdx.x & 31) == 0 ? ld_cluster_u32(p, rank) : 0;
    return __shfl_sync(0xffffffffu, v, 0);
}
__device__ __forceinline__ unsigned long long ask_cluster_u64(const void *p, unsigned rank) {
    const unsigned long long v = (threadIdx.x & 31) == 0 ? ld_cluster_u64(p, rank) : 0;
    return __shfl_sync(0xffffffffu, v, 0);
}

// A block's prefix sums of two values a thread (places 2t and 2t + 1): `v` becomes the sums up to and with each.
__device__ __forceinline__ void block_prefix(Shared *s, unsigned long long (&v)[2]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned long long own = v[0] + v[1];
    unsigned long long up = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long u = __shfl_up_sync(0xffffffffu, up, o);
        if (lane >= o) up += u;
    }
    __syncthreads();
    if (lane == 31) s->warp[warp] = up;
    __syncthreads();
    for (int w = 0; w < warp; ++w) up += s->warp[w];
    v[1] = up;
    v[0] = up - own + v[0];
}

struct Row {
    Shared *s;
    const float *l;          // this row
    unsigned begin, end;     // this warp's indices
    unsigned cta_begin, cta_end, warp_span;
    unsigned rank, ranks;
    bool vec;                // the row is 16-byte aligned
    int meeting, round;      // which of the alternating words and bucket sets is next
    float top, temperature, scale;

    // A token's weight, and that in units of 2^-40 (the rest of a unit is dropped).  scale: log2(e) / T.
    __device__ __forceinline__ float weight(float x) const {
        float w;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(fmaxf(x - top, -3.402823466e38f) * scale));
        return x == top ? 1.0f : w;
    }
    __device__ __forceinline__ static unsigned long long units(float w) {  // 0 <= w <= 1
        const float a = __fadd_rz(w, 8.0f);  // its bits count 2^-20s
        const float b = __fadd_rz(w - (a - 8.0f), 0x1p-17f);  // what is left, in 2^-40s
        return ((unsigned long long)(__float_as_uint(a) - 0x41000000u) << 20) + (__float_as_uint(b) - 0x37000000u);
    }

    // f(index, logit) for every logit of the warp, and now and then for an index behind them with -inf; always by whole warps.  One
    // loop, whose loads alone differ (rows that are 16-byte aligned go by float4): the bodies are inlined eight times as it is.
    // (Loads of the next eight before these are looked at cost registers, and more than they gave: 69 instead of 58 us for 64
    // mixed rows of 128000.)
    template <typename F>
    __device__ __forceinline__ void each(F &&f) const {
        const int lane = threadIdx.x & 31;
        for (unsigned i0 = begin; i0 < end; i0 += 256) {
            float x[8];
            if (vec) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const unsigned i = i0 + h * 128 + lane * 4;
                    float4 q = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
                    if (i + 3 < end) {
                        q = *reinterpret_cast<const float4 *>(l + i);
                    } else {
                        if (i < end) q.x = l[i];
                        if (i + 1 < end) q.y = l[i + 1];
                        if (i + 2 < end) q.z = l[i + 2];
                    }
                    x[4 * h] = q.x, x[4 * h + 1] = q.y, x[4 * h + 2] = q.z, x[4 * h + 3] = q.w;
                }
            } else {
#pragma unroll
                for (int u = 0; u < 8; ++u) x[u] = i0 + u * 32 + lane < end ? l[i0 + u * 32 + lane] : -INFINITY;
            }
#pragma unroll
            for (int u = 0; u < 8; ++u) f(i0 + (vec ? (u >> 2) * 128 + lane * 4 + (u & 3) : u * 32 + lane), x[u]);
        }
    }

    // Every CTA's word to every CTA; `mine` is the same in all threads.  Lane q gets rank q's word (0 behind the last rank): one
    // look into another CTA's shared memory takes as long as eight side by side.
    __device__ __forceinline__ unsigned long long tell(unsigned long long mine) {
        unsigned long long *w = &s->word[meeting & 1];
        ++meeting;
        if (threadIdx.x == 0) *w = mine;
        cluster_meet();
        const unsigned q = threadIdx.x & 31;
        return q < ranks ? ld_cluster_u64(w, q) : 0;
    }
    // Over the lanes of at most 8 ranks.
    __device__ __forceinline__ static unsigned long long ranks_sum(unsigned long long v) {
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return __shfl_sync(0xffffffffu, v, 0);
    }
    __device__ __forceinline__ static unsigned long long ranks_max(unsigned long long v) {
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
        return __shfl_sync(0xffffffffu, v, 0);
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
    // The sum of f(rank), whose looks are on their way together.
    template <typename F>
    __device__ __forceinline__ unsigned long long ranks_total(F &&f) const {
        unsigned long long v[8];
#pragma unroll
        for (unsigned q = 0; q < 8; ++q) v[q] = q < ranks ? f(q) : 0;
        return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
    }

    template <typename F>
    __device__ __forceinline__ unsigned long long total(F &&f) {
        unsigned long long v = 0;
        each([&](unsigned i, float x) { v += f(i, x); });
        return ranks_sum(tell(block_sum(v)));
    }

    // The first index at which the running sum of f, in index order, exceeds goal(sum of all f); all CTAs learn it.
    template <typename F, typename G>
    __device__ __forceinline__ unsigned locate(F &&f, G &&goal) {
        unsigned long long v = 0;
        each([&](unsigned i, float x) { v += f(i, x); });
        const unsigned long long mine = block_sum(v);
        const unsigned long long part = tell(mine);
        const unsigned long long want = goal(ranks_sum(part));
        unsigned long long upto = part;  // of the ranks up to and with this lane's
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            const unsigned long long u = __shfl_up_sync(0xffffffffu, upto, o);
            if ((int)(threadIdx.x & 31) >= o) upto += u;
        }
        const unsigned reached = __ballot_sync(0xffffffffu, upto > want) & ((1u << ranks) - 1);
        const unsigned owner = reached ? __ffs(reached) - 1 : ranks - 1;  // (nothing to locate: the last, which finds no place)
        unsigned long long before = __shfl_sync(0xffffffffu, upto - part, (int)owner);
        if (owner == rank) {  // the warp whose part holds it, then all threads on that part, a few logits each
            int warp = 0;
            while (warp < SM_WARPS - 1 && before + s->warp[warp] <= want) before += s->warp[warp++];
            const unsigned lo = min(cta_begin + warp * warp_span, cta_end), hi = min(lo + warp_span, cta_end);
            const unsigned each_has = (hi - lo + SM_THREADS - 1) / SM_THREADS;
            const unsigned from = min(lo + threadIdx.x * each_has, hi), to = min(from + each_has, hi);
            unsigned long long v[2] = {0, 0};
            for (unsigned i = from; i < to; ++i) v[0] += f(i, l[i]);
            const unsigned long long own = v[0];
            block_prefix(s, v);
            unsigned long long run = before + v[0] - own;
            if (run <= want && run + own > want) {  // one thread
                unsigned i = from;
                for (; i + 1 < to; ++i)
                    if ((run += f(i, l[i])) > want) break;
                s->found = i;
            }
        }
        cluster_meet();
        return ask_cluster_u32(&s->found, owner);
    }

    // The draw itself: the first index at which the mass of what `kept` and min_p leave exceeds u * that mass.
    template <typename F>
    __device__ __forceinline__ unsigned draw(F &&kept, float min_p, float u) {
        return locate(
            [&](unsigned i, float x) {
                const float w = weight(x);
                return units(kept(i, x) & !(w < min_p) ? w : 0.0f);
            },
            [&](unsigned long long sum) {
                const double at = (double)u * (double)sum;
                return at < (double)sum ? min((unsigned long long)at, sum - 1) : sum - 1;
            });
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
                s->all[threadIdx.x] = ranks_total([&](unsigned q) { return ld_cluster_u64(&set[threadIdx.x], q); });
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

// Puts the first n (at most SM_LIST, all different and not 0) of the list in order, largest first; all threads.  Few: each
// counts what is larger than its two (100: 1000 cycles, where a sorting network's barriers take 6000).  Above 384 the counting
// would keep all warps busy for n rounds (1000: 36000 cycles) and the network is the shorter.
__device__ __forceinline__ void order_list(Shared *s, unsigned n) {
    __syncthreads();
    if (n <= 384) {
        const unsigned at = 2 * threadIdx.x;
        const unsigned long long a = at < n ? s->list[at] : 0, b = at + 1 < n ? s->list[at + 1] : 0;
        unsigned ra = 0, rb = 0;
        if (at < n) {
#pragma unroll 4
            for (unsigned j = 0; j < n; ++j) {
                const unsigned long long x = s->list[j];
                ra += x > a, rb += x > b;
            }
        }
        __syncthreads();
        if (at < n) s->list[ra] = a;
        if (at + 1 < n) s->list[rb] = b;
    } else {
        unsigned size = 512;
        while (size < n) size <<= 1;
        for (unsigned i = n + threadIdx.x; i < size; i += SM_THREADS) s->list[i] = 0;
        for (unsigned len = 2; len <= size; len <<= 1)
            for (unsigned gap = len >> 1; gap > 0; gap >>= 1) {
                __syncthreads();
                const unsigned i = threadIdx.x;
                if (i < size / 2) {
                    const unsigned lo = ((i & ~(gap - 1)) << 1) | (i & (gap - 1)), hi = lo | gap;
                    const unsigned long long x = s->list[lo], y = s->list[hi];
                    if ((x < y) == ((lo & len) == 0)) s->list[lo] = y, s->list[hi] = x;
                }
            }
    }
    __syncthreads();
}

struct Settings {
    int k;          // 0: off
    float top_p;    // >= 1: off
    float min_p;    // <= 0: off; at most 1
    float u;
};

// The token (rank 0's return value), where the list holds what is needed for it, or -2 in all CTAs.  `mine`: the largest logit
// that this thread has seen.
__device__ __forceinline__ int draw_from_list_body(Row &r, Settings set, float mine) {
    Shared *s = r.s;
    const float inv = __fdiv_rn(SM_PER_T, r.temperature);
    if (!(inv < 1e30f) || isinf(r.top)) return -2;  // distances need numbers to be measured in
    const bool by_mass = set.top_p < 1.0f;
    // in sixteenths of T; never falls as x falls.  Products and differences that are rounded one by one: every pass has to find a
    // token in the same bucket
    auto distance = [&](float x) { return __fmul_rn(__fsub_rn(r.top, x), inv); };
    // Buckets: of one sixteenth up to 12 T, of a quarter up to 28 T, where a mass is less than a unit and counts as none; or 256
    // in the place of one of those, [lo, hi).
    constexpr float END = 4.0f * SM_BUCKETS - 3.0f * SM_FINE;
    float lo = 0.0f, hi = END, per = 1.0f;
    bool whole = true;
    auto bucket = [&](float d) {  // of a distance in [lo, hi)
        const float t = __fmul_rn(__fsub_rn(d, lo), per);
        return min(whole && t >= (float)SM_FINE ? SM_FINE + (int)__fmul_rn(__fsub_rn(t, (float)SM_FINE), 0.25f) : (int)t, SM_BUCKETS - 1);
    };
    auto first = [&](auto &&reached) {  // of the buckets; SM_BUCKETS: none
        int from = 0, to = SM_BUCKETS;
        while (from < to) {
            const int mid = (from + to) / 2;
            if (reached(mid)) to = mid;
            else from = mid + 1;
        }
        return from;
    };
    // The cluster's counts (and masses) up to and with each bucket, of a set of buckets that all CTAs have filled.
    auto gather_buckets = [&](int level, int split, bool masses) {
        cluster_meet();
        const unsigned j = threadIdx.x & (SM_BUCKETS - 1);
        const int at = whole && (int)j >= SM_FINE ? 12 : split;
        if (threadIdx.x < SM_BUCKETS) {
            unsigned most = 0;
            s->all_count[j] = (unsigned)r.ranks_total([&](unsigned q) {
                const unsigned c = ld_cluster_u32(&s->count[level][j], q);
                most = max(most, c);
                return (unsigned long long)c;
            });
            if (masses && at == 20 && most > 4095) s->kept = 1;  // a half may have run over
        } else if (masses) {
            s->all[j] = (r.ranks_total([&](unsigned q) { return (unsigned long long)ld_cluster_u32(&s->high[level][j], q); }) << at) +
                        r.ranks_total([&](unsigned q) { return (unsigned long long)ld_cluster_u32(&s->low[level][j], q); });
        }
        __syncthreads();
        if (threadIdx.x < 64 && (threadIdx.x < 32 || masses)) {  // one warp the counts, one the masses: eight buckets a lane
            constexpr int N = SM_BUCKETS / 32;
            const int lane = threadIdx.x & 31;
            const bool m = threadIdx.x >= 32;
            unsigned long long v[N], up = 0;
#pragma unroll
            for (int k = 0; k < N; ++k) up += m ? s->all[lane * N + k] : s->all_count[lane * N + k], v[k] = up;
            unsigned long long before = up;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long u = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += u;
            }
            before -= up;
#pragma unroll
            for (int k = 0; k < N; ++k) {
                if (m) s->all[lane * N + k] = before + v[k];
                else s->all_count[lane * N + k] = (unsigned)(before + v[k]);
            }
        }
        __syncthreads();
    };
    // Tokens nearer than `edge` but not than `near` into rank 0's list, as far as it holds them; their number.  Each CTA puts its
    // own aside, and rank 0 fetches them all (put one by one into its list, each had waited for rank 0's counter).
    auto gather_tokens = [&](float near, float edge, auto &&in) {
        const int lane = threadIdx.x & 31;
        r.each([&](unsigned i, float x) {
            const float d = distance(x);
            const bool hit = d < edge && d >= near && in(d);
            const unsigned hits = __ballot_sync(0xffffffffu, hit);
            if (hits) {
                unsigned slot = 0;
                if (lane == 0) slot = atomicAdd(&s->listed, __popc(hits));
                slot = __shfl_sync(0xffffffffu, slot, 0) + __popc(hits & ((1u << lane) - 1));
                if (hit && slot < SM_LIST) s->aside[slot] = (unsigned long long)key_of(x) << 32 | (0xffffffffu - i);
            }
        });
        cluster_meet();
        const unsigned have = (unsigned)lane < r.ranks ? ld_cluster_u32(&s->listed, lane) : 0;
        unsigned upto = have;  // of the ranks up to and with this lane's
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) {
            const unsigned u = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += u;
        }
        const unsigned all = __shfl_sync(0xffffffffu, upto, r.ranks - 1);
        if (r.rank == 0 && all <= SM_LIST) {
            for (unsigned i0 = 0; i0 < all; i0 += SM_THREADS) {
                const unsigned i = i0 + threadIdx.x;
                unsigned q = 0, from = 0;
#pragma unroll
                for (int w = 0; w < 7; ++w) {
                    const unsigned bound = __shfl_sync(0xffffffffu, upto, w);
                    if (w + 1 < (int)r.ranks && i >= bound) q = w + 1, from = bound;
                }
                if (i < all) s->list[i] = ld_cluster_u64(&s->aside[i - from], q);  // (whoever puts it in order begins with a barrier)
            }
        }
        return all;
    };
    const float far = set.min_p > 0.0f ? -logf(set.min_p) * SM_PER_T + 1.0f : END;  // what is farther min_p leaves out

    unsigned n = 0;
    bool listed = false;
    unsigned long long mass = 0;
    if (set.k > 0) {
        // The k-th largest of the threads' maxima is at most the k-th largest logit: all that top-k can keep is nearer than
        // that maximum's bucket ends.
        const float d = distance(mine);
        if (d < END) atomicAdd(&s->count[2][bucket(d)], 1u);
        gather_buckets(2, 20, false);
        const int end = first([&](int j) { return s->all_count[j] >= (unsigned)set.k; });
        if (end < SM_BUCKETS) {
            float edge = end < SM_FINE ? (float)(end + 1) : (float)SM_FINE + 4.0f * (float)(end + 1 - SM_FINE);
            if (!by_mass) edge = fminf(edge, far);  // top-p of a top-k needs the mass of all of these
            n = gather_tokens(0.0f, edge, [](float) { return true; });
            listed = n <= SM_LIST;
        }
    } else if (!by_mass && far < END) {
        n = gather_tokens(0.0f, far, [](float) { return true; });
        listed = n <= SM_LIST;
        if (!listed) {
            cluster_meet();  // the count has been read by everybody
            return (int)r.draw([&](unsigned, float x) { return x > -INFINITY; }, set.min_p, set.u);
        }
    }
    if (!listed) {
        // By counts and masses of all tokens' buckets, and of those inside a crowded one.
        if (n > 0) {
            cluster_meet();
            if (threadIdx.x == 0) s->listed = 0;
        }
        int last = 0;                        // the bucket in which the settings' cut lies
        unsigned from = 0;                   // tokens before it
        unsigned long long mass_from = 0;    // their mass
        double want = 0.0;
        bool cut_only = false;               // more than the list holds up to there: the list holds that bucket alone
#pragma unroll 1
        for (int level = 0; level < 2; ++level) {
            const int split = whole ? 20 : (lo < (float)SM_FINE ? 20 : 12);
            r.each([&](unsigned, float x) {
                const float d = distance(x);
                if (!(d >= lo && d < hi)) return;
                const int j = bucket(d);
                atomicAdd(&s->count[level][j], 1u);
                if (by_mass) {  // in two halves: no carry for up to 4095 tokens of 2^40, or 2^20 of the light ones far off
                    const int at = whole && j >= SM_FINE ? 12 : split;
                    const unsigned long long v = Row::units(r.weight(x));
                    atomicAdd(&s->low[level][j], (unsigned)v & ((1u << at) - 1));
                    atomicAdd(&s->high[level][j], (unsigned)(v >> at));
                }
            });
            gather_buckets(level, split, by_mass);
            if (s->kept) return -2;
            if (whole) {
                mass = s->all[SM_BUCKETS - 1];
                want = (double)set.top_p * (double)mass;
                // what top-k would cut off behind the buckets has no mass
                if (set.k > 0 && s->all_count[SM_BUCKETS - 1] < (unsigned)set.k) set.k = 0;
            }
            // Where each setting ends; top-p of a top-k needs the mass of all of these, so top-k's end comes first.
            int end = SM_BUCKETS;
            if (set.k > 0) end = first([&](int j) { return from + s->all_count[j] >= (unsigned)set.k; });
            else if (by_mass) end = first([&](int j) { return (double)(mass_from + s->all[j]) >= want; });
            bool cuts = end < SM_BUCKETS;
            if (whole && far < END && !(by_mass && set.k > 0)) {
                const int j = bucket(far);
                if (j < end) end = j, cuts = false;
            }
            last = end;
            if (whole && end < SM_BUCKETS && s->all_count[end] <= SM_LIST) {
                n = s->all_count[end];
                break;
            }
            cut_only = true;
            if (!cuts) {  // all that min_p leaves, or all: the draw looks at the weights
                n = 0;
                break;
            }
            if (by_mass && set.k > 0) return -2;
            n = s->all_count[end] - (end > 0 ? s->all_count[end - 1] : 0);
            if (end > 0) from += s->all_count[end - 1], mass_from += s->all[end - 1];
            if (n <= SM_LIST) break;
            if (level == 1) return -2;
            // once more, inside the bucket
            lo = end < SM_FINE ? (float)end : (float)SM_FINE + 4.0f * (float)(end - SM_FINE);
            hi = lo + (end < SM_FINE ? 1.0f : 4.0f);
            per = (float)SM_BUCKETS / (hi - lo);
            whole = false;
            __syncthreads();  // all_count and all have been read
        }
        if (cut_only) {
            float edge = -3.402823466e38f;  // without a cut: all
            unsigned index = 0xffffffffu;
            if (n > 0) {
                gather_tokens(lo, hi, [&](float d) { return bucket(d) == last; });
                if (r.rank == 0) {
                    order_list(s, n);
                    const unsigned at = 2 * threadIdx.x;
                    unsigned long long w[2], upto[2];
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        upto[e] = w[e] = at + e < n && by_mass ? Row::units(r.weight(logit_of((uint32_t)(s->list[at + e] >> 32)))) : 0;
                    if (threadIdx.x == 0) s->above = s->list[n - 1];
                    block_prefix(s, upto);
                    const unsigned long long target = set.top_p > 0.0f ? (unsigned long long)ceil((double)set.top_p * (double)mass) : 1ull;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const bool here = set.k > 0 ? from + at + e + 1 == (unsigned)set.k
                                                    : w[e] && mass_from + upto[e] - w[e] < target && mass_from + upto[e] >= target;
                        if (at + e < n && here) s->above = s->list[at + e];
                    }
                }
                cluster_meet();
                const unsigned long long cut = ask_cluster_u64(&s->above, 0);
                edge = logit_of((uint32_t)(cut >> 32));
                index = 0xffffffffu - (unsigned)cut;
                cluster_meet();  // rank 0 goes on to use the word
            }
            return (int)r.draw([&](unsigned i, float x) { return (x > edge) | ((x == edge) & (i <= index)); }, set.min_p, set.u);
        }
        const float edge = last < SM_FINE ? (float)(last + 1) : (float)SM_FINE + 4.0f * (float)(last + 1 - SM_FINE);
        gather_tokens(0.0f, edge, [](float) { return true; });
    }
    if (r.rank != 0) return 0;

    order_list(s, n);
    if (set.k > 0 && (unsigned)set.k > n) set.k = 0;  // min_p's end came first, and what is farther it leaves out
    const unsigned at = 2 * threadIdx.x;
    unsigned long long entry[2], w[2], upto[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        entry[e] = at + e < n ? s->list[at + e] : 0;
        w[e] = at + e < n ? Row::units(r.weight(logit_of((uint32_t)(entry[e] >> 32)))) : 0;
        upto[e] = w[e];
    }
    block_prefix(s, upto);
    const unsigned most = set.k > 0 ? (unsigned)set.k : SM_LIST;  // top-k: places below this
    if (set.k > 0 && at <= most - 1 && most - 1 < at + 2) s->above = (most - 1) & 1 ? upto[1] : upto[0];
    if (threadIdx.x == 0) s->kept = 0;
    __syncthreads();
    const unsigned long long of = set.k > 0 ? s->above : mass;
    const unsigned long long target = set.top_p > 0.0f ? (unsigned long long)ceil((double)set.top_p * (double)of) : 1ull;
    unsigned keeps = 0;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const unsigned place = at + e;
        bool in = place < n && place < most;
        if (by_mass) in = in && (place == 0 || upto[e] - w[e] < target);
        if (set.min_p > 0.0f) in = in && r.weight(logit_of((uint32_t)(entry[e] >> 32))) >= set.min_p;
        keeps += in;
    }
    keeps = __reduce_add_sync(0xffffffffu, keeps);
    if ((threadIdx.x & 31) == 0 && keeps) atomicAdd(&s->kept, keeps);
    __syncthreads();
    const unsigned kept = s->kept;  // the first places: each condition holds up to some place
    // In index order: (2^32 - 1 - index, key), largest first.
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (at + e < kept) s->list[at + e] = (entry[e] << 32) | (entry[e] >> 32);
    order_list(s, kept);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        entry[e] = at + e < kept ? s->list[at + e] : 0;
        upto[e] = w[e] = at + e < kept ? Row::units(r.weight(logit_of((uint32_t)entry[e]))) : 0;
    }
    block_prefix(s, upto);
    if (threadIdx.x == SM_THREADS - 1) s->above = upto[1];
    __syncthreads();
    const unsigned long long sum = s->above;
    const double point = (double)set.u * (double)sum;
    const unsigned long long goal = point < (double)sum ? min((unsigned long long)point, sum - 1) : sum - 1;
#pragma unroll
    for (int e = 0; e < 2; ++e)
        if (w[e] && upto[e] > goal && upto[e] - w[e] <= goal) s->found = 0xffffffffu - (unsigned)(entry[e] >> 32);
    __syncthreads();
    return (int)s->found;
}

// A row of its own: one that others point to is read again from memory behind every atomic (64 mixed rows of 128000: 65 us, so 58).
__device__ __noinline__ int draw_from_list(Row &given, Settings set, float mine) {
    Row r = given;
    const int token = draw_from_list_body(r, set, mine);
    given.meeting = r.meeting, given.round = r.round;
    return token;
}

// The token, whatever the settings leave.
__device__ __noinline__ int draw_by_search(const Row &given, uint32_t top_key, unsigned vocab, Settings set) {
    Row r = given;
    uint32_t cut = KEY_NONE + 1;  // kept: key > cut, or key == cut and index <= cut_index
    unsigned cut_index = 0xffffffffu;
    auto kept = [&](unsigned i, float x) {
        const uint32_t key = key_of(x);
        return key > cut || (key == cut && i <= cut_index);
    };
    if (set.k > 0) {
        const unsigned long long k = (unsigned long long)set.k;
        auto one = [&](unsigned, float x) { return (unsigned long long)(key_of(x) > KEY_NONE); };
        if (r.total(one) > k) {
            unsigned long long above, at;
            const uint32_t key = r.search(one, top_key, k, &above, &at);
            if (above + at > k)
                cut_index = r.locate([&](unsigned, float x) { return (unsigned long long)(key_of(x) == key); },
                                     [&](unsigned long long) { return k - above - 1; });
            cut = key;
        }
    }
    if (set.top_p < 1.0f) {
        auto mass = [&](unsigned i, float x) { return kept(i, x) ? Row::units(r.weight(x)) : 0ull; };
        const unsigned long long sum = r.total(mass);
        unsigned long long target = set.top_p > 0.0f ? (unsigned long long)ceil((double)set.top_p * (double)sum) : 1ull;
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
    return (int)r.draw(kept, set.min_p, set.u);
}

__global__ void __launch_bounds__(SM_THREADS, 2) sample_kernel(const SampleArgs p) {
    __shared__ Shared sh;
    grid_dependency_wait();
    grid_launch_dependents();
    Row r;
    r.s = &sh;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r.rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r.ranks));
    const size_t row = blockIdx.x / r.ranks;
    r.l = p.logits + row * p.row_stride;
    r.vec = (reinterpret_cast<uintptr_t>(r.l) & 15) == 0;
    r.meeting = r.round = 0;
    // indices of a CTA, and of a warp in it: contiguous, in whole 128-byte lines
    const unsigned span = ((p.vocab + r.ranks - 1) / r.ranks + 31) & ~31u;
    r.warp_span = ((span + SM_WARPS - 1) / SM_WARPS + 31) & ~31u;
    r.cta_begin = min(r.rank * span, p.vocab), r.cta_end = min(r.cta_begin + span, p.vocab);
    r.begin = min(r.cta_begin + (threadIdx.x >> 5) * r.warp_span, r.cta_end);
    r.end = min(r.begin + r.warp_span, r.cta_end);
    for (int i = threadIdx.x; i < 2 * SM_BUCKETS; i += SM_THREADS) (&sh.mass[0][0])[i] = 0;
    for (int i = threadIdx.x; i < 3 * SM_BUCKETS; i += SM_THREADS) (&sh.count[0][0])[i] = 0;
    for (int i = threadIdx.x; i < 2 * SM_BUCKETS; i += SM_THREADS) (&sh.low[0][0])[i] = (&sh.high[0][0])[i] = 0;
    if (threadIdx.x == 0) sh.listed = sh.kept = sh.found = 0;

    // Settings now: their latency passes under the first pass.
    const float t = p.temperature ? p.temperature[row] : 1.0f, u = p.uniform[row];
    Settings set;
    set.k = p.top_k ? p.top_k[row] : 0;
    set.top_p = p.top_p ? p.top_p[row] : 1.0f;
    set.min_p = p.min_p ? p.min_p[row] : 0.0f;
    set.k = set.k > 0 && (unsigned)set.k < p.vocab ? set.k : 0;
    set.top_p = set.top_p < 1.0f ? set.top_p : 1.0f;  // NaN: off
    set.min_p = set.min_p > 0.0f ? fminf(set.min_p, 1.0f) : 0.0f;
    set.u = u > 0.0f ? u : 0.0f;

    // The largest logit (NaN is passed over).
    float top = -INFINITY;
    r.each([&](unsigned, float x) { top = fmaxf(top, x); });
    const uint32_t top_key = (uint32_t)Row::ranks_max(r.tell(r.block_max(key_of(top))));
    int token;
    if (top_key <= KEY_NONE) {
        token = -1;  // no logit to choose
    } else if (!(t > 0.0f)) {
        unsigned long long place = 0;  // the lowest index, as the largest of 2^32 - 1 - index
        const float largest = logit_of(top_key);
        r.each([&](unsigned i, float x) {
            if (x == largest && 0xffffffffu - i > place) place = 0xffffffffu - i;
        });
        place = Row::ranks_max(r.tell(r.block_max(place)));
        token = (int)(0xffffffffu - (unsigned)place);
    } else {
        r.top = logit_of(top_key);
        r.temperature = t;
        // finite, so that 0 * scale is 0; beside an infinite logit all others weigh nothing, whatever the temperature
        r.scale = isinf(r.top) ? 3.402823466e38f : fminf(__fdiv_rn(1.44269504088896340736f, r.temperature), 3.402823466e38f);
        token = -2;
        // (under a temperature near or at infinity -inf would get a weight there: the search asks for the key first)
        Row at = r;
        if (t < 1e30f && (set.k > 0 || set.top_p < 1.0f || set.min_p > 0.0f)) token = draw_from_list(at, set, top);
        if (token == -2) {
            cluster_meet();  // the buckets have been read by everybody
            for (int i = threadIdx.x; i < 2 * SM_BUCKETS; i += SM_THREADS) (&sh.mass[0][0])[i] = 0;
            token = draw_by_search(at, top_key, p.vocab, set);
        }
    }
    if (r.rank == 0 && threadIdx.x == 0) p.tokens[row] = token;
    cluster_part();
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
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a->logits) | reinterpret_cast<uintptr_t>(a->temperature) | reinterpret_cast<uintptr_t>(a->top_k) |
                           reinterpret_cast<uintptr_t>(a->top_p) | reinterpret_cast<uintptr_t>(a->min_p) | reinterpret_cast<uintptr_t>(a->uniform) |
                           reinterpret_cast<uintptr_t>(a->tokens);
    if (bits & 3) return fail(NNE_ERR_INVALID_ARGUMENT, "device pointers must be 4-byte aligned");
    // CTAs a row: as many as leave each at least 2048 logits (four a thread), up to the 8 of a portable cluster.
    unsigned ranks = 1;
    while (ranks < 8 && a->vocab >= (size_t)ranks * 2 * 2048) ranks *= 2;
    // and not more than run at once, two an SM: a second round would wait for the first one's meetings
    while (ranks > 1 && a->rows * ranks > 2 * (size_t)ctx->sm_count) ranks /= 2;
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
