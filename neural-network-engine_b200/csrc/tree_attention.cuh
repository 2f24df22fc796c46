// Attention of drafted token trees over the paged cache: the kernel.  tree_attention.cu has the host side, and one
// source file a cache type instantiates it.
//
// A row is one query head of one node.  The rows that share a key/value head - all nodes of a sequence times the
// query heads of the group - meet each key together.  The scores are formed as S^T = K Q^T: mma.sync m16n8k16 with 16
// keys on the M side and 8 rows on the N side, so that one node of a grouped head (4 or 8 rows) fills a tile that the
// other way round would leave half empty; O^T = V^T P^T takes the probabilities back in by an 8x8 transpose in
// registers (movmatrix).  Keys and values are the MMA's operands as they lie in the cache, exact.  q and P are f32: they
// enter as sums of two (f16) or three (bf16) numbers of the cache's type, 22 or 24 bits, after a power of two
// that keeps the small parts above f16's subnormals.  One part instead would be 2 to 3 times fewer MMAs and an error of 2^-11 or 2^-8
// where the rest of the decode step keeps 2^-23.  A tile's products with P are summed from zero and join O by an f32 FMA that also
// takes the rescaling by exp2(old max - new max): the running sum rounds once a tile, to nearest (the MMA truncates).
//
// One CTA takes up to 64 rows and a share of the keys in tiles of 64, double or triple buffered with
// cp.async (rows of a tile come from up to eight pages); its warps split the tile's keys and the rows.  The
// CTAs of a cluster take the shares of one set of rows and join max, sum and O through each other's shared memory, in rank
// order: no workspace, no second launch, results that do not change from run to run.
#pragma once

#include "kvcache.cuh"
#include "ptx.cuh"

namespace nne {

struct TreeArgs {
    const float *q;
    float *out;
    size_t q_stride, out_stride;
    int group, kv_heads;      // query heads of a key/value head
    int tokens, max_nodes;
    const int32_t *node_start, *context;
    const uint64_t *visible;  // or null: a chain
    const int32_t *page_table;
    size_t table_stride, pages;
    int page_shift;
    float scale;              // times log2(e)
    const void *k, *v;
    int vec_out;
    // Shares that a cluster cannot hold: each CTA leaves its rows here, [set of rows][share][row][D + 4] with the maximum and
    // the sum behind a row's D numbers, and tree_gather_kernel joins them.
    float *part;
};

constexpr int TREE_KEYS = 64;   // keys of a tile
constexpr int TREE_IDS = 8;     // tiles whose row numbers are held
constexpr int TREE_SHARES = 128;  // shares that tree_gather_kernel joins at most: one a thread

template <typename T>
struct TreeType;
template <>
struct TreeType<__half> {
    static constexpr int PARTS = 2;
    static constexpr float P_BIAS = 15.0f;  // P is held times 2^15: its second part stays above the subnormals
};
template <>
struct TreeType<__nv_bfloat16> {
    static constexpr int PARTS = 3;
    static constexpr float P_BIAS = 0.0f;
};

// NT: 8-row tiles of a warp; WN, WK: warps side by side along rows and along a tile's keys.
template <typename T, int D, int NT, int WN, int WK>
struct TreeShape {
    static constexpr int PARTS = TreeType<T>::PARTS;
    static constexpr int THREADS = WN * WK * 32;
    static constexpr int ROWS = 8 * NT * WN;
    static constexpr int KM = TREE_KEYS / (16 * WK);        // 16-key tiles of a warp
    static constexpr int PITCH = 2 * D + 16;                // bytes of a key in shared memory: ldmatrix without conflicts
    static constexpr int TILE = TREE_KEYS * PITCH;
    static constexpr int STAGES = D <= 64 ? 4 : 2;
    static constexpr int Q_BYTES = PARTS * (ROWS / 8) * (D / 16) * 256;
    static constexpr int OPITCH = D + 4;                    // floats of a row of O at the end
    static constexpr int RING = STAGES * 2 * TILE;
    static constexpr int O_BYTES = WK * ROWS * OPITCH * 4;
    static constexpr int MAIN = RING > O_BYTES ? RING : O_BYTES;
    static constexpr int SMEM = MAIN + Q_BYTES + ROWS * 8 + ROWS * 4 + (2 * WK + 2) * ROWS * 4 + TREE_IDS * (TREE_KEYS / 8) * 4 + 16;
    static constexpr int PER_SM = 2 * (SMEM + 1024) <= 227 * 1024 ? 2 : 1;
};

__device__ __forceinline__ void ldsm_x4(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
template <typename T>
__device__ __forceinline__ void mma_16x8x16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_16x8x16<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma_16x8x16<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// The same from an accumulator of 0, which is no register: the first MMA of a chain.
template <typename T>
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma_first<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
template <>
__device__ __forceinline__ void mma_first<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// 2^x; below 2^-126: 0.
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// 16 bytes into shared memory, or zeros.
__device__ __forceinline__ void cp_async_16_or_zero(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ float ld_cluster_f32(uint32_t at, uint32_t rank) {
    uint32_t peer;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(peer) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster_f4(uint32_t at, uint32_t rank) {
    uint32_t peer;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(peer) : "memory");
    return v;
}

// Queries: scale * log2(e) * q, as parts of the cache's type in the MMA's operand order [part][8-row tile][step][lane].
// f16: times a power of two that brings a row's largest to [2^13, 2^14), undone by qfac.  vis: what a row's node sees.
template <typename T, int D, int ROWS, int THREADS>
__device__ __forceinline__ void tree_queries(const TreeArgs &p, uint2 *qfrag, uint64_t *vis, float *qfac, int start, int row_base, int nrows, int kvh) {
    constexpr int PARTS = TreeType<T>::PARTS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = warp; r < ROWS; r += THREADS / 32) {
        constexpr int PL = (D / 2 + 31) / 32;  // pairs of a lane
        float2 x[PL];
        float top = 0.0f;
        const int row = row_base + r, node = row / p.group;
        const bool there = r < nrows;
        const float *src = p.q + (size_t)(there ? start + node : 0) * p.q_stride + (size_t)(kvh * p.group + row % p.group) * D;
#pragma unroll
        for (int i = 0; i < PL; ++i) {
            const int c = lane + i * 32;
            x[i] = make_float2(0.0f, 0.0f);
            if (there && c < D / 2) x[i] = make_float2(src[2 * c] * p.scale, src[2 * c + 1] * p.scale);
            top = fmaxf(top, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
        }
        float up = 1.0f, down = 1.0f;
        if (sizeof(T) == 2 && PARTS == 2) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            int e = 13 + 127 - ((int)(__float_as_uint(top) >> 23) & 255);
            e = e > 120 ? 120 : (e < -114 ? -114 : e);
            up = __uint_as_float((uint32_t)(e + 127) << 23);
            down = __uint_as_float((uint32_t)(127 - e) << 23);
        }
#pragma unroll
        for (int i = 0; i < PL; ++i) {
            const int c = lane + i * 32;
            if (c >= D / 2) continue;
            float2 v = make_float2(x[i].x * up, x[i].y * up);
            const int step = c / 8, word = (c % 8) / 4, at = (r % 8) * 4 + c % 4;
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
                const uint32_t w = pack_pair<T>(v.x, v.y);
                const float2 back = unpack_pair<T>(w);
                v = make_float2(v.x - back.x, v.y - back.y);
                reinterpret_cast<uint32_t *>(qfrag + ((q * (ROWS / 8) + r / 8) * (D / 16) + step) * 32 + at)[word] = w;
            }
        }
        if (lane == 0) {
            qfac[r] = down;
            uint64_t bits = 0;
            if (there) bits = p.visible ? p.visible[start + node] : (node >= 63 ? ~0ull : (2ull << node) - 1);
            vis[r] = bits;
        }
    }
}

// Joins what the warps along the keys and the CTAs of the cluster have of each row, and writes the rows.  o: 16 dimensions x 8
// rows a tile as the MMA leaves them; m, l: maximum and (this lane's part of the) sum.  `smem`: WK * ROWS * (D + 4) floats.
template <int D, int NT, int WN, int WK>
__device__ __forceinline__ void tree_join(const TreeArgs &p, const float (&o)[D / 16][NT][4], const float (&m)[NT][2], float (&l)[NT][2], uint8_t *smem,
                                          float *m_w, float *l_w, float *m_row, float *l_row, int start, int row_base, int nrows, int kvh) {
    constexpr int ROWS = 8 * NT * WN, THREADS = WN * WK * 32, OPITCH = D + 4;
    constexpr float NEG = -INFINITY;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int wn = warp % WN, wk = warp / WN, g = lane >> 2, t4 = lane & 3;
    const unsigned split = gridDim.x, rank = blockIdx.x;
    // The warps along the keys join: maximum and sum of a row, then O, warp after warp.
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], w);
            if (g == 0) {
                const int r = (wn * NT + n) * 8 + 2 * t4 + e;
                m_w[wk * ROWS + r] = m[n][e];
                l_w[wk * ROWS + r] = l[n][e];
            }
        }
    __syncthreads();  // m, l; and nobody reads the ring any more: O goes over it
    float *om = reinterpret_cast<float *>(smem);  // [WK][ROWS][OPITCH], the sum into the first
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                om[(wk * ROWS + (wn * NT + n) * 8 + 2 * t4 + (e & 1)) * OPITCH + i * 16 + (e >> 1) * 8 + g] = o[i][n][e];
    __syncthreads();
    for (int i = tid; i < nrows * (D / 4); i += THREADS) {
        const int r = i / (D / 4), c = (i % (D / 4)) * 4;
        float top = NEG, sum = 0.0f;
#pragma unroll
        for (int w = 0; w < WK; ++w) top = fmaxf(top, m_w[w * ROWS + r]);
        const float ref = top == NEG ? 0.0f : top;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < WK; ++w) {
            const float k = ex2(m_w[w * ROWS + r] - ref);
            const float4 x = *reinterpret_cast<const float4 *>(om + (w * ROWS + r) * OPITCH + c);
            sum = fmaf(l_w[w * ROWS + r], k, sum);
            v.x = fmaf(x.x, k, v.x), v.y = fmaf(x.y, k, v.y), v.z = fmaf(x.z, k, v.z), v.w = fmaf(x.w, k, v.w);
        }
        *reinterpret_cast<float4 *>(om + r * OPITCH + c) = v;
        if (c == 0) m_row[r] = top, l_row[r] = sum;
    }
    __syncthreads();

    if (p.part) {
        float *mine = p.part + (((size_t)blockIdx.z * gridDim.y + blockIdx.y) * split + rank) * ROWS * (D + 4);
        for (int i = tid; i < nrows * (D / 4); i += THREADS) {
            const int r = i / (D / 4), c = (i % (D / 4)) * 4;
            *reinterpret_cast<float4 *>(mine + r * (D + 4) + c) = *reinterpret_cast<const float4 *>(om + r * OPITCH + c);
            if (c == 0) mine[r * (D + 4) + D] = m_row[r], mine[r * (D + 4) + D + 1] = l_row[r];
        }
        return;
    }

    // The CTAs of the cluster join, rank after rank; each writes its share of the rows' elements.
    if (split > 1) cluster_meet();
    const uint32_t om_at = smem_u32(om), m_at = smem_u32(m_row), l_at = smem_u32(l_row);
    for (int i = (int)rank * THREADS + tid; i < nrows * (D / 4); i += (int)split * THREADS) {
        const int r = i / (D / 4), c = (i % (D / 4)) * 4;
        float top = NEG;
        for (unsigned w = 0; w < split; ++w) top = fmaxf(top, ld_cluster_f32(m_at + r * 4, w));
        const float ref = top == NEG ? 0.0f : top;
        float sum = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (unsigned w = 0; w < split; ++w) {
            const float k = ex2(ld_cluster_f32(m_at + r * 4, w) - ref);
            const float4 x = ld_cluster_f4(om_at + (r * OPITCH + c) * 4, w);
            sum = fmaf(ld_cluster_f32(l_at + r * 4, w), k, sum);
            v.x = fmaf(x.x, k, v.x), v.y = fmaf(x.y, k, v.y), v.z = fmaf(x.z, k, v.z), v.w = fmaf(x.w, k, v.w);
        }
        if (sum == 0.0f) {
            v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // a row that sees nothing
        } else {
            v.x = __fdiv_rn(v.x, sum), v.y = __fdiv_rn(v.y, sum), v.z = __fdiv_rn(v.z, sum), v.w = __fdiv_rn(v.w, sum);
        }
        const int row = row_base + r;
        float *dst = p.out + (size_t)(start + row / p.group) * p.out_stride + (size_t)(kvh * p.group + row % p.group) * D + c;
        if (p.vec_out) {
            *reinterpret_cast<float4 *>(dst) = v;
        } else {
            dst[0] = v.x, dst[1] = v.y, dst[2] = v.z, dst[3] = v.w;
        }
    }
    if (split > 1) cluster_meet();  // nobody leaves while a peer may still read its shared memory
}

template <typename T, int D, int NT, int WN, int WK>
__global__ void __launch_bounds__(TreeShape<T, D, NT, WN, WK>::THREADS, TreeShape<T, D, NT, WN, WK>::PER_SM)
tree_attention_kernel(const TreeArgs p) {
    using S = TreeShape<T, D, NT, WN, WK>;
    constexpr int PARTS = S::PARTS, KM = S::KM, ROWS = S::ROWS, THREADS = S::THREADS, STAGES = S::STAGES;
    constexpr float NEG = -INFINITY;
    extern __shared__ __align__(16) uint8_t smem[];
    uint2 *qfrag = reinterpret_cast<uint2 *>(smem + S::MAIN);                     // [part][8-row tile][step][lane]
    uint64_t *vis = reinterpret_cast<uint64_t *>(smem + S::MAIN + S::Q_BYTES);    // [ROWS]
    float *qfac = reinterpret_cast<float *>(vis + ROWS);                          // [ROWS]
    float *m_w = qfac + ROWS, *l_w = m_w + WK * ROWS;                             // [WK][ROWS] each
    float *m_row = l_w + WK * ROWS, *l_row = m_row + ROWS;                        // [ROWS] each
    int *ids = reinterpret_cast<int *>(l_row + ROWS);                             // [TREE_IDS][TREE_KEYS / 8]
    unsigned long long *odd_keys = reinterpret_cast<unsigned long long *>(
        (reinterpret_cast<uintptr_t>(ids + TREE_IDS * (TREE_KEYS / 8)) + 7) & ~(uintptr_t)7);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int wn = warp % WN, wk = warp / WN, g = lane >> 2, t4 = lane & 3;
    const unsigned split = gridDim.x, rank = blockIdx.x;
    const int kvh = blockIdx.y % p.kv_heads, b = blockIdx.z;
    const int row_base = (int)(blockIdx.y / p.kv_heads) * ROWS;

    grid_dependency_wait();
    grid_launch_dependents();

    const int start = p.node_start[b];
    int nodes = p.node_start[b + 1] - start;
    nodes = start < 0 || start > p.tokens ? 0 : min(min(nodes, p.max_nodes), p.tokens - start);
    const int rows = max(nodes, 0) * p.group;
    if (row_base >= rows) return;  // the whole cluster
    const int nrows = min(ROWS, rows - row_base);
    const int ctx = max(p.context[b], 0);
    const long long room = (long long)p.table_stride << p.page_shift;  // places that the table can name
    const int total = (int)min((long long)ctx + nodes, min(room, 0x7fffffc0ll));
    const int tiles = (total + TREE_KEYS - 1) / TREE_KEYS;
    const int per = (tiles + (int)split - 1) / (int)split;
    const int t0 = min((int)rank * per, tiles), t1 = min(t0 + per, tiles);
    const int32_t *table = p.page_table + (size_t)b * p.table_stride;

    // Row of the pool of eight keys of a tile (thread < 8), or -1: eight in a row lie in one page.
    auto id_of = [&](int tile) {
        const int key = tile * TREE_KEYS + tid * 8;
        return key < total ? kv_row(table, p.table_stride, key, p.page_shift, p.pages, p.kv_heads, kvh) : -1;
    };
    const uint32_t ring = smem_u32(smem);
    auto issue = [&](int tile) {
        if (tile < t1) {
            const int *id = ids + (tile % TREE_IDS) * (TREE_KEYS / 8);
            const uint32_t dst = ring + ((tile - t0) % STAGES) * 2 * S::TILE;
            const int left = total - tile * TREE_KEYS;
            static_assert(TREE_KEYS * (D / 8) % THREADS == 0, "whole rounds of copies");
#pragma unroll
            for (int j = 0; j < TREE_KEYS * (D / 8) / THREADS; ++j) {
                const int i = tid + j * THREADS, r = i / (D / 8), c = i % (D / 8), row = id[r >> 3];
                const bool there = row >= 0 && r < left;
                const size_t at = ((size_t)(there ? row + (r & 7) : 0) * D + c * 8) * 2;
                cp_async_16_or_zero(dst + r * S::PITCH + c * 16, static_cast<const uint8_t *>(p.k) + at, there);
                cp_async_16_or_zero(dst + S::TILE + r * S::PITCH + c * 16, static_cast<const uint8_t *>(p.v) + at, there);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if (tid < TREE_KEYS / 8) {
#pragma unroll
        for (int j = 0; j < STAGES; ++j)
            if (t0 + j < t1) ids[((t0 + j) % TREE_IDS) * (TREE_KEYS / 8) + tid] = id_of(t0 + j);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < STAGES - 1; ++j) issue(t0 + j);

    tree_queries<T, D, ROWS, THREADS>(p, qfrag, vis, qfac, start, row_base, nrows, kvh);

    float o[D / 16][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = NEG, l[n][0] = l[n][1] = 0.0f;

    for (int t = t0; t < t1; ++t) {
        asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
        __syncthreads();  // tile t is there for everybody; tile t - 1's buffer is free
        issue(t + STAGES - 1);
        int next_id = -1;  // looked up now, stored below: the table's latency passes under the tile's work
        const bool looks = tid < TREE_KEYS / 8 && t + STAGES < t1;
        if (looks) next_id = id_of(t + STAGES);
        const uint32_t kt = ring + ((t - t0) % STAGES) * 2 * S::TILE, vt = kt + S::TILE;
        const int *id = ids + (t % TREE_IDS) * (TREE_KEYS / 8);
        const int key0 = t * TREE_KEYS;
        const bool drafted = key0 + TREE_KEYS > ctx;  // the tile holds keys that not every node sees (or none)

        // A drafted key that some row does not see must not reach it through 0 * Inf or 0 * NaN: values that are not
        // finite are taken out of the tile and added by hand to the rows that see them.
        unsigned long long odd = 0;
        if (drafted) {
            if (tid == 0) *odd_keys = 0;
            __syncthreads();
            for (int i = tid; i < TREE_KEYS * (D / 8); i += THREADS) {
                const int r = i / (D / 8), c = i % (D / 8);
                if (key0 + r < ctx || key0 + r >= total) continue;
                const uint4 w = *reinterpret_cast<const uint4 *>(smem + (vt - ring) + r * S::PITCH + c * 16);
                const uint32_t e = PARTS == 2 ? 0x7c00u : 0x7f80u;
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
                bool bad = false;
#pragma unroll
                for (int q = 0; q < 4; ++q) bad |= (x[q] & e) == e || ((x[q] >> 16) & e) == e;
                if (bad) atomicOr(odd_keys, 1ull << r);
            }
            __syncthreads();
            odd = *odd_keys;
            if (odd) {  // the same for the whole CTA
                for (int i = tid; i < TREE_KEYS * (D / 8); i += THREADS) {
                    const int r = i / (D / 8), c = i % (D / 8);
                    if (odd >> r & 1) *reinterpret_cast<uint4 *>(smem + (vt - ring) + r * S::PITCH + c * 16) = make_uint4(0, 0, 0, 0);
                }
                __syncthreads();
            }
        }

        if (wn * 8 * NT < nrows) {  // a warp without rows only helps to load
            // S^T: the small parts of q in one accumulator, the large one in another
            float s[KM][NT][4], s2[KM][NT][4];
            const uint32_t ka = kt + (wk * KM * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * S::PITCH + (lane >> 4) * 16;
            const uint2 *qf = qfrag + (wn * NT) * (D / 16) * 32 + lane;
#pragma unroll
            for (int step = 0; step < D / 16; ++step) {
                uint32_t a[KM][4];
#pragma unroll
                for (int k = 0; k < KM; ++k) ldsm_x4(a[k], ka + k * 16 * S::PITCH + step * 32);
#pragma unroll
                for (int q = 0; q < PARTS; ++q)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const uint2 w = qf[((q * (ROWS / 8) + n) * (D / 16) + step) * 32];
#pragma unroll
                        for (int k = 0; k < KM; ++k) {
                            float(&acc)[4] = q == 0 ? s[k][n] : s2[k][n];
                            if (step == 0 && q < 2) mma_first<T>(acc, a[k], w.x, w.y);
                            else mma_16x8x16<T>(acc, a[k], w.x, w.y);
                        }
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float f0 = PARTS == 2 ? qfac[(wn * NT + n) * 8 + 2 * t4] : 1.0f;
                const float f1 = PARTS == 2 ? qfac[(wn * NT + n) * 8 + 2 * t4 + 1] : 1.0f;
#pragma unroll
                for (int k = 0; k < KM; ++k)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[k][n][e] = (s[k][n][e] + s2[k][n][e]) * ((e & 1) ? f1 : f0);
            }
            // What a row does not see, and keys without a place in the pool.
            bool gap = false;
#pragma unroll
            for (int k = 0; k < KM; ++k) gap |= id[(wk * KM + k) * 2 + (lane & 1)] < 0;
            if (drafted || __any_sync(0xffffffffu, gap)) {
#pragma unroll
                for (int k = 0; k < KM; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int r = (wk * KM + k) * 16 + h * 8 + g, j = key0 + r - ctx;
                        const bool there = id[r >> 3] >= 0 && key0 + r < total;
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const bool sees = there && (j < 0 || (vis[(wn * NT + n) * 8 + 2 * t4 + e] >> j & 1));
                                if (!sees) s[k][n][2 * h + e] = NEG;
                            }
                    }
            }
            // Running maximum, probabilities, their sum.
            float alpha[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float top = m[n][e];
#pragma unroll
                    for (int k = 0; k < KM; ++k) top = fmaxf(top, fmaxf(s[k][n][e], s[k][n][2 + e]));
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                    const float ref = top == NEG ? 0.0f : top;
                    alpha[n][e] = ex2(m[n][e] - ref);
                    m[n][e] = top;
                    float sum = 0.0f;
#pragma unroll
                    for (int k = 0; k < KM; ++k)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float v = ex2(s[k][n][2 * h + e] - ref + TreeType<T>::P_BIAS);
                            s[k][n][2 * h + e] = v;
                            sum += v;
                        }
                    l[n][e] = fmaf(l[n][e], alpha[n][e], sum);
                }
            // P^T in parts, transposed into operand order, the smallest part first.
            uint32_t pf[KM][NT][PARTS][2];
#pragma unroll
            for (int k = 0; k < KM; ++k)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        float2 v = make_float2(s[k][n][2 * h], s[k][n][2 * h + 1]);
#pragma unroll
                        for (int q = 0; q < PARTS; ++q) {
                            const uint32_t w = pack_pair<T>(v.x, v.y);
                            const float2 back = unpack_pair<T>(w);
                            v = make_float2(v.x - back.x, v.y - back.y);
                            pf[k][n][PARTS - 1 - q][h] = transpose_8x8(w);
                        }
                    }
            const uint32_t va = vt + (wk * KM * 16 + (lane & 7) + (lane >> 4) * 8) * S::PITCH + ((lane >> 3) & 1) * 16;
            constexpr int W = 2;  // dimension tiles side by side: no MMA waits for the one before it
#pragma unroll
            for (int i = 0; i < D / 16; i += W) {
                float add[W][NT][4];
#pragma unroll
                for (int k = 0; k < KM; ++k) {
                    uint32_t a[W][4];
#pragma unroll
                    for (int w = 0; w < W; ++w) ldsm_x4_trans(a[w], va + k * 16 * S::PITCH + (i + w) * 32);
#pragma unroll
                    for (int q = 0; q < PARTS; ++q)
#pragma unroll
                        for (int w = 0; w < W; ++w)
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                if (k == 0 && q == 0) mma_first<T>(add[w][n], a[w], pf[k][n][q][0], pf[k][n][q][1]);
                                else mma_16x8x16<T>(add[w][n], a[w], pf[k][n][q][0], pf[k][n][q][1]);
                            }
                }
#pragma unroll
                for (int w = 0; w < W; ++w)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i + w][n][e] = fmaf(o[i + w][n][e], alpha[n][e & 1], add[w][n][e]);
            }
            if (odd) {
                const T *vg = static_cast<const T *>(p.v);
#pragma unroll
                for (int k = 0; k < KM; ++k)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        for (int j = 0; j < 8; ++j) {
                            const int r = (wk * KM + k) * 16 + h * 8 + j;
                            if (!(odd >> r & 1)) continue;
                            const size_t at = (size_t)(max(id[r >> 3], 0) + (r & 7)) * D;
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const float w = __shfl_sync(0xffffffffu, s[k][n][2 * h + e], j * 4 + t4);
                                    if (w == 0.0f) continue;
#pragma unroll
                                    for (int i = 0; i < D / 16; ++i) {
                                        o[i][n][e] += w * (float)vg[at + i * 16 + g];
                                        o[i][n][2 + e] += w * (float)vg[at + i * 16 + 8 + g];
                                    }
                                }
                        }
            }
        }
        if (looks) ids[((t + STAGES) % TREE_IDS) * (TREE_KEYS / 8) + tid] = next_id;
    }

    tree_join<D, NT, WN, WK>(p, o, m, l, smem, m_w, l_w, m_row, l_row, start, row_base, nrows, kvh);
}

// Few rows (one node, or a few of a small group): the keys are all the work.  Each of the CTA's four warps takes every
// fourth group of 16 keys of the share and loads it for itself, so that no warp ever waits for another: with tiles shared by the CTA a
// tile of 64 keys took 1950 cycles, most of them at barriers and in address arithmetic.  Eight keys in a row lie in one page (pages are
// 8 places or more), so a group is two look-ups, made one group ahead of the copies they serve.
template <typename T, int D, int NT>
struct DecodeShape {
    static constexpr int PARTS = TreeType<T>::PARTS;
    static constexpr int WARPS = 4;
    static constexpr int ROWS = 8 * NT, THREADS = WARPS * 32;
    static constexpr int PITCH = 2 * D + 16;
    static constexpr int HALF = 16 * PITCH;                 // 16 keys; a slot is keys and values
    static constexpr int SLOTS = 3;
    static constexpr int RING = WARPS * SLOTS * 2 * HALF;
    static constexpr int O_BYTES = WARPS * ROWS * (D + 4) * 4;
    static constexpr int MAIN = RING > O_BYTES ? RING : O_BYTES;
    static constexpr int Q_BYTES = PARTS * NT * (D / 16) * 256;
    static constexpr int SMEM = MAIN + Q_BYTES + ROWS * 8 + ROWS * 4 + (2 * WARPS + 2) * ROWS * 4 + WARPS * SLOTS * 2 * 4;
    static constexpr int FIT = 227 * 1024 / (SMEM + 1024);
    static constexpr int PER_SM = FIT < 1 ? 1 : (FIT > 3 ? 3 : FIT);  // three: 168 registers a thread
    static constexpr bool Q_REGS = NT * (D / 16) * PARTS * 2 <= 48;
};

template <typename T, int D, int NT>
__global__ void __launch_bounds__(DecodeShape<T, D, NT>::THREADS, DecodeShape<T, D, NT>::PER_SM) tree_decode_kernel(const TreeArgs p) {
    using S = DecodeShape<T, D, NT>;
    constexpr int PARTS = S::PARTS, ROWS = S::ROWS, SLOTS = S::SLOTS, WARPS = S::WARPS;
    constexpr float NEG = -INFINITY;
    extern __shared__ __align__(16) uint8_t smem[];
    uint2 *qfrag = reinterpret_cast<uint2 *>(smem + S::MAIN);
    uint64_t *vis = reinterpret_cast<uint64_t *>(smem + S::MAIN + S::Q_BYTES);
    float *qfac = reinterpret_cast<float *>(vis + ROWS);
    float *m_w = qfac + ROWS, *l_w = m_w + WARPS * ROWS, *m_row = l_w + WARPS * ROWS, *l_row = m_row + ROWS;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    int *ids = reinterpret_cast<int *>(l_row + ROWS) + warp * SLOTS * 2;  // [slot][2]: rows of the pool of the group's halves
    const int kvh = blockIdx.y % p.kv_heads, b = blockIdx.z;
    const int row_base = (int)(blockIdx.y / p.kv_heads) * ROWS;

    grid_dependency_wait();
    grid_launch_dependents();

    const int start = p.node_start[b];
    int nodes = p.node_start[b + 1] - start;
    nodes = start < 0 || start > p.tokens ? 0 : min(min(nodes, p.max_nodes), p.tokens - start);
    const int rows = max(nodes, 0) * p.group;
    if (row_base >= rows) return;  // the whole cluster
    const int nrows = min(ROWS, rows - row_base);
    const int ctx = max(p.context[b], 0);
    const long long room = (long long)p.table_stride << p.page_shift;
    const int total = (int)min((long long)ctx + nodes, min(room, 0x7fffffc0ll));
    const int groups = (total + 15) / 16, per = (groups + (int)gridDim.x - 1) / (int)gridDim.x;
    const int g0 = min((int)blockIdx.x * per, groups) + warp, g1 = min((int)blockIdx.x * per + per, groups);
    const int32_t *table = p.page_table + (size_t)b * p.table_stride;

    // Row of the pool of half `lane` (0, 1) of a group, or -1.
    auto look = [&](int grp) {
        const int key = grp * 16 + lane * 8;
        return lane < 2 && grp < g1 && key < total ? kv_row(table, p.table_stride, key, p.page_shift, p.pages, p.kv_heads, kvh) : -1;
    };
    const uint32_t ring = smem_u32(smem) + warp * (SLOTS * 2 * S::HALF);
    auto issue = [&](int grp, int slot, int row) {
        if (grp < g1) {
            const int r0 = __shfl_sync(0xffffffffu, row, 0), r1 = __shfl_sync(0xffffffffu, row, 1);
            if (lane < 2) ids[slot * 2 + lane] = row;
            const int left = total - grp * 16;
            const uint32_t dst = ring + slot * 2 * S::HALF;
            if (left >= 16 && r0 >= 0 && r1 >= 0) {
                const uint8_t *k0 = static_cast<const uint8_t *>(p.k) + (size_t)r0 * D * 2, *k1 = static_cast<const uint8_t *>(p.k) + ((size_t)r1 - 8) * D * 2;
                const ptrdiff_t to_v = static_cast<const uint8_t *>(p.v) - static_cast<const uint8_t *>(p.k);
#pragma unroll
                for (int j = 0; j < D / 16; ++j) {
                    const int i = lane + 32 * j, r = i / (D / 8), c = i % (D / 8);
                    const uint8_t *src = (r < 8 ? k0 : k1) + (r * D + c * 8) * 2;
                    cp_async_16(dst + r * S::PITCH + c * 16, src);
                    cp_async_16(dst + S::HALF + r * S::PITCH + c * 16, src + to_v);
                }
            } else {
                for (int j = 0; j < D / 16; ++j) {
                    const int i = lane + 32 * j, r = i / (D / 8), c = i % (D / 8), base = r < 8 ? r0 : r1;
                    const bool there = r < left && base >= 0;
                    const size_t at = ((size_t)(there ? base + (r & 7) : 0) * D + c * 8) * 2;
                    cp_async_16_or_zero(dst + r * S::PITCH + c * 16, static_cast<const uint8_t *>(p.k) + at, there);
                    cp_async_16_or_zero(dst + S::HALF + r * S::PITCH + c * 16, static_cast<const uint8_t *>(p.v) + at, there);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    {
        int row[SLOTS];
#pragma unroll
        for (int j = 0; j < SLOTS - 1; ++j) row[j] = look(g0 + WARPS * j);
#pragma unroll
        for (int j = 0; j < SLOTS - 1; ++j) issue(g0 + WARPS * j, j, row[j]);
    }
    int next = look(g0 + WARPS * (SLOTS - 1));

    tree_queries<T, D, ROWS, WARPS * 32>(p, qfrag, vis, qfac, start, row_base, nrows, kvh);
    __syncthreads();
    uint2 qr[S::Q_REGS ? NT * (D / 16) * PARTS : 1];
    if constexpr (S::Q_REGS) {
#pragma unroll
        for (int i = 0; i < NT * (D / 16) * PARTS; ++i) qr[i] = qfrag[i * 32 + lane];
    }
    float qf[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) qf[n][0] = qfac[n * 8 + 2 * t4], qf[n][1] = qfac[n * 8 + 2 * t4 + 1];

    float o[D / 16][NT][4];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int i = 0; i < D / 16; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n) o[i][n][0] = o[i][n][1] = o[i][n][2] = o[i][n][3] = 0.0f;
#pragma unroll
    for (int n = 0; n < NT; ++n) m[n][0] = m[n][1] = NEG, l[n][0] = l[n][1] = 0.0f;

    int slot = 0;
    for (int grp = g0; grp < g1; grp += WARPS) {
        asm volatile("cp.async.wait_group %0;" ::"n"(SLOTS - 2) : "memory");
        __syncwarp();  // the group is there for every lane, and every lane is done with the slot before
        issue(grp + WARPS * (SLOTS - 1), slot == 0 ? SLOTS - 1 : slot - 1, next);
        next = look(grp + WARPS * SLOTS);
        const uint32_t kt = ring + slot * 2 * S::HALF, vt = kt + S::HALF;
        const int key0 = grp * 16;
        const bool drafted = key0 + 16 > ctx;

        // Values of drafted keys that are not finite leave the slot and are added by hand to the rows that see them:
        // 0 * Inf must not reach the others.
        unsigned odd = 0;
        if (drafted) {
            for (int i = lane; i < 16 * (D / 8); i += 32) {
                const int r = i / (D / 8), c = i % (D / 8);
                if (key0 + r < ctx || key0 + r >= total) continue;
                const uint4 w = *reinterpret_cast<const uint4 *>(smem + (vt - smem_u32(smem)) + r * S::PITCH + c * 16);
                const uint32_t e = PARTS == 2 ? 0x7c00u : 0x7f80u;
                const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if ((x[q] & e) == e || ((x[q] >> 16) & e) == e) odd |= 1u << r;
            }
            odd = __reduce_or_sync(0xffffffffu, odd);
            if (odd) {
                for (int i = lane; i < 16 * (D / 8); i += 32) {
                    const int r = i / (D / 8), c = i % (D / 8);
                    if (odd >> r & 1) *reinterpret_cast<uint4 *>(smem + (vt - smem_u32(smem)) + r * S::PITCH + c * 16) = make_uint4(0, 0, 0, 0);
                }
                __syncwarp();
            }
        }

        // S^T, in chains of their own for each part and, one tile of rows, for even and odd steps: an MMA waits for
        // the one before it in its chain
        constexpr int CH = NT == 1 ? 2 : 1;
        float s[NT][4], sp[CH][PARTS][NT][4];
        const uint32_t ka = kt + ((lane & 7) + ((lane >> 3) & 1) * 8) * S::PITCH + (lane >> 4) * 16;
#pragma unroll
        for (int step = 0; step < D / 16; ++step) {
            uint32_t a[4];
            ldsm_x4(a, ka + step * 32);
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const int at = (q * NT + n) * (D / 16) + step;
                    uint2 w;
                    if constexpr (S::Q_REGS) w = qr[at];
                    else w = qfrag[at * 32 + lane];
                    if (step < CH) mma_first<T>(sp[step % CH][q][n], a, w.x, w.y);
                    else mma_16x8x16<T>(sp[step % CH][q][n], a, w.x, w.y);
                }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = 0.0f;
#pragma unroll
                for (int q = PARTS - 1; q >= 0; --q)
#pragma unroll
                    for (int c = 0; c < CH; ++c) v += sp[c][q][n][e];
                s[n][e] = PARTS == 2 ? v * qf[n][e & 1] : v;
            }
        const int id0 = ids[slot * 2], id1 = ids[slot * 2 + 1];
        if (drafted || id0 < 0 || id1 < 0) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int r = h * 8 + g, j = key0 + r - ctx;
                const bool there = (h ? id1 : id0) >= 0 && key0 + r < total;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const bool sees = there && (j < 0 || (vis[n * 8 + 2 * t4 + e] >> j & 1));
                        if (!sees) s[n][2 * h + e] = NEG;
                    }
            }
        }
        float alpha[NT][2];
        uint32_t pf[NT][PARTS][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float top = fmaxf(m[n][e], fmaxf(s[n][e], s[n][2 + e]));
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
                const float ref = top == NEG ? 0.0f : top;
                alpha[n][e] = ex2(m[n][e] - ref);
                m[n][e] = top;
                s[n][e] = ex2(s[n][e] - ref + TreeType<T>::P_BIAS);
                s[n][2 + e] = ex2(s[n][2 + e] - ref + TreeType<T>::P_BIAS);
                l[n][e] = fmaf(l[n][e], alpha[n][e], s[n][e] + s[n][2 + e]);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float2 v = make_float2(s[n][2 * h], s[n][2 * h + 1]);
#pragma unroll
                for (int q = 0; q < PARTS; ++q) {
                    const uint32_t w = pack_pair<T>(v.x, v.y);
                    const float2 back = unpack_pair<T>(w);
                    v = make_float2(v.x - back.x, v.y - back.y);
                    pf[n][PARTS - 1 - q][h] = transpose_8x8(w);
                }
            }
        }
        const uint32_t va = vt + ((lane & 7) + (lane >> 4) * 8) * S::PITCH + ((lane >> 3) & 1) * 16;
        constexpr int W = NT == 1 ? (D % 64 ? 2 : 4) : 2;  // dimension tiles side by side
#pragma unroll
        for (int i = 0; i < D / 16; i += W) {
            uint32_t a[W][4];
            float add[W][NT][4];
#pragma unroll
            for (int w = 0; w < W; ++w) {
                ldsm_x4_trans(a[w], va + (i + w) * 32);
            }
#pragma unroll
            for (int q = 0; q < PARTS; ++q)
#pragma unroll
                for (int w = 0; w < W; ++w)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (q == 0) mma_first<T>(add[w][n], a[w], pf[n][q][0], pf[n][q][1]);
                        else mma_16x8x16<T>(add[w][n], a[w], pf[n][q][0], pf[n][q][1]);
                    }
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i + w][n][e] = fmaf(o[i + w][n][e], alpha[n][e & 1], add[w][n][e]);
        }
        if (odd) {
            const T *vg = static_cast<const T *>(p.v);
#pragma unroll
            for (int h = 0; h < 2; ++h)
                for (int j = 0; j < 8; ++j) {
                    if (!(odd >> (h * 8 + j) & 1)) continue;
                    const size_t at = (size_t)(max(h ? id1 : id0, 0) + j) * D;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float w = __shfl_sync(0xffffffffu, s[n][2 * h + e], j * 4 + t4);
                            if (w == 0.0f) continue;
#pragma unroll
                            for (int i = 0; i < D / 16; ++i) {
                                o[i][n][e] += w * (float)vg[at + i * 16 + g];
                                o[i][n][2 + e] += w * (float)vg[at + i * 16 + 8 + g];
                            }
                        }
                }
        }
        slot = slot + 1 == SLOTS ? 0 : slot + 1;
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    tree_join<D, NT, 1, WARPS>(p, o, m, l, smem, m_w, l_w, m_row, l_row, start, row_base, nrows, kvh);
}

// One CTA a row: the weights of its shares (one a thread; at most 128), then each warp every fourth share, then the warps in
// order.  (One warp a row, share after share, took longer than the attention: 19 us for 37 shares.)
template <int D>
__global__ void __launch_bounds__(TREE_SHARES) tree_gather_kernel(const TreeArgs p, int rows_of_cta, int shares) {
    constexpr int V = (D / 4 + 31) / 32;  // float4s of a lane
    __shared__ float weight[TREE_SHARES], tops[4], sums[4];
    __shared__ __align__(16) float acc[4][D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, r = blockIdx.x;
    const int kvh = blockIdx.y % p.kv_heads, b = blockIdx.z, row = (int)(blockIdx.y / p.kv_heads) * rows_of_cta + r;
    grid_dependency_wait();
    grid_launch_dependents();
    const int start = p.node_start[b];
    int nodes = p.node_start[b + 1] - start;
    nodes = start < 0 || start > p.tokens ? 0 : min(min(nodes, p.max_nodes), p.tokens - start);
    if (row >= max(nodes, 0) * p.group) return;
    const size_t pitch = (size_t)rows_of_cta * (D + 4);
    const float *src = p.part + ((size_t)b * gridDim.y + blockIdx.y) * shares * pitch + (size_t)r * (D + 4);
    const float m = tid < shares ? src[tid * pitch + D] : -INFINITY, l = tid < shares ? src[tid * pitch + D + 1] : 0.0f;
    float top = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    const float w = ex2(m - (top == -INFINITY ? 0.0f : top));
    weight[tid] = w;
    float sum = l * w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    sum = sums[0] + sums[1] + sums[2] + sums[3];
    float4 v[V];
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
    for (int q = warp; q < shares; q += 4) {
        const float k = weight[q];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (lane + i * 32) * 4;
            if (c >= D) continue;
            const float4 x = *reinterpret_cast<const float4 *>(src + q * pitch + c);
            v[i].x = fmaf(x.x, k, v[i].x), v[i].y = fmaf(x.y, k, v[i].y), v[i].z = fmaf(x.z, k, v[i].z), v[i].w = fmaf(x.w, k, v[i].w);
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if ((lane + i * 32) * 4 < D) *reinterpret_cast<float4 *>(&acc[warp][(lane + i * 32) * 4]) = v[i];
    __syncthreads();
    float *dst = p.out + (size_t)(start + row / p.group) * p.out_stride + (size_t)(kvh * p.group + row % p.group) * D;
    for (int c = tid; c < D; c += TREE_SHARES)
        dst[c] = sum == 0.0f ? 0.0f : __fdiv_rn(acc[0][c] + acc[1][c] + acc[2][c] + acc[3][c], sum);  // 0: a row that sees nothing
}

// How the keys of one set of rows are split.  A CTA's time is its keys and, in their measure, about 400 for starting,
// queries and the join.  `resident[i]`: how many clusters of TREE_SIZES[i] CTAs the GPU holds at once (a cluster lies in one
// GPC: of 148 SMs with one CTA each, 120 serve clusters of 8 and 112 those of 16).  Beyond a cluster's 16 the shares are
// joined by a second kernel through a workspace, worth about 300 more.
constexpr int TREE_SIZES[] = {1, 2, 3, 4, 6, 8, 16};
constexpr int TREE_SIZE_COUNT = 7;
struct TreeSplit {
    unsigned shares;
    bool gather;
};
inline TreeSplit tree_split(size_t have, size_t slots, const int *resident, long long keys, bool may_gather) {
    TreeSplit best = {1, false};
    double least = 1e300;
    for (int i = 0; i < TREE_SIZE_COUNT; ++i) {
        const int s = TREE_SIZES[i];
        if (s > 1 && (keys < (long long)s * 2 * TREE_KEYS || resident[i] < 1)) break;
        const double cost = (double)((have + resident[i] - 1) / resident[i]) * ((double)keys / s + 400.0);
        if (cost < least * 0.98) best = {(unsigned)s, false}, least = cost;
    }
    const long long most = keys / (2 * TREE_KEYS) < TREE_SHARES ? keys / (2 * TREE_KEYS) : TREE_SHARES;
    const long long s = have ? (long long)(slots / have) : 0;  // one full round
    if (may_gather && s > best.shares) {
        const long long g = s < most ? s : most;
        if (g > best.shares && (double)keys / g + 400.0 + 300.0 < least) best = {(unsigned)g, true};
    }
    return best;
}

// What launching asks of the driver once a kernel and device.
struct TreeKernelInfo {
    std::mutex mu;
    std::atomic<uint64_t> known{0};
    int resident[64][TREE_SIZE_COUNT];
};

template <typename K>
int tree_kernel_info(const nne_ctx *ctx, K kernel, TreeKernelInfo &info, int threads, size_t smem, const int **resident) {
    const int dev = ctx->device & 63;
    if (!(info.known.load(std::memory_order_acquire) >> dev & 1)) {
        std::lock_guard<std::mutex> lock(info.mu);
        NNE_TRY(ensure_dynamic_smem(ctx->device, kernel, smem));
        NNE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        for (int i = 0; i < TREE_SIZE_COUNT; ++i) {
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = (unsigned)TREE_SIZES[i];
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)TREE_SIZES[i], 64, 1);
            cfg.blockDim = dim3((unsigned)threads);
            cfg.dynamicSmemBytes = smem;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) {
                cudaGetLastError();
                n = 0;
            }
            info.resident[dev][i] = i == 0 && n < 1 ? 1 : n;
        }
        info.known.fetch_or(1ull << dev, std::memory_order_release);
    }
    *resident = info.resident[dev];
    return NNE_OK;
}

template <typename K>
int launch_tree_kernel(nne_ctx *ctx, K kernel, TreeKernelInfo &info, int threads, size_t smem, int per_sm, int rows_of_cta, int d, const TreeArgs &args,
                       int sequences, int max_rows, long long max_keys, bool may_gather, cudaStream_t s) {
    const size_t blocks = (size_t)args.kv_heads * ((max_rows + rows_of_cta - 1) / rows_of_cta);
    if (blocks > 65535 || sequences > 65535) return fail(NNE_ERR_INVALID_ARGUMENT, "too many heads or sequences for one launch");
    const int *resident;
    NNE_TRY(tree_kernel_info(ctx, kernel, info, threads, smem, &resident));
    // Of the sets of rows, those that have rows at all: what the tokens of the call fill, and half a set a sequence for the
    // rounding (4 trees of up to 33 nodes counted as four of 33: 92 us instead of 79).
    size_t sets = blocks * sequences;
    const size_t filled = (size_t)args.kv_heads * (((size_t)args.tokens * args.group + rows_of_cta - 1) / rows_of_cta + (size_t)sequences / 2);
    if (filled < sets) sets = filled;
    const TreeSplit split = tree_split(sets, (size_t)ctx->sm_count * per_sm, resident, max_keys, may_gather);
    TreeArgs a = args;
    void *work = nullptr;
    if (split.gather) {
        NNE_CUDA_TRY(cudaMallocAsync(&work, blocks * sequences * split.shares * rows_of_cta * (d + 4) * sizeof(float), s));
        a.part = static_cast<float *>(work);
    }
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = split.gather ? 1 : split.shares;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(split.shares, (unsigned)blocks, (unsigned)sequences);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a);
    count_launch();
    if (e == cudaSuccess && split.gather) {
        cfg.gridDim = dim3((unsigned)rows_of_cta, (unsigned)blocks, (unsigned)sequences);
        cfg.blockDim = dim3(TREE_SHARES);
        cfg.dynamicSmemBytes = 0;
        cfg.numAttrs = 1;
        const int shares = (int)split.shares;
        switch (d) {
            case 64: e = cudaLaunchKernelEx(&cfg, tree_gather_kernel<64>, a, rows_of_cta, shares); break;
            case 96: e = cudaLaunchKernelEx(&cfg, tree_gather_kernel<96>, a, rows_of_cta, shares); break;
            case 128: e = cudaLaunchKernelEx(&cfg, tree_gather_kernel<128>, a, rows_of_cta, shares); break;
            default: e = cudaLaunchKernelEx(&cfg, tree_gather_kernel<256>, a, rows_of_cta, shares); break;
        }
        count_launch();
    }
    if (work) cudaFreeAsync(work, s);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NNE_ERR_CUDA, "tree attention launch failed: %s", cudaGetErrorString(e));
    }
    return NNE_OK;
}

template <typename T, int D, int NT>
int launch_decode(nne_ctx *ctx, const TreeArgs &a, int sequences, int max_rows, long long max_keys, cudaStream_t s) {
    using S = DecodeShape<T, D, NT>;
    static TreeKernelInfo info;
    return launch_tree_kernel(ctx, tree_decode_kernel<T, D, NT>, info, S::THREADS, S::SMEM, S::PER_SM, S::ROWS, D, a, sequences, max_rows, max_keys, true, s);
}
template <typename T, int D, int NT, int WN, int WK>
int launch_tree_shape(nne_ctx *ctx, const TreeArgs &a, int sequences, int max_rows, long long max_keys, cudaStream_t s) {
    using S = TreeShape<T, D, NT, WN, WK>;
    static TreeKernelInfo info;
    return launch_tree_kernel(ctx, tree_attention_kernel<T, D, NT, WN, WK>, info, S::THREADS, S::SMEM, S::PER_SM, S::ROWS, D, a, sequences, max_rows,
                              max_keys, false, s);
}

// Shapes by the rows a key/value head meets at most: the fewest idle MMA columns.  O takes D/16 * NT * 4 registers a
// thread, so heads of 256 keep to one 8-row tile a warp.
template <typename T, int D>
int launch_tree_d(nne_ctx *ctx, const TreeArgs &a, int sequences, long long max_keys, cudaStream_t s) {
    const int rows = a.max_nodes * a.group;
    if (rows <= 8) return launch_decode<T, D, 1>(ctx, a, sequences, rows, max_keys, s);
    if constexpr (D <= 128) {
        if (rows <= 16) return launch_decode<T, D, 2>(ctx, a, sequences, rows, max_keys, s);
        // 8 rows a warp: twice the warps to hide each other's latency (8 trees of 8, bf16: 62 -> 58 us); 16 rows a warp: half
        // the shared-memory traffic a product (64 nodes, f16: 92 -> 86 us)
        if (rows <= 32) return launch_tree_shape<T, D, 1, 4, 2>(ctx, a, sequences, rows, max_keys, s);
        return launch_tree_shape<T, D, 2, 2, 2>(ctx, a, sequences, rows, max_keys, s);
    } else {
        if (rows <= 16) return launch_tree_shape<T, D, 1, 2, 2>(ctx, a, sequences, rows, max_keys, s);
        return launch_tree_shape<T, D, 1, 4, 2>(ctx, a, sequences, rows, max_keys, s);
    }
}

template <typename T>
int launch_tree(nne_ctx *ctx, int d, const TreeArgs &a, int sequences, long long max_keys, cudaStream_t s) {
    switch (d) {
        case 64: return launch_tree_d<T, 64>(ctx, a, sequences, max_keys, s);
        case 96: return launch_tree_d<T, 96>(ctx, a, sequences, max_keys, s);
        case 128: return launch_tree_d<T, 128>(ctx, a, sequences, max_keys, s);
        default: return launch_tree_d<T, 256>(ctx, a, sequences, max_keys, s);
    }
}
int launch_tree_f16(nne_ctx *ctx, int d, const TreeArgs &a, int sequences, long long max_keys, cudaStream_t s);
int launch_tree_bf16(nne_ctx *ctx, int d, const TreeArgs &a, int sequences, long long max_keys, cudaStream_t s);

}  // namespace nne
