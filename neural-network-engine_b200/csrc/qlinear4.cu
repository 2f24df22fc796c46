// Linear layer with 4-bit weights and one f32 scale per group of 32, 64 or 128 consecutive inputs:
//
//   scale[j,g] = max|w_g| > 0 ? max|w_g| / 7 : 1,   q = clamp(round_half_away(w * (1/scale)), -8, 7)
//   y[r,j]     = sum_g scale[j,g] * sum_{i in g} q[j,i] * x[r,i]   (+ bias[j])
//
// the rounding rule of Int8Tensor / QLinear (src/nn/quantized.rs:107-127) with 7 in the place of 127 and a
// scale per group in the place of one per row.
//
// Public layout: codes [n, ceil(k/2)] bytes, two's complement, the even column in the low four bits; scales
// [n, ceil(k/group)].  On the device the layer keeps one private copy, laid out for the forward kernel: tiles of
// 16 rows x 64 columns, 512 bytes each, in which lane l's 16 bytes hold its operand fragments of four
// m16n8k16 MMAs (a code as q + 8, which two integer operations make f16 pairs of), and the
// scales as [tile][group][8][2] (rows r and r + 8 side by side: what one lane needs).  k is padded to 64 and n to
// 16 with zero codes.
#include <cuda_fp16.h>

#include <atomic>
#include <mutex>
#include <new>

#include "common.cuh"
#include "ptx.cuh"

struct nne_qlinear4 {
    nne_ctx *ctx = nullptr;
    int device = 0;
    size_t n = 0, k = 0;
    int group = 0;
    size_t tiles = 0, chunks = 0, groups = 0;  // ceil(n/16), ceil(k/64), ceil(k/group)
    uint4 *words = nullptr;                    // [tiles][chunks][32]
    float2 *scales = nullptr;                  // [tiles][groups of the padded k][8]
    float *bias = nullptr;                     // [n] or null
};

namespace nne {
namespace {

constexpr int Q4_ROWS = 16;        // rows of a tile
constexpr int Q4_CHUNK = 64;       // columns of a tile
constexpr int Q4_PREP = 4;         // activation pieces whose loads a warp has on their way
constexpr int Q4_MAX_SPLIT = 8;    // CTAs of a cluster that share a row block's columns

__host__ __device__ inline size_t padded_groups(size_t chunks, int group) {
    return group >= Q4_CHUNK ? (chunks * Q4_CHUNK + group - 1) / group : chunks * (Q4_CHUNK / group);
}

// ---- quantize ---------------------------------------------------------------------------------------------
// A warp takes 512 columns of a row, four runs of 128 with four consecutive columns a lane; a group is 8, 16 or 32 lanes,
// whose maximum is found by shuffles, so a matrix is read once, 64 bytes a lane on their way.  HBM bound: 4 bytes in and half a
// byte out per weight.
//
// round_half_away(t): |t| + 1/2 and the integer below it, both additions rounding towards zero, which crosses no integer
// (0.49999997 + 0.5 rounded to nearest would be 1).  t is at most 7 but for its rounding, or, under a scale that has underflowed,
// anything: the clamp comes first, to the same effect.
__device__ __forceinline__ uint32_t code4(float v, float inv) {
    float t = __fmul_rn(v, inv);
    t = t == t ? fminf(fmaxf(t, -8.0f), 7.0f) : 0.0f;  // NaN: 0
    const uint32_t magnitude = __float_as_uint(__fadd_rz(__fadd_rz(fabsf(t), 0.5f), 8388608.0f));  // the integer in the low bits
    const uint32_t sign = (uint32_t)((int32_t)__float_as_uint(t) >> 31);
    return ((magnitude ^ sign) - sign) & 15u;
}

template <bool VEC, int GROUP>
__global__ void __launch_bounds__(256)
quantize_rows4_kernel(const float *__restrict__ w, size_t rows, size_t cols, uint8_t *__restrict__ q, float *__restrict__ scales) {
    constexpr int RUNS = 4, WIDE = RUNS * 128;
    constexpr int width = GROUP / 4, per_run = 32 / width;  // lanes of a group, groups of a run
    const int lane = threadIdx.x & 31;
    const size_t segs = (cols + WIDE - 1) / WIDE, bytes = (cols + 1) / 2, groups = (cols + GROUP - 1) / GROUP;
    const size_t step = (size_t)gridDim.x * 8, step_r = step / segs, step_s = step - step_r * segs;
    const size_t first = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    size_t r = first / segs, seg = first - r * segs;
    while (r < rows) {
        float v[RUNS][4];
#pragma unroll
        for (int k = 0; k < RUNS; ++k) {
            const size_t c = seg * WIDE + k * 128 + lane * 4;
            const float *p = w + r * cols + c;
            if (VEC) {  // cols % 4 == 0: a lane's columns are all there or all behind the row
                const float4 f = c < cols ? __ldcs(reinterpret_cast<const float4 *>(p)) : make_float4(0, 0, 0, 0);
                v[k][0] = f.x, v[k][1] = f.y, v[k][2] = f.z, v[k][3] = f.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[k][i] = c + i < cols ? p[i] : 0.0f;
            }
        }
        // The 4 to 16 groups of the warp's columns, a lane each for the two divisions: in every lane they were half of
        // the kernel's instructions.
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < RUNS; ++k) {
            float t = fmaxf(fmaxf(fabsf(v[k][0]), fabsf(v[k][1])), fmaxf(fabsf(v[k][2]), fabsf(v[k][3])));  // NaN is passed over
#pragma unroll
            for (int o = 1; o < width; o <<= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
            t = __shfl_sync(0xffffffffu, t, (lane % per_run) * width);
            if (lane / per_run == k) top = t;
        }
        const float scale_of = top > 0.0f ? __fdiv_rn(top, 7.0f) : 1.0f;
        const float inv_of = __fdiv_rn(1.0f, scale_of);
#pragma unroll
        for (int k = 0; k < RUNS; ++k) {
            const size_t c = seg * WIDE + k * 128 + lane * 4;
            const float scale = __shfl_sync(0xffffffffu, scale_of, k * per_run + lane / width);
            const float inv = __shfl_sync(0xffffffffu, inv_of, k * per_run + lane / width);
            uint32_t word = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) word |= code4(v[k][i], inv) << (4 * i);
            if (c >= cols) continue;  // after the shuffles
            if (lane % width == 0) scales[r * groups + c / GROUP] = scale;
            uint8_t *o = q + r * bytes + c / 2;
            if (VEC) {
                *reinterpret_cast<uint16_t *>(o) = (uint16_t)word;
            } else {
                o[0] = (uint8_t)word;  // codes behind the row are 0
                if (c + 2 < cols) o[1] = (uint8_t)(word >> 8);
            }
        }
        seg += step_s, r += step_r;
        if (seg >= segs) seg -= segs, ++r;
    }
}

// Column (within a 16 x 16 step) and row of a lane's code `i` of a fragment word: bits 4i..4i+3.  The order makes
// (w & 0x000f000f) the pair of A register 0, (w & 0x00f000f0) that of register 1, and the same of w >> 8 those of
// registers 2 and 3.
__host__ __device__ inline void code_place(int lane, int i, int *row, int *col) {
    const int g = lane >> 2, t = lane & 3;
    const int reg = (i & 1) + ((i & 2) ? 2 : 0), high = i >> 2;
    *row = g + ((reg & 1) ? 8 : 0);
    *col = 2 * t + ((reg & 2) ? 8 : 0) + high;
}

// Public layout -> the forward's (one thread a 16-byte lane item), and back (one thread a byte).
__global__ void __launch_bounds__(256)
pack_words_kernel(const uint8_t *__restrict__ q, size_t n, size_t k, size_t chunks, size_t total, uint4 *__restrict__ words) {
    const size_t bytes = (k + 1) / 2;
    for (size_t it = (size_t)blockIdx.x * 256 + threadIdx.x; it < total; it += (size_t)gridDim.x * 256) {
        const int lane = (int)(it & 31);
        const size_t tc = it >> 5, tile = tc / chunks, chunk = tc - tile * chunks;
        uint32_t out[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            out[s] = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                int row, col;
                code_place(lane, i, &row, &col);
                const size_t r = tile * Q4_ROWS + row, c = chunk * Q4_CHUNK + s * 16 + col;
                uint32_t code = 0;
                if (r < n && c < k) code = (q[r * bytes + c / 2] >> (4 * (c & 1))) & 15u;
                out[s] |= (code ^ 8u) << (4 * i);  // two's complement -> q + 8
            }
        }
        words[it] = make_uint4(out[0], out[1], out[2], out[3]);
    }
}
__global__ void __launch_bounds__(256)
pack_scales_kernel(const float *__restrict__ s, size_t n, size_t groups, size_t pgroups, size_t total, float2 *__restrict__ out) {
    for (size_t it = (size_t)blockIdx.x * 256 + threadIdx.x; it < total; it += (size_t)gridDim.x * 256) {
        const size_t g8 = it & 7, tg = it >> 3, tile = tg / pgroups, grp = tg - tile * pgroups;
        const size_t r = tile * Q4_ROWS + g8;
        float2 v = make_float2(0.0f, 0.0f);  // rows and groups behind the matrix add nothing
        if (grp < groups) {
            if (r < n) v.x = s[r * groups + grp];
            if (r + 8 < n) v.y = s[(r + 8) * groups + grp];
        }
        out[it] = v;
    }
}

__device__ __forceinline__ int code_at(const uint4 *words, size_t chunks, size_t r, size_t c) {
    const size_t tile = r / Q4_ROWS, chunk = c / Q4_CHUNK;
    const int row = (int)(r % Q4_ROWS), step = (int)(c % Q4_CHUNK) / 16, col = (int)(c % 16);
    const int reg = (row >= 8 ? 1 : 0) + (col >= 8 ? 2 : 0);
    const int lane = (row & 7) * 4 + (col & 7) / 2, i = reg + 4 * (col & 1);
    const uint32_t w = reinterpret_cast<const uint32_t *>(words)[((tile * chunks + chunk) * 32 + lane) * 4 + step];
    return (int)((w >> (4 * i)) & 15u) - 8;
}
__global__ void __launch_bounds__(256)
unpack_codes_kernel(const uint4 *__restrict__ words, size_t n, size_t k, size_t chunks, uint8_t *__restrict__ q) {
    const size_t bytes = (k + 1) / 2, total = n * bytes;
    for (size_t it = (size_t)blockIdx.x * 256 + threadIdx.x; it < total; it += (size_t)gridDim.x * 256) {
        const size_t r = it / bytes, c = (it - r * bytes) * 2;
        int v = code_at(words, chunks, r, c) & 15;
        if (c + 1 < k) v |= (code_at(words, chunks, r, c + 1) & 15) << 4;
        q[it] = (uint8_t)v;
    }
}
__global__ void __launch_bounds__(256)
unpack_scales_kernel(const float2 *__restrict__ s, size_t n, size_t groups, size_t pgroups, float *__restrict__ out) {
    for (size_t it = (size_t)blockIdx.x * 256 + threadIdx.x; it < n * groups; it += (size_t)gridDim.x * 256) {
        const size_t r = it / groups, grp = it - r * groups;
        const float2 v = s[((r / Q4_ROWS) * pgroups + grp) * 8 + (r & 7)];
        out[it] = (r & 8) ? v.y : v.x;
    }
}
// w = q * scale, one product, like QLinear::to_linear (src/nn/quantized.rs:200-209)
__global__ void __launch_bounds__(256)
dequantize4_kernel(const uint4 *__restrict__ words, const float2 *__restrict__ s, size_t n, size_t k, size_t chunks, int group,
                   size_t pgroups, float *__restrict__ out) {
    for (size_t it = (size_t)blockIdx.x * 256 + threadIdx.x; it < n * k; it += (size_t)gridDim.x * 256) {
        const size_t r = it / k, c = it - r * k;
        const float2 v = s[((r / Q4_ROWS) * pgroups + c / group) * 8 + (r & 7)];
        out[it] = __fmul_rn((float)code_at(words, chunks, r, c), (r & 8) ? v.y : v.x);
    }
}

// ---- forward ----------------------------------------------------------------------------------------------
// The weights are the 16-row side of mma.sync m16n8k16 (f16), the activations the 8-column side, and all a group
// adds up is exact integers:
//  - A code enters as q + 8 in 0..15, its four bits being the low mantissa bits of an f16 number: (q + 8) * 2^-24 (rows
//    0..7 of a tile) or (q + 8) * 2^-20 (rows 8..15), exact subnormals that cost one AND for two codes.  The 8 comes
//    off again through the MMA's initial accumulator, -8 * sum of the group's activations.
//  - An activation is put on the grid 2^-e of its group, v = rint(x * 2^e), max|v| in [2^22, 2^23], and split as
//    v = 4096 h + l, |h|, |l| <= 2048: two f16 integers, the columns 2r and 2r + 1.  (q + 8) h summed over 128 columns
//    stays below 2^22, so the f32 accumulators hold the integer exactly.
//  At a group's end 4096 * (hi sum) + (lo sum) rounds once and joins the row's f32 sum with scale * 2^-e.  The error is
//  that of f32 (x off by 2^-23 of its group's largest); one f16 for x would give 2^-11.
//
// A CTA takes 128 or 256 rows (Q4Shape) and a share of the columns; the CTAs of a cluster take the shares of one
// row block and add their sums up through each other's shared memory in rank order, so results do not change from
// run to run.  Each warp streams its weights through a ring of its own, filled by asynchronous copies up to seven tiles ahead
// that start before the wait for the kernel that makes x (a layer never changes); no other warp is waited for.  (The same
// ring in registers spilled, and a spilled load is a load waited for: 95 us instead of 47 on 8192 -> 28672, group 32.)  Up to four activation rows are put on the
// grid by the CTAs themselves; more are put there once by a kernel before (q4_prepare_kernel): with 12 rows of
// 4091 -> 11003 every CTA preparing its own share took 50 us in all.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two f32 operations in one instruction, each rounded as by itself.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 d;
    asm("{.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 d, a, b;\nmov.b64 {%0, %1}, d;}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{.reg .b64 a, b, c, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmov.b64 c, {%6, %7};\nfma.rn.f32x2 d, a, b, c;\n"
        "mov.b64 {%0, %1}, d;}"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

struct Q4Args {
    const uint4 *words;
    const float2 *scales;
    const float *bias, *x;
    float *y;
    const uint8_t *frag;   // prepared activations [row block][chunk][CHUNK_BYTES], or null: the CTAs prepare theirs
    const float4 *info;    // [row block][group][COLS]
    size_t n, k, m, ldy;
    unsigned tiles, chunks, pgroups;
    unsigned span;    // chunks of a CTA's share
    unsigned stage;   // chunks whose activations are in one shared-memory buffer
    int vec;          // rows of x can be read as float4
};

template <int NT, int TPW>  // TPW: row tiles of a warp
struct Q4Shape {
    static constexpr int COLS = 4 * NT;                  // activation rows of a CTA
    static constexpr int CHUNK_BYTES = 4 * NT * 256;     // fragments of 64 columns
    // The way out of shared memory is the limit (four rows: 58 % of it busy at one tile a warp, with 32 rows 79 %), so the
    // fragments a warp reads serve two tiles: 28672 -> 8192, one row 30 -> 25 us, 12 rows of 4091 -> 11003 22.7 -> 20.8 us, 48 rows of
    // 4096 -> 11008 79 -> 66 us.  One tile where two would leave SMs without a CTA.  5 to 16 rows: CTAs of four warps, whose 128 rows
    // split a layer as finely as eight of one tile (with 256 rows 24.7 us).
    static constexpr int WARPS = NT > 1 && NT < 8 ? 4 : 8;
    static constexpr int PER_SM = NT >= 8 ? 1 : 2;       // CTAs of an SM
    static constexpr int TILES = WARPS * TPW;
    static constexpr int DEPTH = NT == 1 && TPW == 2 ? 4 : 8;  // tile copies on their way: 8 KB a scheduler or more
    static constexpr int STAGE = NT > 1 ? DEPTH : 56;          // chunks whose activations are in shared memory, whole ring rounds
    template <int GROUP>
    __host__ __device__ static constexpr int slot() {  // bytes of a tile in a ring slot: codes, scales
        return Q4_CHUNK * Q4_ROWS / 2 + (GROUP >= Q4_CHUNK ? 1 : Q4_CHUNK / GROUP) * 64;
    }
};

// A piece is 128 columns of one activation row, four a lane: columns blk * 128 + lane * 4 ...
__device__ __forceinline__ void q4_load_piece(const float *row, size_t c, size_t k, int vec, float (&v)[4]) {
    v[0] = v[1] = v[2] = v[3] = 0.0f;
    if (vec) {
        if (c < k) {
            const float4 f = *reinterpret_cast<const float4 *>(row + c);
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c + i < k) v[i] = row[c + i];
    }
}
// The piece on its groups' grids.  `frag`: where the fragments of the lane's chunk start; r: row within the block.
// Fragment words: [step pair][n-tile][lane][step of the pair][2].  `info` (lanes that start a group): the initial
// accumulators -8 * sum of h and of l, and 2^-e for rows 0..7 and 8..15 of a tile, all in units of the MMA's products.
template <int GROUP, int NT>
__device__ __forceinline__ void q4_put_piece(const float (&v)[4], int lane, unsigned r, bool there, uint32_t *frag, float4 *info) {
    float top = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int o = 1; o < GROUP / 4; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    // 2^e by its bits: top * 2^e in [2^22, 2^23); e stays within -105 .. 126, so that 2^e and 2^(20-e) are normal
    int e = 22 + 127 - ((int)(__float_as_uint(top) >> 23) & 255);
    e = e > 126 ? 126 : (e < -105 ? -105 : e);
    const float up = __uint_as_float((uint32_t)(e + 127) << 23);
    float h[4], l[4], hs = 0.0f, ls = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float t = rintf(v[i] * up);
        h[i] = rintf(t * (1.0f / 4096.0f));
        l[i] = fmaf(h[i], -4096.0f, t);
        hs += h[i], ls += l[i];
    }
#pragma unroll
    for (int o = 1; o < GROUP / 4; o <<= 1) {
        hs += __shfl_xor_sync(0xffffffffu, hs, o);
        ls += __shfl_xor_sync(0xffffffffu, ls, o);
    }
    if (!there) return;
    const int kk = (lane & 3) * 4, step = (lane & 15) >> 2;
    const int t = (kk & 7) / 2, word = kk >> 3, g = 2 * (r & 3);
    uint32_t *f = frag + (((step >> 1) * NT + r / 4) * 32 + g * 4 + t) * 4 + (step & 1) * 2 + word;
#pragma unroll
    for (int i = 0; i < 2; ++i) {  // 16 h and 16 l: at most 32768, exact in f16
        const __half2 hh = __floats2half2_rn(h[2 * i] * 16.0f, h[2 * i + 1] * 16.0f);
        const __half2 ll = __floats2half2_rn(l[2 * i] * 16.0f, l[2 * i + 1] * 16.0f);
        f[i * 4] = *reinterpret_cast<const uint32_t *>(&hh);
        f[i * 4 + 16] = *reinterpret_cast<const uint32_t *>(&ll);
    }
    if ((lane * 4) % GROUP == 0)
        *info = make_float4(hs * -0x1p-17f, ls * -0x1p-17f, __uint_as_float((uint32_t)(127 + 20 - e) << 23),
                            __uint_as_float((uint32_t)(127 + 16 - e) << 23));
}

// Groups of 64-column chunk c's column `col`, counted from chunk c0 (a multiple of two).
template <int GROUP>
__device__ __forceinline__ unsigned q4_group(unsigned c, int col) {
    return GROUP >= Q4_CHUNK ? c / (GROUP >= Q4_CHUNK ? GROUP / Q4_CHUNK : 1) : c * (Q4_CHUNK / GROUP) + col / GROUP;
}

// Groups that start in the first c chunks.
template <int GROUP>
__host__ __device__ __forceinline__ unsigned q4_groups(unsigned c) {
    return GROUP >= Q4_CHUNK ? (c + (GROUP >= Q4_CHUNK ? GROUP / Q4_CHUNK : 1) - 1) / (GROUP >= Q4_CHUNK ? GROUP / Q4_CHUNK : 1)
                             : c * (Q4_CHUNK / GROUP);
}

template <int GROUP, int NT>
__global__ void __launch_bounds__(256) q4_prepare_kernel(const Q4Args p, uint8_t *frag, float4 *info) {
    constexpr int COLS = 4 * NT, CHUNK_BYTES = 4 * NT * 256;
    grid_dependency_wait();
    grid_launch_dependents();
    const int lane = threadIdx.x & 31;
    const unsigned blocks = (p.chunks + 1) / 2;
    const size_t total = (size_t)blocks * p.m;
    for (size_t b = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5); b < total; b += (size_t)gridDim.x * 8) {
        const size_t row = b / blocks;
        const unsigned ck = 2 * (unsigned)(b - row * blocks) + (lane >> 4), r = (unsigned)(row % COLS);
        const size_t mb = row / COLS;
        float v[4];
        q4_load_piece(p.x + row * p.k, (size_t)ck * Q4_CHUNK + (lane & 15) * 4, p.k, p.vec, v);
        const bool there = ck < p.chunks;
        q4_put_piece<GROUP, NT>(v, lane, r, there,
                                reinterpret_cast<uint32_t *>(frag + (mb * p.chunks + ck) * CHUNK_BYTES),
                                info + (mb * p.pgroups + q4_group<GROUP>(ck, (lane & 15) * 4)) * COLS + r);
    }
}

template <int GROUP, int NT, int TPW, bool READY>
__global__ void __launch_bounds__(Q4Shape<NT, TPW>::WARPS * 32, Q4Shape<NT, TPW>::PER_SM) q4_forward_kernel(const Q4Args p) {
    using S = Q4Shape<NT, TPW>;
    constexpr int WARPS = S::WARPS, ROWS = S::TILES * Q4_ROWS, D = S::DEPTH;
    constexpr int GPC = GROUP >= Q4_CHUNK ? 1 : Q4_CHUNK / GROUP;   // groups of a chunk
    constexpr int CPG = GROUP >= Q4_CHUNK ? GROUP / Q4_CHUNK : 1;   // chunks of a group
    constexpr int SLOT = S::template slot<GROUP>();
    extern __shared__ __align__(16) uint8_t smem[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const unsigned split = gridDim.x, rank = blockIdx.x;
    const unsigned tile = blockIdx.y * S::TILES + warp * TPW;  // the warp's first
    const size_t row0 = (size_t)blockIdx.z * S::COLS;  // first activation row
    const unsigned cols = (unsigned)(p.m - row0 < (size_t)S::COLS ? p.m - row0 : S::COLS);
    const unsigned c_begin = rank * p.span < p.chunks ? rank * p.span : p.chunks;
    const unsigned c_end = c_begin + p.span < p.chunks ? c_begin + p.span : p.chunks;
    const bool mine = tile < p.tiles;

    // The warp's ring of weight tiles: slot j holds chunk c with (c - c_begin) % D == j, a lane's 16 bytes copied by
    // that lane, and behind the codes the scales of the chunk's groups.  One copy group a chunk, also where a chunk has
    // no copy to make, so that "all but the last D - 2 groups" is always chunk c.
    uint8_t *ring = smem + warp * (D * TPW * SLOT);
    uint8_t *xbuf = smem + S::TILES * D * SLOT;
    const uint32_t ring_at = smem_u32(ring) + lane * 16;
    const uint4 *wp = p.words + ((size_t)(mine ? tile : 0) * p.chunks + c_begin) * 32 + lane;
    const float2 *sp = p.scales + ((size_t)(mine ? tile : 0) * p.pgroups + q4_group<GROUP>(c_begin, 0)) * 8 + lane * 2;
    const size_t w_next = tile + 1 < p.tiles ? (size_t)p.chunks * 32 : 0, s_next = tile + 1 < p.tiles ? (size_t)p.pgroups * 8 : 0;
    // chunk c_begin + at + j: `at` a multiple of D, so that the slot and the offsets are known when compiled
    auto fetch = [&](unsigned at, int j, bool there) {
        if (there) {
#pragma unroll
            for (int u = 0; u < TPW; ++u) {
                // a tile behind the last reads the last's: its sums are not stored
                const size_t w_off = u == 0 ? 0 : w_next, s_off = u == 0 ? 0 : s_next;
                const uint32_t dst = ring_at + ((j % D) * TPW + u) * SLOT;
                cp_async_16(dst, wp + w_off + (size_t)at * 32 + j * 32);
                if (lane < GPC * 4) cp_async_16(dst + 512, sp + s_off + (size_t)(at / CPG * GPC) * 8 + (j / CPG) * GPC * 8);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const unsigned share = c_end - c_begin;
#pragma unroll
    for (int j = 0; j < D - 1; ++j) fetch(0, j, mine && (unsigned)j < share);

    grid_dependency_wait();
    grid_launch_dependents();

    float2 sum[TPW][NT];  // rows r and r + 8
    float part[TPW][NT][4];
#pragma unroll
    for (int u = 0; u < TPW; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t) sum[u][t] = make_float2(0.0f, 0.0f);

    // Prepared activations of the chunks from s0 (counted in the share) on: 16-byte copies into buffer `buf`, part of
    // the copy group that is committed next.
    const unsigned buf_bytes = p.stage * S::CHUNK_BYTES + q4_groups<GROUP>(p.stage) * S::COLS * (unsigned)sizeof(float4);
    auto copy_in = [&](unsigned s0, unsigned buf) {
        const unsigned s1 = s0 + p.stage < share ? s0 + p.stage : share;
        const uint32_t dst = smem_u32(xbuf) + buf * buf_bytes;
        const uint8_t *src = p.frag + (blockIdx.z * (size_t)p.chunks + c_begin + s0) * S::CHUNK_BYTES;
        for (unsigned i = threadIdx.x; i < (s1 - s0) * (S::CHUNK_BYTES / 16); i += WARPS * 32) cp_async_16(dst + i * 16, src + (size_t)i * 16);
        const float4 *isrc = p.info + (blockIdx.z * (size_t)p.pgroups + q4_group<GROUP>(c_begin + s0, 0)) * S::COLS;
        for (unsigned i = threadIdx.x; i < q4_groups<GROUP>(s1 - s0) * S::COLS; i += WARPS * 32)
            cp_async_16(dst + p.stage * S::CHUNK_BYTES + i * 16, isrc + i);
    };

    unsigned buf = 0;
    for (unsigned s0 = 0; s0 < share; s0 += p.stage) {
        const unsigned s1 = s0 + p.stage < share ? s0 + p.stage : share;
        uint8_t *here = xbuf + buf * buf_bytes;
        float4 *info = reinterpret_cast<float4 *>(here + p.stage * S::CHUNK_BYTES);  // [group][COLS]
        if (READY) {
            if (s0 == 0) {
                copy_in(0, 0);
                asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory");
            } else if (!mine) {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            }
            __syncthreads();  // this stage's copies (D chunks old) are there for everybody, the other buffer is free
            if (s1 < share) copy_in(s1, buf ^ 1);
            buf ^= 1;
        } else {
            // Columns of rows that are not there keep whatever the memory held: the sums they lead to are not stored.
            if (s0 != 0) __syncthreads();
            const unsigned pieces = ((s1 - s0 + 1) / 2) * cols;
            for (unsigned b0 = warp; b0 < pieces; b0 += WARPS * Q4_PREP) {
                float v[Q4_PREP][4];
#pragma unroll
                for (int u = 0; u < Q4_PREP; ++u) {
                    const unsigned b = b0 + u * WARPS, ck = c_begin + s0 + 2 * (b / cols) + (lane >> 4);
                    v[u][0] = v[u][1] = v[u][2] = v[u][3] = 0.0f;
                    if (b < pieces && ck < c_begin + s1)
                        q4_load_piece(p.x + (row0 + b % cols) * p.k, (size_t)ck * Q4_CHUNK + (lane & 15) * 4, p.k, p.vec, v[u]);
                }
#pragma unroll
                for (int u = 0; u < Q4_PREP; ++u) {
                    const unsigned b = b0 + u * WARPS, r = b % cols;
                    if (b >= pieces) break;  // the same for the whole warp
                    const unsigned ck = 2 * (b / cols) + (lane >> 4);
                    q4_put_piece<GROUP, NT>(v[u], lane, r, s0 + ck < s1, reinterpret_cast<uint32_t *>(here + ck * S::CHUNK_BYTES),
                                            info + q4_group<GROUP>(ck, (lane & 15) * 4) * S::COLS + r);
                }
            }
            __syncthreads();
        }
        if (!mine) {  // a warp behind the last tile only helps to prepare
            asm volatile("cp.async.commit_group;" ::: "memory");
            continue;
        }

        // Chunk at + j of the share; `end`: the last one of an unfinished group of 128 columns.
        auto chunk = [&](unsigned at, int j, bool more, bool end) {
            asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
            __syncwarp();  // the slot's scales are there for every lane, and the slot before has been read by every lane
            fetch(at, j + D - 1, more);
            const uint8_t *slot = ring + j * TPW * SLOT;
            uint32_t w[TPW][4];
#pragma unroll
            for (int u = 0; u < TPW; ++u) {
                const uint4 w4 = reinterpret_cast<const uint4 *>(slot + u * SLOT)[lane];
                w[u][0] = w4.x, w[u][1] = w4.y, w[u][2] = w4.z, w[u][3] = w4.w;
            }
            const uint4 *fc = reinterpret_cast<const uint4 *>(here + (at - s0) * S::CHUNK_BYTES) + j * (S::CHUNK_BYTES / 16) + lane;
            const float4 *ic = info + (at - s0) / CPG * GPC * S::COLS + (lane & 3);
#pragma unroll
            for (int pair = 0; pair < 2; ++pair) {
                uint32_t a[TPW][2][4];
#pragma unroll
                for (int u = 0; u < TPW; ++u)
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const uint32_t lo = w[u][2 * pair + q], up = lo >> 8;
                        a[u][q][0] = lo & 0x000f000fu, a[u][q][1] = lo & 0x00f000f0u, a[u][q][2] = up & 0x000f000fu, a[u][q][3] = up & 0x00f000f0u;
                    }
                const bool first = pair == 0 ? (CPG == 1 || j % CPG == 0) : GPC == 2;
                const bool last = pair == 0 ? GPC == 2 : (CPG == 1 || j % CPG == CPG - 1 || end);
                const int grp = CPG > 1 ? j / CPG : j * GPC + (GPC == 2 ? pair : 0);
                float2 f2[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    const uint4 b = fc[(pair * NT + t) * 32];
                    if (first) {
                        float2 i0;
                        if (last) {  // what the group's end needs in the same load
                            const float4 i4 = ic[grp * S::COLS + t * 4];
                            i0 = make_float2(i4.x, i4.y), f2[t] = make_float2(i4.z, i4.w);
                        } else {
                            i0 = *reinterpret_cast<const float2 *>(ic + grp * S::COLS + t * 4);
                        }
                        const float2 i8 = mul2(i0, make_float2(16.0f, 16.0f));
#pragma unroll
                        for (int u = 0; u < TPW; ++u) part[u][t][0] = i0.x, part[u][t][1] = i0.y, part[u][t][2] = i8.x, part[u][t][3] = i8.y;
                    }
#pragma unroll
                    for (int u = 0; u < TPW; ++u) mma_f16(part[u][t], a[u][0], b.x, b.y);
#pragma unroll
                    for (int u = 0; u < TPW; ++u) mma_f16(part[u][t], a[u][1], b.z, b.w);
                }
                if (last) {
                    float2 s2[TPW];
#pragma unroll
                    for (int u = 0; u < TPW; ++u)
                        s2[u] = reinterpret_cast<const float2 *>(slot + u * SLOT + 512)[(lane >> 2) + (GPC == 2 ? pair * 8 : 0)];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        if (!first) f2[t] = *(reinterpret_cast<const float2 *>(ic + grp * S::COLS + t * 4) + 1);
#pragma unroll
                        for (int u = 0; u < TPW; ++u) {
                            const float (&d)[4] = part[u][t];
                            sum[u][t] = fma2(mul2(s2[u], f2[t]), make_float2(fmaf(d[0], 4096.0f, d[1]), fmaf(d[2], 4096.0f, d[3])), sum[u][t]);
                        }
                    }
                }
            }
        };
        unsigned at = s0;
        for (; at + 2 * D <= share && at + D <= s1; at += D) {  // rounds whose fetches all exist
#pragma unroll
            for (int j = 0; j < D; ++j) chunk(at, j, true, false);
        }
        for (; at < s1; at += D) {
#pragma unroll
            for (int j = 0; j < D; ++j)
                if (at + j < s1) chunk(at, j, at + j + D - 1 < share, at + j + 1 == share);
        }
    }

    // Sums of the cluster's CTAs: each leaves [ROWS][COLS] in its shared memory, and rank i adds up its share of the
    // rows of all of them, rank after rank.
    float *mysum = reinterpret_cast<float *>(smem);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < TPW; ++u)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            const int r = (warp * TPW + u) * Q4_ROWS + (lane >> 2);
            mysum[r * S::COLS + t * 4 + (lane & 3)] = sum[u][t].x;
            mysum[(r + 8) * S::COLS + t * 4 + (lane & 3)] = sum[u][t].y;
        }
    if (split > 1) {
        cluster_meet();
    } else {
        __syncthreads();
    }
    const size_t out0 = (size_t)blockIdx.y * ROWS;
    const unsigned per = (ROWS + split - 1) / split;  // rows of this rank
    for (unsigned i = threadIdx.x; i < per * cols; i += WARPS * 32) {
        // neighbouring threads take neighbouring rows: y is written in runs along n
        const unsigned r = rank * per + i % per, c = i / per;
        if (r >= ROWS || out0 + r >= p.n) continue;
        float v = 0.0f;
        const uint32_t at = smem_u32(mysum + r * S::COLS + c);
        for (unsigned q = 0; q < split; ++q) {
            float u;
            uint32_t peer;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at), "r"(q));
            asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(u) : "r"(peer) : "memory");
            v += u;
        }
        if (p.bias) v = __fadd_rn(v, p.bias[out0 + r]);
        p.y[(row0 + c) * p.ldy + out0 + r] = v;
    }
    if (split > 1) cluster_part();
}

// Shared memory: the weights' rings and activations of `stage` chunks, once or twice; at the end the sums.
template <int GROUP, int NT, int TPW>
size_t q4_bytes(size_t stage, bool twice) {
    using S = Q4Shape<NT, TPW>;
    const size_t ring = (size_t)S::TILES * S::DEPTH * S::template slot<GROUP>();
    const size_t x = stage * S::CHUNK_BYTES + q4_groups<GROUP>((unsigned)stage) * S::COLS * sizeof(float4);
    const size_t sums = (size_t)S::TILES * Q4_ROWS * S::COLS * sizeof(float), bytes = ring + x * (twice ? 2 : 1);
    return bytes > sums ? bytes : sums;
}

// Clusters of 1 .. Q4_MAX_SPLIT CTAs that the GPU holds at once, asked once a device.
template <int GROUP, int NT, int TPW>
int q4_resident(const nne_ctx *ctx, const int **resident) {
    using S = Q4Shape<NT, TPW>;
    constexpr bool READY = NT > 1;
    static std::atomic<uint64_t> known{0};
    static int table[64][Q4_MAX_SPLIT];
    static std::mutex mu;
    const int dev = ctx->device & 63;
    if (!(known.load(std::memory_order_acquire) >> dev & 1)) {
        std::lock_guard<std::mutex> lock(mu);
        const size_t bytes = q4_bytes<GROUP, NT, TPW>(S::STAGE, READY);
        NNE_TRY(ensure_dynamic_smem(ctx->device, q4_forward_kernel<GROUP, NT, TPW, READY>, bytes));
        for (int c = 1; c <= Q4_MAX_SPLIT; ++c) {
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = (unsigned)c;
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3((unsigned)c, 64, 1);
            cfg.blockDim = dim3(S::WARPS * 32);
            cfg.dynamicSmemBytes = bytes;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, q4_forward_kernel<GROUP, NT, TPW, READY>, &cfg) != cudaSuccess) {
                cudaGetLastError();
                n = 0;
            }
            table[dev][c - 1] = c == 1 && n < 1 ? 1 : n;
        }
        known.fetch_or(1ull << dev, std::memory_order_release);
    }
    *resident = table[dev];
    return NNE_OK;
}

template <int GROUP, int NT, int TPW>
int launch_q4(const nne_qlinear4 *ql, const float *x, size_t m, float *y, size_t ldy, cudaStream_t s) {
    using S = Q4Shape<NT, TPW>;
    constexpr bool READY = NT > 1;
    const nne_ctx *ctx = ql->ctx;
    const size_t blocks_n = (ql->tiles + S::TILES - 1) / S::TILES;
    const size_t blocks_m = (m + S::COLS - 1) / S::COLS;
    // Split the columns over the CTAs of a cluster: a CTA's time is its chunks and, in their measure, about ten for starting,
    // activations and the join, and clusters run in rounds of what the GPU holds (28672 -> 8192, one row, in 320 CTAs: 54
    // us, in 256: 31; 4096 -> 6144 in clusters of 6, of which 45 find a place and not 49: 12.6 us, otherwise 7.4).  A share keeps
    // eight chunks of 64.
    const int *resident;
    NNE_TRY((q4_resident<GROUP, NT, TPW>(ctx, &resident)));
    const size_t have = blocks_n * blocks_m;
    size_t split = 1;
    double least = 1e300;
    for (size_t c = 1; c <= Q4_MAX_SPLIT && (c == 1 || ql->chunks >= c * 8); ++c) {
        if (resident[c - 1] < 1) continue;
        const size_t rounds = (have + resident[c - 1] - 1) / resident[c - 1];
        const double cost = (double)rounds * ((double)ql->chunks / (double)c + 10.0);
        if (cost < least * 0.98) split = c, least = cost;
    }
    // shares in whole pairs of chunks, so that a group of 128 columns never lies in two
    size_t span = (ql->chunks + split - 1) / split;
    span = (span + 1) & ~(size_t)1;
    split = (ql->chunks + span - 1) / span;
    const size_t stage = (size_t)S::STAGE < span ? S::STAGE : span;
    Q4Args a = {};
    a.words = ql->words;
    a.scales = ql->scales;
    a.bias = ql->bias;
    a.x = x;
    a.y = y;
    a.n = ql->n;
    a.k = ql->k;
    a.m = m;
    a.ldy = ldy;
    a.tiles = (unsigned)ql->tiles;
    a.chunks = (unsigned)ql->chunks;
    a.pgroups = (unsigned)padded_groups(ql->chunks, GROUP);
    a.span = (unsigned)span;
    a.stage = (unsigned)stage;
    a.vec = ql->k % 4 == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    const size_t bytes = q4_bytes<GROUP, NT, TPW>(stage, READY && stage < span);
    NNE_TRY(ensure_dynamic_smem(ctx->device, q4_forward_kernel<GROUP, NT, TPW, READY>, bytes));

    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.attrs = attr;
    cfg.stream = s;
    cudaError_t e = cudaSuccess;
    void *work = nullptr;
    if (READY) {
        const size_t fb = blocks_m * ql->chunks * S::CHUNK_BYTES, ib = blocks_m * a.pgroups * S::COLS * sizeof(float4);
        NNE_CUDA_TRY(cudaMallocAsync(&work, fb + ib, s));
        uint8_t *frag = static_cast<uint8_t *>(work);
        float4 *info = reinterpret_cast<float4 *>(frag + fb);
        a.frag = frag;
        a.info = info;
        const size_t pieces = (ql->chunks + 1) / 2 * m, cap = (size_t)ctx->sm_count * 8;
        cfg.gridDim = dim3((unsigned)((pieces + 7) / 8 < cap ? (pieces + 7) / 8 : cap));
        cfg.blockDim = dim3(256);
        cfg.numAttrs = 1;
        e = cudaLaunchKernelEx(&cfg, q4_prepare_kernel<GROUP, NT>, a, frag, info);
        count_launch();
    }
    if (e == cudaSuccess) {
        cfg.gridDim = dim3((unsigned)split, (unsigned)blocks_n, (unsigned)blocks_m);
        cfg.blockDim = dim3(S::WARPS * 32);
        cfg.dynamicSmemBytes = bytes;
        cfg.numAttrs = 2;
        e = cudaLaunchKernelEx(&cfg, q4_forward_kernel<GROUP, NT, TPW, READY>, a);
        count_launch();
    }
    if (work) cudaFreeAsync(work, s);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(NNE_ERR_CUDA, "4-bit forward launch failed: %s", cudaGetErrorString(e));
    }
    return NNE_OK;
}

template <int GROUP>
int launch_q4_group(const nne_qlinear4 *ql, const float *x, size_t m, float *y, size_t ldy, cudaStream_t s) {
    if (m <= 4) {
        // Two tiles a warp where CTAs of 256 rows, split as far as may be, are enough for every SM (4096 -> 4096: 128; 11008 ->
        // 4096 so 10.5 us, with one tile 8.8).
        const size_t most = ql->chunks / 8 < 1 ? 1 : (ql->chunks / 8 < Q4_MAX_SPLIT ? ql->chunks / 8 : Q4_MAX_SPLIT);
        const size_t rows = Q4Shape<1, 2>::TILES * Q4_ROWS;
        if ((ql->n + rows - 1) / rows * most < (size_t)ql->ctx->sm_count) return launch_q4<GROUP, 1, 1>(ql, x, m, y, ldy, s);
        return launch_q4<GROUP, 1, 2>(ql, x, m, y, ldy, s);
    }
    if (m <= 8) return launch_q4<GROUP, 2, 2>(ql, x, m, y, ldy, s);
    if (m <= 12) return launch_q4<GROUP, 3, 2>(ql, x, m, y, ldy, s);
    if (m <= 16) return launch_q4<GROUP, 4, 2>(ql, x, m, y, ldy, s);
    return launch_q4<GROUP, 8, 2>(ql, x, m, y, ldy, s);
}

__global__ void __launch_bounds__(256)
fill_bias_kernel(const float *__restrict__ bias, size_t n, size_t m, size_t ldy, float *__restrict__ y) {
    for (size_t it = (size_t)blockIdx.x * 256 + threadIdx.x; it < n * m; it += (size_t)gridDim.x * 256)
        y[(it / n) * ldy + it % n] = bias ? bias[it % n] : 0.0f;
}

unsigned grid_of(const nne_ctx *ctx, size_t items, size_t per_block) {
    size_t b = (items + per_block - 1) / per_block;
    const size_t cap = (size_t)ctx->sm_count * 8;
    return (unsigned)(b < 1 ? 1 : (b > cap ? cap : b));
}

int launch_quantize4(nne_ctx *ctx, const float *w, size_t rows, size_t cols, int group, uint8_t *q, float *scales, cudaStream_t s) {
    if (rows == 0 || cols == 0) return NNE_OK;
    const unsigned grid = grid_of(ctx, rows * ((cols + 511) / 512), 8);
    const bool vec = cols % 4 == 0 && (reinterpret_cast<uintptr_t>(w) & 15) == 0 && (reinterpret_cast<uintptr_t>(q) & 1) == 0;
    auto kernel = group == 32   ? (vec ? quantize_rows4_kernel<true, 32> : quantize_rows4_kernel<false, 32>)
                  : group == 64 ? (vec ? quantize_rows4_kernel<true, 64> : quantize_rows4_kernel<false, 64>)
                                : (vec ? quantize_rows4_kernel<true, 128> : quantize_rows4_kernel<false, 128>);
    kernel<<<grid, 256, 0, s>>>(w, rows, cols, q, scales);
    NNE_LAUNCH_CHECK();
    return NNE_OK;
}

int check_f32(const float *p) {
    if (reinterpret_cast<uintptr_t>(p) & 3) return fail(NNE_ERR_INVALID_ARGUMENT, "an f32 device pointer is not 4-byte aligned");
    return NNE_OK;
}

int check_group(size_t group) {
    if (group != 32 && group != 64 && group != 128)
        return fail(NNE_ERR_INVALID_ARGUMENT, "group must be 32, 64 or 128 columns, got %zu", group);
    return NNE_OK;
}

// Sizes whose byte counts fit size_t, and tile counts that fit the kernels' 32-bit ones.
int check_sizes(size_t n, size_t k) {
    size_t t;
    if (__builtin_mul_overflow(n, k, &t) || __builtin_mul_overflow(t, sizeof(float), &t))
        return fail(NNE_ERR_INVALID_ARGUMENT, "n*k overflows size_t");
    if (n > ((size_t)1 << 22) || k > ((size_t)1 << 30))
        return fail(NNE_ERR_INVALID_ARGUMENT, "a 4-bit layer holds at most 2^22 rows of 2^30 columns, got %zu x %zu", n, k);
    return NNE_OK;
}

int alloc_layer4(nne_ctx *ctx, size_t n, size_t k, size_t group, bool has_bias, nne_qlinear4 **out) {
    NNE_TRY(check_group(group));
    NNE_TRY(check_sizes(n, k));
    nne_qlinear4 *ql = new (std::nothrow) nne_qlinear4();
    if (!ql) return fail(NNE_ERR_OUT_OF_MEMORY, "host allocation failed");
    ql->ctx = ctx;
    ql->device = ctx->device;
    ql->n = n;
    ql->k = k;
    ql->group = (int)group;
    ql->tiles = (n + Q4_ROWS - 1) / Q4_ROWS;
    ql->chunks = (k + Q4_CHUNK - 1) / Q4_CHUNK;
    ql->groups = (k + group - 1) / group;
    const size_t wb = ql->tiles * ql->chunks * 32 * sizeof(uint4);
    const size_t sb = ql->tiles * padded_groups(ql->chunks, ql->group) * 8 * sizeof(float2);
    cudaError_t e = cudaMalloc(&ql->words, wb ? wb : 16);
    if (e == cudaSuccess) e = cudaMalloc(&ql->scales, sb ? sb : 16);
    if (e == cudaSuccess && has_bias) e = cudaMalloc(&ql->bias, (n ? n : 1) * sizeof(float));
    if (e != cudaSuccess) {
        cudaGetLastError();
        const int st = fail(e == cudaErrorMemoryAllocation ? NNE_ERR_OUT_OF_MEMORY : NNE_ERR_CUDA,
                            "device allocation for a %zu x %zu 4-bit layer failed: %s", n, k, cudaGetErrorString(e));
        nne_qlinear4_destroy(ql);
        return st;
    }
    *out = ql;
    return NNE_OK;
}

// Fills a layer from codes and scales in the public layout (device pointers) and waits for it: the layer is handed
// out complete, since forwards read the weights ahead of the stream's earlier work.
int fill_layer4(nne_qlinear4 *ql, const uint8_t *q, const float *scales, const float *bias, cudaMemcpyKind bias_from, cudaStream_t s) {
    const size_t pg = padded_groups(ql->chunks, ql->group);
    const size_t words = ql->tiles * ql->chunks * 32, pairs = ql->tiles * pg * 8;
    if (words) {
        pack_words_kernel<<<grid_of(ql->ctx, words, 256), 256, 0, s>>>(q, ql->n, ql->k, ql->chunks, words, ql->words);
        NNE_LAUNCH_CHECK();
        pack_scales_kernel<<<grid_of(ql->ctx, pairs, 256), 256, 0, s>>>(scales, ql->n, ql->groups, pg, pairs, ql->scales);
        NNE_LAUNCH_CHECK();
    }
    if (bias && ql->n) NNE_CUDA_TRY(cudaMemcpyAsync(ql->bias, bias, ql->n * sizeof(float), bias_from, s));
    NNE_CUDA_TRY(cudaStreamSynchronize(s));
    return NNE_OK;
}

int forward4(nne_qlinear4 *ql, const float *x, size_t m, size_t k, float *y, size_t ldy, cudaStream_t s) {
    if (!ql || !ql->ctx) return fail(NNE_ERR_INVALID_ARGUMENT, "null layer handle");
    if (k != ql->k) return fail(NNE_ERR_SHAPE_MISMATCH, "shape mismatch: expected [%zu], got [%zu]", ql->k, k);
    if (ldy < ql->n) return fail(NNE_ERR_INVALID_ARGUMENT, "ldy %zu < out_features %zu", ldy, ql->n);
    size_t t;
    if (__builtin_mul_overflow(m, ql->k, &t) || __builtin_mul_overflow(m, ldy, &t) || __builtin_mul_overflow(t, sizeof(float), &t))
        return fail(NNE_ERR_INVALID_ARGUMENT, "m*k or m*ldy overflows size_t");
    if (m > ((size_t)1 << 18)) return fail(NNE_ERR_INVALID_ARGUMENT, "at most 2^18 activation rows a call, got %zu", m);
    if (m == 0 || ql->n == 0) return NNE_OK;
    if (!y || (ql->k && !x)) return fail(NNE_ERR_INVALID_ARGUMENT, "null activation or output pointer");
    if ((reinterpret_cast<uintptr_t>(x) & 3) || (reinterpret_cast<uintptr_t>(y) & 3))
        return fail(NNE_ERR_INVALID_ARGUMENT, "activation or output pointer is not 4-byte aligned");
    NNE_TRY(use_ctx(ql->ctx));
    if (ql->k == 0) {  // an empty contraction
        fill_bias_kernel<<<grid_of(ql->ctx, ql->n * m, 256), 256, 0, s>>>(ql->bias, ql->n, m, ldy, y);
        NNE_LAUNCH_CHECK();
        return NNE_OK;
    }
    switch (ql->group) {
        case 32: return launch_q4_group<32>(ql, x, m, y, ldy, s);
        case 64: return launch_q4_group<64>(ql, x, m, y, ldy, s);
        default: return launch_q4_group<128>(ql, x, m, y, ldy, s);
    }
}

// A stream-ordered device buffer for the length of a creation or download.
struct Scratch {
    void *p = nullptr;
    cudaStream_t s;
    explicit Scratch(cudaStream_t stream) : s(stream) {}
    int get(size_t bytes) {
        NNE_CUDA_TRY(cudaMallocAsync(&p, bytes ? bytes : 16, s));
        return NNE_OK;
    }
    ~Scratch() {
        if (p) cudaFreeAsync(p, s);
    }
};

// Quantizes device weights into `ql`.
int quantize_into4(nne_qlinear4 *ql, const float *w_dev, const float *bias, cudaMemcpyKind bias_from, cudaStream_t s) {
    Scratch q(s), sc(s);
    NNE_TRY(q.get(ql->n * ((ql->k + 1) / 2)));
    NNE_TRY(sc.get(ql->n * ql->groups * sizeof(float)));
    NNE_TRY(launch_quantize4(ql->ctx, w_dev, ql->n, ql->k, ql->group, (uint8_t *)q.p, (float *)sc.p, s));
    return fill_layer4(ql, (const uint8_t *)q.p, (const float *)sc.p, bias, bias_from, s);
}

}  // namespace
}  // namespace nne

using namespace nne;

extern "C" {

int nne_quantize_rows4_dev(nne_ctx *ctx, const float *w_dev, size_t rows, size_t cols, size_t group, uint8_t *q_dev,
                           float *scales_dev, void *stream) {
    NNE_GUARD_BEGIN
    NNE_TRY(use_ctx(ctx));
    NNE_TRY(check_group(group));
    size_t t;
    if (__builtin_mul_overflow(rows, cols, &t) || __builtin_mul_overflow(t, sizeof(float), &t))
        return fail(NNE_ERR_INVALID_ARGUMENT, "rows*cols overflows size_t");
    if (rows == 0 || cols == 0) return NNE_OK;
    if (!w_dev || !q_dev || !scales_dev) return fail(NNE_ERR_INVALID_ARGUMENT, "null device pointer");
    NNE_TRY(check_f32(w_dev));
    NNE_TRY(check_f32(scales_dev));
    return launch_quantize4(ctx, w_dev, rows, cols, (int)group, q_dev, scales_dev, (cudaStream_t)stream);
    NNE_GUARD_END
}

int nne_qlinear4_create_from_f32_dev(nne_ctx *ctx, const float *w_dev, const float *bias_dev_or_null, size_t n, size_t k,
                                     size_t group, void *stream, nne_qlinear4 **out) {
    NNE_GUARD_BEGIN
    if (!out) return fail(NNE_ERR_INVALID_ARGUMENT, "null out pointer");
    *out = nullptr;
    NNE_TRY(use_ctx(ctx));
    if (n && k && !w_dev) return fail(NNE_ERR_INVALID_ARGUMENT, "null weight pointer");
    NNE_TRY(check_f32(w_dev));
    nne_qlinear4 *ql = nullptr;
    NNE_TRY(alloc_layer4(ctx, n, k, group, bias_dev_or_null != nullptr, &ql));
    const int st = quantize_into4(ql, w_dev, bias_dev_or_null, cudaMemcpyDeviceToDevice, (cudaStream_t)stream);
    if (st != NNE_OK) {
        nne_qlinear4_destroy(ql);
        return st;
    }
    *out = ql;
    return NNE_OK;
    NNE_GUARD_END
}

int nne_qlinear4_create_from_f32(nne_ctx *ctx, const float *w_host, const float *bias_host_or_null, size_t n, size_t k,
                                 size_t group, nne_qlinear4 **out) {
    NNE_GUARD_BEGIN
    if (!out) return fail(NNE_ERR_INVALID_ARGUMENT, "null out pointer");
    *out = nullptr;
    NNE_TRY(use_ctx(ctx));
    if (n && k && !w_host) return fail(NNE_ERR_INVALID_ARGUMENT, "null weight pointer");
    nne_qlinear4 *ql = nullptr;
    NNE_TRY(alloc_layer4(ctx, n, k, group, bias_host_or_null != nullptr, &ql));
    int st = NNE_OK;
    {
        std::lock_guard<std::mutex> lock(ctx->mu);
        const size_t bytes = n * k * sizeof(float);
        st = ctx->stage_a.reserve(bytes ? bytes : 4);
        cudaError_t e = cudaSuccess;
        if (st == NNE_OK && bytes) e = cudaMemcpyAsync(ctx->stage_a.ptr, w_host, bytes, cudaMemcpyHostToDevice, ctx->stream);
        if (e != cudaSuccess) st = fail(NNE_ERR_CUDA, "layer upload failed: %s", cudaGetErrorString(e));
        if (st == NNE_OK) st = quantize_into4(ql, (const float *)ctx->stage_a.ptr, bias_host_or_null, cudaMemcpyHostToDevice, ctx->stream);
    }
    if (st != NNE_OK) {
        nne_qlinear4_destroy(ql);
        return st;
    }
    *out = ql;
    return NNE_OK;
    NNE_GUARD_END
}

int nne_qlinear4_create_from_i4_dev(nne_ctx *ctx, const uint8_t *q_dev, const float *scales_dev, const float *bias_dev_or_null,
                                    size_t n, size_t k, size_t group, void *stream, nne_qlinear4 **out) {
    NNE_GUARD_BEGIN
    if (!out) return fail(NNE_ERR_INVALID_ARGUMENT, "null out pointer");
    *out = nullptr;
    NNE_TRY(use_ctx(ctx));
    if (n && k && (!q_dev || !scales_dev)) return fail(NNE_ERR_INVALID_ARGUMENT, "null codes or scales pointer");
    NNE_TRY(check_f32(scales_dev));
    nne_qlinear4 *ql = nullptr;
    NNE_TRY(alloc_layer4(ctx, n, k, group, bias_dev_or_null != nullptr, &ql));
    const int st = fill_layer4(ql, q_dev, scales_dev, bias_dev_or_null, cudaMemcpyDeviceToDevice, (cudaStream_t)stream);
    if (st != NNE_OK) {
        nne_qlinear4_destroy(ql);
        return st;
    }
    *out = ql;
    return NNE_OK;
    NNE_GUARD_END
}

int nne_qlinear4_create_from_i4(nne_ctx *ctx, const uint8_t *q_host, const float *scales_host, const float *bias_host_or_null,
                                size_t n, size_t k, size_t group, nne_qlinear4 **out) {
    NNE_GUARD_BEGIN
    if (!out) return fail(NNE_ERR_INVALID_ARGUMENT, "null out pointer");
    *out = nullptr;
    NNE_TRY(use_ctx(ctx));
    if (n && k && (!q_host || !scales_host)) return fail(NNE_ERR_INVALID_ARGUMENT, "null codes or scales pointer");
    nne_qlinear4 *ql = nullptr;
    NNE_TRY(alloc_layer4(ctx, n, k, group, bias_host_or_null != nullptr, &ql));
    int st = NNE_OK;
    {
        std::lock_guard<std::mutex> lock(ctx->mu);
        cudaStream_t s = ctx->stream;
        const size_t qb = n * ((k + 1) / 2), sb = n * ql->groups * sizeof(float);
        Scratch q(s), sc(s);
        st = q.get(qb);
        if (st == NNE_OK) st = sc.get(sb);
        cudaError_t e = cudaSuccess;
        if (st == NNE_OK && qb) e = cudaMemcpyAsync(q.p, q_host, qb, cudaMemcpyHostToDevice, s);
        if (st == NNE_OK && e == cudaSuccess && sb) e = cudaMemcpyAsync(sc.p, scales_host, sb, cudaMemcpyHostToDevice, s);
        if (st == NNE_OK && e != cudaSuccess) st = fail(NNE_ERR_CUDA, "layer upload failed: %s", cudaGetErrorString(e));
        if (st == NNE_OK) st = fill_layer4(ql, (const uint8_t *)q.p, (const float *)sc.p, bias_host_or_null, cudaMemcpyHostToDevice, s);
    }
    if (st != NNE_OK) {
        nne_qlinear4_destroy(ql);
        return st;
    }
    *out = ql;
    return NNE_OK;
    NNE_GUARD_END
}

int nne_qlinear4_destroy(nne_qlinear4 *ql) {
    NNE_GUARD_BEGIN
    if (!ql) return NNE_OK;
    cudaSetDevice(ql->device);
    if (ql->words) cudaFree(ql->words);
    if (ql->scales) cudaFree(ql->scales);
    if (ql->bias) cudaFree(ql->bias);
    delete ql;
    return NNE_OK;
    NNE_GUARD_END
}

int nne_qlinear4_download(const nne_qlinear4 *ql, uint8_t *q_host, float *scales_host, float *bias_host) {
    NNE_GUARD_BEGIN
    if (!ql || !ql->ctx) return fail(NNE_ERR_INVALID_ARGUMENT, "null layer handle");
    if (ql->n == 0) return NNE_OK;
    NNE_TRY(use_ctx(ql->ctx));
    std::lock_guard<std::mutex> lock(ql->ctx->mu);
    cudaStream_t s = ql->ctx->stream;
    const size_t qb = ql->n * ((ql->k + 1) / 2), sb = ql->n * ql->groups * sizeof(float);
    Scratch q(s), sc(s);
    if (bias_host && ql->bias) NNE_CUDA_TRY(cudaMemcpyAsync(bias_host, ql->bias, ql->n * sizeof(float), cudaMemcpyDeviceToHost, s));
    if (q_host && ql->k) {
        NNE_TRY(q.get(qb));
        unpack_codes_kernel<<<grid_of(ql->ctx, qb, 256), 256, 0, s>>>(ql->words, ql->n, ql->k, ql->chunks, (uint8_t *)q.p);
        NNE_LAUNCH_CHECK();
        NNE_CUDA_TRY(cudaMemcpyAsync(q_host, q.p, qb, cudaMemcpyDeviceToHost, s));
    }
    if (scales_host && ql->k) {
        NNE_TRY(sc.get(sb));
        unpack_scales_kernel<<<grid_of(ql->ctx, ql->n * ql->groups, 256), 256, 0, s>>>(
            ql->scales, ql->n, ql->groups, padded_groups(ql->chunks, ql->group), (float *)sc.p);
        NNE_LAUNCH_CHECK();
        NNE_CUDA_TRY(cudaMemcpyAsync(scales_host, sc.p, sb, cudaMemcpyDeviceToHost, s));
    }
    NNE_CUDA_TRY(cudaStreamSynchronize(s));
    return NNE_OK;
    NNE_GUARD_END
}

int nne_qlinear4_dequantize(const nne_qlinear4 *ql, float *w_host) {
    NNE_GUARD_BEGIN
    if (!ql || !ql->ctx) return fail(NNE_ERR_INVALID_ARGUMENT, "null layer handle");
    if (ql->n == 0 || ql->k == 0) return NNE_OK;
    if (!w_host) return fail(NNE_ERR_INVALID_ARGUMENT, "null host pointer");
    NNE_TRY(use_ctx(ql->ctx));
    std::lock_guard<std::mutex> lock(ql->ctx->mu);
    cudaStream_t s = ql->ctx->stream;
    Scratch w(s);
    const size_t bytes = ql->n * ql->k * sizeof(float);
    NNE_TRY(w.get(bytes));
    dequantize4_kernel<<<grid_of(ql->ctx, ql->n * ql->k, 256), 256, 0, s>>>(ql->words, ql->scales, ql->n, ql->k, ql->chunks, ql->group,
                                                                          padded_groups(ql->chunks, ql->group), (float *)w.p);
    NNE_LAUNCH_CHECK();
    NNE_CUDA_TRY(cudaMemcpyAsync(w_host, w.p, bytes, cudaMemcpyDeviceToHost, s));
    NNE_CUDA_TRY(cudaStreamSynchronize(s));
    return NNE_OK;
    NNE_GUARD_END
}

int nne_qlinear4_info(const nne_qlinear4 *ql, size_t *n, size_t *k, size_t *group, int *has_bias) {
    if (!ql || !ql->ctx) return fail(NNE_ERR_INVALID_ARGUMENT, "null layer handle");
    if (n) *n = ql->n;
    if (k) *k = ql->k;
    if (group) *group = (size_t)ql->group;
    if (has_bias) *has_bias = ql->bias != nullptr;
    return NNE_OK;
}

size_t nne_qlinear4_memory_bytes(const nne_qlinear4 *ql) {
    if (!ql) return 0;
    return ql->tiles * ql->chunks * 32 * sizeof(uint4) + ql->tiles * padded_groups(ql->chunks, ql->group) * 8 * sizeof(float2) +
           (ql->bias ? ql->n * sizeof(float) : 0);
}

int nne_qlinear4_forward_dev(nne_qlinear4 *ql, const float *x_dev, size_t m, size_t k, float *y_dev, void *stream) {
    NNE_GUARD_BEGIN
    return forward4(ql, x_dev, m, k, y_dev, ql ? ql->n : 0, (cudaStream_t)stream);
    NNE_GUARD_END
}

int nne_qlinear4_forward_dev_strided(nne_qlinear4 *ql, const float *x_dev, size_t m, size_t k, float *y_dev, size_t ldy, void *stream) {
    NNE_GUARD_BEGIN
    return forward4(ql, x_dev, m, k, y_dev, ldy, (cudaStream_t)stream);
    NNE_GUARD_END
}

int nne_qlinear4_forward_host(nne_qlinear4 *ql, const float *x_host, size_t m, size_t k, float *y_host) {
    NNE_GUARD_BEGIN
    if (!ql || !ql->ctx) return fail(NNE_ERR_INVALID_ARGUMENT, "null layer handle");
    if (k != ql->k) return fail(NNE_ERR_SHAPE_MISMATCH, "shape mismatch: expected [%zu], got [%zu]", ql->k, k);
    size_t xb, yb;
    if (__builtin_mul_overflow(m, ql->k, &xb) || __builtin_mul_overflow(xb, sizeof(float), &xb) ||
        __builtin_mul_overflow(m, ql->n, &yb) || __builtin_mul_overflow(yb, sizeof(float), &yb))
        return fail(NNE_ERR_INVALID_ARGUMENT, "m*k or m*n overflows size_t");
    if (m == 0 || ql->n == 0) return NNE_OK;
    if ((xb && !x_host) || !y_host) return fail(NNE_ERR_INVALID_ARGUMENT, "null host pointer");
    nne_ctx *ctx = ql->ctx;
    NNE_TRY(use_ctx(ctx));
    std::lock_guard<std::mutex> lock(ctx->mu);
    NNE_TRY(ctx->stage_a.reserve(xb ? xb : 4));
    NNE_TRY(ctx->stage_b.reserve(yb));
    if (xb) NNE_CUDA_TRY(cudaMemcpyAsync(ctx->stage_a.ptr, x_host, xb, cudaMemcpyHostToDevice, ctx->stream));
    NNE_TRY(forward4(ql, (const float *)ctx->stage_a.ptr, m, k, (float *)ctx->stage_b.ptr, ql->n, ctx->stream));
    NNE_CUDA_TRY(cudaMemcpyAsync(y_host, ctx->stage_b.ptr, yb, cudaMemcpyDeviceToHost, ctx->stream));
    NNE_CUDA_TRY(cudaStreamSynchronize(ctx->stream));
    return NNE_OK;
    NNE_GUARD_END
}

}  // extern "C"
