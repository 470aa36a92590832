// Matrix-vector products with 4-bit weights: y[v][r] = xs[v] * sum_g s[r][g] * sum_{k in g} (q[r][k] - z[r][g]) * x[v][k]
// for 1 to 16 vectors at once.
//
// The weights are read once and set the pace (HBM), so the kernel is built around having enough of them in flight:
//   * A CTA owns 64 rows and a slice of K (512, 1024 or 2048 weights of each row, 16 to 64 KB).  It asks for the whole
//     slice at once with 16-byte asynchronous copies into shared memory, stages x and the scales while they fly, and
//     several CTAs share an SM, so that one computes while others wait.  No ring, no waits that could expire.
//   * The CTAs of a row block's slices form a cluster and add their partial sums through distributed shared memory, in
//     slice order: one launch, no workspace, no atomics, the same result every time.
//   * The products run on the warp-level tensor path, m16n8k16 with fp32 accumulators: 16 rows times up to 8 vectors
//     per instruction, for the price of one vector.  tcgen05 would need the unpacked weights in shared memory, which
//     costs more than the arithmetic.
// Exactness.  A nibble q is put into the mantissa of an fp16 number (1024 + q, or 1024 + 16 q for the upper one of a
// byte), from which one fp16 subtraction or fused multiply-add leaves exactly q - z.  x is fp16 or e4m3, which fp16
// holds exactly.  Sums over a group are fp32, multiplied by the fp32 form of the group's scale and added in fp32;
// the only other rounding is the one to an fp16 result.
//
// Order of K inside an instruction.  The lane that the instruction gives columns 2t, 2t+1, 2t+8, 2t+9 holds one 32-bit
// word, weights 8t .. 8t+7 of a 32-weight step, and the unpacking yields pairs (0,4), (1,5), (2,6), (3,7).  Since a sum
// does not care, x is staged in shared memory with each group of eight in that order and one 16-byte load of it
// feeds both instructions of the step.
#pragma once
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "sm100_ptx.cuh"

namespace dxb {

struct GemvQ4Params {
    const uint8_t* W;          // rows x ceil(cols / 2) bytes, ldw bytes apart (16-byte aligned)
    const __half* scales;      // rows x groups
    const uint8_t* zeros;      // rows x groups, or nullptr: 8 everywhere
    const void* x;             // n_vec x cols, fp16 or e4m3
    const float* xs;           // n_vec, or nullptr: 1
    void* y;                   // n_vec x rows
    uint64_t ldw, lds, ldz, ldx, ldy;
    uint32_t rows, cols, n_vec;
    uint32_t slice;            // weights of a row per CTA and round: 512, 1024 or 2048
    uint32_t n_slices;
    uint32_t ranks;            // CTAs of a row block = cluster size, at most 8
};

constexpr int Q4_ROWS = 64;          // rows per CTA
constexpr int Q4_THREADS = 256;      // 2 row halves x 4 parts of the slice

__host__ __device__ constexpr uint32_t q4_w_pitch(uint32_t slice) { return slice / 2; }
// fp16 row of x: 64 bytes more than the slice, so that the two rows a quarter-warp reads fall on different banks
__host__ __device__ constexpr uint32_t q4_x_pitch(uint32_t slice) { return slice * 2 + 64; }
__host__ __device__ constexpr uint32_t q4_red_bytes(uint32_t n_tiles) { return 4u * Q4_ROWS * (8 * n_tiles + 1) * 4; }
__host__ __device__ constexpr uint32_t q4_smem_bytes(uint32_t slice, uint32_t group, uint32_t n_tiles, uint32_t n_vec,
                                                     bool zeros) {
    const uint32_t w = Q4_ROWS * q4_w_pitch(slice);
    const uint32_t x = n_vec * q4_x_pitch(slice);
    const uint32_t s = Q4_ROWS * (slice / group + 1) * (zeros ? 8 : 4);
    const uint32_t red = q4_red_bytes(n_tiles) + Q4_ROWS * 8 * n_tiles * 4;   // reuses the weights' and x's space
    const uint32_t total = w + x + s;
    return total > red ? total : red;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ uint32_t ld_shared_u32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// a word of eight nibbles -> q - z as half2 pairs (0,4) (1,5) (2,6) (3,7); zl = 1024 + z twice, zh = 64 + z twice
__device__ __forceinline__ void q4_unpack(uint32_t w, __half2 zl, __half2 zh, uint32_t (&o)[4]) {
    const __half2 sixteenth = __float2half2_rn(0.0625f);
    const uint32_t magic = 0x64006400u;
    const uint32_t w8 = w >> 8;
    o[0] = h2_bits(__hsub2(bits_h2((w & 0x000f000fu) | magic), zl));
    o[1] = h2_bits(__hfma2(bits_h2((w & 0x00f000f0u) | magic), sixteenth, __hneg2(zh)));
    o[2] = h2_bits(__hsub2(bits_h2((w8 & 0x000f000fu) | magic), zl));
    o[3] = h2_bits(__hfma2(bits_h2((w8 & 0x00f000f0u) | magic), sixteenth, __hneg2(zh)));
}

template <typename OUT>
__device__ __forceinline__ OUT q4_out(float v);
template <> __device__ __forceinline__ float q4_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __half q4_out<__half>(float v) { return __float2half_rn(v); }

// NT: tiles of eight vectors (1 or 2).  X8: x is e4m3.  grid = row blocks x ranks, ranks innermost (a cluster).
template <int GROUP, int NT, bool ZEROS, bool X8, typename OUT>
__global__ void __launch_bounds__(Q4_THREADS)
gemv_q4_kernel(const GemvQ4Params p) {
    extern __shared__ __align__(16) uint8_t q4_smem[];
    const uint32_t base = smem_u32(q4_smem);
    const uint32_t wp = q4_w_pitch(p.slice), xp = q4_x_pitch(p.slice);
    const uint32_t x_off = Q4_ROWS * wp, s_off = x_off + p.n_vec * xp;
    constexpr uint32_t S_BYTES = ZEROS ? 8 : 4;               // fp32 scale, and 1024 + z twice in fp16
    const uint32_t gps = p.slice / GROUP, s_pitch = (gps + 1) * S_BYTES;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t half = warp & 1, part = warp >> 1;         // rows [32 half, +32), quarter `part` of the slice
    const uint32_t ranks = p.ranks, rank = blockIdx.x % ranks;
    const uint32_t row0 = blockIdx.x / ranks * Q4_ROWS;
    const uint32_t row_bytes = (p.cols + 1) / 2;

    float acc[2][NT][4];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.f;

    for (uint32_t sl = rank; sl < p.n_slices; sl += ranks) {
        const uint32_t k0 = sl * p.slice;
        const uint32_t kn = min(p.slice, p.cols - k0);        // weights of a row in this slice
        const uint32_t steps = (kn + 31) / 32;                // 32-weight steps
        if (sl != rank) __syncthreads();                      // the previous slice has been consumed
        // ---- weights: 16-byte units, swizzled within groups of eight so that eight rows' words fall on all banks
        const uint32_t units = steps;                         // 16 bytes = 32 weights
        for (uint32_t i = threadIdx.x; i < Q4_ROWS * units; i += Q4_THREADS) {
            const uint32_t r = i / units, u = i - r * units;
            const uint32_t byte = k0 / 2 + u * 16;
            const bool in = row0 + r < p.rows;
            const uint32_t n = in ? min(16u, row_bytes - byte) : 0u;
            const uint8_t* src = p.W + (in ? uint64_t(row0 + r) * p.ldw + byte : 0);
            cp_async16(base + r * wp + ((u & ~7u) | ((u ^ r) & 7u)) * 16, src, n);
        }
        // ---- x as fp16, each group of eight in the order 0 4 1 5 2 6 3 7, zeros behind the last column
        const uint32_t xunits = steps * 4;
        for (uint32_t i = threadIdx.x; i < p.n_vec * xunits; i += Q4_THREADS) {
            const uint32_t v = i / xunits, u = i - v * xunits, k = k0 + u * 8;
            __half e[8];
            if constexpr (X8) {
                const uint8_t* src = static_cast<const uint8_t*>(p.x) + uint64_t(v) * p.ldx;
                uint32_t b[2] = {0u, 0u};
                if (k + 8 <= p.cols && ((reinterpret_cast<uintptr_t>(src + k)) & 7) == 0) {
                    const uint2 d = *reinterpret_cast<const uint2*>(src + k);
                    b[0] = d.x;
                    b[1] = d.y;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (k + j < p.cols) b[j >> 2] |= uint32_t(src[k + j]) << (8 * (j & 3));
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t h;
                    const uint16_t two = uint16_t(b[j >> 1] >> (16 * (j & 1)));
                    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(two));
                    const __half2 hh = bits_h2(h);
                    e[2 * j] = __low2half(hh);
                    e[2 * j + 1] = __high2half(hh);
                }
            } else {
                const __half* src = static_cast<const __half*>(p.x) + uint64_t(v) * p.ldx;
                if (k + 8 <= p.cols && ((reinterpret_cast<uintptr_t>(src + k)) & 15) == 0) {
                    const uint4 d = *reinterpret_cast<const uint4*>(src + k);
                    *reinterpret_cast<uint4*>(e) = d;
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) e[j] = k + j < p.cols ? src[k + j] : __float2half(0.f);
                }
            }
            st_shared_v4(base + x_off + v * xp + u * 16, h2_bits(__halves2half2(e[0], e[4])),
                         h2_bits(__halves2half2(e[1], e[5])), h2_bits(__halves2half2(e[2], e[6])),
                         h2_bits(__halves2half2(e[3], e[7])));
        }
        // ---- scales (and zero points) of the slice
        const uint32_t g0 = k0 / GROUP, gn = (kn + GROUP - 1) / GROUP;
        for (uint32_t i = threadIdx.x; i < Q4_ROWS * gn; i += Q4_THREADS) {
            const uint32_t r = i / gn, gi = i - r * gn;
            const bool in = row0 + r < p.rows;
            const float s = in ? __half2float(p.scales[uint64_t(row0 + r) * p.lds + g0 + gi]) : 0.f;
            uint8_t* at = q4_smem + s_off + r * s_pitch + gi * S_BYTES;
            if constexpr (ZEROS) {
                const uint32_t z = in ? p.zeros[uint64_t(row0 + r) * p.ldz + g0 + gi] : 0u;
                const __half2 zl = __half2half2(__uint2half_rn(1024u + z));
                *reinterpret_cast<uint2*>(at) = make_uint2(__float_as_uint(s), h2_bits(zl));
            } else {
                *reinterpret_cast<float*>(at) = s;
            }
        }
        cp_async_wait_all();
        __syncthreads();

        // ---- multiply: this warp's 32 rows, its quarter of the slice in whole groups
        const uint32_t per = ((gn + 3) / 4) * (GROUP / 32);   // steps of a quarter
        const uint32_t st0 = part * per, st1 = min(steps, st0 + per);
        const uint32_t wrow = base + (half * 32 + g) * wp;    // row g of the first tile; +8, +16, +24 rows follow
        const uint32_t xrow = base + x_off;
        for (uint32_t st = st0; st < st1; st += GROUP / 32) {
            float gacc[2][NT][4];
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) gacc[m][n][i] = 0.f;
            const uint32_t gi = st / (GROUP / 32);
            float sc[4];
            __half2 zl[4], zh[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const uint32_t at = base + s_off + (half * 32 + m * 8 + g) * s_pitch + gi * S_BYTES;
                if constexpr (ZEROS) {
                    uint32_t a, b;
                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(a), "=r"(b) : "r"(at));
                    sc[m] = __uint_as_float(a);
                    zl[m] = bits_h2(b);
                    zh[m] = __hsub2(zl[m], __float2half2_rn(960.f));
                } else {
                    sc[m] = __uint_as_float(ld_shared_u32(at));
                    zl[m] = __float2half2_rn(1032.f);
                    zh[m] = __float2half2_rn(72.f);
                }
            }
#pragma unroll
            for (int j = 0; j < GROUP / 32; ++j) {
                const uint32_t u = st + j;
                if (GROUP > 32 && u >= st1) break;            // the last group of the row is short
                uint4 xb[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    // lanes of vectors that do not exist read the last one; their columns are never stored
                    const uint32_t v = min(uint32_t(n * 8) + g, p.n_vec - 1);
                    xb[n] = ld_shared_v4(xrow + v * xp + (u * 4 + t) * 16);
                }
                uint32_t a[4][4];
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    // rows m * 8 + g: all have the same row & 7 = g, hence the same swizzle
                    const uint32_t w = ld_shared_u32(wrow + m * 8 * wp + ((u & ~7u) | ((u ^ g) & 7u)) * 16 + t * 4);
                    q4_unpack(w, zl[m], zh[m], a[m]);
                }
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        mma_16816(gacc[m][n], a[2 * m][0], a[2 * m + 1][0], a[2 * m][1], a[2 * m + 1][1], xb[n].x, xb[n].y);
                        mma_16816(gacc[m][n], a[2 * m][2], a[2 * m + 1][2], a[2 * m][3], a[2 * m + 1][3], xb[n].z, xb[n].w);
                    }
            }
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    acc[m][n][0] = fmaf(sc[2 * m], gacc[m][n][0], acc[m][n][0]);
                    acc[m][n][1] = fmaf(sc[2 * m], gacc[m][n][1], acc[m][n][1]);
                    acc[m][n][2] = fmaf(sc[2 * m + 1], gacc[m][n][2], acc[m][n][2]);
                    acc[m][n][3] = fmaf(sc[2 * m + 1], gacc[m][n][3], acc[m][n][3]);
                }
        }
    }

    // ---- join: the four quarters through shared memory, then the slices through distributed shared memory
    __syncthreads();
    constexpr int NV = 8 * NT, RP = NV + 1;
    float* red = reinterpret_cast<float*>(q4_smem);                       // [part][row][RP]
    float* sums = red + 4 * Q4_ROWS * RP;                                 // [vector][row]
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t r = half * 32 + m * 16 + g + (i >> 1) * 8, v = n * 8 + 2 * t + (i & 1);
                red[(part * Q4_ROWS + r) * RP + v] = acc[m][n][i];
            }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < Q4_ROWS * p.n_vec; i += Q4_THREADS) {
        const uint32_t v = i / Q4_ROWS, r = i % Q4_ROWS;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) s += red[(q * Q4_ROWS + r) * RP + v];
        sums[i] = s;
    }
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    if (ranks > 1) cluster.sync(); else __syncthreads();
    for (uint32_t i = rank * Q4_THREADS + threadIdx.x; i < Q4_ROWS * p.n_vec; i += ranks * Q4_THREADS) {
        const uint32_t v = i / Q4_ROWS, r = i % Q4_ROWS;
        float s = 0.f;
        if (ranks > 1)
            for (uint32_t c = 0; c < ranks; ++c) s += *cluster.map_shared_rank(sums + i, c);
        else
            s = sums[i];
        if (row0 + r < p.rows) {
            if (p.xs != nullptr) s *= p.xs[v];
            static_cast<OUT*>(p.y)[uint64_t(v) * p.ldy + row0 + r] = q4_out<OUT>(s);
        }
    }
    if (ranks > 1) cluster.sync();                            // nobody leaves while its sums are being read
}

}  // namespace dxb
