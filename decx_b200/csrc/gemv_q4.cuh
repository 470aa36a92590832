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
// Exactness and cost.  A nibble q left in the low bits of an fp16 number IS the subnormal q * 2^-24 (16 q * 2^-24 for the
// upper nibble of a byte), and the tensor path multiplies subnormals exactly: one mask per pair of weights is all the
// unpacking there is.  Products of lower and of upper nibbles go to accumulators of their own, and the zero point
// leaves the sum: sum (q - z) x = sum q x - z sum x, with the group sums of x computed once per CTA.  x is fp16 or e4m3,
// which fp16 holds exactly.  All sums are fp32; the group's scale multiplies in fp32; the only other rounding is the
// one to an fp16 result.
//
// Order of K.  A sum does not care, so each lane takes whole words of a row: of a group of 32 / 64 / 128 weights the lane
// that the instruction gives columns 2t, 2t+1, 2t+8, 2t+9 holds words t*w .. t*w+w-1 (w = 1 / 2 / 4, one shared-memory
// load), and x is staged in shared memory in the order that this and the masks produce (0 4 2 6 1 5 3 7 within eight),
// so that one 16-byte load feeds both instructions of a word.
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
    int vec_s, vec_z;          // four neighbouring scales / zero points may be read at once
};

constexpr int Q4_ROWS = 64;          // rows per CTA
constexpr int Q4_THREADS = 256;      // 2 row halves x 4 parts of the slice

__host__ __device__ constexpr uint32_t q4_w_pitch(uint32_t slice) { return slice / 2; }
// fp16 row of x: 64 bytes more than the slice, so that the two rows a quarter-warp reads fall on different banks
__host__ __device__ constexpr uint32_t q4_x_pitch(uint32_t slice) { return slice * 2 + 64; }
// a row's scales (fp32, or fp32 pairs with the zero point), padded against bank conflicts
__host__ __device__ constexpr uint32_t q4_s_pitch(uint32_t groups, bool zeros) { return zeros ? (groups + 2) * 8 : (groups + 4) * 4; }
__host__ __device__ constexpr uint32_t q4_red_bytes(uint32_t n_tiles) { return 4u * Q4_ROWS * (8 * n_tiles + 1) * 4; }
__host__ __device__ constexpr uint32_t q4_smem_bytes(uint32_t slice, uint32_t group, uint32_t n_tiles, uint32_t n_vec,
                                                     bool zeros) {
    const uint32_t w = Q4_ROWS * q4_w_pitch(slice);
    const uint32_t x = n_vec * q4_x_pitch(slice);
    const uint32_t s = Q4_ROWS * q4_s_pitch(slice / group, zeros);
    const uint32_t sums = slice / group * 8 * n_tiles * 4;                    // group sums of x
    const uint32_t red = q4_red_bytes(n_tiles) + Q4_ROWS * 8 * n_tiles * 4;   // reuses the weights' and x's space
    const uint32_t total = w + x + s + sums;
    return total > red ? total : red;
}
// 16-byte unit u of row r lies at unit u ^ q4_swizzle(r): loads of 4, 8 and 16 bytes per lane, eight rows by four
// lanes, then meet no bank twice (bit-reversed row number within eight)
__host__ __device__ constexpr uint32_t q4_swizzle(uint32_t r) { return ((r & 1) << 2) | (r & 2) | ((r >> 2) & 1); }

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
// the first of a chain: d = a * b
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t u) { return *reinterpret_cast<__half2*>(&u); }

// W words (1, 2 or 4) from shared memory
template <int W>
__device__ __forceinline__ void q4_words(uint32_t at, uint32_t (&w)[W]) {
    if constexpr (W == 1) {
        w[0] = ld_shared_u32(at);
    } else if constexpr (W == 2) {
        asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at));
    } else {
        const uint4 v = ld_shared_v4(at);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
}

template <typename OUT>
__device__ __forceinline__ OUT q4_out(float v);
template <> __device__ __forceinline__ float q4_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __half q4_out<__half>(float v) { return __float2half_rn(v); }

// NT: tiles of eight vectors (1 or 2).  X8: x is e4m3.  grid = row blocks x ranks, ranks innermost (a cluster).
template <int GROUP, int NT, bool ZEROS, bool X8, typename OUT>
__global__ void __launch_bounds__(Q4_THREADS)
gemv_q4_kernel(const GemvQ4Params p) {
    extern __shared__ __align__(128) uint8_t q4_smem[];      // the swizzle works on address bits 4 to 6
    constexpr int WPL = GROUP / 32;                           // words a lane holds of a row's group
    constexpr int GU = GROUP / 8;                             // 16-byte units of x in a group
    constexpr int NV = 8 * NT;
    const uint32_t base = smem_u32(q4_smem);
    const uint32_t wp = q4_w_pitch(p.slice), xp = q4_x_pitch(p.slice);
    const uint32_t gps = p.slice / GROUP, gps_log = 31 - __clz(gps), s_pitch = q4_s_pitch(gps, ZEROS);
    const uint32_t x_off = Q4_ROWS * wp, s_off = x_off + p.n_vec * xp, xs_off = s_off + Q4_ROWS * s_pitch;
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
        const uint32_t gn = (kn + GROUP - 1) / GROUP;         // its groups; the last one may be short
        if (sl != rank) __syncthreads();                      // the previous slice has been consumed
        // ---- weights: warp w brings rows 8w .. 8w+7, a lane every 32nd 16-byte unit.  Bytes behind the row's end and
        // rows behind the last one become zeros.
        for (uint32_t u = lane; u < gn * (GROUP / 32); u += 32) {
            const uint32_t byte = k0 / 2 + u * 16;
            const uint32_t n = byte < row_bytes ? min(16u, row_bytes - byte) : 0u;
            const uint8_t* src = p.W + uint64_t(row0 + warp * 8) * p.ldw + byte;
            const uint32_t dst = base + warp * 8 * wp + u * 16;
#pragma unroll
            for (uint32_t r = 0; r < 8; ++r) {
                const bool in = n != 0 && row0 + warp * 8 + r < p.rows;
                cp_async16((dst ^ (q4_swizzle(r) * 16)) + r * wp, in ? src : p.W, in ? n : 0u);
                src += p.ldw;
            }
        }
        // ---- x as fp16 in the order of the products, zeros behind the last column, and the sums of its groups
        for (uint32_t v = 0; v < p.n_vec; ++v) {
            for (uint32_t u = threadIdx.x; u < gps * GU; u += Q4_THREADS) {      // a multiple of 32: whole warps
                const uint32_t k = k0 + u * 8;
                uint32_t e[4];                                // pairs (0,1) (2,3) (4,5) (6,7)
                if constexpr (X8) {
                    const uint8_t* src = static_cast<const uint8_t*>(p.x) + uint64_t(v) * p.ldx + k;
                    uint32_t b[2] = {0u, 0u};
                    if (k + 8 <= p.cols && (reinterpret_cast<uintptr_t>(src) & 7) == 0) {
                        const uint2 d = *reinterpret_cast<const uint2*>(src);
                        b[0] = d.x;
                        b[1] = d.y;
                    } else if (k < p.cols) {
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (k + j < p.cols) b[j >> 2] |= uint32_t(src[j]) << (8 * (j & 3));
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint16_t two = uint16_t(b[j >> 1] >> (16 * (j & 1)));
                        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(e[j]) : "h"(two));
                    }
                } else {
                    const __half* src = static_cast<const __half*>(p.x) + uint64_t(v) * p.ldx + k;
                    if (k + 8 <= p.cols && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {
                        const uint4 d = *reinterpret_cast<const uint4*>(src);
                        e[0] = d.x; e[1] = d.y; e[2] = d.z; e[3] = d.w;
                    } else {
                        __half h[8];
#pragma unroll
                        for (int j = 0; j < 8; ++j) h[j] = k + j < p.cols ? src[j] : __float2half(0.f);
#pragma unroll
                        for (int j = 0; j < 4; ++j) e[j] = h2_bits(__halves2half2(h[2 * j], h[2 * j + 1]));
                    }
                }
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 f = __half22float2(bits_h2(e[j]));
                    sum += f.x + f.y;
                }
#pragma unroll
                for (int m = 1; m < GU; m *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, m);
                const uint32_t gi = u / GU, w = u % GU;       // word w of the group belongs to lane w / WPL
                if (w == 0) *reinterpret_cast<float*>(q4_smem + xs_off + (gi * NV + v) * 4) = sum * 0x1p-24f;
                st_shared_v4(base + x_off + v * xp + (gi * GU + (w % WPL) * 4 + w / WPL) * 16,
                             __byte_perm(e[0], e[2], 0x5410), __byte_perm(e[1], e[3], 0x5410),
                             __byte_perm(e[0], e[2], 0x7632), __byte_perm(e[1], e[3], 0x7632));
            }
        }
        // ---- scales (times 2^24) and zero points (negative), four neighbouring groups at a time
        const uint32_t g0 = k0 / GROUP;
        for (uint32_t i = threadIdx.x; i < Q4_ROWS * gps / 4; i += Q4_THREADS) {
            const uint32_t r = i >> (gps_log - 2), gi = (i & (gps / 4 - 1)) * 4;
            if (gi >= gn || row0 + r >= p.rows) continue;
            const __half* sp = p.scales + uint64_t(row0 + r) * p.lds + g0 + gi;
            float s[4], z[4];
            if (p.vec_s && gi + 4 <= gn) {
                const uint2 d = *reinterpret_cast<const uint2*>(sp);
                const float2 a = __half22float2(bits_h2(d.x)), b = __half22float2(bits_h2(d.y));
                s[0] = a.x; s[1] = a.y; s[2] = b.x; s[3] = b.y;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[j] = gi + j < gn ? __half2float(sp[j]) : 0.f;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) s[j] *= 0x1p24f;
            const uint32_t at = base + s_off + r * s_pitch + gi * (ZEROS ? 8 : 4);
            if constexpr (ZEROS) {
                const uint8_t* zp = p.zeros + uint64_t(row0 + r) * p.ldz + g0 + gi;
                if (p.vec_z && gi + 4 <= gn) {
                    const uint32_t d = *reinterpret_cast<const uint32_t*>(zp);
#pragma unroll
                    for (int j = 0; j < 4; ++j) z[j] = -float((d >> (8 * j)) & 255u);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) z[j] = gi + j < gn ? -float(zp[j]) : 0.f;
                }
                st_shared_v4(at, __float_as_uint(s[0]), __float_as_uint(z[0]), __float_as_uint(s[1]), __float_as_uint(z[1]));
                st_shared_v4(at + 16, __float_as_uint(s[2]), __float_as_uint(z[2]), __float_as_uint(s[3]), __float_as_uint(z[3]));
            } else {
                st_shared_v4(at, __float_as_uint(s[0]), __float_as_uint(s[1]), __float_as_uint(s[2]), __float_as_uint(s[3]));
            }
        }
        cp_async_wait_all();
        __syncthreads();

        // ---- multiply: this warp's 32 rows, its quarter of the slice's groups
        const uint32_t per = (gn + 3) / 4, gi1 = min(gn, (part + 1) * per);
        const uint32_t wrow = base + (half * 32 + g) * wp, sw = q4_swizzle(g) * 16;   // rows 8 apart share a swizzle
        uint32_t xv[NT];                                      // lanes of vectors that do not exist read the last one;
#pragma unroll                                                // their columns are never stored
        for (int n = 0; n < NT; ++n) xv[n] = base + x_off + min(uint32_t(n * 8) + g, p.n_vec - 1) * xp + t * 16;
#pragma unroll 1
        for (uint32_t gi = part * per; gi < gi1; ++gi) {
            uint32_t w[4][WPL];
#pragma unroll
            for (int m = 0; m < 4; ++m) q4_words<WPL>(wrow + m * 8 * wp + ((gi * (GROUP / 2) + t * WPL * 4) ^ sw), w[m]);
            float lo[2][NT][4], hi[2][NT][4];
#pragma unroll
            for (int j = 0; j < WPL; ++j) {
                uint4 xb[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) xb[n] = ld_shared_v4(xv[n] + (gi * GU + j * 4) * 16);
#pragma unroll
                for (int m = 0; m < 2; ++m) {
                    const uint32_t wa = w[2 * m][j], wb = w[2 * m + 1][j], wa8 = wa >> 8, wb8 = wb >> 8;
                    constexpr uint32_t L = 0x000f000fu, H = 0x00f000f0u;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        if (j == 0) {
                            mma_16816_first(lo[m][n], wa & L, wb & L, wa8 & L, wb8 & L, xb[n].x, xb[n].y);
                            mma_16816_first(hi[m][n], wa & H, wb & H, wa8 & H, wb8 & H, xb[n].z, xb[n].w);
                        } else {
                            mma_16816(lo[m][n], wa & L, wb & L, wa8 & L, wb8 & L, xb[n].x, xb[n].y);
                            mma_16816(hi[m][n], wa & H, wb & H, wa8 & H, wb8 & H, xb[n].z, xb[n].w);
                        }
                    }
                }
            }
            float sc[4], nz[4];
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const uint32_t at = base + s_off + (half * 32 + m * 8 + g) * s_pitch + gi * (ZEROS ? 8 : 4);
                if constexpr (ZEROS) {
                    uint32_t v[2];
                    q4_words<2>(at, v);
                    sc[m] = __uint_as_float(v[0]);
                    nz[m] = __uint_as_float(v[1]);
                } else {
                    sc[m] = __uint_as_float(ld_shared_u32(at));
                    nz[m] = -8.f;
                }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t v[2];
                q4_words<2>(base + xs_off + (gi * NV + n * 8 + 2 * t) * 4, v);
                const float xs[2] = {__uint_as_float(v[0]), __uint_as_float(v[1])};
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {             // i >> 1: row g or g + 8; i & 1: vector 2t or 2t + 1
                        float d = fmaf(hi[m][n][i], 0.0625f, lo[m][n][i]);
                        d = fmaf(nz[2 * m + (i >> 1)], xs[i & 1], d);
                        acc[m][n][i] = fmaf(sc[2 * m + (i >> 1)], d, acc[m][n][i]);
                    }
            }
        }
    }

    // ---- join: the four quarters through shared memory, then the slices through distributed shared memory
    __syncthreads();
    constexpr int RP = NV + 1;
    float* red = reinterpret_cast<float*>(q4_smem);                       // [part][row][RP]
    float* sums = red + 4 * Q4_ROWS * RP;                                 // [vector][row]
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t r = half * 32 + m * 16 + g + (i >> 1) * 8, v = n * 8 + 2 * t + (i & 1);
                if (v < p.n_vec) red[(part * Q4_ROWS + r) * RP + v] = acc[m][n][i];
            }
    __syncthreads();
    auto store = [&](uint32_t v, uint32_t r, float s) {
        if (row0 + r < p.rows) {
            if (p.xs != nullptr) s *= __ldg(p.xs + v);
            static_cast<OUT*>(p.y)[uint64_t(v) * p.ldy + row0 + r] = q4_out<OUT>(s);
        }
    };
    for (uint32_t i = threadIdx.x; i < Q4_ROWS * p.n_vec; i += Q4_THREADS) {
        const uint32_t v = i / Q4_ROWS, r = i % Q4_ROWS;
        float s = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) s += red[(q * Q4_ROWS + r) * RP + v];
        if (ranks > 1) sums[i] = s;
        else store(v, r, s);
    }
    if (ranks > 1) {
        namespace cg = cooperative_groups;
        const cg::cluster_group cluster = cg::this_cluster();
        cluster_sync_all();
        for (uint32_t i = rank * Q4_THREADS + threadIdx.x; i < Q4_ROWS * p.n_vec; i += ranks * Q4_THREADS) {
            float d[8];                                                   // requested together, added in slice order
#pragma unroll
            for (uint32_t c = 0; c < 8; ++c) d[c] = c < ranks ? *cluster.map_shared_rank(sums + i, c) : 0.f;
            float s = 0.f;
#pragma unroll
            for (uint32_t c = 0; c < 8; ++c) s += d[c];
            store(i / Q4_ROWS, i % Q4_ROWS, s);
        }
        cluster_sync_all();                                               // nobody leaves while its sums are being read
    }
}

}  // namespace dxb
