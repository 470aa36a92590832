// Matrix-vector products with 4-bit weights: y[v][r] = xs[v] * sum_g s[r][g] * sum_{k in g} (q[r][k] - z[r][g]) * x[v][k]
// for 1 to 16 vectors at once.
//
// The weights are read once and set the pace (HBM).  The kernel gives every warp a piece of K that never changes, 256
// columns (128 for more than eight vectors), and lets it walk down the rows:
//   * its part of x sits in registers for the whole launch, already in the order the products want;
//   * weights stream through a ring of 16-row tiles in shared memory that belongs to the warp alone, filled by 16-byte
//     asynchronous copies: no barrier between copying and multiplying, and no wait that could expire;
//   * the warps of a CTA (up to 16) cover neighbouring pieces of K and, every 32 or 64 rows, add their partial sums
//     through shared memory; the CTAs of a cluster (2 to 16, when K needs more than one) do so through distributed shared
//     memory, several blocks at a time and one round later, so that nobody waits for the slowest.  Fixed order, no atomics,
//     one launch, no workspace.
// The products run on the warp-level tensor path, m16n8k16 with fp32 accumulators: 16 rows times up to 8 vectors per
// instruction, for the price of one vector.  tcgen05 would need unpacked weights in shared memory, which costs more than
// the arithmetic.
//
// Exactness and cost.  A nibble q left in the low bits of an fp16 number IS the subnormal q * 2^-24 (16 q * 2^-24 for the
// upper nibble of a byte), and the tensor path multiplies subnormals exactly: a mask, or the difference of two such numbers
// (exact as well, and not on the integer pipe, which is what limits the unpacking), is all there is per pair of weights.
// Products of lower and of upper nibbles go to accumulators of their own, and the zero point leaves the sum:
// sum (q - z) x = sum q x - z sum x, with the group sums of x computed once.  (With an e4m3 x the 16 of the upper nibbles
// is taken from x instead, exactly, and one accumulator does.)  x is fp16 or e4m3, which fp16 holds exactly.  All sums
// are fp32; the group's scale multiplies in fp32; 2^24 comes back at the end; the only other rounding is the one to an
// fp16 result.
//
// Order of K.  A sum does not care, so each lane takes whole words of a row: of a group of 32 / 64 / 128 weights the lane
// that the instruction gives columns 2t, 2t+1, 2t+8, 2t+9 holds words t*w .. t*w+w-1 (w = 1 / 2 / 4, one shared-memory
// load), and its registers hold the matching x as 0 4 2 6 1 5 3 7 within eight.
//
// A weight that is its group's zero point therefore adds no exact zero, but the rounding of two sums that cancel.
//
// Measured (16384 x 16384, fp16 x and y, share of a copy's 6456 GB/s): one vector 31.6 us with groups of 128, 68 %, and 48.9
// with groups of 32 and zero points, 50 %; eight vectors 36.3 us, 59 %.  What bounds it is the length of a warp's chains (word,
// mask, product, scale) with four warps per scheduler, all that the registers of x leave room for: 222 instructions for a tile
// of 16 x 256 with groups of 128 are issued at 2.0 of 4 per clock, 461 with groups of 32 and zero points (a scale, a zero point
// and a sum of x per group and row) at 2.7; the tensor path is busy for 30 and 19 %, DRAM for 47 and 37.  Clusters of four CTAs
// leave 20 of the 148 SMs without one.  Nine to sixteen vectors halve a warp's columns, for the registers of x, and so double
// the partial sums: 4096 x 4096 7.8 us for 16 against 4.9 for 8.  Small products wait for latencies: 1024 x 1024 2.2 us.
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
    uint32_t ranks;            // CTAs that share a block of rows = cluster size, at most 16
    uint32_t tiles;            // tiles of a cluster: its share of the rows
    int vec_s, vec_z, vec_x;   // a tile's scales / zero points of one row, eight entries of x may be read at once
};

template <int NT>
struct Q4Cfg {
    static constexpr int KW = NT == 1 ? 256 : 128;            // columns of a warp
    static constexpr int UNITS = KW / 32;                     // 16-byte units of a row of a tile
    static constexpr int SUB = NT;                            // 16-row parts of a tile
    static constexpr int TR = 16 * SUB;                       // rows of a tile
    static constexpr uint32_t TILE = TR * UNITS * 16;         // bytes: 2 KB
    static constexpr int STAGES = 4;
    static constexpr int BLOCK = NT == 1 ? 4 : 1;             // tiles between two joins of the CTA's warps
    static constexpr int R = TR * BLOCK;
    static constexpr int RS = R + 4;                          // floats between vectors: no bank twice
    static constexpr int WARPS = 16;                          // most per CTA
    static constexpr uint32_t JOIN = 2048;                    // sums a CTA collects before its cluster joins them
    static constexpr uint32_t PART = 8 * NT * RS * 4;         // bytes of one warp's partial sums
    static constexpr uint32_t smem(uint32_t warps) { return warps * (STAGES * TILE + 2 * PART) + 2 * JOIN * 4; }
    static_assert(8 * NT * R <= JOIN, "at least one block");
};
static_assert(Q4Cfg<1>::smem(16) <= 227 * 1024 && Q4Cfg<2>::smem(16) <= 227 * 1024, "one CTA's shared memory");

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
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
__device__ __forceinline__ float half_bits(uint32_t u) { return __half2float(__ushort_as_half(uint16_t(u))); }

// A word of eight nibbles as fp16 subnormals: q * 2^-24 of weights (0,4) and (2,6), 16 q * 2^-24 of (1,5) and (3,7).
__device__ __forceinline__ void q4_pairs(uint32_t w, uint32_t (&o)[4]) {
    const uint32_t odd = __byte_perm(w, 0, 0x4341);           // bytes 1 and 3: lower nibble + 16 * upper nibble
    o[0] = w & 0x000f000fu;
    o[1] = w & 0x00f000f0u;
    o[2] = odd & 0x000f000fu;
    o[3] = h2_bits(__hsub2(bits_h2(odd), bits_h2(o[2])));
}

// W words (1, 2 or 4) from shared memory
template <int W>
__device__ __forceinline__ void q4_words(const uint8_t* at, uint32_t (&w)[W]) {
    if constexpr (W == 1) {
        w[0] = *reinterpret_cast<const uint32_t*>(at);
    } else if constexpr (W == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(at);
        w[0] = v.x; w[1] = v.y;
    } else {
        const uint4 v = *reinterpret_cast<const uint4*>(at);
        w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
    }
}

// 16-byte unit u of row r of a tile lies at unit u ^ q4_swizzle(r): loads of 4, 8 and 16 bytes per lane, eight rows by
// four lanes, then meet no bank twice (bits of the row number reversed; with rows of 64 bytes, two of them share a line)
template <int UNITS>
__host__ __device__ constexpr uint32_t q4_swizzle(uint32_t r) {
    return UNITS == 8 ? ((r & 1) << 2) | (r & 2) | ((r >> 2) & 1) : (r & 2) | ((r >> 2) & 1);
}

// BYTES consecutive bytes (1, 2, 4, 8 or 16) from a naturally aligned address, as words.  Ordinary loads: the kernel lives while
// the one in front of it may still be writing x, so the read-only path is not open to it.
template <int BYTES>
__device__ __forceinline__ void q4_load_bytes(const void* p, uint32_t (&w)[(BYTES + 3) / 4]) {
    // volatile: a load asked for a tile ahead must not sink to where its value is used
    if constexpr (BYTES == 1) asm volatile("{\n\t.reg .u16 t;\n\tld.global.u8 t, [%1];\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(w[0]) : "l"(p));
    else if constexpr (BYTES == 2) asm volatile("{\n\t.reg .u16 t;\n\tld.global.u16 t, [%1];\n\tcvt.u32.u16 %0, t;\n\t}" : "=r"(w[0]) : "l"(p));
    else if constexpr (BYTES == 4) asm volatile("ld.global.b32 %0, [%1];" : "=r"(w[0]) : "l"(p));
    else if constexpr (BYTES == 8) asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "l"(p));
    else asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
}

// -(byte i of w): the byte becomes the low mantissa bits of 2^23
__device__ __forceinline__ float q4_minus_byte(uint32_t w, int i) {
    return 8388608.f - __uint_as_float(__byte_perm(w, 0x4B000000u, 0x7440 | i));
}

template <typename OUT>
__device__ __forceinline__ OUT q4_out(float v);
template <> __device__ __forceinline__ float q4_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __half q4_out<__half>(float v) { return __float2half_rn(v); }

// eight e4m3 values as four fp16 pairs (0,1) (2,3) (4,5) (6,7)
__device__ __forceinline__ void q4_widen(uint32_t lo, uint32_t hi, uint32_t (&e)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint16_t two = uint16_t((j < 2 ? lo : hi) >> (16 * (j & 1)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(e[j]) : "h"(two));
    }
}
// pairs (0,1) (2,3) (4,5) (6,7) -> (0,4) (2,6) (1,5) (3,7).  e4m3: the odd ones divided by 16, which is exact.
template <bool X8>
__device__ __forceinline__ uint4 q4_product_order(const uint32_t (&e)[4]) {
    uint4 x = make_uint4(__byte_perm(e[0], e[2], 0x5410), __byte_perm(e[1], e[3], 0x5410), __byte_perm(e[0], e[2], 0x7632),
                         __byte_perm(e[1], e[3], 0x7632));
    if constexpr (X8) {
        x.z = h2_bits(__hmul2(bits_h2(x.z), __float2half2_rn(0.0625f)));
        x.w = h2_bits(__hmul2(bits_h2(x.w), __float2half2_rn(0.0625f)));
    }
    return x;
}

// Eight entries of x, element by element: any alignment, zeros behind the last column
template <bool X8>
__device__ __forceinline__ void q4_load_x(const GemvQ4Params& p, uint32_t v, uint32_t k, uint32_t (&e)[4]) {
    uint32_t b[2] = {0u, 0u};
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = 0u;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (k + j < p.cols) {
            const uint64_t at = uint64_t(v) * p.ldx + k + j;
            if constexpr (X8) b[j >> 2] |= uint32_t(static_cast<const uint8_t*>(p.x)[at]) << (8 * (j & 3));
            else e[j >> 1] |= uint32_t(__half_as_ushort(static_cast<const __half*>(p.x)[at])) << (16 * (j & 1));
        }
    if constexpr (X8) q4_widen(b[0], b[1], e);
}

// NT: tiles of eight vectors (1 or 2).  X8: x is e4m3.  grid = clusters x ranks, ranks innermost; a cluster takes
// p.tiles neighbouring tiles of rows.
template <int GROUP, int NT, bool ZEROS, bool X8, typename OUT>
__global__ void __launch_bounds__(32 * Q4Cfg<NT>::WARPS, 1)
gemv_q4_kernel(const GemvQ4Params p) {
    using Cfg = Q4Cfg<NT>;
    constexpr int KW = Cfg::KW, UNITS = Cfg::UNITS, STAGES = Cfg::STAGES, RS = Cfg::RS, SUB = Cfg::SUB, TR = Cfg::TR;
    constexpr int WPL = GROUP / 32;                           // words a lane holds of a row's group
    constexpr int GC = KW / GROUP;                            // groups of a warp's piece
    constexpr uint32_t PITCH = UNITS * 16;
    extern __shared__ __align__(128) uint8_t q4_smem[];      // the swizzle works on address bits 4 to 6
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const uint32_t warps = blockDim.x >> 5, ranks = p.ranks, rank = blockIdx.x % ranks;
    const uint32_t tile0 = blockIdx.x / ranks * p.tiles;      // the cluster's rows: [row0, row0 + n_tiles * TR)
    const uint32_t row0 = tile0 * TR, all_tiles = (p.rows + TR - 1) / TR;
    const uint32_t n_tiles = min(p.tiles, all_tiles - tile0);
    const uint32_t row_bytes = (p.cols + 1) / 2, groups = (p.cols + GROUP - 1) / GROUP;
    const uint32_t pieces = (p.cols + KW - 1) / KW, piece = rank * warps + warp;      // this warp's columns: piece * KW ..
    const uint32_t active = min(warps, pieces > rank * warps ? pieces - rank * warps : 0u);   // warps that have some
    float* const parts = reinterpret_cast<float*>(q4_smem + warps * STAGES * Cfg::TILE);      // [2][warp][vector][RS]
    float* const sums = parts + 2 * warps * (Cfg::PART / 4);                                  // [2][block][vector][R]

    // ---- weights, tile after tile.  Addresses are a base that all threads share plus a 32-bit offset of the lane (the host
    // sees to that they fit).  Bytes behind a row's end, and all bytes of a warp without columns, become zeros.
    const uint32_t lrow = lane / UNITS, lunit = lane % UNITS; // this lane's first unit of a tile; the others 32 / UNITS rows on
    constexpr uint32_t ROWS = 32 / UNITS, COPIES = TR / ROWS; // rows per instruction, instructions per tile
    const uint8_t* const my_ring = q4_smem + warp * STAGES * Cfg::TILE;
    const uint32_t rq_byte = piece * (KW / 2) + lunit * 16, rq_bytes = rq_byte < row_bytes ? min(16u, row_bytes - rq_byte) : 0u;
    uint32_t rq_dst[2], rq_off[COPIES];                       // rows ROWS apart have one of two swizzles
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i)
        rq_dst[i] = smem_u32(my_ring) + (lrow + i * ROWS) * PITCH + ((lunit ^ q4_swizzle<UNITS>(lrow + i * ROWS)) * 16);
#pragma unroll
    for (uint32_t i = 0; i < COPIES; ++i) rq_off[i] = (lrow + i * ROWS) * uint32_t(p.ldw) + (rq_bytes ? rq_byte : 0u);
    const uint8_t* rq_base = p.W + uint64_t(row0) * p.ldw;
    auto request = [&](uint32_t tile, uint32_t stage) {
        if (tile < n_tiles) {
            const uint32_t row = row0 + tile * TR;
            if (row + TR <= p.rows) {
#pragma unroll
                for (uint32_t i = 0; i < COPIES; ++i)
                    cp_async16(stage + rq_dst[i & 1] + (i >> 1) * 2 * ROWS * PITCH, rq_base + rq_off[i], rq_bytes);
            } else {                                          // rows behind the last one become zeros
#pragma unroll
                for (uint32_t i = 0; i < COPIES; ++i) {
                    const bool in = row + lrow + i * ROWS < p.rows;
                    cp_async16(stage + rq_dst[i & 1] + (i >> 1) * 2 * ROWS * PITCH, in ? rq_base + rq_off[i] : p.W, in ? rq_bytes : 0u);
                }
            }
            rq_base += TR * p.ldw;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    static_assert((STAGES & (STAGES - 1)) == 0, "the ring wraps by a mask");
    griddep_launch();
    griddep_wait();
    for (int d = 0; d < STAGES - 1; ++d) request(d, d * Cfg::TILE);

    // ---- scales and zero points of rows g, g + 8, ... of a tile, asked for one tile ahead
    uint32_t sraw[2 * SUB][(2 * GC + 3) / 4], zraw[2 * SUB][(GC + 3) / 4];
    const uint32_t g0 = piece * GC;
    const bool sq_fast = p.vec_s && (!ZEROS || p.vec_z) && g0 + GC <= groups;
    const __half* sq_s = p.scales + uint64_t(row0) * p.lds;
    const uint8_t* sq_z = ZEROS ? p.zeros + uint64_t(row0) * p.ldz : nullptr;
    const uint32_t sq_soff = g * uint32_t(p.lds) + g0, sq_zoff = g * uint32_t(p.ldz) + g0;
    auto request_scales = [&](uint32_t tile) {
        if (tile >= n_tiles) return;
        const uint32_t row = row0 + tile * TR;
        if (sq_fast && row + TR <= p.rows) {
#pragma unroll
            for (int h = 0; h < 2 * SUB; ++h) {
                q4_load_bytes<2 * GC>(sq_s + h * 8 * p.lds + sq_soff, sraw[h]);
                if constexpr (ZEROS) q4_load_bytes<GC>(sq_z + h * 8 * p.ldz + sq_zoff, zraw[h]);
            }
        } else {
#pragma unroll
            for (int h = 0; h < 2 * SUB; ++h) {
                // rows behind the last one repeat it: their sums are never stored
                const uint64_t r = min(row + h * 8 + g, p.rows - 1);
                const __half* sp = p.scales + r * p.lds + g0;
#pragma unroll
                for (int j = 0; j < GC; ++j) {
                    const uint32_t b = g0 + j < groups ? __half_as_ushort(sp[j]) : 0u;
                    sraw[h][j / 2] = (j & 1) ? (sraw[h][j / 2] | (b << 16)) : b;
                }
                if constexpr (ZEROS) {
                    const uint8_t* zp = p.zeros + r * p.ldz + g0;
#pragma unroll
                    for (int j = 0; j < GC; ++j) {
                        const uint32_t b = g0 + j < groups ? zp[j] : 0u;
                        zraw[h][j / 4] = (j & 3) ? (zraw[h][j / 4] | (b << (8 * (j & 3)))) : b;
                    }
                }
            }
        }
        sq_s += TR * p.lds;
        if constexpr (ZEROS) sq_z += TR * p.ldz;
    };
    request_scales(0);

    // ---- this warp's x: registers in product order.  Lanes of vectors that do not exist hold the last one's: the columns
    // they lead to are never stored.
    uint4 xr[GC * WPL][NT];
    float xsum[GC][NT][2];
    if (p.vec_x && (piece + 1) * KW <= p.cols) {              // all loads first
        constexpr uint32_t B = X8 ? 1 : 2;
        const uint8_t* const xb = static_cast<const uint8_t*>(p.x) + (piece * KW + t * WPL * 8) * B;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint8_t* const row = xb + uint64_t(min(uint32_t(n * 8) + g, p.n_vec - 1)) * p.ldx * B;
#pragma unroll
            for (int i = 0; i < GC * WPL; ++i) {
                const uint8_t* at = row + (i / WPL * GROUP + i % WPL * 8) * B;
                if constexpr (X8) {
                    uint32_t w[2];
                    q4_load_bytes<8>(at, w);
                    xr[i][n].x = w[0];
                    xr[i][n].y = w[1];
                } else {
                    uint32_t w[4];
                    q4_load_bytes<16>(at, w);
                    xr[i][n] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < GC * WPL; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t e[4] = {xr[i][n].x, xr[i][n].y, xr[i][n].z, xr[i][n].w};
                if constexpr (X8) q4_widen(xr[i][n].x, xr[i][n].y, e);
                xr[i][n] = q4_product_order<X8>(e);
            }
    } else {
#pragma unroll
        for (int i = 0; i < GC * WPL; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                uint32_t e[4];
                q4_load_x<X8>(p, min(uint32_t(n * 8) + g, p.n_vec - 1), piece * KW + i / WPL * GROUP + (t * WPL + i % WPL) * 8, e);
                xr[i][n] = q4_product_order<X8>(e);
            }
    }
    // its group sums, by products with ones: every lane gets those of its two columns
#pragma unroll
    for (int gi = 0; gi < GC; ++gi)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            constexpr uint32_t ONE = 0x3C003C00u, UP = X8 ? 0x4C004C00u /* 16 */ : ONE;
            float s[4];
#pragma unroll
            for (int j = 0; j < WPL; ++j) {
                const uint4 x = xr[gi * WPL + j][n];
                if (j == 0) mma_16816_first(s, ONE, ONE, ONE, ONE, x.x, x.y);
                else mma_16816(s, ONE, ONE, ONE, ONE, x.x, x.y);
                mma_16816(s, UP, UP, UP, UP, x.z, x.w);
            }
            xsum[gi][n][0] = s[0] * 0x1p-24f;
            xsum[gi][n][1] = s[1] * 0x1p-24f;
        }

    auto scale_of = [&](uint32_t i) { return p.xs != nullptr ? p.xs[i / Cfg::R] : 1.f; };      // asked for before the sum is there
    auto store = [&](uint32_t block, uint32_t i, float s, float xs) {   // i = vector * R + row
        const uint32_t v = i / Cfg::R, r = block * Cfg::R + i % Cfg::R, row = row0 + r;
        if (r < n_tiles * TR && row < p.rows)                 // the last block may have fewer tiles
            static_cast<OUT*>(p.y)[uint64_t(v) * p.ldy + row] = q4_out<OUT>(s * 0x1p24f * xs);
    };
    // A cluster joins several blocks at a time: its barrier has to wait for a CTA's outstanding memory accesses.
    const uint32_t block_sums = Cfg::R * p.n_vec, per_join = Cfg::JOIN / block_sums;
    const uint32_t blocks = (n_tiles + Cfg::BLOCK - 1) / Cfg::BLOCK;
    auto join_cluster = [&](uint32_t b0, uint32_t n) {        // n of this cluster's blocks from b0 on, in rank order
        namespace cg = cooperative_groups;
        const cg::cluster_group cluster = cg::this_cluster();
        float* const from = sums + ((b0 / per_join) & 1u) * Cfg::JOIN;
        for (uint32_t i = rank * blockDim.x + threadIdx.x; i < n * block_sums; i += ranks * blockDim.x) {
            const uint32_t k = i / block_sums;
            const float xs = scale_of(i - k * block_sums);
            float s = 0.f;
            for (uint32_t c0 = 0; c0 < ranks; c0 += 8) {
                float d[8];                                   // requested together
#pragma unroll
                for (uint32_t c = 0; c < 8; ++c) d[c] = c0 + c < ranks ? *cluster.map_shared_rank(from + i, c0 + c) : 0.f;
#pragma unroll
                for (uint32_t c = 0; c < 8; ++c) s += d[c];
            }
            store(b0 + k, i - k * block_sums, s, xs);
        }
    };

    const uint32_t sw = q4_swizzle<UNITS>(g) * 16;            // rows 8 apart share it
    uint32_t tile = 0, stage = 0;
    for (uint32_t b = 0; b < blocks; ++b) {
        const uint32_t buf = b & 1u, in_block = min(uint32_t(Cfg::BLOCK), n_tiles - tile);
        float* part = parts + (buf * warps + warp) * (Cfg::PART / 4) + 2 * t * RS + g;
        for (uint32_t k = 0; k < in_block; ++k, ++tile) {
            // the stage that is asked for now was read in the previous turn, by all lanes
            __syncwarp();
            request(tile + STAGES - 1, (stage + (STAGES - 1) * Cfg::TILE) & (STAGES * Cfg::TILE - 1));
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
            __syncwarp();                                     // every lane's copies of this tile have landed
            float sc[2 * SUB][GC], nz[2 * SUB][GC];
#pragma unroll
            for (int h = 0; h < 2 * SUB; ++h)
#pragma unroll
                for (int j = 0; j < GC; ++j) {
                    sc[h][j] = half_bits(sraw[h][j / 2] >> (16 * (j & 1)));
                    if constexpr (ZEROS) nz[h][j] = q4_minus_byte(zraw[h][j / 4], j & 3);
                    else nz[h][j] = -8.f;
                }
            request_scales(tile + 1);
#pragma unroll
            for (int sub = 0; sub < SUB; ++sub) {
                float acc[NT][4];
                const uint8_t* const wrow = my_ring + stage + (sub * 16 + g) * PITCH;
#pragma unroll
                for (int gi = 0; gi < GC; ++gi) {
                    uint32_t wa[WPL], wb[WPL];                // rows g and g + 8
                    q4_words<WPL>(wrow + ((gi * (GROUP / 2) + t * WPL * 4) ^ sw), wa);
                    q4_words<WPL>(wrow + 8 * PITCH + ((gi * (GROUP / 2) + t * WPL * 4) ^ sw), wb);
                    float lo[NT][4], hi[NT][4];
#pragma unroll
                    for (int j = 0; j < WPL; ++j) {
                        uint32_t a[4], c[4];                  // pairs (0,4) (1,5) (2,6) (3,7) of rows g and g + 8
                        q4_pairs(wa[j], a);
                        q4_pairs(wb[j], c);
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            const uint4 x = xr[gi * WPL + j][n];
                            if (j == 0) mma_16816_first(lo[n], a[0], c[0], a[2], c[2], x.x, x.y);
                            else mma_16816(lo[n], a[0], c[0], a[2], c[2], x.x, x.y);
                            if (X8) mma_16816(lo[n], a[1], c[1], a[3], c[3], x.z, x.w);
                            else if (j == 0) mma_16816_first(hi[n], a[1], c[1], a[3], c[3], x.z, x.w);
                            else mma_16816(hi[n], a[1], c[1], a[3], c[3], x.z, x.w);
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {         // i >> 1: row g or g + 8; i & 1: vector 2t or 2t + 1
                            float d = X8 ? lo[n][i] : fmaf(hi[n][i], 0.0625f, lo[n][i]);
                            d = fmaf(nz[2 * sub + (i >> 1)][gi], xsum[gi][n][i & 1], d);
                            const float sg = sc[2 * sub + (i >> 1)][gi];
                            acc[n][i] = gi == 0 ? sg * d : fmaf(sg, d, acc[n][i]);
                        }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) part[(n * 8 + (i & 1)) * RS + sub * 16 + (i >> 1) * 8] = acc[n][i];
            }
            part += TR;
            stage = (stage + Cfg::TILE) & (STAGES * Cfg::TILE - 1);
        }
        // ---- join.  Two sets of partial sums: what the next block writes is not what this one reads.
        __syncthreads();
        const uint32_t in_join = b % per_join;
        if (ranks > 1 && in_join == 0 && b > 0) {             // before its half of `sums` is written again
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
            join_cluster(b - per_join, per_join);
        }
        float* const own = sums + ((b / per_join) & 1u) * Cfg::JOIN + in_join * block_sums;
        for (uint32_t i = threadIdx.x; i < block_sums; i += blockDim.x) {
            const float* at = parts + buf * warps * (Cfg::PART / 4) + i / Cfg::R * RS + i % Cfg::R;
            const float xs = ranks > 1 ? 1.f : scale_of(i);
            float s = 0.f;
#pragma unroll 4
            for (uint32_t w = 0; w < active; ++w) s += at[w * (Cfg::PART / 4)];
            if (ranks > 1) own[i] = s;
            else store(b, i, s, xs);
        }
        if (ranks > 1 && (in_join + 1 == per_join || b + 1 == blocks))
            asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    }
    if (ranks > 1) {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        const uint32_t b0 = (blocks - 1) / per_join * per_join;
        join_cluster(b0, blocks - b0);
        cluster_sync_all();                                   // nobody leaves while its sums are being read
    }
}

}  // namespace dxb
