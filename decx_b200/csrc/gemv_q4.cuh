// Matrix-vector products with 4-bit weights: y[v][r] = xs[v] * sum_g s[r][g] * sum_{k in g} (q[r][k] - z[r][g]) * x[v][k]
// for 1 to 16 vectors at once.
//
// The weights are read once and set the pace (HBM).  The kernel gives every warp a piece of K that never changes, 256
// columns (128 for more than eight vectors), and lets it walk down the rows:
//   * its part of x sits in registers for the whole launch, already in the order the products want;
//   * weights stream through a ring of 16-row tiles in shared memory that belongs to the warp alone, filled by 16-byte
//     asynchronous copies: no barrier between copying and multiplying, and no wait that could expire;
//   * the warps of a CTA (up to 16) cover neighbouring pieces of K and, every 16 to 64 rows, add their partial sums
//     through shared memory; up to eight CTAs of a cluster do so through distributed shared memory, one round later, so
//     that nobody waits for the slowest.  Fixed order, no atomics, one launch, no workspace.
// The products run on the warp-level tensor path, m16n8k16 with fp32 accumulators: 16 rows times up to 8 vectors per
// instruction, for the price of one vector.  tcgen05 would need unpacked weights in shared memory, which costs more than
// the arithmetic.
//
// Exactness and cost.  A nibble q left in the low bits of an fp16 number IS the subnormal q * 2^-24 (16 q * 2^-24 for the
// upper nibble of a byte), and the tensor path multiplies subnormals exactly: a mask, or the difference of two such numbers
// (exact as well, and not on the integer pipe, which is what limits the unpacking), is all there is per pair of weights.  Products of lower and of upper nibbles go to accumulators of their own, and the zero point
// leaves the sum: sum (q - z) x = sum q x - z sum x, with the group sums of x computed once.  x is fp16 or e4m3, which
// fp16 holds exactly.  All sums are fp32; the group's scale multiplies in fp32; 2^24 comes back at the end; the only
// other rounding is the one to an fp16 result.
//
// Order of K.  A sum does not care, so each lane takes whole words of a row: of a group of 32 / 64 / 128 weights the lane
// that the instruction gives columns 2t, 2t+1, 2t+8, 2t+9 holds words t*w .. t*w+w-1 (w = 1 / 2 / 4, one shared-memory
// load), and its registers hold the matching x as 0 4 2 6 1 5 3 7 within eight.
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
    uint32_t ranks;            // CTAs that share a block of rows = cluster size, at most 8
    uint32_t passes;           // 1 unless K is longer than ranks * warps pieces
    uint32_t tiles;            // tiles of a cluster: its share of the rows
    int vec_s, vec_z;          // a tile's scales / zero points of one row may be read at once
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

// 16-byte unit u of row r of a tile lies at unit u ^ q4_swizzle(r): loads of 4, 8 and 16 bytes per lane, eight rows by
// four lanes, then meet no bank twice (bits of the row number reversed; with rows of 64 bytes, two of them share a line)
template <int UNITS>
__host__ __device__ constexpr uint32_t q4_swizzle(uint32_t r) {
    return UNITS == 8 ? ((r & 1) << 2) | (r & 2) | ((r >> 2) & 1) : (r & 2) | ((r >> 2) & 1);
}

// BYTES consecutive bytes (1, 2, 4, 8 or 16) from a naturally aligned address, as words
template <int BYTES>
__device__ __forceinline__ void q4_load_bytes(const void* p, uint32_t (&w)[(BYTES + 3) / 4]) {
    if constexpr (BYTES == 1) w[0] = __ldg(static_cast<const uint8_t*>(p));
    else if constexpr (BYTES == 2) w[0] = __ldg(static_cast<const uint16_t*>(p));
    else if constexpr (BYTES == 4) w[0] = __ldg(static_cast<const uint32_t*>(p));
    else if constexpr (BYTES == 8) { const uint2 v = __ldg(static_cast<const uint2*>(p)); w[0] = v.x; w[1] = v.y; }
    else { const uint4 v = __ldg(static_cast<const uint4*>(p)); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
}

template <typename OUT>
__device__ __forceinline__ OUT q4_out(float v);
template <> __device__ __forceinline__ float q4_out<float>(float v) { return v; }
template <> __device__ __forceinline__ __half q4_out<__half>(float v) { return __float2half_rn(v); }

// Eight entries of x as four fp16 pairs (0,1) (2,3) (4,5) (6,7); zeros behind the last column
template <bool X8>
__device__ __forceinline__ void q4_load_x(const GemvQ4Params& p, uint32_t v, uint32_t k, uint32_t (&e)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = 0u;
    if (v >= p.n_vec || k >= p.cols) return;
    if constexpr (X8) {
        const uint8_t* src = static_cast<const uint8_t*>(p.x) + uint64_t(v) * p.ldx + k;
        uint32_t b[2] = {0u, 0u};
        if (k + 8 <= p.cols && (reinterpret_cast<uintptr_t>(src) & 7) == 0) {
            q4_load_bytes<8>(src, b);
        } else {
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
            q4_load_bytes<16>(src, e);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (k + j < p.cols) e[j >> 1] |= uint32_t(__half_as_ushort(src[j])) << (16 * (j & 1));
        }
    }
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
    const uint32_t pieces = (p.cols + KW - 1) / KW;
    const uint32_t ring = smem_u32(q4_smem) + warp * STAGES * Cfg::TILE;
    float* const parts = reinterpret_cast<float*>(q4_smem + warps * STAGES * Cfg::TILE);      // [2][warp][vector][RS]
    float* const sums = parts + 2 * warps * (Cfg::PART / 4);                                  // [2][block][vector][R]
    // pieces this CTA covers in pass 0 (later passes have at most as many: their missing warps add nothing)
    const uint32_t piece0 = rank * warps + warp, pass_step = ranks * warps;
    const uint32_t active = min(warps, pieces > rank * warps ? pieces - rank * warps : 0u);

    // ---- the stream of tiles: down the rows; with several passes over K, pass by pass within a block of BLOCK tiles
    struct Place {                                            // where a stream is
        uint32_t row, left, tile, pass;
    };
    // moves a stream on; true: to another place than the next tile down
    auto advance = [&](Place& s) {
        s.row += TR;
        --s.left;
        if (p.passes == 1) return false;
        const uint32_t in_block = min(uint32_t(Cfg::BLOCK), n_tiles - (s.row - TR * (s.tile + 1) - row0) / TR);
        if (++s.tile < in_block) return false;
        s.tile = 0;
        if (++s.pass == p.passes) s.pass = 0;
        else s.row -= TR * in_block;
        return true;
    };

    const uint32_t lrow = lane / UNITS, lunit = lane % UNITS; // this lane's first unit of a tile; the others 32 / UNITS rows on
    constexpr uint32_t ROWS = 32 / UNITS, COPIES = TR / ROWS; // rows per instruction, instructions per tile
    uint32_t rq_dst[2];                                       // rows that many apart have one of two swizzles
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) rq_dst[i] = (lrow + i * ROWS) * PITCH + ((lunit ^ q4_swizzle<UNITS>(lrow + i * ROWS)) * 16);
    Place rq = {row0, n_tiles * p.passes, 0, 0};
    uint32_t rq_stage = ring, rq_bytes = 0;
    const uint8_t* rq_src = nullptr;
    auto weights_at = [&]() {
        const uint32_t byte = (piece0 + rq.pass * pass_step) * (KW / 2) + lunit * 16;
        rq_bytes = byte < row_bytes ? min(16u, row_bytes - byte) : 0u;
        rq_src = p.W + uint64_t(rq.row + lrow) * p.ldw + (rq_bytes ? byte : 0u);
    };
    weights_at();
    const uint64_t copy_step = ROWS * p.ldw;
    auto request = [&]() {
        if (rq.left != 0) {
            if (piece0 + rq.pass * pass_step < pieces) {
                const uint8_t* src = rq_src;
                if (rq.row + TR <= p.rows) {
#pragma unroll
                    for (uint32_t i = 0; i < COPIES; ++i, src += copy_step)
                        cp_async16(rq_stage + rq_dst[i & 1] + (i >> 1) * 2 * ROWS * PITCH, src, rq_bytes);
                } else {                                      // rows behind the last one become zeros
#pragma unroll
                    for (uint32_t i = 0; i < COPIES; ++i, src += copy_step) {
                        const bool in = rq.row + lrow + i * ROWS < p.rows;
                        cp_async16(rq_stage + rq_dst[i & 1] + (i >> 1) * 2 * ROWS * PITCH, in ? src : p.W, in ? rq_bytes : 0u);
                    }
                }
            }
            rq_src += TR * p.ldw;
            if (advance(rq)) weights_at();
            rq_stage = rq_stage + Cfg::TILE == ring + STAGES * Cfg::TILE ? ring : rq_stage + Cfg::TILE;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int d = 0; d < STAGES - 1; ++d) request();

    // ---- scales and zero points of rows g, g + 8, ... of a tile, asked for one tile ahead
    uint32_t sraw[2 * SUB][(2 * GC + 3) / 4], zraw[2 * SUB][(GC + 3) / 4];
    Place sq = {row0, n_tiles * p.passes, 0, 0};
    const __half* sq_s = nullptr;
    const uint8_t* sq_z = nullptr;
    bool sq_fast = false;
    auto scales_at = [&]() {
        const uint32_t g0 = (piece0 + sq.pass * pass_step) * GC;
        sq_fast = p.vec_s && (!ZEROS || p.vec_z) && g0 + GC <= groups;
        sq_s = p.scales + uint64_t(sq.row + g) * p.lds + g0;
        if constexpr (ZEROS) sq_z = p.zeros + uint64_t(sq.row + g) * p.ldz + g0;
    };
    scales_at();
    auto request_scales = [&]() {
        if (sq.left == 0) return;
        if (sq_fast && sq.row + TR <= p.rows) {
#pragma unroll
            for (int h = 0; h < 2 * SUB; ++h) {
                q4_load_bytes<2 * GC>(sq_s + h * 8 * p.lds, sraw[h]);
                if constexpr (ZEROS) q4_load_bytes<GC>(sq_z + h * 8 * p.ldz, zraw[h]);
            }
        } else {
            const uint32_t g0 = (piece0 + sq.pass * pass_step) * GC;
#pragma unroll
            for (int h = 0; h < 2 * SUB; ++h) {
                // rows behind the last one repeat it: their sums are never stored
                const uint64_t row = min(sq.row + h * 8 + g, p.rows - 1);
                const __half* sp = p.scales + row * p.lds + g0;
#pragma unroll
                for (int j = 0; j < GC; ++j) {
                    const uint32_t b = g0 + j < groups ? __half_as_ushort(sp[j]) : 0u;
                    sraw[h][j / 2] = (j & 1) ? (sraw[h][j / 2] | (b << 16)) : b;
                }
                if constexpr (ZEROS) {
                    const uint8_t* zp = p.zeros + row * p.ldz + g0;
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
        if (advance(sq)) scales_at();
    };
    request_scales();

    // ---- this warp's x: registers in product order, and the group sums of the vectors whose columns this lane gets
    uint4 xr[GC * WPL][NT];
    float xsum[GC][NT][2];
    auto load_x = [&](uint32_t piece) {
#pragma unroll
        for (int gi = 0; gi < GC; ++gi)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                float sum = 0.f;
#pragma unroll
                for (int j = 0; j < WPL; ++j) {
                    uint32_t e[4];
                    q4_load_x<X8>(p, n * 8 + g, piece * KW + gi * GROUP + (t * WPL + j) * 8, e);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 f = __half22float2(bits_h2(e[i]));
                        sum += f.x + f.y;
                    }
                    xr[gi * WPL + j][n] = make_uint4(__byte_perm(e[0], e[2], 0x5410), __byte_perm(e[1], e[3], 0x5410),
                                                     __byte_perm(e[0], e[2], 0x7632), __byte_perm(e[1], e[3], 0x7632));
                }
                sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                sum *= 0x1p-24f;
                xsum[gi][n][0] = __shfl_sync(0xffffffffu, sum, 8 * t);
                xsum[gi][n][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4);
            }
    };
    if (p.passes == 1) load_x(piece0);

    auto store = [&](uint32_t block, uint32_t i, float s) {   // i = vector * R + row
        const uint32_t v = i / Cfg::R, r = block * Cfg::R + i % Cfg::R, row = row0 + r;
        if (r < n_tiles * TR && row < p.rows) {               // the last block may have fewer tiles
            s *= 0x1p24f;
            if (p.xs != nullptr) s *= __ldg(p.xs + v);
            static_cast<OUT*>(p.y)[uint64_t(v) * p.ldy + row] = q4_out<OUT>(s);
        }
    };
    // A cluster joins several blocks at a time: its barrier has to wait for a CTA's outstanding memory accesses.
    const uint32_t block_sums = Cfg::R * p.n_vec, per_join = Cfg::JOIN / block_sums;
    const uint32_t blocks = (n_tiles + Cfg::BLOCK - 1) / Cfg::BLOCK;
    auto join_cluster = [&](uint32_t b0, uint32_t n) {        // n of this cluster's blocks from b0 on, in rank order
        namespace cg = cooperative_groups;
        const cg::cluster_group cluster = cg::this_cluster();
        float* const from = sums + ((b0 / per_join) & 1u) * Cfg::JOIN;
        for (uint32_t i = rank * blockDim.x + threadIdx.x; i < n * block_sums; i += ranks * blockDim.x) {
            float d[8];                                       // requested together
#pragma unroll
            for (uint32_t c = 0; c < 8; ++c) d[c] = c < ranks ? *cluster.map_shared_rank(from + i, c) : 0.f;
            float s = 0.f;
#pragma unroll
            for (uint32_t c = 0; c < 8; ++c) s += d[c];
            const uint32_t k = i / block_sums;
            store(b0 + k, i - k * block_sums, s);
        }
    };

    uint32_t stage = ring;
    const uint32_t sw = q4_swizzle<UNITS>(g) * 16;            // rows 8 apart share it
    for (uint32_t b = 0; b < blocks; ++b) {
        const uint32_t buf = b & 1u, in_block = min(uint32_t(Cfg::BLOCK), n_tiles - b * Cfg::BLOCK);
        float* const part = parts + (buf * warps + warp) * (Cfg::PART / 4) + 2 * t * RS + g;
        for (uint32_t pass = 0; pass < p.passes; ++pass) {
            const uint32_t piece = piece0 + pass * pass_step;
            if (p.passes > 1) load_x(piece);
            for (uint32_t tile = 0; tile < in_block; ++tile) {
                // the stage that is asked for now was read in the previous turn, by all lanes
                __syncwarp();
                request();
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
                __syncwarp();                                 // every lane's copies of this tile have landed
                float sc[2 * SUB][GC], nz[2 * SUB][GC];
#pragma unroll
                for (int h = 0; h < 2 * SUB; ++h)
#pragma unroll
                    for (int j = 0; j < GC; ++j) {
                        sc[h][j] = half_bits(sraw[h][j / 2] >> (16 * (j & 1)));
                        if constexpr (ZEROS) nz[h][j] = -float((zraw[h][j / 4] >> (8 * (j & 3))) & 255u);
                        else nz[h][j] = -8.f;
                    }
                request_scales();
#pragma unroll
                for (int sub = 0; sub < SUB; ++sub) {
                    float acc[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[n][i] = 0.f;
                    if (piece < pieces) {
                        const uint32_t wrow = stage + (sub * 16 + g) * PITCH;
#pragma unroll
                        for (int gi = 0; gi < GC; ++gi) {
                            uint32_t wa[WPL], wb[WPL];        // rows g and g + 8
                            q4_words<WPL>(wrow + ((gi * (GROUP / 2) + t * WPL * 4) ^ sw), wa);
                            q4_words<WPL>(wrow + 8 * PITCH + ((gi * (GROUP / 2) + t * WPL * 4) ^ sw), wb);
                            float lo[NT][4], hi[NT][4];
#pragma unroll
                            for (int j = 0; j < WPL; ++j) {
                                uint32_t a[4], c[4];          // pairs (0,4) (1,5) (2,6) (3,7) of rows g and g + 8
                                q4_pairs(wa[j], a);
                                q4_pairs(wb[j], c);
#pragma unroll
                                for (int n = 0; n < NT; ++n) {
                                    const uint4 x = xr[gi * WPL + j][n];
                                    if (j == 0) {
                                        mma_16816_first(lo[n], a[0], c[0], a[2], c[2], x.x, x.y);
                                        mma_16816_first(hi[n], a[1], c[1], a[3], c[3], x.z, x.w);
                                    } else {
                                        mma_16816(lo[n], a[0], c[0], a[2], c[2], x.x, x.y);
                                        mma_16816(hi[n], a[1], c[1], a[3], c[3], x.z, x.w);
                                    }
                                }
                            }
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int i = 0; i < 4; ++i) { // i >> 1: row g or g + 8; i & 1: vector 2t or 2t + 1
                                    float d = fmaf(hi[n][i], 0.0625f, lo[n][i]);
                                    d = fmaf(nz[2 * sub + (i >> 1)][gi], xsum[gi][n][i & 1], d);
                                    acc[n][i] = fmaf(sc[2 * sub + (i >> 1)][gi], d, acc[n][i]);
                                }
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float* at = part + (n * 8 + (i & 1)) * RS + tile * TR + sub * 16 + (i >> 1) * 8;
                            if (n * 8 + 2 * t + (i & 1) < p.n_vec) *at = pass == 0 ? acc[n][i] : *at + acc[n][i];
                        }
                }
                stage = stage + Cfg::TILE == ring + STAGES * Cfg::TILE ? ring : stage + Cfg::TILE;
            }
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
            float s = 0.f;
            for (uint32_t w = 0; w < active; ++w) s += at[w * (Cfg::PART / 4)];
            if (ranks > 1) own[i] = s;
            else store(b, i, s);
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
