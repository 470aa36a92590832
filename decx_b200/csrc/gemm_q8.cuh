// D(M x N) = alpha * diag(sa) * A(M x K) * B(N x K)^T * diag(sb) + beta * C        A, B e4m3, fp32 accumulation
//
// Both operands have K innermost, as a row-quantised operand has (its scale belongs to a row of the product's K sum
// and factors out of it), so both go to tcgen05.mma.kind::f8f6f4 as K-major tiles of 128 rows x 128 bytes, loaded by
// TMA with the 128-byte swizzle.  The scales are applied to the finished fp32 sums in the epilogue.
//
// Two kernels:
//   gemm_q8_pair   large products: persistent CTA pairs (cta_group::2), 256 x 256 tiles, two TMEM accumulators so that
//                  one tile's epilogue runs under the next tile's MMAs.  The pair form halves what each SM's shared
//                  memory has to deliver per MMA: each CTA holds its own 128 rows of A and of B only.
//   gemm_q8_thin   few rows of A (tokens) or few tiles: the operands swap places.  128 rows of B (weights) fill the
//                  128 lanes of the MMA whatever M is, and the rows of A are its N side, 16 to 128 at a time.  Such
//                  products are bound by reading B, so K is cut over a cluster of up to 8 CTAs until the GPU is full;
//                  the cluster adds its partial tiles through distributed shared memory in rank order: one launch,
//                  no workspace, no atomics.
// Every wait is bounded: on time-out the role writes a code to *status and the kernel unwinds.
#pragma once
#include <cooperative_groups.h>
#include <cuda_fp16.h>
#include "sm100_ptx.cuh"

namespace dxb {

struct GemmQ8Params {
    uint32_t M, N, K;
    const float* sa;           // M
    const float* sb;           // N
    const void* C;             // same type as D, or nullptr
    void* D;
    uint64_t ldc, ldd;
    float alpha, beta;
    int vec_d;                 // thin kernel: four neighbouring elements of D may be written at once
    int d_tma;                 // pair kernel: D through a staging tile and TMA stores (tmD); else per-thread stores
    int vec_c;                 // pair kernel: rows of C are 16-byte aligned
    uint32_t tiles_m, tiles_n;
    uint32_t group_m;          // pair kernel: height of the rasterisation groups, in tiles
    uint32_t ranks;            // thin kernel: CTAs that share a tile's K = cluster size
    unsigned* status;
    unsigned long long wait_limit_ns;
};

enum Q8Status : unsigned {
    Q8_TIMEOUT_PRODUCER = 0x201,
    Q8_TIMEOUT_MMA_FULL = 0x202,
    Q8_TIMEOUT_MMA_ACC = 0x203,
    Q8_TIMEOUT_EPILOGUE = 0x204,
    Q8_TIMEOUT_TAIL = 0x205,
};

__device__ __forceinline__ void q8_report(const GemmQ8Params& p, unsigned code) {
    if (p.status != nullptr) atomicCAS(p.status, 0u, code);
}

template <int CTAS>
__device__ __forceinline__ void umma_q8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CTAS == 1)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
            ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
            : "memory");
}

constexpr uint32_t Q8_KB = 128;                                     // bytes = elements of K per stage
constexpr uint32_t Q8_TILE = 128 * Q8_KB;                           // 128 rows of an operand
constexpr uint64_t Q8_DESC = smem_desc(SMEM_LAYOUT_SW128, 16, 1024);  // K-major, 8-row swizzle atoms

__device__ __forceinline__ float q8_to_f32(float v) { return v; }
__device__ __forceinline__ float q8_to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ void q8_put(float* p, float v) { *p = v; }
__device__ __forceinline__ void q8_put(__half* p, float v) { *p = __float2half_rn(v); }

// =============================================================================================== thin kernel
template <int BN>
struct ThinCfg {
    static constexpr uint32_t STAGE = Q8_TILE + BN * Q8_KB;
    static constexpr int STAGES = (108 * 1024) / STAGE;               // two CTAs per SM
    static constexpr uint32_t TMEM_COLS = BN < 32 ? 32 : BN;
    static constexpr uint32_t SMEM_BYTES = STAGES * STAGE + 1024 /*alignment slack*/ + 256 /*barriers*/ + BN * 4 /*scales of A*/;
    static constexpr uint32_t IDESC = umma_idesc(0u, false, false, 128, BN);
    static_assert(STAGES * STAGE >= 128 * BN * 4, "the partial tile is exchanged in the ring");
    static_assert(16 * STAGES + 16 <= 256, "barrier area");
};

// four neighbouring columns of one row of D
template <typename T>
__device__ __forceinline__ void q8_put4(const GemmQ8Params& p, uint32_t m, uint32_t n, float (&d)[4]) {
    T* at = static_cast<T*>(p.D) + uint64_t(m) * p.ldd + n;
    if (p.C != nullptr) {
        const T* c = static_cast<const T*>(p.C) + uint64_t(m) * p.ldc + n;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.N) d[i] = fmaf(p.beta, q8_to_f32(c[i]), d[i]);
    }
    if (p.vec_d && n + 4 <= p.N) {
        if constexpr (sizeof(T) == 2) {
            uint2 o;
            q8_put(reinterpret_cast<T*>(&o) + 0, d[0]);
            q8_put(reinterpret_cast<T*>(&o) + 1, d[1]);
            q8_put(reinterpret_cast<T*>(&o) + 2, d[2]);
            q8_put(reinterpret_cast<T*>(&o) + 3, d[3]);
            *reinterpret_cast<uint2*>(at) = o;
        } else {
            *reinterpret_cast<float4*>(at) = make_float4(d[0], d[1], d[2], d[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.N) q8_put(at + i, d[i]);
    }
}

// Adds the cluster's partial tiles ([token][128] floats at `partial` in every CTA) in rank order: this CTA's share.
// All ranks' values of a unit are requested before the first is used: a remote access takes a few hundred cycles.
template <int RANKS, typename T>
__device__ __forceinline__ void q8_join(const GemmQ8Params& p, float* partial, const float* sa, uint32_t rank, uint32_t tm0,
                                        uint32_t tn0, uint32_t tokens) {
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const float4* from[RANKS];
#pragma unroll
    for (int c = 0; c < RANKS; ++c) from[c] = reinterpret_cast<const float4*>(cluster.map_shared_rank(partial, c));
    for (uint32_t i = rank * blockDim.x + threadIdx.x; i < tokens * 32; i += RANKS * blockDim.x) {
        const uint32_t j = i >> 5, n = tn0 + (i & 31u) * 4;
        if (n >= p.N) continue;
        float4 v[RANKS];
#pragma unroll
        for (int c = 0; c < RANKS; ++c) v[c] = from[c][i];
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < RANKS; ++c) {
            d[0] += v[c].x; d[1] += v[c].y; d[2] += v[c].z; d[3] += v[c].w;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] *= sa[j] * (n + e < p.N ? p.alpha * __ldg(p.sb + n + e) : 0.f);
        q8_put4<T>(p, tm0 + j, n, d);
    }
}

template <int BN, typename T>
__global__ void __launch_bounds__(192)
gemm_q8_thin_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmQ8Params p) {
    using Cfg = ThinCfg<BN>;
    constexpr int STAGES = Cfg::STAGES;
    extern __shared__ uint8_t q8_smem[];
    const uint32_t base = (smem_u32(q8_smem) + 1023u) & ~1023u;
    const uint32_t full = base + STAGES * Cfg::STAGE, empty = full + 8 * STAGES, accf = empty + 8 * STAGES, slot = accf + 8;
    uint8_t* const smem = q8_smem + (base - smem_u32(q8_smem));
    float* partial = reinterpret_cast<float*>(smem);                                       // [token][128], reuses the ring
    float* sa = reinterpret_cast<float*>(smem + STAGES * Cfg::STAGE + 256);                // the tile's scales of A

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x % p.ranks, tile = blockIdx.x / p.ranks;
    const uint32_t tm = tile % p.tiles_m, tn = tile / p.tiles_m;
    const uint32_t n_kb = (p.K + Q8_KB - 1) / Q8_KB;
    const uint32_t kb0 = uint32_t(uint64_t(n_kb) * rank / p.ranks), kb1 = uint32_t(uint64_t(n_kb) * (rank + 1) / p.ranks);
    const uint64_t limit = p.wait_limit_ns;

    if (threadIdx.x == 0) {
        tma_prefetch_desc(&tmA);
        tma_prefetch_desc(&tmB);
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        mbar_init(accf, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<1>(slot, Cfg::TMEM_COLS);
        tmem_relinquish<1>();
    }
    griddep_launch();
    griddep_wait();                                                   // nothing of the operands is touched before
    if (warp >= 2 && threadIdx.x - 64 < BN) {
        const uint32_t m = tm * BN + threadIdx.x - 64;
        sa[threadIdx.x - 64] = m < p.M ? p.sa[m] : 0.f;
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + (slot - base));

    bool ok = true;
    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait_bounded(empty + 8 * s, ph ^ 1u, limit)) {
                    q8_report(p, Q8_TIMEOUT_PRODUCER);
                    ok = false;
                    break;
                }
                const uint32_t stage = base + s * Cfg::STAGE;
                mbar_arrive_expect_tx(full + 8 * s, Cfg::STAGE);
                tma_load_2d(stage, &tmB, full + 8 * s, int32_t(kb * Q8_KB), int32_t(tn * 128));
                tma_load_2d(stage + Q8_TILE, &tmA, full + 8 * s, int32_t(kb * Q8_KB), int32_t(tm * BN));
                if (++s == STAGES) { s = 0; ph ^= 1u; }
            }
            // every stage has been released: nothing is in flight towards this CTA's shared memory any more
            for (int i = 0; i < STAGES; ++i) {
                if (!mbar_wait_bounded(empty + 8 * s, ph ^ 1u, limit)) {
                    q8_report(p, Q8_TIMEOUT_TAIL);
                    // the MMA side is stuck: at least the copies have to land before the memory is given back
                    if (ok) for (int j = 0; j < STAGES; ++j) (void)mbar_wait_bounded(full + 8 * s, ph ^ 1u, limit);
                    break;
                }
                if (++s == STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            uint32_t s = 0, ph = 0;
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                if (!mbar_wait_bounded(full + 8 * s, ph, limit)) {
                    q8_report(p, Q8_TIMEOUT_MMA_FULL);
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                const uint32_t stage = base + s * Cfg::STAGE;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_q8<1>(tmem, smem_desc_at(Q8_DESC, stage + k * 32), smem_desc_at(Q8_DESC, stage + Q8_TILE + k * 32),
                               Cfg::IDESC, (kb > kb0 || k > 0) ? 1u : 0u);
                umma_commit<1>(empty + 8 * s);
                if (++s == STAGES) { s = 0; ph ^= 1u; }
            }
            if (ok) umma_commit<1>(accf);
        }
    } else {
        const uint32_t quarter = warp & 3u;
        const uint32_t n = tn * 128 + quarter * 32 + lane;
        const float sbn = n < p.N ? p.alpha * __ldg(p.sb + n) : 0.f;
        if (!mbar_wait_bounded(accf, 0, limit)) {
            if (lane == 0) q8_report(p, Q8_TIMEOUT_EPILOGUE);
            ok = false;
        }
        tc_fence_after_sync();
        const uint32_t taddr = tmem + ((quarter * 32u) << 16);
        constexpr int CH = BN < 32 ? BN : 32;
#pragma unroll 1
        for (uint32_t c = 0; c < BN && ok; c += CH) {
            const uint32_t m0 = tm * BN + c;
            if (m0 >= p.M) break;
            uint32_t v[32];
            tmem_ld_32x32(taddr + c, v);
            tmem_ld_wait();
            if (p.ranks == 1) {
                // lane = column: a warp writes 32 neighbouring elements of one row of D at a time
                float d[CH];
#pragma unroll
                for (int j = 0; j < CH; ++j) d[j] = __uint_as_float(v[j]) * (sa[c + j] * sbn);
                if (n < p.N) {
                    if (p.C != nullptr) {
                        const T* cp = static_cast<const T*>(p.C) + uint64_t(m0) * p.ldc + n;
#pragma unroll
                        for (int j = 0; j < CH; ++j)
                            if (m0 + j < p.M) d[j] = fmaf(p.beta, q8_to_f32(cp[uint64_t(j) * p.ldc]), d[j]);
                    }
                    T* dp = static_cast<T*>(p.D) + uint64_t(m0) * p.ldd + n;
#pragma unroll
                    for (int j = 0; j < CH; ++j)
                        if (m0 + j < p.M) q8_put(dp + uint64_t(j) * p.ldd, d[j]);
                }
            } else {
                // the ring is free: the MMAs that read it have completed
#pragma unroll
                for (int j = 0; j < CH; ++j) partial[(c + j) * 128 + quarter * 32 + lane] = __uint_as_float(v[j]);
            }
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<1>(tmem, Cfg::TMEM_COLS);
    }
    if (p.ranks > 1) {
        cluster_sync_all();
        const uint32_t tokens = min(uint32_t(BN), p.M - tm * BN);
        if (p.ranks == 2) q8_join<2, T>(p, partial, sa, rank, tm * BN, tn * 128, tokens);
        else if (p.ranks == 4) q8_join<4, T>(p, partial, sa, rank, tm * BN, tn * 128, tokens);
        else q8_join<8, T>(p, partial, sa, rank, tm * BN, tn * 128, tokens);
        cluster_sync_all();                                           // nobody leaves while its partial tile is being read
    }
}

// =============================================================================================== pair kernel
struct PairCfg {
    static constexpr uint32_t STAGE = 2 * Q8_TILE;                    // 128 rows of A, 128 rows of B
    static constexpr int STAGES = 6;
    static constexpr int EPI_WARPS = 8;                               // four lane quarters x two column halves
    static constexpr uint32_t STAGING = EPI_WARPS * 4096;             // per epilogue warp: 32 rows x 128 bytes of D
    static constexpr uint32_t SMEM_BYTES = STAGES * STAGE + STAGING + 1024 /*alignment slack*/ + 256 /*barriers*/ + 1024 /*scales of B*/;
    static constexpr uint32_t IDESC = umma_idesc(0u, false, false, 256, 256);
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static_assert(16 * STAGES + 32 + 8 <= 256, "barrier area");
    static_assert(SMEM_BYTES <= 227 * 1024, "one CTA's shared memory");
};

__device__ __forceinline__ void q8_tile_coords(uint32_t t, const GemmQ8Params& p, uint32_t& tm, uint32_t& tn) {
    const uint32_t per_group = p.group_m * p.tiles_n;
    const uint32_t g = t / per_group, first = g * p.group_m;
    const uint32_t rows = min(p.group_m, p.tiles_m - first), r = t - g * per_group;
    tm = first + r % rows;
    tn = r / rows;
}

// 32 columns col0.. of one row of C, if there are that many: a lane reads whole 128-byte lines (64 for fp16)
template <typename T>
__device__ __forceinline__ void q8_load_c(const GemmQ8Params& p, uint32_t row, uint32_t col0, uint4 (&c)[sizeof(T) * 2]) {
    if (row >= p.M || col0 >= p.N) return;
    const T* at = static_cast<const T*>(p.C) + uint64_t(row) * p.ldc + col0;
    if (p.vec_c && col0 + 32 <= p.N) {
#pragma unroll
        for (int u = 0; u < int(sizeof(T)) * 2; ++u) c[u] = reinterpret_cast<const uint4*>(at)[u];
    } else {
        T* e = reinterpret_cast<T*>(&c);
#pragma unroll
        for (int i = 0; i < 32; ++i) e[i] = col0 + i < p.N ? at[i] : T(0.f);
    }
}

// 32 finished columns col0.. of `row`, scaled by sa * sb[0..31], (+ beta * C), to the staging row (16-byte units unit0..,
// swizzled) or to D
template <typename T>
__device__ __forceinline__ void q8_store_chunk(const GemmQ8Params& p, uint32_t row, uint32_t col0, const uint32_t (&v)[32], float sa,
                                               const float* sb, const uint4 (&c)[sizeof(T) * 2], uint32_t stage_row, uint32_t unit0) {
    constexpr int PER = 16 / sizeof(T);                               // elements per 16-byte unit
    const uint32_t ncols = min(32u, p.N - col0), sw = (stage_row >> 7) & 7u;
    T* drow = static_cast<T*>(p.D) + uint64_t(row) * p.ldd + col0;
#pragma unroll
    for (int u = 0; u < 32 / PER; ++u) {
        float d[PER];
#pragma unroll
        for (int i = 0; i < PER; i += 4) {
            const float4 b = reinterpret_cast<const float4*>(sb)[(u * PER + i) / 4];
            d[i] = __uint_as_float(v[u * PER + i]) * (sa * b.x);
            d[i + 1] = __uint_as_float(v[u * PER + i + 1]) * (sa * b.y);
            d[i + 2] = __uint_as_float(v[u * PER + i + 2]) * (sa * b.z);
            d[i + 3] = __uint_as_float(v[u * PER + i + 3]) * (sa * b.w);
        }
        if (p.C != nullptr) {
            const T* e = reinterpret_cast<const T*>(&c[u]);
#pragma unroll
            for (int i = 0; i < PER; ++i) d[i] = fmaf(p.beta, q8_to_f32(e[i]), d[i]);
        }
        uint4 o;
        T* e = reinterpret_cast<T*>(&o);
#pragma unroll
        for (int i = 0; i < PER; ++i) q8_put(e + i, d[i]);
        if (stage_row != 0) {
            st_shared_v4(stage_row + (((unit0 + u) ^ sw) << 4), o.x, o.y, o.z, o.w);
        } else if (row < p.M) {
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (u * PER + i < ncols) drow[u * PER + i] = e[i];
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(PairCfg::THREADS, 1)
gemm_q8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmD, const GemmQ8Params p) {
    constexpr int STAGES = PairCfg::STAGES;
    extern __shared__ uint8_t q8_smem[];
    const uint32_t base = (smem_u32(q8_smem) + 1023u) & ~1023u;
    const uint32_t staging = base + STAGES * PairCfg::STAGE;
    const uint32_t full = staging + PairCfg::STAGING, empty = full + 8 * STAGES, accf = empty + 8 * STAGES, acce = accf + 16;
    const uint32_t slot = acce + 16;
    uint8_t* const smem = q8_smem + (base - smem_u32(q8_smem));
    float* const sb_tile = reinterpret_cast<float*>(smem + (full + 256 - base));       // the tile's 256 scales of B

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = cluster_ctarank();
    const bool leader = cta == 0;
    const uint32_t workers = gridDim.x / 2, worker = blockIdx.x / 2;
    const uint32_t n_tiles = p.tiles_m * p.tiles_n, n_kb = (p.K + Q8_KB - 1) / Q8_KB;
    const uint64_t limit = p.wait_limit_ns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(accf + 8 * a, 1);
            mbar_init(acce + 8 * a, 2 * PairCfg::EPI_WARPS);          // the epilogue warps of both CTAs
        }
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<2>(slot, 512);
        tmem_relinquish<2>();
    }
    griddep_launch();
    griddep_wait();                                                   // nothing of the operands is touched before
    tc_fence_before_sync();
    cluster_sync_all();
    tc_fence_after_sync();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(smem + (slot - base));

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        if (lane == 0) {
            tma_prefetch_desc(&tmA);
            tma_prefetch_desc(&tmB);
            const uint32_t full0 = map_to_cta(full, 0);
            uint32_t s = 0, ph = 0;
            bool ok = true;
            for (uint32_t t = worker; t < n_tiles && ok; t += workers) {
                uint32_t tm, tn;
                q8_tile_coords(t, p, tm, tn);
                const int32_t arow = int32_t((tm * 2 + cta) * 128), brow = int32_t((tn * 2 + cta) * 128);
                for (uint32_t kb = 0; kb < n_kb; ++kb) {
                    if (!mbar_wait_bounded(empty + 8 * s, ph ^ 1u, limit)) {
                        q8_report(p, Q8_TIMEOUT_PRODUCER);
                        ok = false;
                        break;
                    }
                    const uint32_t stage = base + s * PairCfg::STAGE, fb = full0 + 8 * s;
                    if (leader) mbar_arrive_expect_tx(full + 8 * s, 2 * PairCfg::STAGE);
                    tma_load_2d_pair(stage, &tmA, fb, int32_t(kb * Q8_KB), arow);
                    tma_load_2d_pair(stage + Q8_TILE, &tmB, fb, int32_t(kb * Q8_KB), brow);
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
            }
            // every stage this CTA filled has been released: no copy and no arrival of the peer is still on its way
            for (int i = 0; i < STAGES && ok; ++i) {
                if (!mbar_wait_bounded(empty + 8 * s, ph ^ 1u, limit)) {
                    q8_report(p, Q8_TIMEOUT_TAIL);
                    break;
                }
                if (++s == STAGES) { s = 0; ph ^= 1u; }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        if (leader && lane == 0) {
            const uint32_t peer_empty = map_to_cta(empty, 1), peer_accf = map_to_cta(accf, 1);
            uint32_t s = 0, ph = 0, it = 0;
            bool ok = true;
            for (uint32_t t = worker; t < n_tiles && ok; t += workers, ++it) {
                const uint32_t a = it & 1u, aph = (it >> 1) & 1u;
                if (!mbar_wait_bounded(acce + 8 * a, aph ^ 1u, limit)) {
                    q8_report(p, Q8_TIMEOUT_MMA_ACC);
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                for (uint32_t kb = 0; kb < n_kb; ++kb) {
                    if (!mbar_wait_bounded(full + 8 * s, ph, limit)) {
                        q8_report(p, Q8_TIMEOUT_MMA_FULL);
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t stage = base + s * PairCfg::STAGE;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_q8<2>(tmem + a * 256, smem_desc_at(Q8_DESC, stage + k * 32),
                                   smem_desc_at(Q8_DESC, stage + Q8_TILE + k * 32), PairCfg::IDESC, (kb | uint32_t(k)) ? 1u : 0u);
                    umma_commit<2>(empty + 8 * s);
                    umma_commit<2>(peer_empty + 8 * s);
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
                if (ok) {
                    umma_commit<2>(accf + 8 * a);
                    umma_commit<2>(peer_accf + 8 * a);
                }
            }
            for (int i = 0; i < 2 && ok; ++i, ++it) {                 // both accumulators drained by both CTAs
                if (!mbar_wait_bounded(acce + 8 * (it & 1u), ((it >> 1) & 1u) ^ 1u, limit)) {
                    q8_report(p, Q8_TIMEOUT_TAIL);
                    break;
                }
            }
        }
    } else {
        // ------------------------------------------------------------------ epilogue
        const uint32_t quarter = warp & 3u, half = (warp - 2u) >> 2;  // TMEM lanes [32 quarter, +32), columns [128 half, +128)
        const uint32_t acce0 = map_to_cta(acce, 0);
        const uint32_t stage_warp = staging + (warp - 2u) * 4096u;
        const uint32_t stage_row = p.d_tma ? stage_warp + lane * 128u : 0u;
        constexpr uint32_t BOX = 128 / sizeof(T);                     // columns of one staged box
        constexpr uint32_t SUB = BOX / 32;                            // 32-column chunks per box
        // TMA clips a column edge in 16-byte units: a box that crosses an edge N which is not 16-byte aligned is
        // written by predicated per-thread stores
        const bool ragged = ((p.N * uint32_t(sizeof(T))) & 15u) != 0u;
        uint32_t it = 0;
        bool ok = true;
        for (uint32_t t = worker; t < n_tiles; t += workers, ++it) {
            uint32_t tm, tn;
            q8_tile_coords(t, p, tm, tn);
            const uint32_t warp_row0 = (tm * 2 + cta) * 128 + quarter * 32, row = warp_row0 + lane, colbase = tn * 256 + half * 128;
            const float sa = row < p.M ? p.alpha * p.sa[row] : 0.f;
            // while the tile is being multiplied: its scales of B, once nobody reads the previous tile's any more, and C
            const uint32_t sb_col = tn * 256 + threadIdx.x - 64;
            const float sb_mine = sb_col < p.N ? __ldg(p.sb + sb_col) : 0.f;
            uint4 cbuf[2][sizeof(T) * 2];
            if (p.C != nullptr) q8_load_c<T>(p, row, colbase, cbuf[0]);
            asm volatile("bar.sync 1, 256;" ::: "memory");
            sb_tile[threadIdx.x - 64] = sb_mine;
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const uint32_t a = it & 1u, aph = (it >> 1) & 1u;
            if (ok && !mbar_wait_bounded(accf + 8 * a, aph, limit)) {
                if (lane == 0) q8_report(p, Q8_TIMEOUT_EPILOGUE);
                ok = false;                                           // keeps to the barriers above, touches nothing more
            }
            tc_fence_after_sync();
            const uint32_t taddr = tmem + a * 256 + half * 128 + ((quarter * 32u) << 16);
#pragma unroll
            for (uint32_t c = 0; c < 4; ++c) {
                const uint32_t col0 = colbase + c * 32;
                if (!ok || col0 >= p.N) break;
                if (p.C != nullptr && c < 3) q8_load_c<T>(p, row, col0 + 32, cbuf[(c + 1) & 1]);
                uint32_t v[32];
                tmem_ld_32x32(taddr + c * 32, v);
                tmem_ld_wait();
                const uint32_t sub = c & (SUB - 1), box0 = col0 - sub * 32;
                const bool boxed = p.d_tma && !(ragged && box0 + BOX > p.N);
                if (boxed && sub == 0) {
                    if (lane == 0) bulk_wait_read_all();              // the previous box has left the staging tile
                    __syncwarp();
                }
                q8_store_chunk<T>(p, row, col0, v, sa, sb_tile + half * 128 + c * 32, cbuf[c & 1], boxed ? stage_row : 0u, sub * (8 / SUB));
                if (boxed && (sub == SUB - 1 || col0 + 32 >= p.N)) {
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0 && warp_row0 < p.M) {
                        tma_store_2d(&tmD, stage_warp, int32_t(box0), int32_t(warp_row0));
                        bulk_commit_group();
                    }
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive_cluster(acce0 + 8 * a);
        }
        if (lane == 0 && p.d_tma) bulk_wait_all();
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<2>(tmem, 512);
    }
    cluster_sync_all();
}

}  // namespace dxb
