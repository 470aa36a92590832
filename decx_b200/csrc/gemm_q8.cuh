// D(M x N) = alpha * diag(sa) * A(M x K) * B(N x K)^T * diag(sb) + beta * C        A, B e4m3, fp32 accumulation
//
// Both operands have K innermost, as a row-quantised operand has (its scale belongs to a row of the product's K sum
// and factors out of it), so both go to tcgen05.mma.kind::f8f6f4 as K-major tiles of 128 rows x 128 bytes, loaded by
// TMA with the 128-byte swizzle.  The scales are applied to the finished fp32 sums in the epilogue.
//
// Two kernels:
//   gemm_q8_pair   large products: persistent CTA pairs (cta_group::2) on tiles of 256 x 256, two TMEM accumulators so
//                  that one tile's epilogue runs under the next tile's MMAs.  The pair form halves what each SM's shared
//                  memory has to deliver per MMA: each CTA holds its own 128 rows of A and of B only.  What bounds it is
//                  that memory: 64 bytes per clock read by the MMAs and 64 written by TMA at the full rate.  One 128 of K
//                  takes 630 to 660 clocks of a run, 512 at that rate (4096 x 8192 x 8192: 626, tensor pipe 82 % busy).  (256 x 512 tiles, two accumulators sharing A, were
//                  measured: 2048 x 16384 x 4096 118 us against 102, 2048 x 4096 x 16384 99 against 102.)  8192 x 8192 x
//                  8192: 375 us, 2.9 PFLOP/s, in a short run, 437 to 460 in a long one under the power limit.  Few tiles (512 x
//                  8192 x 4096, 18.5 us, 1.86 PFLOP/s) add what is paid once: 2 us until the first MMA, 2.5 for the epilogue.
//   gemm_q8_thin   few rows of A (tokens) or few tiles: the operands swap places.  128 rows of B (weights) fill the
//                  128 lanes of the MMA whatever M is, and the rows of A are its N side, 16 to 128 at a time.  Such
//                  products are bound by reading B, so K is cut over a cluster of up to 8 CTAs until the GPU is full.
//                  Each CTA then sends its partial sums into the shared memory of the CTA that finishes these tokens
//                  (st.async, counted by an mbarrier there), which adds them in rank order: one launch, no workspace,
//                  no atomics, and no barrier between the last partial sum and the tokens that wait for it (one at the very
//                  end keeps the shared memory that is sent to alive).  16 tokens, 16384 x 4096: 15.0 us, 70 % of a copy's
//                  bandwidth; 4096 x 4096: 6.0 us, 43 %, since a product that short is the sum of its latencies (first load
//                  1 us, ring, join 1.3 us).
// Sums are fp32 in the tensor path, whose adder truncates: up to 2^-23 of the running sum for every 32 products.
// Every wait is bounded: on time-out the role writes a code to *status and the kernel unwinds.
#pragma once
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
    int d_tma;                 // pair kernel: D through a staging tile and TMA stores (tmD); else per-thread stores
    int c_tma;                 // pair kernel: boxes of C through TMA loads (tmC), into the same buffers
    uint32_t tiles_m, tiles_n;
    uint32_t group_m;          // pair kernel: height of the rasterisation groups, in tiles
    uint32_t ranks;            // thin kernel: CTAs that share a tile's K = cluster size
    int wide;                  // alpha is not ordinary (q8_ordinary)
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

// The epilogues multiply a sum by one fp32 factor, alpha and the two scales.  That is right as long as no product of them can
// leave the fp32 range: scales of 2^-50 to 2^50 or zero, alpha of 2^-20 to 2^20.  A tile with others ("wide") is finished by a
// plain loop in 64 bits; the epilogue warps agree on that while the tile is being multiplied.
constexpr float Q8_REACH = 0x1p50f, Q8_ALPHA_REACH = 0x1p20f;
__host__ __device__ __forceinline__ bool q8_ordinary(float s, float reach) {
    return s == 0.f || (fabsf(s) <= reach && fabsf(s) >= 1.f / reach);
}
// a barrier of the epilogue's `THREADS` threads that also says whether `mine` holds in any of them
template <int THREADS>
__device__ __forceinline__ bool q8_any(bool mine) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(uint32_t(mine)), "n"(THREADS)
        : "memory");
    return any != 0;
}
// one element of D, if it exists, from its finished sum
template <typename T>
__device__ __forceinline__ void q8_put_wide(const GemmQ8Params& p, uint32_t row, uint32_t col, float v, float sa) {
    if (row >= p.M || col >= p.N) return;
    float d = float(double(v) * (double(p.alpha) * double(sa)) * double(p.sb[col]));
    if (p.C != nullptr) d = fmaf(p.beta, q8_to_f32(static_cast<const T*>(p.C)[uint64_t(row) * p.ldc + col]), d);
    q8_put(static_cast<T*>(p.D) + uint64_t(row) * p.ldd + col, d);
}

// =============================================================================================== thin kernel
template <int BN, bool SPLIT>
struct ThinCfg {
    static constexpr uint32_t STAGE = Q8_TILE + BN * Q8_KB;
    // two CTAs per SM; 128 tokens with the inbox: one
    static constexpr int STAGES = BN == 16 ? 5 : BN == 32 ? 4 : BN == 64 ? 3 : (SPLIT ? 5 : 3);
    static constexpr uint32_t TMEM_COLS = BN < 32 ? 32 : BN;
    static constexpr uint32_t INBOX = SPLIT ? BN * 512 : 0;           // partial sums of this CTA's tokens, from all ranks
    static constexpr uint32_t SMEM_BYTES = STAGES * STAGE + 1024 /*alignment slack*/ + 256 /*barriers*/ + BN * 4 /*scales of A*/ + INBOX;
    static constexpr uint32_t IDESC = umma_idesc(0u, false, false, 128, BN);
    static_assert(16 * STAGES + 24 <= 256, "barrier area");
    // No CTA ever waits for tensor memory, whatever other kernels run: as many as shared memory admits leave enough of it,
    // and a kernel that takes all of it takes more than half of the shared memory, too.
    static_assert(228 * 1024 / (SMEM_BYTES + 1024) * TMEM_COLS <= 512 && SMEM_BYTES > 68 * 1024, "tensor memory for all CTAs of an SM");
};

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// Remote stores of 8 / 16 bytes whose arrival is counted on an mbarrier of the CTA they go to
__device__ __forceinline__ void st_async(uint32_t at, uint32_t bar, uint32_t a, uint32_t b) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.b32 [%0], {%1, %2}, [%3];" ::"r"(at), "r"(a), "r"(b), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void st_async(uint32_t at, uint32_t bar, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(at), "r"(a),
                 "r"(b), "r"(c), "r"(d), "r"(bar)
                 : "memory");
}
// bounded wait that also orders what other CTAs of the cluster wrote
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, uint64_t limit_ns) {
    const uint64_t t0 = global_timer_ns();
    for (uint32_t polls = 0;; ++polls) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
        if ((polls & 63u) == 63u && global_timer_ns() - t0 > limit_ns) return false;
    }
}

// C of tokens m0 .. m0 + N - 1 in column `col` (a lane's column: a warp reads 32 neighbouring elements of a row).  Asked for
// well before q8_thin_store needs it: these loads are what a small product with a C waits for.
template <int N, typename T>
__device__ __forceinline__ void q8_thin_c(const GemmQ8Params& p, uint32_t m0, uint32_t col, float (&c)[N]) {
    if (col >= p.N) return;
    const T* at = static_cast<const T*>(p.C) + uint64_t(m0) * p.ldc + col;
#pragma unroll
    for (int j = 0; j < N; ++j) c[j] = m0 + j < p.M ? q8_to_f32(at[uint64_t(j) * p.ldc]) : 0.f;
}
// N finished sums of the same tokens and column
template <int N, bool HASC, typename T>
__device__ __forceinline__ void q8_thin_store(const GemmQ8Params& p, uint32_t m0, uint32_t col, const float (&v)[N], const float (&c)[N],
                                              const float* sa, float sbn) {
    if (col >= p.N) return;
    T* at = static_cast<T*>(p.D) + uint64_t(m0) * p.ldd + col;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        float d = v[j] * (sa[j] * sbn);
        if constexpr (HASC) d = fmaf(p.beta, c[j], d);
        if (m0 + j < p.M) q8_put(at + uint64_t(j) * p.ldd, d);
    }
}

// Sends this thread's sums (column `n` of the tile, all its tokens) to the ranks that finish them: inbox layout
// [sender][token / U][128 columns][U], U = 2 or 4 tokens per store.
template <int BN, int RANKS>
__device__ __forceinline__ void q8_send(uint32_t taddr, uint32_t inbox, uint32_t bar, uint32_t rank, uint32_t n) {
    constexpr int TPO = BN / RANKS, U = TPO < 4 ? 2 : 4, CH = BN < 32 ? BN : 32;
#pragma unroll 1
    for (int c = 0; c < BN; c += CH) {
        uint32_t v[32];
        tmem_ld_32x32(taddr + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < CH; j += U) {
            const uint32_t token = c + j, owner = token / TPO, mine = token % TPO;
            const uint32_t at = map_to_cta(inbox + ((rank * (TPO / U) + mine / U) * 128 + n) * (U * 4), owner), to = map_to_cta(bar, owner);
            if constexpr (U == 2) st_async(at, to, v[j], v[j + 1]);
            else st_async(at, to, v[j], v[j + 1], v[j + 2], v[j + 3]);
        }
    }
}
// Waits for what the ranks send, adds it in rank order and finishes this rank's tokens.  Without a C they
// go by twos or fours, so that the first stores leave early; with one, up to 16 at a time, so that as many loads are in flight.
template <int BN, int RANKS, bool HASC, typename T>
__device__ __forceinline__ bool q8_finish(const GemmQ8Params& p, const float* inbox, uint32_t bar, uint64_t limit, const float* sa, uint32_t rank,
                                          uint32_t n, uint32_t tm, uint32_t col, float sbn) {
    constexpr int TPO = BN / RANKS, U = TPO < 4 ? 2 : 4, NB = !HASC ? U : TPO < 16 ? TPO : 16;
    const uint32_t m0 = tm * BN + rank * TPO;
    float c[NB], next[NB];
    if constexpr (HASC) q8_thin_c<NB, T>(p, m0, col, c);
    if (!__all_sync(0xffffffffu, mbar_wait_cluster(bar, 0, limit))) return false;
#pragma unroll 1
    for (int b = 0; b < TPO / NB; ++b) {
        if (m0 + b * NB >= p.M) break;
        if constexpr (HASC) {
            if (b + 1 < TPO / NB) q8_thin_c<NB, T>(p, m0 + (b + 1) * NB, col, next);
        }
        float s[NB];
#pragma unroll
        for (int k = 0; k < NB / U; ++k) {
#pragma unroll
            for (int e = 0; e < U; ++e) s[k * U + e] = 0.f;
#pragma unroll
            for (int r = 0; r < RANKS; ++r) {
                const float* at = inbox + ((r * (TPO / U) + b * (NB / U) + k) * 128 + n) * U;
                if constexpr (U == 2) {
                    const float2 f = *reinterpret_cast<const float2*>(at);
                    s[k * U] += f.x; s[k * U + 1] += f.y;
                } else {
                    const float4 f = *reinterpret_cast<const float4*>(at);
                    s[k * U] += f.x; s[k * U + 1] += f.y; s[k * U + 2] += f.z; s[k * U + 3] += f.w;
                }
            }
        }
        q8_thin_store<NB, HASC, T>(p, m0 + b * NB, col, s, c, sa + rank * TPO + b * NB, sbn);
        if constexpr (HASC) {
#pragma unroll
            for (int j = 0; j < NB; ++j) c[j] = next[j];
        }
    }
    return true;
}

template <int BN, int RANKS, typename T>
__device__ __forceinline__ bool q8_finish_c(const GemmQ8Params& p, const float* inbox, uint32_t bar, uint64_t limit, const float* sa, uint32_t rank,
                                            uint32_t n, uint32_t tm, uint32_t col, float sbn) {
    return p.C == nullptr ? q8_finish<BN, RANKS, false, T>(p, inbox, bar, limit, sa, rank, n, tm, col, sbn)
                          : q8_finish<BN, RANKS, true, T>(p, inbox, bar, limit, sa, rank, n, tm, col, sbn);
}
// The tile whose K is not cut: the accumulator straight to D, up to 32 tokens at a time.
template <int BN, bool HASC, typename T>
__device__ __forceinline__ bool q8_direct(const GemmQ8Params& p, uint32_t bar, uint64_t limit, uint32_t taddr, uint32_t tm, uint32_t col,
                                          const float* sa, float sbn) {
    constexpr int CH = BN < 32 ? BN : 32;
    float c[CH], next[CH];
    if constexpr (HASC) q8_thin_c<CH, T>(p, tm * BN, col, c);
    if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar, 0, limit))) return false;
    tc_fence_after_sync();
#pragma unroll 1
    for (uint32_t k = 0; k < BN / CH; ++k) {
        const uint32_t m0 = tm * BN + k * CH;
        if (m0 >= p.M) break;
        if constexpr (HASC) {
            if (k + 1 < BN / CH) q8_thin_c<CH, T>(p, m0 + CH, col, next);
        }
        uint32_t v[32];
        tmem_ld_32x32(taddr + k * CH, v);
        tmem_ld_wait();
        float f[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) f[j] = __uint_as_float(v[j]);
        q8_thin_store<CH, HASC, T>(p, m0, col, f, c, sa + k * CH, sbn);
        if constexpr (HASC) {
#pragma unroll
            for (int j = 0; j < CH; ++j) c[j] = next[j];
        }
    }
    return true;
}

// The same for a wide tile: this rank's tokens, column `col`, from the inbox or (K not cut) from the accumulator
template <int BN, bool SPLIT, typename T>
__device__ __forceinline__ void q8_thin_wide(const GemmQ8Params& p, const float* inbox, uint32_t taddr, const float* sa, uint32_t rank, uint32_t n,
                                             uint32_t tm, uint32_t col) {
    const uint32_t tokens = SPLIT ? BN / p.ranks : BN, u = tokens < 4 ? 2 : 4;
#pragma unroll 1
    for (uint32_t t = 0; t < tokens; ++t) {
        float s = 0.f;
        if constexpr (SPLIT) {
#pragma unroll 1
            for (uint32_t r = 0; r < p.ranks; ++r) s += inbox[((r * (tokens / u) + t / u) * 128 + n) * u + t % u];
        } else {
            uint32_t v;
            __syncwarp();                                             // lanes without a column are back
            tmem_ld_32x1(taddr + t, v);
            tmem_ld_wait();
            s = __uint_as_float(v);
        }
        q8_put_wide<T>(p, tm * BN + rank * tokens + t, col, s, sa[rank * tokens + t]);
    }
}

template <int BN, bool SPLIT, typename T>
__global__ void __launch_bounds__(192)
gemm_q8_thin_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const GemmQ8Params p) {
    using Cfg = ThinCfg<BN, SPLIT>;
    constexpr int STAGES = Cfg::STAGES;
    extern __shared__ uint8_t q8_smem[];
    const uint32_t base = (smem_u32(q8_smem) + 1023u) & ~1023u;
    const uint32_t full = base + STAGES * Cfg::STAGE, empty = full + 8 * STAGES, accf = empty + 8 * STAGES, inbar = accf + 8, slot = inbar + 8;
    uint8_t* const smem = q8_smem + (base - smem_u32(q8_smem));
    float* const sa = reinterpret_cast<float*>(smem + STAGES * Cfg::STAGE + 256);          // the tile's scales of A
    const float* const inbox = sa + BN;                                                    // only with several ranks

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = blockIdx.x % p.ranks, tile = blockIdx.x / p.ranks;
    const uint32_t tm = tile % p.tiles_m, tn = tile / p.tiles_m;
    const uint32_t n_kb = (p.K + Q8_KB - 1) / Q8_KB;
    const uint32_t kb0 = uint32_t(uint64_t(n_kb) * rank / p.ranks), kb1 = uint32_t(uint64_t(n_kb) * (rank + 1) / p.ranks);
    const uint64_t limit = p.wait_limit_ns;
    constexpr bool split = SPLIT;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        mbar_init(accf, 1);
        mbar_init(inbar, 1);
        fence_mbar_init();
        if (split) mbar_arrive_expect_tx(inbar, Cfg::INBOX);
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
    if (split) cluster_arrive();                                      // the inbox barrier is ready
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
        __syncwarp();
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
        __syncwarp();
    }
    const uint32_t quarter = warp & 3u, n = quarter * 32 + lane, col = tn * 128 + n;       // of an epilogue thread
    float sbn = 0.f;
    bool wide = false;
    if (warp >= 2) {
        sbn = col < p.N ? p.sb[col] : 0.f;
        wide = q8_any<128>(p.wide || !q8_ordinary(sbn, Q8_REACH) || (threadIdx.x - 64 < BN && !q8_ordinary(sa[threadIdx.x - 64], Q8_REACH)));
        sbn *= p.alpha;
        if (split) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(accf, 0, limit));
            tc_fence_after_sync();
        } else if (wide) {
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(accf, 0, limit));
            tc_fence_after_sync();
            if (ok) q8_thin_wide<BN, SPLIT, T>(p, inbox, tmem + ((quarter * 32u) << 16), sa, 0, n, tm, col);
        } else if (p.C == nullptr) {
            ok = q8_direct<BN, false, T>(p, accf, limit, tmem + ((quarter * 32u) << 16), tm, col, sa, sbn);
        } else {
            ok = q8_direct<BN, true, T>(p, accf, limit, tmem + ((quarter * 32u) << 16), tm, col, sa, sbn);
        }
        if (!ok && lane == 0) q8_report(p, Q8_TIMEOUT_EPILOGUE);
    }
    if (split) {
        cluster_wait();                                               // every CTA of the cluster is there, its inbox ready
        if (warp >= 2 && ok) {
            const uint32_t taddr = tmem + ((quarter * 32u) << 16), in = base + STAGES * Cfg::STAGE + 256 + BN * 4;
            if (p.ranks == 2) q8_send<BN, 2>(taddr, in, inbar, rank, n);
            else if (p.ranks == 4) q8_send<BN, 4>(taddr, in, inbar, rank, n);
            else q8_send<BN, 8>(taddr, in, inbar, rank, n);
        }
        __syncwarp();
        cluster_arrive();                                             // this CTA sends nothing more
        if (warp >= 2 && ok) {
            bool got;
            if (wide) {
                got = __all_sync(0xffffffffu, mbar_wait_cluster(inbar, 0, limit));
                if (got) q8_thin_wide<BN, SPLIT, T>(p, inbox, 0, sa, rank, n, tm, col);
            } else {
                got = p.ranks == 2   ? q8_finish_c<BN, 2, T>(p, inbox, inbar, limit, sa, rank, n, tm, col, sbn)
                      : p.ranks == 4 ? q8_finish_c<BN, 4, T>(p, inbox, inbar, limit, sa, rank, n, tm, col, sbn)
                                     : q8_finish_c<BN, 8, T>(p, inbox, inbar, limit, sa, rank, n, tm, col, sbn);
            }
            if (!got && lane == 0) q8_report(p, Q8_TIMEOUT_EPILOGUE);
        }
        __syncwarp();
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc<1>(tmem, Cfg::TMEM_COLS);
    }
    if (split) cluster_wait();                                        // nobody is still being sent to by this CTA, nor this one
}

// =============================================================================================== pair kernel
struct PairCfg {
    static constexpr uint32_t STAGE = 2 * Q8_TILE;                    // 128 rows of A, 128 rows of B
    static constexpr int STAGES = 5;
    static constexpr int EPI_WARPS = 8;                               // four lane quarters x two column halves
    static constexpr int BUFS = 4;                                    // per epilogue warp: boxes of 32 rows x 64 bytes of C and D
    static constexpr uint32_t BOX = 2048;
    static constexpr uint32_t STAGING = EPI_WARPS * BUFS * BOX;
    static constexpr uint32_t BARS = 512;
    static constexpr uint32_t SMEM_BYTES = STAGES * STAGE + STAGING + 1024 /*alignment slack*/ + BARS + 1024 /*scales of B*/;
    static constexpr uint32_t IDESC = umma_idesc(0u, false, false, 256, 256);
    static constexpr int THREADS = 64 + 32 * EPI_WARPS;
    static constexpr uint32_t INBOX = 128 * 128 * 4;                  // SPLIT: the other pair's sums of this CTA's columns, in the
    static_assert(INBOX <= STAGES * STAGE, "inbox");                  // ring's place
    static_assert(16 * STAGES + 32 + 8 * EPI_WARPS * BUFS + 16 <= BARS, "barrier area");
    static_assert(SMEM_BYTES <= 227 * 1024, "one CTA's shared memory");
};

__device__ __forceinline__ void q8_tile_coords(uint32_t t, const GemmQ8Params& p, uint32_t& tm, uint32_t& tn) {
    const uint32_t per_group = p.group_m * p.tiles_n;
    const uint32_t g = t / per_group, first = g * p.group_m;
    const uint32_t rows = min(p.group_m, p.tiles_m - first), r = t - g * per_group;
    tm = first + r % rows;
    tn = r / rows;
}

// A thread's row of a wide tile, `count` columns from `col` on.  `in`: what the other pair sent (SPLIT)
template <bool SPLIT, typename T>
__device__ __forceinline__ void q8_pair_wide(const GemmQ8Params& p, uint32_t taddr, const float* in, uint32_t row, uint32_t col, uint32_t count,
                                             float sa) {
#pragma unroll 1
    for (uint32_t c = 0; c < count; ++c) {
        uint32_t v;
        __syncwarp();                                                 // lanes without a row are back
        tmem_ld_32x1(taddr + c, v);
        tmem_ld_wait();
        q8_put_wide<T>(p, row, col + c, __uint_as_float(v) + (SPLIT ? in[c / 4 * 512 + c % 4] : 0.f), sa);
    }
}

// SPLIT: two pairs (a cluster of four CTAs) share a tile, each half of K.  Pair r finishes columns [128 r, +128): the CTAs that
// hold the same rows send each other the other half, as the thin kernel does, and into the ring, which is free once
// both pairs' MMAs are done.
template <bool SPLIT, typename T>
__global__ void __launch_bounds__(PairCfg::THREADS, 1)
gemm_q8_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmD, const __grid_constant__ CUtensorMap tmC, const GemmQ8Params p) {
    using Cfg = PairCfg;
    constexpr int STAGES = Cfg::STAGES;
    extern __shared__ uint8_t q8_smem[];
    const uint32_t base = (smem_u32(q8_smem) + 1023u) & ~1023u;
    const uint32_t staging = base + STAGES * Cfg::STAGE;
    const uint32_t full = staging + Cfg::STAGING, empty = full + 8 * STAGES, accf = empty + 8 * STAGES, acce = accf + 16;
    const uint32_t cbar0 = acce + 16, inbar = cbar0 + 8 * Cfg::EPI_WARPS * Cfg::BUFS, slot = inbar + 8;
    uint8_t* const smem = q8_smem + (base - smem_u32(q8_smem));
    float* const sb_tile = reinterpret_cast<float*>(smem + (full + Cfg::BARS - base));     // the tile's scales of B

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t in_cluster = cluster_ctarank(), cta = in_cluster & 1u, rank = SPLIT ? in_cluster >> 1 : 0u;
    const uint32_t lead = in_cluster & ~1u, peer = in_cluster | 1u;   // this pair's CTAs within the cluster
    const bool leader = cta == 0;
    constexpr uint32_t ranks = SPLIT ? 2 : 1;
    const uint32_t workers = gridDim.x / (2 * ranks), worker = blockIdx.x / (2 * ranks);
    const uint32_t n_tiles = p.tiles_m * p.tiles_n, all_kb = (p.K + Q8_KB - 1) / Q8_KB;
    const uint32_t kb0 = uint32_t(uint64_t(all_kb) * rank / ranks), n_kb = uint32_t(uint64_t(all_kb) * (rank + 1) / ranks) - kb0;
    const uint64_t limit = p.wait_limit_ns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(accf + 8 * a, 1);
            mbar_init(acce + 8 * a, 2 * Cfg::EPI_WARPS);              // the epilogue warps of both CTAs
        }
        for (int w = 0; w < Cfg::EPI_WARPS * Cfg::BUFS; ++w) mbar_init(cbar0 + 8 * w, 1);
        mbar_init(inbar, 1);
        fence_mbar_init();
        if (SPLIT) mbar_arrive_expect_tx(inbar, Cfg::INBOX);
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
            const uint32_t full0 = map_to_cta(full, lead);
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
                    const uint32_t stage = base + s * Cfg::STAGE, fb = full0 + 8 * s;
                    if (leader) mbar_arrive_expect_tx(full + 8 * s, 2 * Cfg::STAGE);
                    tma_load_2d_pair(stage, &tmA, fb, int32_t((kb0 + kb) * Q8_KB), arow);
                    tma_load_2d_pair(stage + Q8_TILE, &tmB, fb, int32_t((kb0 + kb) * Q8_KB), brow);
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
            }
            // every stage this CTA filled has been released: no copy and no arrival of the peer is still on its way
            for (int i = 0; i < STAGES && ok; ++i) {
                if (!mbar_wait_bounded(empty + 8 * s, ph ^ 1u, limit)) {
                    q8_report(p, Q8_TIMEOUT_TAIL);
                    ok = false;
                    break;
                }
                if (++s == STAGES) { s = 0; ph ^= 1u; }
            }
            // the MMA side is stuck: at least both CTAs' copies (counted on the leader's barriers) have to land
            if (!ok && leader)
                for (int i = 0; i < STAGES; ++i) {
                    (void)mbar_wait_bounded(full + 8 * s, ph ^ 1u, limit / 8);
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        if (leader && lane == 0) {
            const uint32_t peer_empty = map_to_cta(empty, peer), peer_accf = map_to_cta(accf, peer);
            uint32_t s = 0, ph = 0, it = 0;
            bool ok = true;
            for (uint32_t t = worker; t < n_tiles && ok; t += workers, ++it) {
                const uint32_t a = it & 1u, aph = (it >> 1) & 1u;     // tiles alternate between two accumulators
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
                    const uint32_t stage = base + s * Cfg::STAGE;
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        umma_q8<2>(tmem + a * 256, smem_desc_at(Q8_DESC, stage + k * 32), smem_desc_at(Q8_DESC, stage + Q8_TILE + k * 32),
                                   Cfg::IDESC, (kb | uint32_t(k)) ? 1u : 0u);
                    umma_commit<2>(empty + 8 * s);
                    umma_commit<2>(peer_empty + 8 * s);
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
                if (ok) {
                    umma_commit<2>(accf + 8 * a);
                    umma_commit<2>(peer_accf + 8 * a);
                }
            }
            // both accumulators drained by both CTAs (SPLIT: the barrier at the end sees to that; the epilogue waits for this
            // warp first)
            for (int i = 0; i < 2 && ok && !SPLIT; ++i, ++it) {
                if (!mbar_wait_bounded(acce + 8 * (it & 1u), ((it >> 1) & 1u) ^ 1u, limit)) {
                    q8_report(p, Q8_TIMEOUT_TAIL);
                    break;
                }
            }
        }
    }
    if (warp < 2) {
        __syncwarp();
        if (SPLIT) {                                                  // the epilogue's handshake needs all threads
            cluster_arrive();
            cluster_wait();
        }
    } else {
        // ------------------------------------------------------------------ epilogue
        // Warp (quarter, half): TMEM lanes [32 quarter, +32), columns [128 half, +128), 64 bytes of D
        // per row at a time.  A box of C arrives by TMA in one of the warp's four buffers, is turned into D in place and
        // leaves by TMA; the boxes two ahead are asked for meanwhile, those of a tile's start while it is multiplied.
        constexpr uint32_t CW = 64 / sizeof(T);                       // columns of a box
        constexpr uint32_t share = 128 / ranks, BOXES = share / CW;   // columns this warp finishes of a tile, in so many boxes
        constexpr int PER = 16 / sizeof(T);                           // elements of a 16-byte unit
        const uint32_t quarter = warp & 3u, half = (warp - 2u) >> 2;
        const uint32_t acce0 = map_to_cta(acce, lead);
        const uint32_t bufs = staging + (warp - 2u) * Cfg::BUFS * Cfg::BOX, cbar = cbar0 + 8 * (warp - 2u) * Cfg::BUFS;
        const uint32_t sw = (lane >> 1) & 3u;                         // 64-byte swizzle: unit ^ (row / 2) % 4
        // TMA clips a column edge in 16-byte units: a box that crosses an edge N which is not 16-byte aligned is
        // written by predicated per-thread stores
        const bool ragged = ((p.N * uint32_t(sizeof(T))) & 15u) != 0u;
        uint32_t it = 0, q = 0, cphase = 0, asked = 0;                // q: boxes so far; a phase bit, and whether C is on its way, per buffer
        bool ok = true;
        for (uint32_t t = worker; t < n_tiles; t += workers, ++it) {
            uint32_t tm, tn;
            q8_tile_coords(t, p, tm, tn);
            const uint32_t warp_row0 = (tm * 2 + cta) * 128 + quarter * 32, row = warp_row0 + lane;
            const uint32_t col_in_tile = SPLIT ? rank * 128 + half * share : half * 128;
            auto box_col = [&](uint32_t i) { return tn * 256 + col_in_tile + i * CW; };
            auto boxed = [&](uint32_t col) { return p.d_tma && col < p.N && warp_row0 < p.M && !(ragged && col + CW > p.N); };
            auto fetch_c = [&](uint32_t i) {                          // box i of this tile into buffer (q + i) % 4
                if (i < BOXES && p.c_tma && boxed(box_col(i))) {
                    const uint32_t b = (q + i) % Cfg::BUFS;
                    asked |= 1u << b;
                    if (lane == 0) {
                        mbar_arrive_expect_tx(cbar + 8 * b, Cfg::BOX);
                        tma_load_2d(bufs + b * Cfg::BOX, &tmC, cbar + 8 * b, int32_t(box_col(i)), int32_t(warp_row0));
                    }
                }
            };
            const float sa_mine = row < p.M ? p.sa[row] : 0.f, sa = p.alpha * sa_mine;
            // while the tile is being multiplied: its scales of B, once nobody reads the previous tile's any more, and C
            const uint32_t sb_col = tn * 256 + threadIdx.x - 64;
            const float sb_mine = sb_col < p.N ? p.sb[sb_col] : 0.f;
            if (ok && p.c_tma) {
                if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 2;" ::: "memory");     // buffers q, q + 1 are free
                fetch_c(0);
                fetch_c(1);
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");
            sb_tile[threadIdx.x - 64] = sb_mine;
            const bool wide = q8_any<256>(p.wide || !q8_ordinary(sa_mine, Q8_REACH) || !q8_ordinary(sb_mine, Q8_REACH));
            const uint32_t a = it & 1u, aph = (it >> 1) & 1u;
            if (ok && !__all_sync(0xffffffffu, mbar_wait_bounded(accf + 8 * a, aph, limit))) {
                if (lane == 0) q8_report(p, Q8_TIMEOUT_EPILOGUE);
                ok = false;                                       // keeps to the barriers above, touches nothing more
            }
            tc_fence_after_sync();
            if constexpr (SPLIT) {
                __syncwarp();
                cluster_arrive();                                     // this pair's MMAs have read the ring
                cluster_wait();                                       // the other pair's have, too
                if (ok) {
                    // this warp's 64 of the columns that the other pair finishes: inbox layout [column / 4][128 rows][4]
                    const uint32_t other = (rank ^ 1u) * 2 + cta, to = map_to_cta(inbar, other);
                    const uint32_t at = map_to_cta(base + (half * share / 4 * 128 + quarter * 32 + lane) * 16, other);
                    const uint32_t src = tmem + (rank ^ 1u) * 128 + half * share + ((quarter * 32u) << 16);
#pragma unroll
                    for (uint32_t c = 0; c < share / 32; ++c) {
                        uint32_t v[32];
                        tmem_ld_32x32(src + c * 32, v);
                        tmem_ld_wait();
#pragma unroll
                        for (uint32_t j = 0; j < 32; j += 4) st_async(at + (c * 32 + j) / 4 * 2048, to, v[j], v[j + 1], v[j + 2], v[j + 3]);
                    }
                    if (!__all_sync(0xffffffffu, mbar_wait_cluster(inbar, 0, limit))) {
                        if (lane == 0) q8_report(p, Q8_TIMEOUT_EPILOGUE);
                        ok = false;
                    }
                }
            }
            if (wide && ok) {
#pragma unroll 1
                for (uint32_t i = 0; i < 2; ++i) {                    // boxes of C that are on their way
                    const uint32_t b = (q + i) % Cfg::BUFS;
                    if (!((asked >> b) & 1u)) continue;
                    if (!__all_sync(0xffffffffu, mbar_wait_bounded(cbar + 8 * b, (cphase >> b) & 1u, limit))) {
                        if (lane == 0) q8_report(p, Q8_TIMEOUT_EPILOGUE);
                        ok = false;
                    }
                    cphase ^= 1u << b;
                    asked ^= 1u << b;
                }
                __syncwarp();
                if (ok)
                    q8_pair_wide<SPLIT, T>(p, tmem + a * 256 + col_in_tile + ((quarter * 32u) << 16),
                                           reinterpret_cast<const float*>(smem) + (half * share / 4 * 128 + quarter * 32 + lane) * 4, row, box_col(0),
                                           share, sa_mine);
                for (uint32_t k = 0; k < BOXES; ++k) {                // its boxes keep their place
                    if (lane == 0) bulk_commit_group();
                }
            }
#pragma unroll 1
            for (uint32_t c = 0; c < share / 32 && ok && !wide; ++c) {    // 32 columns at a time: one box of fp16, two of fp32
                if (box_col(c * (32 / CW)) >= p.N) {
                    for (uint32_t k = 0; k < 32 / CW; ++k) {      // boxes that do not exist keep their place
                        if (lane == 0) bulk_commit_group();
                    }
                    continue;
                }
                uint32_t v[32];
                tmem_ld_32x32(tmem + a * 256 + col_in_tile + c * 32 + ((quarter * 32u) << 16), v);
                tmem_ld_wait();
                if constexpr (SPLIT) {                                // and what has arrived (two terms: the order does not matter)
                    const float4* in = reinterpret_cast<const float4*>(smem) + (half * share + c * 32) / 4 * 128 + quarter * 32 + lane;
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const float4 g = in[j * 128];
                        v[4 * j] = __float_as_uint(__uint_as_float(v[4 * j]) + g.x);
                        v[4 * j + 1] = __float_as_uint(__uint_as_float(v[4 * j + 1]) + g.y);
                        v[4 * j + 2] = __float_as_uint(__uint_as_float(v[4 * j + 2]) + g.z);
                        v[4 * j + 3] = __float_as_uint(__uint_as_float(v[4 * j + 3]) + g.w);
                    }
                }
#pragma unroll
                for (uint32_t k = 0; k < 32 / CW; ++k) {
                    const uint32_t i = c * (32 / CW) + k, col = box_col(i), b = (q + i) % Cfg::BUFS;
                    const bool box = boxed(col);
                    // the store that left from this buffer four boxes ago, and the one two ahead's, have been read
                    if (lane == 0) {
                        if (p.c_tma) asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                        else asm volatile("cp.async.bulk.wait_group.read 3;" ::: "memory");
                    }
                    __syncwarp();
                    fetch_c(i + 2);
                    const bool c_box = box && p.c_tma;
                    if (c_box) {
                        if (!__all_sync(0xffffffffu, mbar_wait_bounded(cbar + 8 * b, (cphase >> b) & 1u, limit))) {
                            if (lane == 0) q8_report(p, Q8_TIMEOUT_EPILOGUE);
                            ok = false;
                        }
                        cphase ^= 1u << b;
                        asked ^= 1u << b;
                    }
                    const uint32_t at = bufs + b * Cfg::BOX + lane * 64;
                    const float* sbp = sb_tile + col_in_tile + c * 32 + k * CW;
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u) {
                        float d[PER];
#pragma unroll
                        for (int e = 0; e < PER; e += 4) {
                            const float4 f = *reinterpret_cast<const float4*>(sbp + u * PER + e);
                            d[e] = __uint_as_float(v[k * CW + u * PER + e]) * (sa * f.x);
                            d[e + 1] = __uint_as_float(v[k * CW + u * PER + e + 1]) * (sa * f.y);
                            d[e + 2] = __uint_as_float(v[k * CW + u * PER + e + 2]) * (sa * f.z);
                            d[e + 3] = __uint_as_float(v[k * CW + u * PER + e + 3]) * (sa * f.w);
                        }
                        const uint32_t unit = at + ((u ^ sw) << 4);
                        const uint32_t left = col + u * PER < p.N ? p.N - col - u * PER : 0u;      // columns from here on
                        if (p.C != nullptr) {
                            if (c_box) {
                                const uint4 w = ld_shared_v4(unit);
                                const T* cp = reinterpret_cast<const T*>(&w);
#pragma unroll
                                for (int e = 0; e < PER; ++e) d[e] = fmaf(p.beta, q8_to_f32(cp[e]), d[e]);
                            } else if (row < p.M) {
                                const T* cp = static_cast<const T*>(p.C) + uint64_t(row) * p.ldc + col + u * PER;
#pragma unroll
                                for (int e = 0; e < PER; ++e)
                                    if (uint32_t(e) < left) d[e] = fmaf(p.beta, q8_to_f32(cp[e]), d[e]);
                            }
                        }
                        uint4 o;
                        T* op = reinterpret_cast<T*>(&o);
#pragma unroll
                        for (int e = 0; e < PER; ++e) q8_put(op + e, d[e]);
                        if (box) {
                            st_shared_v4(unit, o.x, o.y, o.z, o.w);
                        } else if (row < p.M) {
                            T* dp = static_cast<T*>(p.D) + uint64_t(row) * p.ldd + col + u * PER;
#pragma unroll
                            for (int e = 0; e < PER; ++e)
                                if (uint32_t(e) < left) dp[e] = op[e];
                        }
                    }
                    if (box) {
                        fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) tma_store_2d(&tmD, bufs + b * Cfg::BOX, int32_t(col), int32_t(warp_row0));
                    }
                    if (lane == 0) bulk_commit_group();           // one group per box, stored or not
                }
            }
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0 && ok) mbar_arrive_cluster(acce0 + 8 * a);
            q += BOXES;
        }
        if (lane == 0) bulk_wait_all();
        if (!ok)                                                      // copies still on their way have to land first
            for (uint32_t b = 0; b < Cfg::BUFS; ++b)
                if ((asked >> b) & 1u) (void)mbar_wait_bounded(cbar + 8 * b, (cphase >> b) & 1u, limit);
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
