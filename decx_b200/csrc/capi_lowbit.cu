// extern "C" layer, third part: the operators on 8-bit and 4-bit operands.  See include/decx_b200.h for the contracts.
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <cstring>

#include "../../include/decx_b200.h"
#include "capi_shared.h"
#include "gemm_q8.cuh"
#include "gemv_q4.cuh"
#include "per_device.h"
#include "rownorm_q8.cuh"
#include "rownorm_q8_plan.h"

using namespace dxb;
using dxb_host::aligned16;
using dxb_host::PerDevice;

namespace {

int sm_count() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
    return n;
}
int current_device() {
    int dev = 0;
    return cudaGetDevice(&dev) == cudaSuccess ? dev : -1;
}

// Launch configuration with a cluster of CTAs.  All kernels here wait for the grids before them themselves
// (griddep_wait), so they are launched programmatically dependent on them: their CTAs start while the last ones of the
// previous kernel drain.  DECXB200_PDL=0 turns that off.
void cluster_config(cudaLaunchConfig_t& cfg, cudaLaunchAttribute (&attr)[2], unsigned blocks, unsigned threads, unsigned smem,
                    unsigned cluster, cudaStream_t s) {
    static const int pdl_env = [] { const char* e = getenv("DECXB200_PDL"); return e ? atoi(e) : 1; }();
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(blocks);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = attr;
    if (pdl_env != 0) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = cluster;
        attr[cfg.numAttrs].val.clusterDim.y = 1;
        attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
}

template <typename K, typename... Args>
int launch_cluster(K kern, unsigned blocks, unsigned threads, unsigned smem, unsigned cluster, cudaStream_t s, const Args&... args) {
    cudaLaunchConfig_t cfg;
    cudaLaunchAttribute attr[2];
    cluster_config(cfg, attr, blocks, threads, smem, cluster, s);
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) return int(e);
    dxb_host::count_launch();
    return 0;
}

// Dynamic shared memory beyond 48 KB has to be allowed once per kernel and device.
template <typename K>
int allow_smem(K kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return int(e);
    if (dev < 64 && ((done.load(std::memory_order_relaxed) >> dev) & 1)) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return int(e);
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
    return 0;
}

template <typename T, bool NORM, bool RES, bool WARP, bool SHIFT, int NCH>
int launch_row_q8_ring(cudaStream_t s, RowQ8Params p, uint32_t threads) {
    const uint32_t slot = q8_ring_slot(threads, SHIFT, NCH * 8 * sizeof(T) / 16 * (RES ? 2 : 1));
    auto kern = row_q8_ring_kernel<T, NORM, RES, WARP, SHIFT, NCH>;
    static std::atomic<uint64_t> done{0};
    static std::atomic<int> regs{0};
    int rc = allow_smem(kern, Q8_RING_SMEM, done);
    if (rc != 0) return rc;
    int r = regs.load(std::memory_order_relaxed);
    if (r == 0) {
        cudaFuncAttributes a;
        const cudaError_t e = cudaFuncGetAttributes(&a, kern);
        if (e != cudaSuccess) return int(e);
        regs.store(r = a.numRegs, std::memory_order_relaxed);
    }
    const Q8RingPlan plan = q8_ring_plan(slot, threads, uint32_t(r));
    p.depth = plan.depth;
    const uint64_t want = WARP ? (uint64_t(p.rows) + threads / 32 - 1) / (threads / 32) : p.rows;
    const uint64_t have = uint64_t(sm_count()) * plan.per_sm;
    return launch_cluster(kern, unsigned(want < have ? want : have), threads, slot * p.depth, 1, s, p);
}

// Kernels that keep one row per CTA or warp: rows that do not fit a ring, or operands that only single elements fit (VEC false:
// any alignment, and fewer columns than a warp has lanes).  The ring is the faster one wherever it works, from a single row
// on (norm of 37 x 512 fp16 with a residual 2.0 against 2.6 us, 296 x 8192 3.7 against 5.4, 1184 x 8192 13.4 against 20.6).
template <typename T, bool NORM, bool VEC>
int launch_row_q8(cudaStream_t s, const RowQ8Params& p) {
    const unsigned blocks = p.rows < 0x7fffffffu ? p.rows : 0x7fffffffu;
    if (p.cols > 8 * 4 * 1024) return launch_cluster(row_q8_long_kernel<T, NORM>, blocks, 1024, 0, 1, s, p);
    const uint32_t chunks = (p.cols + 7) / 8;
    auto threads = [&](uint32_t nch) { return (chunks + 32 * nch - 1) / (32 * nch) * 32; };
    if constexpr (!VEC) {
        const unsigned warps = unsigned((uint64_t(p.rows) + 7) / 8);
        if (p.cols <= 256) return launch_cluster(row_q8_kernel<T, NORM, true, false, 1>, warps, 256, 0, 1, s, p);
        if (p.cols <= 512) return launch_cluster(row_q8_kernel<T, NORM, true, false, 2>, warps, 256, 0, 1, s, p);
        if (p.cols <= 1024) return launch_cluster(row_q8_kernel<T, NORM, true, false, 4>, warps, 256, 0, 1, s, p);
    }
    if constexpr (!VEC || (NORM && sizeof(T) == 4)) {         // two slots of fp32 rows and residuals end at 12800 columns
        if (chunks <= 2048) return launch_cluster(row_q8_kernel<T, NORM, false, VEC, 2>, blocks, threads(2), 0, 1, s, p);
    }
    return launch_cluster(row_q8_kernel<T, NORM, false, VEC, 4>, blocks, threads(4), 0, 1, s, p);
}

template <typename T, bool NORM, bool RES, bool SHIFT>
int launch_row_q8_shape(cudaStream_t s, const RowQ8Params& p) {
    if (p.cols <= 256) return launch_row_q8_ring<T, NORM, RES, true, SHIFT, 1>(s, p, 256);
    if (p.cols <= 512) return launch_row_q8_ring<T, NORM, RES, true, SHIFT, 2>(s, p, 256);
    if (p.cols <= 1024) return launch_row_q8_ring<T, NORM, RES, true, SHIFT, 4>(s, p, 256);
    return launch_row_q8_ring<T, NORM, RES, false, SHIFT, 2>(s, p, (p.cols + 511) / 512 * 32);
}

template <typename T, bool NORM>
int run_row_q8(cudaStream_t s, const RowQ8Params& p) {
    const uint64_t e = sizeof(T);
    auto elem = [&](const void* a) { return reinterpret_cast<uintptr_t>(a) % e == 0; };
    if (!elem(p.x) || !elem(p.r) || !elem(p.sum) || !elem(p.w) || (reinterpret_cast<uintptr_t>(p.scales) & 3) != 0)
        return DECXB200_EALIGN;
    const bool rows16 = aligned16(p.x) && (p.ldx * e) % 16 == 0 && (p.r == nullptr || (aligned16(p.r) && (p.ldr * e) % 16 == 0)) &&
                        (p.sum == nullptr || (aligned16(p.sum) && (p.lds * e) % 16 == 0));
    const bool out8 = (reinterpret_cast<uintptr_t>(p.q) & 7) == 0 && p.ldq % 8 == 0 && aligned16(p.w);
    // two slots of the ring have to fit: the limit is 1024 threads times two pieces of 8, or shared memory
    const uint64_t slot = uint64_t(p.cols + 511) / 512 * (rows16 ? 512 : 528) * e * (p.r != nullptr ? 2 : 1);
    const bool ring = out8 && p.cols >= 16 && p.cols <= 16384 && 2 * slot <= Q8_RING_SLOTS;
    if (!ring) return rows16 && out8 && p.cols >= 16 ? launch_row_q8<T, NORM, true>(s, p) : launch_row_q8<T, NORM, false>(s, p);
    if constexpr (NORM) {
        if (p.r != nullptr)
            return rows16 ? launch_row_q8_shape<T, true, true, false>(s, p) : launch_row_q8_shape<T, true, true, true>(s, p);
    }
    return rows16 ? launch_row_q8_shape<T, NORM, false, false>(s, p) : launch_row_q8_shape<T, NORM, false, true>(s, p);
}

constexpr uint32_t Q4_MAX_VEC = 16, Q4_MAX_RANKS = 16;

template <int GROUP, int NT, bool ZEROS, bool X8, typename OUT>
int launch_gemv_q4(cudaStream_t s, GemvQ4Params p) {
    using Cfg = Q4Cfg<NT>;
    auto kern = gemv_q4_kernel<GROUP, NT, ZEROS, X8, OUT>;
    static std::atomic<uint64_t> done{0};
    int rc = allow_smem(kern, Cfg::smem(Cfg::WARPS), done);
    if (rc != 0) return rc;
    const uint32_t pieces = (p.cols + Cfg::KW - 1) / Cfg::KW;
    p.ranks = (pieces + Cfg::WARPS - 1) / Cfg::WARPS;
    if (p.ranks > Q4_MAX_RANKS) return DECXB200_ETOOLARGE;
    const uint32_t warps = (pieces + p.ranks - 1) / p.ranks;
    if (p.ranks > 8) {                       // beyond the portable cluster size
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return int(e);
    }
    constexpr uint32_t GC = Cfg::KW / GROUP;
    p.vec_s = reinterpret_cast<uintptr_t>(p.scales) % (2 * GC) == 0 && p.lds % GC == 0;
    p.vec_z = reinterpret_cast<uintptr_t>(p.zeros) % GC == 0 && p.ldz % GC == 0;
    constexpr uint32_t X = X8 ? 8 : 16;
    p.vec_x = reinterpret_cast<uintptr_t>(p.x) % X == 0 && p.ldx % 8 == 0;
    // clusters the GPU holds at once: the grid, since they stay and take turns over the blocks of rows
    static PerDevice held[Q4_MAX_RANKS][Cfg::WARPS];
    const int device = current_device();
    cudaError_t e = cudaSuccess;
    const int clusters = held[p.ranks - 1][warps - 1].get(device, [&] {
        int n = 0;
        if (p.ranks == 1) {
            e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, int(32 * warps), Cfg::smem(warps));
            n *= sm_count();
        } else {
            cudaLaunchConfig_t cfg;
            cudaLaunchAttribute attr[2];
            cluster_config(cfg, attr, p.ranks, 32 * warps, Cfg::smem(warps), p.ranks, s);
            e = cudaOccupancyMaxActiveClusters(&n, kern, &cfg);
        }
        return e == cudaSuccess ? n : 0;
    });
    if (e != cudaSuccess) return int(e);
    if (clusters < 1) return DECXB200_ETOOLARGE;
    const uint64_t tiles = (uint64_t(p.rows) + Cfg::TR - 1) / Cfg::TR;
    p.tiles = uint32_t((tiles + clusters - 1) / clusters);
    const uint64_t n = (tiles + p.tiles - 1) / p.tiles;
    return launch_cluster(kern, unsigned(n * p.ranks), 32 * warps, Cfg::smem(warps), p.ranks, s, p);
}

template <int GROUP, int NT, bool ZEROS>
int run_gemv_q4(cudaStream_t s, bool x8, bool f32, const GemvQ4Params& p) {
    if (x8) return f32 ? launch_gemv_q4<GROUP, NT, ZEROS, true, float>(s, p) : launch_gemv_q4<GROUP, NT, ZEROS, true, __half>(s, p);
    return f32 ? launch_gemv_q4<GROUP, NT, ZEROS, false, float>(s, p) : launch_gemv_q4<GROUP, NT, ZEROS, false, __half>(s, p);
}
template <int GROUP>
int run_gemv_q4_group(cudaStream_t s, bool x8, bool f32, const GemvQ4Params& p) {
    const bool z = p.zeros != nullptr;
    // Sixteen vectors at once take half as many columns per warp: with more than 16384 columns, which 8 CTAs hold, two rounds
    // of eight do.  Up to there one round is faster: 4096 x 4096 7.9 against 10.0 us for 16 vectors and 6.8 against 9.5 for
    // 9, 16384 x 4096 19.7 against 20.5; at the border, 16384 x 16384, 9 vectors 63.5 against 68.1 us, 16 77.5 against 72.8.
    if (p.n_vec > 8 && p.cols <= 8 * Q4Cfg<2>::WARPS * Q4Cfg<2>::KW)
        return z ? run_gemv_q4<GROUP, 2, true>(s, x8, f32, p) : run_gemv_q4<GROUP, 2, false>(s, x8, f32, p);
    for (uint32_t v = 0; v < p.n_vec; v += 8) {
        GemvQ4Params q = p;
        q.n_vec = p.n_vec - v < 8 ? p.n_vec - v : 8;
        q.x = static_cast<const uint8_t*>(p.x) + uint64_t(v) * p.ldx * (x8 ? 1 : 2);
        q.y = static_cast<uint8_t*>(p.y) + uint64_t(v) * p.ldy * (f32 ? 4 : 2);
        if (p.xs != nullptr) q.xs = p.xs + v;
        const int rc = z ? run_gemv_q4<GROUP, 1, true>(s, x8, f32, q) : run_gemv_q4<GROUP, 1, false>(s, x8, f32, q);
        if (rc != 0) return rc;
    }
    return 0;
}

// ------------------------------------------------------------------------------------------------ 8-bit GEMM
// How many clusters of `size` CTAs of a kernel the GPU holds at once (0: it does not say)
template <typename K>
int clusters_at_once(K kern, unsigned threads, unsigned smem, unsigned size, PerDevice& known) {
    const int device = current_device();
    return known.get(device, [&] {
        int n = 0;
        cudaLaunchConfig_t cfg;
        cudaLaunchAttribute attr[2];
        cluster_config(cfg, attr, size, threads, smem, size, nullptr);
        return cudaOccupancyMaxActiveClusters(&n, kern, &cfg) == cudaSuccess ? n : 0;
    });
}

// How many CTAs cut a tile's K in the thin kernel, at least two stages each: as many as are on the GPU at once; up to 64
// tokens, whose CTAs are short and share their SMs, as many as two turns take (64 x 8192 x 8192 17.2 against 20.5 us, 16 x
// 6144 x 4096 6.7 against 8.5, though 16 x 16384 x 4096 15.0 against 14.4; 128 x 8192 x 8192 would take 28.3 for 20.3)
template <int BN, typename T>
uint32_t q8_thin_ranks(uint64_t tiles, uint32_t n_kb) {
    static std::atomic<uint64_t> done{0};
    static PerDevice held[4];
    auto kern = gemm_q8_thin_kernel<BN, true, T>;
    using Cfg = ThinCfg<BN, true>;
    if (allow_smem(kern, Cfg::SMEM_BYTES, done) != 0) return 1;
    uint32_t ranks = 1;
    for (int i = 1; i < 4; ++i)
        if (n_kb >= (2u << i) && int64_t(tiles) * (BN < 128 ? 1 : 2) <= 2 * int64_t(clusters_at_once(kern, 192, Cfg::SMEM_BYTES, 1u << i, held[i])))
            ranks = 1u << i;
    return ranks;
}
// Whether two pairs share a tile's K in the pair kernel: if all tiles are on the GPU at once
template <typename T>
bool q8_pair_split(uint64_t tiles, uint32_t n_kb) {
    static std::atomic<uint64_t> done{0};
    static PerDevice held;
    auto kern = gemm_q8_pair_kernel<true, T>;
    if (n_kb < 8 || allow_smem(kern, PairCfg::SMEM_BYTES, done) != 0) return false;
    return int64_t(tiles) <= clusters_at_once(kern, PairCfg::THREADS, PairCfg::SMEM_BYTES, 4, held);
}

template <int BN, bool SPLIT, typename T>
int launch_q8_thin(cudaStream_t s, const GemmQ8Params& p, const CUtensorMap& ma, const CUtensorMap& mb) {
    using Cfg = ThinCfg<BN, SPLIT>;
    auto kern = gemm_q8_thin_kernel<BN, SPLIT, T>;
    static std::atomic<uint64_t> done{0};
    const int rc = allow_smem(kern, Cfg::SMEM_BYTES, done);
    if (rc != 0) return rc;
    const uint64_t blocks = uint64_t(p.tiles_m) * p.tiles_n * p.ranks;
    if (blocks > 0x7fffffffull) return DECXB200_ETOOLARGE;
    return launch_cluster(kern, unsigned(blocks), 192, Cfg::SMEM_BYTES, p.ranks, s, ma, mb, p);
}

template <int BN, typename T>
int run_q8_thin(cudaStream_t s, GemmQ8Params p, const void* A, uint64_t lda, const void* B, uint64_t ldb) {
    CUtensorMap ma, mb;
    int rc;
    if ((rc = dxb_host::tensor_map_2d(&ma, 1, A, p.M, p.K, lda, Q8_KB, BN)) != 0) return rc;
    if ((rc = dxb_host::tensor_map_2d(&mb, 1, B, p.N, p.K, ldb, Q8_KB, 128)) != 0) return rc;
    p.tiles_m = (p.M + BN - 1) / BN;
    p.tiles_n = (p.N + 127) / 128;
    const uint64_t tiles = uint64_t(p.tiles_m) * p.tiles_n;
    const uint32_t n_kb = (p.K + Q8_KB - 1) / Q8_KB;
    p.ranks = q8_thin_ranks<BN, T>(tiles, n_kb);
    return p.ranks > 1 ? launch_q8_thin<BN, true, T>(s, p, ma, mb) : launch_q8_thin<BN, false, T>(s, p, ma, mb);
}

template <typename T>
int launch_q8_pair(cudaStream_t s, GemmQ8Params p, const void* A, uint64_t lda, const void* B, uint64_t ldb) {
    using Cfg = PairCfg;
    CUtensorMap ma, mb, md, mc;
    int rc;
    if ((rc = dxb_host::tensor_map_2d(&ma, 1, A, p.M, p.K, lda, Q8_KB, 128)) != 0) return rc;
    if ((rc = dxb_host::tensor_map_2d(&mb, 1, B, p.N, p.K, ldb, Q8_KB, 128)) != 0) return rc;
    md = mc = ma;
    const uint64_t e = sizeof(T);
    if (aligned16(p.D) && (p.ldd * e) % 16 == 0 &&
        dxb_host::tensor_map_2d(&md, int(e), p.D, p.M, p.N, p.ldd, uint32_t(64 / e), 32) == 0)
        p.d_tma = 1;
    if (p.d_tma && p.C != nullptr && aligned16(p.C) && (p.ldc * e) % 16 == 0 &&
        dxb_host::tensor_map_2d(&mc, int(e), p.C, p.M, p.N, p.ldc, uint32_t(64 / e), 32) == 0)
        p.c_tma = 1;
    p.tiles_m = uint32_t((uint64_t(p.M) + 255) / 256);
    p.tiles_n = uint32_t((uint64_t(p.N) + 255) / 256);
    const uint64_t tiles = uint64_t(p.tiles_m) * p.tiles_n;
    if (tiles > 0x7fffffffull) return DECXB200_ETOOLARGE;
    p.group_m = p.tiles_m < 8 ? p.tiles_m : 8;
    if (q8_pair_split<T>(tiles, (p.K + Q8_KB - 1) / Q8_KB))
        return launch_cluster(gemm_q8_pair_kernel<true, T>, unsigned(4 * tiles), Cfg::THREADS, Cfg::SMEM_BYTES, 4, s, ma, mb, md, mc, p);
    static std::atomic<uint64_t> done{0};
    auto kern = gemm_q8_pair_kernel<false, T>;
    if ((rc = allow_smem(kern, Cfg::SMEM_BYTES, done)) != 0) return rc;
    uint64_t pairs = uint64_t(sm_count()) / 2;
    if (pairs > tiles) pairs = tiles;
    if (pairs == 0) pairs = 1;
    return launch_cluster(kern, unsigned(2 * pairs), Cfg::THREADS, Cfg::SMEM_BYTES, 2, s, ma, mb, md, mc, p);
}

template <typename T>
int run_gemm_q8(cudaStream_t s, const GemmQ8Params& p, const void* A, uint64_t lda, const void* B, uint64_t ldb, int tile) {
    if (tile == DECXB200_TILE_AUTO) {
        // Clocks of either kernel: turns on the SMs x 128s of K (700 each, measured, for a 256 x 256 tile of a pair as for a
        // 128 x 128 tile of one SM), and what comes after the sums, longer when they are joined.
        tile = DECXB200_TILE_Q8_THIN;
        if (p.M > 128) {
            const uint64_t n_kb = (uint64_t(p.K) + Q8_KB - 1) / Q8_KB;
            const uint64_t tiles = (uint64_t(p.M) + 255) / 256 * ((uint64_t(p.N) + 255) / 256);
            const uint64_t thin_tiles = (uint64_t(p.M) + 127) / 128 * ((uint64_t(p.N) + 127) / 128);
            const uint64_t r = q8_pair_split<T>(tiles, uint32_t(n_kb)) ? 2 : 1, tr = q8_thin_ranks<128, T>(thin_tiles, uint32_t(n_kb));
            const uint64_t sms = uint64_t(sm_count()), pairs = sms > 1 ? sms / 2 : 1;
            const uint64_t pair = (tiles * r + pairs - 1) / pairs * (n_kb / r) * 700 + (r > 1 ? 12000 : 5000);
            const uint64_t thin = (thin_tiles * tr + sms - 1) / sms * (n_kb / tr) * 700 + (tr > 1 ? 8500 : 3000);
            if (pair < thin) tile = DECXB200_TILE_Q8_PAIR;
        }
    }
    if (tile == DECXB200_TILE_Q8_PAIR) return launch_q8_pair<T>(s, p, A, lda, B, ldb);
    if (p.M <= 16) return run_q8_thin<16, T>(s, p, A, lda, B, ldb);
    if (p.M <= 32) return run_q8_thin<32, T>(s, p, A, lda, B, ldb);
    if (p.M <= 64) return run_q8_thin<64, T>(s, p, A, lda, B, ldb);
    return run_q8_thin<128, T>(s, p, A, lda, B, ldb);
}

}  // namespace

extern "C" {

int decxb200_gemm_q8(int d_dtype, void* stream, uint32_t M, uint32_t N, uint32_t K, const void* A, uint64_t lda,
                     const float* a_scales, const void* B, uint64_t ldb, const float* b_scales, const void* C, uint64_t ldc,
                     void* D, uint64_t ldd, const float* alpha, const float* beta, unsigned* status, int tile) {
    dxb_host::reset_launches();
    if (d_dtype != DECXB200_FP16 && d_dtype != DECXB200_FP32) return DECXB200_EINVAL;
    if (A == nullptr || B == nullptr || D == nullptr || a_scales == nullptr || b_scales == nullptr) return DECXB200_EINVAL;
    if (M == 0 || N == 0 || K == 0 || lda < K || ldb < K || ldd < N || (C != nullptr && ldc < N)) return DECXB200_EINVAL;
    if (C == D && ldc != ldd) return DECXB200_EINVAL;         // in place only element by element
    if (tile < DECXB200_TILE_AUTO || tile > DECXB200_TILE_Q8_PAIR) return DECXB200_EINVAL;
    if (M > 0x7fffff00u || N > 0x7fffff00u || K > 0x7fffff00u) return DECXB200_ETOOLARGE;   // TMA coordinates are signed
    if (!aligned16(A) || !aligned16(B) || (lda % 16) != 0 || (ldb % 16) != 0) return DECXB200_EALIGN;
    const uintptr_t e = d_dtype == DECXB200_FP16 ? 2 : 4;
    if ((reinterpret_cast<uintptr_t>(a_scales) & 3) != 0 || (reinterpret_cast<uintptr_t>(b_scales) & 3) != 0 ||
        reinterpret_cast<uintptr_t>(C) % e != 0 || reinterpret_cast<uintptr_t>(D) % e != 0)
        return DECXB200_EALIGN;
    GemmQ8Params p;
    memset(&p, 0, sizeof(p));
    p.M = M; p.N = N; p.K = K;
    p.sa = a_scales; p.sb = b_scales;
    p.alpha = alpha != nullptr ? *alpha : 1.f;
    p.beta = beta != nullptr ? *beta : 0.f;
    p.wide = !q8_ordinary(p.alpha, Q8_ALPHA_REACH);
    p.C = p.beta != 0.f ? C : nullptr;
    p.ldc = ldc;
    p.D = D; p.ldd = ldd;
    p.status = status;
    p.wait_limit_ns = dxb_host::wait_limit_ns();
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return d_dtype == DECXB200_FP16 ? run_gemm_q8<__half>(s, p, A, lda, B, ldb, tile) : run_gemm_q8<float>(s, p, A, lda, B, ldb, tile);
}

int decxb200_gemv_q4(int x_dtype, int y_dtype, void* stream, uint32_t rows, uint32_t cols, uint32_t n_vec, uint32_t group,
                     const void* W, uint64_t ldw, const void* scales, uint64_t ld_scales, const void* zeros,
                     uint64_t ld_zeros, const void* x, uint64_t ldx, const float* x_scales, void* y, uint64_t ldy) {
    dxb_host::reset_launches();
    if ((x_dtype != DECXB200_FP16 && x_dtype != DECXB200_E4M3) || (y_dtype != DECXB200_FP16 && y_dtype != DECXB200_FP32))
        return DECXB200_EINVAL;
    if (W == nullptr || scales == nullptr || x == nullptr || y == nullptr || rows == 0 || cols == 0 || n_vec == 0)
        return DECXB200_EINVAL;
    if (group != 32 && group != 64 && group != 128) return DECXB200_EINVAL;
    const uint64_t groups = (uint64_t(cols) + group - 1) / group;
    if (ldw < (uint64_t(cols) + 1) / 2 || ld_scales < groups || (zeros != nullptr && ld_zeros < groups) || ldx < cols || ldy < rows)
        return DECXB200_EINVAL;
    // columns that 16 CTAs hold; 32-bit offsets within a tile of 32 rows
    if (n_vec > Q4_MAX_VEC || cols > 65536 || rows > 0x7fffff00u || ldw > (1u << 26) || ld_scales > (1u << 26) || ld_zeros > (1u << 26)) return DECXB200_ETOOLARGE;
    if (!aligned16(W) || (ldw % 16) != 0) return DECXB200_EALIGN;
    auto at = [](const void* a, uintptr_t e) { return (reinterpret_cast<uintptr_t>(a) & (e - 1)) == 0; };
    if (!at(scales, 2) || (x_dtype == DECXB200_FP16 && !at(x, 2)) || !at(x_scales, 4) || !at(y, y_dtype == DECXB200_FP32 ? 4 : 2))
        return DECXB200_EALIGN;
    GemvQ4Params p;
    memset(&p, 0, sizeof(p));
    p.W = static_cast<const uint8_t*>(W); p.ldw = ldw;
    p.scales = static_cast<const __half*>(scales); p.lds = ld_scales;
    p.zeros = static_cast<const uint8_t*>(zeros); p.ldz = ld_zeros;
    p.x = x; p.ldx = ldx; p.xs = x_scales;
    p.y = y; p.ldy = ldy;
    p.rows = rows; p.cols = cols; p.n_vec = n_vec;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const bool x8 = x_dtype == DECXB200_E4M3, f32 = y_dtype == DECXB200_FP32;
    if (group == 32) return run_gemv_q4_group<32>(s, x8, f32, p);
    if (group == 64) return run_gemv_q4_group<64>(s, x8, f32, p);
    return run_gemv_q4_group<128>(s, x8, f32, p);
}

int decxb200_cast_q8(int dtype, void* stream, uint32_t rows, uint32_t cols, const void* src, uint64_t lds, void* q,
                     uint64_t ldq, float* scales) {
    dxb_host::reset_launches();
    if (dtype != DECXB200_FP16 && dtype != DECXB200_FP32) return DECXB200_EINVAL;
    if (src == nullptr || q == nullptr || scales == nullptr || rows == 0 || cols == 0 || lds < cols || ldq < cols)
        return DECXB200_EINVAL;
    RowQ8Params p;
    memset(&p, 0, sizeof(p));
    p.x = src; p.ldx = lds;
    p.q = static_cast<uint8_t*>(q); p.ldq = ldq;
    p.scales = scales;
    p.rows = rows; p.cols = cols;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return dtype == DECXB200_FP16 ? run_row_q8<__half, false>(s, p) : run_row_q8<float, false>(s, p);
}

int decxb200_rmsnorm_q8(int dtype, void* stream, uint32_t rows, uint32_t cols, const void* x, uint64_t ldx,
                        const void* residual, uint64_t ldr, void* sum, uint64_t ldsum, const void* weight, float eps,
                        void* q, uint64_t ldq, float* scales) {
    dxb_host::reset_launches();
    if (dtype != DECXB200_FP16 && dtype != DECXB200_FP32) return DECXB200_EINVAL;
    if (x == nullptr || weight == nullptr || q == nullptr || scales == nullptr || rows == 0 || cols == 0 || ldx < cols ||
        ldq < cols || (residual != nullptr && ldr < cols) || (sum != nullptr && ldsum < cols))
        return DECXB200_EINVAL;
    if (residual == nullptr && sum != nullptr) return DECXB200_EINVAL;
    if (sum != nullptr && ((sum == x && ldsum != ldx) || (sum == residual && ldsum != ldr))) return DECXB200_EINVAL;
    if (!std::isnormal(eps) || eps < 0.f) return DECXB200_EINVAL;
    RowQ8Params p;
    memset(&p, 0, sizeof(p));
    p.x = x; p.ldx = ldx;
    p.r = residual; p.ldr = ldr;
    p.sum = sum; p.lds = ldsum;
    p.w = weight;
    p.q = static_cast<uint8_t*>(q); p.ldq = ldq;
    p.scales = scales;
    p.rows = rows; p.cols = cols;
    p.eps = eps;
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return dtype == DECXB200_FP16 ? run_row_q8<__half, true>(s, p) : run_row_q8<float, true>(s, p);
}

}  // extern "C"
