// extern "C" layer, third part: the operators on 8-bit and 4-bit operands.  See include/decx_b200.h for the contracts.
#include <atomic>
#include <cmath>
#include <cstring>

#include "../../include/decx_b200.h"
#include "capi_shared.h"
#include "gemv_q4.cuh"
#include "rownorm_q8.cuh"

using namespace dxb;
using dxb_host::aligned16;
using dxb_host::round_up;

namespace {

inline int last_error() {
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 0 : int(e);
}

template <typename T, bool NORM, bool VEC>
int launch_row_q8(cudaStream_t s, const RowQ8Params& p) {
    if (p.cols <= 1024) {
        // a warp per row: eight rows share a CTA, no barrier
        const unsigned blocks = unsigned((uint64_t(p.rows) + 7) / 8);
        if (p.cols <= 256) row_q8_kernel<T, NORM, true, VEC, 1><<<blocks, 256, 0, s>>>(p);
        else if (p.cols <= 512) row_q8_kernel<T, NORM, true, VEC, 2><<<blocks, 256, 0, s>>>(p);
        else row_q8_kernel<T, NORM, true, VEC, 4><<<blocks, 256, 0, s>>>(p);
    } else {
        const unsigned blocks = p.rows < 0x7fffffffu ? p.rows : 0x7fffffffu;
        const uint32_t chunks = (p.cols + 7) / 8;
        auto threads = [&](uint32_t nch) { return (chunks + 32 * nch - 1) / (32 * nch) * 32; };
        if (p.cols > 8 * 4 * 1024) row_q8_long_kernel<T, NORM><<<blocks, 1024, 0, s>>>(p);
        else if (chunks <= 1024 && p.rows <= 296) row_q8_kernel<T, NORM, false, VEC, 1><<<blocks, threads(1), 0, s>>>(p);
        else if (chunks <= 2048) row_q8_kernel<T, NORM, false, VEC, 2><<<blocks, threads(2), 0, s>>>(p);
        else row_q8_kernel<T, NORM, false, VEC, 4><<<blocks, threads(4), 0, s>>>(p);
    }
    dxb_host::count_launch();
    return last_error();
}

template <typename T, bool NORM>
int run_row_q8(cudaStream_t s, const RowQ8Params& p) {
    const uint64_t e = sizeof(T);
    auto elem = [&](const void* a) { return reinterpret_cast<uintptr_t>(a) % e == 0; };
    if (!elem(p.x) || !elem(p.r) || !elem(p.sum) || !elem(p.w) || (reinterpret_cast<uintptr_t>(p.scales) & 3) != 0)
        return DECXB200_EALIGN;
    const bool vec = aligned16(p.x) && (p.ldx * e) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.q) & 7) == 0 && p.ldq % 8 == 0 &&
                     (p.r == nullptr || (aligned16(p.r) && (p.ldr * e) % 16 == 0)) &&
                     (p.sum == nullptr || (aligned16(p.sum) && (p.lds * e) % 16 == 0)) && aligned16(p.w);
    return vec ? launch_row_q8<T, NORM, true>(s, p) : launch_row_q8<T, NORM, false>(s, p);
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

constexpr uint32_t Q4_MAX_VEC = 16, Q4_MAX_RANKS = 8;

template <int GROUP, int NT, bool ZEROS, bool X8, typename OUT>
int launch_gemv_q4(cudaStream_t s, const GemvQ4Params& p) {
    auto kern = gemv_q4_kernel<GROUP, NT, ZEROS, X8, OUT>;
    static std::atomic<uint64_t> done{0};
    const int rc = allow_smem(kern, 227 * 1024, done);
    if (rc != 0) return rc;
    const uint64_t blocks = (uint64_t(p.rows) + Q4_ROWS - 1) / Q4_ROWS * p.ranks;
    if (blocks > 0x7fffffffull) return DECXB200_ETOOLARGE;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(unsigned(blocks));
    cfg.blockDim = dim3(Q4_THREADS);
    cfg.dynamicSmemBytes = q4_smem_bytes(p.slice, GROUP, NT, p.n_vec, ZEROS);
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.ranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return int(e);
    dxb_host::count_launch();
    return 0;
}

template <int GROUP, int NT, bool ZEROS>
int run_gemv_q4(cudaStream_t s, bool x8, bool f32, const GemvQ4Params& p) {
    if (x8) return f32 ? launch_gemv_q4<GROUP, NT, ZEROS, true, float>(s, p) : launch_gemv_q4<GROUP, NT, ZEROS, true, __half>(s, p);
    return f32 ? launch_gemv_q4<GROUP, NT, ZEROS, false, float>(s, p) : launch_gemv_q4<GROUP, NT, ZEROS, false, __half>(s, p);
}
template <int GROUP>
int run_gemv_q4_group(cudaStream_t s, bool x8, bool f32, const GemvQ4Params& p) {
    const bool z = p.zeros != nullptr;
    if (p.n_vec > 8) return z ? run_gemv_q4<GROUP, 2, true>(s, x8, f32, p) : run_gemv_q4<GROUP, 2, false>(s, x8, f32, p);
    return z ? run_gemv_q4<GROUP, 1, true>(s, x8, f32, p) : run_gemv_q4<GROUP, 1, false>(s, x8, f32, p);
}

}  // namespace

extern "C" {

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
    if (n_vec > Q4_MAX_VEC || cols > 0x7fffffffu || rows > 0x7fffffffu) return DECXB200_ETOOLARGE;
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
    // the longest slice that still gives every SM two CTAs
    const uint64_t row_blocks = (uint64_t(rows) + Q4_ROWS - 1) / Q4_ROWS;
    for (p.slice = 2048; p.slice > 512; p.slice /= 2) {
        const uint64_t n = (uint64_t(cols) + p.slice - 1) / p.slice;
        if (row_blocks * (n < Q4_MAX_RANKS ? n : Q4_MAX_RANKS) >= 296 && q4_smem_bytes(p.slice, group, n_vec > 8 ? 2 : 1, n_vec, zeros != nullptr) <= 112 * 1024) break;
    }
    p.n_slices = (cols + p.slice - 1) / p.slice;
    p.ranks = p.n_slices < Q4_MAX_RANKS ? p.n_slices : Q4_MAX_RANKS;
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
