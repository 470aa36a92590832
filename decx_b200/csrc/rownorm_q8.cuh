// Row kernels that write 8-bit operands: a pitched e4m3 matrix q and one fp32 scale per row, value = q * scale[row].
//
//   cast     y = x
//   norm     h = x (+ r);  sum = h rounded to the element type;  y = h * rsqrt(mean(h^2) + eps) * w
//   both     scale = max|y| / 448,  q = e4m3(y / scale)                     (448 = the largest finite e4m3 value)
//
// One pass over the data.  The norm's factor rsqrt(...) is the same for the whole row, so it cancels in y / scale:
//     q = e4m3(h w * 448 / max|h w|),    scale = rsqrt(...) * max|h w| / 448.
// Sum of squares and maximum are therefore found in ONE reduction while the products h w stay in registers.
// The norm sees the 32-bit h, not the rounded sum that is stored.
//
// The maximum is taken over the bit patterns of |h w| as unsigned integers, which orders NaN above infinity above
// every finite value: a row that holds one (or whose sum of squares overflows) gets NaN for its scale and all its q.
#pragma once
#include <cuda_fp16.h>
#include <cstdint>

namespace dxb {

struct RowQ8Params {
    const void* x;
    const void* r;             // nullptr: nothing to add
    void* sum;                 // nullptr: not stored; may be x or r themselves (same pitch)
    const void* w;             // norm only
    uint8_t* q;
    float* scales;
    uint64_t ldx, ldr, lds, ldq;
    uint32_t rows, cols;
    float eps;
};

constexpr float E4M3_MAX = 448.f;

// two fp32 -> two e4m3 bytes (first value in the low byte), nearest even, saturating, NaN stays NaN
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
    uint16_t v;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(v) : "f"(hi), "f"(lo));
    return v;
}

__device__ __forceinline__ float q8_load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float q8_load(const float* p) { return *p; }
__device__ __forceinline__ void q8_store(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void q8_store(float* p, float v) { *p = v; }

// 8 consecutive elements, 16-byte aligned
__device__ __forceinline__ void q8_load8(const __half* p, float (&f)[8]) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __half22float2(h[i]);
        f[2 * i] = a.x;
        f[2 * i + 1] = a.y;
    }
}
__device__ __forceinline__ void q8_load8(const float* p, float (&f)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
    f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}
__device__ __forceinline__ void q8_store8(__half* p, const float (&f)[8]) {
    uint4 u;
    __half2* h = reinterpret_cast<__half2*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = u;
}
__device__ __forceinline__ void q8_store8(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// What the threads of a row found: sum of squares, bits of the largest magnitude.
// WARP: a row belongs to one warp; else to the whole CTA.
template <bool WARP>
__device__ __forceinline__ void q8_reduce(float& ss, uint32_t& top, float* red_ss, uint32_t* red_top) {
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
    top = __reduce_max_sync(0xffffffffu, top);
    if constexpr (!WARP) {
        const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
        if (lane == 0) {
            red_ss[warp] = ss;
            red_top[warp] = top;
        }
        __syncthreads();
        ss = lane < warps ? red_ss[lane] : 0.f;
        top = lane < warps ? red_top[lane] : 0u;
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        top = __reduce_max_sync(0xffffffffu, top);
        __syncthreads();                       // the next row may write red_* again
    }
}

// The row's scale and the two factors with q = e4m3((v * pre) * mul).  `pre` lifts rows of tiny values so that
// 448 / max does not overflow.
template <bool NORM>
__device__ __forceinline__ void q8_factors(const RowQ8Params& p, float ss, uint32_t top, float& scale, float& pre,
                                           float& mul) {
    const float big = __uint_as_float(top);
    const float nan = __uint_as_float(0x7fffffffu);
    const bool bad = top >= 0x7f800000u || (NORM && !(ss <= 3.402823466e38f));
    const float rms = NORM ? rsqrtf(ss / float(p.cols) + p.eps) : 1.f;
    scale = bad ? nan : big * rms / E4M3_MAX;
    pre = big < 1e-30f ? 0x1p100f : 1.f;
    mul = bad ? nan : (top == 0 ? 0.f : E4M3_MAX / (big * pre));
}

// Rows of up to 8 * NCH * (threads of a row) columns: the whole row sits in registers between the reduction and the
// stores.  VEC: a thread owns chunks of 8 consecutive elements (16-byte accesses; every row of every operand 16-byte
// aligned); else single elements a row's thread count apart, which any alignment allows and stays coalesced.
template <typename T, bool NORM, bool WARP, bool VEC, int NCH>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
row_q8_kernel(const RowQ8Params p) {
    __shared__ float red_ss[32];
    __shared__ uint32_t red_top[32];
    const uint32_t tpr = WARP ? 32u : blockDim.x;
    const uint32_t tid = WARP ? (threadIdx.x & 31u) : threadIdx.x;
    const uint32_t row_step = WARP ? gridDim.x * (blockDim.x >> 5) : gridDim.x;
    const T* w = static_cast<const T*>(p.w);
    for (uint32_t row = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x; row < p.rows; row += row_step) {
        const T* x = static_cast<const T*>(p.x) + uint64_t(row) * p.ldx;
        const T* r = p.r != nullptr ? static_cast<const T*>(p.r) + uint64_t(row) * p.ldr : nullptr;
        T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + uint64_t(row) * p.lds : nullptr;
        uint8_t* q = p.q + uint64_t(row) * p.ldq;
        float v[NCH][8];
        float ss = 0.f;
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const uint32_t col = VEC ? (c * tpr + tid) * 8 : c * 8 * tpr + tid;
            if (VEC && col + 8 <= p.cols) {
                q8_load8(x + col, v[c]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t k = col + (VEC ? i : i * tpr);
                    v[c][i] = k < p.cols ? q8_load(x + k) : 0.f;
                }
            }
        }
        if (NORM && r != nullptr) {
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
                const uint32_t col = VEC ? (c * tpr + tid) * 8 : c * 8 * tpr + tid;
                if (VEC && col + 8 <= p.cols) {
                    float a[8];
                    q8_load8(r + col, a);
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[c][i] += a[i];
                    if (sum != nullptr) q8_store8(sum + col, v[c]);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t k = col + (VEC ? i : i * tpr);
                        if (k < p.cols) {
                            v[c][i] += q8_load(r + k);
                            if (sum != nullptr) q8_store(sum + k, v[c][i]);
                        }
                    }
                }
            }
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            if (NORM) {
                const uint32_t col = VEC ? (c * tpr + tid) * 8 : c * 8 * tpr + tid;
                if (VEC && col + 8 <= p.cols) {
                    float a[8];
                    q8_load8(w + col, a);
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        ss = fmaf(v[c][i], v[c][i], ss);
                        v[c][i] *= a[i];
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t k = col + (VEC ? i : i * tpr);
                        if (k < p.cols) {
                            ss = fmaf(v[c][i], v[c][i], ss);
                            v[c][i] *= q8_load(w + k);
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[c][i]) & 0x7fffffffu);
        }
        q8_reduce<WARP>(ss, top, red_ss, red_top);
        float scale, pre, mul;
        q8_factors<NORM>(p, ss, top, scale, pre, mul);
        if (tid == 0) p.scales[row] = scale;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const uint32_t col = VEC ? (c * tpr + tid) * 8 : c * 8 * tpr + tid;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = v[c][i] * pre * mul;
            if (VEC && col + 8 <= p.cols) {
                uint2 o;
                o.x = e4m3x2(v[c][0], v[c][1]) | (e4m3x2(v[c][2], v[c][3]) << 16);
                o.y = e4m3x2(v[c][4], v[c][5]) | (e4m3x2(v[c][6], v[c][7]) << 16);
                *reinterpret_cast<uint2*>(q + col) = o;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t k = col + (VEC ? i : i * tpr);
                    if (k < p.cols) q[k] = uint8_t(e4m3x2(v[c][i], 0.f));
                }
            }
        }
    }
}

// Rows too long for the registers: the row is read twice, the second time mostly from L2.  Nothing is written in the
// first pass and every element is read and written by the same thread in the second, so `sum` may be x or r here too.
template <typename T, bool NORM>
__global__ void __launch_bounds__(1024) row_q8_long_kernel(const RowQ8Params p) {
    __shared__ float red_ss[32];
    __shared__ uint32_t red_top[32];
    const T* w = static_cast<const T*>(p.w);
    for (uint32_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + uint64_t(row) * p.ldx;
        const T* r = p.r != nullptr ? static_cast<const T*>(p.r) + uint64_t(row) * p.ldr : nullptr;
        T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + uint64_t(row) * p.lds : nullptr;
        uint8_t* q = p.q + uint64_t(row) * p.ldq;
        float ss = 0.f;
        uint32_t top = 0;
        for (uint64_t k = threadIdx.x; k < p.cols; k += blockDim.x) {
            float h = q8_load(x + k);
            if (NORM && r != nullptr) h += q8_load(r + k);
            if (NORM) {
                ss = fmaf(h, h, ss);
                h *= q8_load(w + k);
            }
            top = max(top, __float_as_uint(h) & 0x7fffffffu);
        }
        q8_reduce<false>(ss, top, red_ss, red_top);
        float scale, pre, mul;
        q8_factors<NORM>(p, ss, top, scale, pre, mul);
        if (threadIdx.x == 0) p.scales[row] = scale;
        for (uint64_t k = threadIdx.x; k < p.cols; k += blockDim.x) {
            float h = q8_load(x + k);
            if (NORM && r != nullptr) {
                h += q8_load(r + k);
                if (sum != nullptr) q8_store(sum + k, h);
            }
            if (NORM) h *= q8_load(w + k);
            q[k] = uint8_t(e4m3x2(h * pre * mul, 0.f));
        }
    }
}

}  // namespace dxb
