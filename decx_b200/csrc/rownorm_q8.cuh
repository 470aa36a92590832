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

#include "sm100_ptx.cuh"

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
    uint32_t depth;            // ring kernel: rows in the ring, 2 to 4
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

// ---- ring kernel -------------------------------------------------------------------------------------------
// Many rows: what limits row_q8_kernel is that a CTA's loads, reduction and stores follow one another (fp16
// cast of 4096 x 16384: 72 us against 31 us of traffic).  Here the CTAs stay, and every thread asks for its own pieces
// of the rows to come with asynchronous copies into its own slots of a ring in shared memory.  Nobody else reads a slot,
// so the ring needs no barrier; the only one per row is the reduction's.
//
// SHIFT: rows of x, r and sum that start anywhere (an odd row length).  A thread then copies the aligned 16-byte units that
// its 8 elements touch and shifts them into place; on the way out the lanes of a warp pass each other what an aligned
// unit of the other side needs.

__device__ __forceinline__ void q8_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// SHIFT: neighbouring threads ask for overlapping units, so these go through L1
__device__ __forceinline__ void q8_async16_l1(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void q8_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest `ahead` groups of this thread have landed
__device__ __forceinline__ void q8_async_wait(uint32_t ahead) {
    if (ahead == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (ahead == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// N words of `s` from byte `o` (below 16; whole words only when WORDS) on
template <bool WORDS, int WS, int N, int S>
__device__ __forceinline__ void q8_pick_at(const uint32_t (&s)[S], uint32_t o, uint32_t (&out)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if constexpr (WORDS) out[i] = s[WS + i];
        else out[i] = __funnelshift_r(s[WS + i], s[WS + i + 1 < S ? WS + i + 1 : S - 1], (o & 2) * 8);
    }
}
template <bool WORDS, int N, int S>
__device__ __forceinline__ void q8_pick(const uint32_t (&s)[S], uint32_t o, uint32_t (&out)[N]) {
    switch (o >> 2) {                                     // the same for a whole row
        case 0: q8_pick_at<WORDS, 0, N, S>(s, o, out); break;
        case 1: q8_pick_at<WORDS, 1, N, S>(s, o, out); break;
        case 2: q8_pick_at<WORDS, 2, N, S>(s, o, out); break;
        default: q8_pick_at<WORDS, 3, N, S>(s, o, out); break;
    }
}

__device__ __forceinline__ void q8_to_floats(const uint32_t (&w)[4], float (&f)[8], __half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = a.x;
        f[2 * i + 1] = a.y;
    }
}
__device__ __forceinline__ void q8_to_floats(const uint32_t (&w)[8], float (&f)[8], float) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
}

// 8 elements per lane, consecutive over the warp, to a row that starts anywhere; every lane has all 8
template <typename T>
__device__ __forceinline__ void q8_store8_shift(T* at, const float (&f)[8], uint32_t lane) {
    constexpr int W = 8 * sizeof(T) / 4;                  // words of a lane
    uint32_t s[W + 4];
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
            s[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) s[i] = __float_as_uint(f[i]);
    }
    const uint32_t o = uint32_t(reinterpret_cast<uintptr_t>(at)) & 15u;
    if (o == 0) {
#pragma unroll
        for (int u = 0; u < W / 4; ++u)
            reinterpret_cast<uint4*>(at)[u] = make_uint4(s[4 * u], s[4 * u + 1], s[4 * u + 2], s[4 * u + 3]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) s[W + i] = __shfl_down_sync(0xffffffffu, s[i], 1);
    const uint32_t d = 16 - o, head = d / sizeof(T);      // the first aligned unit starts this many elements in
    uint32_t out[W];
    q8_pick<sizeof(T) == 4, W, W + 4>(s, d, out);
    uint4* unit = reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(at) + d);
#pragma unroll
    for (int u = 0; u < W / 4; ++u)
        if (lane < 31 || u + 1 < W / 4) unit[u] = make_uint4(out[4 * u], out[4 * u + 1], out[4 * u + 2], out[4 * u + 3]);
    // what lies before the warp's first and behind its last whole unit
    const uint32_t tail = head + 8 * (W / 4 - 1) / (W / 4);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if ((lane == 0 && i < head) || (lane == 31 && i >= tail)) q8_store(at + i, f[i]);
}

template <typename T, bool NORM, bool RES, bool WARP, bool SHIFT, int NCH>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
row_q8_ring_kernel(const RowQ8Params p) {
    extern __shared__ __align__(128) uint8_t q8_ring[];
    __shared__ float red_ss[2][32];
    __shared__ uint32_t red_top[2][32];
    constexpr int U = 8 * sizeof(T) / 16, UL = U + (SHIFT ? 1 : 0);   // 16-byte units of 8 elements, and loaded
    constexpr int UT = UL * (RES ? 2 : 1);
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t tpr = WARP ? 32u : blockDim.x, tid = WARP ? lane : threadIdx.x;
    const uint32_t step = WARP ? gridDim.x * (blockDim.x >> 5) : gridDim.x;
    const uint32_t first = WARP ? blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x;
    const uint32_t unit_step = blockDim.x * 16;                       // a thread's units lie this far apart
    const uint32_t mine = smem_u32(q8_ring) + threadIdx.x * 16;
    const T* const w = static_cast<const T*>(p.w);

    // ask for this thread's pieces of a row
    auto request = [&](uint32_t slot, const T* mat, uint64_t ld, uint64_t row, int u0) {
        const T* const rp = mat + row * ld;
        const uint8_t* const end = reinterpret_cast<const uint8_t*>(rp + p.cols);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const uint32_t col = (c * tpr + tid) * 8;
            if (col >= p.cols) continue;
            const uint8_t* at = reinterpret_cast<const uint8_t*>(rp + col);
            const uint32_t dst = mine + ((slot * NCH + c) * UT + u0) * unit_step;
            if constexpr (SHIFT) {
                const uint32_t o = uint32_t(reinterpret_cast<uintptr_t>(at)) & 15u;
                at -= o;
                if (at < reinterpret_cast<const uint8_t*>(mat)) {     // the matrix itself starts inside this unit
                    T* const own = reinterpret_cast<T*>(q8_ring + (dst - smem_u32(q8_ring)));
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const uint32_t b = o + i * sizeof(T);         // byte within the units, which lie unit_step apart
                        own[(b / 16 * unit_step + b % 16) / sizeof(T)] = col + i < p.cols ? rp[col + i] : T(0.f);
                    }
                    continue;
                }
                if (o == 0) {                                         // nothing of the last unit is needed
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int64_t left = end - (at + u * 16);
                        q8_async16_l1(dst + u * unit_step, left > 0 ? at + u * 16 : at, left >= 16 ? 16u : (left > 0 ? uint32_t(left) : 0u));
                    }
                    continue;
                }
            }
#pragma unroll
            for (int u = 0; u < UL; ++u) {
                const int64_t left = end - (at + u * 16);
                const uint32_t n = left >= 16 ? 16u : (left > 0 ? uint32_t(left) : 0u);
                if constexpr (SHIFT) q8_async16_l1(dst + u * unit_step, n ? at + u * 16 : at, n);
                else q8_async16(dst + u * unit_step, n ? at + u * 16 : at, n);
            }
        }
    };
    auto request_row = [&](uint32_t slot, uint64_t row) {
        if (row < p.rows) {
            request(slot, static_cast<const T*>(p.x), p.ldx, row, 0);
            if constexpr (RES) request(slot, static_cast<const T*>(p.r), p.ldr, row, UL);
        }
        q8_async_commit();
    };
    auto take = [&](uint32_t slot, int c, const T* mat, uint64_t ld, uint64_t row, int u0, float (&f)[8]) {
        const uint32_t src = mine + ((slot * NCH + c) * UT + u0) * unit_step;
        uint32_t s[4 * UL], o4[4 * U];
#pragma unroll
        for (int u = 0; u < UL; ++u) {
            const uint4 v = ld_shared_v4(src + u * unit_step);
            s[4 * u] = v.x; s[4 * u + 1] = v.y; s[4 * u + 2] = v.z; s[4 * u + 3] = v.w;
        }
        if constexpr (SHIFT) {
            q8_pick<sizeof(T) == 4, 4 * U, 4 * UL>(s, uint32_t(reinterpret_cast<uintptr_t>(mat + row * ld)) & 15u, o4);
            q8_to_floats(o4, f, T());
        } else {
            q8_to_floats(s, f, T());
        }
    };

    uint64_t ahead = first;                                           // the next row to ask for
    uint32_t put = 0, get = 0, odd = 0;
    for (uint32_t d = 0; d + 1 < p.depth; ++d, ahead += step) {
        request_row(put, ahead);
        if (++put == p.depth) put = 0;
    }
    for (uint64_t row = first; row < p.rows; row += step, odd ^= 1u) {
        request_row(put, ahead);
        ahead += step;
        if (++put == p.depth) put = 0;
        q8_async_wait(p.depth - 1);
        T* const sum = RES && p.sum != nullptr ? static_cast<T*>(p.sum) + row * p.lds : nullptr;
        uint8_t* const q = p.q + row * p.ldq;
        float v[NCH][8];
        float ss = 0.f, big = 0.f;
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const uint32_t col = (c * tpr + tid) * 8;
            const bool any = col < p.cols, all = col + 8 <= p.cols;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = 0.f;
            if (any) take(get, c, static_cast<const T*>(p.x), p.ldx, row, 0, v[c]);
            if constexpr (RES) {
                float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (any) take(get, c, static_cast<const T*>(p.r), p.ldr, row, UL, a);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] += a[i];
                if (sum != nullptr) {
                    if (SHIFT && (c * tpr + (tid | 31u)) * 8 + 8 <= p.cols) {          // the whole warp has whole pieces
                        q8_store8_shift(sum + col, v[c], lane);
                    } else if (!SHIFT && all) {
                        q8_store8(sum + col, v[c]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (col + i < p.cols) q8_store(sum + col + i, v[c][i]);
                    }
                }
            }
            if constexpr (NORM) {
                float a[8];
                if (all) {
                    q8_load8(w + col, a);
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) a[i] = col + i < p.cols ? q8_load(w + col + i) : 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    ss = fmaf(v[c][i], v[c][i], ss);
                    v[c][i] *= a[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) asm("max.NaN.f32 %0, %0, %1;" : "+f"(big) : "f"(fabsf(v[c][i])));
        }
        if (++get == p.depth) get = 0;
        // ---- the row's sum of squares and largest magnitude (two sets of slots: one barrier a row)
        uint32_t top = __float_as_uint(big);
        if constexpr (NORM) {
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if constexpr (!WARP) {
            const uint32_t wid = threadIdx.x >> 5, warps = blockDim.x >> 5;
            if (lane == 0) {
                red_ss[odd][wid] = ss;
                red_top[odd][wid] = top;
            }
            __syncthreads();
            top = lane < warps ? red_top[odd][lane] : 0u;
            if constexpr (NORM) {
                ss = lane < warps ? red_ss[odd][lane] : 0.f;
#pragma unroll
                for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            }
            top = __reduce_max_sync(0xffffffffu, top);
        }
        float scale, pre, mul;
        q8_factors<NORM>(p, ss, top, scale, pre, mul);
        if (tid == 0) p.scales[row] = scale;
        if (pre != 1.f) {
#pragma unroll
            for (int c = 0; c < NCH; ++c)
#pragma unroll
                for (int i = 0; i < 8; ++i) v[c][i] *= pre;
        }
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const uint32_t col = (c * tpr + tid) * 8;
            uint2 o;
            o.x = e4m3x2(v[c][0] * mul, v[c][1] * mul) | (e4m3x2(v[c][2] * mul, v[c][3] * mul) << 16);
            o.y = e4m3x2(v[c][4] * mul, v[c][5] * mul) | (e4m3x2(v[c][6] * mul, v[c][7] * mul) << 16);
            if (col + 8 <= p.cols) {
                *reinterpret_cast<uint2*>(q + col) = o;
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (col + i < p.cols) q[col + i] = uint8_t((i < 4 ? o.x : o.y) >> (8 * (i & 3)));
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
