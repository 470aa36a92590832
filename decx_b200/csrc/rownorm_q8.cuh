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
// HBM bounds it: (3 e + 1) bytes per element with a residual, e + 1 without (e bytes per element of x), against six or so
// operations.  Measured, share of a copy's 6456 GB/s: cast of 4096 x 16384 fp16 31.1 us, 100 %, in a short run, 33 to 35 in a long
// one under the power limit; norm with a residual of 8192 x 4096 fp16 43.4 us, 84 %, fp32 72.7 us, 93 %; 16384 x 512 fp16
// 11.1 us, 82 %.  Rows that start anywhere are bound by instructions, 83 per element in fp32 where aligned fp16 rows take 26:
// 8192 x 4099 fp16 69 us, 53 %, fp32 107 us, 63 %.  A single row is latency: 1.9 us for 4096 fp16.
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

// NaN or infinity in the row, or a sum of squares beyond fp32
template <bool NORM>
__device__ __forceinline__ bool q8_bad(float ss, uint32_t top) {
    return top >= 0x7f800000u || (NORM && !(ss <= 3.402823466e38f));
}
// The row's scale: for the one thread that stores it.
template <bool NORM>
__device__ __forceinline__ float q8_scale(const RowQ8Params& p, float ss, uint32_t top) {
    const float rms = NORM ? rsqrtf(ss / float(p.cols) + p.eps) : 1.f;
    return q8_bad<NORM>(ss, top) ? __uint_as_float(0x7fffffffu) : __uint_as_float(top) * rms / E4M3_MAX;
}

// What e4m3 rounds is v * pre times mul, 448 / max|v * pre|; `pre` keeps rows of tiny and of huge values where mul does not leave
// the fp32 range.  The norm's values come out of fp32 roundings, and mul's does them no more harm.  The cast's are given, often
// with 11 bits, and may lie half way between two e4m3 neighbours, where mul's rounding, the same for a whole row, took all of
// them to one side: 1700 of the 67 million elements of a 4096 x 16384 fp16 cast did not go to the even neighbour.
// A half-way value m, at most 31/16 of its power of two, is what v * mul rounds to as long as mul's relative error is below
// 2^-24 * 16/31, half a last place of m.  For the one row in four whose mul is not that good, `low` is what it lacks, and the
// quotient is v * mul + v * low, rounded once (division by a divisor known in advance: Brisebarre, Muller and Raina, IEEE Trans.
// Computers 53, 2004).  Both pieces for every row cost 1.4 % of a cast under the power limit.
struct Q8Factors {
    float pre, mul, low;
};
template <bool NORM>
__device__ __forceinline__ Q8Factors q8_factors(float ss, uint32_t top) {
    const float big = __uint_as_float(top), nan = __uint_as_float(0x7fffffffu);
    Q8Factors f;
    f.pre = big < 0x1p-100f ? 0x1p100f : big > 0x1p100f ? 0x1p-100f : 1.f;
    const float d = big * f.pre;
    f.mul = q8_bad<NORM>(ss, top) ? nan : top == 0 ? 0.f : E4M3_MAX / d;
    f.low = 0.f;
    if constexpr (!NORM) {
        const float r = fmaf(-f.mul, d, E4M3_MAX);                   // exact: 448 times mul's relative error
        if (fabsf(r) > E4M3_MAX * 0x1p-24f * 0.515f) f.low = r * f.mul * (1.f / E4M3_MAX);
    }
    return f;
}
__device__ __forceinline__ float q8_quotient(float v, const Q8Factors& f) {
    return f.low == 0.f ? v * f.mul : fmaf(v, f.mul, v * f.low);
}
// two quotients as e4m3 bytes, by paired instructions; LOW: of a row that has a low
template <bool LOW>
__device__ __forceinline__ uint32_t q8_two(float a, float b, const Q8Factors& f) {
    const float2 v = make_float2(a, b), m = make_float2(f.mul, f.mul);
    const float2 t = LOW ? __ffma2_rn(v, m, __fmul2_rn(v, make_float2(f.low, f.low))) : __fmul2_rn(v, m);
    return e4m3x2(t.x, t.y);
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
    const uint64_t row_step = WARP ? uint64_t(gridDim.x) * (blockDim.x >> 5) : gridDim.x;
    griddep_launch();
    griddep_wait();
    const T* w = static_cast<const T*>(p.w);
    for (uint64_t row = WARP ? uint64_t(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5) : blockIdx.x; row < p.rows; row += row_step) {
        const T* x = static_cast<const T*>(p.x) + row * p.ldx;
        const T* r = p.r != nullptr ? static_cast<const T*>(p.r) + row * p.ldr : nullptr;
        T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + row * p.lds : nullptr;
        uint8_t* q = p.q + row * p.ldq;
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
        const Q8Factors f = q8_factors<NORM>(ss, top);
        if (tid == 0) p.scales[row] = q8_scale<NORM>(p, ss, top);
#pragma unroll
        for (int c = 0; c < NCH; ++c) {
            const uint32_t col = VEC ? (c * tpr + tid) * 8 : c * 8 * tpr + tid;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[c][i] = q8_quotient(v[c][i] * f.pre, f);
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
// What limits row_q8_kernel is that a CTA's loads, reduction and stores follow one another (fp16 cast of 4096 x 16384:
// 72 us against 32 here and 31 of traffic).  Here the CTAs stay, and every thread asks for its own 16-byte units of the
// rows to come with asynchronous copies into its own slots of a ring in shared memory.  Nobody else reads a slot, so the
// ring needs no barrier; the only one per row is the reduction's.
//
// SHIFT: rows of x, r and sum that start anywhere (an odd row length).  The warps then copy the aligned units that their
// elements touch (33 for 32 lanes), and the lanes take single elements, 32 neighbours at a time: that reads shared memory
// without bank conflicts and writes whole segments whatever the alignment.  (Units shifted into place in registers and
// passed between lanes took 85 instructions per element, and 180 us for 8192 x 4099 fp32 with a residual; this takes 107.)

__device__ __forceinline__ void q8_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void q8_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the newest `ahead` groups of this thread have landed
__device__ __forceinline__ void q8_async_wait(uint32_t ahead) {
    if (ahead == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (ahead == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// one 16-byte unit as floats and back
__device__ __forceinline__ void q8_unit(const uint32_t (&w)[4], float (&f)[8], __half) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        f[2 * i] = a.x;
        f[2 * i + 1] = a.y;
    }
}
__device__ __forceinline__ void q8_unit(const uint32_t (&w)[4], float (&f)[4], float) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
}
__device__ __forceinline__ void q8_words(const float (&f)[8], uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
}
__device__ __forceinline__ void q8_words(const float (&f)[4], uint32_t* w) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __float_as_uint(f[i]);
}

// the larger of big, |a| and |b|; NaN if one of them is
__device__ __forceinline__ void q8_max3(float& big, float a, float b) {
    asm("max.NaN.abs.f32 %0, %0, %1, %2;" : "+f"(big) : "f"(a), "f"(b));
}

template <typename T, bool NORM, bool RES, bool WARP, bool SHIFT, int NCH>
__global__ void __launch_bounds__(WARP ? 256 : 1024)
row_q8_ring_kernel(const RowQ8Params p) {
    extern __shared__ __align__(128) uint8_t q8_ring[];
    __shared__ float red_ss[2][32];
    __shared__ uint32_t red_top[2][32];
    constexpr int E = 16 / sizeof(T), NC = NCH * 8 / E;               // elements of a unit, units of a thread
    constexpr int MATS = RES ? 2 : 1;
    const uint32_t lane = threadIdx.x & 31u, wid = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const uint32_t tpr = WARP ? 32u : blockDim.x, tid = WARP ? lane : threadIdx.x;
    const uint32_t step = WARP ? gridDim.x * warps : gridDim.x;
    const uint32_t first = WARP ? blockIdx.x * warps + wid : blockIdx.x;
    constexpr uint32_t WARP_BYTES = (SHIFT ? 33 : 32) * 16;           // of one warp's units
    const uint32_t unit_bytes = warps * WARP_BYTES, slot_bytes = unit_bytes * NC * MATS;
    const uint32_t mine = smem_u32(q8_ring) + wid * WARP_BYTES + lane * 16;
    const int32_t row_bytes = int32_t(p.cols * sizeof(T));
    // column of element i of a thread's unit c.  SHIFT: lanes are neighbours, with one element each (fp32) or two (fp16: the
    // pair's q bytes go out together)
    auto column = [&](int c, int i) {
        if (!SHIFT) return (c * tpr + tid) * E + i;
        return (c * tpr + (tid & ~31u)) * E + (E == 4 ? i * 32 + lane : i / 2 * 64 + lane * 2 + i % 2);
    };
    griddep_launch();
    griddep_wait();

    // what stays the same for every row: the thread's first bytes, and its pieces of the weight
    uint32_t w[NORM ? NC : 1][4];
    if constexpr (NORM) {
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const T* const wp = static_cast<const T*>(p.w);
            if (!SHIFT && column(c, E - 1) < p.cols) {
                const uint4 u = *reinterpret_cast<const uint4*>(wp + column(c, 0));
                w[c][0] = u.x; w[c][1] = u.y; w[c][2] = u.z; w[c][3] = u.w;
            } else {
                float a[E];
#pragma unroll
                for (int i = 0; i < E; ++i) a[i] = column(c, i) < p.cols ? q8_load(wp + column(c, i)) : 0.f;
                q8_words(a, w[c]);
            }
        }
    }

    // ask for this thread's units of a row
    const uint8_t* next_x = reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.x) + uint64_t(first) * p.ldx);
    const uint8_t* next_r = RES ? reinterpret_cast<const uint8_t*>(static_cast<const T*>(p.r) + uint64_t(first) * p.ldr) : nullptr;
    auto request = [&](uint32_t dst, const uint8_t* rp, const void* mat) {
        const uint32_t o = SHIFT ? uint32_t(reinterpret_cast<uintptr_t>(rp)) & 15u : 0u;
        const uint8_t* const begin = rp - o;
        if (SHIFT && rp == mat && o != 0) {
            // the matrix itself starts inside its first unit: that one element by element
            if (tid == 0) {
                const T* from = reinterpret_cast<const T*>(rp);
                T* const own = reinterpret_cast<T*>(q8_ring + (dst - smem_u32(q8_ring)) + o);
                for (uint32_t i = 0; i * sizeof(T) + o < 16 && i < p.cols; ++i) own[i] = from[i];
            }
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const uint32_t off = (c * tpr + tid) * 16;
            const int32_t left = row_bytes + int32_t(o) - int32_t(off);
            if (left > 0 && !(SHIFT && off == 0 && rp == mat && o != 0))
                q8_async16(dst + c * unit_bytes, begin + off, left >= 16 ? 16u : uint32_t(left));
            if (SHIFT && lane == 31 && left > 16)                     // the unit behind the warp's last one
                q8_async16(dst + c * unit_bytes + 16, begin + off + 16, left >= 32 ? 16u : uint32_t(left - 16));
        }
    };
    uint64_t ahead = first;                                           // the next row to ask for
    uint32_t put = 0, get = 0, odd = 0;                               // byte offsets of slots
    auto request_row = [&]() {
        if (ahead < p.rows) {
            request(mine + put, next_x, p.x);
            next_x += uint64_t(step) * p.ldx * sizeof(T);
            if constexpr (RES) {
                request(mine + put + NC * unit_bytes, next_r, p.r);
                next_r += uint64_t(step) * p.ldr * sizeof(T);
            }
        }
        q8_async_commit();
        ahead += step;
        put += slot_bytes;
        if (put == p.depth * slot_bytes) put = 0;
    };
    // this thread's elements of its unit at `src` (of a row that starts at byte `o` of its first unit); what lies behind the
    // row's end is not zero
    auto take = [&](uint32_t src, uint32_t o, float (&f)[E]) {
        if constexpr (SHIFT) {
            const T* const at = reinterpret_cast<const T*>(q8_ring + (src - smem_u32(q8_ring)) - lane * 16 + o) + lane * (E / 4);
            if constexpr (E == 4) {
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] = q8_load(at + i * 32);
            } else if ((o & 2) == 0) {                                // the same for a whole row
#pragma unroll
                for (int i = 0; i < E; i += 2) {
                    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(at + i * 32));
                    f[i] = a.x;
                    f[i + 1] = a.y;
                }
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i) f[i] = q8_load(at + i / 2 * 64 + i % 2);
            }
        } else {
            const uint4 v = ld_shared_v4(src);
            const uint32_t u4[4] = {v.x, v.y, v.z, v.w};
            q8_unit(u4, f, T());
        }
    };

    for (uint32_t d = 0; d + 1 < p.depth; ++d) request_row();
    const uint64_t lx = p.ldx * sizeof(T), lr = p.ldr * sizeof(T);
    T* sum = RES && p.sum != nullptr ? static_cast<T*>(p.sum) + uint64_t(first) * p.lds : nullptr;
    uint8_t* q = p.q + uint64_t(first) * p.ldq;
    for (uint64_t row = first; row < p.rows; row += step, odd ^= 1u) {
        if constexpr (SHIFT) __syncwarp();                            // the neighbours have read the slot that is filled now
        request_row();
        q8_async_wait(p.depth - 1);
        if constexpr (SHIFT) __syncwarp();                            // the neighbours' copies have landed, too
        const uint32_t ox = SHIFT ? uint32_t(reinterpret_cast<uintptr_t>(p.x) + row * lx) & 15u : 0u;
        const uint32_t orr = SHIFT && RES ? uint32_t(reinterpret_cast<uintptr_t>(p.r) + row * lr) & 15u : 0u;
        float v[NC][E];
        float ss = 0.f, big = 0.f;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const bool all = column(c, E - 1) < p.cols;               // of this thread (columns grow with i)
            take(mine + get + c * unit_bytes, ox, v[c]);
            if constexpr (RES) {
                float a[E];
                take(mine + get + (NC + c) * unit_bytes, orr, a);
#pragma unroll
                for (int i = 0; i < E; ++i) v[c][i] += a[i];
            }
            if (!all) {
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (column(c, i) >= p.cols) v[c][i] = 0.f;
            }
            if constexpr (RES) {
                if (sum != nullptr) {
                    if (!SHIFT && all) {
                        uint32_t o[4];
                        q8_words(v[c], o);
                        *reinterpret_cast<uint4*>(sum + column(c, 0)) = make_uint4(o[0], o[1], o[2], o[3]);
                    } else if (SHIFT && E == 8 && all && (reinterpret_cast<uintptr_t>(sum) & 2) == 0) {
                        uint32_t o[4];
                        q8_words(v[c], o);
#pragma unroll
                        for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(sum + column(c, 2 * i)) = o[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < E; ++i)
                            if (all || column(c, i) < p.cols) q8_store(sum + column(c, i), v[c][i]);
                    }
                }
            }
            if constexpr (NORM) {
                float a[E];
                q8_unit(w[c], a, T());
#pragma unroll
                for (int i = 0; i < E; ++i) {
                    ss = fmaf(v[c][i], v[c][i], ss);
                    v[c][i] *= a[i];
                }
            }
#pragma unroll
            for (int i = 0; i < E; i += 2) q8_max3(big, v[c][i], v[c][i + 1]);
        }
        get += slot_bytes;
        if (get == p.depth * slot_bytes) get = 0;
        // ---- the row's sum of squares and largest magnitude (two sets of slots: one barrier a row)
        uint32_t top = __float_as_uint(big);
        if constexpr (NORM) {
#pragma unroll
            for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if constexpr (!WARP) {
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
        const Q8Factors f = q8_factors<NORM>(ss, top);
        if (tid == 0) p.scales[row] = q8_scale<NORM>(p, ss, top);
        if (f.pre != 1.f) {
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < E; ++i) v[c][i] *= f.pre;
        }
        auto store = [&](auto two) {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                uint32_t o[E / 4];
#pragma unroll
                for (int i = 0; i < E / 4; ++i)
                    o[i] = two(v[c][4 * i], v[c][4 * i + 1]) | (two(v[c][4 * i + 2], v[c][4 * i + 3]) << 16);
                const bool all = column(c, E - 1) < p.cols;
                if (!SHIFT && all) {
                    if constexpr (E == 8) *reinterpret_cast<uint2*>(q + column(c, 0)) = make_uint2(o[0], o[1]);
                    else *reinterpret_cast<uint32_t*>(q + column(c, 0)) = o[0];
                } else if (SHIFT && E == 8 && all) {
#pragma unroll
                    for (int i = 0; i < E; i += 2) *reinterpret_cast<uint16_t*>(q + column(c, i)) = uint16_t(o[i / 4] >> (8 * (i & 3)));
                } else {
#pragma unroll
                    for (int i = 0; i < E; ++i)
                        if (all || column(c, i) < p.cols) q[column(c, i)] = uint8_t(o[i / 4] >> (8 * (i & 3)));
                }
            }
        };
        if (NORM || f.low == 0.f) store([&](float a, float b) { return q8_two<false>(a, b, f); });
        else store([&](float a, float b) { return q8_two<true>(a, b, f); });
        q += uint64_t(step) * p.ldq;
        if (RES && sum != nullptr) sum += uint64_t(step) * p.lds;
    }
}

// Rows too long for the registers: the row is read twice, the second time mostly from L2.  Nothing is written in the
// first pass and every element is read and written by the same thread in the second, so `sum` may be x or r here too.
template <typename T, bool NORM>
__global__ void __launch_bounds__(1024) row_q8_long_kernel(const RowQ8Params p) {
    __shared__ float red_ss[32];
    __shared__ uint32_t red_top[32];
    const T* w = static_cast<const T*>(p.w);
    griddep_launch();
    griddep_wait();
    for (uint64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const T* x = static_cast<const T*>(p.x) + row * p.ldx;
        const T* r = p.r != nullptr ? static_cast<const T*>(p.r) + row * p.ldr : nullptr;
        T* sum = p.sum != nullptr ? static_cast<T*>(p.sum) + row * p.lds : nullptr;
        uint8_t* q = p.q + row * p.ldq;
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
        const Q8Factors f = q8_factors<NORM>(ss, top);
        if (threadIdx.x == 0) p.scales[row] = q8_scale<NORM>(p, ss, top);
        for (uint64_t k = threadIdx.x; k < p.cols; k += blockDim.x) {
            float h = q8_load(x + k);
            if (NORM && r != nullptr) {
                h += q8_load(r + k);
                if (sum != nullptr) q8_store(sum + k, h);
            }
            if (NORM) h *= q8_load(w + k);
            q[k] = uint8_t(e4m3x2(q8_quotient(h * f.pre, f), 0.f));
        }
    }
}

}  // namespace dxb
