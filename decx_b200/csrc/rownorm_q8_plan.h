// How many rows the ring kernel of rownorm_q8.cuh keeps in shared memory, and how many of its CTAs an SM then holds.
// Plain C++, so that every shape can be checked without a GPU.
#pragma once
#include <cstdint>

namespace dxb {

constexpr uint32_t Q8_RING_SMEM = 223 * 1024;   // what a CTA's ring may take: allowed once per kernel, and the limit of every plan
constexpr uint32_t Q8_RING_SLOTS = 200 * 1024;  // rows of which two slots take more go another way
constexpr uint32_t Q8_RING_FIXED = 2 * 1024;    // of an SM's 228 KB, what each CTA takes besides its ring (system, static arrays)

// bytes of one row in the ring; `units` 16-byte units per thread.  Unaligned rows have 33 units per warp.
constexpr uint32_t q8_ring_slot(uint32_t threads, bool shift, uint32_t units) { return threads / 32 * (shift ? 33 : 32) * 16 * units; }

struct Q8RingPlan {
    uint32_t depth;                             // rows in the ring, 2 to 4
    uint32_t per_sm;                            // CTAs per SM
};
inline Q8RingPlan q8_ring_plan(uint32_t slot, uint32_t threads, uint32_t regs) {
    auto fits = [&](uint32_t d) { return d * slot > Q8_RING_SMEM ? 0u : (Q8_RING_SMEM + Q8_RING_FIXED) / (d * slot + Q8_RING_FIXED); };
    const uint32_t by_regs = 65536u / ((regs + 7) / 8 * 8 * threads), by_threads = 2048u / threads;
    const uint32_t most = by_regs < by_threads ? by_regs : by_threads;
    Q8RingPlan r{4, 1};
    while (r.depth > 2 && fits(r.depth) < (most ? most : 1u)) --r.depth;       // as many CTAs as registers and threads allow
    while (r.depth < 4 && fits(r.depth) == 1 && fits(r.depth + 1) == 1) ++r.depth;
    r.per_sm = fits(r.depth) < most ? fits(r.depth) : most;
    if (r.per_sm == 0) r.per_sm = 1;
    return r;
}

}  // namespace dxb
