// The split of a batch's work, laid end to end, into equal ranges: sequence i has len(i) units a segment (its context is
// known on the device only) and `segs` segments.
#pragma once

#include "device.hpp"

namespace mako {

// A value the whole wave holds, in a scalar register.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane(x); }

// The inclusive sum of x over a wave's lanes up to this one, by row shifts and broadcasts.
__device__ __forceinline__ uint32_t scan_lanes(uint32_t x)
{
    x += __builtin_amdgcn_update_dpp(0u, x, 0x111, 0xf, 0xf, false);  // row_shr 1
    x += __builtin_amdgcn_update_dpp(0u, x, 0x112, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x114, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x118, 0xf, 0xf, false);
    x += __builtin_amdgcn_update_dpp(0u, x, 0x142, 0xa, 0xf, false);  // lane 15 of rows 0 and 2 to rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0u, x, 0x143, 0xc, 0xf, false);  // lane 31 to rows 2 and 3
    return x;
}

// T units cut into n equal ranges: range w starts at floor(w T / n), without a 64-bit division (w r < n^2 fits 32 bits).
struct Ranges {
    uint32_t q, r, n;
    Ranges() = default;
    __device__ Ranges(uint32_t T, uint32_t ranges) : q(T / ranges), r(T % ranges), n(ranges) {}
    __device__ __forceinline__ uint32_t start(uint32_t w) const { return w * q + (w * r) / n; }
};

// What a workgroup (or wave) with range `range` of n begins with: its units [x0, x1) (x0 = x1: none), and the sequence b
// whose segments hold x0, their first unit `first` and a segment's length. No range of the n' = min(n, units) is empty. All
// lanes hold the results in scalar registers. Up to 64 sequences are looked up once, a lane each.
struct Place {
    uint32_t x0, x1, b, first, len;
};
template <class F>
__device__ __forceinline__ Place place_of(uint32_t batch, uint32_t segs, uint32_t range, uint32_t n, uint32_t lane, F len)
{
    Place at{0, 0, 0, 0, 0};
    uint32_t total = 0, v = 0, inc = 0;
    for (uint32_t i0 = 0; i0 < batch; i0 += 64) {
        v = i0 + lane < batch ? len(i0 + lane) : 0u;
        inc = scan_lanes(v * segs);
        total += (uint32_t)__builtin_amdgcn_readlane(inc, 63);
    }
    if (range >= min(n, total))
        return at;
    const Ranges rg(total, min(n, total));
    at.x0 = rg.start(range);
    at.x1 = rg.start(range + 1);
    uint32_t base = 0;
    for (uint32_t i0 = 0; i0 < batch; i0 += 64) {
        if (batch > 64) {
            v = i0 + lane < batch ? len(i0 + lane) : 0u;
            inc = scan_lanes(v * segs);
        }
        const uint64_t hit = __ballot(at.x0 < base + inc);
        if (hit) {
            const uint32_t l = (uint32_t)__builtin_ctzll(hit);
            at.b = i0 + l;
            at.len = (uint32_t)__builtin_amdgcn_readlane(v, l);
            at.first = base + (uint32_t)__builtin_amdgcn_readlane(inc, l) - at.len * segs;
            break;
        }
        base += (uint32_t)__builtin_amdgcn_readlane(inc, 63);
    }
    return at;
}

}  // namespace mako
