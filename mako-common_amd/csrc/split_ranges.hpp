// The split of a batch's work, laid end to end, into equal ranges: sequence i has len(i) units a segment (its context is
// known on the device only) and `segs` segments.
#pragma once

#include "device.hpp"

namespace mako {

// A value the whole wave holds, in a scalar register.
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane(x); }

// The sum of len(0) .. len(n - 1), 64 sequences at a time.
template <class F>
__device__ __forceinline__ uint32_t sum_of(uint32_t n, uint32_t lane, F len)
{
    uint32_t s = 0;
    for (uint32_t i0 = 0; i0 < n; i0 += 64) {
        uint32_t v = i0 + lane < n ? len(i0 + lane) : 0u;
        #pragma unroll
        for (int o = 32; o > 0; o >>= 1)
            v += __shfl_xor(v, o);
        s += v;
    }
    return s;
}

// The sequence whose segments hold unit x, and its first unit; b = batch when x lies past them all.
template <class F>
__device__ __forceinline__ void seq_of(uint32_t batch, uint32_t x, uint32_t lane, F len, uint32_t segs, uint32_t& b,
                                       uint32_t& first)
{
    uint32_t base = 0;
    for (uint32_t i0 = 0; i0 < batch; i0 += 64) {
        const uint32_t n = i0 + lane < batch ? len(i0 + lane) * segs : 0u;
        uint32_t inc = n;
        #pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t t = __shfl_up(inc, o);
            inc += lane >= (uint32_t)o ? t : 0u;
        }
        const uint64_t hit = __ballot(i0 + lane < batch && x < base + inc);
        if (hit) {
            const uint32_t at = (uint32_t)__builtin_ctzll(hit);
            b = i0 + at;
            first = base + __shfl(inc - n, at);
            return;
        }
        base += __shfl(inc, 63);
    }
    b = batch;
    first = base;
}

// T units cut into n equal ranges: range w starts at floor(w T / n), without a 64-bit division (w r < n^2 fits 32 bits).
struct Ranges {
    uint32_t T, n, q, r;
    __device__ Ranges(uint32_t total, uint32_t ranges) : T(total), n(ranges), q(total / ranges), r(total % ranges) {}
    __device__ __forceinline__ uint32_t start(uint32_t w) const { return w * q + (w * r) / n; }
    // The range that holds unit x < T.
    __device__ __forceinline__ uint32_t of(uint32_t x) const
    {
        uint32_t w = (uint32_t)(((uint64_t)x * n) / T);
        while (w + 1 < n && start(w + 1) <= x)
            ++w;
        while (w > 0 && start(w) > x)
            --w;
        return w;
    }
};

}  // namespace mako
