// What the kernels of a cache kept in pages share: a step's new rows, and the checks of its sizes.
#pragma once

#include "device.hpp"

namespace mako {

constexpr uint32_t kNoPage = 0xffffffffu;

// The new rows of sequence b: n of them from row s0 on (nothing past `rows`).
struct NewRows {
    uint32_t s0, n;
};
__device__ __forceinline__ NewRows new_rows(const uint32_t* starts, uint32_t rows, uint32_t b)
{
    if (!starts)
        return {b, b < rows ? 1u : 0u};
    const uint32_t s0 = min(starts[b], rows), s1 = min(starts[b + 1], rows);
    return {s0, s1 > s0 ? s1 - s0 : 0u};
}

inline bool page_size_ok(uint32_t page) { return page >= 64 && page <= 4096 && (page & (page - 1)) == 0; }
inline uint32_t log2_of(uint32_t x) { return 31u - (uint32_t)__builtin_clz(x); }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

}  // namespace mako
