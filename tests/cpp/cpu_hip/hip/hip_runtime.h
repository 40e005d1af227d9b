// HIP kernels run on the CPU, for tests of a kernel's indexing: a source compiled for the host with this header first in
// its include path runs each workgroup's threads as fibers, one workgroup after another. A wave's lanes meet at cross-lane
// operations and a workgroup's threads at barriers; between them a thread runs alone. Only what the kernels tested so use
// is here; the rest of device.hpp's builtins are declared, to compile, and not defined.
#pragma once

#include <stdint.h>
#include <ucontext.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <memory>
#include <vector>

using std::max;
using std::min;

#define __global__
#define __device__
#define __host__
#define __forceinline__ inline __attribute__((always_inline))
#define __launch_bounds__(...)
#define __shared__ static

typedef struct ihipStream_t* hipStream_t;
typedef int hipError_t;
constexpr hipError_t hipSuccess = 0;
struct dim3 {
    uint32_t x, y, z;
    dim3(uint32_t a = 1, uint32_t b = 1, uint32_t c = 1) : x(a), y(b), z(c) {}
};

namespace cpu_hip {

struct Fiber {
    ucontext_t ctx;
    std::unique_ptr<char[]> stack;
    bool done = false;
    int barrier = 0;  // barriers passed or waited at
};
struct Wave {
    uint32_t slot[2][64];
    int arrived = 0, round = 0;
};

inline dim3 thread_idx, block_idx;
inline std::vector<Fiber> fibers;
inline std::vector<Wave> waves;
inline ucontext_t scheduler;
inline Fiber* current = nullptr;
inline const std::function<void()>* body = nullptr;
inline int barriers = 0;  // that every thread has reached

inline void yield() { swapcontext(&current->ctx, &scheduler); }

inline void enter()
{
    (*body)();
    current->done = true;
    yield();
}

inline void sync()
{
    ++current->barrier;
    while (current->barrier > barriers)
        yield();
}

// The 64 lanes' values of x, once all have come.
inline const uint32_t* exchange(uint32_t x)
{
    const uint32_t lane = thread_idx.x & 63u;
    Wave& w = waves[thread_idx.x / 64];
    const int round = w.round;
    w.slot[round & 1][lane] = x;
    if (++w.arrived == 64) {
        w.arrived = 0;
        ++w.round;
    }
    while (w.round == round)
        yield();
    return waves[thread_idx.x / 64].slot[round & 1];
}

inline void launch(dim3 grid, dim3 block, const std::function<void()>& kernel)
{
    body = &kernel;
    fibers.resize(std::max<size_t>(fibers.size(), block.x));
    waves.assign(block.x / 64, Wave{});
    for (uint32_t g = 0; g < grid.x; ++g) {
        block_idx = dim3(g);
        barriers = 0;
        for (uint32_t t = 0; t < block.x; ++t) {
            Fiber& f = fibers[t];
            if (!f.stack)
                f.stack.reset(new char[64 << 10]);
            f.done = false;
            f.barrier = 0;
            getcontext(&f.ctx);
            f.ctx.uc_stack.ss_sp = f.stack.get();
            f.ctx.uc_stack.ss_size = 64 << 10;
            f.ctx.uc_link = &scheduler;
            makecontext(&f.ctx, enter, 0);
        }
        for (bool live = true; live;) {
            live = false;
            for (uint32_t w = 0; w < block.x / 64; ++w)
                for (bool runs = true; runs;) {  // until its lanes wait at the barrier or are done
                    runs = false;
                    for (uint32_t t = 64 * w; t < 64 * w + 64; ++t) {
                        Fiber& f = fibers[t];
                        if (f.done || f.barrier > barriers)
                            continue;
                        runs = live = true;
                        thread_idx = dim3(t);
                        current = &f;
                        swapcontext(&scheduler, &f.ctx);
                    }
                }
            bool all = true;
            for (uint32_t t = 0; t < block.x; ++t)
                all = all && (fibers[t].done || fibers[t].barrier > barriers);
            if (all && live)
                ++barriers;
        }
    }
}

}  // namespace cpu_hip

#define threadIdx cpu_hip::thread_idx
#define blockIdx cpu_hip::block_idx
#define hipLaunchKernelGGL(kernel, grid, block, shared, stream, ...) \
    ((void)(shared), (void)(stream), cpu_hip::launch(grid, block, [&] { kernel(__VA_ARGS__); }))

inline void __syncthreads() { cpu_hip::sync(); }
inline uint64_t __ballot(bool x)
{
    const uint32_t* s = cpu_hip::exchange(x);
    uint64_t m = 0;
    for (int i = 0; i < 64; ++i)
        m |= (uint64_t)(s[i] & 1u) << i;
    return m;
}
inline bool __any(bool x) { return __ballot(x) != 0; }
inline uint32_t atomicAdd(uint32_t* p, uint32_t x)
{
    const uint32_t old = *p;
    *p = old + x;
    return old;
}
float __shfl_xor(float x, int mask);

inline uint32_t __builtin_amdgcn_readfirstlane(uint32_t x) { return cpu_hip::exchange(x)[0]; }
inline uint32_t __builtin_amdgcn_readlane(uint32_t x, uint32_t lane) { return cpu_hip::exchange(x)[lane]; }
inline uint32_t __builtin_amdgcn_mbcnt_lo(uint32_t m, uint32_t add)
{
    const uint32_t lane = threadIdx.x & 63u;
    return add + __builtin_popcount(lane < 32 ? m & ((1u << lane) - 1) : m);
}
inline uint32_t __builtin_amdgcn_mbcnt_hi(uint32_t m, uint32_t add)
{
    const uint32_t lane = threadIdx.x & 63u;
    return add + (lane < 32 ? 0 : __builtin_popcount(m & ((1u << (lane - 32)) - 1)));
}
// row_shr 1-15 within rows of 16 lanes, row_bcast 15 (lane 15 of a row to the next row) and 31 (lane 31 to rows 2 and 3);
// rows outside row_mask, and lanes without a source, keep old.
inline uint32_t __builtin_amdgcn_update_dpp(uint32_t old, uint32_t x, int ctrl, int row_mask, int, bool)
{
    const uint32_t* s = cpu_hip::exchange(x);
    const uint32_t lane = threadIdx.x & 63u, row = lane / 16;
    if (!(row_mask >> row & 1))
        return old;
    if (ctrl > 0x110 && ctrl < 0x120)
        return lane % 16 >= uint32_t(ctrl - 0x110) ? s[lane - (ctrl - 0x110)] : old;
    if (ctrl == 0x142)
        return row ? s[16 * row - 1] : old;
    return row >= 2 ? s[31] : old;
}

typedef struct cpu_hip_rsrc* __amdgpu_buffer_rsrc_t;
__amdgpu_buffer_rsrc_t __builtin_amdgcn_make_buffer_rsrc(void*, short, int, int);
typedef uint32_t cpu_hip_u32x4 __attribute__((ext_vector_type(4)));
typedef float cpu_hip_f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 cpu_hip_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 cpu_hip_f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 cpu_hip_f16x2 __attribute__((ext_vector_type(2)));
cpu_hip_u32x4 __builtin_amdgcn_raw_buffer_load_b128(__amdgpu_buffer_rsrc_t, int, int, int);
cpu_hip_f32x16 __builtin_amdgcn_mfma_f32_32x32x16_bf16(cpu_hip_bf16x8, cpu_hip_bf16x8, cpu_hip_f32x16, int, int, int);
cpu_hip_f32x16 __builtin_amdgcn_mfma_f32_32x32x16_f16(cpu_hip_f16x8, cpu_hip_f16x8, cpu_hip_f32x16, int, int, int);
cpu_hip_f16x2 __builtin_amdgcn_cvt_pkrtz(float, float);
float __builtin_amdgcn_fdot2(cpu_hip_f16x2, cpu_hip_f16x2, float, bool);
inline float __builtin_amdgcn_exp2f(float x) { return std::exp2(x); }
