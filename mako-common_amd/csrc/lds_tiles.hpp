// Device helpers of the kernels that stage K / V tiles raw by LDS DMA and read V^T by transpose reads.
#pragma once

#include "device.hpp"

namespace mako {

// An LDS DMA of 16 bytes a lane: rsrc + voff + soff to LDS m0 + 16 lane.
__device__ __forceinline__ void dma16_at(uint32_t m0, uint32_t voff, uint32_t soff, u32x4 rsrc)
{
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"s"(m0), "v"(voff),
                 "s"(rsrc), "s"(soff)
                 : "memory", "m0");
#pragma clang diagnostic pop
}

// The same as a streaming (non-temporal) load, for bytes that one workgroup reads once.
__device__ __forceinline__ void dma16_nt(uint32_t m0, uint32_t voff, u32x4 rsrc)
{
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds" ::"s"(m0), "v"(voff),
                 "s"(rsrc)
                 : "memory", "m0");
#pragma clang diagnostic pop
}

// A buffer descriptor over `bytes` bytes at base, for dma16_at: rows past them load zeros.
__device__ __forceinline__ u32x4 tile_rsrc(const void* base, uint32_t bytes)
{
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return u32x4{(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, bytes, 0x00020000u};
}

// Where 16-byte chunk c of row s (16-bit heads of D) sits in its LDS row: XORed so that the 16 rows a ds_read_b128 spans start in distinct
// banks (rows of 128 bytes: two fill the 64 banks).
template <int D>
__device__ __forceinline__ uint32_t k_xor(uint32_t s)
{
    return D == 64 ? (s >> 1) & 7u : s & 15u;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// x over lanes l and l ^ 32 (the two halves of a wave hold the two key halves of a row): the larger and the sum,
// both halves getting the same bits. v_permlane32_swap exchanges the upper 32 lanes of its first operand with the
// lower 32 of its second, so with x in both, one holds x of lanes 0-31 in every lane and the other x of lanes 32-63:
// no LDS round trip. The instruction goes through inline asm because this compiler's builtin returns the first
// operand for both results; the s_nop gives the preceding VALU write its wait states.
__device__ __forceinline__ void lane_halves(float x, float& lo, float& hi)
{
    uint32_t a = __builtin_bit_cast(uint32_t, x), b = a;
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
    lo = __builtin_bit_cast(float, a);
    hi = __builtin_bit_cast(float, b);
}
// max(a, b, c) by one v_max3_f32: fmaxf on values the compiler cannot prove canonical (MFMA results) is a
// canonicalising v_max per operand and then the v_max, three instructions for two values.
__device__ __forceinline__ float max3(float a, float b, float c)
{
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

__device__ __forceinline__ float pair_max(float x)
{
    float lo, hi;
    lane_halves(x, lo, hi);
    return max3(lo, hi, -INFINITY);
}
__device__ __forceinline__ float pair_sum(float x)
{
    float lo, hi;
    lane_halves(x, lo, hi);
    return lo + hi;
}

// Four f16 of V^T by a transpose read at LDS byte `at` of this wave's group pattern.
__device__ __forceinline__ s16x4 tr_read(const unsigned char* at)
{
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at));
}

}  // namespace mako
