// mx4.cuh -- numbers to codes and back (format: mx4.h)
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace nb {

// two numbers to two codes, the first in the lower four bits: nearest, ties to even, beyond 6 (NaN too) to 6
__device__ __forceinline__ uint32_t codes_of(float lo, float hi) {
    uint32_t r;
    asm("{\n.reg .b8 c;\ncvt.rn.satfinite.e2m1x2.f32 c, %2, %1;\ncvt.u32.u8 %0, c;\n}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}
// what two codes stand for, as fp16: exact
__device__ __forceinline__ __half2 numbers_of(uint32_t byte) {
    uint32_t r;
    asm("{\n.reg .b8 c;\ncvt.u8.u32 c, %1;\ncvt.rn.f16x2.e2m1x2 %0, c;\n}" : "=r"(r) : "r"(byte));
    return *reinterpret_cast<__half2 *>(&r);
}
__device__ __forceinline__ float scale_of(uint32_t e) { return e == 255u ? __uint_as_float(0x7fc00000u) : e == 0u ? __uint_as_float(1u << 22) : __uint_as_float(e << 23); }

// of a group whose largest magnitude has these bits, 2^(f - 127) m with 1 <= m < 2: f - 2, not below 0 (NaN and infinity: 255)
__device__ __forceinline__ uint32_t scale_byte(uint32_t top) { const uint32_t f = top >> 23; return f == 255u ? 255u : f > 2u ? f - 2u : 0u; }
__device__ __forceinline__ float inverse_of(uint32_t e) { return __uint_as_float((254u - min(e, 252u)) << 23); }          // 2^(127 - e): division by a scale is exact

}  // namespace nb
