// mx4.cuh -- numbers to codes and back (format: mx4.h)
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace nb {

// eight numbers to eight codes, the first in the lowest four bits: nearest, ties to even, beyond 6 (NaN too) to 6
__device__ __forceinline__ uint32_t codes_of(const float *x) {
    uint32_t r;
    asm("{\n.reg .b8 a, b, c, d;\ncvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\ncvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\ncvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\ncvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        "mov.b32 %0, {a, b, c, d};\n}" : "=r"(r) : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]), "f"(x[4]), "f"(x[5]), "f"(x[6]), "f"(x[7]));
    return r;
}
// the largest magnitude of three, NaN if one is
__device__ __forceinline__ float top_of(float a, float b, float c) { float r; asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
template <uint32_t N>
__device__ __forceinline__ uint32_t top_bits(const float (&x)[N]) {          // its bits, of N numbers (a multiple of 8)
    float t[4] = {};
#pragma unroll
    for (uint32_t j = 0; j < N; j += 2) t[j / 2 % 4u] = top_of(t[j / 2 % 4u], x[j], x[j + 1]);
    return __float_as_uint(top_of(top_of(t[0], t[1], t[2]), t[3], 0.0f)) & 0x7fffffffu;
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
