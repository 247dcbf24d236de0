// pairs.cuh -- two fp32 numbers in one 64-bit register, and the instructions of sm_100 that work on both at once; the largest of three
#pragma once

namespace nb {

typedef unsigned long long pair_t;
__device__ __forceinline__ pair_t pair(float a, float b) { pair_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void unpair(pair_t p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ pair_t fma2(pair_t a, pair_t b, pair_t c) { pair_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ pair_t mul2(pair_t a, pair_t b) { pair_t r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ pair_t add2(pair_t a, pair_t b) { pair_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

}  // namespace nb
