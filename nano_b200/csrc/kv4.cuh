// kv4.cuh -- device code that the kernels of the cache in 4 bits share (kv4.cu: rows of keys and values, single tokens and short portions; kv4_tc.cu: long portions).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include "kv4.h"

namespace nb {
namespace {

__device__ __forceinline__ void pdl_enter4() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

constexpr float kSlack = 3.0f, kCap = 15.0f;          // with s < 2 no weight above 2^15
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 half2_of(uint32_t v) { return *reinterpret_cast<__half2 *>(&v); }
// the codes at bits 0-3 and 16-19 (HIGH: 4-7 and 20-23) of w as c s + m
template <bool HIGH>
__device__ __forceinline__ uint32_t stand_for(uint32_t w, __half2 s, __half2 m) {
    uint32_t x;          // (one instruction with both constants in registers; written in C++ it became two with immediates)
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(w), "r"(HIGH ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
    const __half2 h = half2_of(x);
    const __half2 c = HIGH ? __hfma2(h, __float2half2_rn(0.0625f), __float2half2_rn(-64.0f)) : __hsub2(h, __float2half2_rn(1024.0f));
    return bits(__hfma2(c, s, m));
}
// BYTES (a multiple of 2) bytes of shared memory in words
template <int BYTES>
__device__ __forceinline__ void take(const unsigned char *p, uint32_t (&w)[(BYTES + 3) / 4]) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 16; i++) { const uint4 v = reinterpret_cast<const uint4 *>(p)[i]; w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w; }
    } else if constexpr (BYTES == 8) { const uint2 v = *reinterpret_cast<const uint2 *>(p); w[0] = v.x; w[1] = v.y; }
    else if constexpr (BYTES % 4 == 0) {
#pragma unroll
        for (int i = 0; i < BYTES / 4; i++) w[i] = reinterpret_cast<const uint32_t *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < BYTES / 2; i++) {
            const uint32_t v = reinterpret_cast<const uint16_t *>(p)[i];
            if (i & 1) w[i / 2] |= v << 16; else w[i / 2] = v;
        }
    }
}

// tanh for the soft cap: where |x| < kTanhNear, x times the polynomial of x^2 whose largest relative error there is least (5.5e-7; the special function unit would be the bound);
// else 1 - 2 / (1 + e^2x)
constexpr float kTanhNear = 0.5f, kTanh0 = 0.99999946f, kTanh1 = -0.33326318f, kTanh2 = 0.13190297f, kTanh3 = -0.044402226f;
__device__ __forceinline__ float tanh_near(float x) {
    const float y = x * x;
    return x * fmaf(y, fmaf(y, fmaf(y, kTanh3, kTanh2), kTanh1), kTanh0);
}
__device__ __forceinline__ float tanh_any(float x) { return 1.0f - __fdividef(2.0f, 1.0f + ex2(2.0f * kLog2e * x)); }

__device__ __forceinline__ int first_seen(int pos, uint32_t window, uint32_t block) {
    int f = 0;
    if (window && pos >= (int)window) f = pos - (int)window + 1;
    if (block) f = max(f, pos - (int)((uint32_t)pos % block));
    return f;
}
__device__ __forceinline__ int seq_len(const Kv4Attn &a, uint32_t b) {
    const long long most = (long long)a.width * kKv4Page;
    const long long n = a.lens ? a.lens[b] : (long long)a.pos0 + (a.pos_ptr ? *a.pos_ptr : 0u) + a.T;
    return (int)(n < 0 ? 0 : n < most ? n : most);
}
// what is left to do with a column's sums: the sink, the division, the gate.  l and the values are in units of 2^r; returns the values' factor
__device__ __forceinline__ float last_factor(const Kv4Attn &a, uint32_t t, uint32_t h, float r, float l) {
    if (l == 0.0f) return 0.0f;          // no key in sight (a NaN is no zero)
    float f = 1.0f;
    if (a.sink) {
        const float s = a.sink[h] * kLog2e, top = fmaxf(r, s);
        f = ex2(r - top);
        l = fmaf(l, f, ex2(s - top));
    }
    f /= l;
    if (a.gate) f *= 1.0f / (1.0f + expf(-a.gate[(uint64_t)t * a.ldg + h]));
    return f;
}
__device__ __forceinline__ void store_four(const Kv4Attn &a, uint32_t b, uint32_t t, uint32_t h, uint32_t d, float x0, float x1, float x2, float x3) {
    const uint64_t at = b * a.o_batch + t * a.o_token + h * a.o_head + d;
    if (a.type == T_F32) *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = make_float4(x0, x1, x2, x3);
    else {
        const __nv_bfloat162 u = __floats2bfloat162_rn(x0, x1), v = __floats2bfloat162_rn(x2, x3);
        *reinterpret_cast<uint2 *>(static_cast<__nv_bfloat16 *>(a.out) + at) = make_uint2(*reinterpret_cast<const uint32_t *>(&u), *reinterpret_cast<const uint32_t *>(&v));
    }
}

struct Shape { uint32_t nsplit, tiles, cols, sorted; };          // splits of the keys, blocks along the columns of a head, columns of a block; whether blocks take the longest sequences first

// the sums of a row's splits: values [B][G][tiles][nsplit][columns of a block][D], then (r, l) of each
__device__ __forceinline__ uint64_t part_places(const Kv4Attn &a, const Shape &sh) { return (uint64_t)a.B * a.G * sh.tiles * sh.nsplit * sh.cols; }

}  // namespace
// kv4_tc.cu: rows in blocks of 128, heads of up to 128.  Returns what the launch returned
constexpr uint32_t kKv4TcRows = 128;
cudaError_t kv4_tc_launch(const Kv4Attn &a, uint32_t nsplit, uint32_t tiles, cudaStream_t stream, bool pdl);
}  // namespace nb
