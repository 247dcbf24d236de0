// rows.cuh -- rows of numbers that start anywhere (mx4.cu, experts.cu): neighbours read as whole 16-byte pieces of memory, of which the wanted part is shifted out, and written as whole pieces.  What
// lies beside a row is never written, and read (without being used) only between the first and the last row of its tensor.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

namespace nb {

// n / d and the rest, for n below 2^31: m = ceil(2^(31 + s) / d), 2^(s - 1) < d <= 2^s, is off by less than 2^-31 of 2^(31 + s) / d, so the quotient is never a whole one too large
struct Divider {
    uint32_t d, m, s;
    static Divider of(uint32_t d) {
        uint32_t s = 0;
        while (s < 31u && (1u << s) < d) s++;
        return Divider{d, (uint32_t)(((1ull << (31u + s)) + d - 1u) / d), s};
    }
    __device__ __forceinline__ uint32_t over(uint32_t n) const { return (uint32_t)((uint64_t)n * m >> (31u + s)); }
};

template <typename T> struct Num;
template <> struct Num<float> {
    static __device__ __forceinline__ float widen(float v) { return v; }
    static __device__ __forceinline__ float narrow(float v) { return v; }
};
template <> struct Num<__nv_bfloat16> {
    static __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Num<__half> {
    static __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
};

// W words (a multiple of four) of memory from p on, any number of bytes behind a 16-byte border: whole pieces are read, the one that holds the last word and (of no use where p is on a border)
// the one behind it among them.  No branches, so that several such loads are under way at once
template <uint32_t W, bool BYTES>
__device__ __forceinline__ void load_words(const void *p, uint32_t (&w)[W]) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(p);
    const uint32_t shift = (uint32_t)(at & 15u), bits = BYTES ? (shift & 3u) * 8u : (shift & 2u) * 8u;
    const uint4 *from = reinterpret_cast<const uint4 *>(at & ~(uintptr_t)15u);
    uint32_t v[W + 4];
#pragma unroll
    for (uint32_t i = 0; i < W / 4 + 1; i++) { const uint4 q = __ldg(from + i); v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w; }
#pragma unroll
    for (uint32_t i = 0; i < W + 2; i++) v[i] = shift & 8u ? v[i + 2] : v[i];
#pragma unroll
    for (uint32_t i = 0; i < W + 1; i++) v[i] = shift & 4u ? v[i + 1] : v[i];
#pragma unroll
    for (uint32_t i = 0; i < W; i++) w[i] = __funnelshift_r(v[i], v[i + 1], bits);
}
template <uint32_t W>
__device__ __forceinline__ void load_even(const void *p, uint32_t (&w)[W]) {          // p is on a border
#pragma unroll
    for (uint32_t i = 0; i < W / 4; i++) { const uint4 q = __ldg(static_cast<const uint4 *>(p) + i); w[4 * i] = q.x; w[4 * i + 1] = q.y; w[4 * i + 2] = q.z; w[4 * i + 3] = q.w; }
}
template <int P, typename T, uint32_t W>
__device__ __forceinline__ void widen_words(const uint32_t (&w)[W], float (&x)[P]) {
    static_assert(W * 4 == P * sizeof(T), "P numbers");
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (uint32_t i = 0; i < P; i++) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < P; i++) { const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i % 2))); x[i] = Num<T>::widen(*reinterpret_cast<const T *>(&h)); }
    }
}

// Numbers k .. k + P - 1 (16 or 32 bytes) of the row of n numbers at `first`.  EVEN: rows start on 16-byte borders and n is a multiple of P.  INSIDE: so far from the row's ends (`inside`) that
// every piece read belongs to it, or in a row between the first and the last of its tensor (`between`): numbers outside of the row are anything.  ANY: zeros outside of the row (k may be negative)
enum Where { EVEN, INSIDE, ANY };
template <int P, typename T> __device__ __forceinline__ bool inside(uint32_t n, int k) { constexpr int Q = 16 / (int)sizeof(T); return k >= Q && (uint32_t)(k + P + Q) <= n; }
template <Where WHERE, int P, typename T>
__device__ __forceinline__ void load_row(const T *first, uint32_t n, int k, float (&x)[P]) {
    if constexpr (WHERE == ANY) {
#pragma unroll
        for (int i = 0; i < P; i++) x[i] = k + i >= 0 && (uint32_t)(k + i) < n ? Num<T>::widen(first[k + i]) : 0.0f;
    } else {
        uint32_t w[P * sizeof(T) / 4];
        if constexpr (WHERE == EVEN) load_even(first + k, w); else load_words<P * sizeof(T) / 4, false>(first + k, w);
        widen_words<P, T>(w, x);
    }
}
// The row of n numbers at `first` as pieces of memory of 16 bytes, P numbers each: piece b holds the numbers from piece_at(b) on, the first and the last of them perhaps in part
template <typename T> __device__ __forceinline__ int piece_at(const T *first, uint32_t b) { return (int)(b * (16u / sizeof(T))) - (int)((reinterpret_cast<uintptr_t>(first) & 15u) / sizeof(T)); }
template <typename T> inline uint32_t most_pieces(uint32_t n, bool aligned) { constexpr uint32_t P = 16u / sizeof(T); return aligned ? (n + P - 1u) / P : (n + 2u * P - 2u) / P; }          // of a row that starts anywhere
template <Where WHERE, int P, typename T>
__device__ __forceinline__ void store_piece(T *first, uint32_t n, int k, const float (&x)[P]) {
    static_assert(P * sizeof(T) == 16, "a piece");
    if (WHERE != ANY || (k >= 0 && (uint32_t)k + P <= n)) {
        struct alignas(16) { T v[P]; } out;
#pragma unroll
        for (int i = 0; i < P; i++) out.v[i] = Num<T>::narrow(x[i]);
        *reinterpret_cast<uint4 *>(first + k) = *reinterpret_cast<const uint4 *>(&out);
    } else
#pragma unroll
        for (int i = 0; i < P; i++) if (k + i >= 0 && (uint32_t)(k + i) < n) first[k + i] = Num<T>::narrow(x[i]);
}

// rows at each end of a tensor beside which 32 bytes of it need not lie; all, where rows lie upon one another.  The pieces of a row between them may be read from its first number's to its last's
inline uint32_t margin_rows(uint64_t stride_bytes) { return stride_bytes ? (uint32_t)((31u + stride_bytes) / stride_bytes) : 0xffffffffu; }
__device__ __forceinline__ bool between(uint32_t r, uint32_t rows, uint32_t margin) { return r >= margin && r < rows && rows - r > margin; }
// all rows on 16-byte borders
template <typename T> inline bool on_borders(const void *at, uint64_t stride, uint32_t rows) { return (reinterpret_cast<uintptr_t>(at) | (rows > 1 ? stride * sizeof(T) : 0u)) % 16u == 0; }

}  // namespace nb
