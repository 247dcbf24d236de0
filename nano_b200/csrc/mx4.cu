// mx4.cu -- rows in microscaled 4-bit floating point: quantised, read back, multiplied, and their C entry points (format: mx4.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "family.h"
#include "mx4.h"
#include "portions.h"

namespace nb {
namespace {

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

// Eight neighbours at p as numbers; `in` of them are the row's, the others zero.  Rows start anywhere: the 16-byte pieces of memory that hold the eight are read, and what is wanted is
// shifted out of them, where all of the pieces lie within the row [first, end); number by number at its ends.
template <typename T>
__device__ __forceinline__ void load8(const T *p, uint32_t in, const T *first, const T *end, float (&x)[8]) {
    constexpr uint32_t W = 8 * sizeof(T) / 4;          // words of eight numbers
    const uintptr_t at = reinterpret_cast<uintptr_t>(p), low = at & ~(uintptr_t)15u;
    const uint32_t shift = (uint32_t)(at & 15u);
    uint32_t w[W];
    if (shift == 0 && in == 8u) {
#pragma unroll
        for (uint32_t i = 0; i < W / 4; i++) { const uint4 v = __ldg(reinterpret_cast<const uint4 *>(p) + i); w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w; }
    } else if (in == 8u && low >= reinterpret_cast<uintptr_t>(first) && low + W * 4u + 16u <= reinterpret_cast<uintptr_t>(end)) {
        uint32_t v[W + 4];
#pragma unroll
        for (uint32_t i = 0; i < W / 4 + 1; i++) { const uint4 q = __ldg(reinterpret_cast<const uint4 *>(low) + i); v[4 * i] = q.x; v[4 * i + 1] = q.y; v[4 * i + 2] = q.z; v[4 * i + 3] = q.w; }
        if (shift & 8u)
#pragma unroll
            for (uint32_t i = 0; i < W + 2; i++) v[i] = v[i + 2];
        if (shift & 4u)
#pragma unroll
            for (uint32_t i = 0; i < W + 1; i++) v[i] = v[i + 1];
#pragma unroll
        for (uint32_t i = 0; i < W; i++) w[i] = sizeof(T) == 2 && (shift & 2u) ? __funnelshift_r(v[i], v[i + 1], 16) : v[i];
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) x[i] = i < in ? Num<T>::widen(p[i]) : 0.0f;
        return;
    }
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) x[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) { const uint16_t h = (uint16_t)(w[i / 2] >> (16 * (i % 2))); x[i] = Num<T>::widen(*reinterpret_cast<const T *>(&h)); }
    }
}

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

// ------------------------------------------------------------------------------------------------
// Quantisation.  Four threads to a group, eight numbers each: the largest magnitude's bits by two exchanges; of a number 2^(f - 127) m, 1 <= m < 2, the scale's byte is f - 2, and division by a
// power of two is exact, so the one rounding is the conversion's.  Bound by memory: a number is read and 17/32 bytes are written, in whole words.
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kThreads = 256;
template <typename T>
__global__ void __launch_bounds__(kThreads) k_mx4_quantize(const Mx4Rows a, const uint32_t per_row, const uint32_t items) {
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    const bool live = i < items;
    const uint32_t row = live ? i / per_row : 0u, q = live ? i % per_row : 0u, k = q * 8u;
    float x[8] = {};
    if (live && k < a.columns) {
        const T *first = static_cast<const T *>(a.x) + (uint64_t)row * a.x_stride;
        load8(first + k, min(8u, a.columns - k), first, first + a.columns, x);
    }
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);          // (NaN above infinity above all others)
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const uint32_t f = top >> 23, e = f == 255u ? 255u : f > 2u ? f - 2u : 0u;
    const float by = __uint_as_float((254u - min(e, 252u)) << 23);          // 2^(127 - e)
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) w |= codes_of(x[2 * j] * by, x[2 * j + 1] * by) << (8 * j);
    if (!live) return;
    *reinterpret_cast<uint32_t *>(a.codes + (uint64_t)row * a.code_stride + q * 4u) = e == 255u ? 0u : w;
    if ((q & 3u) == 0) a.scales[(uint64_t)row * a.scale_stride + (q >> 2)] = (uint8_t)e;
}

// And back, V neighbours to a thread: as many as stores of whole vectors allow for every row
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) k_mx4_read(const Mx4Rows a, const uint32_t per_row, const uint32_t items) {
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= items) return;
    const uint32_t row = i / per_row, k = i % per_row * V;
    const uint8_t *codes = a.codes + (uint64_t)row * a.code_stride + k / 2u;
    const float s = scale_of(a.scales[(uint64_t)row * a.scale_stride + k / kMx4Group]);
    uint32_t w;
    if constexpr (V == 8) w = __ldg(reinterpret_cast<const uint32_t *>(codes));
    else if constexpr (V == 4) w = __ldg(reinterpret_cast<const uint16_t *>(codes));
    else w = V == 2 || k % 2u == 0 ? *codes : *codes >> 4;
    struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Vec { T v[V]; } out;
#pragma unroll
    for (int j = 0; j < V; j += 2) {
        const float2 n = __half22float2(numbers_of(w >> (4 * j)));
        out.v[j] = Num<T>::narrow(n.x * s);
        if constexpr (V > 1) out.v[j + 1] = Num<T>::narrow(n.y * s);
    }
    T *to = static_cast<T *>(a.x) + (uint64_t)row * a.x_stride + k;
    if (k + V <= a.columns) *reinterpret_cast<Vec *>(to) = out;
    else
#pragma unroll
        for (int j = 0; j < V; j++) if (k + j < a.columns) to[j] = out.v[j];
}

// rows in portions whose items are counted in 31 bits
template <typename F>
cudaError_t by_rows(const Mx4Rows &a, uint32_t per_row, F f) {
    if (!a.rows || !a.columns) return cudaSuccess;
    return in_portions(a.rows, std::max(1u, 0x7fffff00u / per_row), [&](uint32_t r0, uint32_t n) {
        Mx4Rows b = a;
        b.rows = n;
        b.codes += (uint64_t)r0 * a.code_stride; b.scales += (uint64_t)r0 * a.scale_stride;
        if (a.type != T_MX4) b.x = static_cast<char *>(a.x) + (uint64_t)r0 * a.x_stride * elem_size(a.type);
        f(b, n * per_row, (n * per_row + kThreads - 1u) / kThreads);
        return cudaGetLastError();
    });
}
template <typename T>
cudaError_t read_launch_t(const Mx4Rows &a, cudaStream_t stream) {
    const uint64_t at = reinterpret_cast<uintptr_t>(a.x) | a.x_stride * sizeof(T);
    auto go = [&](auto k, uint32_t v) {
        const uint32_t per_row = (a.columns + v - 1u) / v;
        return by_rows(a, per_row, [&](const Mx4Rows &b, uint32_t items, uint32_t blocks) { k<<<blocks, kThreads, 0, stream>>>(b, per_row, items); });
    };
    if (at % std::min<uint64_t>(16, 8 * sizeof(T)) == 0) return go(k_mx4_read<T, 8>, 8);
    if (at % (4 * sizeof(T)) == 0) return go(k_mx4_read<T, 4>, 4);
    if (at % (2 * sizeof(T)) == 0) return go(k_mx4_read<T, 2>, 2);
    return go(k_mx4_read<T, 1>, 1);
}

// Rows of codes as a product wants them where a row ends inside a byte: what fills up the last group is zeros.  A group to a thread.
__global__ void __launch_bounds__(kThreads) k_mx4_clean(const Mx4Rows a, const uint8_t *codes, const uint64_t code_stride, const uint8_t *scales, const uint64_t scale_stride, const uint32_t per_row,
                                                        const uint32_t items) {
    const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
    if (i >= items) return;
    const uint32_t row = i / per_row, g = i % per_row, live = min(kMx4Group, a.columns - g * kMx4Group);
    uint4 v = __ldg(reinterpret_cast<const uint4 *>(codes + (uint64_t)row * code_stride) + g);
    auto keep = [&](uint32_t w, uint32_t from) { return live >= from + 8u ? w : live <= from ? 0u : w & ((1u << (4u * (live - from))) - 1u); };
    v = make_uint4(keep(v.x, 0), keep(v.y, 8), keep(v.z, 16), keep(v.w, 24));
    reinterpret_cast<uint4 *>(a.codes + (uint64_t)row * a.code_stride)[g] = v;
    a.scales[(uint64_t)row * a.scale_stride + g] = scales[(uint64_t)row * scale_stride + g];
}

}  // namespace

cudaError_t mx4_quantize_launch(const Mx4Rows &a, cudaStream_t stream) {
    const uint32_t per_row = mx4_groups(a.columns) * 4u;
    return by_rows(a, per_row, [&](const Mx4Rows &b, uint32_t items, uint32_t blocks) {
        if (a.type == T_F32) k_mx4_quantize<float><<<blocks, kThreads, 0, stream>>>(b, per_row, items);
        else if (a.type == T_BF16) k_mx4_quantize<__nv_bfloat16><<<blocks, kThreads, 0, stream>>>(b, per_row, items);
        else k_mx4_quantize<__half><<<blocks, kThreads, 0, stream>>>(b, per_row, items);
    });
}
cudaError_t mx4_read_launch(const Mx4Rows &a, cudaStream_t stream) {
    return a.type == T_F32 ? read_launch_t<float>(a, stream) : a.type == T_BF16 ? read_launch_t<__nv_bfloat16>(a, stream) : read_launch_t<__half>(a, stream);
}
cudaError_t mx4_clean_launch(const Mx4Rows &a, const uint8_t *codes, uint64_t code_stride, const uint8_t *scales, uint64_t scale_stride, cudaStream_t stream) {
    const uint32_t per_row = mx4_groups(a.columns);
    uint32_t r0 = 0;
    return by_rows(a, per_row, [&](const Mx4Rows &b, uint32_t items, uint32_t blocks) {
        k_mx4_clean<<<blocks, kThreads, 0, stream>>>(b, codes + r0 * code_stride, code_stride, scales + r0 * scale_stride, scale_stride, per_row, items);
        r0 += b.rows;
    });
}

}  // namespace nb

using nb::fail;

namespace {
int rows_checked(const nb200_mx4_rows *p, nb::Mx4Rows *a) {
    if (!p) return fail(NB200_EINVAL, "null argument");
    if (p->type > nb::T_F16) return fail(NB200_EINVAL, "rows are fp32, bf16 or fp16 (type %u)", p->type);
    if (p->rows && !p->columns) return fail(NB200_EINVAL, "rows of no numbers");
    if (p->columns > 0x7fffffffu) return fail(NB200_EINVAL, "rows of %u numbers are too long", p->columns);
    if (!p->rows) return 0;
    if (!p->codes || !p->scales || !p->x) return fail(NB200_EINVAL, "null argument");
    const uint64_t groups = nb::mx4_groups(p->columns);
    if (reinterpret_cast<uintptr_t>(p->codes) % 16u || p->code_stride % 16u) return fail(NB200_EINVAL, "codes start and go on in multiples of 16 bytes");
    if (reinterpret_cast<uintptr_t>(p->x) % nb::elem_size(p->type)) return fail(NB200_EINVAL, "numbers are not aligned to their type");
    if (p->rows > 1 && (p->code_stride < groups * 16u || p->scale_stride < groups)) return fail(NB200_EINVAL, "rows of codes or scales overlap");
    *a = nb::Mx4Rows{static_cast<uint8_t *>(p->codes), static_cast<uint8_t *>(p->scales), p->code_stride, p->scale_stride, p->x, p->x_stride, p->type, p->rows, p->columns};
    return 0;
}

// checks the call; *work: bytes of x as it is quantised
int product_checked(const nb200_mx4_product *p, uint64_t *work) {
    if (!p || !work) return fail(NB200_EINVAL, "null argument");
    if (p->x_type > NB200_T_MX4) return fail(NB200_EINVAL, "rows are fp32, bf16, fp16 or in microscaled 4-bit floating point (type %u)", p->x_type);
    if (p->out_type > nb::T_F16) return fail(NB200_EINVAL, "results are fp32, bf16 or fp16 (type %u)", p->out_type);
    if (p->rows > 1u << 30 || p->outputs > 1u << 30 || p->columns > 1u << 30) return fail(NB200_EINVAL, "a product of %u x %u x %u is too large", p->rows, p->outputs, p->columns);
    if (p->experts > 1024u) return fail(NB200_EINVAL, "%u experts: at most 1024", p->experts);
    *work = 0;
    if (!p->rows || !p->outputs) return 0;
    if (!p->columns) return fail(NB200_EINVAL, "rows of no numbers");
    const bool codes = p->x_type == NB200_T_MX4;
    const uint64_t groups = nb::mx4_groups(p->columns), row = groups * 16u;
    if (!p->x || !p->w || !p->w_scales || !p->out || (codes && !p->x_scales) || (p->experts && !p->offsets)) return fail(NB200_EINVAL, "null argument");
    if (reinterpret_cast<uintptr_t>(p->w) % 16u || p->w_stride % 16u || p->w_expert % 16u || (codes && (reinterpret_cast<uintptr_t>(p->x) % 16u || p->x_stride % 16u)))
        return fail(NB200_EINVAL, "codes start and go on in multiples of 16 bytes");
    if (p->w_stride >> 38 || p->w_expert >> 38 || (codes && p->x_stride >> 38)) return fail(NB200_EINVAL, "strides of codes are below 2^38 bytes");
    if ((p->outputs > 1 && p->w_stride < row) || (codes && p->rows > 1 && p->x_stride < row)) return fail(NB200_EINVAL, "rows of codes overlap");
    if (!codes && reinterpret_cast<uintptr_t>(p->x) % nb::elem_size(p->x_type)) return fail(NB200_EINVAL, "numbers are not aligned to their type");
    if (reinterpret_cast<uintptr_t>(p->out) % nb::elem_size(p->out_type)) return fail(NB200_EINVAL, "results are not aligned to their type");
    if (p->rows > 1 && p->out_stride < p->outputs) return fail(NB200_EINVAL, "rows of results overlap");
    if (p->experts && reinterpret_cast<uintptr_t>(p->offsets) % 4u) return fail(NB200_EINVAL, "offsets are not aligned to their type");
    if (!codes || p->columns % 2u) *work = p->rows * (row + groups);
    return 0;
}
}  // namespace

extern "C" {

int nb200_dev_mx4_quantize(const nb200_mx4_rows *rows, void *stream) {
    nb::Mx4Rows a{};
    if (const int r = rows_checked(rows, &a)) return r;
    if (!a.rows) return 0;
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    NB_CK(nb::mx4_quantize_launch(a, static_cast<cudaStream_t>(stream)));
    return 0;
}

int nb200_dev_mx4_read(const nb200_mx4_rows *rows, void *stream) {
    nb::Mx4Rows a{};
    if (const int r = rows_checked(rows, &a)) return r;
    if (!a.rows) return 0;
    if (a.rows > 1 && a.x_stride < a.columns) return fail(NB200_EINVAL, "rows of numbers overlap");
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    NB_CK(nb::mx4_read_launch(a, static_cast<cudaStream_t>(stream)));
    return 0;
}

int nb200_dev_mx4_product_workspace(const nb200_mx4_product *p, uint64_t *bytes) { return product_checked(p, bytes); }

int nb200_dev_mx4_product(const nb200_mx4_product *p, void *workspace, uint64_t workspace_bytes, void *stream) {
    uint64_t need = 0;
    if (const int r = product_checked(p, &need)) return r;
    if (!p->rows || !p->outputs) return 0;
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16u))
        return fail(NB200_EINVAL, "the workspace has %llu bytes, 16-byte aligned: %llu are needed", (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)need);
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    nb::Mx4Product a{static_cast<const uint8_t *>(p->x), static_cast<const uint8_t *>(p->x_scales), static_cast<const uint8_t *>(p->w), static_cast<const uint8_t *>(p->w_scales),
                     p->x_stride, p->xs_stride, p->w_stride, p->ws_stride, p->w_expert, p->ws_expert, p->out, p->out_stride, p->experts ? p->offsets : nullptr,
                     p->out_type, p->rows, p->outputs, p->columns, p->experts};
    if (need) {
        const uint64_t groups = nb::mx4_groups(p->columns);
        uint8_t *codes = static_cast<uint8_t *>(workspace), *scales = codes + p->rows * groups * 16u;
        const nb::Mx4Rows rows{codes, scales, groups * 16u, groups, const_cast<void *>(p->x), p->x_stride, p->x_type, p->rows, p->columns};
        NB_CK(p->x_type == NB200_T_MX4 ? nb::mx4_clean_launch(rows, a.x, a.x_stride, a.xs, a.xs_stride, s) : nb::mx4_quantize_launch(rows, s));
        a.x = codes; a.xs = scales; a.x_stride = groups * 16u; a.xs_stride = groups;
    }
    NB_CK(nb::mx4_tc_launch(a, need != 0, s));
    return 0;
}

}  // extern "C"
