// mx4.cu -- rows in microscaled 4-bit floating point: quantised, read back, multiplied, and their C entry points (format: mx4.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "family.h"
#include "mx4.cuh"
#include "mx4.h"
#include "portions.h"
#include "rows.cuh"

namespace nb {
namespace {

// ------------------------------------------------------------------------------------------------
// Quantisation.  A thread has 32 bytes of a group (a quarter of its fp32 numbers, half of its 16-bit ones): the largest magnitude's bits by one or two exchanges; of a number 2^(f - 127) m,
// 1 <= m < 2, the scale's byte is f - 2, and division by a power of two is exact, so the one rounding is the conversion's.  Bound by memory: a number is read and 17/32 bytes are written, in
// whole words.
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kThreads = 256;
__device__ __forceinline__ uint8_t *scale_at(const Mx4Rows &a, uint32_t row, uint32_t g) { return a.scales + (uint64_t)row * a.scale_stride + (g >> 4) * a.scale_step + (g & 15u); }
// in the second order the last sixteen are filled up with zeros
__device__ __forceinline__ void fill_scales(const Mx4Rows &a, uint32_t row, uint32_t g, uint32_t groups) {
    if (a.scale_step != 16u && g + 1u == groups) for (uint32_t i = groups; i & 15u; i++) *scale_at(a, row, i) = 0;
}
template <typename T> constexpr uint32_t kEach = 32u / sizeof(T);          // numbers to a thread
template <typename T>
__device__ __forceinline__ void quantise(const Mx4Rows &a, const Divider &per_row, uint32_t items, uint32_t i) {          // by all threads of a warp
    constexpr uint32_t P = kEach<T>, SHARE = kMx4Group / P;          // threads to a group
    const bool live = i < items;
    const uint32_t row = live ? per_row.over(i) : 0u, q = live ? i - row * per_row.d : 0u;
    float x[P] = {};
    if (live) {
        const T *first = static_cast<const T *>(a.x) + (uint64_t)row * a.x_stride;
        const int k = (int)(q * P);
        if ((reinterpret_cast<uintptr_t>(first) & 15u) == 0 && q * P + P <= a.columns) load_row<EVEN>(first, a.columns, k, x);
        else if (inside<P, T>(a.columns, k)) load_row<INSIDE>(first, a.columns, k, x);
        else load_row<ANY>(first, a.columns, k, x);
    }
    uint32_t top = top_bits(x);          // (as whole numbers NaN stands above infinity, above all others)
#pragma unroll
    for (uint32_t s = 1; s < SHARE; s *= 2u) top = max(top, __shfl_xor_sync(0xffffffffu, top, s));
    const uint32_t e = scale_byte(top);
    const float by = inverse_of(e);
#pragma unroll
    for (uint32_t j = 0; j < P; j++) x[j] *= by;
    uint32_t w[P / 8];
#pragma unroll
    for (uint32_t j = 0; j < P / 8; j++) w[j] = codes_of(x + 8 * j);
    if (!live) return;
    uint8_t *to = a.codes + (uint64_t)row * a.code_stride + q * (P / 2u);
    if constexpr (P == 8) *reinterpret_cast<uint32_t *>(to) = e == 255u ? 0u : w[0];
    else *reinterpret_cast<uint2 *>(to) = e == 255u ? make_uint2(0u, 0u) : make_uint2(w[0], w[1]);
    if (q % SHARE == 0) { *scale_at(a, row, q / SHARE) = (uint8_t)e; fill_scales(a, row, q / SHARE, per_row.d / SHARE); }
}
template <typename T>
__global__ void __launch_bounds__(kThreads) k_mx4_quantize(const Mx4Rows a, const Divider per_row, const uint32_t items) { quantise<T>(a, per_row, items, blockIdx.x * kThreads + threadIdx.x); }

// And back, by pieces of 32 bytes of the result, two to a thread, whose loads are under way at once: the codes of a piece's numbers are nibbles of neighbouring words, its scales one or two (of its
// own words and one where rows start on borders of 32 bytes).  8192 rows of 2560 fp32 numbers 15.6 us (6.1 TB/s), 8191 of 2570
// 18.3 (with pieces of 16 bytes 16.2 and 22.4); in bf16 8192 of 2560 7.8, 8191 of 2561 12.3
constexpr uint32_t kReadPieces = 2;
template <typename T, bool BORDERS>
__global__ void __launch_bounds__(kThreads) k_mx4_read(const Mx4Rows a, const Divider per_row, const uint32_t items) {
    constexpr int P = 32 / sizeof(T), W = P / 8, U = (int)kReadPieces;
    const uint32_t groups = (a.columns + kMx4Group - 1u) / kMx4Group, i0 = blockIdx.x * (kThreads * U) + threadIdx.x;
    uint32_t w[U][W + 1], e0[U], e1[U];
    T *first[U];
    int k[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const uint32_t i = i0 + u * kThreads, row = i < items ? per_row.over(i) : 0u;
        first[u] = static_cast<T *>(a.x) + (uint64_t)row * a.x_stride;
        k[u] = i >= items ? 0x7fffffff - P : (int)((i - row * per_row.d) * P) - (BORDERS ? 0 : (int)((reinterpret_cast<uintptr_t>(first[u]) & 31u) / sizeof(T)));
        const uint32_t from = k[u] >= (int)a.columns ? 0u : (uint32_t)max(k[u], 0), at = from / 8u, g = from / kMx4Group;
        const uint8_t *scales = a.scales + (uint64_t)row * a.scale_stride;
        const uint32_t *codes = reinterpret_cast<const uint32_t *>(a.codes + (uint64_t)row * a.code_stride);
        if (BORDERS && W == 2) { const uint2 v = __ldg(reinterpret_cast<const uint2 *>(codes + at)); w[u][0] = v.x; w[u][W - 1] = v.y; }
        else {
#pragma unroll
            for (int j = 0; j < W + (BORDERS ? 0 : 1); j++) w[u][j] = __ldg(codes + min(at + j, groups * 4u - 1u));
        }
        e0[u] = scales[g];
        if (!BORDERS) e1[u] = scales[min((from + P - 1u) / kMx4Group, groups - 1u)];
    }
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (k[u] >= (int)a.columns) continue;
        const uint32_t from = (uint32_t)max(k[u], 0), border = (from / kMx4Group + 1u) * kMx4Group, bits = 4u * (from % 8u);
        uint64_t v = W == 2 ? (uint64_t)w[u][W - 1] << 32 | w[u][0] : w[u][0];
        if (!BORDERS) {
            if (W == 2) v = (uint64_t)__funnelshift_r(w[u][W - 1], w[u][W], bits) << 32 | __funnelshift_r(w[u][0], w[u][W - 1], bits);
            else v = __funnelshift_r(w[u][0], w[u][1], bits);
            if (k[u] < 0) v <<= -4 * k[u];          // (the row's first piece: its numbers are the last of it)
        }
        const float s0 = scale_of(e0[u]), s1 = BORDERS ? s0 : scale_of(e1[u]);
        float x[P];
#pragma unroll
        for (int j = 0; j < P; j += 2) {
            const float2 n = __half22float2(numbers_of((uint32_t)(v >> (4 * j))));
            x[j] = n.x * (BORDERS || k[u] + j < (int)border ? s0 : s1);
            x[j + 1] = n.y * (BORDERS || k[u] + j + 1 < (int)border ? s0 : s1);
        }
        union { uint32_t w[8]; T v[P]; } out;
#pragma unroll
        for (int j = 0; j < P; j++) out.v[j] = Num<T>::narrow(x[j]);
        if (k[u] >= 0 && (uint32_t)k[u] + P <= a.columns) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(first[u] + k[u]), "r"(out.w[0]), "r"(out.w[1]), "r"(out.w[2]), "r"(out.w[3]), "r"(out.w[4]), "r"(out.w[5]), "r"(out.w[6]), "r"(out.w[7]) : "memory");
        } else
#pragma unroll
            for (int h = 0; h < P; h += P / 2) {
                const int kh = k[u] + h;
                if (kh >= 0 && (uint32_t)kh + P / 2 <= a.columns) *reinterpret_cast<uint4 *>(first[u] + kh) = make_uint4(out.w[h / (P / 8)], out.w[h / (P / 8) + 1], out.w[h / (P / 8) + 2], out.w[h / (P / 8) + 3]);
                else
#pragma unroll
                    for (int j = 0; j < P / 2; j++) if (kh + j >= 0 && kh + j < (int)a.columns) first[u][kh + j] = out.v[h + j];
            }
    }
}

// rows in portions whose items are counted in 31 bits
template <typename F>
cudaError_t by_rows(const Mx4Rows &a, uint32_t per_row, F f) {
    if (!a.rows || !a.columns) return cudaSuccess;
    return in_portions(a.rows, std::max(1u, 0x7fffff00u / per_row), [&](uint32_t r0, uint32_t n) {
        Mx4Rows b = a;
        b.rows = n;
        b.codes += (uint64_t)r0 * a.code_stride; b.scales += (uint64_t)r0 * a.scale_stride;
        b.x = static_cast<char *>(a.x) + (uint64_t)r0 * a.x_stride * elem_size(a.type);
        f(b, n * per_row, (n * per_row + kThreads - 1u) / kThreads);
        return cudaGetLastError();
    });
}
template <typename T>
cudaError_t read_launch_t(const Mx4Rows &a, cudaStream_t stream) {
    constexpr uint32_t P = 32u / sizeof(T);
    const bool borders = (reinterpret_cast<uintptr_t>(a.x) | (a.rows > 1 ? a.x_stride * sizeof(T) : 0u)) % 32u == 0;
    const uint32_t per_row = borders ? (a.columns + P - 1u) / P : (a.columns + 2u * P - 2u) / P;
    const Divider by = Divider::of(per_row);
    return by_rows(a, per_row, [&](const Mx4Rows &b, uint32_t items, uint32_t blocks) {
        blocks = (blocks + kReadPieces - 1u) / kReadPieces;
        if (borders) k_mx4_read<T, true><<<blocks, kThreads, 0, stream>>>(b, by, items);
        else k_mx4_read<T, false><<<blocks, kThreads, 0, stream>>>(b, by, items);
    });
}

// ------------------------------------------------------------------------------------------------
// What a product wants made before it, in one launch: its rows quantised (or, where codes end inside a byte, what fills up their last group set to zeros), and scales in the second order: blocks
// [0, first) work on x, the others on the scales of w.
// ------------------------------------------------------------------------------------------------
struct Scales { const uint8_t *from; uint64_t stride, expert; uint8_t *to; uint32_t rows, groups, chunks, unit; };          // of `rows` rows of each expert
__device__ __forceinline__ void second_order(const Scales &a, uint64_t i, uint64_t items) {          // sixteen scales of a row to a thread
    if (i >= items) return;
    const uint32_t row = (uint32_t)(i % a.rows), chunk = (uint32_t)(i / a.rows % a.chunks);
    const uint8_t *from = a.from + i / a.rows / a.chunks * a.expert + (uint64_t)row * a.stride + chunk * 16u;
    const uint32_t in = min(16u, a.groups - chunk * 16u);
    uint32_t w[4] = {};
    if (a.unit == 16u) { const uint4 v = __ldg(reinterpret_cast<const uint4 *>(from)); w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w; }
    else if (a.unit >= 4u)
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) w[j] = j * 4u < in ? __ldg(reinterpret_cast<const uint32_t *>(from) + j) : 0u;
    else
#pragma unroll
        for (uint32_t j = 0; j < 16; j++) w[j / 4] |= (j < in ? (uint32_t)__ldg(from + j) : 0u) << (8u * (j % 4u));
    reinterpret_cast<uint4 *>(a.to)[i] = make_uint4(w[0], w[1], w[2], w[3]);
}
struct Codes { const uint8_t *codes, *scales; uint64_t code_stride, scale_stride; };
// a group to a thread
__device__ __forceinline__ void clean(const Mx4Rows &a, const Codes &from, uint32_t groups, uint32_t items, uint32_t i) {
    if (i >= items) return;
    const uint32_t row = i / groups, g = i % groups, live = min(kMx4Group, a.columns - g * kMx4Group);
    uint4 v = __ldg(reinterpret_cast<const uint4 *>(from.codes + (uint64_t)row * from.code_stride) + g);
    auto keep = [&](uint32_t w, uint32_t at) { return live >= at + 8u ? w : live <= at ? 0u : w & ((1u << (4u * (live - at))) - 1u); };
    v = make_uint4(keep(v.x, 0), keep(v.y, 8), keep(v.z, 16), keep(v.w, 24));
    reinterpret_cast<uint4 *>(a.codes + (uint64_t)row * a.code_stride)[g] = v;
    *scale_at(a, row, g) = from.scales[(uint64_t)row * from.scale_stride + g];
    fill_scales(a, row, g, groups);
}
struct Prepare { Mx4Rows rows; Codes codes; Scales xs, ws; uint64_t x_items, w_items; uint32_t per_row, first; Divider by; };
enum { kOfF32, kOfBf16, kOfF16, kOfCodes, kOfScales };          // what x is: numbers, codes to be cleaned, codes whose scales are put in order
template <int KIND>
__global__ void __launch_bounds__(kThreads) k_mx4_prepare(const __grid_constant__ Prepare a) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");          // the product sets itself up and brings its first weights meanwhile
    if (blockIdx.x >= a.first) { second_order(a.ws, (uint64_t)(blockIdx.x - a.first) * kThreads + threadIdx.x, a.w_items); return; }
    const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    if constexpr (KIND == kOfF32) quantise<float>(a.rows, a.by, (uint32_t)a.x_items, (uint32_t)i);
    else if constexpr (KIND == kOfBf16) quantise<__nv_bfloat16>(a.rows, a.by, (uint32_t)a.x_items, (uint32_t)i);
    else if constexpr (KIND == kOfF16) quantise<__half>(a.rows, a.by, (uint32_t)a.x_items, (uint32_t)i);
    else if constexpr (KIND == kOfCodes) clean(a.rows, a.codes, a.per_row, (uint32_t)a.x_items, (uint32_t)i);
    else second_order(a.xs, i, a.x_items);
}

}  // namespace

cudaError_t mx4_quantize_launch(const Mx4Rows &a, cudaStream_t stream) {
    const uint32_t per_row = mx4_groups(a.columns) * (a.type == T_F32 ? 4u : 2u);
    const Divider by = Divider::of(std::max(1u, per_row));
    return by_rows(a, per_row, [&](const Mx4Rows &b, uint32_t items, uint32_t blocks) {
        if (a.type == T_F32) k_mx4_quantize<float><<<blocks, kThreads, 0, stream>>>(b, by, items);
        else if (a.type == T_BF16) k_mx4_quantize<__nv_bfloat16><<<blocks, kThreads, 0, stream>>>(b, by, items);
        else k_mx4_quantize<__half><<<blocks, kThreads, 0, stream>>>(b, by, items);
    });
}
cudaError_t mx4_read_launch(const Mx4Rows &a, cudaStream_t stream) {
    return a.type == T_F32 ? read_launch_t<float>(a, stream) : a.type == T_BF16 ? read_launch_t<__nv_bfloat16>(a, stream) : read_launch_t<__half>(a, stream);
}
cudaError_t mx4_prepare_launch(const Mx4Product &p, const Mx4Plan &plan, uint8_t *workspace, cudaStream_t stream) {
    const uint32_t groups = mx4_groups(p.columns), chunks = (groups + 15u) / 16u;
    uint8_t *xs = workspace + plan.x_scales_at;
    auto unit = [&](const uint8_t *at, uint64_t stride, uint64_t expert) { const uint64_t all = reinterpret_cast<uintptr_t>(at) | stride | expert | groups; return all % 16u == 0 ? 16u : all % 4u == 0 ? 4u : 1u; };
    Prepare a{};
    a.ws = Scales{p.ws, p.ws_stride, p.ws_expert, workspace + plan.w_scales_at, p.outputs, groups, chunks, unit(p.ws, p.ws_stride, p.ws_expert)};
    a.w_items = plan.w_scales ? (uint64_t)std::max(1u, p.experts) * p.outputs * chunks : 0;
    a.rows = Mx4Rows{workspace, xs, groups * 16ull, plan.x_second ? 16ull : groups, plan.x_second ? p.rows * 16ull : 16ull, const_cast<void *>(p.x), p.x_stride, p.x_type, p.rows, p.columns};
    a.codes = Codes{static_cast<const uint8_t *>(p.x), p.xs, p.x_stride, p.xs_stride};
    a.xs = Scales{p.xs, p.xs_stride, 0, xs, p.rows, groups, chunks, p.x_type == T_MX4 ? unit(p.xs, p.xs_stride, 0) : 1u};
    const uint32_t kind = p.x_type != T_MX4 ? p.x_type : plan.x_codes ? (uint32_t)kOfCodes : (uint32_t)kOfScales;
    a.per_row = kind == kOfF32 ? groups * 4u : kind < kOfCodes ? groups * 2u : kind == kOfCodes ? groups : chunks;
    a.by = Divider::of(a.per_row);
    // x in portions whose items are counted in 31 bits, w's scales with the first
    return in_portions(plan.x_codes || plan.x_scales ? p.rows : 1u, std::max(1u, 0x7fffff00u / a.per_row), [&](uint32_t r0, uint32_t n) {
        Prepare b = a;
        if (plan.x_codes || plan.x_scales) b.x_items = kind == kOfScales ? (uint64_t)p.rows * chunks : (uint64_t)n * a.per_row;
        if (kind == kOfScales && r0) return cudaSuccess;          // (all rows at once: counted in 64 bits)
        if (r0) b.w_items = 0;
        b.rows.rows = n;
        b.rows.codes += r0 * a.rows.code_stride; b.rows.scales += r0 * a.rows.scale_stride;
        if (kind < kOfCodes) b.rows.x = static_cast<char *>(a.rows.x) + r0 * p.x_stride * elem_size(p.x_type);
        else { b.codes.codes += r0 * p.x_stride; if (p.xs) b.codes.scales += r0 * p.xs_stride; }
        b.first = (uint32_t)((b.x_items + kThreads - 1u) / kThreads);
        const uint32_t blocks = b.first + (uint32_t)((b.w_items + kThreads - 1u) / kThreads);
        switch (kind) {
            case kOfF32: k_mx4_prepare<kOfF32><<<blocks, kThreads, 0, stream>>>(b); break;
            case kOfBf16: k_mx4_prepare<kOfBf16><<<blocks, kThreads, 0, stream>>>(b); break;
            case kOfF16: k_mx4_prepare<kOfF16><<<blocks, kThreads, 0, stream>>>(b); break;
            case kOfCodes: k_mx4_prepare<kOfCodes><<<blocks, kThreads, 0, stream>>>(b); break;
            default: k_mx4_prepare<kOfScales><<<blocks, kThreads, 0, stream>>>(b);
        }
        return cudaGetLastError();
    });
}

}  // namespace nb

using nb::fail;

namespace {
int rows_checked(const nb200_mx4_rows *p, nb::Mx4Rows *a) {
    if (!p) return fail(NB200_EINVAL, "null argument");
    if (p->type > nb::T_F16) return fail(NB200_EINVAL, "rows are fp32, bf16 or fp16 (type %u)", p->type);
    if (p->rows && !p->columns) return fail(NB200_EINVAL, "rows of no numbers");
    if (p->columns > 1u << 30) return fail(NB200_EINVAL, "rows of %u numbers are too long", p->columns);
    if (!p->rows) return 0;
    if (!p->codes || !p->scales || !p->x) return fail(NB200_EINVAL, "null argument");
    const uint64_t groups = nb::mx4_groups(p->columns);
    if (reinterpret_cast<uintptr_t>(p->codes) % 16u || (p->rows > 1 && p->code_stride % 16u)) return fail(NB200_EINVAL, "codes start and go on in multiples of 16 bytes");
    if (reinterpret_cast<uintptr_t>(p->x) % nb::elem_size(p->type)) return fail(NB200_EINVAL, "numbers are not aligned to their type");
    if (p->rows > 1 && (p->code_stride < groups * 16u || p->scale_stride < groups)) return fail(NB200_EINVAL, "rows of codes or scales overlap");
    *a = nb::Mx4Rows{static_cast<uint8_t *>(p->codes), static_cast<uint8_t *>(p->scales), p->code_stride, p->scale_stride, 16, p->x, p->x_stride, p->type, p->rows, p->columns};
    return 0;
}

int product_checked(const nb200_mx4_product *p, nb::Mx4Product *a) {
    if (!p) return fail(NB200_EINVAL, "null argument");
    if (p->x_type > NB200_T_MX4) return fail(NB200_EINVAL, "rows are fp32, bf16, fp16 or in microscaled 4-bit floating point (type %u)", p->x_type);
    if (p->out_type > nb::T_F16) return fail(NB200_EINVAL, "results are fp32, bf16 or fp16 (type %u)", p->out_type);
    if (p->rows > 1u << 30 || p->outputs > 1u << 30 || p->columns > 1u << 30) return fail(NB200_EINVAL, "a product of %u x %u x %u is too large", p->rows, p->outputs, p->columns);
    if (p->experts > 1024u) return fail(NB200_EINVAL, "%u experts: at most 1024", p->experts);
    *a = nb::Mx4Product{};
    if (!p->rows || !p->outputs) return 0;
    if (!p->columns) return fail(NB200_EINVAL, "rows of no numbers");
    const bool codes = p->x_type == NB200_T_MX4;
    const uint64_t groups = nb::mx4_groups(p->columns), row = groups * 16u;
    if (!p->x || !p->w || !p->w_scales || !p->out || (codes && !p->x_scales) || (p->experts && !p->offsets)) return fail(NB200_EINVAL, "null argument");
    if (reinterpret_cast<uintptr_t>(p->w) % 16u || (p->outputs > 1 && p->w_stride % 16u) || (p->experts > 1 && p->w_expert % 16u) || (codes && (reinterpret_cast<uintptr_t>(p->x) % 16u || (p->rows > 1 && p->x_stride % 16u))))
        return fail(NB200_EINVAL, "codes start and go on in multiples of 16 bytes");
    if (p->w_stride >> 38 || p->w_expert >> 38 || (codes && p->x_stride >> 38)) return fail(NB200_EINVAL, "strides of codes are below 2^38 bytes");
    if ((p->outputs > 1 && p->w_stride < row) || (codes && p->rows > 1 && p->x_stride < row)) return fail(NB200_EINVAL, "rows of codes overlap");
    if (!codes && reinterpret_cast<uintptr_t>(p->x) % nb::elem_size(p->x_type)) return fail(NB200_EINVAL, "numbers are not aligned to their type");
    if (reinterpret_cast<uintptr_t>(p->out) % nb::elem_size(p->out_type)) return fail(NB200_EINVAL, "results are not aligned to their type");
    if (p->rows > 1 && p->out_stride < p->outputs) return fail(NB200_EINVAL, "rows of results overlap");
    if (p->experts && reinterpret_cast<uintptr_t>(p->offsets) % 4u) return fail(NB200_EINVAL, "offsets are not aligned to their type");
    *a = nb::Mx4Product{p->x, static_cast<const uint8_t *>(p->x_scales), static_cast<const uint8_t *>(p->w), static_cast<const uint8_t *>(p->w_scales), p->x_stride, p->xs_stride, p->w_stride,
                        p->ws_stride, p->w_expert, p->ws_expert, p->out, p->out_stride, p->experts ? p->offsets : nullptr, p->x_type, p->out_type, p->rows, p->outputs, p->columns, p->experts};
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

int nb200_dev_mx4_product_workspace(const nb200_mx4_product *p, uint64_t *bytes) {
    nb::Mx4Product a{};
    if (!bytes) return fail(NB200_EINVAL, "null argument");
    if (const int r = product_checked(p, &a)) return r;
    *bytes = a.rows ? nb::mx4_plan(a).bytes : 0;
    return 0;
}

int nb200_dev_mx4_product(const nb200_mx4_product *p, void *workspace, uint64_t workspace_bytes, void *stream) {
    nb::Mx4Product a{};
    if (const int r = product_checked(p, &a)) return r;
    if (!a.rows) return 0;
    const nb::Mx4Plan plan = nb::mx4_plan(a);
    if (plan.bytes && (!workspace || workspace_bytes < plan.bytes || reinterpret_cast<uintptr_t>(workspace) % 16u))
        return fail(NB200_EINVAL, "the workspace has %llu bytes, 16-byte aligned: %llu are needed", (unsigned long long)(workspace ? workspace_bytes : 0), (unsigned long long)plan.bytes);
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    uint8_t *made = static_cast<uint8_t *>(workspace);
    uint64_t xs_step = 16, ws_step = 16;
    if (plan.bytes) {
        NB_CK(nb::mx4_prepare_launch(a, plan, made, s));
        if (plan.x_codes) { a.x = made; a.x_stride = nb::mx4_groups(a.columns) * 16ull; }
        if (plan.x_scales) { a.xs = made + plan.x_scales_at; a.xs_stride = plan.x_second ? 16 : nb::mx4_groups(a.columns); xs_step = plan.x_second ? a.rows * 16ull : 16; }
        if (plan.w_scales) { a.ws = made + plan.w_scales_at; a.ws_stride = 16; ws_step = a.outputs * 16ull; a.ws_expert = ws_step * ((nb::mx4_groups(a.columns) + 15u) / 16u); }
    }
    NB_CK(nb::mx4_tc_launch(a, plan, xs_step, ws_step, plan.bytes != 0, s));
    return 0;
}

}  // extern "C"
