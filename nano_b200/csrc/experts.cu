// experts.cu -- rows of tokens sorted by expert and back, with their weights and gradients, and their C entry points.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "family.h"
#include "ops.h"
#include "portions.h"

namespace nb {
namespace {

// ------------------------------------------------------------------------------------------------
// Sorting places by expert: counts, their running sums, and a second walk that hands out the places in order.  A warp owns a run of neighbouring places and a row of counts in shared memory, a
// block the runs of its warps, a cluster of up to eight blocks the list: sums run over experts, then blocks, then warps, so the result is the stable one whatever the order of arrival, in one
// launch without a workspace.  Within 32 places __match_any_sync gives a place its rank.  Bound by the walks' latency: 2 x places / (32 warps) rounds of some 100 cycles.
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortCluster = 8, kMaxExperts = 1024;

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t peer_u32(const uint32_t *mine, uint32_t rank) {
    uint32_t there, v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"((uint32_t)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(there) : "memory");
    return v;
}

struct SortArgs { const void *ids; int32_t *order, *offsets, *place; uint32_t wide, n, experts; };

__global__ void __launch_bounds__(kSortThreads) k_experts_sort(const SortArgs a, const uint32_t C) {
    extern __shared__ uint32_t counts[];          // [warps][experts], then the block's sums [experts] and where its runs begin [experts]
    __shared__ uint32_t sums[kSortWarps];
    const uint32_t E = a.experts, tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, rank = C > 1 ? cluster_rank() : 0u;
    uint32_t *mine = counts + warp * E, *block = counts + kSortWarps * E, *begin = block + E;
    for (uint32_t i = tid; i < kSortWarps * E; i += kSortThreads) counts[i] = 0;
    // runs of whole 32 places, as even as that allows
    const uint32_t pieces = (a.n + 31u) / 32u, runs = C * kSortWarps, per = (pieces + runs - 1u) / runs;
    const uint32_t p0 = min(pieces, (rank * kSortWarps + warp) * per), p1 = min(pieces, p0 + per);
    auto expert = [&](uint32_t i) {          // E: none
        if (i >= a.n) return E;
        const long long id = a.wide ? static_cast<const long long *>(a.ids)[i] : (long long)static_cast<const int *>(a.ids)[i];
        return id >= 0 && id < (long long)E ? (uint32_t)id : E;
    };
    __syncthreads();
    for (uint32_t p = p0; p < p1; p++) {
        const uint32_t e = expert(p * 32u + lane), same = __match_any_sync(0xffffffffu, e);
        if (e < E && lane == (uint32_t)__ffs(same) - 1u) mine[e] += __popc(same);
        __syncwarp();
    }
    __syncthreads();
    for (uint32_t e = tid; e < E; e += kSortThreads) {
        uint32_t run = 0;
        for (uint32_t w = 0; w < kSortWarps; w++) { const uint32_t c = counts[w * E + e]; counts[w * E + e] = run; run += c; }
        block[e] = run;
    }
    if (C > 1) cluster_sync(); else __syncthreads();
    uint32_t all = 0, before = 0;          // of expert tid: in the whole list, in the blocks before this one
    if (tid < E)
        for (uint32_t c = 0; c < C; c++) { const uint32_t x = C > 1 ? peer_u32(block + tid, c) : block[tid]; all += x; before += c < rank ? x : 0u; }
    uint32_t up = all;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, up, o); up += lane >= o ? x : 0u; }
    if (lane == 31u) sums[warp] = up;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = sums[lane];
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, s, o); s += lane >= o ? x : 0u; }
        sums[lane] = s;
    }
    __syncthreads();
    const uint32_t from = up - all + (warp ? sums[warp - 1u] : 0u), known = sums[kSortWarps - 1u];
    if (tid < E) {
        begin[tid] = from + before;
        if (rank == 0) { a.offsets[tid] = (int32_t)from; if (tid == E - 1u) a.offsets[E] = (int32_t)known; }
    }
    __syncthreads();
    for (uint32_t p = p0; p < p1; p++) {
        const uint32_t i = p * 32u + lane, e = expert(i), same = __match_any_sync(0xffffffffu, e);
        uint32_t at = 0;
        if (e < E) at = begin[e] + mine[e] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (e < E && lane == (uint32_t)__ffs(same) - 1u) mine[e] += __popc(same);
        __syncwarp();
        if (i < a.n) a.place[i] = e < E ? (int32_t)at : -1;
        if (e < E) a.order[at] = (int32_t)i;
    }
    for (uint64_t r = known + (uint64_t)rank * kSortThreads + tid; r < a.n; r += C * kSortThreads) a.order[r] = -1;
    if (C > 1) cluster_sync();          // nobody leaves while its shared memory is read
}

// ------------------------------------------------------------------------------------------------
// Rows to their places.  Pure movement, bound by memory: units of U bytes, the widest that every row's start and length allow, two to a thread.
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kMoveThreads = 256, kMoveUnits = 2;
struct GatherArgs { char *out; const char *x; const int32_t *order; uint64_t out_stride, x_stride; uint32_t units, top, tokens; };
template <int U> struct Unit;
template <> struct Unit<16> { typedef uint4 T; };
template <> struct Unit<8> { typedef uint2 T; };
template <> struct Unit<4> { typedef uint32_t T; };
template <> struct Unit<2> { typedef uint16_t T; };
template <> struct Unit<1> { typedef uint8_t T; };

template <int U>
__global__ void __launch_bounds__(kMoveThreads) k_experts_gather(const GatherArgs a, const uint32_t items) {
    typedef typename Unit<U>::T T;
    T v[kMoveUnits] = {};
    const uint32_t i0 = blockIdx.x * kMoveThreads * kMoveUnits + threadIdx.x;
#pragma unroll
    for (uint32_t j = 0; j < kMoveUnits; j++) {
        const uint32_t i = i0 + j * kMoveThreads;
        if (i >= items) break;
        const int32_t o = a.order[i / a.units];
        const uint32_t t = (uint32_t)o / a.top;
        if (o >= 0 && t < a.tokens) v[j] = __ldg(reinterpret_cast<const T *>(a.x + t * a.x_stride) + i % a.units);
    }
#pragma unroll
    for (uint32_t j = 0; j < kMoveUnits; j++) {
        const uint32_t i = i0 + j * kMoveThreads;
        if (i >= items) break;
        reinterpret_cast<T *>(a.out + (uint64_t)(i / a.units) * a.out_stride)[i % a.units] = v[j];
    }
}

// ------------------------------------------------------------------------------------------------
// And back.  V neighbours of a token's row to a thread, which adds up the rows of its experts in fp32, in the list's order; the gradient by rows of the sorted list, a warp to each, which reads
// the token's gradient (the other experts of the token find it in L2) and its own row once.  Both bound by memory.
// ------------------------------------------------------------------------------------------------
struct CombineArgs {
    void *out; const void *y; const float *weights; const int32_t *place, *order; uint64_t out_stride, y_stride; uint32_t tokens, top, rows, columns;
    const void *grad; void *dy; float *dweights; uint64_t grad_stride, dy_stride;
};
template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen(float v) { return v; }
template <> __device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow(float v) { return __float2half_rn(v); }
template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };

template <typename T, int V>
__global__ void __launch_bounds__(kMoveThreads) k_experts_combine(const CombineArgs a, const uint32_t per_row, const uint32_t items) {
    const uint32_t i = blockIdx.x * kMoveThreads + threadIdx.x;
    if (i >= items) return;
    const uint32_t t = i / per_row, c = i % per_row * V;
    const uint64_t first = (uint64_t)t * a.top;
    float sum[V] = {};
#pragma unroll 4
    for (uint32_t j = 0; j < a.top; j++) {
        const uint32_t r = (uint32_t)a.place[first + j];          // (-1: beyond all rows)
        const float w = a.weights ? a.weights[first + j] : 1.0f;
        if (r < a.rows) {
            const Vec<T, V> y = *reinterpret_cast<const Vec<T, V> *>(static_cast<const T *>(a.y) + r * a.y_stride + c);
#pragma unroll
            for (int k = 0; k < V; k++) sum[k] = fmaf(w, widen(y.v[k]), sum[k]);
        }
    }
    Vec<T, V> out;
#pragma unroll
    for (int k = 0; k < V; k++) out.v[k] = narrow<T>(sum[k]);
    *reinterpret_cast<Vec<T, V> *>(static_cast<T *>(a.out) + t * a.out_stride + c) = out;
}

template <typename T, int V>
__global__ void __launch_bounds__(kMoveThreads) k_experts_combine_grad(const CombineArgs a, const uint32_t n) {
    const uint32_t r = blockIdx.x * (kMoveThreads / 32u) + threadIdx.x / 32u, lane = threadIdx.x & 31u;
    if (a.dweights && r < n && lane == 0 && (uint32_t)a.place[r] >= a.rows) a.dweights[r] = 0.0f;          // of place r of the list
    if (r >= a.rows) return;
    const uint32_t o = (uint32_t)a.order[r], t = o / a.top;
    const bool known = o < n;
    const float w = known && a.weights ? a.weights[o] : 1.0f;
    const T *g = static_cast<const T *>(a.grad) + t * a.grad_stride, *y = static_cast<const T *>(a.y) + r * a.y_stride;
    T *dy = a.dy ? static_cast<T *>(a.dy) + r * a.dy_stride : nullptr;
    float dot = 0.0f;
#pragma unroll 4
    for (uint32_t c = lane * V; c < a.columns; c += 32u * V) {
        Vec<T, V> d = {};
        if (known) {
            const Vec<T, V> gv = *reinterpret_cast<const Vec<T, V> *>(g + c);
            if (a.dweights) {
                const Vec<T, V> yv = *reinterpret_cast<const Vec<T, V> *>(y + c);
#pragma unroll
                for (int k = 0; k < V; k++) dot = fmaf(widen(gv.v[k]), widen(yv.v[k]), dot);
            }
#pragma unroll
            for (int k = 0; k < V; k++) d.v[k] = narrow<T>(w * widen(gv.v[k]));
        }
        if (dy) *reinterpret_cast<Vec<T, V> *>(dy + c) = d;
    }
    if (!a.dweights || !known) return;
#pragma unroll
    for (uint32_t s = 16; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
    if (lane == 0) a.dweights[o] = dot;
}

// neighbours that one load may bring: all that the pointers, strides and the width are multiples of, at most 16 bytes
template <typename T>
uint32_t width_of(std::initializer_list<uint64_t> all, uint32_t columns) {
    uint64_t at = (uint64_t)columns * sizeof(T);
    for (const uint64_t x : all) at |= x;
    uint32_t v = 16u / sizeof(T);
    while (v > 1u && at % (v * sizeof(T))) v /= 2u;
    return v;
}
inline uint64_t bits(const void *p) { return reinterpret_cast<uintptr_t>(p); }

template <typename T>
cudaError_t combine_launch(const CombineArgs &a, cudaStream_t stream) {
    const uint32_t v = width_of<T>({bits(a.out), bits(a.y), a.out_stride * sizeof(T), a.y_stride * sizeof(T)}, a.columns), per_row = a.columns / v;
    return in_portions(a.tokens, std::max(1u, 0x7fffff00u / per_row), [&](uint32_t t0, uint32_t nt) {
        CombineArgs b = a;
        b.tokens = nt;
        b.out = static_cast<T *>(a.out) + t0 * a.out_stride;
        b.place += (uint64_t)t0 * a.top;
        if (a.weights) b.weights += (uint64_t)t0 * a.top;
        const uint32_t items = nt * per_row, blocks = (items + kMoveThreads - 1u) / kMoveThreads;
        if (v * sizeof(T) == 16) k_experts_combine<T, 16 / sizeof(T)><<<blocks, kMoveThreads, 0, stream>>>(b, per_row, items);
        else if (v * sizeof(T) == 8) k_experts_combine<T, 8 / sizeof(T)><<<blocks, kMoveThreads, 0, stream>>>(b, per_row, items);
        else if (v * sizeof(T) == 4) k_experts_combine<T, 4 / sizeof(T)><<<blocks, kMoveThreads, 0, stream>>>(b, per_row, items);
        else k_experts_combine<T, 1><<<blocks, kMoveThreads, 0, stream>>>(b, per_row, items);
        return cudaGetLastError();
    });
}
template <typename T>
cudaError_t grad_launch(const CombineArgs &a, cudaStream_t stream) {
    const uint32_t v = width_of<T>({bits(a.y), bits(a.grad), bits(a.dy), a.y_stride * sizeof(T), a.grad_stride * sizeof(T), a.dy_stride * sizeof(T)}, a.columns), n = a.tokens * a.top;
    const uint32_t blocks = (std::max(n, a.rows) + kMoveThreads / 32u - 1u) / (kMoveThreads / 32u);
    if (v * sizeof(T) == 16) k_experts_combine_grad<T, 16 / sizeof(T)><<<blocks, kMoveThreads, 0, stream>>>(a, n);
    else if (v * sizeof(T) == 8) k_experts_combine_grad<T, 8 / sizeof(T)><<<blocks, kMoveThreads, 0, stream>>>(a, n);
    else if (v * sizeof(T) == 4) k_experts_combine_grad<T, 4 / sizeof(T)><<<blocks, kMoveThreads, 0, stream>>>(a, n);
    else k_experts_combine_grad<T, 1><<<blocks, kMoveThreads, 0, stream>>>(a, n);
    return cudaGetLastError();
}

}  // namespace
}  // namespace nb

using nb::fail;

namespace {
constexpr uint32_t kMostPlaces = 1u << 30;

cudaError_t sort_launch(const nb::SortArgs &a, cudaStream_t stream) {
    using namespace nb;
    // blocks: one for each 4096 places, up to the eight that any cluster may have
    uint32_t C = 1;
    while (C < kSortCluster && a.n > C * 4096u) C *= 2u;
    const uint32_t smem = (kSortWarps + 2u) * a.experts * 4u;
    if (smem > 40u * 1024u) {
        const cudaError_t e = smem_at_least(reinterpret_cast<const void *>(k_experts_sort), (int)smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(C); cfg.blockDim = dim3(kSortThreads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr; cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_experts_sort, a, C);
}

int combine_checked(const nb200_experts_rows *p, bool gradient, nb::CombineArgs *a) {
    if (!p) return fail(NB200_EINVAL, "null argument");
    if (p->type > nb::T_F16) return fail(NB200_EINVAL, "rows are fp32, bf16 or fp16 (type %u)", p->type);
    if ((uint64_t)p->tokens * p->top > kMostPlaces || p->rows > kMostPlaces || p->columns > kMostPlaces)
        return fail(NB200_EINVAL, "%u tokens of %u experts, %u rows of %u are too many for one call", p->tokens, p->top, p->rows, p->columns);
    const uint32_t size = nb::elem_size(p->type);
    auto aligned = [&](const void *x, uint32_t to) { return reinterpret_cast<uintptr_t>(x) % to == 0; };
    if (!aligned(p->out, size) || !aligned(p->y, size) || !aligned(p->grad, size) || !aligned(p->dy, size)) return fail(NB200_EINVAL, "rows are not aligned to their type");
    if (!aligned(p->weights, 4) || !aligned(p->place, 4) || !aligned(p->order, 4) || !aligned(p->dweights, 4)) return fail(NB200_EINVAL, "weights and places are not aligned to their type");
    *a = nb::CombineArgs{p->out, p->y, p->weights, p->place, p->order, p->out_stride, p->y_stride, p->tokens, p->top, p->rows, p->columns, p->grad, p->dy, p->dweights, p->grad_stride, p->dy_stride};
    if (gradient) {
        if (p->rows > (uint64_t)p->tokens * p->top) return fail(NB200_EINVAL, "%u rows of %u places", p->rows, p->tokens * p->top);
        const bool some = p->rows && p->columns;
        if ((p->dy && p->rows && (!p->order || (some && !p->grad))) || (p->dweights && p->tokens && p->top && (!p->place || (some && (!p->order || !p->y || !p->grad))))) return fail(NB200_EINVAL, "null argument");
        if (p->dy && p->rows > 1 && p->dy_stride < p->columns) return fail(NB200_EINVAL, "rows of the gradient overlap");
    } else if (p->tokens && p->columns) {
        if (!p->out || (p->top && (!p->place || (p->rows && !p->y)))) return fail(NB200_EINVAL, "null argument");
        if (p->tokens > 1 && p->out_stride < p->columns) return fail(NB200_EINVAL, "rows of the result overlap");
    }
    return 0;
}
}  // namespace

extern "C" {

int nb200_dev_experts_sort(int32_t *order, int32_t *offsets, int32_t *place, const void *ids, uint32_t id_bytes, uint32_t n, uint32_t experts, void *stream) {
    if (!experts || experts > nb::kMaxExperts) return fail(NB200_EINVAL, "%u experts: 1 to %u", experts, nb::kMaxExperts);
    if (n > kMostPlaces) return fail(NB200_EINVAL, "%u places are too many for one call", n);
    if (id_bytes != 4 && id_bytes != 8) return fail(NB200_EINVAL, "ids are 32-bit or 64-bit numbers");
    if (!offsets || (n && (!order || !place || !ids))) return fail(NB200_EINVAL, "null argument");
    if (reinterpret_cast<uintptr_t>(ids) % id_bytes || (reinterpret_cast<uintptr_t>(order) | reinterpret_cast<uintptr_t>(offsets) | reinterpret_cast<uintptr_t>(place)) % 4u)
        return fail(NB200_EINVAL, "ids, order, offsets or place are not aligned to their type");
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    NB_CK(sort_launch(nb::SortArgs{ids, order, offsets, place, id_bytes == 8 ? 1u : 0u, n, experts}, static_cast<cudaStream_t>(stream)));
    return 0;
}

int nb200_dev_experts_gather(void *out, uint64_t out_stride, const void *x, uint64_t x_stride, uint64_t row_bytes, const int32_t *order, uint32_t n, uint32_t top, uint32_t tokens, void *stream) {
    if (n > kMostPlaces || row_bytes > 1u << 30) return fail(NB200_EINVAL, "%u rows of %llu bytes are too many for one call", n, (unsigned long long)row_bytes);
    if (!n || !row_bytes) return 0;
    if (!out || !order || !top || (tokens && !x)) return fail(NB200_EINVAL, "null argument");
    if (reinterpret_cast<uintptr_t>(order) % 4u) return fail(NB200_EINVAL, "order is not aligned to its type");
    if (n > 1 && out_stride < row_bytes) return fail(NB200_EINVAL, "rows of the result overlap");
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    const uint64_t at = reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(x) | out_stride | x_stride | row_bytes;
    uint32_t unit = 16;
    while (at % unit) unit /= 2u;
    const uint32_t units = (uint32_t)(row_bytes / unit), each = nb::kMoveThreads * nb::kMoveUnits;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    NB_CK(nb::in_portions(n, std::max(1u, 0x7fffff00u / units), [&](uint32_t r0, uint32_t rows) {
        const nb::GatherArgs a{static_cast<char *>(out) + r0 * out_stride, static_cast<const char *>(x), order + r0, out_stride, x_stride, units, top, tokens};
        const uint32_t items = rows * units, blocks = (items + each - 1u) / each;
        switch (unit) {
            case 16: nb::k_experts_gather<16><<<blocks, nb::kMoveThreads, 0, s>>>(a, items); break;
            case 8: nb::k_experts_gather<8><<<blocks, nb::kMoveThreads, 0, s>>>(a, items); break;
            case 4: nb::k_experts_gather<4><<<blocks, nb::kMoveThreads, 0, s>>>(a, items); break;
            case 2: nb::k_experts_gather<2><<<blocks, nb::kMoveThreads, 0, s>>>(a, items); break;
            default: nb::k_experts_gather<1><<<blocks, nb::kMoveThreads, 0, s>>>(a, items);
        }
        return cudaGetLastError();
    }));
    return 0;
}

int nb200_dev_experts_combine(const nb200_experts_rows *p, void *stream) {
    nb::CombineArgs a{};
    if (const int r = combine_checked(p, false, &a)) return r;
    if (!a.tokens || !a.columns) return 0;
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    NB_CK(p->type == nb::T_F32 ? nb::combine_launch<float>(a, s) : p->type == nb::T_BF16 ? nb::combine_launch<__nv_bfloat16>(a, s) : nb::combine_launch<__half>(a, s));
    return 0;
}

int nb200_dev_experts_combine_grad(const nb200_experts_rows *p, void *stream) {
    nb::CombineArgs a{};
    if (const int r = combine_checked(p, true, &a)) return r;
    if (!a.tokens || !a.top || (!a.dy && !a.dweights)) return 0;
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    NB_CK(p->type == nb::T_F32 ? nb::grad_launch<float>(a, s) : p->type == nb::T_BF16 ? nb::grad_launch<__nv_bfloat16>(a, s) : nb::grad_launch<__half>(a, s));
    return 0;
}

}  // extern "C"
