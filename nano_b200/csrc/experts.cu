// experts.cu -- rows of tokens sorted by expert and back, with their weights and gradients, and their C entry points.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "family.h"
#include "ops.h"
#include "portions.h"
#include "rows.cuh"

namespace nb {
namespace {

// ------------------------------------------------------------------------------------------------
// Sorting places by expert: counts, their running sums, and a second walk that hands out the places in order.  A warp owns a run of neighbouring places and a row of counts in shared memory, a
// block the runs of its warps, a cluster of up to sixteen blocks the list: sums run over experts, then blocks, then warps, so the result is the stable one whatever the order of arrival, in one
// launch without a workspace.  Within 32 places a place's rank is counted from ballots over the bits of its expert's number.  Bound by latency: eight loads of a warp are under way at once, and the first eight of its run stay in
// registers for the second walk.
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kSortThreads = 1024, kSortWarps = kSortThreads / 32, kSortCluster = 16, kMaxExperts = 1024, kSortAhead = 8;

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
    uint32_t *mine = counts + warp * E, *block = counts + (blockDim.x / 32u) * E, *begin = block + E;
    const uint32_t threads = blockDim.x, warps = threads / 32u;
    for (uint32_t i = tid; i < warps * E; i += threads) counts[i] = 0;
    // runs of whole 32 places, as even as that allows
    const uint32_t pieces = (a.n + 31u) / 32u, runs = C * warps, per = (pieces + runs - 1u) / runs;
    const uint32_t p0 = min(pieces, (rank * warps + warp) * per), p1 = min(pieces, p0 + per);
    auto expert = [&](uint32_t i) {          // E: none
        if (i >= a.n) return E;
        const long long id = a.wide ? __ldg(static_cast<const long long *>(a.ids) + i) : (long long)__ldg(static_cast<const int *>(a.ids) + i);
        return id >= 0 && id < (long long)E ? (uint32_t)id : E;
    };
    const uint32_t bits = 32u - __clz(E);          // (of 0 .. E)
    auto alike = [&](uint32_t e) {          // the lanes with the same number
        uint32_t same = 0xffffffffu;
        for (uint32_t b = 0; b < bits; b++) { const bool one = e >> b & 1u; const uint32_t m = __ballot_sync(0xffffffffu, one); same &= one ? m : ~m; }
        return same;
    };
    uint32_t held[kSortAhead];
    auto load = [&](uint32_t p) {
#pragma unroll
        for (uint32_t j = 0; j < kSortAhead; j++) held[j] = p + j < p1 ? expert((p + j) * 32u + lane) : E;
    };
    load(p0);
    __syncthreads();
    for (uint32_t p = p0; p < p1; p += kSortAhead) {
        if (p != p0) load(p);
#pragma unroll
        for (uint32_t j = 0; j < kSortAhead; j++) if (held[j] < E) atomicAdd(mine + held[j], 1u);          // (a count does not depend on the order)
    }
    if (p1 - p0 > kSortAhead) load(p0);
    __syncthreads();
    for (uint32_t e = tid; e < E; e += threads) {
        uint32_t c[kSortWarps], run = 0;
#pragma unroll
        for (uint32_t w = 0; w < kSortWarps; w++) c[w] = w < warps ? counts[w * E + e] : 0u;
#pragma unroll
        for (uint32_t w = 0; w < kSortWarps; w++) { const uint32_t x = c[w]; c[w] = run; run += x; }
#pragma unroll
        for (uint32_t w = 0; w < kSortWarps; w++) if (w < warps) counts[w * E + e] = c[w];          // those of the warps before
        block[e] = run;
    }
    if (C > 1) cluster_sync(); else __syncthreads();
    uint32_t all = 0, before = 0;          // of expert tid: in the whole list, in the blocks before this one
    if (tid < E)
#pragma unroll 8
        for (uint32_t c = 0; c < C; c++) { const uint32_t x = C > 1 ? peer_u32(block + tid, c) : block[tid]; all += x; before += c < rank ? x : 0u; }
    uint32_t up = all;
#pragma unroll
    for (uint32_t o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, up, o); up += lane >= o ? x : 0u; }
    if (lane == 31u) sums[warp] = up;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = lane < warps ? sums[lane] : 0u;
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, s, o); s += lane >= o ? x : 0u; }
        sums[lane] = s;          // (all 32)
    }
    __syncthreads();
    const uint32_t from = up - all + (warp ? sums[warp - 1u] : 0u), known = sums[31];
    if (tid < E) {
        begin[tid] = from + before;
        if (rank == 0) { a.offsets[tid] = (int32_t)from; if (tid == E - 1u) a.offsets[E] = (int32_t)known; }
    }
    __syncthreads();
    for (uint32_t i = tid; i < warps * E; i += threads) counts[i] += begin[i % E];          // where a warp's first place of an expert goes
    __syncthreads();
    for (uint32_t p = p0; p < p1; p += kSortAhead) {
        if (p != p0) load(p);
#pragma unroll
        for (uint32_t j = 0; j < kSortAhead; j++) {
            if (p + j >= p1) break;
            const uint32_t i = (p + j) * 32u + lane, e = held[j], same = alike(e);
            uint32_t at = 0;
            if (e < E) at = mine[e];
            __syncwarp();
            if (e < E && lane == (uint32_t)__ffs(same) - 1u) mine[e] = at + __popc(same);
            __syncwarp();
            at += __popc(same & ((1u << lane) - 1u));
            if (i < a.n) a.place[i] = e < E ? (int32_t)at : -1;
            if (e < E) a.order[at] = (int32_t)i;
        }
    }
    for (uint64_t r = known + (uint64_t)rank * threads + tid; r < a.n; r += C * threads) a.order[r] = -1;
    if (C > 1) cluster_sync();          // nobody leaves while its shared memory is read
}

// ------------------------------------------------------------------------------------------------
// Rows to their places.  Pure movement, bound by memory.  Where every row starts on a 16-byte border, pieces of 16 bytes, four to a thread; elsewhere pieces of the result's memory, whose bytes are
// shifted out of two of the row's.
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kMoveThreads = 256, kMoveUnits = 4;
struct GatherArgs { uint8_t *out; const uint8_t *x; const int32_t *order; uint64_t out_stride, x_stride; uint32_t bytes, top, tokens, margin; };
__device__ __forceinline__ uint32_t token_of(const GatherArgs &a, uint32_t r) {          // `tokens` and more: none
    const int32_t o = __ldg(a.order + r);
    return o >= 0 ? (uint32_t)o / a.top : 0xffffffffu;
}
__global__ void __launch_bounds__(kMoveThreads) k_experts_gather(const GatherArgs a, const Divider per_row, const uint32_t items) {
    uint4 v[kMoveUnits] = {};
    const uint32_t i0 = blockIdx.x * kMoveThreads * kMoveUnits + threadIdx.x;
#pragma unroll
    for (uint32_t j = 0; j < kMoveUnits; j++) {
        const uint32_t i = i0 + j * kMoveThreads, r = per_row.over(i);
        if (i >= items) break;
        const uint32_t t = token_of(a, r);
        if (t < a.tokens) v[j] = __ldg(reinterpret_cast<const uint4 *>(a.x + t * a.x_stride) + (i - r * per_row.d));
    }
#pragma unroll
    for (uint32_t j = 0; j < kMoveUnits; j++) {
        const uint32_t i = i0 + j * kMoveThreads, r = per_row.over(i);
        if (i >= items) break;
        reinterpret_cast<uint4 *>(a.out + (uint64_t)r * a.out_stride)[i - r * per_row.d] = v[j];
    }
}
// UNIT: bytes that every row's start and length are multiples of
template <typename UNIT>
__global__ void __launch_bounds__(kMoveThreads) k_experts_gather_any(const GatherArgs a, const Divider per_row, const uint32_t items) {
    constexpr int S = sizeof(UNIT), U = 2;
    union Piece { uint32_t w[4]; UNIT u[16 / S]; };
    Piece v[U] = {};
    int k[U];
    uint8_t *to[U];
    const uint32_t i0 = blockIdx.x * kMoveThreads * U + threadIdx.x;
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
        const uint32_t i = i0 + u * kMoveThreads, r = per_row.over(i);
        k[u] = 0x7fffffff - 16;
        if (i >= items) continue;
        to[u] = a.out + (uint64_t)r * a.out_stride;
        k[u] = piece_at(to[u], i - r * per_row.d);
        if (k[u] >= (int)a.bytes) continue;
        const uint32_t t = token_of(a, r);
        if (t >= a.tokens) continue;
        const uint8_t *row = a.x + t * a.x_stride;
        if (between(t, a.tokens, a.margin) || inside<16, uint8_t>(a.bytes, k[u])) load_words<4, (S < 2)>(row + k[u], v[u].w);
        else
#pragma unroll
            for (int j = 0; j < 16; j += S) if (k[u] + j >= 0 && k[u] + j < (int)a.bytes) v[u].u[j / S] = *reinterpret_cast<const UNIT *>(row + k[u] + j);
    }
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
        if (k[u] >= (int)a.bytes) continue;
        if (k[u] >= 0 && (uint32_t)k[u] + 16u <= a.bytes) *reinterpret_cast<uint4 *>(to[u] + k[u]) = make_uint4(v[u].w[0], v[u].w[1], v[u].w[2], v[u].w[3]);
        else
#pragma unroll
            for (int j = 0; j < 16; j += S) if (k[u] + j >= 0 && k[u] + j < (int)a.bytes) *reinterpret_cast<UNIT *>(to[u] + k[u] + j) = v[u].u[j / S];
    }
}

// ------------------------------------------------------------------------------------------------
// And back.  A piece of 16 bytes of a token's row to a thread, which adds up the rows of its experts in fp32, in the list's order; the gradient by rows of the sorted list, which read the token's
// gradient (the other experts of the token find it in L2) and their own row once.  Both bound by memory.
// ------------------------------------------------------------------------------------------------
struct CombineArgs {
    void *out; const void *y; const float *weights; const int32_t *place, *order; uint64_t out_stride, y_stride; uint32_t tokens, top, rows, columns;
    const void *grad; void *dy; float *dweights; uint64_t grad_stride, dy_stride;
    uint32_t y_margin, grad_margin;          // (margin_rows)
};
template <typename T, Where WHERE>
__device__ __forceinline__ void combine_piece(const CombineArgs &a, T *out, uint64_t first, int c) {
    constexpr int P = 16 / sizeof(T);
    float sum[P] = {};
#pragma unroll 4
    for (uint32_t j = 0; j < a.top; j++) {
        const uint32_t r = (uint32_t)__ldg(a.place + first + j);          // (-1: beyond all rows)
        const float w = a.weights ? __ldg(a.weights + first + j) : 1.0f;
        if (r < a.rows) {
            float y[P];
            load_row<WHERE>(static_cast<const T *>(a.y) + r * a.y_stride, a.columns, c, y);
#pragma unroll
            for (int k = 0; k < P; k++) sum[k] = fmaf(w, y[k], sum[k]);
        }
    }
    store_piece<WHERE == EVEN ? EVEN : ANY>(out, a.columns, c, sum);
}
// BORDERS: every row starts on a 16-byte border and is whole pieces
template <typename T, bool BORDERS>
__global__ void __launch_bounds__(kMoveThreads) k_experts_combine(const CombineArgs a, const Divider per_row, const uint32_t items) {
    constexpr int P = 16 / sizeof(T);
    const uint32_t i = blockIdx.x * kMoveThreads + threadIdx.x, t = per_row.over(i);
    if (i >= items) return;
    T *out = static_cast<T *>(a.out) + t * a.out_stride;
    const uint64_t first = (uint64_t)t * a.top;
    if constexpr (BORDERS) combine_piece<T, EVEN>(a, out, first, (int)((i - t * per_row.d) * P));
    else {
        const int c = piece_at(out, i - t * per_row.d);
        if (c >= (int)a.columns) return;
        bool plain = inside<P, T>(a.columns, c);
        if (!plain) {
            plain = true;
            for (uint32_t j = 0; j < a.top; j++) { const uint32_t r = (uint32_t)__ldg(a.place + first + j); plain = plain && (r >= a.rows || between(r, a.rows, a.y_margin)); }
        }
        if (plain) combine_piece<T, INSIDE>(a, out, first, c);
        else combine_piece<T, ANY>(a, out, first, c);
    }
}

template <typename T> struct GradRow { const T *g, *y; T *dy; bool known, wanted, weigh; float w; uint32_t columns; };
template <Where WHERE, typename T>
__device__ __forceinline__ float grad_piece(const GradRow<T> &r, int c) {
    constexpr int P = 16 / sizeof(T);
    float d[P] = {}, dot = 0.0f;
    if (r.known) {
        load_row<WHERE>(r.g, r.columns, c, d);
        if (r.weigh) {
            float v[P];
            load_row<WHERE>(r.y, r.columns, c, v);
            if (WHERE == INSIDE && (c < 0 || (uint32_t)(c + P) > r.columns))
#pragma unroll
                for (int k = 0; k < P; k++) if (c + k < 0 || (uint32_t)(c + k) >= r.columns) d[k] = v[k] = 0.0f;
#pragma unroll
            for (int k = 0; k < P; k++) dot = fmaf(d[k], v[k], dot);
        }
#pragma unroll
        for (int k = 0; k < P; k++) d[k] *= r.w;
    }
    if (r.wanted) store_piece<WHERE == EVEN ? EVEN : ANY>(r.dy, r.columns, c, d);
    return dot;
}
// LANES threads to a row
template <typename T, int LANES, bool BORDERS>
__global__ void __launch_bounds__(kMoveThreads) k_experts_combine_grad(const CombineArgs a, const uint32_t n) {
    constexpr int P = 16 / sizeof(T);
    const uint32_t r = blockIdx.x * (kMoveThreads / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES;
    if (a.dweights && r < n && lane == 0 && (uint32_t)__ldg(a.place + r) >= a.rows) a.dweights[r] = 0.0f;          // of place r of the list
    const uint32_t o = r < a.rows ? (uint32_t)__ldg(a.order + r) : 0xffffffffu, t = o / a.top;
    const bool known = o < n;
    // (dy's address shares the columns out whether it is wanted or not: the same sums)
    const GradRow<T> row{static_cast<const T *>(a.grad) + t * a.grad_stride, static_cast<const T *>(a.y) + r * a.y_stride, static_cast<T *>(a.dy) + r * a.dy_stride, known, a.dy != nullptr,
                         a.dweights != nullptr, known && a.weights ? __ldg(a.weights + o) : 1.0f, a.columns};
    float dot = 0.0f;
    if (r < a.rows) {
        if constexpr (BORDERS) {
#pragma unroll 4
            for (uint32_t c = lane * P; c < a.columns; c += LANES * P) dot += grad_piece<EVEN>(row, (int)c);
        } else {
            const uint32_t pieces = (a.columns + (uint32_t)-piece_at(row.dy, 0) + P - 1u) / P;
            if (!known || ((!row.weigh || between(r, a.rows, a.y_margin)) && between(t, a.tokens, a.grad_margin))) {          // (y is read for the weights' gradient alone)
#pragma unroll 2
                for (uint32_t b = lane; b < pieces; b += LANES) dot += grad_piece<INSIDE>(row, piece_at(row.dy, b));
            } else
                for (uint32_t b = lane; b < pieces; b += LANES) dot += grad_piece<ANY>(row, piece_at(row.dy, b));
        }
    }
    if (!a.dweights) return;
#pragma unroll
    for (uint32_t s = LANES / 2; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
    if (lane == 0 && known) a.dweights[o] = dot;
}

template <typename T>
cudaError_t combine_launch(const CombineArgs &a, cudaStream_t stream) {
    const bool out = on_borders<T>(a.out, a.out_stride, a.tokens), all = out && on_borders<T>(a.y, a.y_stride, a.rows) && a.columns * sizeof(T) % 16u == 0;
    const uint32_t per_row = most_pieces<T>(a.columns, out);
    return in_portions(a.tokens, std::max(1u, 0x7fffff00u / per_row), [&](uint32_t t0, uint32_t nt) {
        CombineArgs b = a;
        b.tokens = nt;
        b.out = static_cast<T *>(a.out) + t0 * a.out_stride;
        b.place += (uint64_t)t0 * a.top;
        if (a.weights) b.weights += (uint64_t)t0 * a.top;
        const uint32_t items = nt * per_row, blocks = (items + kMoveThreads - 1u) / kMoveThreads;
        if (all) k_experts_combine<T, true><<<blocks, kMoveThreads, 0, stream>>>(b, Divider::of(per_row), items);
        else k_experts_combine<T, false><<<blocks, kMoveThreads, 0, stream>>>(b, Divider::of(per_row), items);
        return cudaGetLastError();
    });
}
template <typename T>
cudaError_t grad_launch(const CombineArgs &a, cudaStream_t stream) {
    const bool even = on_borders<T>(a.dy, a.dy_stride, a.rows) && on_borders<T>(a.y, a.y_stride, a.rows) && on_borders<T>(a.grad, a.grad_stride, a.tokens) && a.columns * sizeof(T) % 16u == 0;
    const uint32_t pieces = (a.columns * (uint32_t)sizeof(T) + 15u) / 16u, n = a.tokens * a.top, all = std::max(n, a.rows);
    // Threads to a row: as many as it has pieces, up to a warp; eight for rows of up to 64 pieces that start anywhere, whose ends are stores of single numbers (rows and places are at most 2^30).
    // us with 8 / 32: 131072 rows of 267 bf16 numbers 61 / 127, but 32768 of 2047 133 / 108, 8000 of 2534 fp32 158 / 62
    auto go = [&](auto kernel, uint32_t lanes) { kernel<<<(uint32_t)(((uint64_t)all * lanes + kMoveThreads - 1u) / kMoveThreads), kMoveThreads, 0, stream>>>(a, n); return cudaGetLastError(); };
    if (!even) return pieces <= 64u ? go(k_experts_combine_grad<T, 8, false>, 8) : go(k_experts_combine_grad<T, 32, false>, 32);
    return pieces <= 4u ? go(k_experts_combine_grad<T, 4, true>, 4) : pieces <= 8u ? go(k_experts_combine_grad<T, 8, true>, 8) : go(k_experts_combine_grad<T, 32, true>, 32);
}

}  // namespace
}  // namespace nb

using nb::fail;

namespace {
constexpr uint32_t kMostPlaces = 1u << 30;

cudaError_t sort_launch(const nb::SortArgs &a, cudaStream_t stream) {
    using namespace nb;
    // blocks: one for each 1024 places, up to the sixteen that a cluster may have if it is asked for.  us with 4096 / 1024, 64 experts: 4096 places 7.2 / 6.0, 8192 8.3 / 6.0, 32768 8.4 / 7.1 (the
    // second walk's stores go to places far apart, one after the other)
    uint32_t C = 1;
    while (C < kSortCluster && a.n > C * 1024u) C *= 2u;
    if (C > 8u) {
        const cudaError_t e = cudaFuncSetAttribute(k_experts_sort, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    // warps: one for each 32 places, up to the block's 32, and threads for all experts
    const uint32_t warps = std::min(kSortWarps, std::max((a.n + 32u * C - 1u) / (32u * C), (a.experts + 31u) / 32u)), smem = (warps + 2u) * a.experts * 4u;
    if (smem > 40u * 1024u) {
        const cudaError_t e = smem_at_least(reinterpret_cast<const void *>(k_experts_sort), (int)smem);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(C); cfg.blockDim = dim3(std::max(1u, warps) * 32u); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
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
    *a = nb::CombineArgs{p->out, p->y, p->weights, p->place, p->order, p->out_stride, p->y_stride, p->tokens, p->top, p->rows, p->columns, p->grad, p->dy, p->dweights, p->grad_stride, p->dy_stride,
                          nb::margin_rows(p->y_stride * size), nb::margin_rows(p->grad_stride * size)};
    if (gradient) {
        if (p->rows > (uint64_t)p->tokens * p->top) return fail(NB200_EINVAL, "%u rows of %u places", p->rows, p->tokens * p->top);
        const bool some = p->rows && p->columns;
        if ((p->dy && p->rows && (!p->order || (some && !p->grad))) || (p->dweights && p->tokens && p->top && (!p->place || (p->rows && !p->order) || (some && (!p->y || !p->grad))))) return fail(NB200_EINVAL, "null argument");
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
    const uint32_t bytes = (uint32_t)row_bytes, per_row = unit == 16u ? bytes / 16u : nb::most_pieces<uint8_t>(bytes, false);
    const nb::Divider by = nb::Divider::of(per_row);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    NB_CK(nb::in_portions(n, std::max(1u, 0x7fffff00u / per_row), [&](uint32_t r0, uint32_t rows) {
        const nb::GatherArgs a{static_cast<uint8_t *>(out) + r0 * out_stride, static_cast<const uint8_t *>(x), order + r0, out_stride, x_stride, bytes, top, tokens, nb::margin_rows(x_stride)};
        const uint32_t items = rows * per_row, each = nb::kMoveThreads * (unit >= 16u ? nb::kMoveUnits : 2u), blocks = (items + each - 1u) / each;
        switch (unit) {
            case 16: nb::k_experts_gather<<<blocks, nb::kMoveThreads, 0, s>>>(a, by, items); break;
            case 8: nb::k_experts_gather_any<uint2><<<blocks, nb::kMoveThreads, 0, s>>>(a, by, items); break;
            case 4: nb::k_experts_gather_any<uint32_t><<<blocks, nb::kMoveThreads, 0, s>>>(a, by, items); break;
            case 2: nb::k_experts_gather_any<uint16_t><<<blocks, nb::kMoveThreads, 0, s>>>(a, by, items); break;
            default: nb::k_experts_gather_any<uint8_t><<<blocks, nb::kMoveThreads, 0, s>>>(a, by, items);
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
