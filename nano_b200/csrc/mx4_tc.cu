// mx4_tc.cu -- products of rows in microscaled 4-bit floating point on the fifth-generation tensor cores, which multiply the codes as they are (format: mx4.h).
//
// out^T = W X^T in tiles of 128 rows of W x TN rows of X: tcgen05.mma kind::mxf4 takes 64 columns of both and two scales for each row, which lie in tensor memory (tcgen05.cp brings them there).
// A stage is 256 columns: codes by cp.async.bulk.tensor into 128-byte-swizzled rows, scales by two warps, which lay 128 rows x 4 scales out as that copy wants them (32 lines of 16 bytes: row r's word
// is word r / 32 of line r % 32).  A lane of tensor memory is an output column, so a warp's stores of one row are neighbours.
// Every wait has a limit; a block in which one runs out leaves with NaN in its results.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "family.h"
#include "mx4.h"
#include "tc_ptx.cuh"

namespace nb {
namespace {

constexpr uint32_t kRows = 128, kDepth = 256, kStageGroups = kDepth / kMx4Group;          // rows of W in a tile; columns of a stage
template <int TN> struct Tile {
    static constexpr uint32_t blocks = (TN + 127) / 128;          // of 128 rows, as scales are laid out
    static constexpr uint32_t x_at = kRows * 128u, ws_at = x_at + TN * 128u, xs_at = ws_at + 1024u, bytes = xs_at + 1024u * blocks;          // of a stage
    static constexpr uint32_t stages = TN <= 16 ? 5 : TN <= 64 ? 4 : 3;          // up to 104 KB: two blocks to an SM
    static constexpr uint32_t scale_cols = 8u + 8u * blocks, cols_used = (TN < 32 ? 32u : TN) + stages * scale_cols;
    static constexpr uint32_t cols = cols_used <= 128 ? 128 : cols_used <= 256 ? 256 : 512;
    static constexpr uint32_t smem = stages * bytes + 1024u;
};

struct alignas(64) TcArgs { CUtensorMap wmap, xmap; Mx4Product p; uint32_t groups, steps, ks, wtiles, pairs, w_align, x_align, made; };

__device__ __forceinline__ bool soon(uint32_t bar, uint32_t parity) { return mbar_try(bar, parity) || mbar_wait(bar, parity); }
__device__ __forceinline__ bool soon_warp(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, soon(bar, parity)); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// d (+)= a b^T: 64 columns of 128 rows of codes and of the instruction's N, each with its two scales
__device__ __forceinline__ void mma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t a_scales, uint32_t b_scales, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %6, 0;\ntcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"((uint32_t)add) : "memory");
}
// 32 lines of 16 bytes to four columns of tensor memory, the same in all four quarters of its lanes
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint64_t desc) { asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory"); }
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) { return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)8 << 32) | ((uint64_t)1 << 46); }          // no swizzle, 8 lines every 128 bytes
// e2m1 x e2m1, scales in 8 bits of exponent, N columns; scales from byte `id` (0 or 2) of their words
__host__ __device__ constexpr uint32_t idesc_of(uint32_t n, uint32_t id) { return (id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((kRows >> 4) << 24) | (id << 29); }

// eight neighbouring scales of a row, from group g on; zeros behind its last
__device__ __forceinline__ uint2 scales8(const uint8_t *row, uint32_t g, uint32_t groups, uint32_t align) {
    uint2 v = make_uint2(0u, 0u);
    if (g + 8u <= groups && align >= 8u) return __ldg(reinterpret_cast<const uint2 *>(row + g));
    if (g + 8u <= groups && align >= 4u) return make_uint2(__ldg(reinterpret_cast<const uint32_t *>(row + g)), __ldg(reinterpret_cast<const uint32_t *>(row + g + 4u)));
#pragma unroll
    for (uint32_t i = 0; i < 8; i++) {
        const uint32_t b = g + i < groups ? (uint32_t)row[g + i] : 0u;
        if (i < 4) v.x |= b << (8u * i); else v.y |= b << (8u * (i - 4u));
    }
    return v;
}

// A warp brings the scales of up to 128 * BLOCKS rows, stage after stage: a lane has rows lane, lane + 32, ..., and writes the words of four of them at once
template <uint32_t BLOCKS>
struct ScaleWarp {
    const uint8_t *row[BLOCKS * 4];
    uint32_t groups, align;
    // rows [0, live) at `base`; what lies behind them counts for nothing and is read from the first
    __device__ __forceinline__ void at(const uint8_t *base, uint64_t stride, uint32_t live, uint32_t lane) {
#pragma unroll
        for (uint32_t i = 0; i < BLOCKS * 4; i++) { const uint32_t r = lane + 32u * i; row[i] = base + (r < live ? r : 0u) * stride; }
    }
    __device__ __forceinline__ void load(uint32_t step, uint2 (&v)[BLOCKS * 4]) const {
#pragma unroll
        for (uint32_t i = 0; i < BLOCKS * 4; i++) v[i] = scales8(row[i], step * kStageGroups, groups, align);
    }
    __device__ __forceinline__ static void store(uint32_t to, const uint2 (&v)[BLOCKS * 4], uint32_t lane) {          // [half of the stage][block][line]
#pragma unroll
        for (uint32_t b = 0; b < BLOCKS; b++) {
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + b * 512u + lane * 16u), "r"(v[4 * b].x), "r"(v[4 * b + 1].x), "r"(v[4 * b + 2].x), "r"(v[4 * b + 3].x) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + (BLOCKS + b) * 512u + lane * 16u), "r"(v[4 * b].y), "r"(v[4 * b + 1].y), "r"(v[4 * b + 2].y), "r"(v[4 * b + 3].y) : "memory");
        }
    }
};
template <uint32_t BLOCKS>
__device__ __forceinline__ bool bring_scales(const ScaleWarp<BLOCKS> &w, uint32_t s0, uint32_t ns, uint32_t ring, uint32_t bytes, uint32_t off, uint32_t stages, uint32_t full, uint32_t empty, uint32_t lane) {
    uint2 v[2][BLOCKS * 4];
    if (ns > 0) w.load(s0, v[0]);
    if (ns > 1) w.load(s0 + 1u, v[1]);
#pragma unroll 2
    for (uint32_t i = 0; i < ns; i++) {
        const uint32_t st = i % stages;
        if (i >= stages && !soon_warp(empty + st * 8u, ((i / stages) - 1u) & 1u)) return false;
        ScaleWarp<BLOCKS>::store(ring + st * bytes + off, v[i & 1u], lane);
        if (i + 2u < ns) w.load(s0 + i + 2u, v[i & 1u]);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");          // plain stores, read by the tensor core
        __syncwarp();
        if (lane == 0) mbar_arrive(full + st * 8u);
    }
    return true;
}

// one stage's products
template <int TN>
__device__ __forceinline__ void stage_products(uint32_t at, uint32_t d, uint32_t scales, bool first) {
    using Z = Tile<TN>;
#pragma unroll
    for (uint32_t h = 0; h < 2; h++) {
        copy_scales(scales + h * 4u, scale_desc(at + Z::ws_at + h * 512u));
#pragma unroll
        for (uint32_t b = 0; b < Z::blocks; b++) copy_scales(scales + 8u + (h * Z::blocks + b) * 4u, scale_desc(at + Z::xs_at + (h * Z::blocks + b) * 512u));
    }
    const uint64_t wd = tc_desc(at), xd = tc_desc(at + Z::x_at);
#pragma unroll
    for (uint32_t k = 0; k < 4; k++)
        mma_mx4(d, wd + 2u * k, xd + 2u * k, idesc_of(TN, (k & 1u) * 2u), scales + (k >> 1) * 4u, scales + 8u + (k >> 1) * Z::blocks * 4u, !first || k > 0);
}

__device__ __forceinline__ uint32_t clamp_row(int32_t o, uint32_t rows) { return o < 0 ? 0u : min((uint32_t)o, rows); }
// Which expert's rows [r0, r1) are pair `pair` of (expert, tile of TN rows): a warp walks over the experts, 32 at a time
struct Span { uint32_t e, r0, r1; };
template <int TN>
__device__ __forceinline__ Span span_of(const Mx4Product &p, uint32_t pair) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t run = 0;
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 32u) {
        const uint32_t e = e0 + lane;
        const uint32_t a = e < p.experts ? clamp_row(p.offsets[e], p.rows) : 0u, b = e < p.experts ? clamp_row(p.offsets[e + 1u], p.rows) : 0u, tiles = b > a ? (b - a + TN - 1u) / TN : 0u;
        uint32_t up = tiles;
#pragma unroll
        for (uint32_t o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, up, o); up += lane >= o ? x : 0u; }
        const uint32_t mine = __ballot_sync(0xffffffffu, run + up > pair);
        if (mine) {
            const int at = __ffs(mine) - 1;
            const uint32_t before = run + __shfl_sync(0xffffffffu, up - tiles, at), first = __shfl_sync(0xffffffffu, a, at) + (pair - before) * TN;
            return Span{e0 + at, first, min(first + TN, __shfl_sync(0xffffffffu, b, at))};
        }
        run += __shfl_sync(0xffffffffu, up, 31);
    }
    return Span{0u, 0u, 0u};
}

__device__ __forceinline__ void put(const Mx4Product &p, uint64_t row, uint32_t n, float v) {
    const uint64_t at = row * p.out_stride + n;
    if (p.out_type == T_F32) static_cast<float *>(p.out)[at] = v;
    else if (p.out_type == T_BF16) static_cast<__nv_bfloat16 *>(p.out)[at] = __float2bfloat16_rn(v);
    else static_cast<__half *>(p.out)[at] = __float2half_rn(v);
}
// J neighbouring rows' results of one output column, `live` of them
template <int J, typename T, typename F>
__device__ __forceinline__ void put_column(T *to, uint64_t stride, uint32_t live, F value) {
    if (live >= (uint32_t)J) {
#pragma unroll
        for (uint32_t j = 0; j < J; j++) to[j * stride] = value(j);
    } else
#pragma unroll
        for (uint32_t j = 0; j < J; j++) if (j < live) to[j * stride] = value(j);
}
template <int J>
__device__ __forceinline__ void put_rows(const Mx4Product &p, uint64_t row, uint32_t n, const float (&v)[J], uint32_t live) {
    const uint64_t at = row * p.out_stride + n;
    if (p.out_type == T_F32) put_column<J>(static_cast<float *>(p.out) + at, p.out_stride, live, [&](uint32_t j) { return v[j]; });
    else if (p.out_type == T_BF16) put_column<J>(static_cast<__nv_bfloat16 *>(p.out) + at, p.out_stride, live, [&](uint32_t j) { return __float2bfloat16_rn(v[j]); });
    else put_column<J>(static_cast<__half *>(p.out) + at, p.out_stride, live, [&](uint32_t j) { return __float2half_rn(v[j]); });
}

// grid (tiles of W x (pairs + 1 with experts), 1, ks), clusters of ks blocks that share a tile's depth
template <int TN>
__global__ void __launch_bounds__(192) k_mx4_tiles(const __grid_constant__ TcArgs t) {
    using Z = Tile<TN>;
    constexpr uint32_t ST = Z::stages;
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[2 * ST + 1];
    __shared__ uint32_t tmem_s, bad_s;
    __shared__ Span span_s;
    const Mx4Product &p = t.p;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, part = blockIdx.z, n0 = blockIdx.x % t.wtiles * kRows, pair = blockIdx.x / t.wtiles;
    const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u, full = smem_u32(bars), empty = full + ST * 8u, done = full + 2u * ST * 8u;
    Span span{0u, pair * TN, min(pair * TN + TN, p.rows)};
    if (p.offsets) {
        if (pair == t.pairs) {          // rows of no expert
            const uint32_t first = clamp_row(p.offsets[0], p.rows), last = clamp_row(p.offsets[p.experts], p.rows), n = n0 + threadIdx.x;
            if (threadIdx.x < kRows && n < p.outputs)
                for (uint32_t r = part; r < first + (p.rows - last); r += t.ks) put(p, r < first ? r : last + (r - first), n, 0.0f);
            pdl_wait();          // no block ends before the kernel that quantises
            return;
        }
        if (warp == 0) { const Span s = span_of<TN>(p, pair); if (lane == 0) span_s = s; }
        __syncthreads();
        span = span_s;
        if (span.r0 >= span.r1) { pdl_wait(); return; }          // (all blocks of a cluster)
    }
    if (threadIdx.x == 0) {
        bad_s = 0;
        for (uint32_t i = 0; i < ST; i++) { mbar_init(full + i * 8u, 3); mbar_init(empty + i * 8u, 1); }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) { tc_alloc(smem_u32(&tmem_s), Z::cols); tc_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s, scales_at = tmem + (TN < 32 ? 32u : TN), per = (t.steps + t.ks - 1u) / t.ks, s0 = min(t.steps, part * per), ns = min(t.steps, s0 + per) - s0;
    if (warp == 0 && lane == 0) {
        const uint32_t npre = min(ST, ns);
        auto weights = [&](uint32_t i) {
            const uint32_t st = i % ST;
            mbar_expect(full + st * 8u, Z::ws_at);
            tma_3d(ring + st * Z::bytes, &t.wmap, (s0 + i) * (kDepth / 2u), n0, span.e, full + st * 8u);
        };
        for (uint32_t i = 0; i < npre; i++) weights(i);          // these do not depend on the kernel before, which quantises the rows
        pdl_wait();
        for (uint32_t i = 0; i < ns; i++) {
            const uint32_t st = i % ST;
            if (i >= ST) {
                if (!soon(empty + st * 8u, ((i / ST) - 1u) & 1u)) { bad_s = 1; break; }
                weights(i);
            }
            tma_3d(ring + st * Z::bytes + Z::x_at, &t.xmap, (s0 + i) * (kDepth / 2u), span.r0, 0, full + st * 8u);
        }
    } else if (warp == 1 && lane == 0) {
        bool ok = true;
        for (uint32_t i = 0; i < ns; i++) {
            const uint32_t st = i % ST;
            ok = soon(full + st * 8u, (i / ST) & 1u);
            if (!ok) break;
            tc_fence_after();
            stage_products<TN>(ring + st * Z::bytes, tmem, scales_at + st * Z::scale_cols, i == 0);
            tc_commit(empty + st * 8u);
        }
        if (ok) tc_commit(done); else bad_s = 1;          // (the waits on it run out too)
    } else if (warp == 2) {
        ScaleWarp<1> w;
        w.groups = t.groups; w.align = t.w_align;
        w.at(p.ws + span.e * p.ws_expert + (uint64_t)n0 * p.ws_stride, p.ws_stride, p.outputs - n0, lane);
        if (!bring_scales(w, s0, ns, ring, Z::bytes, Z::ws_at, ST, full, empty, lane)) bad_s = 1;
    } else if (warp == 3) {
        pdl_wait();
        ScaleWarp<Z::blocks> w;
        w.groups = t.groups; w.align = t.x_align;
        w.at(p.xs + (uint64_t)span.r0 * p.xs_stride, p.xs_stride, span.r1 - span.r0, lane);
        if (!bring_scales(w, s0, ns, ring, Z::bytes, Z::xs_at, ST, full, empty, lane)) bad_s = 1;
    }
    __syncwarp();
    const uint32_t quad = warp & 3u, n = n0 + quad * 32u + lane;
    bool ok = true;
    if (warp >= 2) { ok = ns == 0 || soon_warp(done, 0); tc_fence_after(); if (!ok) bad_s = 1; }
    float *mine = reinterpret_cast<float *>(raw + (ring - smem_u32(raw))) + quad * 32u + lane;          // partial tiles, [TN][128], where the stages were
    if (warp >= 2) {
#pragma unroll 1
        for (uint32_t c = 0; c < TN; c += 16u) {
            if (span.r0 + c >= span.r1) break;
            uint32_t v[16];
            if (ns && ok) tc_ld16(tmem + ((quad * 32u) << 16) + c, v);
            float f[16];
#pragma unroll
            for (uint32_t j = 0; j < 16; j++) f[j] = !ok ? NAN : ns ? __uint_as_float(v[j]) : 0.0f;
            if (t.ks > 1) {
#pragma unroll
                for (uint32_t j = 0; j < 16; j++) mine[(c + j) * kRows] = f[j];
            } else if (n < p.outputs) put_rows<16>(p, span.r0 + c, n, f, span.r1 - span.r0 - c);
        }
    }
    if (t.ks > 1) {          // every block of the cluster finishes TN / ks rows, its parts added up in the order of the depth
        cluster_sync_all();
        if (warp >= 2 && n < p.outputs) {
            const uint32_t each = TN / t.ks, j1 = min((part + 1u) * each, span.r1 - span.r0), at = smem_u32(mine);
            for (uint32_t j = part * each; j < j1; j++) {
                float f = 0.0f;
                for (uint32_t q = 0; q < t.ks; q++) {
                    uint32_t peer;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at + j * kRows * 4u), "r"(q));
                    f += ld_cluster_f32(peer);
                }
                put(p, span.r0 + j, n, f);
            }
        }
        cluster_sync_all();          // no block leaves while another reads its part
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (bad_s) {          // copies still in flight land in this block's shared memory before it is given back
        const long long t0 = clock64();
        while (clock64() - t0 < 20000000ll) __nanosleep(1000);
    }
    if (warp == 1) tc_dealloc(tmem, Z::cols);
}

// ---- host side ----
typedef decltype(&cuTensorMapEncodeTiled) Encode;
Encode encoder() {
    static std::atomic<Encode> found{nullptr};
    Encode e = found.load(std::memory_order_acquire);
    if (e) return e;
    void *fn = nullptr;
    cudaDriverEntryPointQueryResult got;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &got) != cudaSuccess || got != cudaDriverEntryPointSuccess) return nullptr;
    e = reinterpret_cast<Encode>(fn);
    found.store(e, std::memory_order_release);
    return e;
}
// rows of codes in boxes of 128 bytes x `box`; what lies behind a row's last whole byte reads as zeros
bool map_of(CUtensorMap *m, const void *base, uint32_t columns, uint64_t rows, uint64_t experts, uint64_t stride, uint64_t expert, uint32_t box) {
    const uint64_t bytes = (columns + 1u) / 2u, least = (bytes + 15u) & ~15ull;
    if (rows == 1) stride = std::max<uint64_t>(stride, least);
    if (experts == 1) expert = std::max<uint64_t>(stride, least);
    const cuuint64_t dims[3] = {bytes, rows, experts}, strides[2] = {stride, expert};
    const cuuint32_t boxes[3] = {kDepth / 2u, box, 1}, step[3] = {1, 1, 1};
    const Encode e = encoder();
    return e && e(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(base), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TN>
cudaError_t launch_tiles(TcArgs &t, uint32_t pairs, cudaStream_t stream) {
    static std::atomic<uint64_t> asked{0};          // devices (of the first 64) whose shared-memory limit has been raised
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev > 63 || !(asked.load(std::memory_order_acquire) >> dev & 1u))) {
        e = smem_at_least(reinterpret_cast<const void *>(k_mx4_tiles<TN>), (int)Tile<TN>::smem);
        if (e == cudaSuccess && dev <= 63) asked.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (e != cudaSuccess) return e;
    if (!map_of(&t.xmap, t.p.x, t.p.columns, t.p.rows, 1, t.p.x_stride, 0, TN) || !map_of(&t.wmap, t.p.w, t.p.columns, t.p.outputs, std::max(1u, t.p.experts), t.p.w_stride, t.p.w_expert, kRows))
        return cudaErrorInvalidValue;
    t.pairs = pairs;
    const uint64_t tiles = (uint64_t)t.wtiles * pairs;
    t.ks = 1;
    while (t.ks < 8u && tiles * t.ks < 148u && t.steps >= 2u * t.ks) t.ks *= 2u;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((uint32_t)(t.wtiles * (pairs + (t.p.offsets ? 1u : 0u))), 1, t.ks); cfg.blockDim = dim3(192); cfg.dynamicSmemBytes = Tile<TN>::smem; cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (t.made) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (t.ks > 1) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = 1; attr[cfg.numAttrs].val.clusterDim.y = 1; attr[cfg.numAttrs++].val.clusterDim.z = t.ks;
    }
    return cudaLaunchKernelEx(&cfg, k_mx4_tiles<TN>, t);
}
uint32_t align_of(const void *base, uint64_t stride, uint64_t expert) {
    const uint64_t at = reinterpret_cast<uintptr_t>(base) | stride | expert;
    return at % 8u == 0 ? 8u : at % 4u == 0 ? 4u : 1u;
}

}  // namespace

cudaError_t mx4_tc_launch(const Mx4Product &a, bool made, cudaStream_t stream) {
    TcArgs t{};
    t.p = a; t.groups = mx4_groups(a.columns); t.steps = (t.groups + kStageGroups - 1u) / kStageGroups; t.wtiles = (a.outputs + kRows - 1u) / kRows; t.made = made;
    t.w_align = align_of(a.ws, a.ws_stride, a.ws_expert); t.x_align = align_of(a.xs, a.xs_stride, 0);
    const uint32_t each = a.offsets ? (a.rows + a.experts - 1u) / a.experts : a.rows;          // rows to a matrix, on average
    auto pairs = [&](uint32_t tn) { return a.offsets ? std::min(a.rows, a.rows / tn + std::min(a.rows, a.experts)) : (a.rows + tn - 1u) / tn; };
    if (each <= 16u) return launch_tiles<16>(t, pairs(16), stream);
    if (each <= 32u) return launch_tiles<32>(t, pairs(32), stream);
    if (each <= 64u) return launch_tiles<64>(t, pairs(64), stream);
    return launch_tiles<128>(t, pairs(128), stream);
}

}  // namespace nb
