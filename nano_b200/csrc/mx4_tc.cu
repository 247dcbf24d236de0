// mx4_tc.cu -- products of rows in microscaled 4-bit floating point on the fifth-generation tensor cores, which multiply the codes as they are (format: mx4.h).
//
// out^T = W X^T in tiles of 128 rows of W x TN rows of X: tcgen05.mma kind::mxf4 takes 64 columns of both and two scales for each row, which lie in tensor memory.
// A stage is 256 columns: codes by cp.async.bulk.tensor into 128-byte-swizzled rows, scales by four warps.  A lane of tensor memory is an output column, so a warp's stores of one row are
// neighbours.
// Every wait has a limit; a block in which one runs out leaves with NaN in its results, those of a tile that it shares among them.
// Products are named rows x outputs x columns, times are those on the device with W in memory, not in L2.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "family.h"
#include "mx4.cuh"
#include "mx4.h"
#include "rows.cuh"
#include "tc_ptx.cuh"

namespace nb {
namespace {

constexpr uint32_t kRows = 128, kDepth = 256, kStageGroups = kDepth / kMx4Group, kMostExperts = 1024;          // rows of W in a tile; columns of a stage
template <int TN> struct Tile {
    static constexpr uint32_t blocks = (TN + 127) / 128;          // of 128 rows, as tensor memory holds scales: row r's word in lane r % 32, column r / 32
    static constexpr uint32_t x_at = kRows * 128u;          // in a stage
    static constexpr uint32_t scale_cols = 8u + 8u * blocks, sum_cols = TN < 32 ? 32 : TN;          // of tensor memory
    static constexpr uint32_t staged = (kRows + 128u * blocks) * 16u;          // two stages' scales, sixteen to a row, on their way
};
__host__ __device__ constexpr uint32_t cols_for(uint32_t used) { return used <= 128u ? 128u : used <= 256u ? 256u : 512u; }

struct alignas(64) TcArgs { CUtensorMap wmap, xmap; Mx4Product p; uint64_t w_step, x_step; uint32_t groups, steps, ks, per, wtiles, pairs, w_unit, x_unit, made; };

__device__ __forceinline__ bool soon(uint32_t bar, uint32_t parity) { return mbar_try(bar, parity) || mbar_wait(bar, parity); }
__device__ __forceinline__ bool soon_warp(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, soon(bar, parity)); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// d (+)= a b^T: 64 columns of 128 rows of codes and of the instruction's N, each with its two scales.  PAIR: two blocks' 128 rows each, and half of the N rows in each block's shared memory; sums and
// scales of a block's rows, and those of all N, are in its own tensor memory
template <bool PAIR>
__device__ __forceinline__ void mma_mx4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t a_scales, uint32_t b_scales, bool add) {
    if constexpr (PAIR)
        asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %6, 0;\ntcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"((uint32_t)add) : "memory");
    else
        asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %6, 0;\ntcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"((uint32_t)add) : "memory");
}
// e2m1 x e2m1, scales in 8 bits of exponent, N columns; scales from byte `id` (0 or 2) of their words
__host__ __device__ constexpr uint32_t idesc_of(uint32_t m, uint32_t n, uint32_t id) { return (id << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24) | (id << 29); }

// Sixteen neighbouring scales of a row, from group g (a multiple of 16, or of 8 for UNIT 8) on; zeros behind its last.  UNIT: bytes that one load may bring, for every row and every g
template <int UNIT>
__device__ __forceinline__ uint4 scales16(const uint8_t *at, uint32_t g, uint32_t groups) {
    if constexpr (UNIT == 16) return __ldg(reinterpret_cast<const uint4 *>(at));
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if constexpr (UNIT == 8) {
        uint2 lo = make_uint2(0u, 0u), hi = lo;
        if (g < groups) lo = __ldg(reinterpret_cast<const uint2 *>(at));
        if (g + 8u < groups) hi = __ldg(reinterpret_cast<const uint2 *>(at) + 1);
        return make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else if constexpr (UNIT == 4) {
        if (g < groups) v.x = __ldg(reinterpret_cast<const uint32_t *>(at));
        if (g + 4u < groups) v.y = __ldg(reinterpret_cast<const uint32_t *>(at) + 1);
        if (g + 8u < groups) v.z = __ldg(reinterpret_cast<const uint32_t *>(at) + 2);
        if (g + 12u < groups) v.w = __ldg(reinterpret_cast<const uint32_t *>(at) + 3);
    } else {
        uint32_t w[4] = {};
#pragma unroll
        for (uint32_t i = 0; i < 16; i++) w[i / 4] |= (g + i < groups ? (uint32_t)__ldg(at + i) : 0u) << (8u * (i % 4u));
        v = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return v;
}

// Four warps bring the scales of tile after tile to tensor memory: a thread loads those of one row of W and of one or two of X, eight at a time and kAhead stages ahead, the four exchange them
// through shared memory, and each writes all of them to its quarter of the lanes.  (tcgen05.cp, which replicates by itself, takes its turn with the products, some 55 cycles for each 128 x 4
// scales, a quarter of a stage of 128 x 256: 8192 x 8192 x 8192 took 266 us with it.)  Pairs of SMs, whose ring has six stages, hand two of them over at once: one wait for the
// stores of both (8192 x 8192 x 8192 212 us, one by one 227); shorter rings would run dry.
constexpr uint32_t kAhead = 2, kScaleThreads = 128, kScaleBar = 1;
__device__ __forceinline__ void tc_st8(uint32_t addr, const uint32_t (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t bar, uint32_t rank) {          // at the same barrier of block `rank`
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(bar), "r"(rank));
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(there) : "memory");
}
struct ScaleRows { const uint8_t *base; uint64_t stride; uint32_t live; };          // rows [0, live); what lies behind them counts for nothing
struct ScaleRing { uint32_t staged, tmem, stages, full, empty, groups; uint64_t w_step, x_step; uint32_t w_unit, x_unit; };
template <int TN, bool PAIR, int WU, int XU, typename F>
__device__ __forceinline__ bool bring_scales(const ScaleRing &r, uint32_t tiles, uint32_t s0, uint32_t ns, F &next) {
    using Z = Tile<TN>;
    constexpr uint32_t XR = Z::blocks;          // rows of X to a thread
    const uint32_t tid = threadIdx.x & (kScaleThreads - 1u), warp = tid >> 5, lane = tid & 31u, pairs = (ns + 1u) / 2u, total = tiles * pairs;          // two stages at a time
    const uint8_t *w_row = nullptr, *x_row[XR] = {};
    uint4 v[kAhead][1 + XR];
    uint32_t asked = 0, pair = pairs;
    auto ask = [&](uint4 (&to)[1 + XR]) {
        if (asked == total) return;
        if (pair == pairs) {
            ScaleRows w, x;
            next(w, x);
            w_row = w.base + (tid < w.live ? tid : 0u) * w.stride + (s0 >> 1) * r.w_step + (s0 & 1u) * 8u;
#pragma unroll
            for (uint32_t i = 0; i < XR; i++) { const uint32_t q = tid + i * kScaleThreads; x_row[i] = x.base + (q < x.live ? q : 0u) * x.stride + (s0 >> 1) * r.x_step + (s0 & 1u) * 8u; }
            pair = 0;
        }
        const uint32_t g = (s0 + 2u * pair) * kStageGroups;
        to[0] = scales16<WU>(w_row, g, r.groups);
        w_row += r.w_step;
#pragma unroll
        for (uint32_t i = 0; i < XR; i++) { to[1 + i] = scales16<XU>(x_row[i], g, r.groups); x_row[i] += r.x_step; }
        pair++; asked++;
    };
#pragma unroll
    for (uint32_t d = 0; d < kAhead; d++) ask(v[d]);
    uint32_t st = 0, turn = 0, done = 0;
    bool ok = true;
    for (uint32_t i = 0; i < total; i += kAhead)
#pragma unroll
        for (uint32_t d = 0; d < kAhead; d++) {
            if (i + d >= total) return ok;
            const uint32_t at = r.staged + (d & 1u) * Z::staged, count = min(2u, ns - done);          // (two buffers in turn: kAhead is even)
#pragma unroll
            for (uint32_t j = 0; j < 1 + XR; j++) {          // the two stages' apart: neighbours, for the loads
                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + (j * kScaleThreads + tid) * 8u), "r"(v[d][j].x), "r"(v[d][j].y) : "memory");
                asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + Z::staged / 2u + (j * kScaleThreads + tid) * 8u), "r"(v[d][j].z), "r"(v[d][j].w) : "memory");
            }
            const uint32_t st1 = st + 1u == r.stages ? 0u : st + 1u, turn1 = st1 ? turn : turn + 1u;          // the second of the two
            ok = ok && (!turn || soon_warp(r.empty + st * 8u, (turn - 1u) & 1u));
            if constexpr (PAIR) ok = ok && (count < 2u || !turn1 || soon_warp(r.empty + st1 * 8u, (turn1 - 1u) & 1u));
            if (bar_any(kScaleBar, kScaleThreads, !ok)) return false;          // one verdict for the four warps, which meet here
            ask(v[d]);
            auto write = [&](uint32_t from, uint32_t st) {
                uint32_t w[8], x[8 * XR];          // [half of the stage][row / 32]
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[j]), "=r"(w[4 + j]) : "r"(from + (j * 32u + lane) * 8u) : "memory");
#pragma unroll
                for (uint32_t j = 0; j < 4 * XR; j++) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x[j]), "=r"(x[4 * XR + j]) : "r"(from + (kRows + j * 32u + lane) * 8u) : "memory");
                const uint32_t to = r.tmem + ((warp * 32u) << 16) + st * Z::scale_cols;
                tc_st8(to, w);
                if constexpr (XR == 1) tc_st8(to + 8u, x); else tc_st16(to + 8u, x);
            };
            if constexpr (PAIR) {
                tc_fence_after();
                write(at, st);
                if (count == 2u) write(at + Z::staged / 2u, st1);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane < count) arrive_at(r.full + (lane ? st1 : st) * 8u, 0);
                st += count;
                if (st >= r.stages) { st -= r.stages; turn++; }
            } else
                for (uint32_t h = 0; h < count; h++) {
                    if (h && turn) {          // (the others learn of a wait that runs out where they meet again)
                        ok = soon_warp(r.empty + st * 8u, (turn - 1u) & 1u);
                        if (!ok) break;
                    }
                    tc_fence_after();
                    write(at + h * (Z::staged / 2u), st);
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(r.full + st * 8u);
                    if (++st == r.stages) { st = 0; turn++; }
                }
            done = done + count == ns ? 0u : done + count;
        }
    return ok;
}
// next(w, x) names the rows of the next of `tiles` tiles, of which steps [s0, s0 + ns) of the depth are wanted
template <int TN, bool PAIR, typename F>
__device__ __forceinline__ bool bring_scales(const ScaleRing &r, uint32_t tiles, uint32_t s0, uint32_t ns, F next) {
    if (r.x_unit == 16u) {
        if (r.w_unit == 16u) return bring_scales<TN, PAIR, 16, 16>(r, tiles, s0, ns, next);
        if (r.w_unit >= 4u) return bring_scales<TN, PAIR, 4, 16>(r, tiles, s0, ns, next);
        return bring_scales<TN, PAIR, 1, 16>(r, tiles, s0, ns, next);
    }
    if (r.w_unit >= 8u && r.x_unit >= 8u) return bring_scales<TN, PAIR, 8, 8>(r, tiles, s0, ns, next);
    if (r.w_unit >= 4u && r.x_unit >= 4u) return bring_scales<TN, PAIR, 4, 4>(r, tiles, s0, ns, next);
    return bring_scales<TN, PAIR, 1, 1>(r, tiles, s0, ns, next);
}

// Rows of X that are numbers, up to 16 of them: the same four warps quantise all that their block needs of them while W's first stages are on their way, a group to a thread, into swizzled rows as a
// bulk copy would leave them.  Every block of a tile does so for itself: a launch and a wait less than quantising first.
struct RawRows { const void *x; uint64_t stride; uint32_t r0, live, columns; };
constexpr uint32_t kRawStep = 16u * 128u, kRawScales = 16u * kStageGroups, kRawStages = 5;          // bytes of codes and of scales of a step of the depth; stages of W
// Steps of the depth that a block has room for where an SM has two blocks of 113 KB: beside W's stages and their alignment, two stages' scales of W and the barriers, 13.  us, so / by a kernel before, with
// 11 steps: 1 x 9728 x 2816 7.9 / 8.7 (10.5 / 15 a call), 1 x 16000 x 2816 9.1 / 9.4
constexpr uint32_t kRawSteps = (113u * 1024u - kRawStages * kRows * 128u - 1024u - 2u * kRows * 16u - 256u) / (kRawStep + kRawScales);
template <typename T>
__device__ __forceinline__ void quantise_rows(const RawRows &x, uint32_t s0, uint32_t ns, uint32_t codes, uint32_t scales) {
    const uint32_t tid = threadIdx.x & (kScaleThreads - 1u), per_row = ns * kStageGroups;
    for (uint32_t i = tid; i < x.live * per_row; i += kScaleThreads) {
        const uint32_t row = i / per_row, g = i - row * per_row, step = g / kStageGroups, c = g % kStageGroups, k = (s0 * kStageGroups + g) * kMx4Group;
        const T *first = static_cast<const T *>(x.x) + (uint64_t)(x.r0 + row) * x.stride;
        float v[kMx4Group];
        if ((reinterpret_cast<uintptr_t>(first) & 15u) == 0 && k + kMx4Group <= x.columns) load_row<EVEN>(first, x.columns, (int)k, v);
        else load_row<ANY>(first, x.columns, (int)k, v);
        const uint32_t e = scale_byte(top_bits(v));
        const float by = inverse_of(e);
#pragma unroll
        for (uint32_t j = 0; j < kMx4Group; j++) v[j] *= by;
        const uint32_t w[4] = {codes_of(v), codes_of(v + 8), codes_of(v + 16), codes_of(v + 24)};
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(codes + step * kRawStep + row * 128u + ((c ^ (row & 7u)) << 4)), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
        asm volatile("st.shared.u8 [%0], %1;" ::"r"(scales + step * kRawScales + row * kStageGroups + c), "r"(e) : "memory");
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");          // plain stores, read by the tensor core
}
// (codes of a group that is NaN may be anything: its scale makes every product NaN, and rows behind the last have no results)
template <int WU>
__device__ __forceinline__ bool bring_w_scales(const ScaleRing &r, const ScaleRows &w, uint32_t x_scales, uint32_t s0, uint32_t ns) {
    using Z = Tile<16>;
    const uint32_t tid = threadIdx.x & (kScaleThreads - 1u), warp = tid >> 5, lane = tid & 31u;
    const uint8_t *w_row = w.base + (tid < w.live ? tid : 0u) * w.stride;
    uint4 v[2];
    auto ask = [&](uint32_t i, uint4 &to) { const uint32_t step = s0 + i; if (i < ns) to = scales16<WU>(w_row + (step >> 1) * r.w_step + (step & 1u) * 8u, step * kStageGroups, r.groups); };
    ask(0, v[0]); ask(2, v[1]);
    bool ok = true;
    uint32_t st = 0, turn = 0;
    for (uint32_t i0 = 0; i0 < ns; i0 += 4u)
#pragma unroll
        for (uint32_t d = 0; d < 2; d++) {
            const uint32_t i = i0 + 2u * d, at = r.staged + d * kRows * 16u;
            if (i >= ns) return ok;
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + tid * 8u), "r"(v[d].x), "r"(v[d].y) : "memory");
            asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at + kRows * 8u + tid * 8u), "r"(v[d].z), "r"(v[d].w) : "memory");
            ok = ok && (!turn || soon_warp(r.empty + st * 8u, (turn - 1u) & 1u));
            if (bar_any(kScaleBar, kScaleThreads, !ok)) return false;
            ask(i + 4u, v[d]);
            for (uint32_t h = 0; h < min(2u, ns - i); h++) {
                if (h && turn) { ok = soon_warp(r.empty + st * 8u, (turn - 1u) & 1u); if (!ok) break; }
                tc_fence_after();
                uint32_t wv[8], xv[8] = {};
#pragma unroll
                for (uint32_t j = 0; j < 4; j++) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(wv[j]), "=r"(wv[4 + j]) : "r"(at + h * kRows * 8u + (j * 32u + lane) * 8u) : "memory");
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(xv[0]), "=r"(xv[4]) : "r"(x_scales + (i + h) * kRawScales + (lane & 15u) * 8u) : "memory");
                const uint32_t to = r.tmem + ((warp * 32u) << 16) + st * Z::scale_cols;
                tc_st8(to, wv);
                tc_st8(to + 8u, xv);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(r.full + st * 8u);
                if (++st == r.stages) { st = 0; turn++; }
            }
        }
    return ok;
}

// a stage's products
template <int TN, bool PAIR = false>
__device__ __forceinline__ void stage_products(uint32_t w_at, uint32_t x_at, uint32_t d, uint32_t scales, bool first) {
    using Z = Tile<TN>;
    const uint64_t wd = tc_desc(w_at), xd = tc_desc(x_at);
#pragma unroll
    for (uint32_t k = 0; k < 4; k++)
        mma_mx4<PAIR>(d, wd + 2u * k, xd + 2u * k, idesc_of(PAIR ? 2u * kRows : kRows, TN, (k & 1u) * 2u), scales + (k >> 1) * 4u, scales + 8u + (k >> 1) * Z::blocks * 4u, !first || k > 0);
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

// Of a tile whose parts lie in the blocks of a cluster, block `part` finishes J rows in every J * ks: the parts added up in the order of the depth.  As many rows at once as there may be: a
// word of another block is some 200 ns away.  lost: 0, or NaN in a block without its sums, whose part may be anything
template <int J>
__device__ __forceinline__ void finish_parts(const Mx4Product &p, uint32_t at, uint32_t lost, uint32_t part, uint32_t ks, uint32_t r0, uint32_t n, uint32_t rows) {
    for (uint32_t j = part * J; j < rows; j += ks * J) {
        float f[J] = {}, none = 0.0f;
#pragma unroll 2
        for (uint32_t q = 0; q < ks; q++) {
            uint32_t peer, peer_lost;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer) : "r"(at + j * kRows * 4u), "r"(q));
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(peer_lost) : "r"(lost), "r"(q));
            none += ld_cluster_f32(peer_lost);
            float v[J];
#pragma unroll
            for (uint32_t i = 0; i < J; i++) v[i] = ld_cluster_f32(peer + i * kRows * 4u);          // (a part has all TN rows' places)
#pragma unroll
            for (uint32_t i = 0; i < J; i++) f[i] += v[i];
        }
#pragma unroll
        for (uint32_t i = 0; i < J; i++) f[i] += none;          // (a sum that began with +0 is not -0: adding 0 changes none)
        put_rows<J>(p, r0 + j, n, f, rows - j);
    }
}

// ------------------------------------------------------------------------------------------------
// Few tiles: a tile's depth is shared by a cluster of ks blocks, each of which finishes some of its rows.  grid (tiles of W x (pairs + 1 with experts), 1, ks)
// ------------------------------------------------------------------------------------------------
template <int TN> struct Few {
    static constexpr uint32_t stages = TN <= 32 ? kRawStages : TN <= 64 ? 4 : 3, cols = cols_for(Tile<TN>::sum_cols + stages * Tile<TN>::scale_cols);          // up to 107 KB: two blocks to an SM
    // codes that bulk copies read come with W's stage by stage; numbers are quantised to a place of their own
    static __host__ __device__ constexpr uint32_t stage(uint32_t x) { return (kRows + (x == T_MX4 ? TN : 0u)) * 128u; }
    static __host__ __device__ constexpr uint32_t smem(uint32_t x) { return stages * stage(x) + (x == T_MX4 ? 0u : kRawSteps * kRawStep) + 1024u; }
};
// X: what the rows of X are, codes that bulk copies read or numbers
template <int TN, uint32_t X>
__global__ void __launch_bounds__(192) k_mx4_few(const __grid_constant__ TcArgs t) {
    using Z = Tile<TN>;
    constexpr uint32_t ST = Few<TN>::stages, SB = Few<TN>::stage(X);
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[2 * ST + 1];
    __shared__ __align__(16) uint8_t staged[X == T_MX4 ? 2u * Z::staged : 2u * kRows * 16u + kRawSteps * kRawScales];
    __shared__ uint32_t tmem_s, bad_s;
    __shared__ float lost_s;
    __shared__ Span span_s;
    const Mx4Product &p = t.p;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, part = blockIdx.z, n0 = blockIdx.x % t.wtiles * kRows, pair = blockIdx.x / t.wtiles;
    const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u, full = smem_u32(bars), empty = full + ST * 8u, done = full + 2u * ST * 8u, raw_at = ring + ST * SB;
    const uint32_t s0 = min(t.steps, part * t.per), ns = min(t.steps, s0 + t.per) - s0;
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
    auto weights = [&](uint32_t i) {
        const uint32_t st = i % ST;
        mbar_expect(full + st * 8u, SB);
        tma_3d(ring + st * SB, &t.wmap, (s0 + i) * (kDepth / 2u), n0, span.e, full + st * 8u);
    };
    const uint32_t npre = min(ST, ns), rows = span.r1 - span.r0;
    if (threadIdx.x == 128u) {
        bad_s = 0; lost_s = 0.0f;
        for (uint32_t i = 0; i < ST; i++) { mbar_init(full + i * 8u, 5); mbar_init(empty + i * 8u, 1); }
        mbar_init(done, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (uint32_t i = 0; i < npre; i++) weights(i);          // these do not depend on the kernel before, which quantises the rows
    }
    if (warp == 5) { tc_alloc(smem_u32(&tmem_s), Few<TN>::cols); tc_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s, scales_at = tmem + Z::sum_cols;
    if (warp == 4) {
        if (lane == 0) {
            pdl_wait();
            for (uint32_t i = 0; i < ns; i++) {
                const uint32_t st = i % ST;
                if (i >= ST) {
                    if (!soon(empty + st * 8u, ((i / ST) - 1u) & 1u)) { bad_s = 1; break; }
                    weights(i);
                }
                if (X == T_MX4) tma_3d(ring + st * SB + Z::x_at, &t.xmap, (s0 + i) * (kDepth / 2u), span.r0, 0, full + st * 8u);
            }
        }
    } else if (warp == 5) {
        if (lane == 0) {
            bool ok = true;
            for (uint32_t i = 0; i < ns; i++) {
                const uint32_t st = i % ST;
                ok = soon(full + st * 8u, (i / ST) & 1u);
                if (!ok) break;
                tc_fence_after();
                stage_products<TN>(ring + st * SB, X == T_MX4 ? ring + st * SB + Z::x_at : raw_at + i * kRawStep, tmem, scales_at + st * Z::scale_cols, i == 0);
                tc_commit(empty + st * 8u);
            }
            if (ok) tc_commit(done); else bad_s = 1;          // (the waits on it run out too)
        }
    } else {
        pdl_wait();
        const ScaleRing r{smem_u32(staged), scales_at, ST, full, empty, t.groups, t.w_step, t.x_step, t.w_unit, t.x_unit};
        const ScaleRows w_rows{p.ws + span.e * p.ws_expert + (uint64_t)n0 * p.ws_stride, p.ws_stride, p.outputs - n0};
        bool brought;
        if constexpr (X == T_MX4) brought = bring_scales<TN, false>(r, 1, s0, ns, [&](ScaleRows &w, ScaleRows &x) { w = w_rows; x = ScaleRows{p.xs + (uint64_t)span.r0 * p.xs_stride, p.xs_stride, span.r1 - span.r0}; });
        else {
            typedef std::conditional_t<X == T_F32, float, std::conditional_t<X == T_BF16, __nv_bfloat16, __half>> T;
            const uint32_t x_scales = r.staged + 2u * kRows * 16u;
            quantise_rows<T>(RawRows{p.x, p.x_stride, span.r0, rows, p.columns}, s0, ns, raw_at, x_scales);
            brought = r.w_unit >= 8u ? bring_w_scales<8>(r, w_rows, x_scales, s0, ns) : r.w_unit >= 4u ? bring_w_scales<4>(r, w_rows, x_scales, s0, ns) : bring_w_scales<1>(r, w_rows, x_scales, s0, ns);
        }
        if (!brought) bad_s = 1;
    }
    __syncwarp();
    const uint32_t quad = warp & 3u, n = n0 + quad * 32u + lane;
    bool ok = true;
    if (warp < 4) { ok = ns == 0 || soon_warp(done, 0); tc_fence_after(); if (!ok) { bad_s = 1; lost_s = NAN; } }
    float *mine = reinterpret_cast<float *>(raw + (ring - smem_u32(raw))) + quad * 32u + lane;          // partial tiles, [TN][128], where the stages were (and, where a wait ran out, copies may still land)
    if (warp < 4) {
#pragma unroll 1
        for (uint32_t c = 0; c < TN; c += 16u) {
            if (c >= rows) break;
            uint32_t v[16];
            if (ns && ok) tc_ld16(tmem + ((quad * 32u) << 16) + c, v);
            float f[16];
#pragma unroll
            for (uint32_t j = 0; j < 16; j++) f[j] = !ok ? NAN : ns ? __uint_as_float(v[j]) : 0.0f;
            if (t.ks > 1) {
#pragma unroll
                for (uint32_t j = 0; j < 16; j++) mine[(c + j) * kRows] = f[j];
            } else if (n < p.outputs) put_rows<16>(p, span.r0 + c, n, f, rows - c);
        }
    }
    if (t.ks > 1) {          // every block of the cluster finishes some of the tile's rows, in turn, its parts added up in the order of the depth
        cluster_sync_all();
        if (warp < 4 && n < p.outputs) {
            if (TN >= 32 && rows > 4u * t.ks) finish_parts<16>(p, smem_u32(mine), smem_u32(&lost_s), part, t.ks, span.r0, n, rows);
            else finish_parts<4>(p, smem_u32(mine), smem_u32(&lost_s), part, t.ks, span.r0, n, rows);
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
    if (warp == 5) tc_dealloc(tmem, Few<TN>::cols);
}

// ------------------------------------------------------------------------------------------------
// Many tiles: a block to each SM takes tiles in turn.  Codes and scales run ahead of the products over the tiles' borders, and a tile's results are written while the next one's products run: in
// another set of columns of tensor memory (tiles of up to 128 rows of X), or, of 256, after the sums have been read out at once, 128 columns to a thread.
// ------------------------------------------------------------------------------------------------
// PAIR: two blocks of a cluster share tiles of 256 x TN, 128 rows of W and half of the rows of X to each: a block's shared memory takes in and gives out two thirds of the bytes, and so does L2
// (8192 x 8192 x 8192 225 us instead of 244 with a block to a tile of 128 x 256, 8192 x 9728 x 2560 102 instead of 106; with scales handed over in twos 212, 5.2 PFLOP/s, and 100).  The
// first block issues the products of both; all copies and scales count on its barriers.
template <int TN, bool PAIR> struct Many {
    static_assert(PAIR == (TN == 256));
    static constexpr uint32_t stages = TN <= 16 ? 11 : TN <= 32 ? 10 : TN <= 64 ? 8 : 6, sets = TN <= 128 ? 2 : 1, drain = TN <= 32 ? 4 : 8, columns = TN / (drain / 4);          // (columns of a thread)
    static constexpr uint32_t tma = 4 + drain, mma = 5 + drain;          // warps 0-3: scales, then those that write results, then one each
    static constexpr uint32_t x_rows = PAIR ? TN / 2 : TN, bytes = (kRows + x_rows) * 128u;          // of a stage
    static constexpr uint32_t cols = cols_for(sets * Tile<TN>::sum_cols + stages * Tile<TN>::scale_cols), threads = 32u * (drain + 6u), smem = stages * bytes + 1024u;
};
// a bulk copy to this block's memory that counts on the first block's barrier
__device__ __forceinline__ void tma_pair(uint32_t dst, const CUtensorMap *map, uint32_t x, uint32_t y, uint32_t z, uint32_t bar) {
    uint32_t there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(bar), "r"(0));
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(there) : "memory");
}
__device__ __forceinline__ void commit_both(uint32_t bar) {          // to the barrier of both blocks
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
template <int TN, bool PAIR>
__global__ void __launch_bounds__(Many<TN, PAIR>::threads, 1) k_mx4_many(const __grid_constant__ TcArgs t) {
    using Z = Tile<TN>;
    using Y = Many<TN, PAIR>;
    constexpr uint32_t ST = Y::stages, SETS = Y::sets, SB = Y::bytes, WIDE = PAIR ? 2u * kRows : kRows;          // WIDE: rows of W in a tile
    extern __shared__ uint8_t raw[];
    __shared__ __align__(8) uint64_t bars[2 * ST + 2 * SETS];
    __shared__ __align__(16) uint8_t staged[2 * Z::staged];
    __shared__ uint32_t tmem_s, bad_s, pairs_s[kMostExperts + 1];          // of (expert, TN rows): those before an expert's
    const Mx4Product &p = t.p;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, rank = PAIR ? blockIdx.x & 1u : 0u, first_tile = PAIR ? blockIdx.x / 2u : blockIdx.x, stride = PAIR ? gridDim.x / 2u : gridDim.x;
    const uint32_t ring = (smem_u32(raw) + 1023u) & ~1023u, full = smem_u32(bars), empty = full + ST * 8u, sums = full + 2u * ST * 8u, room = sums + SETS * 8u;
    if (threadIdx.x == 0) {
        bad_s = 0;
        for (uint32_t i = 0; i < ST; i++) { mbar_init(full + i * 8u, PAIR ? 9 : 5); mbar_init(empty + i * 8u, 1); }
        for (uint32_t i = 0; i < SETS; i++) { mbar_init(sums + i * 8u, 1); mbar_init(room + i * 8u, PAIR ? 2u * Y::drain : Y::drain); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == Y::mma) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(Y::cols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else { tc_alloc(smem_u32(&tmem_s), Y::cols); tc_relinquish(); }
    }
    if (p.offsets && warp == Y::tma) {
        uint32_t run = 0;
        for (uint32_t e0 = 0; e0 < p.experts; e0 += 32u) {
            const uint32_t e = e0 + lane, a = e < p.experts ? clamp_row(p.offsets[e], p.rows) : 0u, b = e < p.experts ? clamp_row(p.offsets[e + 1u], p.rows) : 0u, tiles = b > a ? (b - a + TN - 1u) / TN : 0u;
            uint32_t up = tiles;
#pragma unroll
            for (uint32_t o = 1; o < 32; o <<= 1) { const uint32_t x = __shfl_up_sync(0xffffffffu, up, o); up += lane >= o ? x : 0u; }
            if (e < p.experts) pairs_s[e] = run + up - tiles;
            run += __shfl_sync(0xffffffffu, up, 31);
        }
        if (lane == 0) pairs_s[p.experts] = run;
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();          // both blocks' barriers are there
    tc_fence_after();
    const uint32_t tmem = tmem_s, scales_at = tmem + SETS * Z::sum_cols, ns = t.steps;
    const uint64_t tiles = (uint64_t)t.wtiles * (p.offsets ? pairs_s[p.experts] : t.pairs), mine = tiles > first_tile ? (tiles - 1u - first_tile) / stride + 1u : 0u;
    uint32_t e_now = 0;
    auto span = [&](uint64_t tile) {          // tiles come in ascending order
        const uint32_t pair = (uint32_t)(tile / t.wtiles);
        if (!p.offsets) return Span{0u, pair * TN, min(pair * TN + TN, p.rows)};
        while (pairs_s[e_now + 1u] <= pair) e_now++;
        const uint32_t r0 = clamp_row(p.offsets[e_now], p.rows) + (pair - pairs_s[e_now]) * TN;
        return Span{e_now, r0, min(r0 + TN, clamp_row(p.offsets[e_now + 1u], p.rows))};
    };
    if (warp == Y::tma) {
        if (lane == 0) {
            bool ok = true, waited = false;
            uint32_t st = 0, turn = 0;
            for (uint64_t tile = first_tile; tile < tiles && ok; tile += stride) {
                const Span s = span(tile);
                const uint32_t n0 = (uint32_t)(tile % t.wtiles) * WIDE + rank * kRows;
                auto weights = [&](uint32_t i, uint32_t at) {
                    if (rank == 0) mbar_expect(full + at * 8u, PAIR ? 2u * SB : SB);          // of both blocks
                    if constexpr (PAIR) tma_pair(ring + at * SB, &t.wmap, i * (kDepth / 2u), n0, s.e, full + at * 8u);
                    else tma_3d(ring + at * SB, &t.wmap, i * (kDepth / 2u), n0, s.e, full + at * 8u);
                };
                uint32_t early = 0;
                if (!waited) {          // the first tile's weights do not depend on the kernel before, which quantises the rows
                    for (; early < min(ST, ns); early++) weights(early, early);
                    pdl_wait();
                    waited = true;
                }
                for (uint32_t i = 0; i < ns; i++) {
                    ok = !turn || soon(empty + st * 8u, (turn - 1u) & 1u);
                    if (!ok) { bad_s = 1; break; }
                    if (i >= early) weights(i, st);
                    if constexpr (PAIR) tma_pair(ring + st * SB + Z::x_at, &t.xmap, i * (kDepth / 2u), s.r0 + rank * Y::x_rows, 0, full + st * 8u);
                    else tma_3d(ring + st * SB + Z::x_at, &t.xmap, i * (kDepth / 2u), s.r0, 0, full + st * 8u);
                    if (++st == ST) { st = 0; turn++; }
                }
            }
        }
    } else if (warp == Y::mma) {
        if (lane == 0 && rank == 0) {
            bool ok = true;
            uint32_t st = 0, phase = 0, set = 0, turn = 0;
            for (uint64_t n = 0; n < mine && ok; n++) {
                ok = !turn || soon(room + set * 8u, (turn - 1u) & 1u);
                if (!ok) break;
                tc_fence_after();
                for (uint32_t i = 0; i < ns; i++) {
                    ok = soon(full + st * 8u, phase);
                    if (!ok) break;
                    tc_fence_after();
                    stage_products<TN, PAIR>(ring + st * SB, ring + st * SB + Z::x_at, tmem + set * Z::sum_cols, scales_at + st * Z::scale_cols, i == 0);
                    if constexpr (PAIR) commit_both(empty + st * 8u); else tc_commit(empty + st * 8u);
                    if (++st == ST) { st = 0; phase ^= 1u; }
                }
                if (ok) { if constexpr (PAIR) commit_both(sums + set * 8u); else tc_commit(sums + set * 8u); }
                if (++set == SETS) { set = 0; turn++; }
            }
            if (!ok) bad_s = 1;
        }
    } else if (warp < 4) {
        pdl_wait();
        uint64_t tile = first_tile;
        const ScaleRing r{smem_u32(staged), scales_at, ST, full, empty, t.groups, t.w_step, t.x_step, t.w_unit, t.x_unit};
        if (!bring_scales<TN, PAIR>(r, (uint32_t)mine, 0, ns, [&](ScaleRows &w, ScaleRows &x) {
                const Span s = span(tile);
                const uint32_t n0 = (uint32_t)(tile % t.wtiles) * WIDE + rank * kRows, from = min(n0, p.outputs - 1u);          // (the second block's rows may lie behind the last)
                w = ScaleRows{p.ws + s.e * p.ws_expert + (uint64_t)from * p.ws_stride, p.ws_stride, p.outputs - from};
                x = ScaleRows{p.xs + (uint64_t)s.r0 * p.xs_stride, p.xs_stride, s.r1 - s.r0};
                tile += stride;
            })) bad_s = 1;
    } else {
        constexpr uint32_t CO = Y::columns, LD = CO < 32 ? 16 : 32, HELD = CO < 64 ? CO : 64;          // sums that a thread reads at once: 64 of fp32, all in 16 bits
        const uint32_t quad = warp & 3u, c0 = ((warp - 4u) >> 2) * CO;
        bool ok = true;
        for (uint64_t i = 0; i < mine; i++) {
            const uint64_t tile = first_tile + i * stride;
            const uint32_t set = (uint32_t)i % SETS, n = (uint32_t)(tile % t.wtiles) * WIDE + rank * kRows + quad * 32u + lane;
            const Span s = span(tile);
            ok = ok && soon_warp(sums + set * 8u, (uint32_t)(i / SETS) & 1u);
            tc_fence_after();
            const uint32_t from = tmem + set * Z::sum_cols + ((quad * 32u) << 16) + c0, rows = n < p.outputs && s.r0 + c0 < s.r1 ? s.r1 - s.r0 - c0 : 0u;
            auto read = [&](uint32_t c, uint32_t (&v)[LD]) {
                if (!ok) {
#pragma unroll
                    for (uint32_t j = 0; j < LD; j++) v[j] = 0x7fc00000u;
                } else if constexpr (LD == 16) tc_ld16(from + c, v);
                else tc_ld32(from + c, v);
            };
            auto free = [&] { tc_fence_before(); __syncwarp(); if (lane == 0) { if constexpr (PAIR) arrive_at(room + set * 8u, 0); else mbar_arrive(room + set * 8u); } };
            if (p.out_type == T_F32) {
#pragma unroll
                for (uint32_t h = 0; h < CO; h += HELD) {
                    float f[HELD];
#pragma unroll
                    for (uint32_t c = 0; c < HELD; c += LD) {
                        uint32_t v[LD];
                        read(h + c, v);
#pragma unroll
                        for (uint32_t j = 0; j < LD; j++) f[c + j] = __uint_as_float(v[j]);
                    }
                    if (h + HELD == CO) free();
                    if (rows > h) put_column<HELD>(static_cast<float *>(p.out) + (uint64_t)(s.r0 + c0 + h) * p.out_stride + n, p.out_stride, rows - h, [&](uint32_t j) { return f[j]; });
                }
            } else {
                uint32_t f[CO / 2];
#pragma unroll
                for (uint32_t c = 0; c < CO; c += LD) {
                    uint32_t v[LD];
                    read(c, v);
#pragma unroll
                    for (uint32_t j = 0; j < LD; j += 2) {
                        if (p.out_type == T_BF16) { const __nv_bfloat162 y = __floats2bfloat162_rn(__uint_as_float(v[j]), __uint_as_float(v[j + 1])); f[(c + j) / 2] = *reinterpret_cast<const uint32_t *>(&y); }
                        else { const __half2 y = __floats2half2_rn(__uint_as_float(v[j]), __uint_as_float(v[j + 1])); f[(c + j) / 2] = *reinterpret_cast<const uint32_t *>(&y); }
                    }
                }
                free();
                if (rows) put_column<CO>(static_cast<uint16_t *>(p.out) + (uint64_t)(s.r0 + c0) * p.out_stride + n, p.out_stride, rows, [&](uint32_t j) { return (uint16_t)(f[j / 2] >> (16u * (j & 1u))); });
            }
        }
        if (!ok) bad_s = 1;
        if (p.offsets) {          // rows of no expert
            const uint32_t first = clamp_row(p.offsets[0], p.rows), none = first + (p.rows - clamp_row(p.offsets[p.experts], p.rows));
            for (uint32_t i = blockIdx.x * Y::drain + warp - 4u; i < none; i += gridDim.x * Y::drain)
                for (uint32_t n = lane; n < p.outputs; n += 32u) put(p, i < first ? i : p.rows - none + i, n, 0.0f);
        }
        pdl_wait();          // no block ends before the kernel that quantises
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (bad_s) {          // copies still in flight land in this block's shared memory before it is given back
        const long long t0 = clock64();
        while (clock64() - t0 < 20000000ll) __nanosleep(1000);
    }
    if constexpr (PAIR) cluster_sync_all();          // nor while the other block's products read it
    tc_fence_after();
    if (warp == Y::mma) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Y::cols));
        else tc_dealloc(tmem, Y::cols);
    }
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
    if (rows == 1) stride = least;
    if (experts <= 1) expert = least;
    const cuuint64_t dims[3] = {bytes, rows, experts}, strides[2] = {stride, expert};
    const cuuint32_t boxes[3] = {kDepth / 2u, box, 1}, step[3] = {1, 1, 1};
    const Encode e = encoder();
    return e && e(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(base), dims, strides, boxes, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// scales that a load may bring, of every row and every step of the depth (`odd`: that may start at an odd one)
uint32_t unit_of(const void *base, uint64_t stride, uint64_t expert, uint64_t step, uint32_t groups, bool odd) {
    const uint64_t at = reinterpret_cast<uintptr_t>(base) | stride | expert | step | (step == 16u ? groups : 0u);          // (the second order is filled up)
    return at % 16u == 0 && !odd ? 16u : at % 8u == 0 ? 8u : at % 4u == 0 ? 4u : 1u;
}
constexpr uint32_t kSms = 148;

// ks 0: the kernel for many tiles
template <int TN, uint32_t X>
cudaError_t launch_of(TcArgs &t, cudaStream_t stream) {
    constexpr bool PAIR = TN == 256, CODES = X == T_MX4;
    static std::atomic<uint64_t> asked[2];          // devices (of the first 64) whose shared-memory limit has been raised
    const bool many = PAIR || (CODES && t.ks == 0);
    void (*kernel)(TcArgs) = nullptr;
    uint32_t smem = 0, threads = 192, x_rows = TN;
    if constexpr (CODES) if (many) { kernel = k_mx4_many<TN, PAIR>; smem = Many<TN, PAIR>::smem; threads = Many<TN, PAIR>::threads; x_rows = Many<TN, PAIR>::x_rows; }
    if constexpr (!PAIR) if (!many) { kernel = k_mx4_few<TN, X>; smem = Few<TN>::smem(X); }
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev > 63 || !(asked[many].load(std::memory_order_acquire) >> dev & 1u))) {
        e = smem_at_least(reinterpret_cast<const void *>(kernel), (int)smem);
        if (e == cudaSuccess && dev <= 63) asked[many].fetch_or(1ull << dev, std::memory_order_release);
    }
    if (e != cudaSuccess) return e;
    if ((CODES && !map_of(&t.xmap, t.p.x, t.p.columns, t.p.rows, 1, t.p.x_stride, 0, x_rows)) || !map_of(&t.wmap, t.p.w, t.p.columns, t.p.outputs, std::max(1u, t.p.experts), t.p.w_stride, t.p.w_expert, kRows))
        return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cfg.gridDim = PAIR ? dim3(2u * (uint32_t)std::min<uint64_t>(kSms / 2u, (uint64_t)t.wtiles * t.pairs)) : many ? dim3((uint32_t)std::min<uint64_t>(kSms, (uint64_t)t.wtiles * t.pairs)) : dim3(t.wtiles * (t.pairs + (t.p.offsets ? 1u : 0u)), 1, t.ks);
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    if (t.made) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (t.ks > 1 || PAIR) {
        attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attr[cfg.numAttrs].val.clusterDim.x = PAIR ? 2 : 1; attr[cfg.numAttrs].val.clusterDim.y = 1; attr[cfg.numAttrs++].val.clusterDim.z = PAIR ? 1 : t.ks;
    }
    return cudaLaunchKernelEx(&cfg, kernel, t);
}

}  // namespace

Mx4Plan mx4_plan(const Mx4Product &a) {
    Mx4Plan r{};
    const uint32_t groups = mx4_groups(a.columns), steps = (groups + kStageGroups - 1u) / kStageGroups, chunks = (groups + 15u) / 16u, wtiles = (a.outputs + kRows - 1u) / kRows;
    const uint32_t each = a.experts ? (a.rows + a.experts - 1u) / a.experts : a.rows;          // rows to a matrix, on average
    auto pairs = [&](uint32_t tn) { return a.experts ? std::min(a.rows, a.rows / tn + std::min(a.rows, a.experts)) : (a.rows + tn - 1u) / tn; };
    // Tiles of tn rows of X, ks blocks to one: what takes least by a model of the time in us, fitted to products of 1 to 1024 rows with 1024 x 2048 up to 20000 x 1024 and 2560 x 9728.  A step of the depth
    // takes `one` in the kernel for few tiles (once more for each 296 blocks, which begin anew, a quarter more where SMs have two), parts of a tile and their exchange some more; in the kernel for many tiles `step`,
    // a tile `tile`.  us as measured, with X in codes, few / many: 1 x 9728 x 2560 7.8 / 8.4 (16 rows), 128 9.8 / 9.0 (128 rows), 256 11.0 / 12.9; split 1 / 2 / 4 / 8: 1 x 2560 x 9728 17.7 / 11.5 / 8.6 / 8.7,
    // 1 x 9728 x 2560 7.8 / 7.8 / 10.3 / 15.1; 64 / 128 / 256 rows: 512 x 9728 x 2560 22.3 / 17.8 / 16.6, 128 9.3 / 9.0 / 10.6
    // Bytes have no term of their own: a block's step brings 18 to 64 KB in the time above, and rounds of tiles took longer than W's bytes in all that was measured (24 x 151936 x 1024 20.9 us, its bytes 14.8;
    // 132 rows of 64 experts of 1024 x 2048, 44 of them asked for, 17.4 and 7.6)
    struct Cost { uint32_t tn; float one, step, tile; };
    constexpr Cost costs[5] = {{16, 0.40f, 0.33f, 0.40f}, {32, 0.42f, 0.34f, 0.45f}, {64, 0.45f, 0.36f, 0.50f}, {128, 0.60f, 0.34f, 1.1f}, {256, 0.0f, 0.50f, 1.3f}};
    float best = 3e38f;
    for (const Cost &c : costs) {
        if (c.tn > 16u && c.tn >= 4u * each) break;
        // tiles as they may be expected: half a tile of an expert's rows is empty
        const double rows = a.experts ? std::min<double>(a.rows, a.rows / (double)c.tn + 0.5 * std::min(a.rows, a.experts)) : pairs(c.tn), tiles = std::max(1.0, rows) * wtiles;
        auto take = [&](double us, uint32_t ks) { if (us < best) { best = (float)us; r.tn = c.tn; r.ks = ks; } };
        take(4.0 + std::ceil(tiles / kSms) * (steps * c.step + c.tile), 0);
        if (c.tn == 256u || (uint64_t)wtiles * pairs(c.tn) > (1u << 24)) continue;
        for (uint32_t ks = 1; ks <= 8u && (ks == 1u || steps >= ks); ks *= 2u) {
            const double blocks = tiles * ks, waves = std::ceil(blocks / (2.0 * kSms)), busy = blocks > kSms;
            take(3.5 + waves * ((steps + ks - 1u) / ks) * c.one * (1.0 + 0.25 * busy) + 2.0 * (waves - 1.0) + (ks > 1u ? 0.5 + 0.02 * std::min(c.tn, each) + busy : 0.0), ks);
        }
    }
    r.pairs = pairs(r.tn);
    r.per = (steps + std::max(1u, r.ks) - 1u) / std::max(1u, r.ks);
    r.x_second = r.ks <= 1u || r.per % 2u == 0;          // (two steps of the depth are sixteen scales)
    const bool codes = a.x_type == T_MX4;
    // Numbers are quantised by the product itself where a block has few of them (64 rows x steps: four groups to a thread).  us, so / by a kernel before: 1 x 9728 x 2560 7.6 / 8.4, 1 x 4096 x 4096 7.0 / 7.3,
    // 6 x 9728 x 2560 9.3 / 8.4, 16 12.4 / 9.2; and a launch less of the host's time, 10.9 / 15.2 a call, which is what six rows have it for
    const uint32_t mine = std::min(16u, a.experts ? std::min(a.rows, 4u * each) : a.rows);
    if (!codes && r.tn == 16u && r.ks && r.per <= kRawSteps && mine * r.per <= 64u) { r.raw = true; return r; }
    r.x_codes = !codes || a.columns % 2u;
    r.w_scales = r.tn == 256u && (uint64_t)r.pairs >= 4u * (uint64_t)std::max(1u, a.experts);
    r.x_scales = r.x_codes || (codes && r.tn == 256u);
    r.x_scales_at = r.x_codes ? (uint64_t)a.rows * groups * 16u : 0;
    r.w_scales_at = r.x_scales_at + (r.x_scales ? (uint64_t)a.rows * chunks * 16u : 0);
    r.bytes = r.w_scales_at + (r.w_scales ? (uint64_t)std::max(1u, a.experts) * a.outputs * chunks * 16u : 0);
    return r;
}

cudaError_t mx4_tc_launch(const Mx4Product &a, const Mx4Plan &plan, uint64_t xs_step, uint64_t ws_step, bool made, cudaStream_t stream) {
    TcArgs t{};
    t.p = a; t.groups = mx4_groups(a.columns); t.steps = (t.groups + kStageGroups - 1u) / kStageGroups; t.wtiles = (a.outputs + kRows - 1u) / kRows; t.made = made;
    t.pairs = plan.pairs; t.ks = plan.ks; t.per = plan.per;
    const bool odd = t.ks > 1 && t.per % 2u;
    t.w_step = ws_step; t.x_step = xs_step;
    if (plan.raw) {
        t.w_unit = unit_of(a.ws, a.ws_stride, a.ws_expert, ws_step, t.groups, odd);
        return a.x_type == T_F32 ? launch_of<16, T_F32>(t, stream) : a.x_type == T_BF16 ? launch_of<16, T_BF16>(t, stream) : launch_of<16, T_F16>(t, stream);
    }
    t.w_unit = unit_of(a.ws, a.ws_stride, a.ws_expert, ws_step, t.groups, odd); t.x_unit = unit_of(a.xs, a.xs_stride, 0, xs_step, t.groups, odd);
    switch (plan.tn) {
        case 16: return launch_of<16, T_MX4>(t, stream);
        case 32: return launch_of<32, T_MX4>(t, stream);
        case 64: return launch_of<64, T_MX4>(t, stream);
        case 128: return launch_of<128, T_MX4>(t, stream);
        default: t.wtiles = (a.outputs + 2u * kRows - 1u) / (2u * kRows); return launch_of<256, T_MX4>(t, stream);
    }
}

}  // namespace nb
