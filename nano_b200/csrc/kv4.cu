// kv4.cu -- writing, reading and attending to a paged key/value cache held in 4 bits (layout and formulas: kv4.h).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <algorithm>
#include <atomic>

#include "family.h"
#include "kv4.cuh"
#include "portions.h"

namespace nb {
namespace {

// ------------------------------------------------------------------------------------------------
// Writing.  Four lanes hold a group, eight coordinates each: the extremes take two shuffles, a lane's codes are one word of a key row (two halves of a
// word of a value row).  The code is round_half_even((x - m) / s) of the numbers themselves: the fp32 quotient decides it unless it lies within 1e-5 of a
// border between two codes (its own error is below 3e-6: three roundings of numbers up to 16), where the quotient is taken in 64 bits.
// ------------------------------------------------------------------------------------------------
constexpr float kKv4Most = 32768.0f;          // c s + m of a written group stays inside fp16
constexpr uint32_t kRowThreads = 256;

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

// the place of token t in the pool, or -1
__device__ __forceinline__ long long kv4_place(const Kv4Rows &a, uint32_t t) {
    if (a.slots) {
        const int s = a.slots[t];
        return s >= 0 && (uint32_t)s / kKv4Page < a.n_pages ? (long long)s : -1;
    }
    const uint32_t pos = a.pos0 + t + (a.pos_ptr ? *a.pos_ptr : 0u), page = a.table[pos / kKv4Page];
    return page < a.n_pages ? (long long)page * kKv4Page + pos % kKv4Page : -1;
}

// A lane's eight coordinates of a group are 8 b .. 8 b + 7, but of fp32 rows 4 b .. 4 b + 3 and 16 + 4 b .. 16 + 4 b + 3: four lanes' 16-byte accesses then are 64 bytes side by side
// (with 32 bytes to a lane, half of each sector to an access, 9001 tokens of 8 heads of 128 took 26 us to write and 20 to read; so 22 and 13)
template <typename T> constexpr bool kHalves = sizeof(T) == 4;
template <typename T> __device__ __forceinline__ uint32_t second(uint32_t b) { return kHalves<T> ? 16u + 4u * b : 8u * b + 4u; }
template <typename T> __device__ __forceinline__ uint32_t first(uint32_t b) { return kHalves<T> ? 4u * b : 8u * b; }
template <typename T, bool VEC>
__device__ __forceinline__ void load_eight(const T *group, uint32_t b, float (&x)[8]) {
    if constexpr (VEC && kHalves<T>) {
        const float4 u = __ldcs(reinterpret_cast<const float4 *>(group + first<T>(b))), v = __ldcs(reinterpret_cast<const float4 *>(group + second<T>(b)));
        x[0] = u.x; x[1] = u.y; x[2] = u.z; x[3] = u.w; x[4] = v.x; x[5] = v.y; x[6] = v.z; x[7] = v.w;
    } else if constexpr (VEC) {
        __align__(16) T raw[8];
        *reinterpret_cast<uint4 *>(raw) = __ldcs(reinterpret_cast<const uint4 *>(group + first<T>(b)));
#pragma unroll
        for (int i = 0; i < 8; i++) x[i] = widen(raw[i]);
    } else
#pragma unroll
        for (int i = 0; i < 4; i++) { x[i] = widen(group[first<T>(b) + i]); x[4 + i] = widen(group[second<T>(b) + i]); }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_eight(T *group, uint32_t b, const float (&x)[8]) {
    if constexpr (VEC && kHalves<T>) {
        __stcs(reinterpret_cast<float4 *>(group + first<T>(b)), make_float4(x[0], x[1], x[2], x[3]));
        __stcs(reinterpret_cast<float4 *>(group + second<T>(b)), make_float4(x[4], x[5], x[6], x[7]));
    } else if constexpr (VEC) {
        __align__(16) T y[8];
#pragma unroll
        for (int i = 0; i < 8; i++) y[i] = (T)x[i];
        __stcs(reinterpret_cast<uint4 *>(group + first<T>(b)), *reinterpret_cast<const uint4 *>(y));
    } else
#pragma unroll
        for (int i = 0; i < 4; i++) { group[first<T>(b) + i] = (T)x[i]; group[second<T>(b) + i] = (T)x[4 + i]; }
}
// a thread's place in its call: token t, head g, group j of n, its eight coordinates b of the group's 32 (thread 4 k + b of the groups in order); 32-bit numbers (the
// launch sees to that: divisions of 64-bit ones were a third of the kernels)
struct Eighth { uint32_t t, g, j, b, n; bool live; };
__device__ __forceinline__ Eighth kv4_eighth(const Kv4Rows &a) {
    Eighth e;
    e.n = a.D / kKv4Group; e.b = threadIdx.x & 3u;
    const uint32_t item = blockIdx.x * (kRowThreads / 4u) + (threadIdx.x >> 2), per = a.G * e.n;
    e.t = item / per;
    const uint32_t rest = item - e.t * per;
    e.g = rest / e.n; e.j = rest - e.g * e.n;
    e.live = e.t < a.T;
    return e;
}
__device__ __forceinline__ unsigned char *kv4_block(const Kv4Rows &a, long long place, uint32_t g) {
    return a.pool + (uint64_t)(place / kKv4Page) * a.page_stride + (uint64_t)g * kv4_block_bytes(a.D);
}
// the group that four lanes hold eight coordinates of each: its pair, and this lane's codes
__device__ __forceinline__ uint32_t kv4_codes(const float (&x)[8], __half2 &sm) {
    float lo = x[0], hi = x[0];
    bool fine = true;
#pragma unroll
    for (int i = 0; i < 8; i++) { lo = fminf(lo, x[i]); hi = fmaxf(hi, x[i]); fine = fine && fabsf(x[i]) <= kKv4Most; }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o)); hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        fine = __shfl_xor_sync(0xffffffffu, (int)fine, o) && fine;
    }
    __half m = __float2half_rn(lo), s = __float2half_rn((hi - lo) * (1.0f / 15.0f));
    uint32_t word = 0;
    if (!fine) m = s = __ushort_as_half(0x7fff);
    else if (__half2float(s) > 0.0f) {
        const float mf = __half2float(m), sf = __half2float(s), inv = 1.0f / sf;
        float q[8], r[8], border = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) { q[i] = (x[i] - mf) * inv; r[i] = rintf(q[i]); border = fmaxf(border, fabsf(q[i] - r[i])); }
        if (border > 0.49999f)          // (some one in two hundred warps)
#pragma unroll
            for (int i = 0; i < 8; i++) r[i] = (float)rint(((double)x[i] - (double)mf) / (double)sf);
#pragma unroll
        for (int i = 0; i < 8; i++) word |= (uint32_t)fminf(fmaxf(r[i], 0.0f), 15.0f) << (4 * i);
    }
    sm = __halves2half2(s, m);
    return word;
}

// a thread: the same eight coordinates of a key and of the value beside it, both on their way at once
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRowThreads) k_kv4_write(const Kv4Rows a) {
    pdl_enter4();
    const Eighth e = kv4_eighth(a);
    const long long place = e.live ? kv4_place(a, e.t) : -1;
    float k[8] = {}, v[8] = {};
    if (place >= 0) {
        load_eight<T, VEC>(static_cast<const T *>(a.k) + e.t * a.k_token + e.g * a.k_head + e.j * kKv4Group, e.b, k);
        load_eight<T, VEC>(static_cast<const T *>(a.v) + e.t * a.v_token + e.g * a.v_head + e.j * kKv4Group, e.b, v);
    }
    __half2 ks, vs;
    uint32_t kw = kv4_codes(k, ks);
    const uint32_t vw = kv4_codes(v, vs);
    if constexpr (kHalves<T>) {          // a word's eight codes lie with two lanes
        const uint32_t from = (threadIdx.x & 28u) + 2u * (e.b & 1u), u = __shfl_sync(0xffffffffu, kw, from), w = __shfl_sync(0xffffffffu, kw, from + 1u);
        kw = __byte_perm(u, w, e.b < 2u ? 0x5410u : 0x7632u);
    }
    if (place < 0) return;
    unsigned char *block = kv4_block(a, place, e.g);
    const uint32_t at = (uint32_t)(place % kKv4Page), n = e.n;
    reinterpret_cast<uint32_t *>(block + at * 16u * n)[e.b * n + e.j] = kw;
    uint16_t *codes = reinterpret_cast<uint16_t *>(block + 640u * n + at * 16u * n);
    codes[first<T>(e.b) / 4u * n + e.j] = (uint16_t)vw;
    codes[second<T>(e.b) / 4u * n + e.j] = (uint16_t)(vw >> 16);
    if (e.b == 0) {
        reinterpret_cast<__half2 *>(block + 512u * n)[at * n + e.j] = ks;
        reinterpret_cast<__half2 *>(block + 1152u * n)[at * n + e.j] = vs;
    }
}

// Reading back: c s is exact in fp32, so one rounding is left
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRowThreads) k_kv4_read(const Kv4Rows a) {
    const Eighth e = kv4_eighth(a);
    if (!e.live) return;
    const long long place = kv4_place(a, e.t);
    float k[8] = {}, v[8] = {};
    if (place >= 0) {
        const unsigned char *block = kv4_block(a, place, e.g);
        const uint32_t at = (uint32_t)(place % kKv4Page), n = e.n;
        const uint16_t *kc = reinterpret_cast<const uint16_t *>(block + at * 16u * n), *vc = reinterpret_cast<const uint16_t *>(block + 640u * n + at * 16u * n);
        const uint32_t u = first<T>(e.b) / 4u, w = second<T>(e.b) / 4u;          // fours of coordinates; of a key two to a word
        const uint32_t kw = kc[(u / 2u * n + e.j) * 2u + (u & 1u)] | (uint32_t)kc[(w / 2u * n + e.j) * 2u + (w & 1u)] << 16, vw = vc[u * n + e.j] | (uint32_t)vc[w * n + e.j] << 16;
        const float2 ks = __half22float2(reinterpret_cast<const __half2 *>(block + 512u * n)[at * n + e.j]), vs = __half22float2(reinterpret_cast<const __half2 *>(block + 1152u * n)[at * n + e.j]);
#pragma unroll
        for (int i = 0; i < 8; i++) { k[i] = fmaf((float)((kw >> (4 * i)) & 15u), ks.x, ks.y); v[i] = fmaf((float)((vw >> (4 * i)) & 15u), vs.x, vs.y); }
    }
    store_eight<T, VEC>(static_cast<T *>(a.k) + e.t * a.k_token + e.g * a.k_head + e.j * kKv4Group, e.b, k);
    store_eight<T, VEC>(static_cast<T *>(a.v) + e.t * a.v_token + e.g * a.v_head + e.j * kKv4Group, e.b, v);
}

bool rows_at16(const Kv4Rows &a) {
    const uint64_t unit = 16u / elem_size(a.type);
    return ((reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v)) & 15u) == 0 && a.k_token % unit == 0 && a.v_token % unit == 0 && a.k_head % unit == 0 && a.v_head % unit == 0;
}

// ------------------------------------------------------------------------------------------------
// Attention.  A warp multiplies the keys of one page at a time (32, in two tiles of 16 rows) with NT tiles of 8 columns -- column c of key/value head g is
// query token c / rep, head g rep + c % rep, rep = H / G -- on the matrix instructions: keys and values are the row operand, made in registers from the codes,
// queries and weights the column operand, sums in fp32.  A nibble in the lowest bits of an fp16 number is that number: c 2^-24 (or c 2^-20, four bits up), below the
// smallest normal one and exact.  So:
//   values   o_d += sum_t c_td (p_t s_t),  one instruction per pair of codes; the pairs' second halves are a product of their own, 16 rows of which the groups take the
//            first: sum_t m_tg p_t.  c 2^-24 becomes c when o leaves.
//   keys     NT = 1: the product of the bare codes over one group at a time, s and m times it in fp32 (8 multiply-adds to a group); with more columns that would
//            cost more than the other way, c s + m in fp16 (1024 + c less 1024, then one fp16 multiply-add): 80 + 112 NT instructions for a page against 270
// Softmax in one pass: per column a reference r, the sum l and the weighted values o of weights 2^(x - r), x the score in log2 units.  r need not be the maximum: it is
// renewed when a weight would pass 2^cap, which keeps weights, and weights times s, inside fp16, small ones 2^kSlack below that; most pages leave r and o as they are.
// Rounding to 11 bits: the queries (times a power of two per row, so that any magnitude fits), the weights, the weights times s, and keys where they are c s + m; each
// rounding is at most 2^-11 of its number, against the 2^-8 of a bf16 output and the cache's own 1/30 of a group's range.
// Each warp brings its own pages into its own ring of shared memory (cp.async, one group of copies to a page) and waits for nobody else until the end.
// WK warps of a block share the columns and take every WK-th page (single tokens: the keys are what there is to share out); with WK = 1 (heads of 256,
// more than 16 columns) each warp has columns of its own.  The pages of a row are also split over nsplit blocks, whose parts k_kv4_join puts together.
// Measured: 32 heads over 8 of 128 behind 131000 tokens 44 us, with k_kv4_join (3.8 TB/s of the cache's bytes); bound by the chain of a warp's page -- 632 instructions, a scheduler issues in 54 % of its
// cycles -- not by mma.sync (34 to a page, one every 8.5 cycles of 1170).
// Values that stand for NaN are taken out of the product (0 times NaN would reach columns that do not see them) and make the rows that do see them NaN.
// ------------------------------------------------------------------------------------------------
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) { uint32_t r; asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v)); return r; }
constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;          // the bare codes: c 2^-24 and c 2^-20
constexpr int kStages = 2;
template <int NG, int NT, int WK, int W>
struct Room {
    static constexpr bool after = NT == 1;          // keys are scaled after the product
    static constexpr uint32_t block = 1280u * NG, ring = W * kStages * block, merge = WK > 1 ? W * NT * 8u * (32u * NG + 2u) * 4u : 0u,
                              q = (W / WK) * NT * NG * 512u, all = (ring > merge ? ring : merge) + q + (W / WK) * NT * 8u * 4u * (after ? 1u + NG : 1u);
};

// Blocks that an SM holds at once.  Four of heads of 128 leave 128 registers to a thread, and the instances spill up to 80 bytes (two tiles of columns: 56 at three blocks and 168 registers; heads
// of 64 with two tiles 72 at four and 128); one block less spills nothing.  As it is / one block less, us: one token of 32 heads of 128 over 8 behind 131000 43.6 / 42.7, three tokens 57.4 / 53.4; 32 sequences
// of up to 8190 42.8 / 45.1, 8 of 8190 26.0 / 26.7, four tokens of 16 heads over 4 in 32 sequences of 4000 37.1 / 36.8, of heads of 64 26.4 / 25.8: many sequences gain by the places
__host__ __device__ constexpr int kv4_blocks(int NG, int NT) { return NG <= 2 || (NG <= 4 && NT == 1) ? 4 : NG <= 4 ? 3 : 2; }

// The sequence that `before` others come before when they are ordered by pages, then by number; up to 32 N of them.  By votes, whose results are known to be the same in all
// lanes: read back from shared memory the number cost the kernel spills and a tenth of its speed
template <int N>
__device__ __forceinline__ uint32_t longest(const Kv4Attn &a, uint32_t before) {
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t own[N], count[N], b = 0;
#pragma unroll
    for (int i = 0; i < N; i++) { const uint32_t at = i * 32u + lane; count[i] = 0; own[i] = at < a.B ? (uint32_t)max(a.lens[at], 0) / kKv4Page * 64u + 63u - at : 0u; }
#pragma unroll 8
    for (uint32_t l = 0; l < 32; l++)
#pragma unroll
        for (int j = 0; j < N; j++) {
            const uint32_t other = __shfl_sync(0xffffffffu, own[j], l);
#pragma unroll
            for (int i = 0; i < N; i++) count[i] += other > own[i] ? 1u : 0u;
        }
#pragma unroll
    for (int i = 0; i < N; i++) { const uint32_t v = __ballot_sync(0xffffffffu, i * 32u + lane < a.B && count[i] == before); if (v) b = i * 32u + __ffs(v) - 1u; }
    return b;
}

// grid (nsplit x tiles, G, B); part: values [B][G][tiles][nsplit][columns of a block][D], then (m, l) of each
template <int NG, int NT, int WK, int W>
__global__ void __launch_bounds__(W * 32, kv4_blocks(NG, NT) * 4 / W > 1 ? kv4_blocks(NG, NT) * 4 / W : 1) k_kv4_attn(const Kv4Attn a, const Shape sh) {
    pdl_enter4();
    using R = Room<NG, NT, WK, W>;
    constexpr uint32_t D = 32u * NG, COLS = NT * 8u;
    extern __shared__ __align__(16) unsigned char sm[];
    __shared__ uint32_t known[W][kStages];          // whether the page in a stage is one of the pool's
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, wr = warp / WK, wk = warp % WK, gq = lane >> 2, tq = lane & 3u;
    const uint32_t split = blockIdx.x % sh.nsplit, tile = blockIdx.x / sh.nsplit, g = blockIdx.y, rep = a.H / a.G, ncols = a.T * rep;
    uint32_t b = blockIdx.z;
    if (sh.sorted) b = a.B <= 32u ? longest<1>(a, b) : longest<2>(a, b);
    unsigned char *ring = sm + warp * kStages * R::block;
    unsigned char *q_s = sm + (R::ring > R::merge ? R::ring : R::merge) + wr * NT * NG * 512u;
    float *scale_s = reinterpret_cast<float *>(sm + (R::ring > R::merge ? R::ring : R::merge) + R::q) + wr * COLS * (R::after ? 1u + NG : 1u), *sum_s = scale_s + COLS;          // sum_s (R::after): [column][group] sums of the rounded queries
    const uint32_t c0 = tile * sh.cols + wr * COLS;
    const int len = seq_len(a, b);

    // pages that any of this warp's columns sees, and the share of this split
    const uint32_t c1 = min(c0 + COLS, ncols);
    const int pos_a = c0 < ncols ? len - (int)a.T + (int)(c0 / rep) : -1, pos_b = c0 < ncols ? len - (int)a.T + (int)((c1 - 1u) / rep) : -1;
    uint32_t p0 = 0, p1 = 0;
    int low_a = 0, low_b = 0;          // the first key that a column sees, and the last column's first
    if (pos_b >= 0) {
        low_a = first_seen(max(pos_a, 0), a.window, a.block);
        const uint32_t first = (uint32_t)low_a / kKv4Page, np = (uint32_t)pos_b / kKv4Page + 1u - first;
        p0 = first + (uint32_t)((uint64_t)np * split / sh.nsplit); p1 = first + (uint32_t)((uint64_t)np * (split + 1u) / sh.nsplit);
        low_b = first_seen(pos_b, a.window, a.block);
    }
    const uint32_t count = p0 + wk < p1 ? (p1 - p0 - wk + WK - 1u) / WK : 0u;

    uint32_t ahead = 0;          // page numbers of 32 steps, one to a lane
    const unsigned char *head = a.pool + (uint64_t)g * R::block;
    const int32_t *table = a.table + (uint64_t)b * a.table_stride;
    auto fetch = [&](uint32_t i) {
        if (i < count) {
            if ((i & 31u) == 0) { const uint32_t p = p0 + wk + (i + lane) * WK; ahead = p < p1 ? (uint32_t)table[p] : 0u; }
            const uint32_t page = __shfl_sync(0xffffffffu, ahead, i & 31u), stage = i % kStages;
            const bool ok = page < a.n_pages;
            if (lane == 0) known[warp][stage] = ok;
            if (ok) {
                const unsigned char *src = head + (uint64_t)page * a.page_stride;
                const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring + stage * R::block);
#pragma unroll
                for (uint32_t v = 0; v < (80u * NG + 31u) / 32u; v++) { const uint32_t k = v * 32u + lane; if (80u * NG % 32u == 0 || k < 80u * NG) copy16(dst + k * 16u, src + k * 16u); }
            }
        }
        copy_commit();
    };
    for (uint32_t i = 0; i < kStages - 1; i++) fetch(i);

    // the queries as the column operand, each row times the power of two that brings its largest number to [1, 2)
    for (uint32_t c = wk; c < COLS; c += WK) {
        const uint32_t col = c0 + c, t = col / rep, h = g * rep + col % rep;
        float x[NG], most = 0.0f;
#pragma unroll
        for (int j = 0; j < NG; j++) {
            x[j] = 0.0f;
            if (col < ncols) {
                const uint64_t at = b * a.q_batch + t * a.q_token + h * a.q_head + j * 32u + lane;
                x[j] = a.type == T_F32 ? static_cast<const float *>(a.q)[at] : __bfloat162float(static_cast<const __nv_bfloat16 *>(a.q)[at]);
            }
            most = fmaxf(most, fabsf(x[j]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
        const int e = most > 0.0f ? min(max((int)(__float_as_uint(most) >> 23) - 127, -126), 126) : 0;
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        // coordinate 32 j + 8 b + i (lane = 8 b + i): step i / 2 % 2 of the group, register i % 2, half i / 4
        const uint32_t bq = lane >> 3, i = lane & 7u;
#pragma unroll
        for (int j = 0; j < NG; j++) {
            // (codes at bits 4-7 count sixteen times as much where they are multiplied as they are)
            const __half y = __float2half_rn(x[j] * down * (R::after && (i & 1u) ? 0.0625f : 1.0f));
            *reinterpret_cast<__half *>(q_s + (((c >> 3) * NG + j) * 2u + ((i >> 1) & 1u)) * 256u + ((c & 7u) * 4u + bq) * 8u + (i & 1u) * 4u + (i >> 2) * 2u) = y;
            if constexpr (R::after) {
                float z = __half2float(y) * (i & 1u ? 16.0f : 1.0f);
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
                if (lane == 0) sum_s[c * NG + j] = z * 0x1p-24f;
            }
        }
        if (lane == 0) scale_s[c] = (R::after ? 0x1p24f : 1.0f) * a.scale * __uint_as_float((uint32_t)(127 + e) << 23) * (a.softcap > 0.0f ? 1.0f / a.softcap : kLog2e);
    }
    if constexpr (WK > 1) __syncthreads(); else __syncwarp();


    float r[NT][2], l[NT][2], o[2 * NG][NT][4], om[NT][4];          // om: row j is the part of the groups' second halves
#pragma unroll
    for (int t = 0; t < NT; t++) {
        r[t][0] = r[t][1] = -INFINITY; l[t][0] = l[t][1] = 0.0f; om[t][0] = om[t][1] = om[t][2] = om[t][3] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * NG; i++) { o[i][t][0] = o[i][t][1] = o[i][t][2] = o[i][t][3] = 0.0f; }
    }
    float f[NT][2]; int pos[NT][2];          // this thread's columns: 2 tq and 2 tq + 1 of each tile
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const uint32_t c = t * 8u + tq * 2u + x;
            f[t][x] = scale_s[c];
            pos[t][x] = c0 + c < ncols ? len - (int)a.T + (int)((c0 + c) / rep) : -1;
        }

    uint32_t qf[NT == 1 ? 2 * NG : 1][2];
    if constexpr (NT == 1)
#pragma unroll
        for (int j = 0; j < 2 * NG; j++) { const uint2 v = *reinterpret_cast<const uint2 *>(q_s + j * 256u + lane * 8u); qf[j][0] = v.x; qf[j][1] = v.y; }
    float qsum[R::after ? NG : 1][2];
    if constexpr (R::after)
#pragma unroll
        for (int j = 0; j < NG; j++) { qsum[j][0] = sum_s[(tq * 2u) * NG + j]; qsum[j][1] = sum_s[(tq * 2u + 1u) * NG + j]; }
    const uint32_t gm = NG == 8 ? gq : gq % NG;          // the group whose second halves this lane's rows hold
    float cap = kCap;
    uint32_t most_s = 0x4000u;          // fp16 bits of the smallest s that cap has no room for
    const uint32_t row = (gq & 1u) * 4u + (gq >> 1);          // row r of eight is token 4 (r % 2) + r / 2 of eight: the transposed weights then pair tokens i and i + 4
    for (uint32_t i = 0; i < count; i++) {
        copy_wait<kStages - 2>();
        __syncwarp();
        fetch(i + kStages - 1);
        const uint32_t stage = i % kStages;
        if (!known[warp][stage]) continue;          // not a page of the pool: its keys are not seen
        unsigned char *pg = ring + stage * R::block;
        const int key0 = (int)((p0 + wk + i * WK) * kKv4Page);

        const bool whole = pos_a >= key0 + (int)kKv4Page - 1 && low_b <= key0;
        // the values' pairs, one token to a lane: steps that the weights have no room for, pairs that are no numbers (behind a sequence's end lies anything)
        uint32_t bad = 0;
        {
            uint32_t w[NG];
            take<4 * NG>(pg + 1152u * NG + lane * 4u * NG, w);
            __half2 top = half2_of(w[0]);
#pragma unroll
            for (int j = 1; j < NG; j++) top = __hmax2_nan(top, half2_of(w[j]));
            if (__any_sync(0xffffffffu, !whole || (bits(top) & 0xffffu) >= most_s)) {
                __half2 zero = __float2half2_rn(0.0f);          // 0 times a pair is 0, or NaN
                float big = 0.0f;
#pragma unroll
                for (int j = 0; j < NG; j++) { zero = __hfma2(half2_of(w[j]), __float2half2_rn(0.0f), zero); big = fmaxf(big, fabsf(__low2float(half2_of(w[j])))); }
                const bool odd = !__hbeq2(zero, __float2half2_rn(0.0f));
                bad = __ballot_sync(0xffffffffu, odd);
                // (a token that no column sees weighs nothing, whatever its step: the room, and with it the roundings, does not follow from it)
                const int at = key0 + (int)lane;
                const bool seen = at <= pos_b && at >= low_a;
                if (odd)
#pragma unroll
                    for (int j = 0; j < NG; j++) reinterpret_cast<uint32_t *>(pg + 1152u * NG + lane * 4u * NG)[j] = 0u;
                big = odd || !seen ? 0.0f : big;
#pragma unroll
                for (int off = 16; off > 0; off >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, off));
                if (big >= 2.0f) {
                    const int e = (int)(__float_as_uint(big) >> 23) - 127;
                    cap = fminf(cap, kCap - (float)e);
                    most_s = max(most_s, (uint32_t)(e + 16) << 10);
                }
                __syncwarp();
            }
        }

        // scores: rows 16 k + row (+ 8) of the page
        float s[2][NT][4];
#pragma unroll
        for (int k = 0; k < 2; k++) {
#pragma unroll
            for (int t = 0; t < NT; t++) s[k][t][0] = s[k][t][1] = s[k][t][2] = s[k][t][3] = 0.0f;
            const uint32_t ra = k * 16u + row, rb = ra + 8u;
            uint32_t wa[NG], wb[NG], sa[NG], sb[NG];
            take<4 * NG>(pg + ra * 16u * NG + tq * 4u * NG, wa); take<4 * NG>(pg + rb * 16u * NG + tq * 4u * NG, wb);
            take<4 * NG>(pg + 512u * NG + ra * 4u * NG, sa); take<4 * NG>(pg + 512u * NG + rb * 4u * NG, sb);
#pragma unroll
            for (int j = 0; j < NG; j++) {
                if constexpr (R::after) {
                    float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    const float2 pa = __half22float2(half2_of(sa[j])), pb = __half22float2(half2_of(sb[j]));
                    mma(c, wa[j] & kLow, wb[j] & kLow, wa[j] & kHigh, wb[j] & kHigh, qf[2 * j][0], qf[2 * j][1]);
                    mma(c, (wa[j] >> 8) & kLow, (wb[j] >> 8) & kLow, (wa[j] >> 8) & kHigh, (wb[j] >> 8) & kHigh, qf[2 * j + 1][0], qf[2 * j + 1][1]);
                    s[k][0][0] = fmaf(pa.x, c[0], fmaf(pa.y, qsum[j][0], s[k][0][0])); s[k][0][1] = fmaf(pa.x, c[1], fmaf(pa.y, qsum[j][1], s[k][0][1]));
                    s[k][0][2] = fmaf(pb.x, c[2], fmaf(pb.y, qsum[j][0], s[k][0][2])); s[k][0][3] = fmaf(pb.x, c[3], fmaf(pb.y, qsum[j][1], s[k][0][3]));
                    continue;
                }
                const __half2 s_a = __low2half2(half2_of(sa[j])), m_a = __high2half2(half2_of(sa[j])), s_b = __low2half2(half2_of(sb[j])), m_b = __high2half2(half2_of(sb[j]));
                const uint32_t x0 = stand_for<false>(wa[j], s_a, m_a), x1 = stand_for<true>(wa[j], s_a, m_a), x2 = stand_for<false>(wa[j] >> 8, s_a, m_a), x3 = stand_for<true>(wa[j] >> 8, s_a, m_a);
                const uint32_t y0 = stand_for<false>(wb[j], s_b, m_b), y1 = stand_for<true>(wb[j], s_b, m_b), y2 = stand_for<false>(wb[j] >> 8, s_b, m_b), y3 = stand_for<true>(wb[j] >> 8, s_b, m_b);
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    uint2 u, v;
                    { u = *reinterpret_cast<const uint2 *>(q_s + ((t * NG + j) * 2u) * 256u + lane * 8u); v = *reinterpret_cast<const uint2 *>(q_s + ((t * NG + j) * 2u + 1u) * 256u + lane * 8u); }
                    mma(s[k][t], x0, y0, x1, y1, u.x, u.y);
                    mma(s[k][t], x2, y2, x3, y3, v.x, v.y);
                }
            }
        }

        // weights, as the column operand of the second product
        uint32_t pw[NT][4];
#pragma unroll
        for (int t = 0; t < NT; t++) {
            float top[2] = {-INFINITY, -INFINITY};
            auto hide = [&](float as) {          // the scores of keys that a column does not see
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int low = first_seen(max(pos[t][x], 0), a.window, a.block) - key0 - (int)row, high = pos[t][x] - key0 - (int)row;          // of the rows 16 k + 8 y
#pragma unroll
                    for (int k = 0; k < 2; k++)
#pragma unroll
                        for (int y = 0; y < 2; y++) if (k * 16 + y * 8 > high || k * 16 + y * 8 < low) s[k][t][2 * y + x] = as;
                }
            };
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int x = 0; x < 4; x++) s[k][t][x] *= f[t][x & 1];
            if (a.softcap > 0.0f) {
                if (!whole) hide(0.0f);          // (which form tanh takes does not follow from them)
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int x = 0; x < 4; x++) top[0] = fmaxf(top[0], fabsf(s[k][t][x]));
                const bool near = __all_sync(0xffffffffu, top[0] < kTanhNear);          // (a NaN goes through either)
                top[0] = -INFINITY;
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int x = 0; x < 4; x++) s[k][t][x] = a.softcap * kLog2e * (near ? tanh_near(s[k][t][x]) : tanh_any(s[k][t][x]));
            }
            if (!whole) hide(-INFINITY);
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int x = 0; x < 4; x++) top[x & 1] = fmaxf(top[x & 1], s[k][t][x]);
            if (__any_sync(0xffffffffu, top[0] > r[t][0] + cap || top[1] > r[t][1] + cap)) {
                float corr[2];
#pragma unroll
                for (int x = 0; x < 2; x++) {
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], off));
                    const float next = fmaxf(top[x] - (cap - kSlack), r[t][x]);
                    corr[x] = next == -INFINITY ? 1.0f : ex2(r[t][x] - next);
                    r[t][x] = next;
                    l[t][x] *= corr[x];
                }
#pragma unroll
                for (int d = 0; d < 2 * NG; d++) { o[d][t][0] *= corr[0]; o[d][t][1] *= corr[1]; o[d][t][2] *= corr[0]; o[d][t][3] *= corr[1]; }
                om[t][0] *= corr[0]; om[t][1] *= corr[1];
            }
            const float use[2] = {r[t][0] == -INFINITY ? 0.0f : r[t][0], r[t][1] == -INFINITY ? 0.0f : r[t][1]};
#pragma unroll
            for (int k = 0; k < 2; k++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const float u = ex2(s[k][t][2 * y] - use[0]), v = ex2(s[k][t][2 * y + 1] - use[1]);
                    l[t][0] += u; l[t][1] += v;
                    pw[t][2 * k + y] = transpose8(bits(__floats2half2_rn(u, v)));
                }
        }

        if (bad) {          // values that are no number make the rows that see them NaN, however little they weigh
#pragma unroll
            for (int t = 0; t < NT; t++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    if (bad >> (k * 8 + row) & 1u) {
                        if (s[k >> 1][t][2 * (k & 1)] != -INFINITY) l[t][0] = NAN;
                        if (s[k >> 1][t][2 * (k & 1) + 1] != -INFINITY) l[t][1] = NAN;
                    }
        }

        // weighted values: depth step k takes tokens 16 k + tq + {0, 4, 8, 12}; rows are coordinates 32 j + 4 gq + {0 .. 3}
#pragma unroll
        for (int k = 0; k < 2; k++) {
            uint32_t w[4][(NG + 1) / 2], sp[4][NG], mw[4];
#pragma unroll
            for (int x = 0; x < 4; x++) {
                const uint32_t at = k * 16u + tq + 4u * x;
                take<2 * NG>(pg + 640u * NG + at * 16u * NG + gq * 2u * NG, w[x]);
                take<4 * NG>(pg + 1152u * NG + at * 4u * NG, sp[x]);
                mw[x] = *reinterpret_cast<const uint32_t *>(pg + 1152u * NG + at * 4u * NG + gm * 4u);
            }
            const uint32_t m_ab = __byte_perm(mw[0], mw[1], 0x7632u), m_cd = __byte_perm(mw[2], mw[3], 0x7632u);
#pragma unroll
            for (int t = 0; t < NT; t++) mma(om[t], m_ab, 0u, m_cd, 0u, pw[t][2 * k], pw[t][2 * k + 1]);
#pragma unroll
            for (int j = 0; j < NG; j++) {
                const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
                const uint32_t ab = __byte_perm(w[0][j / 2], w[1][j / 2], sel), cd = __byte_perm(w[2][j / 2], w[3][j / 2], sel);
                const __half2 s_ab = half2_of(__byte_perm(sp[0][j], sp[1][j], 0x5410u)), s_cd = half2_of(__byte_perm(sp[2][j], sp[3][j], 0x5410u));
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const uint32_t u = bits(__hmul2(half2_of(pw[t][2 * k]), s_ab)), v = bits(__hmul2(half2_of(pw[t][2 * k + 1]), s_cd));
                    mma(o[2 * j][t], ab & kLow, ab & kHigh, cd & kLow, cd & kHigh, u, v);
                    mma(o[2 * j + 1][t], (ab >> 8) & kLow, (ab >> 8) & kHigh, (cd >> 8) & kLow, (cd >> 8) & kHigh, u, v);
                }
            }
        }
    }
    copy_wait<0>();
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) l[t][x] += __shfl_xor_sync(0xffffffffu, l[t][x], off);

    // coordinates 32 j + 4 gq + {0, 1, 2, 3} of column x
    auto four = [&](int t, int x, int j, float k) {
        const float mj = __shfl_sync(0xffffffffu, om[t][x], (j << 2) | tq);
        return make_float4(fmaf(o[2 * j][t][x], 0x1p24f, mj) * k, fmaf(o[2 * j][t][2 + x], 0x1p20f, mj) * k, fmaf(o[2 * j + 1][t][x], 0x1p24f, mj) * k, fmaf(o[2 * j + 1][t][2 + x], 0x1p20f, mj) * k);
    };
    const uint64_t where = (((uint64_t)(b * a.G + g) * sh.tiles + tile) * sh.nsplit + split) * sh.cols, places = (uint64_t)a.B * a.G * sh.tiles * sh.nsplit * sh.cols;
    float2 *ml = reinterpret_cast<float2 *>(a.part + places * D);
    if constexpr (WK > 1) {
        float *mo = reinterpret_cast<float *>(sm), *mm = mo + W * COLS * D;          // [warp][column][D], then [warp][column] (m, l): where the rings were
        __syncthreads();
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t c = warp * COLS + t * 8u + tq * 2u + x;
#pragma unroll
                for (int j = 0; j < NG; j++)
                    *reinterpret_cast<float4 *>(mo + c * D + j * 32u + gq * 4u) = four(t, x, j, 1.0f);
                if (gq == 0) { mm[2 * c] = r[t][x]; mm[2 * c + 1] = l[t][x]; }
            }
        __syncthreads();
        for (uint32_t e = tid; e < COLS * D / 4u; e += W * 32u) {
            const uint32_t c = e / (D / 4u), d = e % (D / 4u) * 4u, col = c0 + c;
            if (col >= ncols) break;
            float top = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < W; w++) top = fmaxf(top, mm[2 * (w * COLS + c)]);
            const float use = top == -INFINITY ? 0.0f : top;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float k = ex2(mm[2 * (w * COLS + c)] - use);
                const float4 u = *reinterpret_cast<const float4 *>(mo + (w * COLS + c) * D + d);
                sum = fmaf(mm[2 * (w * COLS + c) + 1], k, sum);
                v.x = fmaf(u.x, k, v.x); v.y = fmaf(u.y, k, v.y); v.z = fmaf(u.z, k, v.z); v.w = fmaf(u.w, k, v.w);
            }
            if (sh.nsplit > 1) {
                *reinterpret_cast<float4 *>(a.part + (where + c) * D + d) = v;
                if (d == 0) ml[where + c] = make_float2(top, sum);
            } else {
                const uint32_t t = col / rep, h = g * rep + col % rep;
                const float k = last_factor(a, t, h, top, sum);
                const bool none = sum == 0.0f;
                store_four(a, b, t, h, d, none ? 0.0f : v.x * k, none ? 0.0f : v.y * k, none ? 0.0f : v.z * k, none ? 0.0f : v.w * k);
            }
        }
    } else {
#pragma unroll
        for (int t = 0; t < NT; t++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t c = wr * COLS + t * 8u + tq * 2u + x, col = tile * sh.cols + c;
                const bool mine = col < ncols;
                const uint32_t tt = col / rep, h = g * rep + col % rep;
                const float k = !mine || sh.nsplit > 1 ? 1.0f : last_factor(a, tt, h, r[t][x], l[t][x]);
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    const float4 v = four(t, x, j, k);
                    if (!mine) continue;
                    if (sh.nsplit > 1) *reinterpret_cast<float4 *>(a.part + (where + c) * D + j * 32u + gq * 4u) = v;
                    else store_four(a, b, tt, h, j * 32u + gq * 4u, v.x, v.y, v.z, v.w);
                }
                if (mine && sh.nsplit > 1 && gq == 0) ml[where + c] = make_float2(r[t][x], l[t][x]);
            }
    }
}

// The parts of a row's splits put together: a block per row, its warps take every fourth split.  grid (T rep, G, B); shared memory: a weight per split
constexpr uint32_t kJoinThreads = 128;
__global__ void __launch_bounds__(kJoinThreads) k_kv4_join(const Kv4Attn a, const Shape sh) {
    pdl_enter4();
    extern __shared__ __align__(16) unsigned char sm[];
    float *w_s = reinterpret_cast<float *>(sm);
    __shared__ float4 part[kJoinThreads / 32][64];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, rep = a.H / a.G, col = blockIdx.x, g = blockIdx.y, b = blockIdx.z, t = col / rep, h = g * rep + col % rep;
    const uint64_t places = (uint64_t)a.B * a.G * sh.tiles * sh.nsplit * sh.cols, where = ((uint64_t)(b * a.G + g) * sh.tiles + col / sh.cols) * sh.nsplit * sh.cols + col % sh.cols;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + places * a.D);
    // (every warp finds the row's maximum and sum for itself)
    float top = -INFINITY, sum = 0.0f;
    for (uint32_t s = lane; s < sh.nsplit; s += 32u) top = fmaxf(top, ml[where + (uint64_t)s * sh.cols].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float use = top == -INFINITY ? 0.0f : top;
    for (uint32_t s = lane; s < sh.nsplit; s += 32u) {
        const float2 p = ml[where + (uint64_t)s * sh.cols];
        const float k = ex2(p.x - use);
        sum = fmaf(p.y, k, sum);
        if (warp == 0) w_s[s] = k;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    __syncthreads();
    for (uint32_t d0 = 0; d0 < a.D; d0 += 128u) {
        const uint32_t d = d0 + lane * 4u;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (d < a.D)
#pragma unroll 4
            for (uint32_t s = warp; s < sh.nsplit; s += kJoinThreads / 32u) {
                const float4 u = *reinterpret_cast<const float4 *>(a.part + (where + (uint64_t)s * sh.cols) * a.D + d);
                const float k = w_s[s];
                v.x = fmaf(u.x, k, v.x); v.y = fmaf(u.y, k, v.y); v.z = fmaf(u.z, k, v.z); v.w = fmaf(u.w, k, v.w);
            }
        part[warp][d0 / 4u + lane] = v;
    }
    __syncthreads();
    const float k = last_factor(a, t, h, top, sum);
    for (uint32_t e = threadIdx.x; e < a.D / 4u; e += kJoinThreads) {
        float4 v = part[0][e];
#pragma unroll
        for (uint32_t w = 1; w < kJoinThreads / 32u; w++) { const float4 u = part[w][e]; v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w; }
        store_four(a, b, t, h, e * 4u, v.x * k, v.y * k, v.z * k, v.w * k);
    }
}

template <typename K, typename... A>
cudaError_t launch_on(K k, dim3 grid, uint32_t threads, size_t smem, cudaStream_t stream, bool pdl, const A &...args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid; cfg.blockDim = dim3(threads); cfg.dynamicSmemBytes = smem; cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

// ---- which instance, and how the work is shared out ----
struct Plan { int nt; bool rows, tc, wide; Shape sh; };
constexpr uint32_t kWarps = 4, kWide = 8, kShort = 32, kWaves = 3, kMost = 64;
Plan plan_for(uint32_t B, uint32_t T, uint32_t H, uint32_t G, uint32_t D, uint32_t width, uint32_t window, uint32_t block, uint32_t sms) {
    const uint32_t ncols = T * (H / G);
    Plan p{};
    p.nt = ncols <= 8 ? 1 : 2;
    p.rows = ncols > 16;
    p.tc = p.rows && D <= 128;
    p.sh.cols = p.tc ? kKv4TcRows : (uint32_t)p.nt * 8u * (p.rows ? kWarps : 1u);
    p.sh.tiles = (ncols + p.sh.cols - 1u) / p.sh.cols;
    // pages that a block can have in sight
    const uint64_t reach = std::min<uint64_t>(window ? window : ~0u, block ? block : ~0u) + (p.sh.cols + H / G - 1u) / (H / G) + kKv4Page;
    const uint32_t pages = (uint32_t)std::min<uint64_t>(width, reach / kKv4Page + 1u);
    // A block for every place that the device has.  Of several sequences, whose lengths may differ, blocks of no more than kMost pages, but at most three times as many blocks as
    // places.  In the given order of sequences (measured before the longest came first, below), with one, two and three blocks to a place, 32 sequences of up to 8190 tokens take 67, 56 and 57 us,
    // of 8190 each 77, 74 and 79, but 8 of them 20, 24 and 29, 3 of up to 30000 26, 33 and 36 (a block costs some 2 us beside its pages)
    const uint32_t at_once = p.tc ? 1u : (uint32_t)kv4_blocks((int)D / 32, p.nt);
    const uint64_t blocks = std::max<uint64_t>(1, (uint64_t)B * G * p.sh.tiles), places = (uint64_t)at_once * sms;
    const uint32_t least = p.tc ? 16u : p.rows ? 8u : kWarps;          // pages of a split
    uint64_t n = places / blocks;
    if (B > 1) n = std::max(n, std::min<uint64_t>((pages + kMost - 1u) / kMost, kWaves * places / blocks));
    p.sh.nsplit = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(n, std::max(1u, pages / least)));
    // Few blocks with few pages each: twice the warps and no parts to be joined.  One token of 16 heads of 128 over 8 behind 200, 400, 500, 600, 777 and 1000 tokens takes 5.9, 7.2, 7.6, 8.6, 10.0 and 10.3 us on
    // the device, with the keys split 6.4, 8.5, 7.7, 8.5, 8.9 and 7.9; but it is one launch without a workspace, and calls in a row, bound by the host, take 12.6 us instead of 17.  So the border lies where
    // the call gains, beyond the 550 or so where the device does.  (Sixteen warps behind 400: 7.8, 777: 9.7, 60: 6.5 instead of 5.3.)  Heads of 256 behind 200 7.8 instead of 8.3, 400 10.3 as the split, 500 10.8 instead of 9.2
    p.wide = !p.tc && !p.rows && pages <= (D > 128u ? kShort / 2u : kShort) && blocks <= sms;
    if (p.wide) p.sh.nsplit = 1;
    // Of up to 64 sequences the longest first, so that the SMs get long and short ones alike and what is left when others end is short (32 of up to 8190 tokens: 50 us, in the given
    // order 56; 64 of up to 4000, 4 heads of 64: 25 and 28).  It costs some 0.9 us of a block's start: not for blocks of less than 16 pages (48 of up to 1000: 10.6 us, sorted 11.5)
    p.sh.sorted = !p.tc && B > 1 && B <= 64 && pages >= 16u * p.sh.nsplit ? 1u : 0u;
    return p;
}

template <int NG, int NT, int WK, int W = kWarps>
cudaError_t attn_launch(const Kv4Attn &a, const Shape &sh, cudaStream_t stream, bool pdl) {
    constexpr int smem = (int)Room<NG, NT, WK, W>::all;
    const auto k = k_kv4_attn<NG, NT, WK, W>;
    static std::atomic<uint64_t> asked{0};          // devices (of the first 64) whose limit has been raised: asking costs a microsecond
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev > 63 || !(asked.load(std::memory_order_acquire) >> dev & 1u))) {
        e = smem_at_least(reinterpret_cast<const void *>(k), smem);
        if (e == cudaSuccess && dev <= 63) asked.fetch_or(1ull << dev, std::memory_order_release);
    }
    return e != cudaSuccess ? e : launch_on(k, dim3(sh.nsplit * sh.tiles, a.G, a.B), W * 32, smem, stream, pdl, a, sh);
}
template <int NG>
cudaError_t attn_launch_nt(const Kv4Attn &a, const Plan &p, cudaStream_t stream, bool pdl) {
    if constexpr (NG > 4) { if (p.rows) return attn_launch<NG, 2, 1>(a, p.sh, stream, pdl); }          // (of up to 128 the tensor-memory kernel takes them: plan_for)
    if (p.wide) return p.nt == 1 ? attn_launch<NG, 1, kWide, kWide>(a, p.sh, stream, pdl) : attn_launch<NG, 2, kWide, kWide>(a, p.sh, stream, pdl);
    return p.nt == 1 ? attn_launch<NG, 1, kWarps>(a, p.sh, stream, pdl) : attn_launch<NG, 2, kWarps>(a, p.sh, stream, pdl);
}

template <bool WRITE>
cudaError_t rows_launch(const Kv4Rows &all, cudaStream_t stream, bool pdl) {
    const uint32_t per = all.G * (all.D / kKv4Group), most = (1u << 30) / per;          // tokens of a launch
    const bool vec = rows_at16(all);
    return in_portions(all.T, most, [&](uint32_t t0, uint32_t n) {
        Kv4Rows a = all;
        a.T = n;
        a.k = static_cast<char *>(all.k) + t0 * all.k_token * elem_size(all.type); a.v = static_cast<char *>(all.v) + t0 * all.v_token * elem_size(all.type);
        if (all.slots) a.slots += t0; else a.pos0 += t0;
        const dim3 grid((a.T * per + kRowThreads / 4u - 1u) / (kRowThreads / 4u));
#define KV4_ROWS(TYPE)                                                                                                                          \
    (WRITE ? (vec ? launch_on(k_kv4_write<TYPE, true>, grid, kRowThreads, 0, stream, pdl, a) : launch_on(k_kv4_write<TYPE, false>, grid, kRowThreads, 0, stream, pdl, a)) \
           : (vec ? launch_on(k_kv4_read<TYPE, true>, grid, kRowThreads, 0, stream, false, a) : launch_on(k_kv4_read<TYPE, false>, grid, kRowThreads, 0, stream, false, a)))
        return a.type == T_F32 ? KV4_ROWS(float) : a.type == T_BF16 ? KV4_ROWS(__nv_bfloat16) : KV4_ROWS(__half);
#undef KV4_ROWS
    });
}

}  // namespace

cudaError_t kv4_write_launch(const Kv4Rows &a, cudaStream_t stream, bool pdl) { return rows_launch<true>(a, stream, pdl); }
cudaError_t kv4_read_launch(const Kv4Rows &a, cudaStream_t stream) { return rows_launch<false>(a, stream, false); }

size_t kv4_attn_workspace(uint32_t B, uint32_t T, uint32_t H, uint32_t G, uint32_t D, uint32_t width, uint32_t window, uint32_t block, uint32_t sms) {
    const Plan p = plan_for(B, T, H, G, D, width, window, block, sms);
    return p.sh.nsplit == 1 ? 0 : (size_t)B * G * p.sh.tiles * p.sh.nsplit * p.sh.cols * (D + 2u) * 4u;
}

// (keys are split only while blocks times splits stay within the waves of what the device holds at once: one block of 128 rows to an SM, or four of at most 64)
size_t kv4_attn_workspace_most(uint32_t B, uint32_t D, uint32_t sms) { return (size_t)(B > 1 ? kWaves : 1u) * sms * 256u * (D + 2u) * 4u; }

cudaError_t kv4_attn_launch(const Kv4Attn &a, uint32_t sms, cudaStream_t stream, bool pdl, bool pdl_join, uint32_t *launches) {
    const Plan p = plan_for(a.B, a.T, a.H, a.G, a.D, a.width, a.window, a.block, sms);
    cudaError_t e;
    if (p.tc) e = kv4_tc_launch(a, p.sh.nsplit, p.sh.tiles, stream, pdl);
    else switch (a.D / 32u) {
        case 1: e = attn_launch_nt<1>(a, p, stream, pdl); break;
        case 2: e = attn_launch_nt<2>(a, p, stream, pdl); break;
        case 3: e = attn_launch_nt<3>(a, p, stream, pdl); break;
        case 4: e = attn_launch_nt<4>(a, p, stream, pdl); break;
        default: e = attn_launch_nt<8>(a, p, stream, pdl); break;
    }
    if (e == cudaSuccess && p.sh.nsplit > 1)
        e = launch_on(k_kv4_join, dim3(a.T * (a.H / a.G), a.G, a.B), kJoinThreads, p.sh.nsplit * 4u, stream, pdl_join, a, p.sh);
    if (launches) *launches = p.sh.nsplit > 1 ? 2 : 1;
    return e;
}

}  // namespace nb

using nb::fail;

namespace {
int kv4_pool_check(const void *pool, uint64_t page_stride, uint32_t n_pages, uint32_t kv_heads, uint32_t head_dim) {
    if (!head_dim || head_dim % nb::kKv4Group || head_dim > 256u) return fail(NB200_EINVAL, "head_dim %u: a cache in 4 bits holds multiples of 32 up to 256", head_dim);
    if (!kv_heads || kv_heads > 65535u) return fail(NB200_EINVAL, "kv_heads %u unusable", kv_heads);
    if (n_pages > 0x7fffffffu / nb::kKv4Page) return fail(NB200_EINVAL, "%u pages: places are 32-bit numbers", n_pages);
    if ((reinterpret_cast<uintptr_t>(pool) | page_stride) & 15u) return fail(NB200_EINVAL, "the pool's base and page stride are to be multiples of 16 bytes");
    if (n_pages && (!pool || (n_pages > 1 && page_stride < (uint64_t)kv_heads * nb::kv4_block_bytes(head_dim)))) return fail(NB200_EINVAL, "null pool, or pages that overlap");
    return 0;
}
int kv4_rows_check(const nb200_kv4_rows *r, nb::Kv4Rows *a) {
    if (!r) return fail(NB200_EINVAL, "null argument");
    int rc;
    if ((rc = kv4_pool_check(r->pool, r->page_stride, r->n_pages, r->kv_heads, r->head_dim))) return rc;
    if (r->type > nb::T_F16) return fail(NB200_EINVAL, "rows are fp32, bf16 or fp16 (type %u)", r->type);
    if (r->tokens && (!r->k || !r->v || !r->slots)) return fail(NB200_EINVAL, "null argument");
    if ((reinterpret_cast<uintptr_t>(r->k) | reinterpret_cast<uintptr_t>(r->v)) % nb::elem_size(r->type) || reinterpret_cast<uintptr_t>(r->slots) % 4u) return fail(NB200_EINVAL, "rows or slots are not aligned to their type");
    if ((uint64_t)r->tokens * r->kv_heads * (r->head_dim / 8u) > 0x7fffffffull * nb::kRowThreads) return fail(NB200_EINVAL, "%u tokens are too many for one call", r->tokens);
    if (r->tokens && nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    *a = nb::Kv4Rows{r->k, r->v, r->k_token, r->v_token, r->k_head, r->v_head, r->type, r->slots, nullptr, 0, nullptr, r->tokens, r->kv_heads, r->head_dim,
                     static_cast<unsigned char *>(r->pool), r->page_stride, r->n_pages};
    return 0;
}
int sm_count(uint32_t *sms) {
    int dev = 0, n = 0;
    NB_CK(cudaGetDevice(&dev));
    NB_CK(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    *sms = (uint32_t)n;
    return 0;
}
int kv4_attention_check(const nb200_kv4_attention *p) {
    if (!p) return fail(NB200_EINVAL, "null argument");
    int rc;
    if ((rc = kv4_pool_check(p->pool, p->page_stride, p->n_pages, p->kv_heads, p->head_dim))) return rc;
    if (!nb::kv4_dim_ok(p->head_dim)) return fail(NB200_EINVAL, "head_dim %u has no attention kernel (32, 64, 96, 128 and 256 have)", p->head_dim);
    if (p->type > nb::T_BF16) return fail(NB200_EINVAL, "queries are fp32 or bf16 (type %u)", p->type);
    if (!p->heads || p->heads % p->kv_heads) return fail(NB200_EINVAL, "%u heads do not share %u key/value heads evenly", p->heads, p->kv_heads);
    if (p->batch > 65535u) return fail(NB200_EINVAL, "%u sequences are too many for one call", p->batch);
    if ((uint64_t)p->tokens * (p->heads / p->kv_heads) > (1u << 30) || p->tokens > (1u << 30)) return fail(NB200_EINVAL, "%u tokens are too many for one call", p->tokens);
    if ((uint64_t)p->width * nb::kKv4Page > (1u << 30)) return fail(NB200_EINVAL, "%u pages to a sequence are too many", p->width);
    if (p->window > (1u << 30) || p->block > (1u << 30)) return fail(NB200_EINVAL, "window or block above 2^30");
    if (!(p->softcap >= 0.0f) || isinf(p->softcap) || !isfinite(p->scale)) return fail(NB200_EINVAL, "scale %g or softcap %g unusable", p->scale, p->softcap);
    if (p->batch && p->tokens) {
        if (!p->q || !p->out || !p->lens || (p->width && !p->table)) return fail(NB200_EINVAL, "null argument");
        const uint32_t e = nb::elem_size(p->type), four = 4u * e;
        if (reinterpret_cast<uintptr_t>(p->q) % e || reinterpret_cast<uintptr_t>(p->lens) % 4u || reinterpret_cast<uintptr_t>(p->table) % 4u || reinterpret_cast<uintptr_t>(p->sinks) % 4u) return fail(NB200_EINVAL, "an operand is not aligned to its type");
        if (reinterpret_cast<uintptr_t>(p->out) % four || (p->o_batch | p->o_token | p->o_head) % 4u) return fail(NB200_EINVAL, "out's base and strides are to be multiples of four numbers");
    }
    return 0;
}
}  // namespace

extern "C" {

int nb200_dev_kv4_write(const nb200_kv4_rows *rows, void *stream) {
    nb::Kv4Rows a;
    const int r = kv4_rows_check(rows, &a);
    if (r) return r;
    NB_CK(nb::kv4_write_launch(a, static_cast<cudaStream_t>(stream), false));
    return 0;
}

int nb200_dev_kv4_read(const nb200_kv4_rows *rows, void *stream) {
    nb::Kv4Rows a;
    const int r = kv4_rows_check(rows, &a);
    if (r) return r;
    NB_CK(nb::kv4_read_launch(a, static_cast<cudaStream_t>(stream)));
    return 0;
}

int nb200_dev_kv4_attention_workspace(const nb200_kv4_attention *p, uint64_t *bytes) {
    int r;
    uint32_t sms = 0;
    if (!bytes) return fail(NB200_EINVAL, "null argument");
    if ((r = kv4_attention_check(p))) return r;
    *bytes = 0;
    if (!p->batch || !p->tokens) return 0;
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    if ((r = sm_count(&sms))) return r;
    *bytes = nb::kv4_attn_workspace(p->batch, p->tokens, p->heads, p->kv_heads, p->head_dim, p->width, p->window, p->block, sms);
    return 0;
}

int nb200_dev_kv4_attention(const nb200_kv4_attention *p, void *workspace, uint64_t workspace_bytes, void *stream) {
    int r;
    uint32_t sms = 0;
    if ((r = kv4_attention_check(p))) return r;
    if (!p->batch || !p->tokens) return 0;
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    if ((r = sm_count(&sms))) return r;
    const size_t need = nb::kv4_attn_workspace(p->batch, p->tokens, p->heads, p->kv_heads, p->head_dim, p->width, p->window, p->block, sms);
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) & 15u)) return fail(NB200_EINVAL, "the workspace is to have %zu bytes at a multiple of 16", need);
    const nb::Kv4Attn a{p->q, p->q_batch, p->q_token, p->q_head, p->type, p->out, p->o_batch, p->o_token, p->o_head, static_cast<const unsigned char *>(p->pool), p->page_stride, p->n_pages,
                        p->table, p->table_stride, p->width, p->lens, 0, nullptr, p->batch, p->tokens, p->heads, p->kv_heads, p->head_dim, p->scale, p->softcap, p->sinks, p->window, p->block,
                        nullptr, 0, static_cast<float *>(workspace)};
    NB_CK(nb::kv4_attn_launch(a, sms, static_cast<cudaStream_t>(stream), false, true, nullptr));          // (whose kernel comes before is not known; before the join it is this call's own)
    return 0;
}

}  // extern "C"
