// ops.cu -- operators on device memory: log probabilities of given tokens, copies of cache pages, and their C entry points.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <math.h>

#include <algorithm>
#include <tuple>
#include <utility>
#include <vector>

#include "family.h"
#include "ops.h"
#include "pairs.cuh"
#include "portions.h"

namespace nb {
namespace {

// ------------------------------------------------------------------------------------------------
// Log probabilities.  For a row x of V logits with maximum M, Z = sum exp(x_i - M):
//     log p_t = (x_t - M) - log Z,    H = log Z + (1/Z) sum exp(x_i - M) (M - x_i),    alternatives in the order (x descending, index ascending).
// One pass over the row, bound by its bytes: every thread keeps m, z = sum exp(x - m) and s = sum exp(x - m) (x - m) of what it has seen, in log2 units and on
// pairs of numbers (fma.f32x2: some five instructions to a number, where eleven are what bf16 rows at the full rate of HBM leave), and rescales them when m grows.  Two
// such triples join as  z = z1 f1 + z2 f2,  s = f1 (s1 + z1 (m1 - m)) + f2 (...),  f = exp(m_i - m).  Sums are fp32.
// Alternatives: the k-th largest of the threads' maxima is a floor below which no alternative of the block lies.  Of every thread's steps the maxima of eight segments are
// kept, and only segments that reach the floor, about k, are read once more (1024 rows of 151936: whole threads instead were 15 us of fetches from HBM); what reaches it is
// sorted as 64-bit keys, ordered bits of x and complement of the index.  Lists kept during the pass instead cost 3 to 5 times the pass.
// A row belongs to a cluster of C blocks, whose parts are joined over distributed shared memory: one launch, no workspace, no order of arrival in the result.
// Measured: 1024 bf16 rows of 151936 56 us (5.5 TB/s, of 6.5), 68 with twenty alternatives (bound by the exponentials' pipe, 57 % busy, and issue, 63 %); one fp32 row of 151936 4.4 us, 8.4 with
// eight alternatives (start, one trip to memory, the cluster's exchange).
// -inf (a masked token) adds nothing; a row of nothing else has log probabilities -inf and entropy 0; NaN or +inf anywhere makes a row's numbers NaN (its order
// of alternatives counts NaN as -inf).
// ------------------------------------------------------------------------------------------------
constexpr int kLpMaxCluster = 16;
constexpr int kLpUnroll = 4;          // 16-byte vectors in flight per thread
constexpr uint32_t kLpSegs = 8;       // segments of a thread's steps whose maxima are kept

template <typename T> struct Elem;
template <> struct Elem<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void widen(const uint4 &v, float *x) { x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w); }
    static __device__ __forceinline__ float one(const float *p) { return __ldg(p); }
};
template <> struct Elem<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void widen(const uint4 &v, float *x) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ float one(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
};
template <> struct Elem<__half> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void widen(const uint4 &v, float *x) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) { const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i])); x[2 * i] = f.x; x[2 * i + 1] = f.y; }
    }
    static __device__ __forceinline__ float one(const __half *p) { return __half2float(*p); }
};

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
constexpr float kLog2e = 1.4426950408889634f;

// keys: larger is better.  Bits of x ordered as unsigned numbers (-0 as 0, NaN as -inf), then the complement of the index; 0 is "none"
__device__ __forceinline__ unsigned long long top_key(float x, uint32_t idx) {
    x = x != x ? -INFINITY : x + 0.0f;
    uint32_t u = __float_as_uint(x);
    u = (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return ((unsigned long long)u << 32) | (uint32_t)~idx;
}
__device__ __forceinline__ float key_value(unsigned long long k) {
    const uint32_t u = (uint32_t)(k >> 32);
    return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u);
}

// 32 lanes' keys into descending order
__device__ __forceinline__ unsigned long long warp_sort(unsigned long long v) {
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (uint32_t size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (uint32_t step = size >> 1; step > 0; step >>= 1) {
            const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, step);
            const bool down = (lane & size) == 0, first = (lane & step) == 0;
            v = (down == first) == (v > o) ? v : o;
        }
    return v;
}
// the 32 best of two descending lists, descending
__device__ __forceinline__ unsigned long long warp_merge(unsigned long long a, unsigned long long b) {
    const uint32_t lane = threadIdx.x & 31u;
    b = __shfl_xor_sync(0xffffffffu, b, 31u);
    unsigned long long v = a > b ? a : b;
#pragma unroll
    for (uint32_t step = 16; step > 0; step >>= 1) {
        const unsigned long long o = __shfl_xor_sync(0xffffffffu, v, step);
        v = ((lane & step) == 0) == (v > o) ? v : o;
    }
    return v;
}

struct TopList {
    unsigned long long list = 0, kth = 0;
    uint32_t top;
    __device__ __forceinline__ void take(unsigned long long key) {          // every lane brings one key (0: none)
        uint32_t more = __ballot_sync(0xffffffffu, key > kth);
        if (!more) return;
        if (__popc(more) > 5) list = warp_merge(list, warp_sort(key));
        else
            for (; more; more &= more - 1u) {
                const unsigned long long k = __shfl_sync(0xffffffffu, key, __ffs(more) - 1), up = __shfl_up_sync(0xffffffffu, list, 1);
                if (!(list > k)) list = (threadIdx.x & 31u) == 0 || up > k ? k : up;
            }
        kth = __shfl_sync(0xffffffffu, list, top - 1u);
    }
};

struct Sums { float m, z, s; };
__device__ __forceinline__ Sums join(const Sums &a, const Sums &b) {
    Sums r;
    r.m = fmaxf(a.m, b.m);
    const float da = a.m - r.m, db = b.m - r.m, fa = ex2(da * kLog2e), fb = ex2(db * kLog2e);
    r.z = a.z * fa + b.z * fb;
    r.s = (fa > 0.0f ? fa * fmaf(a.z, da, a.s) : 0.0f) + (fb > 0.0f ? fb * fmaf(b.z, db, b.s) : 0.0f);
    if (r.m == INFINITY) r.z = NAN;
    return r;
}
__device__ __forceinline__ Sums shfl(const Sums &a, int step) {
    return Sums{__shfl_xor_sync(0xffffffffu, a.m, step), __shfl_xor_sync(0xffffffffu, a.z, step), __shfl_xor_sync(0xffffffffu, a.s, step)};
}

// What a thread has seen: m, and z, s in units of 2^u, u = m log2 e as it was rounded while m is small (d = x log2 e - u is then one multiply-add), and exact where m is
// not (m - x first: nothing overflows, and the rounding of a large product does not count)
constexpr float kSmallLogit = 4096.0f;
struct Running {
    float m = -FLT_MAX, seg = -INFINITY; pair_t z = 0, s = 0;          // seg: largest number of the present segment; z and s: partial sums of the even and of the odd places
    static __device__ __forceinline__ float off(float m) { return fabsf(m) < kSmallLogit ? fmaf(m, kLog2e, -__fmul_rn(m, kLog2e)) : 0.0f; }          // m log2 e - u
    __device__ __forceinline__ void rescale(float next, float d) {          // d: the old u less the new one
        const float f = ex2(d);
        const pair_t ff = pair(f, f), none = pair(0.0f, 0.0f);
        s = f > 0.0f ? fma2(fma2(z, pair(d, d), s), ff, none) : none;
        z = fma2(z, ff, none);
        m = next;
    }
    // false, and only m renewed, where a number is masked or outsize: -inf log2 e makes s NaN and z not
    template <int N> __device__ __forceinline__ bool see(const float (&x)[N]) {
        float top = x[0];
#pragma unroll
        for (int i = 1; i + 1 < N; i += 2) top = max3(top, x[i], x[i + 1]);
        if constexpr (N % 2 == 0) top = fmaxf(top, x[N - 1]);
        seg = fmaxf(seg, top);
        if (!(fabsf(fmaxf(top, m)) < kSmallLogit)) return false;
        if (top > m) rescale(top, __fsub_rn(__fmul_rn(fmaxf(m, -1e37f), kLog2e), __fmul_rn(top, kLog2e)));
        const float c = __fmul_rn(m, kLog2e);
        const pair_t L = pair(kLog2e, kLog2e), cc = pair(-c, -c);
        pair_t zn = z, sn = s;
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const pair_t d = fma2(pair(x[i], x[i + 1]), L, cc);
            float a, b;
            unpair(d, a, b);
            const pair_t p = pair(ex2(a), ex2(b));
            zn = add2(zn, p);
            sn = fma2(p, d, sn);
        }
        float za, zb, sa, sb;
        unpair(zn, za, zb); unpair(sn, sa, sb);
        const float sum = sa + sb, all = za + zb;
        if (sum != sum && all == all) return false;
        z = zn; s = sn;
        return true;
    }
    // any numbers; what weighs nothing is left out of s (0 times -inf)
    template <int N> __device__ __forceinline__ void see_any(const float (&x)[N]) {
        float top = x[0];
#pragma unroll
        for (int i = 1; i < N; i++) top = fmaxf(top, x[i]);
        seg = fmaxf(seg, top);
        if (top > m) rescale(top, (m - top) * kLog2e - off(m) + off(top));
        float za, zb, sa, sb;
        unpair(z, za, zb); unpair(s, sa, sb);
        const float o = off(m);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float d = fmaf(x[i] - m, kLog2e, o), p = ex2(d);
            if (i & 1) { zb += p; sb = fmaf(p, fmaxf(d, -1e4f), sb); } else { za += p; sa = fmaf(p, fmaxf(d, -1e4f), sa); }
        }
        z = pair(za, zb); s = pair(sa, sb);
    }
    __device__ __forceinline__ Sums done() const {
        float za, zb, sa, sb;
        unpair(z, za, zb); unpair(s, sa, sb);
        const float o = off(m), f = ex2(-o), zz = za + zb;
        return Sums{m, zz * f, fmaf(-o, zz, sa + sb) * f * 0.69314718055994531f};
    }
};

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory"); }
template <typename W>
__device__ __forceinline__ W peer_word(const W *mine, uint32_t rank) {          // the word at the same place of block `rank`'s shared memory
    uint32_t at = (uint32_t)__cvta_generic_to_shared(mine), there;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(at), "r"(rank));
    W v;
    if constexpr (sizeof(W) == 8) asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(there) : "memory");
    else asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
    return v;
}

// The row as 16-byte vectors of memory: vector v holds the places [v N - head, v N - head + N), the first and the last vector possibly in part; [whole0, whole1) are whole
template <typename T>
struct RowVectors {
    const T *row; const uint4 *vecs; uint32_t head, vocab, nv, whole0, whole1;
    __device__ __forceinline__ RowVectors(const T *r, uint32_t V) : row(r), vocab(V) {
        constexpr uint32_t N = Elem<T>::N;
        vecs = reinterpret_cast<const uint4 *>(reinterpret_cast<uintptr_t>(r) & ~(uintptr_t)15u);
        head = (uint32_t)((reinterpret_cast<uintptr_t>(r) & 15u) / sizeof(T));
        nv = (head + V + N - 1u) / N; whole0 = head ? 1u : 0u; whole1 = (head + V) / N;
    }
    __device__ __forceinline__ bool whole(uint32_t v) const { return v >= whole0 && v < whole1; }
    // one of the others, number by number; `none` in the places outside the row
    __device__ __forceinline__ void edge(uint32_t v, float none, float *x) const {
#pragma unroll
        for (int e = 0; e < Elem<T>::N; e++) {
            const uint32_t i = v * Elem<T>::N + e - head;          // wraps below the row's start
            x[e] = i < vocab ? Elem<T>::one(row + i) : none;
        }
    }
    __device__ __forceinline__ uint32_t first(uint32_t v) const { return v ? v * Elem<T>::N - head : 0u; }
};

// 32 lanes' numbers into descending order, and the 32 largest of two such lists
__device__ __forceinline__ float sort32(float v) {
    const uint32_t lane = threadIdx.x & 31u;
#pragma unroll
    for (uint32_t size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (uint32_t step = size >> 1; step > 0; step >>= 1) {
            const float o = __shfl_xor_sync(0xffffffffu, v, step);
            v = ((lane & size) == 0) == ((lane & step) == 0) ? fmaxf(v, o) : fminf(v, o);
        }
    return v;
}
__device__ __forceinline__ float merge32(float a, float b) {
    const uint32_t lane = threadIdx.x & 31u;
    float v = fmaxf(a, __shfl_xor_sync(0xffffffffu, b, 31u));
#pragma unroll
    for (uint32_t step = 16; step > 0; step >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, v, step);
        v = (lane & step) == 0 ? fmaxf(v, o) : fminf(v, o);
    }
    return v;
}

// grid (C, rows), clusters of C blocks
template <typename T, bool TOP, int THREADS>
__global__ void __launch_bounds__(THREADS, 1024 / THREADS) k_logprobs(const LogprobArgs a, const uint32_t C) {
    constexpr int N = Elem<T>::N, WARPS = THREADS / 32;
    __shared__ unsigned long long lists[WARPS > kLpMaxCluster ? WARPS : kLpMaxCluster][32];
    __shared__ float tops[WARPS][32], red[3][WARPS], part[3];
    __shared__ float segs[TOP ? kLpSegs : 1][THREADS];
    __shared__ uint32_t flagged[TOP ? kLpSegs * THREADS : 1], flags, found;          // found: numbers that reach the floor
    const uint32_t tid = threadIdx.x, lane = tid & 31u, warp = tid >> 5, rank = C > 1 ? cluster_rank() : 0u;
    const T *row = static_cast<const T *>(a.logits) + (uint64_t)blockIdx.y * a.row_stride;

    long long token = -1;
    float xt = NAN;
    if (rank == 0 && tid == 0 && a.tokens) {          // (asked for now, used at the end)
        token = a.token_bytes == 8 ? static_cast<const long long *>(a.tokens)[blockIdx.y] : (long long)static_cast<const int *>(a.tokens)[blockIdx.y];
        if (token >= 0 && token < (long long)a.vocab) xt = Elem<T>::one(row + token);
    }

    const RowVectors<T> rv(row, a.vocab);
    const uint32_t nv = rv.nv, head = rv.head, each = (nv + C - 1u) / C;
    const uint32_t v0 = min(nv, rank * each), v1 = min(nv, v0 + each);
    Running run;
    // whole vectors [w0, w1): steps of kLpUnroll vectors to a thread without a test, a step's vectors worked on while the next step's are on their way; the rest one by one
    const uint32_t w0 = min(max(v0, rv.whole0), v1), w1 = max(min(v1, rv.whole1), w0), steps = (w1 - w0) / (THREADS * kLpUnroll);
    bool masked = false;          // rows with masked tokens have many
    auto see = [&](const auto &x) {
        if (!masked && run.see(x)) return;
        masked = true;
        run.see_any(x);
    };
    const uint32_t seg_steps = (steps + kLpSegs) / kLpSegs;          // (the rest is one more step)
    uint4 ahead[kLpUnroll];
    const uint4 *next = rv.vecs + w0 + tid;
    if (steps)
#pragma unroll
        for (int j = 0; j < kLpUnroll; j++) ahead[j] = __ldg(next + j * THREADS);
    for (uint32_t step = 0; step < steps; step++) {
        uint4 raw[kLpUnroll];
#pragma unroll
        for (int j = 0; j < kLpUnroll; j++) raw[j] = ahead[j];
        next += THREADS * kLpUnroll;
        if (step + 1u < steps)
#pragma unroll
            for (int j = 0; j < kLpUnroll; j++) ahead[j] = __ldg(next + j * THREADS);
#pragma unroll
        for (int j = 0; j < kLpUnroll; j += 2) {
            float x[2 * N];
            Elem<T>::widen(raw[j], x);
            Elem<T>::widen(raw[j + 1], x + N);
            see(x);
        }
        if (TOP && (step + 1u) % seg_steps == 0) { segs[step / seg_steps][tid] = run.seg; run.seg = -INFINITY; }
    }
    {
        const uint32_t left = w0 + steps * THREADS * kLpUnroll + tid;
#pragma unroll
        for (int j = 0; j < kLpUnroll; j++) if (left + j * THREADS < w1) ahead[j] = __ldg(next + j * THREADS);
#pragma unroll
        for (int j = 0; j < kLpUnroll; j++) {
            if (left + j * THREADS >= w1) break;
            float x[N];
            Elem<T>::widen(ahead[j], x);
            see(x);
        }
        if (TOP) segs[steps / seg_steps][tid] = run.seg;
        // the row's first and last vector, if they are not whole
        const uint32_t v = tid == 0 ? 0u : nv - 1u;
        if (tid < 2 && v >= v0 && v < v1 && !rv.whole(v) && (tid == 0 || nv > 1u)) {
            float x[N];
            rv.edge(v, -INFINITY, x);
            run.see_any(x);
        }
    }
    Sums t = run.done();
    [[maybe_unused]] const float mine = t.z == 0.0f ? -INFINITY : t.m;          // this thread's largest logit

#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = join(t, shfl(t, o));
    if (lane == 0) { red[0][warp] = t.m; red[1][warp] = t.z; red[2][warp] = t.s; }
    if constexpr (TOP) { tops[warp][lane] = sort32(mine); if (tid == 0) flags = found = 0; }
    __syncthreads();
    bool nan = false;
    if constexpr (TOP) {
#pragma unroll
        for (uint32_t half = WARPS / 2; half > 0; half >>= 1) {
            if (warp < half) tops[warp][lane] = merge32(tops[warp][lane], tops[warp + half][lane]);
            __syncthreads();
        }
#pragma unroll
        for (int w = 0; w < WARPS; w++) nan = nan || red[1][w] != red[1][w];
        const float low = nan ? -INFINITY : tops[0][a.top - 1u];
        // the threads that have alternatives, their vectors dealt out one to a lane
        if (w0 + tid < w1 && (nan || !(mine < low)))
            for (uint32_t g = 0; g <= steps / seg_steps; g++) if (nan || !(segs[g][tid] < low)) flagged[atomicAdd(&flags, 1u)] = g * THREADS + tid;
        __syncthreads();
        // (and the two vectors that are not whole, whoever took them; at most all vectors, rounded up: below 2^32)
        const uint32_t per = seg_steps * kLpUnroll, total = 2u + flags * per;
        auto fetch = [&](uint32_t q, float (&x)[N]) {
            uint32_t v = v1;
            if (q >= 2u && q < total) { const uint32_t f = flagged[(q - 2u) / per]; v = w0 + f % THREADS + (f / THREADS * per + (q - 2u) % per) * THREADS; v = v < w1 ? v : v1; }
            else if (q < 2u && (q == 0 ? rv.whole0 != 0 || rv.whole1 == 0 : nv > 1u && rv.whole1 < nv)) { v = q ? nv - 1u : 0u; v = v >= v0 && v < v1 ? v : v1; }
            if (v < v1 && rv.whole(v)) Elem<T>::widen(__ldg(rv.vecs + v), x);
            else if (v < v1) rv.edge(v, -INFINITY, x);
            else
#pragma unroll
                for (int e = 0; e < N; e++) x[e] = -INFINITY;
            return v;
        };
        bool few = flags <= THREADS / 4u;
        if (tops[0][0] == -INFINITY && !nan) {          // nothing but masked tokens: the first ones
            const uint32_t i = rv.first(v0) + lane;
            if (warp == 0) lists[0][lane] = v0 < v1 && i < min(v1 * N - head, a.vocab) ? top_key(-INFINITY, i) : 0ull;
            __syncthreads();
        } else {
            if (few) {          // whatever reaches the floor, in any order; sorted afterwards
                for (uint32_t q0 = warp * 32u; q0 < total; q0 += THREADS * 2u) {
                    float x[2][N];
                    uint32_t v[2];
#pragma unroll
                    for (int u = 0; u < 2; u++) v[u] = fetch(q0 + u * THREADS + lane, x[u]);
#pragma unroll
                    for (int u = 0; u < 2; u++) {
                        float top = x[u][0];
#pragma unroll
                        for (int e = 1; e < N; e++) top = fmaxf(top, x[u][e]);
                        if (v[u] >= v1 || top < low) continue;
#pragma unroll
                        for (int e = 0; e < N; e++)
                            if (!(x[u][e] < low) && v[u] * N + e - head < a.vocab) {
                                const uint32_t at = atomicAdd(&found, 1u);
                                if (at < WARPS * 32u) (&lists[0][0])[at] = top_key(x[u][e], v[u] * N + e - head);
                            }
                    }
                }
                __syncthreads();
                const uint32_t n = found;
                few = n <= WARPS * 32u;
                if (few) {
                    if (warp * 32u < n || warp == 0) lists[warp][lane] = warp_sort(warp * 32u + lane < n ? lists[warp][lane] : 0ull);
                    for (uint32_t w = 1; w * 32u < n; w <<= 1) {          // (as many lists as there are, by pairs)
                        __syncthreads();
                        if (warp % (2u * w) == 0 && (warp + w) * 32u < n) lists[warp][lane] = warp_merge(lists[warp][lane], lists[warp + w][lane]);
                    }
                }
                __syncthreads();
            }
            if (!few) {          // rows full of equal numbers: a list to a warp, which only a better key enters
                TopList best;
                best.top = a.top;
                for (uint32_t q0 = warp * 32u; q0 < total; q0 += THREADS) {
                    float x[N];
                    const uint32_t v = fetch(q0 + lane, x), first = v * N - head;
                    float top = x[0];
#pragma unroll
                    for (int e = 1; e < N; e++) top = fmaxf(top, x[e]);
                    // (no key of the vector is above that of its largest number at its first place)
                    if (!__any_sync(0xffffffffu, v < v1 && !(top < low) && top_key(top, rv.first(v)) > best.kth)) continue;
#pragma unroll
                    for (int e = 0; e < N; e++) {
                        const bool in = v < v1 && first + e < a.vocab && !(x[e] < low);
                        if (__any_sync(0xffffffffu, in)) best.take(in ? top_key(x[e], first + e) : 0ull);
                    }
                }
                lists[warp][lane] = best.list;
                __syncthreads();
#pragma unroll
                for (uint32_t half = WARPS / 2; half > 0; half >>= 1) {
                    if (warp < half) lists[warp][lane] = warp_merge(lists[warp][lane], lists[warp + half][lane]);
                    __syncthreads();
                }
            }
        }
    }
    if (warp == 0) {
        t = Sums{lane < WARPS ? red[0][lane] : -FLT_MAX, lane < WARPS ? red[1][lane] : 0.0f, lane < WARPS ? red[2][lane] : 0.0f};
#pragma unroll
        for (int o = WARPS / 2; o > 0; o >>= 1) t = join(t, shfl(t, o));
        if (lane == 0) { part[0] = t.m; part[1] = t.z; part[2] = t.s; }
    }
    if (C > 1) {
        cluster_sync();
        if (rank == 0) {
            if constexpr (TOP)
                for (uint32_t peer = warp ? warp : WARPS; peer < C; peer += WARPS) {          // (the block's own list stays where it is)
                    const unsigned long long k = peer_word(&lists[0][lane], peer);
                    __syncwarp();
                    lists[peer][lane] = k;
                }
            if (warp == 0) {
                t = Sums{lane < C ? peer_word(&part[0], lane) : -FLT_MAX, lane < C ? peer_word(&part[1], lane) : 0.0f, lane < C ? peer_word(&part[2], lane) : 0.0f};
#pragma unroll
                for (int o = kLpMaxCluster / 2; o > 0; o >>= 1) t = join(t, shfl(t, o));
            }
            if constexpr (TOP) {
                __syncthreads();
                for (uint32_t half = C / 2; half > 0; half >>= 1) {
                    if (warp < half) lists[warp][lane] = warp_merge(lists[warp][lane], lists[warp + half][lane]);
                    __syncthreads();
                }
            }
        }
        cluster_sync();          // nobody leaves while its shared memory is read
    }
    if (rank || warp) return;
    t.m = __shfl_sync(0xffffffffu, t.m, 0); t.z = __shfl_sync(0xffffffffu, t.z, 0); t.s = __shfl_sync(0xffffffffu, t.s, 0);
    const bool empty = t.z == 0.0f;          // (a NaN is no zero)
    const float lz = logf(t.z);
    const uint64_t r = blockIdx.y;
    if (lane == 0) {
        if (a.logprob) a.logprob[r] = xt != xt ? NAN : empty ? -INFINITY : (xt - t.m) - lz;
        if (a.entropy) a.entropy[r] = empty ? 0.0f : lz - t.s / t.z;
    }
    if (TOP && lane < a.top) {
        const unsigned long long k = lists[0][lane];
        if (a.top_logprob) a.top_logprob[r * a.top + lane] = empty ? -INFINITY : (key_value(k) - t.m) - lz;
        if (a.top_id) a.top_id[r * a.top + lane] = (int32_t)~(uint32_t)k;
    }
}

template <typename T, bool TOP, int THREADS>
cudaError_t logprobs_launch_of(const LogprobArgs &a, cudaStream_t stream) {
    const uint32_t nv = (a.vocab + Elem<T>::N - 1u) / Elem<T>::N;
    // blocks to a row: until there is one for each SM, as long as a thread keeps a step's vectors.  us at 1 / 2 / 4 / 8 / 16 blocks, with eight alternatives: one row of 151936
    // fp32 numbers 24 / 17 / 12 / 9 / 8, 64 of 32000 8.6 / 7.5 / 7.5 / 8.3, 256 bf16 rows of 32000 9.1 / 11.4 / 16.5, 1024 of 151936 77 / 89 / 111
    uint32_t C = 1;
    while (C < kLpMaxCluster && nv >= (uint32_t)kLpUnroll * C * THREADS && (uint64_t)a.rows * C < 148u) C *= 2;
    if (C > 8) {          // more than eight blocks to a cluster are to be asked for, on every device that runs them
        cudaError_t e = cudaFuncSetAttribute(k_logprobs<T, TOP, THREADS>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    return in_portions(a.rows, 65535u, [&](uint32_t r0, uint32_t n) {          // (the grid's second dimension)
        LogprobArgs b = a;
        b.rows = n;
        b.logits = static_cast<const char *>(a.logits) + (uint64_t)r0 * a.row_stride * sizeof(T);
        if (a.tokens) b.tokens = static_cast<const char *>(a.tokens) + (uint64_t)r0 * a.token_bytes;
        if (a.logprob) b.logprob += r0;
        if (a.entropy) b.entropy += r0;
        if (a.top_logprob) b.top_logprob += (uint64_t)r0 * a.top;
        if (a.top_id) b.top_id += (uint64_t)r0 * a.top;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(C, b.rows); cfg.blockDim = dim3(THREADS); cfg.stream = stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = C; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr; cfg.numAttrs = 1;
        return cudaLaunchKernelEx(&cfg, k_logprobs<T, TOP, THREADS>, b, C);
    });
}

// Blocks of 256 threads; of 128 where there are more rows than blocks of 256 run at once (four to an SM) and a row is short, so that what follows a row's pass has more
// blocks beside it: with eight alternatives 2000 rows of 4000 fp32 numbers 15.7 us instead of 22.6, 600 bf16 rows of 16000 11.7 instead of 14.8; but 64 of 7000 7.4 instead of 6.4, 300 of
// 151936 37.7 instead of 32.6
template <typename T, bool TOP>
cudaError_t logprobs_launch_t(const LogprobArgs &a, cudaStream_t stream) {
    return a.rows >= 4u * 148u && a.vocab < 4u * kLpUnroll * 256u * Elem<T>::N ? logprobs_launch_of<T, TOP, 128>(a, stream) : logprobs_launch_of<T, TOP, 256>(a, stream);
}

// ------------------------------------------------------------------------------------------------
// Copies of pages.  Pure movement: a block takes 8 KB of one page of one pool, with every load in flight before the first store.  The pairs and the pools
// travel with the launch, so the call reads no memory of the caller's later and copies nothing to the device.  Bound by memory: 1000 pages of 40 KB in 8 pools 101 us (6.5 TB/s there and back).
// ------------------------------------------------------------------------------------------------
constexpr uint32_t kCopyThreads = 256, kCopyVecs = 2, kCopyChunk = kCopyThreads * kCopyVecs * 16u;
template <uint32_t PAIRS>
struct PageArgs { PagePool pool[kPagePools]; uint32_t src[PAIRS], dst[PAIRS]; };
template <uint32_t PAIRS, bool VEC>
__global__ void __launch_bounds__(kCopyThreads) k_pages_copy(const __grid_constant__ PageArgs<PAIRS> a) {
    const PagePool &p = a.pool[blockIdx.z];
    const uint64_t at = (uint64_t)blockIdx.x * kCopyChunk;
    if (at >= p.page_bytes) return;
    const uint64_t n = min((uint64_t)kCopyChunk, p.page_bytes - at);
    const char *from = static_cast<const char *>(p.base) + a.src[blockIdx.y] * p.page_stride + at;
    char *to = static_cast<char *>(p.base) + a.dst[blockIdx.y] * p.page_stride + at;
    if constexpr (VEC) {
        uint4 v[kCopyVecs];
#pragma unroll
        for (uint32_t i = 0; i < kCopyVecs; i++) { const uint32_t o = (threadIdx.x + i * kCopyThreads) * 16u; if (o < n) v[i] = __ldcs(reinterpret_cast<const uint4 *>(from + o)); }
#pragma unroll
        for (uint32_t i = 0; i < kCopyVecs; i++) { const uint32_t o = (threadIdx.x + i * kCopyThreads) * 16u; if (o < n) *reinterpret_cast<uint4 *>(to + o) = v[i]; }
    } else
        for (uint32_t o = threadIdx.x; o < n; o += kCopyThreads) to[o] = from[o];
}
template <uint32_t PAIRS, bool VEC>
cudaError_t pages_launch(const PagePool *pools, uint32_t n_pools, const uint32_t *src, const uint32_t *dst, uint32_t n, uint64_t bytes, cudaStream_t stream) {
    PageArgs<PAIRS> a;
    for (uint32_t i = 0; i < n_pools; i++) a.pool[i] = pools[i];
    std::copy(src, src + n, a.src);
    std::copy(dst, dst + n, a.dst);
    k_pages_copy<PAIRS, VEC><<<dim3((uint32_t)((bytes + kCopyChunk - 1u) / kCopyChunk), n, n_pools), kCopyThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t logprobs_launch(const LogprobArgs &a, cudaStream_t stream) {
    if (!a.rows) return cudaSuccess;
    return a.type == T_F32 ? (a.top ? logprobs_launch_t<float, true>(a, stream) : logprobs_launch_t<float, false>(a, stream))
         : a.type == T_BF16 ? (a.top ? logprobs_launch_t<__nv_bfloat16, true>(a, stream) : logprobs_launch_t<__nv_bfloat16, false>(a, stream))
                            : (a.top ? logprobs_launch_t<__half, true>(a, stream) : logprobs_launch_t<__half, false>(a, stream));
}

cudaError_t pages_copy_launch(const PagePool *pools, uint32_t n_pools, const uint32_t *src, const uint32_t *dst, uint32_t n, cudaStream_t stream, uint32_t *launches) {
    return in_portions(n_pools, kPagePools, [&](uint32_t p0, uint32_t np) -> cudaError_t {
        uint64_t bytes = 0;
        bool vec = true;
        for (uint32_t i = 0; i < np; i++) {
            const PagePool &p = pools[p0 + i];
            bytes = std::max(bytes, p.page_bytes);
            vec = vec && ((reinterpret_cast<uintptr_t>(p.base) | p.page_bytes | p.page_stride) & 15u) == 0;
        }
        if (!bytes) return cudaSuccess;
        return in_portions(n, kPagePairs, [&](uint32_t i, uint32_t m) {
            cudaError_t e;
            if (m <= 64u) e = vec ? pages_launch<64, true>(pools + p0, np, src + i, dst + i, m, bytes, stream) : pages_launch<64, false>(pools + p0, np, src + i, dst + i, m, bytes, stream);
            else e = vec ? pages_launch<kPagePairs, true>(pools + p0, np, src + i, dst + i, m, bytes, stream) : pages_launch<kPagePairs, false>(pools + p0, np, src + i, dst + i, m, bytes, stream);
            if (e == cudaSuccess && launches) ++*launches;
            return e;
        });
    });
}

}  // namespace nb

using nb::fail;

namespace {
// Pools of one call whose memory meets: pages of several layers may lie side by side in one tensor, but no page that is written may lie over another that is read or written (blocks run in any
// order).  The pool given twice is taken once.  A walk over the pools where their memory is apart, which is the rule; residues of the stride where their pages are interleaved; else every page that is touched is looked at.
int pages_apart(std::vector<nb::PagePool> &list, uint32_t pages, const uint32_t *src, const uint32_t *dst, uint32_t n) {
    typedef unsigned __int128 wide;
    auto start = [](const nb::PagePool &p) { return (uint64_t)reinterpret_cast<uintptr_t>(p.base); };
    auto end = [&](const nb::PagePool &p) { return (wide)start(p) + (wide)(pages - 1u) * p.page_stride + p.page_bytes; };
    list.erase(std::remove_if(list.begin(), list.end(), [](const nb::PagePool &p) { return p.page_bytes == 0; }), list.end());
    bool apart = true;
    for (size_t i = 1; i < list.size(); i++) apart = apart && end(list[i - 1]) <= start(list[i]);
    if (apart) return 0;
    auto key = [&](const nb::PagePool &p) { return std::make_tuple(start(p), p.page_stride, p.page_bytes); };
    std::sort(list.begin(), list.end(), [&](const nb::PagePool &a, const nb::PagePool &b) { return key(a) < key(b); });
    list.erase(std::unique(list.begin(), list.end(), [&](const nb::PagePool &a, const nb::PagePool &b) { return key(a) == key(b); }), list.end());
    bool even = true;
    wide last = 0;
    apart = true;
    for (const nb::PagePool &p : list) { apart = apart && last <= start(p); last = std::max(last, end(p)); even = even && p.page_stride == list[0].page_stride; }
    if (apart) return 0;
    if (even) {
        const uint64_t step = list[0].page_stride;
        std::vector<std::pair<uint64_t, uint64_t>> at;          // where in a step a pool's pages lie
        for (const nb::PagePool &p : list) at.emplace_back((start(p) - start(list[0])) % step, p.page_bytes);
        std::sort(at.begin(), at.end());
        bool free = (wide)at.back().first + at.back().second <= (wide)step + at[0].first;
        for (size_t i = 1; i < at.size(); i++) free = free && at[i - 1].first + at[i - 1].second <= at[i].first;
        if (free) return 0;
    }
    struct Touch { wide from, to; bool write; };
    std::vector<Touch> touched;
    touched.reserve(2u * (size_t)n * list.size());
    for (const nb::PagePool &p : list)
        for (uint32_t i = 0; i < n; i++)
            for (const bool write : {false, true}) { const wide from = (wide)start(p) + (wide)(write ? dst[i] : src[i]) * p.page_stride; touched.push_back(Touch{from, from + p.page_bytes, write}); }
    std::sort(touched.begin(), touched.end(), [](const Touch &a, const Touch &b) { return a.from < b.from; });
    wide written = 0, any = 0;          // where what lies before ends
    for (const Touch &t : touched) {
        if (t.from < written || (t.write && t.from < any)) return fail(NB200_EINVAL, "pools overlap: a page that this call writes in one lies over a page that it reads or writes in another");
        any = std::max(any, t.to);
        if (t.write) written = std::max(written, t.to);
    }
    return 0;
}
}  // namespace

extern "C" {

int nb200_dev_token_logprobs(float *logprob, float *entropy, float *top_logprob, int32_t *top_id, const void *logits, uint32_t type, uint64_t row_stride,
                             uint32_t rows, uint32_t vocab, const void *tokens, uint32_t token_bytes, uint32_t top, void *stream) {
    if (type > nb::T_F16) return fail(NB200_EINVAL, "logits are fp32, bf16 or fp16 (type %u)", type);
    if (rows && (!logits || !vocab || vocab > 0x7fffffffu)) return fail(NB200_EINVAL, "bad logits (%u rows of %u)", rows, vocab);
    if (reinterpret_cast<uintptr_t>(logits) % nb::elem_size(type)) return fail(NB200_EINVAL, "logits are not aligned to their type");
    if (tokens && token_bytes != 4 && token_bytes != 8) return fail(NB200_EINVAL, "tokens are 32-bit or 64-bit numbers");
    if (tokens && reinterpret_cast<uintptr_t>(tokens) % token_bytes) return fail(NB200_EINVAL, "tokens are not aligned to their type");
    if (top > nb::kTopMax || (rows && top > vocab)) return fail(NB200_EINVAL, "%u alternatives asked for: at most %u, and no more than the vocabulary has", top, nb::kTopMax);
    if (logprob && !tokens) return fail(NB200_EINVAL, "log probabilities need tokens");
    if (top && !top_logprob && !top_id) top = 0;
    if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
    const nb::LogprobArgs a{logits, row_stride, type, rows, vocab, logprob ? tokens : nullptr, token_bytes, top, logprob, entropy, top_logprob, top_id};
    NB_CK(nb::logprobs_launch(a, static_cast<cudaStream_t>(stream)));
    return 0;
}

int nb200_dev_pages_copy(void *const *pools, const uint64_t *page_bytes, const uint64_t *page_stride, const uint32_t *n_pages, uint32_t n_pools, const uint32_t *src,
                         const uint32_t *dst, uint32_t n, void *stream) {
    if ((n_pools && (!pools || !page_bytes || !page_stride || !n_pages)) || (n && (!src || !dst))) return fail(NB200_EINVAL, "null argument");
    try {
        uint32_t pages = n_pools ? 0xffffffffu : 0u;
        std::vector<nb::PagePool> list(n_pools);
        for (uint32_t i = 0; i < n_pools; i++) {
            if (!pools[i] && page_bytes[i] && n_pages[i]) return fail(NB200_EINVAL, "pool %u is null", i);
            if (page_bytes[i] > (1ull << 32) || page_stride[i] < page_bytes[i]) return fail(NB200_EINVAL, "pool %u: pages of %llu bytes every %llu", i, (unsigned long long)page_bytes[i], (unsigned long long)page_stride[i]);
            list[i] = nb::PagePool{pools[i], page_bytes[i], page_stride[i]};
            pages = std::min(pages, n_pages[i]);
        }
        if (!n_pools || !n) return 0;
        std::vector<bool> used(pages, false);
        for (uint32_t i = 0; i < n; i++) {
            if (src[i] >= pages || dst[i] >= pages) return fail(NB200_EINVAL, "pair %u copies page %u to %u, one outside: the smallest pool has %u", i, src[i], dst[i], pages);
            used[src[i]] = true;
        }
        for (uint32_t i = 0; i < n; i++) {
            if (used[dst[i]]) return fail(NB200_EINVAL, "page %u is written and read, or written twice, by one call", dst[i]);
            used[dst[i]] = true;
        }
        if (const int r = pages_apart(list, pages, src, dst, n)) return r;
        if (nb200_device_count() <= 0) return fail(NB200_ENODEV, "no CUDA device: nano_b200 has no CPU path");
        NB_CK(nb::pages_copy_launch(list.data(), (uint32_t)list.size(), src, dst, n, static_cast<cudaStream_t>(stream), nullptr));
    } catch (const std::bad_alloc &) { return fail(NB200_ENOMEM, "out of host memory"); }
    return 0;
}

}  // extern "C"
