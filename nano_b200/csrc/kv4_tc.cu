// kv4_tc.cu -- attention of long portions over a cache held in 4 bits, on the fifth-generation tensor cores (formulas: kv4.h).
//
// A block owns 128 rows (query token, query head) of one key/value head and walks their keys in tiles of 128, four pages.  Seven warps make a tile's operands from the codes,
// by the page: a word of eight key codes is one 16-byte piece of a row of the swizzled key operand (the queries are laid out in the nibbles' order, so that nothing is
// shuffled), eight tokens' codes of a coordinate one piece of a row of the value operand, both as c s + m in fp16, rounded once; two tiles' operands have room.  One thread
// issues tcgen05.mma -- scores into tensor memory, two buffers, and weights (fp16, where the scores were) times values onto the running sum there -- and eight warps do the
// softmax, two threads to a row with 64 of its scores in registers each (one thread to a row: 46 us instead of 41 for 1000 tokens of 16 heads of 64 over 4 behind 3100 and a window of 2500,
// 58 instead of 51 with a soft cap).
// Every wait has a limit; a block in which one runs out leaves with NaN in its rows (nothing but its own products is ever in flight) and a code in the engine's error word.
// Softmax as in k_kv4_attn: log2 units, weights times 2^kLift, a reference that is renewed when it lags kSlack behind the maximum, so that the sums in tensor memory
// are seldom touched.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "family.h"
#include "kv4.cuh"
#include "pairs.cuh"
#include "tc_ptx.cuh"

namespace nb {
namespace {

constexpr uint32_t kTile = 128, kPages = kTile / kKv4Page, kThreads = 512, kSoft = 8, kMmaWarp = 8, kMakers = 9, kProducers = 7;          // warps 0-7: softmax, 8: products, 9-15: operands
constexpr uint32_t kKeys = kTile / 2;          // of a tile, to a thread of the softmax
constexpr float kLift = 12.0f;
// byte of the 16-byte piece c8 (8 fp16) of row r in an operand of 64-wide blocks of `rows` rows, 128-byte swizzle
__device__ __forceinline__ uint32_t op_byte(uint32_t rows, uint32_t r, uint32_t c8) { return (c8 >> 3) * rows * 128u + r * 128u + (((c8 & 7u) ^ (r & 7u)) << 4); }
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// waits that mostly find what they wait for there: the first try without the clock
__device__ __forceinline__ bool soon(uint32_t bar, uint32_t parity) { return mbar_try(bar, parity) || mbar_wait(bar, parity); }
__device__ __forceinline__ bool soon_warp(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, soon(bar, parity)); }

template <int NG> struct Sizes {
    static constexpr uint32_t D = 32u * NG, DP = NG <= 2 ? 64u : 128u;          // coordinates; those that an operand of queries or keys has room for
    static constexpr uint32_t qk = kTile * DP * 2u, v = kTile * D * 2u, all = 3u * qk + 2u * v + 1024u;
};

// grid (nsplit x tiles, G, B)
template <int NG>
__global__ void __launch_bounds__(kThreads, 1) k_kv4_attn_tc(const Kv4Attn a, const Shape sh) {
    using Z = Sizes<NG>;
    constexpr uint32_t D = Z::D;
    extern __shared__ uint8_t tc_raw[];
    enum { KFULL = 0, KFREE = 2, VFULL = 4, VFREE = 6, SFULL = 8, PREADY = 10, ODONE = 12, NBAR = 14 };          // two each, tiles in turn.  (PREADY: a warp may be a tile ahead of the others; ODONE: nobody need have seen the tile before last's)
    __shared__ __align__(8) uint64_t bars[NBAR];
    __shared__ uint32_t tmem_s;
    __shared__ uint32_t hide_s[4][kPages], odd_s[4][kPages];          // of a tile's pages (four tiles in turn): keys that nobody sees, keys whose values are no number
    __shared__ float scale_s[kTile], top_s[2][kTile], sum_s[2][kTile];          // (what two warps that share rows tell each other)
    __shared__ uint32_t ok_s[2][kSoft];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t qs = (smem_u32(tc_raw) + 1023u) & ~1023u, ks = qs + Z::qk, vs = ks + 2u * Z::qk;
    unsigned char *base = tc_raw + (qs - smem_u32(tc_raw));
    const uint32_t split = blockIdx.x % sh.nsplit, tile = sh.tiles - 1u - blockIdx.x / sh.nsplit, g = blockIdx.y, b = blockIdx.z;          // the longest rows first
    const uint32_t rep = a.H / a.G, rows = a.T * rep, r0 = tile * kKv4TcRows, last = min(rows, r0 + kKv4TcRows) - 1u;
    const uint32_t b0 = smem_u32(bars);
    auto bar = [&](uint32_t i) { return b0 + i * 8u; };
    if (tid == 0) {
        for (uint32_t i = 0; i < NBAR; i++) mbar_init(bar(i), i < KFREE || (i >= VFULL && i < VFREE) ? kPages : i >= PREADY && i < ODONE ? kSoft : 1u);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kMmaWarp) { tc_alloc(smem_u32(&tmem_s), 512); tc_relinquish(); }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // Only now may the next kernel's blocks come: one that waits for this grid while it holds tensor memory must not be in the way of an allocation here
    asm volatile("griddepcontrol.launch_dependents;\ngriddepcontrol.wait;" ::: "memory");
    const uint32_t tmem = tmem_s;
    const int len = seq_len(a, b), pos_0 = len - (int)a.T;          // position of the first query
    const int first_pos = pos_0 + (int)(r0 / rep), last_pos = pos_0 + (int)(last / rep);
    uint32_t lo = 0, n = 0;
    if (last_pos >= 0) {
        const uint32_t first = (uint32_t)first_seen(max(first_pos, 0), a.window, a.block) / kTile, all = (uint32_t)last_pos / kTile + 1u - first;
        lo = first + (uint32_t)((uint64_t)all * split / sh.nsplit);
        n = first + (uint32_t)((uint64_t)all * (split + 1u) / sh.nsplit) - lo;
    }

    // queries as the row operand, each row times the power of two that brings its largest number to [1, 2); a piece's eight coordinates in the order 0 4 1 5 2 6 3 7
    {
        constexpr uint32_t pieces = 4u * NG, wide = NG == 1 ? 4u : NG == 2 ? 8u : 16u, per = 32u / wide;          // lanes to a row, rows to a warp
        const uint32_t c = lane % wide;
        for (uint32_t r = warp * per + lane / wide; r < kTile; r += kThreads / 32u * per) {
            const uint32_t rr = r0 + r, t = rr / rep, h = g * rep + rr % rep;
            float x[8] = {}, most = 0.0f;
            if (rr <= last && c < pieces) {
                const uint64_t at = b * a.q_batch + t * a.q_token + h * a.q_head + c * 8u;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    x[i] = a.type == T_F32 ? static_cast<const float *>(a.q)[at + i] : __bfloat162float(static_cast<const __nv_bfloat16 *>(a.q)[at + i]);
                    most = fmaxf(most, fabsf(x[i]));
                }
            }
#pragma unroll
            for (uint32_t o = wide / 2u; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            const int e = most > 0.0f ? min(max((int)(__float_as_uint(most) >> 23) - 127, -126), 126) : 0;
            float down = __uint_as_float((uint32_t)(127 - e) << 23);
            if (a.scale < 0.0f) down = -down;          // the largest product is to be the largest score
            if (c < pieces) {
                const uint4 v = make_uint4(bits(__floats2half2_rn(x[0] * down, x[4] * down)), bits(__floats2half2_rn(x[1] * down, x[5] * down)), bits(__floats2half2_rn(x[2] * down, x[6] * down)),
                                           bits(__floats2half2_rn(x[3] * down, x[7] * down)));
                *reinterpret_cast<uint4 *>(base + op_byte(kTile, r, c)) = v;
                if (c == 0) scale_s[r] = fabsf(a.scale) * __uint_as_float((uint32_t)(127 + e) << 23) * (a.softcap > 0.0f ? 1.0f / a.softcap : kLog2e);
            }
        }
        async_fence();
        __syncthreads();
    }

    // tensor memory: scores (two buffers of 128 columns), where a tile's weights take the place of its scores (64 columns), and the sums
    constexpr uint32_t OCOL = 256;
    if (warp == kMmaWarp) {
        if (lane == 0 && n) {
            constexpr uint32_t id_s = (1u << 4) | ((kTile >> 3) << 17) | ((kTile >> 4) << 24), id_o = (1u << 4) | ((D >> 3) << 17) | ((kTile >> 4) << 24);      // fp32 += f16 x f16
            auto scores = [&](uint32_t i) {
                const uint32_t s = i & 1u;
                if (!soon(bar(KFULL + s), (i >> 1) & 1u)) return false;
                tc_fence_after();
#pragma unroll
                for (uint32_t k = 0; k < 2u * NG; k++) {
                    const uint32_t off = (k >> 2) * kTile * 128u + (k & 3u) * 32u;
                    tc_mma_ss(tmem + s * kTile, tc_desc(qs + off), tc_desc(ks + s * Z::qk + off), id_s, k > 0);
                }
                tc_commit(bar(KFREE + s)); tc_commit(bar(SFULL + s));
                return true;
            };
            bool ok = scores(0) && (n < 2u || scores(1));
            for (uint32_t i = 0; i < n && ok; i++) {
                const uint32_t s = i & 1u;
                ok = soon(bar(VFULL + s), (i >> 1) & 1u) && soon(bar(PREADY + s), (i >> 1) & 1u);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (uint32_t k = 0; k < kTile / 16u; k++)
                    tc_mma_ts(tmem + OCOL, tmem + s * kTile + k * 8u, tc_desc(vs + s * Z::v + (k >> 2) * D * 128u + (k & 3u) * 32u), id_o, i > 0 || k > 0);
                tc_commit(bar(VFREE + s)); tc_commit(bar(ODONE + s));
                if (i + 2u < n) ok = soon(bar(ODONE + s), (i >> 1) & 1u) && scores(i + 2u);          // they overwrite the weights that the products before read
            }
        }
    } else if (warp >= kMakers) {
        // operands: a tile is eight pieces of work, the keys and then the values of its four pages, dealt out to seven warps in turn
        const uint32_t eight = lane >> 3, bv = lane & 7u;
        const int32_t *table = a.table + (uint64_t)b * a.table_stride;
        const int low_first = first_seen(max(first_pos, 0), a.window, a.block);          // the block's rows see the keys from here to last_pos, each at least one of them
        auto number = [&](uint32_t q) {          // the page of piece q (a length is no more than the table's width allows)
            const uint32_t p = (lo + q / (2u * kPages)) * kPages + q % kPages;
            return q < n * 2u * kPages && (int)(p * kKv4Page) <= last_pos ? (uint32_t)table[p] : 0xffffffffu;
        };
        uint32_t page = number(warp - kMakers);
        for (uint32_t q = warp - kMakers; q < n * 2u * kPages; q += kProducers) {
            const uint32_t i = q / (2u * kPages), s = i & 1u, pw = q % kPages, next = number(q + kProducers);
            const bool ok = page < a.n_pages;
            const unsigned char *block = a.pool + (uint64_t)(ok ? page : 0u) * a.page_stride + (uint64_t)g * kv4_block_bytes(D);
            if (q % (2u * kPages) < kPages) {
                uint32_t kw[4 * NG], kp[NG], odd = 0;          // odd: tokens whose values are no numbers
                if (ok) {
                    uint32_t own[NG];
                    take<16 * NG>(block + lane * 16u * NG, kw);
                    take<4 * NG>(block + 512u * NG + lane * 4u * NG, kp);
                    take<4 * NG>(block + 1152u * NG + lane * 4u * NG, own);
                    __half2 none = __float2half2_rn(0.0f);          // 0 times a pair is 0, or NaN
#pragma unroll
                    for (int j = 0; j < NG; j++) none = __hfma2(half2_of(own[j]), __float2half2_rn(0.0f), none);
                    odd = __ballot_sync(0xffffffffu, !__hbeq2(none, __float2half2_rn(0.0f)));
                } else {
#pragma unroll
                    for (int j = 0; j < NG; j++) kp[j] = 0u;
#pragma unroll
                    for (int j = 0; j < 4 * NG; j++) kw[j] = 0u;
                }
                if (i >= 2u && !soon_warp(bar(KFREE + s), ((i >> 1) - 1u) & 1u)) break;
                unsigned char *k_s = base + (1u + s) * Z::qk;
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    const __half2 st = __low2half2(half2_of(kp[j])), mn = __high2half2(half2_of(kp[j]));
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const uint32_t w = kw[x * NG + j];
                        *reinterpret_cast<uint4 *>(k_s + op_byte(kTile, pw * 32u + lane, 4u * j + x)) =
                            make_uint4(stand_for<false>(w, st, mn), stand_for<true>(w, st, mn), stand_for<false>(w >> 8, st, mn), stand_for<true>(w >> 8, st, mn));
                    }
                }
                if (lane == 0) { hide_s[i & 3u][pw] = ok ? 0u : 0xffffffffu; odd_s[i & 3u][pw] = odd; }
                async_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(KFULL + s));
            } else {
                uint32_t vp[8][NG], vw[8][(NG + 1) / 2];
                if (ok) {
#pragma unroll
                    for (uint32_t t = 0; t < 8; t++) {
                        take<2 * NG>(block + 640u * NG + (eight * 8u + t) * 16u * NG + bv * 2u * NG, vw[t]);
                        take<4 * NG>(block + 1152u * NG + (eight * 8u + t) * 4u * NG, vp[t]);
                    }
                } else {
#pragma unroll
                    for (uint32_t t = 0; t < 8; t++) {
#pragma unroll
                        for (int j = 0; j < NG; j++) vp[t][j] = 0u;
#pragma unroll
                        for (int j = 0; j < (NG + 1) / 2; j++) vw[t][j] = 0u;
                    }
                }
                // Tokens that no row sees hold any bytes: their weights are 0, but c s + m may be beyond fp16, and 0 times infinity is no number
                const int key = (int)((lo + i) * kTile + pw * kKv4Page + eight * 8u);
                if (key + 7 > last_pos || key < low_first)
#pragma unroll
                    for (uint32_t t = 0; t < 8; t++)
                        if (key + (int)t > last_pos || key + (int)t < low_first)
#pragma unroll
                            for (int j = 0; j < NG; j++) vp[t][j] = 0u;
                // tokens whose pairs are no numbers would spoil rows that do not see them
#pragma unroll
                for (uint32_t t = 0; t < 8; t++) {
                    __half2 none = __float2half2_rn(0.0f);
#pragma unroll
                    for (int j = 0; j < NG; j++) none = __hfma2(half2_of(vp[t][j]), __float2half2_rn(0.0f), none);
                    if (!__hbeq2(none, __float2half2_rn(0.0f)))
#pragma unroll
                        for (int j = 0; j < NG; j++) vp[t][j] = 0u;
                }
                if (i >= 2u && !soon_warp(bar(VFREE + s), ((i >> 1) - 1u) & 1u)) break;
                unsigned char *v_s = base + 3u * Z::qk + s * Z::v;
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    uint32_t y[4][4];          // [coordinate][pair of tokens]
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const uint32_t w = __byte_perm(vw[2 * x][j / 2], vw[2 * x + 1][j / 2], (j & 1) ? 0x7632u : 0x5410u);
                        const __half2 st = half2_of(__byte_perm(vp[2 * x][j], vp[2 * x + 1][j], 0x5410u)), mn = half2_of(__byte_perm(vp[2 * x][j], vp[2 * x + 1][j], 0x7632u));
                        y[0][x] = stand_for<false>(w, st, mn); y[1][x] = stand_for<true>(w, st, mn); y[2][x] = stand_for<false>(w >> 8, st, mn); y[3][x] = stand_for<true>(w >> 8, st, mn);
                    }
#pragma unroll
                    for (uint32_t d = 0; d < 4; d++) *reinterpret_cast<uint4 *>(v_s + op_byte(D, 32u * j + 4u * bv + d, pw * 4u + eight)) = make_uint4(y[d][0], y[d][1], y[d][2], y[d][3]);
                }
                async_fence();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar(VFULL + s));
            }
            page = next;
        }
    } else {
        // Two threads to a row: warps w and w + 4 share 32 rows, keys 0-63 and 64-127 of a tile.  They meet once a tile, when both hold their scores and the weights may take their
        // place, and tell each other more only where the reference moves or a wait ran out
        const uint32_t half = warp >> 2, r = (warp & 3u) * 32u + lane, rr = min(r0 + r, last), t = rr / rep, h = g * rep + rr % rep, id = 1u + (warp & 3u);
        const int pos = pos_0 + (int)t, low = first_seen(max(pos, 0), a.window, a.block), low_last = first_seen(max(last_pos, 0), a.window, a.block);
        const uint32_t lanes = ((warp & 3u) * 32u) << 16, o_at = tmem + lanes + OCOL;
        const float kc = scale_s[r], cap = a.softcap * kLog2e, kk = kc * kc;
        // the soft cap of a score x near 0 is x (c0 + c1 x^2 + c2 x^4 + c3 x^6); factors whose powers leave fp32 take the other way
        const float c0 = cap * kTanh0 * kc, c1 = cap * kTanh1 * kc * kk, c2 = cap * kTanh2 * kc * kk * kk, c3 = cap * kTanh3 * kc * kk * kk * kk, limit = kc > 1e-4f && kc < 1e4f ? kTanhNear / kc : 0.0f;
        float m = -INFINITY, l = 0.0f;
        bool ok = true;
        for (uint32_t i = 0; i < n; i++) {
            const int key0 = (int)((lo + i) * kTile);
            const uint32_t s_at = tmem + lanes + (i & 1u) * kTile;
            ok = ok && soon_warp(bar(SFULL + (i & 1u)), (i >> 1) & 1u);
            tc_fence_after();
            uint32_t w[kKeys];
            tc_ld64(s_at + half * kKeys, w);
            uint32_t hide = 0, odd = 0;
#pragma unroll
            for (uint32_t u = 0; u < kPages; u++) hide |= hide_s[i & 3u][u];
#pragma unroll
            for (uint32_t u = 0; u < 2; u++) odd |= odd_s[i & 3u][half * 2u + u];
            const bool whole = key0 + (int)kTile - 1 <= first_pos && key0 >= low_last && hide == 0;          // every row of the block sees every key
            auto sees = [&](uint32_t u) {          // of 32 keys those that this row sees
                const int at = key0 + 32 * (int)(half * 2u + u), from = low - at, to = pos - at;          // places [from, to]
                uint32_t v = to < 0 || from > 31 ? 0u : 0xffffffffu;
                if (to >= 0 && to < 31) v &= (2u << to) - 1u;
                if (from > 0 && from <= 31) v &= 0xffffffffu << from;
                return v & ~hide_s[i & 3u][half * 2u + u];
            };
            if (!whole)
#pragma unroll
                for (uint32_t u = 0; u < 2; u++) {
                    const uint32_t see = sees(u);
#pragma unroll
                    for (uint32_t j = 0; j < 32; j++) w[u * 32u + j] = see >> j & 1u ? w[u * 32u + j] : 0xff800000u;
                }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY}, fars[4] = {};          // (four at a time: one after the other, each would wait for the one before)
#pragma unroll
            for (uint32_t j = 0; j < kKeys; j += 2) tops[j / 2 & 3u] = max3(tops[j / 2 & 3u], __uint_as_float(w[j]), __uint_as_float(w[j + 1]));
            float top = fmaxf(max3(tops[0], tops[1], tops[2]), tops[3]);
            bool near = false;          // scores whose soft cap is a polynomial, taken where the weights are made
            if (a.softcap > 0.0f) {
#pragma unroll
                for (uint32_t j = 0; j < kKeys; j += 2) fars[j / 2 & 3u] = max3(fars[j / 2 & 3u], fabsf(__uint_as_float(w[j])), fabsf(__uint_as_float(w[j + 1])));
                near = __all_sync(0xffffffffu, fmaxf(max3(fars[0], fars[1], fars[2]), fars[3]) < limit);
                if (!near)
#pragma unroll
                    for (uint32_t j = 0; j < kKeys; j++) w[j] = w[j] == 0xff800000u ? w[j] : __float_as_uint(tanh_any(__uint_as_float(w[j]) * kc));
            }
            if (top != -INFINITY) { top *= kc; if (a.softcap > 0.0f) top = cap * tanh_any(top); }
            if (bar_any(id, 64u, !ok || top > m + kSlack)) {          // (m = -inf: top is taken, if there is one)
                top_s[half][r] = top;
                if (lane == 0) ok_s[0][warp] = ok;
                bar_any(id, 64u, false);
                if (!(ok = ok && ok_s[0][warp ^ 4u])) break;          // both leave
                top = fmaxf(top, top_s[half ^ 1u][r]);
                const float next = top > m + kSlack ? top : m, corr = next == m ? 1.0f : ex2(m - next);
                l *= corr;
                m = next;
                if (i) {          // the sums move to the new reference, once the products before are done; half of the columns each
                    ok = soon_warp(bar(ODONE + ((i - 1u) & 1u)), ((i - 1u) >> 1) & 1u);
                    tc_fence_after();
                    const pair_t k = pair(corr, corr);
#pragma unroll 1
                    for (uint32_t c = half * (D / 2u); ok && c < (half + 1u) * (D / 2u); c += 16u) {
                        uint32_t v[16];
                        tc_ld16(o_at + c, v);
#pragma unroll
                        for (uint32_t j = 0; j < 16; j += 2) {
                            float y, z;
                            unpair(mul2(pair(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), k), y, z);
                            v[j] = __float_as_uint(y); v[j + 1] = __float_as_uint(z);
                        }
                        tc_st16(o_at + c, v);
                    }
                }
            }
            const float use = m == -INFINITY ? 0.0f : m - kLift;
            // (masked scores are -inf, whatever the factor: 0 times -inf would be no number)
            const float by = a.softcap > 0.0f ? cap : whole ? kc : fmaxf(kc, 1e-30f);
            const pair_t k = pair(by, by), less = pair(-use, -use);
            pair_t s2[2] = {pair(0.0f, 0.0f), pair(0.0f, 0.0f)};
            auto weights = [&](auto capped) {
#pragma unroll
                for (uint32_t u = 0; u < 2; u++) {
                    uint32_t wh[16];
#pragma unroll
                    for (uint32_t j = 0; j < 16; j++) {
                        float y, z;
                        const pair_t x = pair(__uint_as_float(w[u * 32u + 2u * j]), __uint_as_float(w[u * 32u + 2u * j + 1u]));
                        if constexpr (capped.value) {
                            const pair_t xx = mul2(x, x);
                            unpair(fma2(x, fma2(xx, fma2(xx, fma2(xx, pair(c3, c3), pair(c2, c2)), pair(c1, c1)), pair(c0, c0)), less), y, z);
                        } else unpair(fma2(x, k, less), y, z);
                        y = ex2(y); z = ex2(z);
                        s2[j & 1u] = add2(s2[j & 1u], pair(y, z));
                        wh[j] = bits(__floats2half2_rn(y, z));
                    }
                    tc_st16(s_at + half * (kKeys / 2u) + u * 16u, wh);
                }
            };
            if (near) weights(std::true_type{}); else weights(std::false_type{});
            float s0, s1;
            unpair(add2(s2[0], s2[1]), s0, s1);
            l += s0 + s1;
            if (odd)          // values that are no number make the rows that see them NaN, however little they weigh
#pragma unroll 1
                for (uint32_t u = 0; u < 2; u++) if (odd_s[i & 3u][half * 2u + u] & sees(u)) l = NAN;
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(PREADY + (i & 1u)));
        }
        // (a tile's scores come after the products of the tile two before it: of the last two products this is known of neither)
        if (ok && n > 1u) ok = soon_warp(bar(ODONE + (n & 1u)), ((n - 2u) >> 1) & 1u);
        if (ok && n) { ok = soon_warp(bar(ODONE + ((n - 1u) & 1u)), ((n - 1u) >> 1) & 1u); tc_fence_after(); }
        sum_s[half][r] = l;
        if (lane == 0) ok_s[1][warp] = ok;
        bar_any(id, 64u, false);
        ok = ok && ok_s[1][warp ^ 4u];
        if (!ok && lane == 0 && a.err) *a.err = 0x300u + warp;          // (whoever's wait it was: without scores and products those of these warps run out too)
        const float ref = m - kLift, sum = ok ? l + sum_s[half ^ 1u][r] : NAN;          // a wait that ran out shows as NaN
        const bool mine = r0 + r <= last;
        const uint64_t where = (((uint64_t)(b * a.G + g) * sh.tiles + tile) * sh.nsplit + split) * sh.cols + r;
        const float k = sh.nsplit > 1 ? 1.0f : last_factor(a, t, h, ref, sum);
#pragma unroll 1
        for (uint32_t c = half * (D / 2u); c < (half + 1u) * (D / 2u); c += 16u) {
            uint32_t w[16] = {};
            if (n && ok) tc_ld16(o_at + c, w);
            if (mine)
#pragma unroll
                for (uint32_t j = 0; j < 16; j += 4) {
                    const float4 v = make_float4(__uint_as_float(w[j]), __uint_as_float(w[j + 1]), __uint_as_float(w[j + 2]), __uint_as_float(w[j + 3]));
                    if (sh.nsplit > 1) *reinterpret_cast<float4 *>(a.part + where * D + c + j) = v;
                    else store_four(a, b, t, h, c + j, v.x * k, v.y * k, v.z * k, v.w * k);
                }
        }
        if (half == 0 && mine && sh.nsplit > 1) reinterpret_cast<float2 *>(a.part + part_places(a, sh) * D)[where] = make_float2(ref, sum);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tc_dealloc(tmem, 512);
}

template <int NG>
cudaError_t launch_ng(const Kv4Attn &a, const Shape &sh, cudaStream_t stream, bool pdl) {
    static std::atomic<uint64_t> asked{0};          // devices (of the first 64) whose shared-memory limit has been raised
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev > 63 || !(asked.load(std::memory_order_acquire) >> dev & 1u))) {
        e = smem_at_least(reinterpret_cast<const void *>(k_kv4_attn_tc<NG>), (int)Sizes<NG>::all);
        if (e == cudaSuccess && dev <= 63) asked.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(sh.nsplit * sh.tiles, a.G, a.B); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = Sizes<NG>::all; cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = pdl ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k_kv4_attn_tc<NG>, a, sh);
}

}  // namespace

cudaError_t kv4_tc_launch(const Kv4Attn &a, uint32_t nsplit, uint32_t tiles, cudaStream_t stream, bool pdl) {
    const Shape sh{nsplit, tiles, kKv4TcRows, 0};
    switch (a.D / 32u) {
        case 1: return launch_ng<1>(a, sh, stream, pdl);
        case 2: return launch_ng<2>(a, sh, stream, pdl);
        case 3: return launch_ng<3>(a, sh, stream, pdl);
        default: return launch_ng<4>(a, sh, stream, pdl);
    }
}

}  // namespace nb
