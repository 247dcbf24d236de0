// kv4.h -- a paged key/value cache held in 4 bits: its layout, and the launchers that write it, read it back and attend to it (kv4.cu).
//
// A pool is [pages][kv heads][block]; a block holds the keys and values of one head's 32 tokens, D coordinates each, n = D / 32 groups:
//     key codes [32][16 n] | key pairs [32][n] of two fp16 | value codes [32][16 n] | value pairs [32][n]          1280 n bytes, 5 bits a coordinate
// A group is 32 neighbouring coordinates x of one token: 4-bit codes c and the pair (s, m), m = f16(min x), s = f16((max x - min x) f32(1/15)),
// c = clamp(round_half_even((x - m) / s), 0, 15); it stands for c s + m.  A group with a coordinate that is no number or beyond +-32768 stands for NaN.
// Where coordinates lie is chosen for the matrix instructions' operands, so that a thread of k_kv4_attn finds what it multiplies side by side:
// coordinate 32 j + 8 b + i of a key is nibble i of the 32-bit word b n + j of its codes, coordinate 32 j + 4 b + i of a value nibble i of the 16-bit word b n + j.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "ops.h"

namespace nb {

constexpr uint32_t kKv4Page = 32, kKv4Group = 32;
__host__ __device__ constexpr uint32_t kv4_block_bytes(uint32_t D) { return 1280u * (D / kKv4Group); }
// head sizes that have an attention kernel (writing and reading take any multiple of 32 up to 256)
inline bool kv4_dim_ok(uint32_t D) { return D == 32 || D == 64 || D == 96 || D == 128 || D == 256; }

// rows of keys and values: token t, head g: D numbers of `type` at k + t * k_token + g * k_head (elements).  Token t goes to (or comes from) place slots[t] =
// page * 32 + place in the page; a slot outside the pool is skipped (read: zeros).  Without slots: token t is position pos0 + *pos_ptr + t of `table`.
struct Kv4Rows {
    void *k, *v; uint64_t k_token, v_token, k_head, v_head; uint32_t type;
    const int32_t *slots; const uint32_t *table; uint32_t pos0; const uint32_t *pos_ptr;
    uint32_t T, G, D; unsigned char *pool; uint64_t page_stride; uint32_t n_pages;
};
cudaError_t kv4_write_launch(const Kv4Rows &a, cudaStream_t stream, bool pdl);
cudaError_t kv4_read_launch(const Kv4Rows &a, cudaStream_t stream);

// out[b][t][h] = sum_j p_j v_j over the keys j that query t of sequence b sees, p the softmax of softcap tanh(scale q . k_j / softcap) (softcap 0: of scale q . k_j);
// head h reads the keys of head h / (H / G).  Query t sits at position lens[b] - T + t and sees the keys up to its own, of these only those less than `window`
// positions back (0: all) and those in its own block of `block` positions (0: all); one whose position is negative, or that sees none, has zeros.  sink[h] (optional)
// joins the denominator as exp(sink_h).  gate (optional): the output of (t, h) is multiplied by sigmoid(gate[t * ldg + h]).
struct Kv4Attn {
    const void *q; uint64_t q_batch, q_token, q_head; uint32_t type;          // elements; type of q and out: fp32 or bf16
    void *out; uint64_t o_batch, o_token, o_head;
    const unsigned char *pool; uint64_t page_stride; uint32_t n_pages;
    const int32_t *table; uint64_t table_stride; uint32_t width;               // [B][width] page numbers
    const int32_t *lens; uint32_t pos0; const uint32_t *pos_ptr;               // without lens: every sequence holds pos0 + *pos_ptr + T tokens
    uint32_t B, T, H, G, D; float scale, softcap; const float *sink; uint32_t window, block;
    const float *gate; uint32_t ldg;
    float *part;                                                               // kv4_attn_workspace bytes
    uint32_t *err;                                                             // optional: receives a code where a wait inside a kernel ran out (its rows are NaN either way)
};
size_t kv4_attn_workspace(uint32_t B, uint32_t T, uint32_t H, uint32_t G, uint32_t D, uint32_t width, uint32_t window, uint32_t block, uint32_t sms);
// the most that any call of B sequences asks for, whatever its tokens and its width
size_t kv4_attn_workspace_most(uint32_t B, uint32_t D, uint32_t sms);
// one launch, or two (the keys of a row split over several blocks, then joined); *launches says how many.  pdl, pdl_join: whether the first and the second may be launched while the
// kernel before them runs
cudaError_t kv4_attn_launch(const Kv4Attn &a, uint32_t sms, cudaStream_t stream, bool pdl, bool pdl_join, uint32_t *launches);

}  // namespace nb
