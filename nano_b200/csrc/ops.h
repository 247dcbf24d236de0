// ops.h -- operators on device memory that the engine and the C-ABI share (ops.cu, kv4.cu).  Launchers queue their kernels on `stream` of the current device,
// allocate nothing and wait for nothing; they return what the launch returned.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace nb {

// element types of operands (NB200_T_* of the C-ABI)
enum ElemType : uint32_t { T_F32 = 0, T_BF16 = 1, T_F16 = 2 };
inline uint32_t elem_size(uint32_t type) { return type == T_F32 ? 4u : 2u; }

constexpr uint32_t kTopMax = 32;          // alternatives of a row: one lane of a warp holds each

// one row of logits per token: row r starts at logits + r * row_stride (elements)
struct LogprobArgs {
    const void *logits; uint64_t row_stride; uint32_t type, rows, vocab;
    const void *tokens; uint32_t token_bytes;          // null: no token is asked for
    uint32_t top; float *logprob, *entropy, *top_logprob; int32_t *top_id;          // [rows], [rows], [rows][top], [rows][top]; each may be null
};
cudaError_t logprobs_launch(const LogprobArgs &a, cudaStream_t stream);

// pages of several pools: page p of pool i is the page_bytes[i] bytes at pool[i] + p * page_stride[i]
struct PagePool { void *base; uint64_t page_bytes, page_stride; };
// copies page src[i] over page dst[i] in every pool.  No destination may be a source or appear twice (the caller has checked); launches of up to
// kPagePairs pairs and kPagePools pools
constexpr uint32_t kPagePairs = 1024, kPagePools = 32;
cudaError_t pages_copy_launch(const PagePool *pools, uint32_t n_pools, const uint32_t *src, const uint32_t *dst, uint32_t n, cudaStream_t stream, uint32_t *launches);

}  // namespace nb
