// mx4.h -- rows in microscaled 4-bit floating point, and their products (mx4.cu, mx4_tc.cu).
//
// A group of 32 neighbours of a row: one byte E, the scale 2^(E - 127) (255: NaN), and 32 codes c of four bits, sign and e2m1 number v(c) in {0, .5, 1, 1.5, 2, 3, 4, 6}.  Code j of a group is
// nibble j % 2 (from the lowest) of byte j / 2.  Products of two such groups:  2^(E_x + E_w - 254) sum v(c_x) v(c_w),  where the sum is a whole multiple of 1/4 below 2^11: exact in fp32.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "ops.h"

namespace nb {

constexpr uint32_t T_MX4 = 3, kMx4Group = 32;
inline uint32_t mx4_groups(uint32_t columns) { return columns / kMx4Group + (columns % kMx4Group != 0); }

// Scales lie row after row (stride bytes apart, sixteen every 16 bytes), or sixteen of every row after the other (16 bytes from row to row, `step` to the next sixteen), which neighbouring threads
// read as neighbours: scale g of row r is byte r stride + (g / 16) step + g % 16
struct Mx4Rows { uint8_t *codes, *scales; uint64_t code_stride, scale_stride, scale_step; void *x; uint64_t x_stride; uint32_t type, rows, columns; };
cudaError_t mx4_quantize_launch(const Mx4Rows &a, cudaStream_t stream);
cudaError_t mx4_read_launch(const Mx4Rows &a, cudaStream_t stream);

// How a product is run: by sizes, types and alignment alone
struct Mx4Plan {
    uint32_t tn, ks, per, pairs;          // rows of X in a tile; blocks that share a tile's depth (0: the kernel for many tiles); steps to each; tiles of rows, over all experts at most
    bool raw;          // the product reads numbers and quantises them itself: nothing is made before it
    bool x_codes, x_scales, w_scales, x_second;          // what a kernel makes before: codes of x, its scales (in the second order?) and those of w in the second order
    uint64_t x_scales_at, w_scales_at, bytes;          // in the workspace; codes come first
};
struct Mx4Product {
    const void *x; const uint8_t *xs, *w, *ws; uint64_t x_stride, xs_stride, w_stride, ws_stride, w_expert, ws_expert;
    void *out; uint64_t out_stride; const int32_t *offsets;          // null: one matrix for all rows
    uint32_t x_type, out_type, rows, outputs, columns, experts;
};
Mx4Plan mx4_plan(const Mx4Product &p);
// the kernel before: to the workspace, what the plan names
cudaError_t mx4_prepare_launch(const Mx4Product &p, const Mx4Plan &plan, uint8_t *workspace, cudaStream_t stream);
// the product, of codes; steps: bytes from sixteen scales to the next.  made: the kernel queued before this one made x, its scales and w's, and nothing else that this one reads
cudaError_t mx4_tc_launch(const Mx4Product &p, const Mx4Plan &plan, uint64_t xs_step, uint64_t ws_step, bool made, cudaStream_t stream);

}  // namespace nb
