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

struct Mx4Rows { uint8_t *codes, *scales; uint64_t code_stride, scale_stride; void *x; uint64_t x_stride; uint32_t type, rows, columns; };
cudaError_t mx4_quantize_launch(const Mx4Rows &a, cudaStream_t stream);
// codes and scales of type T_MX4 with zeros where a row's last group is filled up, to a.codes and a.scales
cudaError_t mx4_clean_launch(const Mx4Rows &a, const uint8_t *codes, uint64_t code_stride, const uint8_t *scales, uint64_t scale_stride, cudaStream_t stream);
cudaError_t mx4_read_launch(const Mx4Rows &a, cudaStream_t stream);

// x and w are codes here
struct Mx4Product {
    const uint8_t *x, *xs, *w, *ws; uint64_t x_stride, xs_stride, w_stride, ws_stride, w_expert, ws_expert;
    void *out; uint64_t out_stride; const int32_t *offsets;          // null: one matrix for all rows
    uint32_t out_type, rows, outputs, columns, experts;
};
// made: the kernel queued before this one made x and xs, and nothing else that this one reads
cudaError_t mx4_tc_launch(const Mx4Product &a, bool made, cudaStream_t stream);

}  // namespace nb
