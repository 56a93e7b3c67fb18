/*
 * Products with 4-bit weights: linear_w4 (y = x . W^T) and experts_w4 (the routed experts' two
 * products with SwiGLU between them, summed with the routing weights).
 *
 *   W[n, k] = scale[n, k / group] * (code[n, k] - zero[n, k / group])      zero: 8 where none is given
 *
 * codes: two per byte, the even column in the low nibble, rows of ceil(K / 2) bytes. scale has the
 * activations' type, zero is a byte of which the low four bits count; both [N, ceil(K / group)].
 */
#pragma once
#include "experts_route.cuh"
#include "moe_common.cuh"

namespace moe {

struct W4Matrix {
  const uint8_t* codes;   // [rows, pitch bytes]
  const void* scale;      // [rows, groups]
  const uint8_t* zero;    // [rows, groups] or null
  int group;              // 32, 64 or 128 columns per scale
};

struct ExpertsW4Args {
  const void* x;          // [T, H], rows x_stride elements apart
  long long x_stride;
  const int* idx;         // [T, k] global experts; outside [offset, offset + E): not on this GPU
  const float* wt;        // [T, k]
  W4Matrix w13;           // [E, 2 I, H]: rows [0, I) multiply silu of rows [I, 2 I)
  W4Matrix w2;            // [E, H, I]
  int T, k, E, offset, H, I;
};

}  // namespace moe
