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

// x[0..K) . W[row], one warp; every lane returns the sum. Sums in 32 bits.
template <typename T, typename X>
__device__ __forceinline__ float w4_dot(const X* x, const W4Matrix& w, long long row, int K) {
  const int lane = threadIdx.x & 31;
  const int bytes = (K + 1) / 2, groups = (K + w.group - 1) / w.group;
  const uint8_t* c = w.codes + row * bytes;
  const T* sc = static_cast<const T*>(w.scale) + row * groups;
  const uint8_t* zp = w.zero ? w.zero + row * groups : nullptr;
  float acc = 0.0f;
  for (int b = lane; b < bytes; b += 32) {
    const int k = 2 * b, g = k / w.group;
    const float z = zp ? static_cast<float>(zp[g] & 15) : 8.0f;
    const int q = c[b];
    float part = to_f32(x[k]) * (static_cast<float>(q & 15) - z);
    if (k + 1 < K) part = fmaf(to_f32(x[k + 1]), static_cast<float>(q >> 4) - z, part);
    acc = fmaf(to_f32(sc[g]), part, acc);
  }
  return warp_sum(acc);
}

template <typename T>
__global__ void __launch_bounds__(256) linear_w4_kernel(const T* x, long long x_stride, W4Matrix w, int M, int N, int K, T* out) {
  const long long i = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (i >= static_cast<long long>(M) * N) return;
  const long long m = i / N, n = i % N;
  const float y = w4_dot<T>(x + m * x_stride, w, n, K);
  if ((threadIdx.x & 31) == 0) out[m * N + n] = from_f32<T>(y);
}

struct ExpertsW4Args {
  const void* x;          // [T, H], rows x_stride elements apart
  long long x_stride;
  const int* idx;         // [T, k] global experts; outside [offset, offset + E): not on this GPU
  const float* wt;        // [T, k]
  W4Matrix w13;           // [E, 2 I, H]: rows [0, I) multiply silu of rows [I, 2 I)
  W4Matrix w2;            // [E, H, I]
  int T, k, E, offset, H, I;
};

template <typename T>
__global__ void __launch_bounds__(256) experts_w4_up_kernel(const __grid_constant__ ExpertsW4Args p, float* h) {
  const long long i = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (i >= static_cast<long long>(p.T) * p.k * p.I) return;
  const long long r = i / p.I, c = i % p.I;
  const int e = p.idx[r] - p.offset;
  if (e < 0 || e >= p.E) return;
  const T* x = static_cast<const T*>(p.x) + r / p.k * p.x_stride;
  const float u1 = w4_dot<T>(x, p.w13, static_cast<long long>(e) * 2 * p.I + c, p.H);
  const float u2 = w4_dot<T>(x, p.w13, static_cast<long long>(e) * 2 * p.I + p.I + c, p.H);
  if ((threadIdx.x & 31) == 0) h[i] = u1 * (u2 / (1.0f + expf(-u2)));
}

template <typename T>
__global__ void __launch_bounds__(256) experts_w4_down_kernel(const __grid_constant__ ExpertsW4Args p, const float* h, T* out) {
  const long long i = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  if (i >= static_cast<long long>(p.T) * p.H) return;
  const long long t = i / p.H, n = i % p.H;
  float acc = 0.0f;
  for (int j = 0; j < p.k; ++j) {
    const long long r = t * p.k + j;
    const int e = p.idx[r] - p.offset;
    if (e < 0 || e >= p.E) continue;
    acc = fmaf(p.wt[r], w4_dot<T>(h + r * p.I, p.w2, static_cast<long long>(e) * p.H + n, p.I), acc);
  }
  if ((threadIdx.x & 31) == 0) out[i] = from_f32<T>(acc);
}

}  // namespace moe
