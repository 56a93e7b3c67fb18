/*
 * Expert router in its general form, and its gradient (moe_route / route_kernel is the one fixed
 * DeepSeek-V3 router inside moe_forward; this one takes any expert count, score and grouping).
 *
 *   s      = softmax(logits) over the row, or sigmoid(logits) per expert
 *   pick   = s + bias (the bias chooses, it never weighs); -inf where the logit is -inf
 *   groups   E / n_group experts each, scored by their best pick or the sum of their two best; only the
 *            topk_group best groups stay (ties to the lower group)
 *   idx    = the top_k best picks, descending, ties to the lower expert; -1 where no expert is left
 *   w      = scale * s[idx], divided by (sum of the row's picked s + 1e-20) if renormalised; 0 for idx -1
 *
 * Without a bias the scores keep the logits' order, so experts are compared by their logits: those whose
 * scores round to the same 32-bit value are still told apart. Only sums of two scores (group_top2) need
 * exponentials for the choice then; groups whose sums round together go by their order.
 *
 * One warp per token, VPT = ceil(E / 32) neighbouring experts per lane in registers. The choice:
 *   1. each lane's best key; k rounds of (warp maximum, lanes holding it drop out) give a key that at
 *      least k experts reach, in k warp reductions and no index bookkeeping;
 *   2. the experts that reach it (k and a few more) go to shared memory, one per lane;
 *   3. each candidate counts the candidates before it; that rank is its place in the output.
 * More than 32 candidates (many equal scores, or the best ones side by side in a few lanes): k rounds of
 * arg-max over the warp instead, with the same result.
 *
 * Measured on a B200 (device time): 16384 tokens, 256 experts, sigmoid, bias, 8 groups, top 8: 14.4 us, 1.2 TB/s of
 * logits; 4.0 us for 4096 tokens without groups and bias; one token 3.1 us. Bound by instructions (771 per token and
 * 76% of the issue slots at 16384 tokens: profiles/route_experts_t16384.md), not by memory: the floor there is
 * 2.8 us. With ex2.approx for the choice it took 13.2 us, and neighbouring logits got one score.
 */
#pragma once
#include "moe_common.cuh"
#include "route.cuh"

#include <cuda_fp16.h>

namespace moe {

constexpr int RX_MAX_E = 1024;
constexpr int RX_MAX_K = 32;
constexpr int RX_MAX_GROUPS = 32;
constexpr int RX_WARPS = 8;   // tokens per block

struct RouteExpertsArgs {
  const void* logits;      // [T, E], rows `row_stride` elements apart
  long long row_stride;
  const float* bias;       // [E] or null
  int T, E, k;
  int n_group, topk_group;
  int group_top2;          // group score: 0 best pick, 1 sum of the two best
  int softmax;             // 1 softmax, 0 sigmoid
  int renormalize;
  float scale;
  int* idx;                // [T, k]
  float* w;                // [T, k]
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// VPT neighbouring values of a row from element `first` on, `fill` past E. `vec`: E == 32 * VPT and every
// lane's values start on a boundary of their own size (or of 16 bytes, if larger).
template <typename T, int VPT>
__device__ __forceinline__ void load_row(const T* row, int first, int E, bool vec, float fill, float (&v)[VPT]) {
  if (vec) {
    constexpr int BYTES = VPT * static_cast<int>(sizeof(T)) < 16 ? VPT * static_cast<int>(sizeof(T)) : 16;
    constexpr int PER = BYTES / static_cast<int>(sizeof(T));
#pragma unroll
    for (int c = 0; c < VPT / PER; ++c) {
      alignas(16) T tmp[PER];
      if constexpr (BYTES == 16)
        *reinterpret_cast<uint4*>(tmp) = __ldg(reinterpret_cast<const uint4*>(row + first) + c);
      else if constexpr (BYTES == 8)
        *reinterpret_cast<uint2*>(tmp) = __ldg(reinterpret_cast<const uint2*>(row + first) + c);
      else if constexpr (BYTES == 4)
        *reinterpret_cast<uint32_t*>(tmp) = __ldg(reinterpret_cast<const uint32_t*>(row + first) + c);
      else
        tmp[0] = row[first];
#pragma unroll
      for (int j = 0; j < PER; ++j) v[c * PER + j] = to_f32(tmp[j]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i) v[i] = first + i < E ? to_f32(row[first + i]) : fill;
  }
}

// Sigmoid of the choice, in 32 bits: expf (2 units of 2^-23 of its value at most), a sum and the hardware's 1/x (one
// unit); below 2^-126 it is 0. ex2.approx of x log2(e) in its place loses |x| / 8 units by rounding the product: at |x| = 12
// neighbouring float32 logits got one score.
__device__ __forceinline__ float sigmoid_choice(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.0f + expf(-x)));
  return y;
}

// Key of a pick: larger pick, larger key. x + 0 makes -0 and +0 equal and every NaN the positive one, the largest key:
// a NaN is chosen and its weight shows it.
__device__ __forceinline__ uint32_t pick_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u ^ (static_cast<uint32_t>(static_cast<int32_t>(u) >> 31) | 0x80000000u);
}
constexpr uint32_t RX_NONE = 0x007FFFFFu;       // the key of -inf: never chosen

__device__ __forceinline__ float key_value(uint32_t key) {
  return __uint_as_float((key & 0x80000000u) ? (key & 0x7FFFFFFFu) : ~key);
}

template <typename T, int VPT>
__global__ void __launch_bounds__(32 * RX_WARPS) route_experts_kernel(const __grid_constant__ RouteExpertsArgs p) {
  extern __shared__ uint32_t rx_dyn[];                    // per warp: E pick keys, n_group group keys (grouped only)
  __shared__ uint2 cand[RX_WARPS][32];                    // key, expert
  __shared__ float cand_x[RX_WARPS][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = static_cast<long long>(blockIdx.x) * RX_WARPS + warp;
  if (t >= p.T) return;
  const int first = lane * VPT;
  const T* row = static_cast<const T*>(p.logits) + t * p.row_stride;
  const bool vec = p.E == 32 * VPT && (reinterpret_cast<uintptr_t>(row) & 15u) == 0;
  float x[VPT];
  load_row<T, VPT>(row, first, p.E, vec, -INFINITY, x);

  // Softmax statistics of the row (the scores' scale; the choice may not need the scores).
  float mx = 0.0f, inv = 0.0f;
  if (p.softmax) {
    mx = x[0];
#pragma unroll
    for (int i = 1; i < VPT; ++i) mx = fmaxf(mx, x[i]);
    mx = warp_max(mx);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) sum += expf(x[i] - mx);
    inv = 1.0f / warp_sum(sum);
  }
  const bool grouped = p.n_group > 1;
  const bool by_logit = p.bias == nullptr && !(grouped && p.group_top2);

  uint32_t key[VPT];
  if (by_logit) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) key[i] = pick_key(x[i]);            // -inf past E
  } else {
    float b[VPT];
    if (p.bias != nullptr) {
      load_row<float, VPT>(p.bias, first, p.E, p.E == 32 * VPT && (reinterpret_cast<uintptr_t>(p.bias) & 15u) == 0, 0.0f, b);
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i) b[i] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const float v = __fadd_rn(p.softmax ? expf(x[i] - mx) * inv : sigmoid_choice(x[i]), b[i]);
      key[i] = x[i] == -INFINITY ? RX_NONE : pick_key(v);
    }
  }

  if (grouped) {
    const int per = p.E / p.n_group, lanes = per / VPT;               // lanes of a group, where it is made of whole lanes
    if (p.E == 32 * VPT && lanes >= 1 && (lanes & (lanes - 1)) == 0) {
      // Two best of the lane's keys, then of the group's lanes.
      uint32_t k1 = RX_NONE, k2 = RX_NONE;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        k2 = max(k2, min(k1, key[i]));
        k1 = max(k1, key[i]);
      }
      for (int o = 1; o < lanes; o <<= 1) {
        const uint32_t o1 = __shfl_xor_sync(0xffffffffu, k1, o), o2 = __shfl_xor_sync(0xffffffffu, k2, o);
        k2 = max(max(k2, o2), min(k1, o1));
        k1 = max(k1, o1);
      }
      const uint32_t mine = p.group_top2 ? pick_key(__fadd_rn(key_value(k1), key_value(k2))) : k1;
      // The group's lanes share the comparisons with the other groups.
      int rank = 0;
      const int own = lane & ~(lanes - 1);
      for (int o = (lane - own) * lanes; o < 32 + (lane - own) * lanes; o += lanes * lanes) {
        const uint32_t other = __shfl_sync(0xffffffffu, mine, o & 31);
        rank += o < 32 && (other > mine || (other == mine && o < own)) ? 1 : 0;
      }
      for (int o = 1; o < lanes; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
      if (rank >= p.topk_group) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) key[i] = RX_NONE;
      }
    } else {
      uint32_t* pk = rx_dyn + warp * (p.E + p.n_group);
      uint32_t* gs = pk + p.E;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (first + i < p.E) pk[first + i] = key[i];
      __syncwarp();
      uint32_t mine = RX_NONE;                            // key of group `lane`'s score
      bool drop = false;
      if (lane < p.n_group) {
        uint32_t k1 = RX_NONE, k2 = RX_NONE;
#pragma unroll 4
        for (int j = 0; j < per; ++j) {
          const uint32_t v = pk[lane * per + j];
          k2 = max(k2, min(k1, v));
          k1 = max(k1, v);
        }
        mine = p.group_top2 ? pick_key(__fadd_rn(key_value(k1), key_value(k2))) : k1;
        gs[lane] = mine;
      }
      __syncwarp();
      if (lane < p.n_group) {
        int rank = 0;
        for (int o = 0; o < p.n_group; ++o) {
          const uint32_t other = gs[o];
          rank += (other > mine || (other == mine && o < lane)) ? 1 : 0;
        }
        drop = rank >= p.topk_group;
      }
      const uint32_t dropped = __ballot_sync(0xffffffffu, drop);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (first + i < p.E && ((dropped >> ((first + i) / per)) & 1u)) key[i] = RX_NONE;
    }
  }

  // Without a bias the kept groups' experts are compared by their logits; the scores were for the groups' sums alone.
  if (p.bias == nullptr && !by_logit) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) key[i] = key[i] == RX_NONE ? RX_NONE : pick_key(x[i]);
  }

  // 1. A key that at least k experts reach (or all that are left).
  uint32_t best = key[0];
#pragma unroll
  for (int i = 1; i < VPT; ++i) best = max(best, key[i]);
  uint32_t left = best, floor_key = 0;
  for (int r = 0; r < p.k; ++r) {
    floor_key = __reduce_max_sync(0xffffffffu, left);
    if (left == floor_key) left = 0u;
  }
  floor_key = max(floor_key, RX_NONE + 1u);

  // 2. The experts that reach it, one per lane.
  int count = 0;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const bool in = key[i] >= floor_key;
    const uint32_t m = __ballot_sync(0xffffffffu, in);
    const int at = count + __popc(m & ((1u << lane) - 1u));
    if (in && at < 32) {
      cand[warp][at] = make_uint2(key[i], static_cast<uint32_t>(first + i));
      cand_x[warp][at] = x[i];
    }
    count += __popc(m);
  }
  __syncwarp();

  int place = p.k, my_idx = -1;
  float my_x = 0.0f;
  if (count <= 32) {
    // 3. Rank among the candidates.
    const uint2 mine = lane < count ? cand[warp][lane] : make_uint2(0u, RX_MAX_E);
    int rank = 0;
#pragma unroll 4
    for (int j = 0; j < count; ++j) {
      const uint2 o = cand[warp][j];
      rank += (o.x > mine.x || (o.x == mine.x && o.y < mine.y)) ? 1 : 0;
    }
    if (lane < count && rank < p.k) {
      place = rank;
      my_idx = static_cast<int>(mine.y);
      my_x = cand_x[warp][lane];
    }
    // Lanes past the candidates take the places that no expert fills.
    if (lane >= count && lane < p.k) place = lane;
  } else {
    for (int r = 0; r < p.k; ++r) {
      uint32_t bk = 0;
      int bi = 0;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (key[i] > bk) {
          bk = key[i];
          bi = i;
        }
      const uint32_t mk = __reduce_max_sync(0xffffffffu, bk);
      if (mk <= RX_NONE) {                              // none left
        if (lane == r) place = r;
        continue;
      }
      const int src = __ffs(__ballot_sync(0xffffffffu, bk == mk)) - 1;
      float xv = 0.0f;
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (lane == src && i == bi) {
          xv = x[i];
          key[i] = RX_NONE;
        }
      const int e = __shfl_sync(0xffffffffu, first + bi, src);
      xv = __shfl_sync(0xffffffffu, xv, src);
      if (lane == r) {
        place = r;
        my_idx = e;
        my_x = xv;
      }
    }
  }

  float s = 0.0f;
  if (my_idx >= 0) s = p.softmax ? expf(my_x - mx) * inv : 1.0f / (1.0f + expf(-my_x));
  if (p.renormalize) {
    s = s / (warp_sum(s) + 1e-20f);
  }
  if (place < p.k) {
    p.idx[t * p.k + place] = my_idx;
    p.w[t * p.k + place] = s * p.scale;
  }
}

struct RouteExpertsBwdArgs {
  const float* grad_w;     // [T, k]
  const void* logits;      // [T, E], rows `row_stride` elements apart
  long long row_stride;
  const int* idx;          // [T, k], distinct per row; outside [0, E): no expert
  int T, E, k;
  int softmax, renormalize;
  float scale;
  void* grad_logits;       // [T, E] contiguous, the logits' type
};

/*
 * Gradient of the weights. With g = scale * grad_w and D = sum of the picked s + 1e-20:
 *   ds_j = g_j                               without renormalisation,
 *   ds_j = (g_j - sum_i g_i s_i / D) / D     with it (0 for experts not picked);
 *   sigmoid: dl_e = ds_e s_e (1 - s_e), so only the picked logits are read;
 *   softmax: dl_e = s_e (ds_e - sum_i ds_i s_i). With renormalisation the sum is
 *            (sum g s / D) (1e-20 / D): the two terms that cancel are never formed.
 * The choice itself (idx) has no gradient, nor has the bias.
 *
 * A row is written twice where it was picked: first every expert's value without a pick, then the picks over it. That
 * needs no shared memory (which took as long). 6.8 us at 16384 x 256, sigmoid; the floor is 2.8 us, most of it the dense
 * output. Half of a warp's time is waiting for loads (the picks, then their logits) before its first store.
 */
template <typename T, int VPT>
__global__ void __launch_bounds__(32 * RX_WARPS) route_experts_backward_kernel(const __grid_constant__ RouteExpertsBwdArgs p) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t = static_cast<long long>(blockIdx.x) * RX_WARPS + warp;
  if (t >= p.T) return;
  const int first = lane * VPT;
  const T* row = static_cast<const T*>(p.logits) + t * p.row_stride;

  int e = -1;
  float g = 0.0f, l = 0.0f;
  if (lane < p.k) {
    e = p.idx[t * p.k + lane];
    if (e < 0 || e >= p.E) e = -1;
    if (e >= 0) {
      g = p.grad_w[t * p.k + lane] * p.scale;
      l = to_f32(row[e]);
    }
  }
  float x[VPT], mx = 0.0f, inv = 0.0f;
  if (p.softmax) {
    const bool vec = p.E == 32 * VPT && (reinterpret_cast<uintptr_t>(row) & 15u) == 0;
    load_row<T, VPT>(row, first, p.E, vec, -INFINITY, x);
    mx = x[0];
#pragma unroll
    for (int i = 1; i < VPT; ++i) mx = fmaxf(mx, x[i]);
    mx = warp_max(mx);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      x[i] = expf(x[i] - mx);
      sum += x[i];
    }
    inv = 1.0f / warp_sum(sum);
  }
  const float ex = expf(-fabsf(l)), r1 = 1.0f / (1.0f + ex);
  const float s = e < 0 ? 0.0f : p.softmax ? expf(l - mx) * inv : (l >= 0.0f ? r1 : ex * r1);
  const float gs = warp_sum(g * s);
  float d = g, dot = gs;
  if (p.renormalize) {
    const float D = warp_sum(s) + 1e-20f;
    d = __fdiv_rn(g - __fdiv_rn(gs, D), D);
    dot = __fdiv_rn(gs, D) * __fdiv_rn(1e-20f, D);
  }
  // Every expert's value without a pick, then the picks over them. A row without a pick has constant weights: zeros, also
  // where all its logits are -inf and the softmax is NaN.
  const bool dense = p.softmax && __any_sync(0xffffffffu, e >= 0);
  float o[VPT];
#pragma unroll
  for (int i = 0; i < VPT; ++i) o[i] = dense ? -(x[i] * inv) * dot : 0.0f;
  T* out = static_cast<T*>(p.grad_logits) + t * p.E;
  if (p.E == 32 * VPT && (reinterpret_cast<uintptr_t>(out) & 15u) == 0) {
    constexpr int BYTES = VPT * static_cast<int>(sizeof(T)) < 16 ? VPT * static_cast<int>(sizeof(T)) : 16;
    constexpr int PER = BYTES / static_cast<int>(sizeof(T));
#pragma unroll
    for (int c = 0; c < VPT / PER; ++c) {
      alignas(16) T tmp[PER];
#pragma unroll
      for (int j = 0; j < PER; ++j) tmp[j] = from_f32<T>(o[c * PER + j]);
      if constexpr (BYTES == 16)
        reinterpret_cast<uint4*>(out + first)[c] = *reinterpret_cast<uint4*>(tmp);
      else if constexpr (BYTES == 8)
        reinterpret_cast<uint2*>(out + first)[c] = *reinterpret_cast<uint2*>(tmp);
      else if constexpr (BYTES == 4)
        reinterpret_cast<uint32_t*>(out + first)[c] = *reinterpret_cast<uint32_t*>(tmp);
      else
        out[first] = tmp[0];
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (first + i < p.E) out[first + i] = from_f32<T>(o[i]);
  }
  __syncwarp();                                           // orders the two stores of a picked expert
  if (e >= 0) out[e] = from_f32<T>(p.softmax ? s * (d - dot) : d * (ex * r1 * r1));
}

// Experts per lane of the smallest instance that holds E experts.
inline int rx_vpt(int E) {
  int v = 1;
  while (32 * v < E) v *= 2;
  return v;
}

template <typename T>
inline void launch_route_experts_t(const RouteExpertsArgs& p, cudaStream_t st) {
  const unsigned grid = (static_cast<unsigned>(p.T) + RX_WARPS - 1) / RX_WARPS;
  // Shared keys only for groups that are not made of whole lanes.
  const int vpt = rx_vpt(p.E), lanes = p.E / p.n_group / vpt;
  const bool whole = p.E == 32 * vpt && lanes >= 1 && (lanes & (lanes - 1)) == 0;
  const size_t smem = p.n_group > 1 && !whole ? sizeof(float) * RX_WARPS * static_cast<size_t>(p.E + p.n_group) : 0;
  switch (rx_vpt(p.E)) {
    case 1: route_experts_kernel<T, 1><<<grid, 32 * RX_WARPS, smem, st>>>(p); break;
    case 2: route_experts_kernel<T, 2><<<grid, 32 * RX_WARPS, smem, st>>>(p); break;
    case 4: route_experts_kernel<T, 4><<<grid, 32 * RX_WARPS, smem, st>>>(p); break;
    case 8: route_experts_kernel<T, 8><<<grid, 32 * RX_WARPS, smem, st>>>(p); break;
    case 16: route_experts_kernel<T, 16><<<grid, 32 * RX_WARPS, smem, st>>>(p); break;
    default: route_experts_kernel<T, 32><<<grid, 32 * RX_WARPS, smem, st>>>(p); break;
  }
}

template <typename T>
inline void launch_route_experts_backward_t(const RouteExpertsBwdArgs& p, cudaStream_t st) {
  const unsigned grid = (static_cast<unsigned>(p.T) + RX_WARPS - 1) / RX_WARPS;
  switch (rx_vpt(p.E)) {
    case 1: route_experts_backward_kernel<T, 1><<<grid, 32 * RX_WARPS, 0, st>>>(p); break;
    case 2: route_experts_backward_kernel<T, 2><<<grid, 32 * RX_WARPS, 0, st>>>(p); break;
    case 4: route_experts_backward_kernel<T, 4><<<grid, 32 * RX_WARPS, 0, st>>>(p); break;
    case 8: route_experts_backward_kernel<T, 8><<<grid, 32 * RX_WARPS, 0, st>>>(p); break;
    case 16: route_experts_backward_kernel<T, 16><<<grid, 32 * RX_WARPS, 0, st>>>(p); break;
    default: route_experts_backward_kernel<T, 32><<<grid, 32 * RX_WARPS, 0, st>>>(p); break;
  }
}

}  // namespace moe
