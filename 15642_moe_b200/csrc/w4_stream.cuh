/*
 * Products with 4-bit weights for up to 8 tokens: the weights are read once, straight from global memory
 * into matrix fragments, and that read is all the time there is (6.45 TB/s measured).
 *
 *   mma m16n8k16: A = 16 weight rows x 16 columns, B = 16 columns x 8 tokens, fp32 accumulators.
 *
 * A thread holds, of rows g and g + 8 of a tile, the four codes at each of two places; which columns those
 * are is free as long as A and B agree. So thread t of a row's four takes g/4 neighbouring columns of each
 * group of g (one 16-, 8- or 4-byte load), a 32-bit word of 8 codes makes the fragments of two mma, and the
 * activations are put into shared memory in that order once per block. Codes become numbers by placing a
 * nibble in the mantissa of 128 (bf16) or 1024 (f16) and subtracting 128 + zero: exact, as is every product.
 * Each group's sum is scaled in fp32: no weight is ever rounded.
 *
 * Split: a block has 8 warps, 4 tiles of 16 rows x 2 column halves; a cluster of up to 8 blocks shares the
 * same rows and splits the columns (for the experts' second product: the active experts and their columns),
 * and adds its parts through distributed shared memory in rank order, so results repeat bit for bit.
 * Each warp keeps 4 steps of 128 columns in flight (4 KB).
 */
#pragma once
#include "gate.cuh"
#include "w4.cuh"

#include <type_traits>

namespace moe {

constexpr int WS_WARPS = 8, WS_THREADS = 32 * WS_WARPS;
constexpr int WS_WK = 2;                        // column halves per block
constexpr int WS_ROWS = 16 * WS_WARPS / WS_WK;  // 64 weight rows per block
constexpr int WS_TOK = 8;                       // tokens per mma
constexpr int WS_STEP = 128;                    // columns per step
constexpr int WS_CHUNK = 16;                    // steps staged at a time
constexpr int WS_DEPTH = 4;                     // steps in flight per warp
constexpr int WS_MAX_PICKS = WS_TOK * RX_MAX_K; // 256

enum { WS_LINEAR = 0, WS_UP = 1, WS_DOWN = 2 };

struct StreamArgs {
  const void* x;           // [M, K] (linear, up)
  long long x_stride;
  W4Matrix w;
  int M, N, K;             // tokens (<= 8); output columns (up: I); reduction length
  int cluster;             // blocks per cluster: gridDim.x = row tiles * cluster
  int parts, spp;          // the K steps of one matrix in `parts` parts of `spp` steps (down: parts at least)
  const int* idx;          // [M, k] (up, down)
  const float* wt;         // [M, k] (down)
  int k, E, offset;
  float* h;                // [M * k, M, I]: entry (r, t) is token t through the expert first picked at r
  void* out;               // [M, N] (linear, down)
};

// mma with bf16 or f16 operands: d += a x b.
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Pair i of a word's codes (columns i and i + 4) as two numbers minus `off` (128 + zero or 1024 + zero, twice).
template <typename T>
__device__ __forceinline__ uint32_t w4_pair(uint32_t word, int i, uint32_t off) {
  constexpr bool F16 = std::is_same_v<T, __half>;
  uint32_t v;
  asm("lop3.b32 %0, %1, 0x000f000f, %2, 0xea;" : "=r"(v) : "r"(word >> (4 * i)), "n"(F16 ? 0x64006400 : 0x43004300));
  if constexpr (F16) {
    const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&v), *reinterpret_cast<const __half2*>(&off));
    return *reinterpret_cast<const uint32_t*>(&d);
  } else {
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&off));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
}
// `off` for a zero point: both halves of 128 + z in bf16 (z < 16: exact) or 1024 + z in f16.
template <typename T>
__device__ __forceinline__ uint32_t w4_offset(int zero) {
  const uint32_t one = (std::is_same_v<T, __half> ? 0x6400u : 0x4300u) + static_cast<uint32_t>(zero);
  return one | (one << 16);
}

// 32 bits at any byte address; bytes at or past `left` are not read (only aligned words that hold a wanted byte).
__device__ __forceinline__ uint32_t ld_u32_any(const uint8_t* p, int left) {
  if (left <= 0) return 0u;
  const uintptr_t a = reinterpret_cast<uintptr_t>(p);
  const uint32_t* w = reinterpret_cast<const uint32_t*>(a & ~static_cast<uintptr_t>(3));
  const int sh = static_cast<int>(a & 3);
  const uint32_t lo = __ldg(w);
  const uint32_t hi = sh + min(left, 4) > 4 ? __ldg(w + 1) : 0u;
  return __funnelshift_r(lo, hi, 8 * sh);
}

__device__ __forceinline__ uint4 ld_stream_v4(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// The four words of one step that thread t of a row's four holds. G4 = group / 32 words per group.
// Word i of the step: columns (i / G4) * group + t * group / 4 + (i % G4) * 8 .. + 8.
template <int G4, bool ALIGNED>
__device__ __forceinline__ uint4 ld_codes(const uint8_t* row, int step, int t, int pitch) {
  const int base = step * (WS_STEP / 2);
  uint32_t v[4] = {0u, 0u, 0u, 0u};
  if constexpr (ALIGNED) {
#pragma unroll
    for (int s = 0; s < 4 / G4; ++s) {
      const int o = base + s * (16 * G4) + t * (4 * G4);
      if (o < pitch) {
        if constexpr (G4 == 4) {
          return ld_stream_v4(row + o);
        } else if constexpr (G4 == 2) {
          const uint2 u = __ldg(reinterpret_cast<const uint2*>(row + o));
          v[2 * s] = u.x;
          v[2 * s + 1] = u.y;
        } else {
          v[s] = __ldg(reinterpret_cast<const uint32_t*>(row + o));
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int o = base + (i / G4) * (16 * G4) + t * (4 * G4) + (i % G4) * 4;
      v[i] = ld_u32_any(row + o, pitch - o);
    }
  }
  return make_uint4(v[0], v[1], v[2], v[3]);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(T a, T b) {
  return static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&a)) |
         (static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(&b)) << 16);
}

// 8 neighbouring activations from column k on (0 past K) as the pairs (0,4), (1,5), (2,6), (3,7).
template <typename T>
__device__ __forceinline__ uint4 ld_x_pairs(const T* row, int k, int K, bool vec) {
  if (vec && k + 8 <= K) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(row + k));
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                      __byte_perm(v.y, v.w, 0x7632));
  }
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = k + i < K ? row[k + i] : from_f32<T>(0.0f);
  return make_uint4(pack2(e[0], e[4]), pack2(e[1], e[5]), pack2(e[2], e[6]), pack2(e[3], e[7]));
}

// The same for 8 fp32 values, as two bf16 terms (hi + lo carry 16 bits).
__device__ __forceinline__ void ld_h_pairs(const float* row, int k, int K, uint4& hi, uint4& lo) {
  float v[8];
  if (k + 8 <= K && (reinterpret_cast<uintptr_t>(row + k) & 15u) == 0) {
    const float4 a = *reinterpret_cast<const float4*>(row + k), b = *reinterpret_cast<const float4*>(row + k + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = k + i < K ? row[k + i] : 0.0f;
  }
  uint32_t h[4], l[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    h[i] = pack_bf16x2(v[i], v[i + 4]);
    const float r0 = v[i] - __uint_as_float(h[i] << 16), r1 = v[i + 4] - __uint_as_float(h[i] & 0xFFFF0000u);
    // A value past bf16's range (or NaN) has no remainder.
    l[i] = pack_bf16x2(fabsf(r0) <= 3.4e38f ? r0 : 0.0f, fabsf(r1) <= 3.4e38f ? r1 : 0.0f);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// Shared memory of one block, in bytes: activations of a chunk, then scales and offsets of its groups.
inline size_t ws_smem(int mode, int M, int chunk_steps, int group) {
  return static_cast<size_t>(chunk_steps) * 16 * M * 16 * (mode == WS_DOWN ? 2 : 1) +
         static_cast<size_t>(WS_ROWS) * (chunk_steps * (WS_STEP / group) + 1) * 8;
}

template <typename T, int G4, int MODE, bool ALIGNED>
__global__ void __launch_bounds__(WS_THREADS, 3) w4_stream_kernel(const __grid_constant__ StreamArgs p) {
  using W = typename std::conditional<MODE == WS_DOWN, __nv_bfloat16, T>::type;   // type of the fragments
  constexpr int NB = MODE == WS_DOWN ? 2 : 1;
  constexpr int GPS = 4 / G4;                    // groups per step
  extern __shared__ __align__(16) uint8_t ws_dyn[];
  __shared__ float red[WS_WK][WS_ROWS][WS_TOK];
  __shared__ int s_idx[MODE == WS_LINEAR ? 1 : WS_MAX_PICKS];
  __shared__ int s_act[MODE == WS_DOWN ? WS_MAX_PICKS : 1];
  __shared__ uint32_t s_mask[WS_WARPS];
  __shared__ float s_wt[WS_TOK];
  __shared__ int s_routed;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int wr = warp / WS_WK, wk = warp % WS_WK;
  const int S = p.cluster, rank = static_cast<int>(blockIdx.x) % S;
  const int tile = static_cast<int>(blockIdx.x) / S, slot = blockIdx.y;
  const int pitch = (p.K + 1) / 2, steps = (p.K + WS_STEP - 1) / WS_STEP;
  const int groups = (p.K + p.w.group - 1) / p.w.group;
  const int picks = p.M * p.k;

  // Which experts: `up` has one block (cluster) per pick, those whose expert an earlier pick has end here;
  // `down` walks the list of the picks' distinct experts.
  int expert = 0, n_act = 1, parts = p.parts, spp = p.spp;
  if constexpr (MODE == WS_UP) {
    for (int r = tid; r < picks; r += WS_THREADS) s_idx[r] = p.idx[r];
    if (tid == 0) s_routed = 0;
    __syncthreads();
    expert = s_idx[slot] - p.offset;
    bool skip = expert < 0 || expert >= p.E;
    if (tid < slot && s_idx[tid] == s_idx[slot]) skip = true;
    if (tid < picks && s_idx[tid] == s_idx[slot]) atomicOr(&s_routed, 1 << (tid / p.k));
    if (__syncthreads_or(skip)) {
      allow_dependent_launch();
      return;
    }
    allow_dependent_launch();
  }
  if constexpr (MODE == WS_DOWN) {
    if (tid < picks) s_idx[tid] = p.idx[tid];
    __syncthreads();
    bool first = false;
    if (tid < picks) {
      const int e = s_idx[tid] - p.offset;
      first = e >= 0 && e < p.E;
      for (int r = 0; r < tid; ++r)
        if (s_idx[r] == s_idx[tid]) first = false;
    }
    const uint32_t m = __ballot_sync(0xffffffffu, first);
    if (lane == 0) s_mask[warp] = m;
    __syncthreads();
    int at = __popc(m & ((1u << lane) - 1u));
    n_act = 0;
#pragma unroll
    for (int i = 0; i < WS_WARPS; ++i) {
      if (i < warp) at += __popc(s_mask[i]);
      n_act += __popc(s_mask[i]);
    }
    if (first) s_act[at] = tid;
    __syncthreads();
    // Few active experts: cut their columns so that every block of the cluster has a part.
    if (n_act > 0 && n_act * parts < S) {
      parts = min(steps, (S + n_act - 1) / n_act);
      spp = (steps + parts - 1) / parts;
      parts = (steps + spp - 1) / spp;
    }
  }

  uint8_t* xs = ws_dyn;
  const int x_units = spp * 16 * p.M;
  float* sc = reinterpret_cast<float*>(ws_dyn + static_cast<size_t>(p.spp) * 16 * p.M * 16 * NB);
  const int sc_pitch = p.spp * GPS + 1;
  uint32_t* zo = reinterpret_cast<uint32_t*>(sc + WS_ROWS * sc_pitch);

  // Weight rows of this thread: g and g + 8 of the warp's tile; `up` puts column i of X1 and of X2 there.
  const int r0 = wr * 16 + g;
  auto matrix_row = [&](int local) -> long long {   // local row 0..63 of the block -> row of the matrix, clamped
    if constexpr (MODE == WS_UP) {
      const int i = min(tile * (WS_ROWS / 2) + (local >> 4) * 8 + (local & 7), p.N - 1);
      return (local & 8) ? static_cast<long long>(p.N) + i : i;
    } else {
      return min(tile * WS_ROWS + local, p.N - 1);
    }
  };
  const int rows_per = MODE == WS_UP ? 2 * p.N : p.N;
  const long long mr0 = matrix_row(r0), mr1 = matrix_row(r0 + 8);

  float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  const int items = n_act * parts;
  bool waited = false;
  for (int item = rank; item < items; item += S) {
    const int part = item % parts;
    int pick = 0;
    if constexpr (MODE == WS_DOWN) {
      pick = s_act[item / parts];
      expert = s_idx[pick] - p.offset;
    }
    const int s_begin = part * spp, s_end = min(steps, s_begin + spp);
    const int half = (s_end - s_begin + WS_WK - 1) / WS_WK;
    const int a = s_begin + wk * half, b = min(s_end, a + half), n = b - a;
    const long long first_row = static_cast<long long>(expert) * rows_per;
    const uint8_t* c0 = p.w.codes + (first_row + mr0) * pitch;
    const uint8_t* c1 = p.w.codes + (first_row + mr1) * pitch;
    uint4 buf[WS_DEPTH][2];
#pragma unroll
    for (int d = 0; d < WS_DEPTH; ++d)
      if (d < n) {
        buf[d][0] = ld_codes<G4, ALIGNED>(c0, a + d, t, pitch);
        buf[d][1] = ld_codes<G4, ALIGNED>(c1, a + d, t, pitch);
      }
    __syncthreads();                              // the last item's shared memory is free
    // Scales and offsets of the block's rows.
    const int g_begin = s_begin * GPS, g_count = min(groups, s_end * GPS) - g_begin;
    for (int i = tid; i < WS_ROWS * g_count; i += WS_THREADS) {
      const int local = i / g_count, q = i % g_count;
      const long long at = (first_row + matrix_row(local)) * groups + g_begin + q;
      sc[local * sc_pitch + q] = to_f32(static_cast<const T*>(p.w.scale)[at]);
      zo[local * sc_pitch + q] = w4_offset<W>(p.w.zero ? p.w.zero[at] & 15 : 8);
    }
    // Activations in fragment order: unit ((step, word, token), t) of 16 bytes.
    const int units = (s_end - s_begin) * 16;
    if constexpr (MODE == WS_DOWN) {
      if (tid < WS_TOK) {
        float w = 0.0f;
        if (tid < p.M)
          for (int j = 0; j < p.k; ++j)
            if (s_idx[tid * p.k + j] == s_idx[pick]) w += p.wt[tid * p.k + j];
        s_wt[tid] = w;
      }
      if (tid == 0) {
        int routed = 0;
        for (int r = 0; r < picks; ++r)
          if (s_idx[r] == s_idx[pick]) routed |= 1 << (r / p.k);
        s_routed = routed;
      }
      if (!waited) {
        wait_prerequisite_grids();                // h comes from the kernel before
        waited = true;
      }
      __syncthreads();
    }
    for (int i = tid; i < units * p.M; i += WS_THREADS) {
      const int tok = i / units, q = i % units;
      const int st = q >> 4, c8 = q & 15;         // 8-column piece c8 of step st
      const int sub = c8 / (4 * G4), in = c8 % (4 * G4), tt = in / G4, word = sub * G4 + in % G4;
      const int k = (s_begin + st) * WS_STEP + c8 * 8;
      const int unit = ((st * 4 + word) * p.M + tok) * 4 + tt;
      if constexpr (MODE == WS_DOWN) {
        uint4 hi = make_uint4(0, 0, 0, 0), lo = hi;
        if ((s_routed >> tok) & 1)
          ld_h_pairs(p.h + (static_cast<long long>(pick) * p.M + tok) * p.K, k, p.K, hi, lo);
        reinterpret_cast<uint4*>(xs)[unit] = hi;
        reinterpret_cast<uint4*>(xs)[x_units + unit] = lo;
      } else {
        const T* row = static_cast<const T*>(p.x) + tok * p.x_stride;
        reinterpret_cast<uint4*>(xs)[unit] = ld_x_pairs<T>(row, k, p.K, (reinterpret_cast<uintptr_t>(row) & 15u) == 0);
      }
    }
    __syncthreads();

    float part_sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto step = [&](const uint4 (&w)[2], int s) {
      const uint32_t u0[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, u1[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
      const int ls = s - s_begin;
      const int q0 = min(ls * GPS, g_count - 1);
#pragma unroll
      for (int gq = 0; gq < GPS; ++gq) {
        const int q = GPS == 1 ? q0 : min(ls * GPS + gq, g_count - 1);
        const uint32_t o0 = zo[r0 * sc_pitch + q], o1 = zo[(r0 + 8) * sc_pitch + q];
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = gq * G4; i < (gq + 1) * G4; ++i) {
          const uint32_t p0 = w4_pair<W>(u0[i], 0, o0), p1 = w4_pair<W>(u0[i], 1, o0), p2 = w4_pair<W>(u0[i], 2, o0),
                         p3 = w4_pair<W>(u0[i], 3, o0);
          const uint32_t q0_ = w4_pair<W>(u1[i], 0, o1), q1_ = w4_pair<W>(u1[i], 1, o1), q2_ = w4_pair<W>(u1[i], 2, o1),
                         q3_ = w4_pair<W>(u1[i], 3, o1);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            uint4 x = make_uint4(0, 0, 0, 0);
            if (g < p.M) x = reinterpret_cast<const uint4*>(xs)[nb * x_units + ((ls * 4 + i) * p.M + g) * 4 + t];
            mma16816<W>(acc, p0, q0_, p1, q1_, x.x, x.y);
            mma16816<W>(acc, p2, q2_, p3, q3_, x.z, x.w);
          }
        }
        const float f0 = sc[r0 * sc_pitch + q], f1 = sc[(r0 + 8) * sc_pitch + q];
        part_sum[0] = fmaf(f0, acc[0], part_sum[0]);
        part_sum[1] = fmaf(f0, acc[1], part_sum[1]);
        part_sum[2] = fmaf(f1, acc[2], part_sum[2]);
        part_sum[3] = fmaf(f1, acc[3], part_sum[3]);
      }
    };
    for (int s = 0; s < n; s += WS_DEPTH) {
#pragma unroll
      for (int d = 0; d < WS_DEPTH; ++d)
        if (s + d < n) {
          step(buf[d], a + s + d);
          if (s + d + WS_DEPTH < n) {
            buf[d][0] = ld_codes<G4, ALIGNED>(c0, a + s + d + WS_DEPTH, t, pitch);
            buf[d][1] = ld_codes<G4, ALIGNED>(c1, a + s + d + WS_DEPTH, t, pitch);
          }
        }
    }
    if constexpr (MODE == WS_DOWN) {
      // Weighted sum over the experts; a token that did not pick this one takes nothing, not even 0 * NaN.
      const int routed = s_routed;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int tok = 2 * t + (c & 1);
        if ((routed >> tok) & 1) total[c] = fmaf(s_wt[tok], part_sum[c], total[c]);
      }
    } else {
#pragma unroll
      for (int c = 0; c < 4; ++c) total[c] += part_sum[c];
    }
  }

  if constexpr (MODE == WS_DOWN)
    if (!waited) wait_prerequisite_grids();       // this grid ends after the one before it, with items or without

  // Sum of the cluster's parts, in rank and half order.
  red[wk][r0][2 * t] = total[0];
  red[wk][r0][2 * t + 1] = total[1];
  red[wk][r0 + 8][2 * t] = total[2];
  red[wk][r0 + 8][2 * t + 1] = total[3];
  if (S > 1) cluster_sync_all(); else __syncthreads();
  const uint32_t red_at = smem_u32(&red[0][0][0]);
  auto sum_at = [&](int row, int tok) {
    float v = 0.0f;
    for (int r = 0; r < S; ++r) {
      const uint32_t base = S > 1 ? cluster_map(red_at, r) : red_at;
#pragma unroll
      for (int q = 0; q < WS_WK; ++q) {
        float x;
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(base + ((q * WS_ROWS + row) * WS_TOK + tok) * 4) : "memory");
        v += x;
      }
    }
    return v;
  };
  if constexpr (MODE == WS_UP) {
    const int routed = s_routed;
    for (int i = rank * WS_THREADS + tid; i < WS_ROWS / 2 * WS_TOK; i += S * WS_THREADS) {
      const int c = i % (WS_ROWS / 2), tok = i / (WS_ROWS / 2), row = (c >> 3) * 16 + (c & 7);
      const int col = tile * (WS_ROWS / 2) + c;
      if (tok < p.M && col < p.N && ((routed >> tok) & 1)) {
        const float u1 = sum_at(row, tok), u2 = sum_at(row + 8, tok);
        p.h[(static_cast<long long>(slot) * p.M + tok) * p.N + col] = u1 * (u2 / (1.0f + expf(-u2)));
      }
    }
  } else {
    for (int i = rank * WS_THREADS + tid; i < WS_ROWS * WS_TOK; i += S * WS_THREADS) {
      const int row = i % WS_ROWS, tok = i / WS_ROWS, col = tile * WS_ROWS + row;
      if (tok < p.M && col < p.N) static_cast<T*>(p.out)[static_cast<long long>(tok) * p.N + col] = from_f32<T>(sum_at(row, tok));
    }
  }
  if (S > 1) cluster_sync_all();                  // no block ends while another reads its sums
}

// One launch of a cluster of S blocks per row tile (and per slot).
template <typename T, int MODE>
inline cudaError_t launch_w4_stream(StreamArgs a, int cluster, int slots, bool programmatic, cudaStream_t st) {
  const int per = MODE == WS_UP ? WS_ROWS / 2 : WS_ROWS;
  cudaLaunchConfig_t cfg{};
  a.cluster = cluster;
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<long long>(a.N) + per - 1) / per * cluster), static_cast<unsigned>(slots));
  cfg.blockDim = dim3(WS_THREADS);
  cfg.dynamicSmemBytes = ws_smem(MODE, a.M, a.spp, a.w.group);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim = {static_cast<unsigned>(cluster), 1, 1};
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = programmatic ? 2 : 1;
  const bool aligned = ((a.K + 1) / 2) % 16 == 0 && (reinterpret_cast<uintptr_t>(a.w.codes) & 15u) == 0;
  auto go = [&](auto kernel) -> cudaError_t {
    // Above 48 KB the size has to be allowed first; a no-op after the first call.
    if (cfg.dynamicSmemBytes > 40 * 1024)
      if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(cfg.dynamicSmemBytes)))
        return e;
    return cudaLaunchKernelEx(&cfg, kernel, a);
  };
  switch (a.w.group) {
    case 128: return aligned ? go(w4_stream_kernel<T, 4, MODE, true>) : go(w4_stream_kernel<T, 4, MODE, false>);
    case 64: return aligned ? go(w4_stream_kernel<T, 2, MODE, true>) : go(w4_stream_kernel<T, 2, MODE, false>);
    default: return aligned ? go(w4_stream_kernel<T, 1, MODE, true>) : go(w4_stream_kernel<T, 1, MODE, false>);
  }
}

}  // namespace moe
