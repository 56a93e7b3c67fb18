/*
 * linear_w4 for up to 8 tokens, in one launch: the weights are read once, straight from global memory into matrix
 * fragments.
 *
 *   mma m16n8k16: A = 16 weight rows x 16 columns, B = 16 columns x 8 tokens, fp32 accumulators.
 *
 * A thread holds, of rows g and g + 8 of a tile, the codes at a few places; which columns those are is free as long as A
 * and B agree. Thread t of a row's four takes group / 4 neighbouring columns of each group (one 16-, 8- or 4-byte load); a
 * 32-bit word of 8 codes makes the fragments of two mma. Codes become numbers by placing a nibble in the mantissa of 128
 * (bf16) or 1024 (f16) and subtracting 128 + zero or 1024 + zero: exact, as is every product (published for f16 by Kim et
 * al., "Who Says Elephants Can't Run", 2022). Each group's sum is scaled in fp32: no weight is rounded.
 *
 * Split: a block has one tile of 16 rows, its 8 warps an eighth of the columns each; their sums meet in shared memory in
 * warp order, so results repeat bit for bit. Nothing is staged: a warp alone uses its columns of x. 1 to 4 steps of 128
 * columns are in flight per warp (1 KB each).
 *
 * Measured on a B200 (device time, group 128): 4096 x 7168 for one token 8.5 to 9.6 us, from one B200 to another (1.5 to
 * 1.7 TB/s of codes; three copies of the weights in turn, which L2 holds), for 8 tokens 9.9 us; 7168 x 2048 6.2 us;
 * 28672 x 7168, which L2 does not hold so, 47.6 us (2.2 TB/s), for 8 tokens 55.6 us. No single part is the limit there
 * (profiles/w4_stream_m1.md): 36 instructions per 256 weights take 56% of the issue slots, DRAM is 25% busy, and with 4
 * warps to a scheduler (128 registers) the slots left empty are waits for memory, for the instruction before and for the
 * arithmetic pipes, in this order. A block's 7 steps per warp begin with an empty pipe each time. An e4m3 mma would need
 * no conversion (a code's byte is an e4m3 number), but mma.sync with it took some 30 issue slots on sm_100a, more than the
 * conversion. Staging activations and scales in shared memory, with the columns split over a cluster, took 14 us for the
 * first shape.
 */
#pragma once
#include "gate.cuh"
#include "w4.cuh"

#include <type_traits>

namespace moe {

constexpr int WS_WARPS = 8, WS_THREADS = 32 * WS_WARPS;
constexpr int WS_ROWS = 16;                     // weight rows per block
constexpr int WS_TOK = 8;                       // tokens per mma
constexpr int WS_STEP = 128;                    // columns per step

enum { WS_LINEAR = 0, WS_UP = 1, WS_DOWN = 2 };  // which product a kernel computes: linear_w4, the experts' first, second

struct StreamArgs {
  const void* x;           // [M, K]
  long long x_stride;
  W4Matrix w;
  int M, N, K;             // tokens (<= 8), output columns, reduction length
  void* out;               // [M, N]
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

// What a code's number is minus: 128 + zero twice in bf16; 1024 + zero and 64 + zero twice in f16 (all exact: zero < 16).
template <typename T>
struct W4Offset {
  uint32_t a, b;
};
template <typename T>
__device__ __forceinline__ W4Offset<T> w4_offset(int zero) {
  const uint32_t z = static_cast<uint32_t>(zero);
  if constexpr (std::is_same_v<T, __half>)
    return {(0x6400u + z) * 0x10001u, (0x5400u + (z << 4)) * 0x10001u};
  else
    return {(0x4300u + z) * 0x10001u, 0u};
}

// Pair i of a word's codes (columns i and i + 4) as two numbers code - zero. A nibble in bits 0-3 of the mantissa of 128
// (bf16) or 1024 (f16) adds its value; f16's ten bits also take one in bits 4-7, of 64, which saves two of three shifts.
template <typename T>
__device__ __forceinline__ uint32_t w4_pair(uint32_t word, int i, const W4Offset<T>& off) {
  uint32_t v;
  if constexpr (std::is_same_v<T, __half>) {
    const uint32_t w = i < 2 ? word : word >> 8;
    if (i % 2 == 0)
      asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(v) : "r"(w));
    else
      asm("lop3.b32 %0, %1, 0x00f000f0, 0x54005400, 0xea;" : "=r"(v) : "r"(w));
    const __half2 d = __hsub2(*reinterpret_cast<__half2*>(&v), *reinterpret_cast<const __half2*>(i % 2 == 0 ? &off.a : &off.b));
    return *reinterpret_cast<const uint32_t*>(&d);
  } else {
    asm("lop3.b32 %0, %1, 0x000f000f, 0x43004300, 0xea;" : "=r"(v) : "r"(word >> (4 * i)));
    const __nv_bfloat162 d = __hsub2(*reinterpret_cast<__nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&off.a));
    return *reinterpret_cast<const uint32_t*>(&d);
  }
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

// The four words of one step that thread t of a row's four holds; `row` is the row's code byte of the step's first column
// plus 4 G4 t. G4 = group / 32 words per group: word i holds columns (i / G4) * group + t * group / 4 + (i % G4) * 8 .. + 8.
// `left`: bytes of the row from `row` on. FULL: the whole step lies inside the row.
template <int G4, bool ALIGNED, bool FULL>
__device__ __forceinline__ uint4 ld_codes(const uint8_t* row, int left) {
  uint32_t v[4] = {0u, 0u, 0u, 0u};
  if constexpr (ALIGNED) {
#pragma unroll
    for (int s = 0; s < 4 / G4; ++s) {
      const int o = s * (16 * G4);
      if (FULL || o < left) {
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
      const int o = (i / G4) * (16 * G4) + (i % G4) * 4;
      v[i] = ld_u32_any(row + o, left - o);
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
  if (k + 8 <= K) {
    uint4 v;
    if (vec) {
      v = __ldg(reinterpret_cast<const uint4*>(row + k));
    } else {
      // Aligned words that hold a wanted value, shifted together where the row starts in the middle of one.
      const uintptr_t at = reinterpret_cast<uintptr_t>(row + k);
      const uint32_t* w = reinterpret_cast<const uint32_t*>(at & ~static_cast<uintptr_t>(3));
      const int sh = static_cast<int>(at & 2) * 8;
      uint32_t u[5];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = __ldg(w + i);
      u[4] = sh ? __ldg(w + 4) : 0u;
      v = make_uint4(__funnelshift_r(u[0], u[1], sh), __funnelshift_r(u[1], u[2], sh), __funnelshift_r(u[2], u[3], sh),
                     __funnelshift_r(u[3], u[4], sh));
    }
    return make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                      __byte_perm(v.y, v.w, 0x7632));
  }
  T e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) e[i] = k + i < K ? row[k + i] : from_f32<T>(0.0f);
  return make_uint4(pack2(e[0], e[4]), pack2(e[1], e[5]), pack2(e[2], e[6]), pack2(e[3], e[7]));
}

template <typename T, int G4, bool ALIGNED>
__global__ void __launch_bounds__(WS_THREADS, 2) w4_stream_kernel(const __grid_constant__ StreamArgs p) {
  constexpr int GPS = 4 / G4;                    // groups per step
  // Steps in flight per warp, which is also how often the step's code is unrolled: the long ones (many groups, byte-wise
  // addresses) would spend more time fetching instructions than they win.
  constexpr int DEPTH = !ALIGNED ? 1 : G4 == 4 ? 4 : 2;
  __shared__ float red[WS_WARPS][WS_ROWS][WS_TOK];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int pitch = (p.K + 1) / 2, steps = (p.K + WS_STEP - 1) / WS_STEP;
  const int groups = (p.K + p.w.group - 1) / p.w.group;
  const int per = (steps + WS_WARPS - 1) / WS_WARPS;
  const int a = warp * per, n = min(steps, a + per) - a;            // this warp's steps (n may be 0 or less)
  const int n0 = blockIdx.x * WS_ROWS;
  const long long r0 = min(n0 + g, p.N - 1), r1 = min(n0 + g + 8, p.N - 1);   // rows past N repeat the last one
  const T *f0 = static_cast<const T*>(p.w.scale) + r0 * groups, *f1 = static_cast<const T*>(p.w.scale) + r1 * groups;
  const uint8_t *z0 = p.w.zero ? p.w.zero + r0 * groups : nullptr, *z1 = p.w.zero ? p.w.zero + r1 * groups : nullptr;
  const T* xrow = static_cast<const T*>(p.x) + min(g, p.M - 1) * p.x_stride;
  const bool vec = __all_sync(0xffffffffu, (reinterpret_cast<uintptr_t>(xrow) & 15u) == 0);

  // Steps that lie wholly inside the rows are read without a check per load (all of them where K is a multiple of 128 and
  // the rows allow 16-byte loads).
  const int whole = ALIGNED && vec ? p.K / WS_STEP : 0;
  const uint8_t *c0 = p.w.codes + r0 * pitch + 4 * G4 * t, *c1 = p.w.codes + r1 * pitch + 4 * G4 * t;
  uint4 buf[DEPTH][2];
  auto codes = [&](int step, uint4 (&o)[2]) {
    const long long at = static_cast<long long>(step) * (WS_STEP / 2);
    const int left = pitch - static_cast<int>(at) - 4 * G4 * t;
    if (step < whole) {
      o[0] = ld_codes<G4, ALIGNED, true>(c0 + at, left);
      o[1] = ld_codes<G4, ALIGNED, true>(c1 + at, left);
    } else {
      o[0] = ld_codes<G4, ALIGNED, false>(c0 + at, left);
      o[1] = ld_codes<G4, ALIGNED, false>(c1 + at, left);
    }
  };
#pragma unroll
  for (int d = 0; d < DEPTH; ++d)
    if (d < n) codes(a + d, buf[d]);
  // One step ahead: activations, scales and zero points.
  uint4 x[4];
  float s0[GPS], s1[GPS];
  W4Offset<T> o0[GPS], o1[GPS];
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < GPS; ++i) o0[i] = o1[i] = w4_offset<T>(8);
  auto side = [&](int step) {
    const int k0 = step * WS_STEP;
    if (g < p.M) {
      if (step < whole) {
        const T* xt = xrow + k0 + 8 * G4 * t;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(xt + (i / G4) * (32 * G4) + (i % G4) * 8));
          x[i] = make_uint4(__byte_perm(v.x, v.z, 0x5410), __byte_perm(v.x, v.z, 0x7632), __byte_perm(v.y, v.w, 0x5410),
                            __byte_perm(v.y, v.w, 0x7632));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = ld_x_pairs<T>(xrow, k0 + (i / G4) * (32 * G4) + t * (8 * G4) + (i % G4) * 8, p.K, vec);
      }
    }
#pragma unroll
    for (int i = 0; i < GPS; ++i) {
      const int q = step < whole ? step * GPS + i : min(step * GPS + i, groups - 1);
      s0[i] = to_f32(f0[q]);
      s1[i] = to_f32(f1[q]);
      if (z0) {
        o0[i] = w4_offset<T>(__ldg(z0 + q) & 15);
        o1[i] = w4_offset<T>(__ldg(z1 + q) & 15);
      }
    }
  };
  float total[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if (n > 0) side(a);
  for (int s = 0; s < n; s += DEPTH) {
#pragma unroll
    for (int d = 0; d < DEPTH; ++d)
      if (s + d < n) {
        const uint32_t u0[4] = {buf[d][0].x, buf[d][0].y, buf[d][0].z, buf[d][0].w};
        const uint32_t u1[4] = {buf[d][1].x, buf[d][1].y, buf[d][1].z, buf[d][1].w};
        if (s + d + DEPTH < n) codes(a + s + d + DEPTH, buf[d]);
        const uint4 xs[4] = {x[0], x[1], x[2], x[3]};
        float fa[GPS], fb[GPS];
        W4Offset<T> oa[GPS], ob[GPS];
#pragma unroll
        for (int i = 0; i < GPS; ++i) {
          fa[i] = s0[i];
          fb[i] = s1[i];
          oa[i] = o0[i];
          ob[i] = o1[i];
        }
        if (s + d + 1 < n) side(a + s + d + 1);
#pragma unroll
        for (int q = 0; q < GPS; ++q) {
          float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = q * G4; i < (q + 1) * G4; ++i) {
            mma16816<T>(acc, w4_pair<T>(u0[i], 0, oa[q]), w4_pair<T>(u1[i], 0, ob[q]), w4_pair<T>(u0[i], 1, oa[q]),
                        w4_pair<T>(u1[i], 1, ob[q]), xs[i].x, xs[i].y);
            mma16816<T>(acc, w4_pair<T>(u0[i], 2, oa[q]), w4_pair<T>(u1[i], 2, ob[q]), w4_pair<T>(u0[i], 3, oa[q]),
                        w4_pair<T>(u1[i], 3, ob[q]), xs[i].z, xs[i].w);
          }
          total[0] = fmaf(fa[q], acc[0], total[0]);
          total[1] = fmaf(fa[q], acc[1], total[1]);
          total[2] = fmaf(fb[q], acc[2], total[2]);
          total[3] = fmaf(fb[q], acc[3], total[3]);
        }
      }
  }
  *reinterpret_cast<float2*>(&red[warp][g][2 * t]) = make_float2(total[0], total[1]);
  *reinterpret_cast<float2*>(&red[warp][g + 8][2 * t]) = make_float2(total[2], total[3]);
  __syncthreads();
  const int row = threadIdx.x % WS_ROWS, tok = threadIdx.x / WS_ROWS;
  if (tok < p.M && n0 + row < p.N) {
    float v = red[0][row][tok];
#pragma unroll
    for (int w = 1; w < WS_WARPS; ++w) v += red[w][row][tok];
    static_cast<T*>(p.out)[static_cast<long long>(tok) * p.N + n0 + row] = from_f32<T>(v);
  }
}

template <typename T>
inline cudaError_t launch_w4_stream(const StreamArgs& a, cudaStream_t st) {
  const bool aligned = ((a.K + 1) / 2) % 16 == 0 && (reinterpret_cast<uintptr_t>(a.w.codes) & 15u) == 0;
  const unsigned grid = (static_cast<unsigned>(a.N) + WS_ROWS - 1) / WS_ROWS;
  auto go = [&](auto kernel) { kernel<<<grid, WS_THREADS, 0, st>>>(a); };
  switch (a.w.group) {
    case 128: aligned ? go(w4_stream_kernel<T, 4, true>) : go(w4_stream_kernel<T, 4, false>); break;
    case 64: aligned ? go(w4_stream_kernel<T, 2, true>) : go(w4_stream_kernel<T, 2, false>); break;
    default: aligned ? go(w4_stream_kernel<T, 1, true>) : go(w4_stream_kernel<T, 1, false>); break;
  }
  return cudaGetLastError();
}

}  // namespace moe
