/*
 * Products with 4-bit weights for more than a few tokens, on tcgen05.mma (kind::f16): the weights are the
 * M = 128 operand in tensor memory, the tokens (16 to NT columns) the N operand in shared memory.
 *
 *   codes -> TMA, 128 rows x 256 columns a stage -> 8 warps turn a row's codes into numbers code - zero, exact in
 *   bf16 and f16 (a nibble in the mantissa of 128 or 1024, minus 128 + zero or 1024 + zero) -> tensor memory ->
 *   one accumulator per group of columns -> 4 warps add scale * accumulator to the row's sums in fp32.
 *
 * No weight is rounded, and the scale of a group multiplies a finished sum. A thread owns a weight row all the way:
 * it reads the row's codes, writes the row's lane of tensor memory, and (in the last warps) scales its sums.
 *
 * A word's codes come out as the pairs (0,4), (1,5), (2,6), (3,7) with two instructions each; the tokens' rows are
 * kept in that order of columns (within each 8), which costs their copy nothing.
 *
 * Roles: warp 0 loads codes, warp 1 issues the mma, warp 2 loads token rows; two warpgroups convert, taking turns with
 * steps of 256 columns; one or two scale and store. Persistent: one block per SM walks
 * the units (token tile, 128 weight rows[, part of the columns]).
 *
 * Measured on a B200 (device time, 32 experts of 7168 x 2048, group 128): T = 64 of a 256-expert layer 187 us, 3.3 TB/s of
 * weights; T = 4096 742 us, 485 TFLOP/s; linear_w4 512 x 4096 x 7168 39 us, 770 TFLOP/s. Counters (profiles/w4_mma.md): T = 64's
 * first product keeps DRAM 42%, the issue slots 59% and the tensor pipe 10% busy, T = 4096's 22%, 55% and 34%: nothing is
 * full, the roles wait for each other. At T = 4096 the likely reason is the way into the SM: a step brings 16 KB of codes
 * and up to 64 KB of token rows, which at 64 bytes a cycle (reckoned, not measured by itself) is as long as its mma. Pairs
 * of SMs that share the token rows (cta_group::2) would halve that.
 */
#pragma once
#include "gate.cuh"
#include "w4_stream.cuh"

namespace moe {

constexpr int WM_STEP = 256;                    // columns per step
constexpr int WM_CODE_BYTES = 128 * WM_STEP / 2;
// Register split of the blocks of 640 threads: warpgroup 0, the two that convert, the two that scale.
constexpr int WM_REGS_CTRL = 40, WM_REGS_CONV = 88, WM_REGS_EPI = 128;
constexpr int WM_LAUNCH_REGS_MIN = (WM_REGS_CTRL + 2 * WM_REGS_CONV + 2 * WM_REGS_EPI + 4) / 5;

// Shared memory: a ring of steps of codes, a ring of token rows. An entry of the second holds B_COLS columns of every
// term (up to 64 KB), so that a step of few tokens is one entry.
// Tensor memory: two batches of accumulators, then the weights of as many steps (128 columns each) as fit.
// A barrier's parity tells only neighbouring uses apart. The converting warpgroups take every second step, so they skip uses
// of a ring whose length is odd; that is safe here because the mma of the steps before them has finished by then (the weights'
// slots are fewer than the codes' stages and are given back in order).
template <int NT, int TERMS, int G>
struct WmShape {
  static constexpr int D_COLS = NT * TERMS * (WM_STEP / G) >= 128 ? 128 : NT * TERMS * (WM_STEP / G);
  static constexpr int A_COL = 2 * D_COLS;
  static constexpr int A_SLOTS = (512 - A_COL) / 128;
  // Warpgroups that scale, each TOK tokens of the tile: above 32 tokens one would be the slowest of the roles (four for 128
  // tokens took 8% longer than two: more warps on the same barriers).
  static constexpr int EPI = NT == 32 ? 1 : 2;
  static constexpr int TOK = NT / EPI;
  static constexpr int THREADS = 128 * (3 + EPI);
  static constexpr int B_COLS = NT * TERMS >= 128 ? 128 : 256;
  static constexpr int B_BYTES = NT * TERMS * B_COLS * 2;
  static constexpr int B_STAGES = 4;
  static constexpr int CODE_STAGES = B_BYTES >= 32768 ? 5 : 8;
  static constexpr int RING = CODE_STAGES * WM_CODE_BYTES + B_STAGES * B_BYTES;
  static_assert(RING <= 212992, "rings too large");
};

struct WmCtrl {
  uint64_t c_full[8], c_empty[8];
  uint64_t b_full[4], b_empty[4];
  uint64_t a_full[3], a_empty[3];
  uint64_t d_full[2], d_empty[2];
  uint64_t mma_done;
  uint32_t tmem_base;
  int abort_flag;
  int tile_off[RX_MAX_E + 1];                   // first token tile of each expert
  int row_off[RX_MAX_E + 1];                    // first row of each expert in the route-ordered buffers
};

template <int NT, int TERMS, int G>
constexpr int WM_SMEM = WmShape<NT, TERMS, G>::RING + static_cast<int>(sizeof(WmCtrl)) + 1024;

// Tensor maps. codes: 4-D (bytes of a row, rows, X1 / X2, experts), one box per step. x: 4-D (64 columns, rows, terms,
// blocks of 64 columns), one map for each box height of 16, 32, ... 128 rows; a box is a ring entry as the mma reads it.
// One copy instruction per entry: a producer's thread needs some hundred cycles for each.
struct WmMaps {
  CUtensorMap codes;
  CUtensorMap x[8];
};

struct WmArgs {
  W4Matrix w;
  int E, N, K;              // experts; output columns (up: I) and reduction length of one
  int M;                    // linear: tokens
  int codes_copied;         // linear: the codes come from the kernel before, too
  const int* counts;        // [E] routes per expert (up, down)
  int row_cap;              // rows of the route-ordered buffers
  int splits, sps;          // linear: parts of the columns, each of `sps` steps
  __nv_bfloat16* h;         // up: [2][row_cap][Ip] hi and lo of the intermediate, columns in pair order
  int h_pitch;              // Ip
  float* y;                 // down: [row_cap][N]; linear with splits: [splits][M][N]
  void* out;                // linear: [M][N]
};

// Position of column c inside the pair order (0,4,1,5,2,6,3,7) of its 8, and back.
__host__ __device__ __forceinline__ int pair_pos(int c) { return (c & ~7) | ((c & 3) << 1) | ((c >> 2) & 1); }

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// D(tmem) (+)= A(tmem, 128 x 16) x B(smem desc)^T, bf16 or f16 operands (idesc), fp32 accumulate.
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 4-D tiled TMA load (no multicast) with an L2 policy.
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.L2::cache_hint "
      "[%0], [%1, {%2, %3, %4, %5}], [%6], %7;" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar)), "l"(policy)
      : "memory");
}

// One lane of a converged warp. The compiler then knows that a single thread runs what follows and keeps the operands of
// mma and copy instructions in uniform registers: an mma with 16 tokens issues every 9 cycles, behind `lane == 0` every 46.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "elect.sync _|q, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(p));
  return p != 0;
}

// 16 columns of this warp's lanes, without waiting; and the wait, tied to the registers that it makes valid.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]),
                 "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
}
// acc[i] += v[i] * f for 16 values, two to an instruction.
__device__ __forceinline__ void fma16_scaled(float* acc, const float (&v)[16], float f) {
  uint64_t ff;
  asm("mov.b64 %0, {%1, %1};" : "=l"(ff) : "f"(f));
#pragma unroll
  for (int i = 0; i < 16; i += 2) {
    uint64_t a, b;
    asm("mov.b64 %0, {%1, %2};" : "=l"(a) : "f"(acc[i]), "f"(acc[i + 1]));
    asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(v[i]), "f"(v[i + 1]));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(b), "l"(ff));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(acc[i]), "=f"(acc[i + 1]) : "l"(a));
  }
}

// Bounded wait of a converged warp, every lane for itself (each needs its own acquire); they agree on giving up. The
// hardware suspends the lanes meanwhile: polling warps take issue slots and shared-memory cycles from the others.
__device__ __forceinline__ bool wait_warp(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int who) {
  // A completed phase is seen by the plain test in a third of the suspending test's time.
  if (__all_sync(0xffffffffu, mbar_test_wait(bar, parity))) return true;
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, who));
}

// Tiles of up to NT tokens: an expert's rows in equal parts.
__host__ __device__ __forceinline__ int wm_tiles(int rows, int nt) { return (rows + nt - 1) / nt; }

// Prefix sums of the experts' tiles and rows; one full warp. Counts outside [0, cap], or adding up to more than cap,
// are reported and taken as none.
__device__ __forceinline__ void wm_build_map(int* tile_off, int* row_off, const int* counts, int E, int cap, int nt) {
  const int lane = threadIdx.x & 31, per = (E + 31) / 32;
  long long rows = 0;
  int tiles = 0;
  bool bad = false;
  for (int i = 0; i < per; ++i) {
    const int e = lane * per + i;
    const int c = e < E ? counts[e] : 0;
    bad |= c < 0 || c > cap;
    rows += c;
    tiles += wm_tiles(c, nt);
  }
  long long r_incl = rows;
  int t_incl = tiles;
  for (int o = 1; o < 32; o <<= 1) {
    const long long rn = __shfl_up_sync(0xffffffffu, r_incl, o);
    const int tn = __shfl_up_sync(0xffffffffu, t_incl, o);
    if (lane >= o) {
      r_incl += rn;
      t_incl += tn;
    }
  }
  bad = __any_sync(0xffffffffu, bad || r_incl > cap);
  if (bad && lane == 0) report_status(ST_BAD_INDEX);
  int t = bad ? 0 : t_incl - tiles, r = bad ? 0 : static_cast<int>(r_incl - rows);
  for (int i = 0; i < per; ++i) {
    const int e = lane * per + i;
    if (e <= E) {
      tile_off[e] = t;
      row_off[e] = r;
    }
    const int c = e < E && !bad ? counts[e] : 0;
    t += wm_tiles(c, nt);
    r += c;
  }
  if (lane == 31 && 32 * per == E) {
    tile_off[E] = t;
    row_off[E] = r;
  }
}

// Operand columns of a tile's tokens: the height of the box that brings them.
__device__ __forceinline__ int wm_cols(int tokens) { return (tokens + 15) & ~15; }

struct WmUnit {
  int expert, row0, tokens;    // first row and count of the tile's tokens
  int rt, split;               // 128-row tile of the weights; part of the columns
};

template <int NT>
__device__ __forceinline__ WmUnit wm_unit(const WmCtrl* ctl, const WmArgs& p, int u, int row_tiles) {
  WmUnit w;
  w.rt = u % row_tiles;
  int tile = u / row_tiles;
  w.split = tile % p.splits;
  tile /= p.splits;
  int lo = 0, hi = p.E;        // tile_off[lo] <= tile < tile_off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (ctl->tile_off[mid] <= tile) lo = mid; else hi = mid;
  }
  w.expert = lo;
  const int rows = ctl->row_off[lo + 1] - ctl->row_off[lo], tiles = ctl->tile_off[lo + 1] - ctl->tile_off[lo];
  const int i = tile - ctl->tile_off[lo];
  const int a = static_cast<int>(static_cast<long long>(rows) * i / tiles), b = static_cast<int>(static_cast<long long>(rows) * (i + 1) / tiles);
  w.row0 = ctl->row_off[lo] + a;
  w.tokens = b - a;
  return w;
}

template <typename T, int MODE, int NT, int G>
__global__ void __launch_bounds__(WmShape<NT, MODE == WS_DOWN ? 2 : 1, G>::THREADS, 1)
    w4_mma_kernel(const __grid_constant__ WmMaps maps, const __grid_constant__ WmArgs p) {
  using W = typename std::conditional<MODE == WS_DOWN, __nv_bfloat16, T>::type;   // the operands' type
  constexpr int TERMS = MODE == WS_DOWN ? 2 : 1;
  using S = WmShape<NT, TERMS, G>;
  constexpr int GPS = WM_STEP / G;                                      // groups per step
  constexpr int NC = NT * TERMS;                                        // columns of one accumulator
  constexpr int GPB = S::D_COLS / NC < GPS ? S::D_COLS / NC : GPS;      // groups per batch of accumulators
  constexpr int ENTRIES = WM_STEP / S::B_COLS;                          // entries of token rows per step
  extern __shared__ uint8_t wm_raw[];
  uint8_t* smem = align_1024(wm_raw);
  uint8_t* ring_c = smem;
  uint8_t* ring_b = smem + S::CODE_STAGES * WM_CODE_BYTES;
  WmCtrl* ctl = reinterpret_cast<WmCtrl*>(smem + S::RING);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < S::CODE_STAGES; ++i) {
      mbar_init(&ctl->c_full[i], 1);
      mbar_init(&ctl->c_empty[i], 4);
    }
    for (int i = 0; i < S::B_STAGES; ++i) {
      mbar_init(&ctl->b_full[i], 1);
      mbar_init(&ctl->b_empty[i], 1);
    }
    for (int i = 0; i < S::A_SLOTS; ++i) {
      mbar_init(&ctl->a_full[i], 4);
      mbar_init(&ctl->a_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ctl->d_full[i], 1);
      mbar_init(&ctl->d_empty[i], 4 * S::EPI);
    }
    mbar_init(&ctl->mma_done, 1);
    ctl->abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
  }
  // Counts come from the kernel before the first product; the second product may read them at once, since the first one
  // lets it start only after its own wait, and load weights while the first still runs.
  if (MODE == WS_UP) wait_prerequisite_grids();
  if (warp == 2) {
    if constexpr (MODE == WS_LINEAR) {
      if (lane == 0) {
        ctl->tile_off[0] = ctl->row_off[0] = 0;
        ctl->tile_off[1] = wm_tiles(p.M, NT);
        ctl->row_off[1] = p.M;
      }
    } else {
      wm_build_map(ctl->tile_off, ctl->row_off, p.counts, p.E, p.row_cap, NT);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (threadIdx.x == 0) allow_dependent_launch();
  const uint32_t tmem = ctl->tmem_base;
  volatile int* abort_flag = &ctl->abort_flag;

  const int per_tile = MODE == WS_UP ? 64 : 128;      // output columns of 128 weight rows
  const int row_tiles = (p.N + per_tile - 1) / per_tile;
  const int units = ctl->tile_off[p.E] * p.splits * row_tiles;
  const int steps = (p.K + WM_STEP - 1) / WM_STEP;
  const int groups = (p.K + G - 1) / G;
  auto range = [&](const WmUnit& w, int& s0, int& s1) {   // steps of the unit
    s0 = w.split * p.sps;
    s1 = min(steps, s0 + p.sps);
  };

  if (warp < 4) {
    if constexpr (S::EPI == 2) regs_dec<WM_REGS_CTRL>();
    if (warp == 0 && elect_one()) {
      // ---------------- codes ----------------
      if (MODE == WS_LINEAR && p.codes_copied) {
        wait_prerequisite_grids();
        fence_proxy_async_global();
      }
      const uint64_t pol = policy_evict_first();
      uint32_t it = 0;
      for (int u = blockIdx.x; u < units && !*abort_flag; u += gridDim.x) {
        const WmUnit w = wm_unit<NT>(ctl, p, u, row_tiles);
        int s0, s1;
        range(w, s0, s1);
        const int y = w.rt * per_tile;
        for (int s = s0; s < s1; ++s, ++it) {
          const int st = it % S::CODE_STAGES;
          if (!mbar_wait(&ctl->c_empty[st], ((it / S::CODE_STAGES) & 1u) ^ 1u, abort_flag, ST_TIMEOUT_PRODUCER)) break;
          mbar_arrive_expect_tx(&ctl->c_full[st], WM_CODE_BYTES);
          tma_load_4d(ring_c + st * WM_CODE_BYTES, &maps.codes, s * (WM_STEP / 2), y, 0, w.expert, &ctl->c_full[st], pol);
        }
      }
      if (*abort_flag)
        for (uint32_t i = 1; i <= S::CODE_STAGES && i <= it; ++i)
          mbar_wait_drain(&ctl->c_full[(it - i) % S::CODE_STAGES], ((it - i) / S::CODE_STAGES) & 1u);
    } else if (warp == 2 && elect_one()) {
      // ---------------- token rows ----------------
      if (MODE != WS_UP) wait_prerequisite_grids();          // rows come from the kernel before
      fence_proxy_async_global();                           // its stores, then this thread's copies
      const uint64_t pol = policy_evict_last();
      uint32_t it = 0;
      for (int u = blockIdx.x; u < units && !*abort_flag; u += gridDim.x) {
        const WmUnit w = wm_unit<NT>(ctl, p, u, row_tiles);
        int s0, s1;
        range(w, s0, s1);
        const int n = wm_cols(w.tokens);                     // rows past the tile's are read for nothing
        const CUtensorMap* map = &maps.x[n / 16 - 1];
        const uint32_t bytes = n * S::B_COLS * 2 * TERMS;
        for (int c = s0 * ENTRIES; c < s1 * ENTRIES; ++c, ++it) {
          const int st = it % S::B_STAGES;
          if (!mbar_wait(&ctl->b_empty[st], ((it / S::B_STAGES) & 1u) ^ 1u, abort_flag, ST_TIMEOUT_PRODUCER)) break;
          mbar_arrive_expect_tx(&ctl->b_full[st], bytes);
          tma_load_4d(ring_b + st * S::B_BYTES, map, 0, w.row0, 0, c * (S::B_COLS / 64), &ctl->b_full[st], pol);
        }
      }
      if (*abort_flag)
        for (uint32_t i = 1; i <= S::B_STAGES && i <= it; ++i)
          mbar_wait_drain(&ctl->b_full[(it - i) % S::B_STAGES], ((it - i) / S::B_STAGES) & 1u);
    } else if (warp == 1 && elect_one()) {
      // ---------------- mma ----------------
      constexpr int BC = S::B_COLS / 64, PARTS = G == 32 ? 2 : 1;      // 64-column pieces per entry, groups per piece
      const uint64_t b_desc0 = sdesc_k_sw128(smem_u32(ring_b));
      uint32_t b_it = 0, a_it = 0, d_it = 0;
      // A wait that gives up leaves at once: a flag tested before each mma would double the cost of issuing it.
      for (int u = blockIdx.x; u < units; u += gridDim.x) {
        const WmUnit w = wm_unit<NT>(ctl, p, u, row_tiles);
        int s0, s1;
        range(w, s0, s1);
        const int n = TERMS * wm_cols(w.tokens);
        const uint64_t chunk = static_cast<uint64_t>(n * 128 >> 4);    // from one block of 64 columns to the next
        constexpr uint32_t fmt = std::is_same_v<W, __half> ? 0u : (1u << 7) | (1u << 10);
        const uint32_t idesc = (1u << 4) | fmt | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
        for (int s = s0; s < s1; ++s, ++a_it) {
          const uint32_t slot = a_it % S::A_SLOTS;
          const uint32_t a = tmem + S::A_COL + slot * 128;
          uint64_t bd = b_desc0;
          uint32_t d = 0;
#pragma unroll
          for (int c = 0; c < WM_STEP / 64; ++c) {                     // 64 columns at a time
            if (c % BC == 0) {
              if (!mbar_wait_spin(&ctl->b_full[b_it % S::B_STAGES], (b_it / S::B_STAGES) & 1u, abort_flag, ST_TIMEOUT_MMA)) goto mma_end;
              bd = b_desc0 + (b_it % S::B_STAGES) * (S::B_BYTES >> 4);
            }
#pragma unroll
            for (int part = 0; part < PARTS; ++part) {
              const int k = c * 64 + part * 32;                        // column of the step
              if (k % (G * GPB) == 0) {                                // a batch of accumulators starts
                if (!mbar_wait_spin(&ctl->d_empty[d_it & 1], ((d_it >> 1) & 1u) ^ 1u, abort_flag, ST_TIMEOUT_MMA)) goto mma_end;
                d = tmem + (d_it & 1) * S::D_COLS;
              }
              // The weights come last, as a rule: nothing else is waited for between them and the step's first mma.
              if (k == 0 && !mbar_wait_spin(&ctl->a_full[slot], (a_it / S::A_SLOTS) & 1u, abort_flag, ST_TIMEOUT_MMA)) goto mma_end;
              if (k % (G * GPB) == 0 || c % BC == 0) tc_fence_after();
#pragma unroll
              for (int kk = 0; kk < 4 / PARTS; ++kk) {
                const int k16 = part * (4 / PARTS) + kk;               // 16 columns of the 64
                tc_mma_ts(d + ((k / G) % GPB) * NC, a + c * 32 + k16 * 8, bd + (c % BC) * chunk + k16 * 2, idesc,
                          k % G == 0 && kk == 0 ? 0u : 1u);
              }
              if ((k + 64 / PARTS) % (G * GPB) == 0) {
                tc_commit(&ctl->d_full[d_it & 1]);
                ++d_it;
              }
            }
            if ((c + 1) % BC == 0) {
              tc_commit(&ctl->b_empty[b_it % S::B_STAGES]);
              ++b_it;
            }
          }
          tc_commit(&ctl->a_empty[slot]);
        }
      }
    mma_end:
      // Everything issued has finished before tensor and shared memory are given back.
      tc_commit(&ctl->mma_done);
      mbar_wait_drain(&ctl->mma_done, 0);
    }
  } else if (warp < 12) {
    // ---------------- codes to numbers: the warpgroups take turns with the steps ----------------
    if constexpr (S::EPI == 2) regs_dec<WM_REGS_CONV>();
    const uint32_t wg = (warp - 4) >> 2;
    const int q4 = warp & 3;
    // Row of the shared tile behind this lane of tensor memory; `up` puts X1's 16 rows and X2's side by side.
    const int srow = MODE == WS_UP ? (lane >> 4) * 64 + q4 * 16 + (lane & 15) : q4 * 32 + lane;
    const uint32_t a_dst0 = tmem + (static_cast<uint32_t>(q4 * 32) << 16) + S::A_COL;
    const uint8_t* row = ring_c + srow * 128;
    uint32_t it = 0;
    bool ok = true;
    for (int u = blockIdx.x; u < units && ok; u += gridDim.x) {
      const WmUnit w = wm_unit<NT>(ctl, p, u, row_tiles);
      int s0, s1;
      range(w, s0, s1);
      const uint8_t* zrow = nullptr;
      if (p.w.zero) {
        const long long r = MODE == WS_UP
            ? static_cast<long long>(w.expert) * 2 * p.N + (lane >> 4) * static_cast<long long>(p.N) + min(w.rt * 64 + q4 * 16 + (lane & 15), p.N - 1)
            : static_cast<long long>(w.expert) * p.N + min(w.rt * 128 + srow, p.N - 1);
        zrow = p.w.zero + r * groups;
      }
      const uint32_t end = it + static_cast<uint32_t>(s1 - s0);
      int s = s0 + static_cast<int>((it ^ wg) & 1u);                   // the warpgroups take turns across units
      for (it += (it ^ wg) & 1u; it < end; it += 2, s += 2) {
        const uint32_t st = it % S::CODE_STAGES, slot = it % S::A_SLOTS;
        W4Offset<W> off[GPS];
#pragma unroll
        for (int i = 0; i < GPS; ++i) off[i] = w4_offset<W>(zrow ? __ldg(zrow + min(s * GPS + i, groups - 1)) & 15 : 8);
        if (!wait_warp(&ctl->c_full[st], (it / S::CODE_STAGES) & 1u, abort_flag, ST_TIMEOUT_EPILOGUE) ||
            !wait_warp(&ctl->a_empty[slot], ((it / S::A_SLOTS) & 1u) ^ 1u, abort_flag, ST_TIMEOUT_EPILOGUE)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint8_t* src = row + st * WM_CODE_BYTES;
        const uint32_t a_dst = a_dst0 + slot * 128;
#pragma unroll
        for (int hf = 0; hf < 4; ++hf) {                               // 64 columns: 32 columns of tensor memory
          uint32_t r[32];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint4 x = *reinterpret_cast<const uint4*>(src + (((hf * 2 + c) ^ (srow & 7)) << 4));
            const W4Offset<W> o = off[(hf * 64 + c * 32) / G];
            const uint32_t word[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) r[c * 16 + i * 4 + j] = w4_pair<W>(word[i], j, o);
          }
          tmem_st32(a_dst + hf * 32, r);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->c_empty[st]);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->a_full[slot]);
      }
      it = end;
    }
  } else {
    // ---------------- scale and store ----------------
    if constexpr (S::EPI == 2) regs_inc<WM_REGS_EPI>();
    constexpr int TOK = S::TOK;
    const int q4 = warp & 3, tok0 = (warp - 12) / 4 * TOK;               // this warpgroup's first token of a tile
    const uint32_t lanes = static_cast<uint32_t>(q4 * 32) << 16;
    const bool vec = groups % 8 == 0 && (reinterpret_cast<uintptr_t>(p.w.scale) & 15u) == 0;
    uint32_t d_it = 0;
    bool stop = false;
    for (int u = blockIdx.x; u < units && !stop; u += gridDim.x) {
      const WmUnit w = wm_unit<NT>(ctl, p, u, row_tiles);
      int s0, s1;
      range(w, s0, s1);
      const int col = MODE == WS_UP ? w.rt * 64 + q4 * 16 + (lane & 15) : w.rt * 128 + q4 * 32 + lane;
      const long long mrow = MODE == WS_UP ? static_cast<long long>(w.expert) * 2 * p.N + (lane >> 4) * static_cast<long long>(p.N) + min(col, p.N - 1)
                                           : static_cast<long long>(w.expert) * p.N + min(col, p.N - 1);
      const T* srow = static_cast<const T*>(p.w.scale) + mrow * groups;
      // The row's scales, 8 at a time (one 16-byte load where the rows allow it) and 8 ahead; 0 past the last group.
      auto load8 = [&](int g, uint32_t (&o)[4]) {
        if (vec) {
          const uint4 v = g < groups ? __ldg(reinterpret_cast<const uint4*>(srow + g)) : make_uint4(0, 0, 0, 0);
          o[0] = v.x; o[1] = v.y; o[2] = v.z; o[3] = v.w;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const T z = from_f32<T>(0.0f);
            o[i] = pack2(g + 2 * i < groups ? srow[g + 2 * i] : z, g + 2 * i + 1 < groups ? srow[g + 2 * i + 1] : z);
          }
        }
      };
      uint32_t cur[4], nxt[4];
      auto shift = [&]() {
#pragma unroll
        for (int i = 0; i < 3; ++i) cur[i] = __funnelshift_r(cur[i], cur[i + 1], 16);
        cur[3] >>= 16;
      };
      const int g_begin = s0 * GPS;
      load8(g_begin & ~7, cur);
      load8((g_begin & ~7) + 8, nxt);
      for (int i = 0; i < (g_begin & 7); ++i) shift();
      float total[TOK];
#pragma unroll
      for (int i = 0; i < TOK; ++i) total[i] = 0.0f;
      for (int g = g_begin; g < s1 * GPS; g += GPB, ++d_it) {
        const uint32_t q = d_it & 1;
        if (!wait_warp(&ctl->d_full[q], (d_it >> 1) & 1u, abort_flag, ST_TIMEOUT_EPILOGUE)) { stop = true; break; }
        tc_fence_after();
        const uint32_t src = tmem + lanes + q * S::D_COLS + tok0;
        const int n = wm_cols(w.tokens);
#pragma unroll
        for (int i = 0; i < GPB; ++i) {
          const uint16_t bits = static_cast<uint16_t>(cur[0]);
          const float f = to_f32(*reinterpret_cast<const T*>(&bits));
          shift();
          if (((g + i) & 7) == 7) {
#pragma unroll
            for (int j = 0; j < 4; ++j) cur[j] = nxt[j];
            load8(g + i + 9, nxt);
          }
          // 16 columns at a time, the next 16 on their way while these are added.
          float v[2][16];
          tmem_ld16(src + i * NC, v[0]);
#pragma unroll
          for (int c = 0; c < TERMS * (TOK / 16); ++c) {
            // Piece c: 16 tokens of one term, the terms of a token side by side. Pieces past the tile's tokens hold nothing;
            // leaving them out pays for small tiles only (it breaks the overlap of loads and sums).
            const int ahead = (c + 1) / TERMS * 16 + (c + 1) % TERMS * n;
            if (NT > 32 || c / TERMS * 16 < n) {
              tmem_wait_ld(v[c & 1]);
              if (c + 1 < TERMS * (TOK / 16) && (NT > 32 || (c + 1) / TERMS * 16 < n)) tmem_ld16(src + i * NC + ahead, v[(c + 1) & 1]);
              fma16_scaled(total + c / TERMS * 16, v[c & 1], f);
            }
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->d_empty[q]);
      }
      if (stop) break;
      const int tokens = w.tokens - tok0;                               // of this warpgroup
      const long long row0 = w.row0 + tok0;
      if constexpr (MODE == WS_LINEAR) {
        if (col < p.N) {
#pragma unroll
          for (int i = 0; i < TOK; ++i)
            if (i < tokens) {
              const long long at = (row0 + i) * p.N + col;
              if (p.splits > 1)
                p.y[static_cast<long long>(w.split) * p.M * p.N + at] = total[i];
              else
                static_cast<T*>(p.out)[at] = from_f32<T>(total[i]);
            }
        }
      } else if constexpr (MODE == WS_DOWN) {
        if (col < p.N) {
#pragma unroll
          for (int i = 0; i < TOK; ++i)
            if (i < tokens) p.y[(row0 + i) * p.N + col] = total[i];
        }
      } else {
        // Lanes 0-15 hold X1, lanes 16-31 X2 of the same columns: even tokens end in the first, odd in the second.
        // hi + lo bf16 carry 16 bits of h (off by 2^-17 at most; one term, off by 2^-8, would add as much as the output's own
        // rounding, and f16 terms would overflow); the columns go in pair order, zeros up to the next 64.
        const int pos = pair_pos(col), mine = lane >> 4;
#pragma unroll
        for (int i = 0; i < TOK; i += 2)
          if (i < tokens) {
            const float give = mine ? total[i] : total[i + 1];
            const float got = __shfl_xor_sync(0xffffffffu, give, 16);
            const float u1 = mine ? got : total[i], u2 = mine ? total[i + 1] : got;
            const float hv = col < p.N ? u1 * (u2 / (1.0f + expf(-u2))) : 0.0f;
            if (i + mine < tokens) {
              const __nv_bfloat16 hi = __float2bfloat16_rn(hv);
              const float rest = hv - __bfloat162float(hi);
              const long long at = (row0 + i + mine) * p.h_pitch + pos;
              p.h[at] = hi;
              // An infinity or NaN has no remainder.
              p.h[static_cast<long long>(p.row_cap) * p.h_pitch + at] = __float2bfloat16_rn(fabsf(rest) <= 3.4e38f ? rest : 0.0f);
            }
          }
      }
    }
  }
  if (MODE != WS_UP) wait_prerequisite_grids();           // this grid ends after the one before it
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ---- the kernels around it ----------------------------------------------------------------

// 8 columns from k on (0 past K), in pair order.
template <typename T>
__device__ __forceinline__ uint4 ld_pairs(const T* row, int k, int K) {
  alignas(16) T e[8];
  if (k + 8 <= K && (reinterpret_cast<uintptr_t>(row + k) & 15u) == 0) {
    *reinterpret_cast<uint4*>(e) = __ldg(reinterpret_cast<const uint4*>(row + k));
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = k + i < K ? row[k + i] : from_f32<T>(0.0f);
  }
  alignas(16) T o[8] = {e[0], e[4], e[1], e[5], e[2], e[6], e[3], e[7]};
  return *reinterpret_cast<const uint4*>(o);
}

// Codes with a row pitch of a multiple of 16 bytes, for shapes whose own rows do not allow TMA: words i, i + stride, ...
__device__ __forceinline__ void pad_codes(const uint8_t* codes, long long rows, int bytes, uint8_t* out, long long i, long long stride) {
  const int words = (bytes + 15) / 16 * 4;
  for (const long long n = rows * words; i < n; i += stride) {
    const long long r = i / words;
    const int o = static_cast<int>(i % words) * 4;
    uint32_t v = ld_u32_any(codes + r * bytes + o, bytes - o);
    if (bytes - o < 4) v = bytes > o ? v & ((1u << (8 * (bytes - o))) - 1u) : 0u;
    reinterpret_cast<uint32_t*>(out)[i] = v;
  }
}
__global__ void __launch_bounds__(256) pad_codes_kernel(const uint8_t* codes, long long rows, int bytes, uint8_t* out) {
  pad_codes(codes, rows, bytes, out, blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll);
}

// What linear_w4 lays out for the product, in one launch: rows of x in pair order, columns padded with zeros to a multiple
// of 64 (the first `row_blocks` blocks, 256 pieces of 8 columns each), and the codes' copy where one is needed.
template <typename T>
__global__ void __launch_bounds__(256) linear_w4_layout_kernel(const T* x, long long x_stride, int M, int K, T* out, int row_blocks,
                                                               const uint8_t* codes, int N, uint8_t* copy) {
  allow_dependent_launch();
  const int per = (K + 63) / 64 * 8, b = blockIdx.x;
  if (b < row_blocks) {
    const int i = b * 256 + threadIdx.x;                  // M * per < 2^31 / 8: at most 65535 rows of 2^31 / 65535 columns
    if (i < M * per) reinterpret_cast<uint4*>(out)[i] = ld_pairs(x + static_cast<long long>(i / per) * x_stride, i % per * 8, K);
  } else {
    pad_codes(codes, N, (K + 1) / 2, copy, (b - row_blocks) * 256ll + threadIdx.x, (gridDim.x - row_blocks) * 256ll);
  }
}

// Sum of the column parts of linear_w4, in order, rounded once.
template <typename T>
__global__ void __launch_bounds__(256) sum_parts_kernel(const float* y, int splits, long long n, T* out) {
  wait_prerequisite_grids();
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += gridDim.x * 256ll) {
    float v = y[i];
    for (int s = 1; s < splits; ++s) v += y[s * n + i];
    out[i] = from_f32<T>(v);
  }
}

// Rows of up to 64 KB or so, 16 bytes per lane and step: four in flight per lane.
template <typename T>
__device__ __forceinline__ void copy_row_pairs(const T* row, int K, uint4* out, int first, int stride) {
  const int per = (K + 63) / 64 * 8;
  int c = first;
  for (; c + 3 * stride < per; c += 4 * stride) {
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = ld_pairs(row, (c + i * stride) * 8, K);
#pragma unroll
    for (int i = 0; i < 4; ++i) out[c + i * stride] = v[i];
  }
  for (; c < per; c += stride) out[c] = ld_pairs(row, c * 8, K);
}

constexpr int WM_PLAN_MAX = 1024;   // picks that the one-kernel plan handles
constexpr int WM_GATHER = 16;       // picks that a block of the gather looks at together

// Few picks: one block per pick finds its row's place by itself (experts in order, picks of an expert in order) and
// copies the row; block 0 also counts the experts' picks. place[r]: the pick's row, or -1.
template <typename T>
__global__ void __launch_bounds__(256) experts_plan_kernel(const T* x, long long x_stride, const int* idx, int n, int k, int offset, int E,
                                                           int H, int* counts, int* place, T* out) {
  __shared__ int hist[RX_MAX_E];
  allow_dependent_launch();
  const int r = blockIdx.x, id = idx[r], e = id >= offset && id - offset < E ? id - offset : -1;
  int before = 0;
  if (r == 0) {
    for (int i = threadIdx.x; i < E; i += 256) hist[i] = 0;
    __syncthreads();
  }
  for (int q = threadIdx.x; q < n; q += 256) {
    const int iq = idx[q], eq = iq >= offset && iq - offset < E ? iq - offset : -1;
    if (eq < 0) continue;
    before += eq < e || (eq == e && q < r) ? 1 : 0;
    if (r == 0) atomicAdd(&hist[eq], 1);
  }
  __shared__ int warp_sum_[8];
  before = __reduce_add_sync(0xffffffffu, before);
  if ((threadIdx.x & 31) == 0) warp_sum_[threadIdx.x >> 5] = before;
  __syncthreads();
  if (r == 0)
    for (int i = threadIdx.x; i < E; i += 256) counts[i] = hist[i];
  int at = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) at += warp_sum_[i];
  if (threadIdx.x == 0) place[r] = e < 0 ? -1 : at;
  if (e < 0) return;
  const int per = (H + 63) / 64 * 8;
  copy_row_pairs(x + static_cast<long long>(r / k) * x_stride, H, reinterpret_cast<uint4*>(out) + static_cast<long long>(at) * per,
                 static_cast<int>(threadIdx.x), 256);
}

// Each local pick takes a place in its expert's list. The order within a list changes from call to call and no
// result with it: a row's products do not depend on the rows beside it.
__global__ void __launch_bounds__(256) experts_slot_kernel(const int* idx, int n, int offset, int E, int* counts, int* slot) {
  for (int r = blockIdx.x * 256 + threadIdx.x; r < n; r += gridDim.x * 256) {
    const int id = idx[r];
    const int e = id >= offset ? id - offset : -1;
    slot[r] = e >= 0 && e < E ? atomicAdd(counts + e, 1) : -1;
  }
}

// Copies each local pick's row to its expert's rows, in pair order; slot[r] becomes the row's place (or -1).
template <typename T>
__global__ void __launch_bounds__(256) experts_gather_kernel(const T* x, long long x_stride, const int* idx, int n, int k, int offset, int E,
                                                             const int* counts, int H, int* slot, T* out) {
  __shared__ int tile_off[RX_MAX_E + 1], row_off[RX_MAX_E + 1];
  allow_dependent_launch();
  if (threadIdx.x < 32) wm_build_map(tile_off, row_off, counts, E, n, 128);
  __syncthreads();
  // A block looks at some picks at a time, then copies the local ones' rows together.
  __shared__ int place[WM_GATHER];
  const int per = (H + 63) / 64 * 8;
  for (int base = blockIdx.x * WM_GATHER; base < n; base += gridDim.x * WM_GATHER) {
    __syncthreads();
    if (threadIdx.x < WM_GATHER) {
      const int r = base + static_cast<int>(threadIdx.x);
      int at = -1;
      if (r < n && slot[r] >= 0) {
        at = row_off[idx[r] - offset] + slot[r];
        if (at >= n) {
          report_status(ST_BAD_INDEX);
          at = -1;
        }
        slot[r] = at;
      }
      place[threadIdx.x] = at;
    }
    __syncthreads();
    for (int i = 0; i < WM_GATHER; ++i)
      if (place[i] >= 0)
        copy_row_pairs(x + static_cast<long long>((base + i) / k) * x_stride, H, reinterpret_cast<uint4*>(out) + static_cast<long long>(place[i]) * per,
                       static_cast<int>(threadIdx.x), 256);
  }
}

// out[t] = sum over the token's local picks, in their order, of weight * y[row], rounded once. A block has `span` columns of
// a token (a multiple of 1024). `vec`: 4 neighbouring columns per thread (H a multiple of 4, out 8-byte aligned).
template <typename T>
__global__ void __launch_bounds__(256) experts_combine_kernel(const float* y, const int* place, const float* wt, int k, int H, int span, int vec,
                                                              T* out) {
  __shared__ int row[RX_MAX_K];
  __shared__ float weight[RX_MAX_K];
  __shared__ int count;
  const long long t = blockIdx.y;
  wait_prerequisite_grids();
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    const int r = lane < k ? place[t * k + lane] : -1;
    const uint32_t m = __ballot_sync(0xffffffffu, r >= 0);
    if (r >= 0) {
      const int at = __popc(m & ((1u << lane) - 1u));
      row[at] = r;
      weight[at] = wt[t * k + lane];
    }
    if (lane == 0) count = __popc(m);
  }
  __syncthreads();
  const int n = count, begin = blockIdx.x * span, end = min(H, begin + span);
  if (vec) {
    // Up to 4 pieces of 1024 columns at a time, their loads together in flight.
    for (int c0 = begin; c0 < end; c0 += 4096) {
      float4 acc[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      for (int j = 0; j < n; ++j) {
        const float* src = y + static_cast<long long>(row[j]) * H + c0 + threadIdx.x * 4;
        const float w = weight[j];
        float4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c0 + i * 1024 + static_cast<int>(threadIdx.x) * 4 < end) v[i] = __ldcs(reinterpret_cast<const float4*>(src + i * 1024));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (c0 + i * 1024 + static_cast<int>(threadIdx.x) * 4 < end) {
            acc[i].x = fmaf(w, v[i].x, acc[i].x);
            acc[i].y = fmaf(w, v[i].y, acc[i].y);
            acc[i].z = fmaf(w, v[i].z, acc[i].z);
            acc[i].w = fmaf(w, v[i].w, acc[i].w);
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + i * 1024 + threadIdx.x * 4;
        if (c < end)
          *reinterpret_cast<uint2*>(out + t * H + c) =
              make_uint2(pack2(from_f32<T>(acc[i].x), from_f32<T>(acc[i].y)), pack2(from_f32<T>(acc[i].z), from_f32<T>(acc[i].w)));
      }
    }
  } else {
    for (int i = begin + threadIdx.x; i < end; i += 256) {
      float acc = 0.0f;
      for (int j = 0; j < n; ++j) acc = fmaf(weight[j], y[static_cast<long long>(row[j]) * H + i], acc);
      out[t * H + i] = from_f32<T>(acc);
    }
  }
}

}  // namespace moe
