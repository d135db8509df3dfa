// Products of up to 64 tokens with 4-bit weights, w = (q - zero) * scale, one scale and zero per group of G columns
// (G = 32, 64 or 128): a plain product (DUAL = false) or the gate/up half of a gated MLP (DUAL = true), dense
// or over the experts of a mixture.
//
// What bounds it: HBM. A weight is half a byte (plus its share of scale and zero), so at the copy bandwidth an SM
// receives about 46 weights a clock and has four instruction slots for them. Two identities make that enough.
//
// 1. A nibble is an 8-bit float. The e4m3 codes 0..15 stand for 0, 1, .., 15 times 2^-9 (0..7 are the subnormals,
//    8..15 the first binade, with the same spacing). So a packed word needs two masks and a shift to become eight
//    operands of tcgen05.mma.kind::f8f6f4, exactly:  q 2^-9.
// 2. An activation is a short sum of 8-bit floats. e4m3 has 4 significant bits, bf16 8, fp16 11: with a power of
//    two per token and group that brings the group's largest value to [128, 256),
//      x 2^e = t_1 + t_2 (bf16)   or   t_1 + t_2 + t_3 (fp16),   t_i the e4m3 rounding of what is left.
//    That is exact for values within 2^-9 (bf16) or 2^-6 (fp16) of the group's largest; below, the error is at most
//    2^-10 (half the spacing of e4m3's subnormals) where the largest is at least 2^7: 2^-17 of the group's largest
//    value, 256 (bf16) or 32 (fp16) times less than that value's own half step.
//    The terms are separate columns of the MMA (the tensor pipe is idle at so few columns), so nothing else changes.
// Per row r, token m:
//   y[r][m] = sum_g 512 s[r][g] * ( 2^-e(m,g) * sum_i acc_i[r][m]  -  z[r][g] * 2^-9 sx[m][g] ),
//   acc_i = sum_{c in g} (q[r][c] 2^-9) t_i[c][m],   sx = sum_{c in g} x[m][c]
// with the scale, the zero point and the power of two applied in 32 bits when a group's sums leave tensor memory:
// neither weights nor activations are rounded (but for the bound above), and that work is per token and group, not per
// weight. (Expanding to 16-bit operands instead was built first: exact integers q - zero in bf16 / fp16. It ran at
// 1.5 TB/s: three times the instructions per weight, twice the tensor-memory traffic, twice the MMAs.)
//
// Path of a weight: HBM -> shared memory by TMA (packed, 128 rows x 128 bytes = 256 columns per tile, two tiles a
// unit) -> registers of the thread that owns its row -> tensor memory (tcgen05.st), from which the MMA takes its A
// operand (128 weight rows; the tokens' terms are the N dimension). Shared memory carries only packed weights.
//
// Kernels of a product: w4_split_kernel (terms, powers of two and group sums of the activations, a few microseconds of
// latency that hide behind the weight stream's start), then w4_stream_kernel.
// Warps of w4_stream_kernel: 0 streams weights (TMA), 1 issues MMA, 2 streams activation terms (TMA), 3 streams scales
// and zeros (4-byte cp.async: their rows have no alignment), 4..11 expand (four per tile, thread = row), then 4 (8 for
// 64 tokens) accumulate and run the epilogue. Everything between two roles is a ring with full / empty barriers.
//
// Work split: stream-K over units of (two row tiles, 256 columns) as in few_token.cuh.
#pragma once
#include "few_token.cuh"
#include <cuda_fp8.h>

namespace gmlp {

constexpr int W4_TILE_BYTES = 16384;  // 128 rows x 128 bytes: 256 columns
constexpr int W4_UNIT_COLS = 256;
constexpr int W4_HALF_COLS = 128;

// Terms per activation and N of the MMA for MT token columns (a multiple of 16).
template <typename T>
__host__ __device__ constexpr int w4_terms() {
  return 2;
}
template <>
__host__ __device__ constexpr int w4_terms<__half>() {
  return 3;
}
template <int MT, int TERMS>
__host__ __device__ constexpr int w4_n() {
  return (MT * TERMS + 15) / 16 * 16;
}

// ---- activations -> terms ----
// x [R][cols] (row pitch ldx) -> t8 [TERMS][R][cols] e4m3 bytes, inside every 8 columns in the order in which
// the masks of expand_word deliver a word's nibbles, and meta [R / M][cols / G][2][MT] floats: 2^-e, 2^-9 * sum.
// 16 lanes take the 128 columns of a half unit (8 each); a group is 4, 8 or 16 lanes.
struct W4SplitArgs {
  const void* x;
  long long ldx;
  long long R;  // rows: M, or active experts * M
  int M, MT, cols, gshift;
  uint8_t* t8;
  float* meta;
  int dependent;
};
constexpr int W4_SPLIT_THREADS = 256;

template <typename T>
__global__ void __launch_bounds__(W4_SPLIT_THREADS)
w4_split_kernel(const W4SplitArgs args) {
  constexpr int TERMS = w4_terms<T>();
  pdl_launch_dependents();
  if (args.dependent) pdl_wait();
  const int lane = threadIdx.x & 31, sub = lane & 15;
  const int blocks = (args.cols + W4_HALF_COLS - 1) / W4_HALF_COLS;  // 128-column blocks of a row
  const long long items = args.R * blocks;
  const long long item = (blockIdx.x * (W4_SPLIT_THREADS / 32LL) + (threadIdx.x >> 5)) * 2 + (lane >> 4);
  const long long row = item / blocks;
  const int col = static_cast<int>(item - row * blocks) * W4_HALF_COLS + sub * 8;
  const bool live = item < items && col < args.cols;
  float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (live) load8(static_cast<const T*>(args.x) + row * args.ldx + col, v);
  float amax = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    amax = fmaxf(amax, fabsf(v[i]));
    bad |= !(fabsf(v[i]) < INFINITY);
  }
  const int width = 4 << args.gshift;  // lanes per group
  for (int o = 1; o < width; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  // 2^e: the largest value goes to [128, 256). e is limited so that 2^e and 2^-e are normal numbers.
  int ex = 7 - (static_cast<int>((__float_as_uint(amax) >> 23) & 255u) - 127);
  ex = ex > 120 ? 120 : ex;
  const float up = __uint_as_float(static_cast<uint32_t>(127 + ex) << 23);
  const float down = __uint_as_float(static_cast<uint32_t>(127 - ex) << 23);
  float rest[8];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = v[i] * up;
#pragma unroll
  for (int t = 0; t < TERMS; ++t) {
    uint32_t code[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __nv_fp8_storage_t c = __nv_cvt_float_to_fp8(rest[i], __NV_SATFINITE, __NV_E4M3);
      const float back = __half2float(__half(__nv_cvt_fp8_to_halfraw(c, __NV_E4M3)));
      rest[i] -= back;
      sum += back;
      code[i] = c;
    }
    // bytes in the order of the nibbles: columns 0 4 1 5 | 2 6 3 7
    const uint32_t lo = code[0] | (code[4] << 8) | (code[1] << 16) | (code[5] << 24);
    const uint32_t hi = code[2] | (code[6] << 8) | (code[3] << 16) | (code[7] << 24);
    if (live) *reinterpret_cast<uint2*>(args.t8 + (t * args.R + row) * args.cols + col) = make_uint2(lo, hi);
  }
  if (bad) sum = __uint_as_float(0x7fc00000u);  // a non-finite activation: the token's outputs become NaN
  for (int o = 1; o < width; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (live && (sub & (width - 1)) == 0) {
    const long long a = row / args.M, m = row - a * args.M;
    const int groups = args.cols >> (5 + args.gshift);
    const long long g = col >> (5 + args.gshift);
    float* const p = args.meta + ((a * groups + g) * 2) * args.MT + m;
    p[0] = sum != sum ? sum : down;
    p[args.MT] = sum * down * 0.001953125f;
  }
}

// ---- the stream ----
struct W4Args {
  int M;
  int rows;        // weight rows per expert (N for DUAL, outputs otherwise)
  int kbt;         // units along an expert's columns: ceil(cols / 256)
  int groups;      // cols / G
  int gshift;      // log2(G / 32): 0, 1, 2
  int gpg;         // groups per accumulator buffer (1, 2, 4): as many of a half unit as fit 128 columns
  int acc_bufs;    // accumulator buffers of gpg * N columns
  long long R;     // rows of a plane of activation terms
  uint32_t idesc;
  int* status;
  const float* meta;     // [experts in h or 1][groups][2][MT]
  const uint16_t* scale0;  // [experts][groups][rows], T
  const uint16_t* scale1;  // DUAL: the up matrix's
  const uint8_t* zero0;  // [experts][groups][rows] or null (8)
  const uint8_t* zero1;
  const void* bias0;     // [rows] or null
  const void* bias1;
  const void* residual;  // [M][rows] or null (DUAL = false)
  void* out;             // [M][rows]; DUAL on experts: [active][M][rows]
  float* slots;
  int* counters;
  int act;
  int early;  // the weights may be streamed before the preceding kernel has finished
  MoeTable moe;
};

template <int MT, int TERMS>
struct W4Conf {
  static constexpr int N = w4_n<MT, TERMS>();
  static constexpr int ACC_WARPS = MT == 64 ? 8 : 4;
  static constexpr int THREADS = 32 * (12 + ACC_WARPS);
  static constexpr int COLS = MT == 64 ? 32 : MT;  // tokens per accumulator thread
  static constexpr int X_TILE = N * 128;           // terms of a half unit: N rows of 128 columns
  static constexpr int X_STAGE = X_TILE + 4 * 2 * MT * 4;  // + meta of up to four groups, rounded to 1 KB
  static constexpr int X_STAGE_AL = (X_STAGE + 1023) / 1024 * 1024;
  static constexpr int X_STAGES = 4;
  static constexpr int M_BYTES = 12800;  // scales and zeros: four half units at G = 32, sixteen at G = 128
  static constexpr int LEFT = 232448 - 1024 - 4096 - X_STAGES * X_STAGE_AL - M_BYTES;
  static constexpr int W_STAGES = LEFT / (2 * W4_TILE_BYTES) > 5 ? 5 : LEFT / (2 * W4_TILE_BYTES);
  static constexpr size_t SMEM = 1024 + static_cast<size_t>(W_STAGES) * 2 * W4_TILE_BYTES + X_STAGES * X_STAGE_AL + M_BYTES;
  // tensor memory: accumulators in front, expanded weights (64 columns per half unit) behind
  static constexpr int A_BUFS = N > 128 ? 2 : 4;
  static constexpr int C_COLS = 512 - A_BUFS * 64;
  static constexpr int MAX_ACC_BUFS = 8;
  static_assert(W_STAGES >= 3, "ring too shallow");
};
constexpr int W4_META_ROW = 400;  // 66 words of scales, 34 words of zeros of one (tile, group)

// ---- tensor memory and MMA ----
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem], e4m3: A is 128 lanes x 8 columns, four elements a column (32 of the reduction).
__device__ __forceinline__ void umma_f8_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Untiled bulk copy (16-byte aligned, a multiple of 16 bytes), completion on `bar`.
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(src)), "r"(bytes), "r"(bar)
      : "memory");
}
// `bytes` (1..4) of a 4-byte word, the rest zero.
__device__ __forceinline__ void cp_async_word(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// Arrives on `bar` when this thread's cp.asyncs so far have landed (the barrier counts the thread from the start).
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint4 ld_shared_u4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared_u16(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t ld_shared_u8(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
  return v;
}

// Bounded wait of a whole warp (or of one thread, WARP = false) that polls without the suspend hint of mbar_wait: the
// hand-over from warp to warp takes 125 clocks instead of 213 (measured), and these roles hand over every few
// hundred clocks.
template <bool WARP>
__device__ __forceinline__ bool quick_wait(uint32_t bar, uint32_t parity, volatile int* abortp) {
  long long t0 = 0;
  for (int i = 0;; ++i) {
    const bool ok = mbar_try_wait(bar, parity);
    if (WARP ? __all_sync(0xffffffffu, ok) : ok) return true;
    if ((i & 63) == 63) {
      const long long t = clock64();
      if (t0 == 0) t0 = t;
      const bool stop = *abortp != 0 || t - t0 > WAIT_LIMIT_CYCLES;
      if (WARP ? __any_sync(0xffffffffu, stop) : stop) return false;
    }
  }
}

// Ring position: index and the parity of its phase.
struct Ring {
  int at = 0;
  uint32_t phase = 0;
  __device__ __forceinline__ void next(int n) {
    if (++at == n) {
      at = 0;
      phase ^= 1u;
    }
  }
};

// Walks the units of a CTA: position inside the list of active experts (a) and along an expert's columns (kb).
struct W4Walk {
  long long left;  // units of the current row tile from here on (of all CTAs)
  long long tile;
  int a, kb, row0;
};

template <int MT, bool DUAL, typename T>
__global__ void __launch_bounds__(W4Conf<MT, w4_terms<T>()>::THREADS, 1)
w4_stream_kernel(const __grid_constant__ CUtensorMap tmW0, const __grid_constant__ CUtensorMap tmW1,
                 const __grid_constant__ CUtensorMap tmX, const W4Args args) {
  constexpr int TERMS = w4_terms<T>();
  using C = W4Conf<MT, TERMS>;
  constexpr int N = C::N, COLS = C::COLS, ACC_WARPS = C::ACC_WARPS, ACC_THREADS = 32 * ACC_WARPS;
  constexpr int NW = C::W_STAGES, NX = C::X_STAGES, NA = C::A_BUFS, MAXC = C::MAX_ACC_BUFS;
  constexpr int ROWS = DUAL ? 128 : 256;  // weight rows per row tile
  constexpr int NM_MAX = 16;

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * NW + 2 * NX + 2 * NM_MAX + 2 * NA + 2 * MAXC + 1];
  __shared__ uint32_t tmem_base_holder;
  __shared__ int abort_flag;
  __shared__ MoeShared moe;

  const uint32_t w_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t x_base = w_base + NW * 2 * W4_TILE_BYTES;
  const uint32_t m_base = x_base + NX * C::X_STAGE_AL;
  uint32_t b_at = smem_u32(bars);
  const uint32_t wfull = b_at, wempty = wfull + 8 * NW, xfull = wempty + 8 * NW, xempty = xfull + 8 * NX,
                 mfull = xempty + 8 * NX, mempty = mfull + 8 * NM_MAX, afull = mempty + 8 * NM_MAX,
                 aempty = afull + 8 * NA, cfull = aempty + 8 * NA, cempty = cfull + 8 * MAXC,
                 drain_bar = cempty + 8 * MAXC;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int gph = 4 >> args.gshift;        // groups per half unit
  const int gpu_ = 2 * gph;                // groups per unit
  const int nm = 16 / gph;                 // ring of scales and zeros, in half units
  const uint32_t m_stage = 2 * gph * W4_META_ROW;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < NW; ++s) {
      mbar_init(wfull + 8 * s, 1);
      mbar_init(wempty + 8 * s, 8);
    }
    for (int s = 0; s < NX; ++s) {
      mbar_init(xfull + 8 * s, 1);
      mbar_init(xempty + 8 * s, 1 + ACC_WARPS);
    }
    for (int s = 0; s < NM_MAX; ++s) {
      mbar_init(mfull + 8 * s, 32);
      mbar_init(mempty + 8 * s, ACC_WARPS);
    }
    for (int b = 0; b < NA; ++b) {
      mbar_init(afull + 8 * b, 8);
      mbar_init(aempty + 8 * b, 1);
    }
    for (int b = 0; b < MAXC; ++b) {
      mbar_init(cfull + 8 * b, 1);
      mbar_init(cempty + 8 * b, ACC_WARPS);
    }
    mbar_init(drain_bar, 1);
    mbar_fence_init();
    fence_proxy_async_smem();
    tma_prefetch_desc(&tmW0);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_base_holder), 512);
    tmem_relinquish();
  }
  const bool is_moe = args.moe.ids != nullptr;
  // The routing table comes from an earlier kernel. The gate/up kernel waits for that kernel before it lets its own
  // dependent start, so the down kernel may read the table (and stream weights) at once.
  if (!args.early) pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  tc_fence_before_sync();
  moe_collect(args.moe, args.M, moe);  // ends with a block barrier
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_holder;
  volatile int* const abortp = &abort_flag;

  // Units: DUAL: tile = (expert, row tile), kbt units each. Else: tile = row tile, units = (expert, kb).
  const int row_tiles = (args.rows + ROWS - 1) / ROWS;
  const long long per_tile = DUAL ? args.kbt : static_cast<long long>(moe.n) * args.kbt;
  const long long total = per_tile * (DUAL ? static_cast<long long>(moe.n) * row_tiles : row_tiles);
  const long long ctas = total < gridDim.x ? total : gridDim.x;
  const long long u_begin = blockIdx.x < ctas ? unit_start(blockIdx.x, total, ctas) : 0;
  const long long u_end = blockIdx.x < ctas ? unit_start(blockIdx.x + 1, total, ctas) : 0;

  auto enter = [&](W4Walk& w, long long tile, long long r) {  // unit r of the tile
    w.tile = tile;
    w.left = per_tile - r;
    if (DUAL) {
      w.a = static_cast<int>(tile / row_tiles);
      w.row0 = static_cast<int>(tile - static_cast<long long>(w.a) * row_tiles) * ROWS;
      w.kb = static_cast<int>(r);
    } else {
      w.row0 = static_cast<int>(tile) * ROWS;
      w.a = static_cast<int>(r / args.kbt);
      w.kb = static_cast<int>(r - static_cast<long long>(w.a) * args.kbt);
    }
  };
  auto start = [&](W4Walk& w) {
    if (u_begin < u_end) {
      const long long tile = u_begin / per_tile;
      enter(w, tile, u_begin - tile * per_tile);
    }
  };
  auto step = [&](W4Walk& w) {
    if (--w.left == 0) {
      enter(w, w.tile + 1, 0);
    } else if (++w.kb == args.kbt) {
      w.kb = 0;
      ++w.a;
    }
  };
  auto groups_in = [&](int kb, int half) {  // groups of a half unit that exist
    const int left = args.groups - kb * gpu_ - half * gph;
    return left < gph ? left : gph;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ weights --
    if (lane == 0) {
      const uint64_t pol = l2_policy_evict_first();
      W4Walk w;
      start(w);
      Ring r;
      long long u = u_begin;
      bool ok = true;
      for (; u < u_end; ++u) {
        if (!(ok = quick_wait<false>(wempty + 8 * r.at, r.phase ^ 1u, abortp))) break;
        const uint32_t dst = w_base + r.at * 2 * W4_TILE_BYTES, fb = wfull + 8 * r.at;
        const int y = moe.list[w.a] * args.rows + w.row0;
        mbar_expect_tx(fb, 2 * W4_TILE_BYTES);
        tma_load_2d_hint(dst, &tmW0, fb, w.kb * 128, y, pol);
        if (DUAL)
          tma_load_2d_hint(dst + W4_TILE_BYTES, &tmW1, fb, w.kb * 128, y, pol);
        else
          tma_load_2d_hint(dst + W4_TILE_BYTES, &tmW0, fb, w.kb * 128, y + 128, pol);
        step(w);
        r.next(NW);
      }
      if (!ok) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_PRODUCER);
        const long long done = u - u_begin;  // see the copies in flight land before the block leaves
        for (long long i = done > NW ? done - NW : 0; i < done; ++i)
          drain_wait(wfull + 8 * static_cast<int>(i % NW), static_cast<uint32_t>(i / NW) & 1u);
      }
    }
  } else if (warp == 2) {
    // -------------------------------------------------------- activations --
    if (lane == 0) {
      if (args.early) pdl_wait();
      const uint64_t pol = l2_policy_evict_last();
      W4Walk w;
      start(w);
      Ring r;
      bool ok = true;
      long long done = 0;
      for (long long u = u_begin; u < u_end && ok; ++u) {
        const int a = DUAL ? 0 : w.a;
        for (int h = 0; h < 2; ++h) {
          const int ng = groups_in(w.kb, h);
          if (ng <= 0) break;
          if (!(ok = quick_wait<false>(xempty + 8 * r.at, r.phase ^ 1u, abortp))) break;
          const uint32_t dst = x_base + r.at * C::X_STAGE_AL, fb = xfull + 8 * r.at;
          const uint32_t meta_bytes = ng * 2 * MT * 4;
          mbar_expect_tx(fb, TERMS * MT * 128 + meta_bytes);
#pragma unroll
          for (int t = 0; t < TERMS; ++t)
            tma_load_2d_hint(dst + t * MT * 128, &tmX, fb, w.kb * W4_UNIT_COLS + h * W4_HALF_COLS,
                             static_cast<int>(t * args.R) + a * args.M, pol);
          bulk_load(dst + C::X_TILE,
                    args.meta + (static_cast<long long>(a) * args.groups + w.kb * gpu_ + h * gph) * 2 * MT, meta_bytes, fb);
          r.next(NX);
          ++done;
        }
        step(w);
      }
      if (!ok) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_PRODUCER);
        for (long long i = done > NX ? done - NX : 0; i < done; ++i)
          drain_wait(xfull + 8 * static_cast<int>(i % NX), static_cast<uint32_t>(i / NX) & 1u);
      }
    }
  } else if (warp == 3) {
    // --------------------------------------------------- scales and zeros --
    W4Walk w;
    start(w);
    Ring r;
    bool ok = true;
    for (long long u = u_begin; u < u_end && ok; ++u) {
      for (int h = 0; h < 2; ++h) {
        const int ng = groups_in(w.kb, h);
        if (ng <= 0) break;
        if (!(ok = quick_wait<true>(mempty + 8 * r.at, r.phase ^ 1u, abortp))) break;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const uint16_t* const sc = (DUAL && t == 1) ? args.scale1 : args.scale0;
          const uint8_t* const ze = (DUAL && t == 1) ? args.zero1 : args.zero0;
          const int row = w.row0 + (DUAL ? 0 : t * 128);
          const int nrow = args.rows - row < 128 ? args.rows - row : 128;
          if (nrow <= 0) continue;
          for (int i = 0; i < ng; ++i) {
            const long long e0 =
                (static_cast<long long>(moe.list[w.a]) * args.groups + w.kb * gpu_ + h * gph + i) * args.rows + row;
            const uint32_t dst = m_base + r.at * m_stage + (t * gph + i) * W4_META_ROW;
            // words that hold rows row .. row + nrow - 1; the last one only as far as the rows go
            const int head = static_cast<int>(e0 & 1) * 2, bytes = head + 2 * nrow;
            const char* const s0 = reinterpret_cast<const char*>(sc + e0) - head;
            for (int k = lane * 4; k < bytes; k += 128)
              cp_async_word(dst + k, s0 + k, bytes - k < 4 ? bytes - k : 4);
            if (ze != nullptr) {
              const int zhead = static_cast<int>(e0 & 3), zbytes = zhead + nrow;
              const uint8_t* const z0 = ze + e0 - zhead;
              for (int k = lane * 4; k < zbytes; k += 128)
                cp_async_word(dst + 264 + k, z0 + k, zbytes - k < 4 ? zbytes - k : 4);
            }
          }
        }
        cp_async_arrive(mfull + 8 * r.at);
        r.next(nm);
      }
      step(w);
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_PRODUCER);
    }
    cp_async_wait_all();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA --
    if (lane == 0) {
      W4Walk w;
      start(w);
      Ring rx, ra, rc;
      const int ksteps = 1 << args.gshift;  // 32-column steps per group
      const uint32_t c_cols = args.gpg * N;
      bool ok = true;
      for (long long u = u_begin; u < u_end && ok; ++u) {
        for (int h = 0; h < 2 && ok; ++h) {
          const int ng = groups_in(w.kb, h);
          if (ng <= 0) break;
          if (!(ok = quick_wait<false>(xfull + 8 * rx.at, rx.phase, abortp))) break;
          if (!(ok = quick_wait<false>(afull + 8 * ra.at, ra.phase, abortp))) break;
          const uint64_t xd = make_smem_desc(x_base + rx.at * C::X_STAGE_AL, 16, 1024);
          const uint32_t a0 = tmem_base + C::C_COLS + ra.at * 64;
          for (int t = 0; t < 2 && ok; ++t) {
            for (int g0 = 0; g0 < ng; g0 += args.gpg) {
              if (!(ok = quick_wait<false>(cempty + 8 * rc.at, rc.phase ^ 1u, abortp))) break;
              tc_fence_after_sync();
              const int ge = g0 + args.gpg < ng ? g0 + args.gpg : ng;
              uint32_t d = tmem_base + rc.at * c_cols;
              for (int g = g0; g < ge; ++g, d += N) {
                const int k0 = g * ksteps;
                for (int k = 0; k < ksteps; ++k)
                  umma_f8_ts(d, a0 + t * 32 + (k0 + k) * 8, xd + static_cast<uint64_t>(2 * (k0 + k)), args.idesc,
                             k > 0 ? 1u : 0u);
              }
              umma_commit(cfull + 8 * rc.at);
              rc.next(args.acc_bufs);
            }
          }
          if (!ok) break;
          umma_commit(aempty + 8 * ra.at);
          umma_commit(xempty + 8 * rx.at);
          ra.next(NA);
          rx.next(NX);
        }
        step(w);
      }
      if (!ok) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_MMA);
        umma_commit(drain_bar);
        drain_wait(drain_bar, 0);
      }
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------- expand --
    const int quarter = warp & 3;
    const int tsel = (warp - 4) >> 2;  // which of the unit's two tiles
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    W4Walk w;
    start(w);
    Ring rw, ra;
    bool ok = true;
    for (long long u = u_begin; u < u_end && ok; ++u) {
      if (!(ok = quick_wait<true>(wfull + 8 * rw.at, rw.phase, abortp))) break;
      const uint32_t src = w_base + rw.at * 2 * W4_TILE_BYTES + tsel * W4_TILE_BYTES + row * 128;
      const int halves = groups_in(w.kb, 1) > 0 ? 2 : 1;
      for (int h = 0; h < halves; ++h) {
        uint4 q[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) q[c] = ld_shared_u4(src + (((h * 4 + c) ^ (row & 7)) << 4));
        uint32_t r[32];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t word[4] = {q[c].x, q[c].y, q[c].z, q[c].w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            r[c * 8 + 2 * i] = word[i] & 0x0F0F0F0Fu;
            r[c * 8 + 2 * i + 1] = (word[i] >> 4) & 0x0F0F0F0Fu;
          }
        }
        if (!(ok = quick_wait<true>(aempty + 8 * ra.at, ra.phase ^ 1u, abortp))) break;
        if (h == halves - 1 && lane == 0) mbar_arrive(wempty + 8 * rw.at);  // the packed weights are in registers
        tc_fence_after_sync();
        tmem_st_32x32(tmem_base + lane_addr + C::C_COLS + ra.at * 64 + tsel * 32, r);
        tmem_st_wait();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(afull + 8 * ra.at);
        ra.next(NA);
      }
      rw.next(NW);
      step(w);
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_MMA);
    }
  } else {
    // ------------------------------------------- accumulate and finish --
    constexpr int CH = COLS < 16 ? COLS : 16;  // token columns per tensor-memory load
    const int quarter = warp & 3;
    const int col0 = ((warp - 12) >> 2) * COLS;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int ep_tid = threadIdx.x - 384;
    const uint32_t c_cols = args.gpg * N;
    if (args.early) pdl_wait();  // slots, counters and outputs may still be in use
    if (!DUAL && total == 0) {
      // no token chose any expert: the outputs are the residual, or zero
      const long long all = static_cast<long long>(args.M) * args.rows;
      for (long long i = blockIdx.x * static_cast<long long>(ACC_THREADS) + ep_tid; i < all;
           i += static_cast<long long>(gridDim.x) * ACC_THREADS)
        static_cast<T*>(args.out)[i] =
            args.residual ? static_cast<const T*>(args.residual)[i] : static_cast<T>(0.f);
    }
    W4Walk w;
    start(w);
    Ring rx, rm, rc;
    long long u = u_begin;
    while (u < u_end) {
      const Segment s = segment_at(u, u_end, per_tile);
      const int a = DUAL ? w.a : 0;
      const int r0 = w.row0 + row, r1 = DUAL ? r0 : r0 + 128;
      f32x2 v[2][COLS / 2];
#pragma unroll
      for (int c = 0; c < COLS / 2; ++c) v[0][c] = v[1][c] = 0ull;
      bool ok = true;
      for (; u < s.end && ok; ++u) {
        for (int h = 0; h < 2 && ok; ++h) {
          const int ng = groups_in(w.kb, h);
          if (ng <= 0) break;
          if (!(ok = quick_wait<true>(mfull + 8 * rm.at, rm.phase, abortp))) break;
          if (!(ok = quick_wait<true>(xfull + 8 * rx.at, rx.phase, abortp))) break;
          const uint32_t xm = x_base + rx.at * C::X_STAGE_AL + C::X_TILE + col0 * 4;
          const uint32_t mm = m_base + rm.at * m_stage;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const bool zeros = ((DUAL && t == 1) ? args.zero1 : args.zero0) != nullptr;
            for (int g0 = 0; g0 < ng && ok; g0 += args.gpg) {
              if (!(ok = quick_wait<true>(cfull + 8 * rc.at, rc.phase, abortp))) break;
              tc_fence_after_sync();
              const int ge = g0 + args.gpg < ng ? g0 + args.gpg : ng;
              uint32_t src = tmem_base + lane_addr + rc.at * c_cols + col0;
              for (int g = g0; g < ge; ++g, src += N) {
                const long long e0 = (static_cast<long long>(moe.list[w.a]) * args.groups + w.kb * gpu_ + h * gph + g) *
                                         args.rows + (w.row0 + (DUAL ? 0 : t * 128));
                const uint32_t mr = mm + (t * gph + g) * W4_META_ROW;
                const uint32_t sbits = ld_shared_u16(mr + static_cast<uint32_t>(e0 & 1) * 2 + row * 2);
                const float sc = 512.0f * Pack2<T>::unpack(sbits).x;
                const float z = zeros ? static_cast<float>(ld_shared_u8(mr + 264 + static_cast<uint32_t>(e0 & 3) + row) & 15u)
                                      : 8.0f;
                const f32x2 s2 = f2_pack(sc, sc), z2 = f2_pack(-z, -z);
#pragma unroll
                for (int c = 0; c < COLS; c += CH) {
                  uint32_t x[TERMS][CH];
#pragma unroll
                  for (int i = 0; i < TERMS; ++i)
#pragma unroll
                    for (int k = 0; k < CH; k += 8) tmem_ld_32x8(src + i * MT + c + k, &x[i][k]);
                  tmem_ld_wait();
#pragma unroll
                  for (int k = 0; k < CH; k += 4) {
                    const float4 p = ld_shared_f4(xm + g * 2 * MT * 4 + (c + k) * 4);
                    const float4 q = ld_shared_f4(xm + g * 2 * MT * 4 + MT * 4 + (c + k) * 4);
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                      const int o = k + 2 * j;
                      f32x2 y = f2_add(f2_pack(__uint_as_float(x[0][o]), __uint_as_float(x[0][o + 1])),
                                       f2_pack(__uint_as_float(x[1][o]), __uint_as_float(x[1][o + 1])));
                      if (TERMS == 3)
                        y = f2_add(y, f2_pack(__uint_as_float(x[TERMS - 1][o]), __uint_as_float(x[TERMS - 1][o + 1])));
                      y = f2_mul(y, j == 0 ? f2_pack(p.x, p.y) : f2_pack(p.z, p.w));
                      y = f2_fma(z2, j == 0 ? f2_pack(q.x, q.y) : f2_pack(q.z, q.w), y);
                      v[t][(c + o) / 2] = f2_fma(s2, y, v[t][(c + o) / 2]);
                    }
                  }
                }
              }
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive(cempty + 8 * rc.at);
              rc.next(args.acc_bufs);
            }
          }
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive(mempty + 8 * rm.at);
            mbar_arrive(xempty + 8 * rx.at);
          }
          rm.next(nm);
          rx.next(NX);
        }
        step(w);
      }
      if (!ok && lane == 0) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_EPILOGUE);
      }
      float f[2][COLS];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int c = 0; c < COLS / 2; ++c) f2_unpack(v[t][c], f[t][2 * c], f[t][2 * c + 1]);
      if (DUAL && is_moe) moe_factors(args.moe, args.M, moe.list[a], ep_tid, moe);  // seen behind the next barrier
      const Split sp{total,       ctas,   args.slots, args.counters,
                     args.status, abortp, w_base,     NW * 2 * W4_TILE_BYTES / (ACC_THREADS * 16)};
      const int what = settle_segment<2, COLS, MT, ACC_THREADS>(f, s, sp, args.M, col0, row, ep_tid);
      if (what == SETTLE_ABORT) break;
      if (what == SETTLE_EMIT) {
        const MoeShared* const mp = is_moe ? &moe : nullptr;
        T* const out = static_cast<T*>(args.out);
        const T* const b0 = static_cast<const T*>(args.bias0);
        const T* const b1 = static_cast<const T*>(args.bias1);
        const T* const res = static_cast<const T*>(args.residual);
        const long long ld = args.rows;
        if (DUAL) {
          if (r0 < args.rows)
            store_hidden<COLS>(args.act, out + static_cast<long long>(a) * args.M * ld + r0, ld, args.M, col0, f[0],
                               f[1], b0 ? static_cast<float>(b0[r0]) : 0.f, b1 ? static_cast<float>(b1[r0]) : 0.f, mp);
        } else {
          if (r0 < args.rows)
            store_product<COLS>(out + r0, res ? res + r0 : nullptr, ld, args.M, col0, f[0],
                                b0 ? static_cast<float>(b0[r0]) : 0.f, mp);
          if (r1 < args.rows)
            store_product<COLS>(out + r1, res ? res + r1 : nullptr, ld, args.M, col0, f[1],
                                b0 ? static_cast<float>(b0[r1]) : 0.f, mp);
        }
      }
      if (DUAL && is_moe) named_bar_sync(1, ACC_THREADS);  // f and hit are overwritten for the next tile
    }
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, 512);
  }
}

}  // namespace gmlp
