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
// 2. An activation is a short sum of 8-bit floats. e5m2 has 3 significant bits and each rounding to the nearest saves one
//    more: three terms carry 3 + 4 + 4 = 11, as many as fp16 has (bf16: 8). With a power of two that brings the largest
//    value of a block of activations to [2^14, 2^15),
//      x 2^e = t_1 + t_2 + t_3,   t_i the e5m2 rounding of what is left.
//    That is exact for values within 2^-23 (bf16) or 2^-20 (fp16) of the block's largest; below, the error is at most
//    2^-17 (half the spacing of e5m2's subnormals) where the largest is at least 2^14: 2^-31 of the block's largest
//    value, below what 32-bit sums keep. (e4m3 terms, two of them for bf16, have a floor of 2^-17 of the largest: with an
//    activation of 16384 among normal ones, outputs that it does not reach were off by 8e-2.)
//    The terms are MMAs into one accumulator (the tensor pipe has the time: an MMA of N <= 64 columns takes N / 2 clocks, at
//    least 16, and the weights of one arrive every 89).
//    The block: up to 4 tokens, a token and group (terms made inside the kernel, unit by unit); above, a whole token.
// Per row r, token m:
//   y[r][m] = sum_g 512 s[r][g] * ( acc[r][m]  -  z[r][g] * sx[m][g] ) * 2^-e,
//   acc = sum_i sum_{c in g} (q[r][c] 2^-9) t_i[c][m],   sx = 2^-9 sum_{c in g} sum_i t_i[c][m]
// with the scale, the zero point and the power of two applied in 32 bits when a group's sums leave tensor memory:
// neither weights nor activations are rounded (but for the bound above), and that work is per token and group, not per
// weight: three operations per token and group while 2^-e belongs to the group, two when it belongs to the token. That
// is why it does from 5 tokens on: those operations, and fetching sx and 2^-e, are what 64 tokens wait for.
// (Expanding to 16-bit operands instead was built first: exact integers q - zero in bf16 / fp16. It ran at
// 1.5 TB/s: three times the instructions per weight, twice the tensor-memory traffic, twice the MMAs.)
//
// Path of a weight: HBM -> shared memory by TMA (packed, 128 rows x 128 bytes = 256 columns per tile, two tiles a
// unit) -> registers of the thread that owns its row -> tensor memory (tcgen05.st), from which the MMA takes its A
// operand (128 weight rows; the tokens' terms are the N dimension). Shared memory carries only packed weights.
//
// Kernels of a product: w4_stream_kernel; from 5 tokens on w4_split_kernel before it (terms, powers of two and group sums of
// the activations, a few microseconds of latency that hide behind the weight stream's start).
// Warps of w4_stream_kernel: 0 streams weights (TMA), 1 issues MMA, 2 streams activation terms, scales and zeros (TMA), 3
// packs scales and zeros, 4..11 expand (four per tile, thread = row), 12..19 take the sums
// and run the epilogue (thread = a row of both tiles; up to 4 tokens 12..15, and 16..19 make activation terms; up to 32 tokens
// four warps per half of the tokens, 64 tokens four per quarter). Everything between two roles is a ring with full / empty barriers, and
// every ring turns once a unit (65,536 weights, 1,400 clocks at the copy bandwidth): a role that is one thread or one warp
// executes an instruction every 5 to 10 clocks, so its instructions per unit are counted, and the group size is a template
// parameter to keep them straight-line. (With hand-overs per 128 columns and run-time group loops the thread that
// issues the MMAs was itself the bound, at 3,000 clocks per 32,768 weights.)
//
// Work split: stream-K over units of (two row tiles, 256 columns) as in few_token.cuh.
//
// Measured (one B200, replayed from a graph, G = 128): gated MLP K=8192, N=28672 of one token 71 us = 5.2 TB/s of the packed
// bytes (the copy rate is 6.56), 8 tokens 83, 16 tokens 88, 32 tokens 111, 64 tokens 168 (G = 64: 235, G = 32: 463);
// product 131072 x 4096, 8 tokens 60 us; 4096 x 4096, one token 8.7 us, of which 7 are the life of a block from its start to
// its join. Of an MLP's time 16 us (one token) to 33 (64 tokens) do not grow with N: starts, joins and the terms. Up to 16
// tokens HBM bounds the rest. Above, the accumulating warps do: two instructions per two (row, token) sums of a group,
// and the trip of the sums through tensor memory (at 64 tokens 55 % of the issue slots, 41 % of the tensor pipe, 29 % of
// HBM). Fetching a group's sums while those of the group before are worked on was slower (64 tokens: 164 us against 158 with
// two terms; that third term costs bf16 9 us at 64 tokens and nothing measurable up to 32).
#pragma once
#include <cuda_fp8.h>

#include "few_token.cuh"

namespace gmlp {

constexpr int W4_TILE_BYTES = 16384;  // 128 rows x 128 bytes: 256 columns
constexpr int W4_UNIT_COLS = 256;
constexpr int W4_HALF_COLS = 128;
// Of one CTA, whether or not the others stream: what its weights take to arrive. Measured at 3 and 5 tokens; many tokens take
// longer to accumulate (64 tokens with G = 128 / 64 / 32: about 3,900 / 5,500 / 10,800 clocks, from the times above), so that
// a short tile of theirs stays whole (see cut_grain) where cutting it would leave fewer SMs idle.
constexpr int W4_UNIT_CLOCKS = 1400;

constexpr int W4_TERMS = 3;  // per activation

// ---- activations -> terms ----
// The power of two, as an exponent, that brings `amax` to [2^14, 2^15); limited so that it and its inverse are normal numbers.
__device__ __forceinline__ int split_exponent(float amax) {
  const int ex = 14 - (static_cast<int>((__float_as_uint(amax) >> 23) & 255u) - 127);
  return ex > 120 ? 120 : ex;
}
// What takes the power off again, 2^-e, is applied as 2^(13 - e) and the scales' 512 as 512 * 2^-13: both are then normal
// numbers for every e, and sums of scale * acc stay finite for scales up to 2^106 over 2^16 columns.
constexpr int W4_LIFT = 13;
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }
// Eight columns of a lane times 2^ex: the terms' codes (bytes in the order in which the expanders' masks deliver a word's
// nibbles: columns 0 4 1 5 | 2 6 3 7); returns the sum of the terms.
__device__ __forceinline__ float split_terms(const float (&v)[8], int ex, uint2 (&codes)[W4_TERMS]) {
  constexpr int PERM[8] = {0, 4, 1, 5, 2, 6, 3, 7};
  const float up = power_of_two(ex);
  float rest[8], sum = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = v[i] * up;
#pragma unroll
  for (int t = 0; t < W4_TERMS; ++t) {
    uint32_t pair[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int a = PERM[2 * i], b = PERM[2 * i + 1];
      const __nv_fp8x2_storage_t c = __nv_cvt_float2_to_fp8x2(make_float2(rest[a], rest[b]), __NV_SATFINITE, __NV_E5M2);
      const float2 back = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(c, __NV_E5M2)));
      rest[a] -= back.x;
      rest[b] -= back.y;
      sum += back.x + back.y;
      pair[i] = c;
    }
    codes[t] = make_uint2(pair[0] | (pair[1] << 16), pair[2] | (pair[3] << 16));
  }
  return sum;
}
// Largest magnitude of eight columns; a NaN or an infinity gives NaN, which then belongs in the token's outputs.
__device__ __forceinline__ float amax8(const float (&v)[8]) {
  float amax = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    amax = fmaxf(amax, fabsf(v[i]));
    bad |= !(fabsf(v[i]) < INFINITY);
  }
  return bad ? __uint_as_float(0x7fc00000u) : amax;
}
__device__ __forceinline__ float nan_max(float a, float b) { return (b > a || b != b) ? b : a; }

// x [active][M][cols] (row pitch ldx) -> t8 [W4_TERMS][R][cols] e5m2 bytes, meta [active][groups][MT] floats sx with
// the groups of a row padded to whole units of 256 columns (zeros there), and per token 2^(13 - e) (NaN where the token
// holds a NaN or an infinity). A cluster of blocks per token: each takes a share of the token's half units (128 columns, 16
// lanes of 8; a group is 4, 8 or 16 lanes), finds their largest value, and goes over them again with the token's. Bound by
// latency (launch, two passes, the cluster's barrier), about 5 us before a stream kernel, which starts meanwhile.
struct W4SplitArgs {
  const void* x;
  long long ldx;
  long long R;  // rows of a plane of t8
  int M, MT, cols, gshift;
  uint8_t* t8;
  float* meta;
  float* rowscale;
  int dependent;
  MoeTable moe;
};
// 8 blocks of 512 threads: a thread's eight columns mostly are its only ones and stay in registers (MLP K=8192, N=28672,
// 8 / 16 / 32 tokens: 81 / 89 / 109 us; blocks of 256 threads 85 / 93 / 113, of 1024 threads 81 / 88 / 117).
constexpr int W4_SPLIT_THREADS = 512;
constexpr int W4_SPLIT_CLUSTER = 8;

template <typename T>
__global__ void __launch_bounds__(W4_SPLIT_THREADS)
w4_split_kernel(const W4SplitArgs args) {
  __shared__ MoeShared moe;
  __shared__ float warp_max[W4_SPLIT_THREADS / 32];
  __shared__ float block_max[W4_SPLIT_CLUSTER];
  pdl_launch_dependents();
  cluster_sync_all();  // the other blocks' shared memory is written below: they have to be there
  if (args.dependent) pdl_wait();
  moe_collect(args.moe, args.M, moe);
  const uint32_t rank = cluster_ctarank();
  const int m = blockIdx.x / W4_SPLIT_CLUSTER;
  const int tid = threadIdx.x, lane = tid & 31, sub = lane & 15;
  const int blocks = (args.cols + W4_UNIT_COLS - 1) / W4_UNIT_COLS * 2;  // half units of a row, padded to whole units
  const int items = moe.n * blocks;
  const int lo = static_cast<int>(static_cast<long long>(items) * rank / W4_SPLIT_CLUSTER);
  const int hi = static_cast<int>(static_cast<long long>(items) * (rank + 1) / W4_SPLIT_CLUSTER);
  auto load = [&](int item, float (&v)[8]) {  // true: the lane's columns exist
    const int a = item / blocks, col = (item - a * blocks) * W4_HALF_COLS + sub * 8;
    const bool live = item < hi && col < args.cols;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.f;
    if (live) load8(static_cast<const T*>(args.x) + (static_cast<long long>(a) * args.M + m) * args.ldx + col, v);
    return live;
  };
  float kept[8];  // the first item's columns, mostly the only ones
  const bool kept_live = load(lo + (tid >> 4), kept);
  float amax = amax8(kept);
  for (int item = lo + (tid >> 4) + W4_SPLIT_THREADS / 16; item < hi; item += W4_SPLIT_THREADS / 16) {
    float v[8];
    load(item, v);
    amax = nan_max(amax, amax8(v));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = nan_max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  if (lane == 0) warp_max[tid >> 5] = amax;
  __syncthreads();
  if (tid < W4_SPLIT_CLUSTER) {
    amax = warp_max[0];
#pragma unroll
    for (int i = 1; i < W4_SPLIT_THREADS / 32; ++i) amax = nan_max(amax, warp_max[i]);
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(smem_u32(&block_max[rank]), tid)), "f"(amax)
                 : "memory");
  }
  __syncwarp();
  cluster_sync_all();
  amax = block_max[0];
#pragma unroll
  for (int i = 1; i < W4_SPLIT_CLUSTER; ++i) amax = nan_max(amax, block_max[i]);
  const bool bad = amax != amax;
  const int ex = bad ? 0 : split_exponent(amax);
  if (rank == 0 && tid == 0) args.rowscale[m] = bad ? amax : power_of_two(W4_LIFT - ex);
  const int width = 4 << args.gshift;  // lanes per group
  for (int first = lo; first < hi; first += W4_SPLIT_THREADS / 16) {
    const int item = first + (tid >> 4);
    float v[8];
    bool live = kept_live;
    if (first == lo) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = kept[i];
    } else {
      live = load(item, v);
    }
    uint2 code[W4_TERMS];
    float sum = split_terms(v, ex, code);
    for (int o = 1; o < width; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (item >= hi) continue;
    const int a = item / blocks, col = (item - a * blocks) * W4_HALF_COLS + sub * 8;
    if (live) {
      uint8_t* const p = args.t8 + (static_cast<long long>(a) * args.M + m) * args.cols + col;
#pragma unroll
      for (int t = 0; t < W4_TERMS; ++t) *reinterpret_cast<uint2*>(p + t * args.R * args.cols) = code[t];
    }
    if ((sub & (width - 1)) == 0) {
      const long long g = static_cast<long long>(a) * (blocks * (4 >> args.gshift)) + (col >> (5 + args.gshift));
      args.meta[g * args.MT + m] = sum * 0.001953125f;
    }
  }
}

// ---- the stream ----
struct W4Maps {
  CUtensorMap w0, w1, x;
  CUtensorMap s0, s1, z0, z1;  // scales and zeros, where W4Args::wide
};
struct W4Args {
  int M;
  int rows;        // weight rows per expert (N for DUAL, outputs otherwise)
  int kbt;         // units along an expert's columns: ceil(cols / 256)
  int groups;      // cols / G
  long long R;     // rows of a plane of activation terms
  const void* x;   // FUSED: the activations, [M] or [active * M] rows of pitch ldx
  long long ldx;
  int cols;
  int* status;
  const float* meta;       // not FUSED: [experts in h or 1][kbt * groups per unit][MT] sx
  const float* rowscale;   // not FUSED: [M] 2^(13 - e)
  const uint16_t* scale0;  // [experts][groups][rows], T
  const uint16_t* scale1;  // DUAL: the up matrix's
  const uint8_t* zero0;    // [experts][groups][rows] or null (8)
  const uint8_t* zero1;
  const void* bias0;       // [rows] or null
  const void* bias1;
  const void* residual;    // [M][rows] or null (DUAL = false)
  void* out;               // [M][rows]; DUAL on experts: [active][M][rows]
  float* slots;
  int* counters;
  int act;
  int wide;   // scales and zeros go by TMA: rows are a multiple of 16 and the arrays 16-byte aligned
  int early;  // the weights may be streamed before the preceding kernel has finished
  Cut cut;    // a dense call's; on experts the kernel makes it from the routing table
  MoeTable moe;
};

// Scales and zeros of a unit in shared memory. As TMA boxes (W4Args::wide): [2 tiles][groups][128] scales, then zeros alike.
// As rows: per (tile, group) the 16-byte blocks that the 128 scales lie in (up to 17), from byte 272 on those of the zeros (up
// to 9).
constexpr int W4_META_ROW = 416;
constexpr int W4_META_ZERO = 272;

// FUSED: the terms are made in the kernel, with a power of two per token and group. Four warps make them, each takes a (unit,
// token) pair in turn; a pair takes about 800 clocks, a unit's weights 1,400 to arrive, which carries four tokens (8
// tokens, 28672 x 8192: 85 us, 73 with six such warps, against 50 with the terms made beforehand).
constexpr int W4_FUSED_TOKENS = 4;
template <int MT, int GSHIFT, bool FUSED>
struct W4Conf {
  static_assert(!FUSED || MT == 8, "one instantiation of each fused form");
  // Up to 8 tokens and with groups of 128 the terms are columns of one MMA, which costs the same 16 clocks with 32 columns as
  // with 16, and the accumulating warps add them up; else they are MMAs into one accumulator, since smaller groups have
  // more sums to add up (K=8192, N=28672 MLP without pause, G = 128 / 64 / 32: one token 77 / 109 / 254 us stacked, 85 / 108
  // / 236 not; 8 tokens 91 / 109 / 256 and 93 / 108 / 190).
  static constexpr bool STACKED = MT == 8 && GSHIFT == 2;
  static constexpr int TOK = STACKED && FUSED ? W4_FUSED_TOKENS : MT;  // rows of a term
  static constexpr int N = STACKED ? (W4_TERMS * TOK + 15) / 16 * 16 : MT < 16 ? 16 : MT;  // columns of the MMA
  // accumulating threads: four warps per share of the tokens; 64 tokens take sixteen warps (with eight, 64 sums a thread)
  static constexpr int SHARES = FUSED ? 1 : (MT == 64 ? 4 : 2);
  static constexpr int EPI = 128 * SHARES;
  static constexpr int CONVERTERS = FUSED ? 4 : 0;
  static constexpr int THREADS = 32 * (12 + 4 * SHARES + CONVERTERS);
  static constexpr int GPH = 4 >> GSHIFT;          // groups per half unit (128 columns)
  static constexpr int GPU = 2 * GPH;              // groups per unit
  static constexpr int FACTORS = FUSED ? 2 : 1;    // per token and group: 2^-e (FUSED) and sx
  // activation terms of a unit: [two halves][W4_TERMS] of TOK rows x 128 columns, then [GPU][FACTORS][MT] factors. (Columns
  // of the MMA behind the last term are whatever lies there.)
  static constexpr int X_TERM = TOK * 128;
  static constexpr int X_HALF = (W4_TERMS * X_TERM + 1023) / 1024 * 1024;
  static constexpr int X_STAGE = (2 * X_HALF + GPU * FACTORS * MT * 4 + 1023) / 1024 * 1024;
  static_assert(X_STAGE >= X_HALF + (STACKED ? 0 : (W4_TERMS - 1) * X_TERM) + N * 128, "the MMA reads N rows");
  static constexpr int M_STAGE = 2 * GPU * W4_META_ROW;  // scales and zeros of a unit as they lie in memory
  static constexpr int S_STAGE = 2 * GPU * 128 * 4;      // and as a word per row: scale << 16 | zero
  static constexpr int SIDE = X_STAGE + M_STAGE + S_STAGE;
  static constexpr int COLS = FUSED ? W4_FUSED_TOKENS : MT / SHARES;  // tokens per accumulator thread
  static constexpr int SMEM_MAX = 232448 - 1024 - 4096;
  static constexpr int X_STAGES = FUSED ? CONVERTERS : 3 * SIDE + 3 * 2 * W4_TILE_BYTES <= SMEM_MAX ? 3 : 2;
  static constexpr int FIT = (SMEM_MAX - X_STAGES * SIDE) / (2 * W4_TILE_BYTES);
  static constexpr int W_STAGES = FIT > 5 ? 5 : FIT;
  static constexpr size_t SMEM = 1024 + static_cast<size_t>(W_STAGES) * 2 * W4_TILE_BYTES + X_STAGES * SIDE;
  // tensor memory: accumulators in front, expanded weights (128 columns per unit) behind. An accumulator buffer holds as
  // many (tile, group) sums of a unit as leave room for two buffers.
  static constexpr int A_BUFS = 2;
  static constexpr int C_COLS = 512 - A_BUFS * 128;
  static constexpr int PAIRS = 2 * GPU;  // (half, group, tile) sums of a unit
  static constexpr int fit_pairs() {
    int p = PAIRS;
    while (p > 1 && 2 * p * N > C_COLS) p /= 2;
    return p;
  }
  static constexpr int BUF_PAIRS = fit_pairs();
  static_assert(BUF_PAIRS >= 2, "a buffer holds both tiles' sums of a group");
  static constexpr int C_BUFS_FIT = C_COLS / (BUF_PAIRS * N);
  static constexpr int C_BUFS = C_BUFS_FIT > 4 ? 4 : C_BUFS_FIT;
  static_assert(W_STAGES >= 2 && C_BUFS >= 2, "rings too shallow");
};

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
// D[tmem] (+)= A[tmem] * B[smem], 8-bit floats: A is 128 lanes x 8 columns, four elements a column (32 of the reduction).
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
__device__ __forceinline__ uint4 ld_shared_u4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// Bounded wait for the producers, which wait most of the time and several units ahead: the hardware parks the warp between
// polls (each poll takes issue slots from the warps that work).
__device__ __forceinline__ bool idle_wait(uint32_t bar, uint32_t parity, volatile int* abortp) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const long long t0 = clock64();
  for (;;) {
    if (__all_sync(0xffffffffu, mbar_try_wait_suspend(bar, parity, 2000u))) return true;
    if (__any_sync(0xffffffffu, *abortp != 0 || clock64() - t0 > WAIT_LIMIT_CYCLES)) return false;
    __nanosleep(100);
  }
}
// Bounded wait of a whole warp that polls without the suspend hint of mbar_wait: the hand-over from warp to warp takes
// 125 clocks instead of 213 (measured), and these roles hand over every few hundred clocks.
__device__ __forceinline__ bool quick_wait(uint32_t bar, uint32_t parity, volatile int* abortp) {
  long long t0 = 0;
  for (int i = 0;; ++i) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((i & 63) == 63) {
      const long long t = clock64();
      if (t0 == 0) t0 = t;
      if (__any_sync(0xffffffffu, *abortp != 0 || t - t0 > WAIT_LIMIT_CYCLES)) return false;
    }
  }
}

// One thread of a converged warp. The single-thread roles run their loops with the whole warp and elect a thread for
// the issue itself: addresses and descriptors then live in uniform registers, and an MMA is issued every 15 clocks
// instead of every 45 from inside an `if (lane == 0)` (measured, N = 16).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred q;\nelect.sync _|q, 0xffffffff;\nselp.u32 %0, 1, 0, q;\n}" : "=r"(p));
  return p != 0;
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

// Position of a unit: a in the list of active experts, kb along that expert's columns, first row of its tile.
struct W4Walk {
  int a, kb, row0;
};

template <int MT, bool DUAL, typename T, int GSHIFT, bool FUSED>
__global__ void __launch_bounds__(W4Conf<MT, GSHIFT, FUSED>::THREADS, 1)
w4_stream_kernel(const __grid_constant__ W4Maps maps, const W4Args args) {
  constexpr int TERMS = W4_TERMS;
  using C = W4Conf<MT, GSHIFT, FUSED>;
  constexpr int N = C::N;
  constexpr int NW = C::W_STAGES, NX = C::X_STAGES, NA = C::A_BUFS, NC = C::C_BUFS;
  constexpr int GPH = C::GPH, GPU = C::GPU, PAIRS = C::PAIRS, BUF_PAIRS = C::BUF_PAIRS;
  constexpr int KSTEPS = 1 << GSHIFT;     // 32-column MMA steps per group
  constexpr int ROWS = DUAL ? 128 : 256;  // weight rows per row tile

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * (NW + NX + NA + NC) + NX + 1];
  __shared__ uint32_t tmem_base_holder;
  __shared__ int abort_flag;
  __shared__ MoeShared moe;

  const uint32_t w_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const smem = smem_raw + (w_base - smem_u32(smem_raw));
  const uint32_t x_base = w_base + NW * 2 * W4_TILE_BYTES;
  const uint32_t m_base = x_base + NX * C::X_STAGE;
  const uint32_t wfull = smem_u32(bars), wempty = wfull + 8 * NW, xfull = wempty + 8 * NW, xempty = xfull + 8 * NX,
                 afull = xempty + 8 * NX, aempty = afull + 8 * NA, cfull = aempty + 8 * NA, cempty = cfull + 8 * NC, sfull = cempty + 8 * NC, drain_bar = sfull + 8 * NX;

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // one barrier a thread
  constexpr int BARS = 2 * (NW + NX + NA + NC) + NX + 1;
  if (threadIdx.x < BARS) {
    const uint32_t bar = wfull + 8 * threadIdx.x;
    int count = 1;  // wfull (TMA), aempty and cfull (MMA), sfull (warp 3), drain
    if (bar >= wempty && bar < xfull) count = 8;                               // expanding warps
    if (bar >= xfull && bar < xempty) count = 1 + (FUSED ? args.M : 0);  // TMA, tokens
    if (bar >= xempty && bar < afull) count = 1 + C::EPI / 32;                 // MMA, accumulating warps
    if (bar >= afull && bar < aempty) count = 8;
    if (bar >= cempty && bar < sfull) count = C::EPI / 32;
    mbar_init(bar, count);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (threadIdx.x == 64) abort_flag = 0;
  if (warp == 2 && lane < 7) tma_prefetch_desc(&maps.w0 + lane);
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
  const int per_tile = DUAL ? args.kbt : moe.n * args.kbt;
  const Cut cut = is_moe ? make_cut(per_tile * (DUAL ? moe.n * row_tiles : row_tiles),
                                           cut_grain(per_tile, W4_UNIT_CLOCKS), gridDim.x)
                                : args.cut;
  const int u_begin = cut_start(cut, blockIdx.x), u_end = cut_start(cut, blockIdx.x + 1);
  const int units = u_end - u_begin;

  auto start = [&](W4Walk& w) {
    w.a = w.kb = w.row0 = 0;
    if (units == 0) return;
    const int tile = u_begin / per_tile, r = u_begin - tile * per_tile;
    if (DUAL) {
      w.a = is_moe ? tile / row_tiles : 0;
      w.row0 = (tile - w.a * row_tiles) * ROWS;
      w.kb = r;
    } else {
      w.row0 = tile * ROWS;
      w.a = is_moe ? r / args.kbt : 0;
      w.kb = r - w.a * args.kbt;
    }
  };
  auto step = [&](W4Walk& w) {  // the next unit, without a division
    if (++w.kb < args.kbt) return;
    w.kb = 0;
    if (DUAL) {
      w.row0 += ROWS;
      if (w.row0 >= args.rows) {
        w.row0 = 0;
        ++w.a;
      }
    } else if (++w.a == moe.n) {
      w.a = 0;
      w.row0 += ROWS;
    }
  };
  // groups of the unit that exist: GPU but for the last unit of an expert's columns
  auto groups_in = [&](int kb) {
    const int left = args.groups - kb * GPU;
    return left < GPU ? left : GPU;
  };

  // 64 tokens: 896 threads leave 72 registers each. Of the block's 896 x 72 = 64,512 the helpers keep 40 and the expanders
  // 56 a thread, the accumulators get 88: 128 x (40 + 2 x 56 + 4 x 88) = 64,512.
  if (warp == 0) {
    // ------------------------------------------------------------ weights --
    if (MT == 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    const uint64_t pol = l2_policy_evict_first();
    W4Walk w;
    start(w);
    Ring r;
    int u = 0;
    bool ok = true;
    for (; u < units; ++u) {
      if (!(ok = idle_wait(wempty + 8 * r.at, r.phase ^ 1u, abortp))) break;
      const uint32_t dst = w_base + r.at * 2 * W4_TILE_BYTES, fb = wfull + 8 * r.at;
      const int y = moe.list[w.a] * args.rows + w.row0;
      if (elect_one()) {
        mbar_expect_tx(fb, 2 * W4_TILE_BYTES);
        tma_load_2d_hint(dst, &maps.w0, fb, w.kb * 128, y, pol);
        if (DUAL)
          tma_load_2d_hint(dst + W4_TILE_BYTES, &maps.w1, fb, w.kb * 128, y, pol);
        else
          tma_load_2d_hint(dst + W4_TILE_BYTES, &maps.w0, fb, w.kb * 128, y + 128, pol);
      }
      __syncwarp();
      step(w);
      r.next(NW);
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_PRODUCER);
      for (int i = u > NW ? u - NW : 0; i < u; ++i)  // see the copies in flight land before the block leaves
        drain_wait(wfull + 8 * (i % NW), static_cast<uint32_t>(i / NW) & 1u);
    }
  } else if (warp == 2) {
    // -------------------------------------------------------- activations --
    if (MT == 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (args.early && !FUSED) pdl_wait();
    const uint64_t pol = l2_policy_evict_last(), pol_w = l2_policy_evict_first();
    W4Walk w;
    start(w);
    Ring r;
    int u = 0;
    bool ok = true;
    for (; u < units; ++u) {
      if (!(ok = idle_wait(xempty + 8 * r.at, r.phase ^ 1u, abortp))) break;
      const int a = DUAL ? 0 : w.a;
      const uint32_t dst = x_base + r.at * C::X_STAGE, fb = xfull + 8 * r.at;
      constexpr uint32_t META_BYTES = GPU * MT * 4;
      const uint32_t md = m_base + r.at * C::M_STAGE;
      uint32_t sz_bytes = args.wide ? 2 * GPU * 128 * (2 + (args.zero0 != nullptr ? 1 : 0)) : 0;
      uint64_t src = 0;  // this lane's copy
      uint32_t len = 0;
      if (!args.wide) {
        const int t = lane >> 1 >= GPU ? 1 : 0, g = (lane >> 1) - t * GPU;  // even lanes: scales, odd ones: zeros
        const int skip = DUAL ? 0 : t * 128, left = args.rows - w.row0 - skip;
        const long long e0 = (static_cast<long long>(moe.list[w.a]) * args.groups + w.kb * GPU + g) * args.rows + w.row0 + skip;
        const uint32_t nrow = static_cast<uint32_t>(left < 128 ? left : 128);
        const uint64_t base = reinterpret_cast<uint64_t>(
            lane & 1 ? static_cast<const void*>(DUAL && t == 1 ? args.zero1 : args.zero0)
                     : static_cast<const void*>(DUAL && t == 1 ? args.scale1 : args.scale0));
        const int sh = 1 - (lane & 1);  // bytes of an element, as a shift
        src = base + (static_cast<uint64_t>(e0) << sh);
        if (base != 0 && left > 0 && lane < 4 * GPU && g < groups_in(w.kb))
          len = ((static_cast<uint32_t>(src) & 15u) + (nrow << sh) + 15u) & ~15u;
        src &= ~15ull;
        sz_bytes = __reduce_add_sync(0xffffffffu, len);
      }
      if (elect_one()) {
        mbar_expect_tx(fb, (FUSED ? 0 : 2 * TERMS * MT * 128 + META_BYTES) + sz_bytes);
        if (args.wide) {
          const int gy = moe.list[w.a] * args.groups + w.kb * GPU;
          tma_load_2d_hint(md, &maps.s0, fb, w.row0, gy, pol_w);
          tma_load_2d_hint(md + GPU * 256, DUAL ? &maps.s1 : &maps.s0, fb, w.row0 + (DUAL ? 0 : 128), gy, pol_w);
          if (args.zero0 != nullptr) {
            tma_load_2d_hint(md + 2 * GPU * 256, &maps.z0, fb, w.row0, gy, pol_w);
            tma_load_2d_hint(md + 2 * GPU * 256 + GPU * 128, DUAL ? &maps.z1 : &maps.z0, fb, w.row0 + (DUAL ? 0 : 128), gy,
                             pol_w);
          }
        }
        if (!FUSED) {
#pragma unroll
          for (int i = 0; i < 2 * TERMS; ++i)  // a half behind the last column arrives as zeros
            tma_load_2d_hint(dst + i / TERMS * C::X_HALF + i % TERMS * C::X_TERM, &maps.x, fb, w.kb * W4_UNIT_COLS + (i / TERMS) * W4_HALF_COLS,
                             static_cast<int>((i % TERMS) * args.R) + a * args.M, pol);
          bulk_load(dst + 2 * C::X_HALF, args.meta + (static_cast<long long>(a) * args.kbt + w.kb) * (GPU * MT),
                    META_BYTES, fb);
        }
      }
      __syncwarp();
      if (len != 0)
        bulk_load(md + (lane >> 1) * W4_META_ROW + (lane & 1) * W4_META_ZERO, reinterpret_cast<const void*>(src), len, fb);
      step(w);
      r.next(NX);
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_PRODUCER);
      for (int i = u > NX ? u - NX : 0; i < u; ++i)
        drain_wait(xfull + 8 * (i % NX), static_cast<uint32_t>(i / NX) & 1u);
    }
  } else if (warp == 3) {
    // --------------------------------------------------- scales and zeros --
    if (MT == 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    // One word per row, tile and group for all the accumulating threads: scale << 16 | zero.
    const bool zeros = args.zero0 != nullptr;
    const uint8_t* const m_stages = smem + NW * 2 * W4_TILE_BYTES + NX * C::X_STAGE;
    uint8_t* const s_stages = smem + NW * 2 * W4_TILE_BYTES + NX * (C::X_STAGE + C::M_STAGE);
    W4Walk w;
    start(w);
    Ring r;
    bool ok = true;
    for (int u = 0; u < units && ok; ++u) {
      if (!(ok = quick_wait(xfull + 8 * r.at, r.phase, abortp))) break;
      const int ng = groups_in(w.kb);
      const uint8_t* const mm = m_stages + r.at * C::M_STAGE;
      uint4* const ss = reinterpret_cast<uint4*>(s_stages + r.at * C::S_STAGE) + lane;  // four rows a lane
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int g = 0; g < GPU; ++g) {
          uint32_t z = 0x08080808u, s01, s23;
          if (args.wide) {
            const uint2 q = *reinterpret_cast<const uint2*>(mm + (t * GPU + g) * 256 + lane * 8);
            s01 = q.x;
            s23 = q.y;
            if (zeros) z = *reinterpret_cast<const uint32_t*>(mm + 2 * GPU * 256 + (t * GPU + g) * 128 + lane * 4);
          } else {
            // where the rows start inside the copied blocks of 16 bytes: low bits of the first one's address
            const uint32_t e = (static_cast<uint32_t>(moe.list[w.a]) * args.groups + w.kb * GPU + g) *
                                   static_cast<uint32_t>(args.rows) + w.row0 + (DUAL ? 0 : t * 128);
            const uint32_t s_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(DUAL && t == 1 ? args.scale1 : args.scale0));
            const uint32_t z_at = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(DUAL && t == 1 ? args.zero1 : args.zero0));
            const uint8_t* const mr = mm + (t * GPU + g) * W4_META_ROW;
            const uint16_t* const sp = reinterpret_cast<const uint16_t*>(mr + ((s_at + 2 * e) & 15u)) + lane * 4;
            s01 = sp[0] | (static_cast<uint32_t>(sp[1]) << 16);
            s23 = sp[2] | (static_cast<uint32_t>(sp[3]) << 16);
            const uint8_t* const zp = mr + W4_META_ZERO + ((z_at + e) & 15u) + lane * 4;
            if (zeros) z = zp[0] | (zp[1] << 8) | (zp[2] << 16) | (static_cast<uint32_t>(zp[3]) << 24);
          }
          uint4 o = make_uint4((s01 << 16) | (z & 15u), (s01 & 0xFFFF0000u) | ((z >> 8) & 15u),
                               (s23 << 16) | ((z >> 16) & 15u), (s23 & 0xFFFF0000u) | ((z >> 24) & 15u));
          if (g >= ng) o = make_uint4(0u, 0u, 0u, 0u);  // a group behind the last column has a scale of zero
          ss[(t * GPU + g) * 32] = o;
        }
      __syncwarp();
      if (lane == 0) mbar_arrive(sfull + 8 * r.at);
      step(w);
      r.next(NX);
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_PRODUCER);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA --
    if (MT == 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    constexpr uint32_t IDESC = make_idesc_f8(128, N, FORMAT_E5M2);
    const uint64_t x0 = make_smem_desc(x_base, 16, 1024);
    Ring rx, ra, rc;
    bool ok = true;
    for (int u = 0; u < units && ok; ++u) {
      if (!(ok = quick_wait(xfull + 8 * rx.at, rx.phase, abortp))) break;
      if (!(ok = quick_wait(afull + 8 * ra.at, ra.phase, abortp))) break;
      const uint64_t xd = x0 + static_cast<uint64_t>(rx.at * (C::X_STAGE >> 4));
      const uint32_t a0 = tmem_base + C::C_COLS + ra.at * 128;
      // sums in the order (half, group, tile); groups behind the last column are zeros
#pragma unroll
      for (int p0 = 0; p0 < PAIRS; p0 += BUF_PAIRS) {
        if (!(ok = quick_wait(cempty + 8 * rc.at, rc.phase ^ 1u, abortp))) break;
        tc_fence_after_sync();
        const uint32_t d = tmem_base + rc.at * (BUF_PAIRS * N);
        if (elect_one()) {
#pragma unroll
          for (int p = p0; p < p0 + BUF_PAIRS; ++p) {
            const int t = p & 1, h = p / (2 * GPH), g = (p >> 1) % GPH;
#pragma unroll
            for (int k = 0; k < KSTEPS; ++k) {
              const int kk = g * KSTEPS + k;  // 32-column step inside the half
#pragma unroll
              for (int i = 0; i < (C::STACKED ? 1 : TERMS); ++i)
                umma_f8_ts(d + (p - p0) * N, a0 + t * 64 + h * 32 + kk * 8,
                           xd + static_cast<uint64_t>(((h * C::X_HALF + i * C::X_TERM) >> 4) + 2 * kk), IDESC,
                           k + i > 0 ? 1u : 0u);
            }
          }
          umma_commit(cfull + 8 * rc.at);
          if (p0 + BUF_PAIRS == PAIRS) {
            umma_commit(aempty + 8 * ra.at);
            umma_commit(xempty + 8 * rx.at);
          }
        }
        __syncwarp();
        rc.next(NC);
      }
      ra.next(NA);
      rx.next(NX);
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_MMA);
      umma_commit(drain_bar);
      drain_wait(drain_bar, 0);
    }
  } else if (warp < 12) {
    // ------------------------------------------------------------- expand --
    if (MT == 64) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    const int quarter = warp & 3;
    const int tsel = (warp - 4) >> 2;  // which of the unit's two tiles
    const int row = quarter * 32 + lane;
    const uint32_t src0 = w_base + tsel * W4_TILE_BYTES + row * 128;
    const uint32_t dst0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + C::C_COLS + tsel * 64;
    Ring rw, ra;
    bool ok = true;
    for (int u = 0; u < units; ++u) {
      if (!(ok = quick_wait(wfull + 8 * rw.at, rw.phase, abortp))) break;
      const uint32_t src = src0 + rw.at * 2 * W4_TILE_BYTES;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t r[32];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint4 q = ld_shared_u4(src + (((h * 4 + c) ^ (row & 7)) << 4));
          const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            r[c * 8 + 2 * i] = word[i] & 0x0F0F0F0Fu;
            r[c * 8 + 2 * i + 1] = (word[i] >> 4) & 0x0F0F0F0Fu;
          }
        }
        if (h == 0) {
          ok = quick_wait(aempty + 8 * ra.at, ra.phase ^ 1u, abortp);
          if (!ok) break;
          tc_fence_after_sync();
        } else {
          __syncwarp();
          if (lane == 0) mbar_arrive(wempty + 8 * rw.at);  // the packed weights are in registers
        }
        tmem_st_32x32(dst0 + ra.at * 128 + h * 32, r);
      }
      if (!ok) break;
      tmem_st_wait();
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(afull + 8 * ra.at);
      ra.next(NA);
      rw.next(NW);
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_MMA);
    }
  } else if (FUSED && warp >= 16) {
    // ------------------------------------------- activations -> terms --
    // (unit, token) pairs in turn, one a warp: the row's 256 columns, eight a lane, the two halves of the warp the two halves
    // of the unit. Written where TMA would have put them (128-byte rows, 16-byte chunks swizzled by the row).
    if (args.early) pdl_wait();
    const int sub = lane & 15, half = lane >> 4;
    W4Walk wn;  // position of the pair being fetched
    start(wn);
    // A parity tells a stage's phase only to a waiter that is not a whole turn of the ring away from it: a warp that goes
    // from unit u to u + d has seen unit u - NX released, and needs u + d - 2 NX to be: d <= NX.
    static_assert(!FUSED || NX >= C::CONVERTERS, "a converting warp would take one phase of a stage for another");
    Ring r;  // stage of `unit`
    bool ok = true;
    auto fetch = [&](int m) {
      const int col = wn.kb * W4_UNIT_COLS + lane * 8;
      uint4 v = make_uint4(0u, 0u, 0u, 0u);
      if (col < args.cols)
        v = *reinterpret_cast<const uint4*>(static_cast<const T*>(args.x) +
                                            ((DUAL ? 0 : static_cast<long long>(wn.a) * args.M) + m) * args.ldx + col);
      return v;
    };
    // (unit, token) of this pair and, one ahead, of the pair being fetched
    int unit = 0, m = 0, next_unit = 0, next_m = warp - 16;
    auto settle_next = [&]() {
      while (next_m >= args.M) {
        next_m -= args.M;
        ++next_unit;
        if (next_unit < units) step(wn);
      }
    };
    uint4 raw = make_uint4(0u, 0u, 0u, 0u);
    settle_next();
    if (next_unit < units) raw = fetch(next_m);
    while (next_unit < units) {
      for (; unit < next_unit; ++unit) r.next(NX);
      m = next_m;
      const uint4 cur = raw;
      next_m += C::CONVERTERS;
      settle_next();
      if (next_unit < units) raw = fetch(next_m);
      float v[8];
      const float2 v0 = Pack2<T>::unpack(cur.x), v1 = Pack2<T>::unpack(cur.y), v2 = Pack2<T>::unpack(cur.z),
                   v3 = Pack2<T>::unpack(cur.w);
      v[0] = v0.x; v[1] = v0.y; v[2] = v1.x; v[3] = v1.y;
      v[4] = v2.x; v[5] = v2.y; v[6] = v3.x; v[7] = v3.y;
      constexpr int WIDTH = 4 << GSHIFT;  // lanes of a group
      float amax = amax8(v);
#pragma unroll
      for (int o = 1; o < WIDTH; o <<= 1) amax = nan_max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      const int ex = amax != amax ? 0 : split_exponent(amax);
      uint2 code[TERMS];
      float sum = split_terms(v, ex, code);
#pragma unroll
      for (int o = 1; o < WIDTH; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const float down = amax != amax ? amax : power_of_two(W4_LIFT - ex);
      ok = quick_wait(xempty + 8 * r.at, r.phase ^ 1u, abortp);
      if (!ok) break;
      uint8_t* const xs = smem + NW * 2 * W4_TILE_BYTES + r.at * C::X_STAGE;
#pragma unroll
      for (int t = 0; t < TERMS; ++t) {
        const int xr = t * C::TOK + m;
        *reinterpret_cast<uint2*>(xs + half * C::X_HALF + xr * 128 + (((sub >> 1) ^ (xr & 7)) << 4) + (sub & 1) * 8) =
            code[t];
      }
      if ((sub & (WIDTH - 1)) == 0) {
        float* const mt = reinterpret_cast<float*>(xs + 2 * C::X_HALF) + (half * GPH + sub / WIDTH) * 2 * MT + m;
        mt[0] = down;
        mt[MT] = sum * 0.001953125f;
      }
      fence_proxy_async_smem();  // the MMA reads the terms
      __syncwarp();
      if (lane == 0) mbar_arrive(xfull + 8 * r.at);
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_PRODUCER);
    }
  } else {
    // ------------------------------------------- accumulate and finish --
    if (MT == 64) asm volatile("setmaxnreg.inc.sync.aligned.u32 88;");
    constexpr int COLS = C::COLS, EPI = C::EPI;
    constexpr int CH = COLS < 16 ? COLS : 16;  // token columns per round of tensor-memory loads
    constexpr int GROUPS = BUF_PAIRS / 2;      // groups in a buffer, both tiles' sums each
    // sums in flight at a time: as many as 32 registers hold
    constexpr int LOADS = C::STACKED ? TERMS : 1;
    constexpr int BATCH = BUF_PAIRS * CH * LOADS <= 32 ? BUF_PAIRS : 32 / (CH * LOADS);
    const int quarter = warp & 3;
    const int col0 = ((warp - 12) >> 2) * COLS;
    const bool idle = col0 >= args.M;  // no tokens in these columns
    const int row = quarter * 32 + lane;
    const uint32_t acc0 = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + col0;
    const int ep_tid = threadIdx.x - 384;
    if (args.early) pdl_wait();  // slots, counters and outputs may still be in use
    if (!DUAL && cut.total == 0) {
      // no token chose any expert: the outputs are the residual, or zero
      const long long all = static_cast<long long>(args.M) * args.rows;
      for (long long i = blockIdx.x * static_cast<long long>(EPI) + ep_tid; i < all; i += gridDim.x * static_cast<long long>(EPI))
        static_cast<T*>(args.out)[i] =
            args.residual ? static_cast<const T*>(args.residual)[i] : static_cast<T>(0.f);
    }
    const MoeShared* const mp = is_moe ? &moe : nullptr;
    const Split sp{cut, args.M, reinterpret_cast<float4*>(args.slots), args.counters, abortp};
    auto emit_tile = [&](int tile, int begin, const Join& join) {
      T* const out = static_cast<T*>(args.out);
      const T* const b0 = static_cast<const T*>(args.bias0);
      const float* const rs = FUSED ? nullptr : args.rowscale;
      const long long ld = args.rows;
      if (DUAL) {
        const T* const b1 = static_cast<const T*>(args.bias1);
        const int a = tile / row_tiles, row0 = (tile - a * row_tiles) * ROWS;
        if (is_moe) {
          moe_factors(args.moe, args.M, moe.list[a], ep_tid, moe);
          named_bar_sync(1, EPI);
        }
        T* const oa = out + static_cast<long long>(a) * args.M * ld;
        finish_tile<2, true, MT, EPI, 1>(begin, join, sp, ep_tid,
                                      [&](int, int r, int i, const float4& gate, const float4& up) {
          const int wr = row0 + r;
          if (wr < args.rows)
            emit_hidden(oa + wr, ld, args.M, i, gate, up, rs, b0 ? static_cast<float>(b0[wr]) : 0.f,
                        b1 ? static_cast<float>(b1[wr]) : 0.f, args.act, mp);
        });
      } else {
        const T* const res = static_cast<const T*>(args.residual);
        finish_tile<2, false, MT, EPI, 1>(begin, join, sp, ep_tid,
                                       [&](int t, int r, int i, const float4& v, const float4&) {
          const int wr = tile * ROWS + t * 128 + r;
          if (wr < args.rows)
            emit_product(out + wr, res ? res + wr : nullptr, ld, args.M, i, v, rs, b0 ? static_cast<float>(b0[wr]) : 0.f, mp);
        });
      }
      named_bar_sync(1, EPI);  // the slot, f and hit are free for the next tile
    };
    Pending pending;
    bool alive = true;
    W4Walk w;
    start(w);
    Ring rx, rc;
    int u = u_begin;
    while (u < u_end) {
      const Segment s = segment_at(u, u_end, per_tile);
      f32x2 v[2][COLS / 2];
#pragma unroll
      for (int c = 0; c < COLS / 2; ++c) v[0][c] = v[1][c] = 0ull;
      bool ok = true;
      for (; u < s.end; ++u) {
        // (warp 3 saw the unit's factors land before it arrived here)
        ok = quick_wait(sfull + 8 * rx.at, rx.phase, abortp);
        // read as ordinary memory, so that the loads between two waits go out together
        const uint8_t* const side = smem + NW * 2 * W4_TILE_BYTES;
        const float* const xm = reinterpret_cast<const float*>(side + rx.at * C::X_STAGE + 2 * C::X_HALF) + col0;
        const uint32_t* const ss =
            reinterpret_cast<const uint32_t*>(side + NX * (C::X_STAGE + C::M_STAGE) + rx.at * C::S_STAGE) + row;
#pragma unroll
        for (int g0 = 0; g0 < GPU; g0 += GROUPS) {
          // scales and zeros of the buffer's sums are fetched before the sums are there
          float sc[BUF_PAIRS], nz[BUF_PAIRS];
#pragma unroll
          for (int b = 0; b < BUF_PAIRS; ++b) {
            const uint32_t sz = ss[((b & 1) * GPU + g0 + (b >> 1)) * 128];
            sc[b] = (512.0f / (1 << W4_LIFT)) * Pack2<T>::unpack(sz >> 16).x;
            // an integer below 2^23 in a float's fraction: 2^23 - (2^23 + z)
            nz[b] = 8388608.0f - __uint_as_float(0x4B000000u | (sz & 15u));
          }
          ok = ok && quick_wait(cfull + 8 * rc.at, rc.phase, abortp);
          tc_fence_after_sync();
          const uint32_t src = acc0 + rc.at * (BUF_PAIRS * N);
#pragma unroll
          for (int b0 = 0; b0 < BUF_PAIRS; b0 += BATCH) {
#pragma unroll
            for (int c = 0; c < COLS; c += CH) {
              uint32_t x[BATCH][CH], more[BATCH][LOADS][CH];
              if (!idle) {
#pragma unroll
                for (int b = 0; b < BATCH; ++b) {
                  tmem_ld_cols<CH>(src + (b0 + b) * N + c, x[b]);
#pragma unroll
                  for (int i = 1; i < LOADS; ++i) tmem_ld_cols<CH>(src + (b0 + b) * N + i * C::TOK + c, more[b][i]);
                }
                tmem_ld_wait();
              }
              if (b0 + BATCH == BUF_PAIRS && c + CH == COLS) {  // the last sums are in registers
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(cempty + 8 * rc.at);
              }
              if (!idle) {
                if constexpr (C::STACKED) {  // the terms' sums, the smallest first
#pragma unroll
                  for (int b = 0; b < BATCH; ++b)
#pragma unroll
                    for (int k = 0; k < CH; ++k) {
                      float sum = __uint_as_float(more[b][LOADS - 1][k]);
#pragma unroll
                      for (int i = LOADS - 2; i > 0; --i) sum += __uint_as_float(more[b][i][k]);
                      x[b][k] = __float_as_uint(__uint_as_float(x[b][k]) + sum);
                    }
                }
#pragma unroll
                for (int k = 0; k < CH; k += 4) {
#pragma unroll
                  for (int b = 0; b < BATCH; ++b) {
                    const int t = (b0 + b) & 1, g = g0 + ((b0 + b) >> 1);
                    const float4 q0 = *reinterpret_cast<const float4*>(xm + g * C::FACTORS * MT + c + k);
                    const float tok[4] = {q0.x, q0.y, q0.z, q0.w};
                    if constexpr (FUSED) {
                      const float4 q1 = *reinterpret_cast<const float4*>(xm + g * 2 * MT + MT + c + k);
                      const float sx[4] = {q1.x, q1.y, q1.z, q1.w};
#pragma unroll
                      for (int j = 0; j < 4; j += 2) {
                        // (scale and power of two first: their product with the sum is the group's share of the output and
                        // overflows only where that does)
                        const f32x2 f = f2_pack(sc[b0 + b] * tok[j], sc[b0 + b] * tok[j + 1]);
                        const f32x2 y = f2_pack(fmaf(nz[b0 + b], sx[j], __uint_as_float(x[b][k + j])),
                                                fmaf(nz[b0 + b], sx[j + 1], __uint_as_float(x[b][k + j + 1])));
                        v[t][(c + k + j) / 2] = f2_fma(f, y, v[t][(c + k + j) / 2]);
                      }
                    } else {
                      // two tokens an instruction: what bounds many tokens is issue slots
                      const f32x2 s2 = f2_pack(sc[b0 + b], sc[b0 + b]), z2 = f2_pack(nz[b0 + b], nz[b0 + b]);
#pragma unroll
                      for (int j = 0; j < 4; j += 2) {
                        f32x2 y = f2_pack(__uint_as_float(x[b][k + j]), __uint_as_float(x[b][k + j + 1]));
                        y = f2_fma(z2, f2_pack(tok[j], tok[j + 1]), y);
                        v[t][(c + k + j) / 2] = f2_fma(s2, y, v[t][(c + k + j) / 2]);
                      }
                    }
                  }
                }
              }
            }
          }
          rc.next(NC);
        }
        if (!ok) break;
        __syncwarp();  // all lanes have read the unit's factors, scales and zeros
        if (lane == 0) mbar_arrive(xempty + 8 * rx.at);
        rx.next(NX);
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
      if (!(alive = end_segment<2, COLS, MT, EPI>(f, s, sp, col0, row, ep_tid, pending, emit_tile))) break;
    }
    if (alive) end_units<EPI>(pending, per_tile, sp, ep_tid, emit_tile);
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
