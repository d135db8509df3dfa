// Products of up to 64 tokens with 4-bit weights, w = (q - zero) * scale, one scale and zero per group of G columns
// (G = 32, 64 or 128): a plain product (DUAL = false) or the gate/up half of a gated MLP (DUAL = true), dense
// or over the experts of a mixture.
//
// What bounds it: HBM. A weight is half a byte (plus its share of scale and zero), so at the copy bandwidth an SM
// receives about 46 weights a clock, and what it must do per weight is small but not nothing: take the nibble out,
// make it a 16-bit number, multiply it with every token. The tokens are the N dimension of tcgen05.mma (16, 32 or
// 64), 128 weight rows its M dimension ("swap-AB" like the 16-bit decode kernel).
//
// Path of a weight: HBM -> shared memory by TMA (packed, 128 rows x 128 bytes = 256 columns per tile, two tiles a
// unit) -> registers of the thread that owns its row -> exact 16-bit integers q - zero -> tensor memory
// (tcgen05.st), from which the MMA takes its A operand. The expanded weights never pass through shared memory,
// whose 128 bytes a clock could not carry them twice (92 written and 92 read) beside the packed stream.
//   nibble -> number: the in-word order of the format puts columns 2i and 2i + 1 at bits 4i and 16 + 4i, so
//   ((word >> 4i) & 0x000F000F) | magic is a pair of 16-bit floats 128 + q (bf16, magic 0x4300) or 1024 + q (fp16,
//   0x6400), and one packed subtraction of 128 + zero leaves q - zero: three instructions for two weights, no rounding.
//   scale: not applied to the weights. A group's products are accumulated by themselves and the 32-bit sums are
//   multiplied by the group's scale when the accumulator warps take them out of tensor memory:
//     y[r][m] = sum_g scale[r][g] * ( sum_{c in g} (q[r][c] - zero[r][g]) x[m][c] )
//   so nothing is rounded to 16 bits on the way, and it costs tokens / G multiply-adds per weight.
//
// Warps: 0 issues TMA, 1 issues MMA, 2..9 expand (four per tile, thread = row), then 4 (8 for 64 tokens)
// accumulate and run the epilogue. Tensor memory: accumulators 2 buffers x 2 tiles x MPAD columns, expanded weights
// 2 buffers x 2 tiles x 64 columns (128 weights each).
//
// Work split: stream-K over units of (two row tiles, 256 columns) as in few_token.cuh.
#pragma once
#include "few_token.cuh"

namespace gmlp {

struct W4Args {
  int M;
  int rows;        // weight rows per expert (N for DUAL, outputs otherwise)
  int kbt;         // units along an expert's columns: ceil(cols / 256)
  int groups;      // cols / G
  int gshift;      // log2(G / 32): 0, 1, 2
  uint32_t idesc;
  int* status;
  const void* scale0;    // [experts][groups][rows], T
  const void* scale1;    // DUAL: the up matrix's
  const uint8_t* zero0;  // [experts][groups][rows] or null (8)
  const uint8_t* zero1;
  const void* bias0;     // [rows] or null
  const void* bias1;
  const void* residual;  // [M][rows] or null (DUAL = false)
  void* out;             // [M][rows]; DUAL on experts: [active][M][rows]
  float* slots;
  int* counters;
  int act;
  int dependent;    // launched as a programmatic dependent
  int early;        // the weights may be streamed before the preceding kernel has finished
  MoeTable moe;
};

constexpr int W4_TILE_BYTES = 16384;  // 128 rows x 128 bytes: 256 columns
constexpr int W4_UNIT_COLS = 256;
template <int MPAD>
__host__ __device__ constexpr int w4_stage_bytes() {
  return 2 * W4_TILE_BYTES + MPAD * 512;
}
template <int MPAD>
__host__ __device__ constexpr int w4_stages() {
  return (232448 - 1024 - 4096) / w4_stage_bytes<MPAD>();
}
template <int MPAD>
constexpr size_t w4_smem_bytes() {
  return static_cast<size_t>(w4_stages<MPAD>()) * w4_stage_bytes<MPAD>() + 1024;
}
template <int MPAD>
__host__ __device__ constexpr int w4_acc_warps() {
  return MPAD == 64 ? 8 : 4;
}
template <int MPAD>
__host__ __device__ constexpr int w4_threads() {
  return 32 * (10 + w4_acc_warps<MPAD>());
}

// ---- tensor-memory operand ----
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// D[tmem] (+)= A[tmem] * B[smem]: A is 128 lanes x 8 columns, two 16-bit elements a column.
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Eight weights of one 32-bit word as four packed pairs (columns 0-1, 2-3, 4-5, 6-7), minus `off` = magic base + zero.
template <typename T>
struct Nibbles;
template <>
struct Nibbles<__nv_bfloat16> {
  static constexpr uint32_t MAGIC = 0x43004300u;  // 128, 128: the nibble is the low end of the 7-bit fraction
  static __device__ __forceinline__ uint32_t offset(int zero) {
    return 0x43004300u + static_cast<uint32_t>(zero) * 0x00010001u;  // 128 + zero
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};
template <>
struct Nibbles<__half> {
  static constexpr uint32_t MAGIC = 0x64006400u;  // 1024, 1024
  static __device__ __forceinline__ uint32_t offset(int zero) {
    return 0x64006400u + static_cast<uint32_t>(zero) * 0x00010001u;
  }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    uint32_t d;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
  }
};
template <typename T>
__device__ __forceinline__ void expand_word(uint32_t w, uint32_t off, uint32_t* r) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = Nibbles<T>::sub(((w >> (4 * i)) & 0x000F000Fu) | Nibbles<T>::MAGIC, off);
}

__device__ __forceinline__ uint4 ld_shared_u4(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "r"(a)
               : "memory");
  return v;
}

// Position of a unit: expert slot a (its index in the active list), unit kb along that expert's columns.
struct W4Pos {
  int a, kb;
};

template <int MPAD, bool DUAL, typename T>
__global__ void __launch_bounds__(w4_threads<MPAD>(), 1)
w4_stream_kernel(const __grid_constant__ CUtensorMap tmW0, const __grid_constant__ CUtensorMap tmW1,
                 const __grid_constant__ CUtensorMap tmX, const W4Args args) {
  constexpr int STAGES = w4_stages<MPAD>();
  constexpr uint32_t STAGE_BYTES = w4_stage_bytes<MPAD>();
  constexpr uint32_t X_OFF = 2 * W4_TILE_BYTES;
  constexpr int ACC_WARPS = w4_acc_warps<MPAD>();
  constexpr int ACC_THREADS = 32 * ACC_WARPS;
  constexpr int COLS = MPAD == 64 ? 32 : MPAD;  // tokens per accumulator thread
  constexpr int ROWS = DUAL ? 128 : 256;        // weight rows per row tile
  constexpr uint32_t TM_A = 256;                // first tensor-memory column of the expanded weights
  static_assert(STAGES >= 3, "ring too shallow");

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * STAGES + 9];
  __shared__ uint32_t tmem_base_holder;
  __shared__ int abort_flag;
  __shared__ MoeShared moe;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar_base = smem_u32(bars);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto afull_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + b); };
  auto aempty_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + 2 + b); };
  auto cfull_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + 4 + b); };
  auto cempty_bar = [&](int b) { return bar_base + 8u * (2 * STAGES + 6 + b); };
  const uint32_t drain_bar = bar_base + 8u * (2 * STAGES + 8);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(afull_bar(b), 8);
      mbar_init(aempty_bar(b), 1);
      mbar_init(cfull_bar(b), 1);
      mbar_init(cempty_bar(b), ACC_WARPS);
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
  if (args.dependent && !args.early) pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  tc_fence_before_sync();
  moe_collect(args.moe, args.M, moe);  // ends with a block barrier
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_holder;
  volatile int* abortp = &abort_flag;

  // Units: DUAL: tile = (expert, row tile), kbt units each. Else: tile = row tile, units = (expert, kb).
  const int row_tiles = (args.rows + ROWS - 1) / ROWS;
  const long long per_tile = DUAL ? args.kbt : static_cast<long long>(moe.n) * args.kbt;
  const long long total = per_tile * (DUAL ? static_cast<long long>(moe.n) * row_tiles : row_tiles);
  const long long ctas = total < gridDim.x ? total : gridDim.x;
  const long long u_begin = blockIdx.x < ctas ? unit_start(blockIdx.x, total, ctas) : 0;
  const long long u_end = blockIdx.x < ctas ? unit_start(blockIdx.x + 1, total, ctas) : 0;
  const int gpu_ = 8 >> args.gshift;  // groups per unit (256 columns)
  const int gps = 4 >> args.gshift;   // groups per half unit (128 columns)

  auto pos_at = [&](long long tile, long long r) {  // r: unit inside the tile
    W4Pos p;
    if (DUAL) {
      p.a = static_cast<int>(tile / row_tiles);
      p.kb = static_cast<int>(r);
    } else {
      p.a = static_cast<int>(r / args.kbt);
      p.kb = static_cast<int>(r - static_cast<long long>(p.a) * args.kbt);
    }
    return p;
  };
  auto step = [&](W4Pos& p) {  // the next unit of the same tile
    if (++p.kb == args.kbt) {
      p.kb = 0;
      if (!DUAL) ++p.a;
    }
  };
  auto row0_of = [&](long long tile) {  // first weight row of the tile inside its expert
    return static_cast<int>(DUAL ? tile % row_tiles : tile) * ROWS;
  };
  auto groups_in = [&](int kb) {  // groups of a unit that exist (the last unit may be short)
    const int left = args.groups - kb * gpu_;
    return left < gpu_ ? left : gpu_;
  };

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA --
    if (lane == 0 && u_begin < u_end) {
      const uint64_t pol_w = l2_policy_evict_first();
      const uint64_t pol_x = l2_policy_evict_last();
      long long tile = u_begin / per_tile;
      W4Pos p = pos_at(tile, u_begin - tile * per_tile);
      long long left = (tile + 1) * per_tile - u_begin;  // units of this tile still to come
      W4Pos px = p;
      long long tile_x = tile, left_x = left;
      auto advance = [&](long long& t, W4Pos& q, long long& l) {
        if (--l == 0) {
          ++t;
          l = per_tile;
          q = pos_at(t, 0);
        } else {
          step(q);
        }
      };
      auto load_w = [&](int st) {
        const long long base = static_cast<long long>(moe.list[p.a]) * args.rows + row0_of(tile);
        const uint32_t sw = smem_base + st * STAGE_BYTES;
        const uint32_t fb = full_bar(st);
        mbar_expect_tx(fb, STAGE_BYTES);
        tma_load_2d_hint(sw, &tmW0, fb, p.kb * 128, static_cast<int>(base), pol_w);
        if (DUAL)
          tma_load_2d_hint(sw + W4_TILE_BYTES, &tmW1, fb, p.kb * 128, static_cast<int>(base), pol_w);
        else
          tma_load_2d_hint(sw + W4_TILE_BYTES, &tmW0, fb, p.kb * 128, static_cast<int>(base) + 128, pol_w);
        advance(tile, p, left);
      };
      auto load_x = [&](int st) {
        const int y = (!DUAL && is_moe) ? px.a * args.M : 0;
        const uint32_t sx = smem_base + st * STAGE_BYTES + X_OFF;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          tma_load_2d_hint(sx + i * MPAD * 128, &tmX, full_bar(st), px.kb * W4_UNIT_COLS + i * 64, y, pol_x);
        advance(tile_x, px, left_x);
      };
      long long u = u_begin;
      if (args.dependent && args.early) {
        const long long n0 = (u_end - u_begin) < STAGES ? (u_end - u_begin) : STAGES;
        for (int i = 0; i < n0; ++i) load_w(i);
        pdl_wait();
        for (int i = 0; i < n0; ++i) load_x(i);
        u += n0;
      }
      bool ok = true;
      for (; u < u_end; ++u) {
        const long long i = u - u_begin;
        const int st = static_cast<int>(i % STAGES);
        const uint32_t ph = static_cast<uint32_t>(i / STAGES) & 1u;
        if (!mbar_wait(empty_bar(st), ph ^ 1u, abortp)) {
          ok = false;
          break;
        }
        load_w(st);
        load_x(st);
      }
      if (!ok) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_PRODUCER);
        // see the copies in flight land before the block leaves
        const long long done = u - u_begin;
        for (long long i = done > STAGES ? done - STAGES : 0; i < done; ++i)
          drain_wait(full_bar(static_cast<int>(i % STAGES)), static_cast<uint32_t>(i / STAGES) & 1u);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA --
    if (lane == 0) {
      long long n = 0;      // units done
      uint32_t na = 0, nc = 0;  // half units expanded, groups accumulated
      const int ksteps = 2 << args.gshift;  // 16-column steps per group
      bool ok = true;
      long long u = u_begin;
      while (u < u_end && ok) {
        const Segment s = segment_at(u, u_end, per_tile);
        W4Pos p = pos_at(s.tile, u - s.tile_begin);
        for (; u < s.end && ok; ++u, ++n, step(p)) {
          const int st = static_cast<int>(n % STAGES);
          if (!(ok = mbar_wait(full_bar(st), static_cast<uint32_t>(n / STAGES) & 1u, abortp))) break;
          const int ng = groups_in(p.kb);
          for (int g = 0; g < ng; ++g, ++nc) {
            const int half = g >= gps ? 1 : 0;
            const int ab = static_cast<int>(na & 1u);
            if (g == half * gps) {  // first group of a half unit
              if (!(ok = mbar_wait(afull_bar(ab), (na >> 1) & 1u, abortp))) break;
            }
            const int cb = static_cast<int>(nc & 1u);
            if (!(ok = mbar_wait(cempty_bar(cb), ((nc >> 1) & 1u) ^ 1u, abortp))) break;
            tc_fence_after_sync();
            const int k0 = (g - half * gps) * ksteps;  // 16-column step inside the half unit
            const uint32_t a0 = tmem_base + TM_A + ab * 128 + k0 * 8;
            const uint32_t d0 = tmem_base + cb * 2 * MPAD;
            for (int k = 0; k < ksteps; ++k) {
              const int kk = half * 8 + k0 + k;  // 16-column step inside the unit: 4 per 128-byte row of x
              const uint64_t xd = make_smem_desc(smem_base + st * STAGE_BYTES + X_OFF + (kk >> 2) * MPAD * 128, 16, 1024) +
                                  static_cast<uint64_t>(2 * (kk & 3));
              umma_f16_ts(d0, a0 + k * 8, xd, args.idesc, k > 0 ? 1u : 0u);
              umma_f16_ts(d0 + MPAD, a0 + 64 + k * 8, xd, args.idesc, k > 0 ? 1u : 0u);
            }
            umma_commit(cfull_bar(cb));
            if (g == half * gps + gps - 1 || g == ng - 1) {  // last group of the half unit
              umma_commit(aempty_bar(ab));
              ++na;
            }
          }
          if (ok) umma_commit(empty_bar(st));
        }
      }
      if (!ok) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_MMA);
        umma_commit(drain_bar);
        drain_wait(drain_bar, 0);
      }
    }
  } else if (warp < 10) {
    // ------------------------------------------------------------- expand --
    const int quarter = warp & 3;
    const int tsel = (warp - 2) >> 2;  // which of the unit's two tiles
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const uint8_t* const zero = (DUAL && tsel == 1) ? args.zero1 : args.zero0;
    const uint32_t off8 = Nibbles<T>::offset(8);
    long long n = 0;
    uint32_t na = 0;
    bool ok = true;
    long long u = u_begin;
    while (u < u_end && ok) {
      const Segment s = segment_at(u, u_end, per_tile);
      W4Pos p = pos_at(s.tile, u - s.tile_begin);
      const int wrow = row0_of(s.tile) + (DUAL ? row : tsel * 128 + row);
      const bool live = zero != nullptr && wrow < args.rows;
      // zeros of the four 32-column chunks of half unit `h` of unit q: one byte each (repeated where G > 32)
      auto zeros_of = [&](const W4Pos& q, int h) {
        uint32_t z = 0x08080808u;
        if (live) {
          const uint8_t* zp = zero + static_cast<long long>(moe.list[q.a]) * args.groups * args.rows + wrow;
          z = 0u;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            int g = q.kb * gpu_ + h * gps + (c >> args.gshift);
            g = g < args.groups ? g : args.groups - 1;
            z |= static_cast<uint32_t>(zp[static_cast<long long>(g) * args.rows] & 15u) << (8 * c);
          }
        }
        return z;
      };
      uint32_t znext = zeros_of(p, 0);
      for (; u < s.end && ok; ++u, ++n) {
        const int st = static_cast<int>(n % STAGES);
        W4Pos pn = p;
        step(pn);
        const int halves = groups_in(p.kb) > gps ? 2 : 1;
        for (int h = 0; h < halves; ++h, ++na) {
          const uint32_t z = znext;
          if (h + 1 < halves)
            znext = zeros_of(p, 1);
          else if (u + 1 < s.end)
            znext = zeros_of(pn, 0);
          if (h == 0 && !(ok = mbar_wait_warp(full_bar(st), static_cast<uint32_t>(n / STAGES) & 1u, abortp, lane)))
            break;
          const int ab = static_cast<int>(na & 1u);
          const uint32_t src = smem_base + st * STAGE_BYTES + tsel * W4_TILE_BYTES + row * 128;
          uint4 q[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) q[c] = ld_shared_u4(src + (((h * 4 + c) ^ (row & 7)) << 4));
          if (!(ok = mbar_wait_warp(aempty_bar(ab), ((na >> 1) & 1u) ^ 1u, abortp, lane))) break;
          tc_fence_after_sync();
          const uint32_t dst = tmem_base + lane_addr + TM_A + ab * 128 + tsel * 64;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t off = zero != nullptr ? Nibbles<T>::offset((z >> (8 * c)) & 15u) : off8;
            uint32_t r[16];
            expand_word<T>(q[c].x, off, r);
            expand_word<T>(q[c].y, off, r + 4);
            expand_word<T>(q[c].z, off, r + 8);
            expand_word<T>(q[c].w, off, r + 12);
            tmem_st_32x16(dst + c * 16, r);
          }
          tmem_st_wait();
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(afull_bar(ab));
        }
        p = pn;
      }
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_MMA);
    }
  } else {
    // ------------------------------------------- accumulate and finish --
    const int quarter = warp & 3;
    const int col0 = ((warp - 10) >> 2) * COLS;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int ep_tid = threadIdx.x - 320;
    if (args.dependent && args.early) pdl_wait();  // slots, counters and outputs may still be in use
    const T* const scale0 = static_cast<const T*>(args.scale0);
    const T* const scale1 = static_cast<const T*>(DUAL ? args.scale1 : args.scale0);
    uint32_t nc = 0;
    long long u = u_begin;
    if (!DUAL && total == 0) {
      // no token chose any expert: the outputs are the residual, or zero
      const long long all = static_cast<long long>(args.M) * args.rows;
      for (long long i = blockIdx.x * static_cast<long long>(ACC_THREADS) + ep_tid; i < all;
           i += static_cast<long long>(gridDim.x) * ACC_THREADS)
        static_cast<T*>(args.out)[i] =
            args.residual ? static_cast<const T*>(args.residual)[i] : static_cast<T>(0.f);
    }
    while (u < u_end) {
      const Segment s = segment_at(u, u_end, per_tile);
      W4Pos p = pos_at(s.tile, u - s.tile_begin);
      const int r0 = row0_of(s.tile) + row;
      const int r1 = DUAL ? r0 : r0 + 128;
      float v[2][COLS];
#pragma unroll
      for (int c = 0; c < COLS; ++c) v[0][c] = v[1][c] = 0.f;
      auto scales_of = [&](const W4Pos& q, int g, float& a, float& b) {
        const long long o =
            (static_cast<long long>(moe.list[q.a]) * args.groups + q.kb * gpu_ + g) * args.rows;
        a = r0 < args.rows ? static_cast<float>(scale0[o + r0]) : 0.f;
        b = r1 < args.rows ? static_cast<float>(scale1[o + r1]) : 0.f;
      };
      float sa, sb;
      scales_of(p, 0, sa, sb);
      bool ok = true;
      for (; u < s.end && ok; ++u) {
        W4Pos pn = p;
        step(pn);
        const int ng = groups_in(p.kb);
        for (int g = 0; g < ng; ++g, ++nc) {
          const float ca = sa, cb_ = sb;
          if (g + 1 < ng)
            scales_of(p, g + 1, sa, sb);
          else if (u + 1 < s.end)
            scales_of(pn, 0, sa, sb);
          const int cb = static_cast<int>(nc & 1u);
          if (!(ok = mbar_wait_warp(cfull_bar(cb), (nc >> 1) & 1u, abortp, lane))) break;
          tc_fence_after_sync();
          const uint32_t src = tmem_base + lane_addr + cb * 2 * MPAD + col0;
#pragma unroll
          for (int c = 0; c < COLS / 16; ++c) {
            uint32_t x0[16], x1[16];
            tmem_ld_32x16(src + c * 16, x0);
            tmem_ld_32x16(src + MPAD + c * 16, x1);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              v[0][c * 16 + i] = fmaf(ca, __uint_as_float(x0[i]), v[0][c * 16 + i]);
              v[1][c * 16 + i] = fmaf(cb_, __uint_as_float(x1[i]), v[1][c * 16 + i]);
            }
          }
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive(cempty_bar(cb));
        }
        p = pn;
      }
      if (!ok && lane == 0) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_EPILOGUE);
      }
      const int a = DUAL ? static_cast<int>(s.tile / row_tiles) : 0;
      if (DUAL && is_moe) moe_factors(args.moe, args.M, moe.list[a], ep_tid, moe);  // seen behind the next barrier
      const Split sp{total,  ctas,  args.slots, args.counters,
                     args.status, abortp, smem_base,  static_cast<int>(STAGES * STAGE_BYTES / (ACC_THREADS * 16))};
      const int what = settle_segment<2, COLS, MPAD, ACC_THREADS>(v, s, sp, args.M, col0, row, ep_tid);
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
            store_hidden<COLS>(args.act, out + static_cast<long long>(a) * args.M * ld + r0, ld, args.M, col0, v[0],
                               v[1], b0 ? static_cast<float>(b0[r0]) : 0.f, b1 ? static_cast<float>(b1[r0]) : 0.f, mp);
        } else {
          if (r0 < args.rows)
            store_product<COLS>(out + r0, res ? res + r0 : nullptr, ld, args.M, col0, v[0],
                                b0 ? static_cast<float>(b0[r0]) : 0.f, mp);
          if (r1 < args.rows)
            store_product<COLS>(out + r1, res ? res + r1 : nullptr, ld, args.M, col0, v[1],
                                b0 ? static_cast<float>(b0[r1]) : 0.f, mp);
        }
      }
      if (DUAL && is_moe) named_bar_sync(1, ACC_THREADS);  // f and hit are overwritten for the next tile
      u = s.end;
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
