// The experts of a mixture layer for up to 64 tokens on 16-bit weights: gate/up (DUAL = true) and down (DUAL = false).
// The scheme (active experts, zero-padded hidden rows, one long reduction) is in few_token.cuh; the weight path is the
// one of the dense decode kernel (decode_stream.cuh): 128 weight rows x 64 columns per tile through a deep TMA ring,
// tokens as the N dimension of tcgen05.mma, stream-K over units. HBM-bound: every byte of the active experts once.
//   DUAL   units = (active expert, row tile of N, 64 columns of K), two tiles (gate, up) a unit; all M tokens are
//          multiplied (the tensor pipe has the time, see MPAD there) and the epilogue keeps the chosen ones
//   !DUAL  units = (row tile of the hidden size, (active expert, 64 columns of N)): one accumulator for all experts
// Measured (one B200, with the router): 8 experts of 4096 x 14336, one token, top 2: 129 us for 705 MB of chosen weights = 5.4
// TB/s; 64 experts of 2048 x 1408, 64 tokens, top 6: 204 us for 1107 MB = 5.4 TB/s (copy rate 6.56; with 64 tokens an SM also
// takes 8 KB of activations from L2 for every 32 KB of weights).
#pragma once
#include "few_token.cuh"

namespace gmlp {

struct MoeArgs {
  int M;
  int rows;  // weight rows per expert: N for DUAL, K (hidden) otherwise
  int kbt;   // 64-wide reduction blocks per expert
  uint32_t idesc;
  int* status;
  const void* residual;  // [M][rows] or null (DUAL = false)
  void* out;             // DUAL: H[active][M][rows]; else Y[M][rows]
  float* slots;
  int* counters;
  int act;
  int early;  // weights may be streamed before the preceding kernel has finished (the down kernel)
  MoeTable moe;
};

struct MoeMaps {
  CUtensorMap w0, w1, x;
};

// Warps 0 and 1 load and multiply, the others finish tiles: two groups of four, each half of the tokens (with one group, 64
// tokens, 64 experts of 1408 x 2048: gate/up 139 us, the last tiles finished 30,000 clocks after the last product).
constexpr int MOE_EPI = 256;
constexpr int MOE_THREADS = 64 + MOE_EPI;
template <int MPAD, bool DUAL>
__host__ __device__ constexpr int moe_stage_bytes() {
  return (DUAL ? 2 : 1) * 16384 + MPAD * 128;
}
template <int MPAD, bool DUAL>
__host__ __device__ constexpr int moe_stages() {
  constexpr int fit = (232448 - 1024 - 4096) / moe_stage_bytes<MPAD, DUAL>();
  return fit > 12 ? 12 : fit;
}
template <int MPAD, bool DUAL>
constexpr size_t moe_smem_bytes() {
  return static_cast<size_t>(moe_stages<MPAD, DUAL>()) * moe_stage_bytes<MPAD, DUAL>() + 1024;
}

template <int MPAD, bool DUAL, typename T>
__global__ void __launch_bounds__(MOE_THREADS, 1)
moe_stream_kernel(const __grid_constant__ MoeMaps maps, const MoeArgs args) {
  constexpr int NACC = DUAL ? 2 : 1;
  constexpr int STAGES = moe_stages<MPAD, DUAL>();
  constexpr uint32_t W_BYTES = 16384;
  constexpr uint32_t X_OFF = NACC * W_BYTES;
  constexpr uint32_t STAGE_BYTES = moe_stage_bytes<MPAD, DUAL>();
  constexpr uint32_t ACC_COLS = NACC * MPAD;
  constexpr uint32_t TMEM_COLS = 2 * ACC_COLS <= 32 ? 32 : 2 * ACC_COLS <= 64 ? 64 : 2 * ACC_COLS <= 128 ? 128 : 256;

  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bars[2 * STAGES + 5];
  __shared__ uint32_t tmem_base_holder;
  __shared__ int abort_flag;
  __shared__ MoeShared moe;

  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bar_base = smem_u32(bars);
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto tfull_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
  auto tempty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
  const uint32_t drain_bar = bar_base + 8u * (2 * STAGES + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  constexpr int BARS = 2 * STAGES + 5;  // one a thread
  if (threadIdx.x < BARS) {
    const uint32_t bar = bar_base + 8 * threadIdx.x;
    mbar_init(bar, bar >= tempty_bar(0) && bar < drain_bar ? MOE_EPI / 32 : 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (threadIdx.x == 64) abort_flag = 0;
  if (warp == 3 && lane < 3) tma_prefetch_desc(&maps.w0 + lane);
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_base_holder), TMEM_COLS);
    tmem_relinquish();
  }
  // The routing table comes from an earlier kernel. The gate/up kernel waits for that kernel before it lets its own
  // dependent start, so the down kernel may read the table (and stream weights) at once.
  if (!args.early) pdl_wait();
  if (threadIdx.x == 0) pdl_launch_dependents();
  tc_fence_before_sync();
  moe_collect(args.moe, args.M, moe);  // ends with a block barrier
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_base_holder;
  volatile int* abortp = &abort_flag;

  const int row_tiles = (args.rows + 127) / 128;
  const int per_tile = DUAL ? args.kbt : moe.n * args.kbt;
  const Cut cut = make_cut(per_tile * (DUAL ? moe.n * row_tiles : row_tiles), cut_grain(per_tile, (DUAL ? 2 : 1) * 300),
                           gridDim.x);  // 300 clocks: 16 KB into one SM while the others are idle
  const int u_begin = cut_start(cut, blockIdx.x), u_end = cut_start(cut, blockIdx.x + 1);

  if (warp == 0) {
    // ---------------------------------------------------------------- TMA --
    if (lane == 0 && u_begin < u_end) {
      const uint64_t pol_w = l2_policy_evict_first();
      const uint64_t pol_x = l2_policy_evict_last();
      struct Pos {
        int a, rt, kb;
      };
      auto pos_at = [&](int u) {
        Pos p;
        const int tile = u / per_tile, r = u - tile * per_tile;
        if (DUAL) {
          p.a = tile / row_tiles;
          p.rt = tile - p.a * row_tiles;
          p.kb = r;
        } else {
          p.rt = tile;
          p.a = r / args.kbt;
          p.kb = r - p.a * args.kbt;
        }
        return p;
      };
      auto step = [&](Pos& p) {  // unit by unit: no division in the issuing thread's loop
        if (++p.kb < args.kbt) return;
        p.kb = 0;
        if (DUAL) {
          if (++p.rt == row_tiles) {
            p.rt = 0;
            ++p.a;
          }
        } else {
          if (++p.a == moe.n) {
            p.a = 0;
            ++p.rt;
          }
        }
      };
      Pos pw = pos_at(u_begin), px = pw;
      auto load_w = [&](int st) {
        const int y = moe.list[pw.a] * args.rows + pw.rt * 128;
        const uint32_t sw = smem_base + st * STAGE_BYTES;
        mbar_expect_tx(full_bar(st), STAGE_BYTES);
        tma_load_2d_hint(sw, &maps.w0, full_bar(st), pw.kb * 64, y, pol_w);
        if (DUAL) tma_load_2d_hint(sw + W_BYTES, &maps.w1, full_bar(st), pw.kb * 64, y, pol_w);
        step(pw);
      };
      auto load_x = [&](int st) {
        tma_load_2d_hint(smem_base + st * STAGE_BYTES + X_OFF, &maps.x, full_bar(st), px.kb * 64,
                         DUAL ? 0 : px.a * args.M, pol_x);
        step(px);
      };
      int u = u_begin;
      if (args.early) {
        const int n0 = (u_end - u_begin) < STAGES ? (u_end - u_begin) : STAGES;
        for (int i = 0; i < n0; ++i) load_w(i);
        pdl_wait();
        for (int i = 0; i < n0; ++i) load_x(i);
        u += n0;
      }
      int st = (u - u_begin) % STAGES;
      uint32_t ph = static_cast<uint32_t>((u - u_begin) / STAGES) & 1u;
      bool ok = true;
      for (; u < u_end; ++u) {
        if (!mbar_wait(empty_bar(st), ph ^ 1u, abortp)) {
          ok = false;
          break;
        }
        load_w(st);
        load_x(st);
        if (++st == STAGES) {
          st = 0;
          ph ^= 1u;
        }
      }
      if (!ok) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_PRODUCER);
        const int done = u - u_begin;  // see the copies in flight land before the block leaves
        for (int i = done > STAGES ? done - STAGES : 0; i < done; ++i)
          drain_wait(full_bar(i % STAGES), static_cast<uint32_t>(i / STAGES) & 1u);
      }
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA --
    if (lane == 0) {
      int st = 0, seg = 0;
      uint32_t ph = 0;
      bool ok = true;
      int u = u_begin;
      while (u < u_end && ok) {
        const Segment s = segment_at(u, u_end, per_tile);
        const int acc = seg & 1;
        if (!(ok = mbar_wait(tempty_bar(acc), ((seg >> 1) & 1u) ^ 1u, abortp))) break;
        tc_fence_after_sync();
        const uint32_t d = tmem_base + acc * ACC_COLS;
        uint32_t accum = 0u;
        for (; u < s.end; ++u) {
          if (!(ok = mbar_wait(full_bar(st), ph, abortp))) break;
          tc_fence_after_sync();
          const uint32_t sw = smem_base + st * STAGE_BYTES;
          const uint64_t xd = make_smem_desc(sw + X_OFF, 16, 1024);
          const uint64_t w0 = make_smem_desc(sw, 16, 1024), w1 = make_smem_desc(sw + W_BYTES, 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            umma_f16(d, w0 + static_cast<uint64_t>(2 * k), xd + static_cast<uint64_t>(2 * k), args.idesc, accum);
            if (DUAL)
              umma_f16(d + MPAD, w1 + static_cast<uint64_t>(2 * k), xd + static_cast<uint64_t>(2 * k), args.idesc, accum);
            accum = 1u;
          }
          umma_commit(empty_bar(st));
          if (++st == STAGES) {
            st = 0;
            ph ^= 1u;
          }
        }
        if (ok) umma_commit(tfull_bar(acc));
        ++seg;
      }
      if (!ok) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_MMA);
        umma_commit(drain_bar);
        drain_wait(drain_bar, 0);
      }
    }
  } else {
    // ------------------------------------------------------------ epilogue --
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>(quarter * 32) << 16;
    const int ep_tid = threadIdx.x - 64;
    constexpr int COLS = MPAD / (MOE_EPI / 128);
    const int col0 = ((warp - 2) >> 2) * COLS;
    if (args.early) pdl_wait();  // slots, counters and outputs may still be in use by the preceding grid
    T* const out = static_cast<T*>(args.out);
    const T* const res = static_cast<const T*>(args.residual);
    const long long ld = args.rows;
    if (!DUAL && cut.total == 0) {
      // no token chose any expert: the outputs are the residual, or zero
      const long long all = static_cast<long long>(args.M) * args.rows;
      for (long long i = blockIdx.x * static_cast<long long>(MOE_EPI) + ep_tid; i < all;
           i += gridDim.x * static_cast<long long>(MOE_EPI))
        out[i] = res ? res[i] : static_cast<T>(0.f);
    }
    const Split sp{cut, args.M, reinterpret_cast<float4*>(args.slots), args.counters, abortp};
    constexpr int ITEMS = MPAD > 16 ? 4 : 1;
    auto emit_tile = [&](int tile, int begin, const Join& join) {
      if (DUAL) {
        const int a = tile / row_tiles, row0 = (tile - a * row_tiles) * 128;
        moe_factors(args.moe, args.M, moe.list[a], ep_tid, moe);
        named_bar_sync(1, MOE_EPI);
        T* const oa = out + static_cast<long long>(a) * args.M * ld;
        finish_tile<NACC, true, MPAD, MOE_EPI, ITEMS>(begin, join, sp, ep_tid,
                                           [&](int, int r, int i, const float4& gate, const float4& up) {
          if (row0 + r < args.rows) emit_hidden(oa + row0 + r, ld, args.M, i, gate, up, nullptr, 0.f, 0.f, args.act, &moe);
        });
      } else {
        finish_tile<NACC, false, MPAD, MOE_EPI, ITEMS>(begin, join, sp, ep_tid,
                                            [&](int, int r, int i, const float4& v, const float4&) {
          const int wr = tile * 128 + r;
          if (wr < args.rows) emit_product(out + wr, res ? res + wr : nullptr, ld, args.M, i, v, nullptr, 0.f, &moe);
        });
      }
      named_bar_sync(1, MOE_EPI);  // the slot, f and hit are free for the next tile
    };
    Pending pending;
    bool alive = true;
    int seg = 0;
    int u = u_begin;
    while (u < u_end) {
      const Segment s = segment_at(u, u_end, per_tile);
      const int acc = seg & 1;
      if (!mbar_wait_warp(tfull_bar(acc), (seg >> 1) & 1u, abortp, lane) && lane == 0) {
        abort_flag = 1;
        atomicCAS(args.status, 0, GMLP_DEV_TIMEOUT_EPILOGUE);
      }
      tc_fence_after_sync();
      float v[NACC][COLS];
      uint32_t r[NACC][COLS];
#pragma unroll
      for (int t = 0; t < NACC; ++t) tmem_ld_cols<COLS>(tmem_base + acc * ACC_COLS + lane_addr + t * MPAD + col0, r[t]);
      tmem_ld_wait();
#pragma unroll
      for (int t = 0; t < NACC; ++t)
#pragma unroll
        for (int c = 0; c < COLS; ++c) v[t][c] = __uint_as_float(r[t][c]);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty_bar(acc));
      if (!(alive = end_segment<NACC, COLS, MPAD, MOE_EPI>(v, s, sp, col0, row, ep_tid, pending, emit_tile))) break;
      u = s.end;
      ++seg;
    }
    if (alive) end_units<MOE_EPI>(pending, per_tile, sp, ep_tid, emit_tile);
  }

  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    tc_fence_after_sync();
    tmem_dealloc(tmem_base, TMEM_COLS);
  }
}

// ---- router ----
// logits l[t][e] = x_t . Wr_e; p = softmax(l); the top_k largest (equal ones: lowest index first; NaN ranks lowest) with
// weights p, or p divided by their sum. A cluster of C blocks per token: each warp takes two experts
// a pass, products exact and summed in fp64: a logit is off by at most K 2^-53 of sum |x_k w_k|, however much of it
// cancels, so that a choice next to a border is that of the exact sums. (Eight products summed in fp32 at a time are off by
// some 2^-24 of sum |x_k w_k|: four channels of 3e4 that cancel turned choices over and moved weights by 6e-3. That took
// 4.4, 5.2 and 32 us for the cases below; products converted one by one instead of widened: 6.0, 8.6 and 62.) The
// logits go to the first block's shared memory (distributed shared memory), whose first warp selects. Latency-bound where
// tokens are few: C spreads the 2 E K bytes of a token over SMs.
// Measured: 8 experts x 4096, one token 4.2 us; 64 x 2048, 64 tokens 7.5; 512 x 4096, 64 tokens 57; 128 x 2048,
// 2048 tokens 174.
constexpr int ROUTE_THREADS = 256;
struct RouteArgs {
  const void* x;
  const void* w;
  long long ldx;
  int M, K, E, top_k, renormalize;
  int* ids;
  float* weights;
};
// Order of logits as an integer whose low 9 bits are the index, larger for lower indices: one maximum finds the largest
// logit and, among equal ones (equal in 43 of the 52 fraction bits), the lowest index. NaN ranks below -inf.
__device__ __forceinline__ unsigned long long sort_key(double v, int e) {
  unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v));
  b = (b >> 63) ? ~b : b | 0x8000000000000000ull;
  if (v != v) b = 0x0008000000000000ull;  // below the key of -inf, above that of a removed entry (0)
  return (b & ~511ull) | static_cast<unsigned long long>(511 - e);
}
// A 16-bit value (as the float it was converted to) times 2^-896, exactly, subnormals too: its exponent and fraction bits
// moved to a double's place, with the exponent's bias left as it is. Not for infinities and NaNs.
constexpr double WIDENED = 0x1p896;
__device__ __forceinline__ double widened(float v) {
  return __hiloint2double((__float_as_int(v) >> 3) & static_cast<int>(0x8fffffffu), 0);
}
// A lane's columns of TOKENS x EXPERTS dot products in CHAINS sums each. FAST: the weights widened; `finite` is
// 0 times every weight, a NaN if one is not finite.
template <bool FAST, int CHAINS, int TOKENS, int EXPERTS, typename T>
__device__ __forceinline__ void route_columns(const T* const (&x)[TOKENS], const T* const (&w)[EXPERTS], int K, int lane,
                                              double (&s)[TOKENS][EXPERTS], f32x2& finite) {
  double t[CHAINS][TOKENS][EXPERTS];
#pragma unroll
  for (int c = 0; c < CHAINS; ++c)
#pragma unroll
    for (int m = 0; m < TOKENS; ++m)
#pragma unroll
      for (int e = 0; e < EXPERTS; ++e) t[c][m][e] = 0.0;
  constexpr int UNROLL = !FAST ? 1 : TOKENS == 1 ? 4 : 2;
#pragma unroll UNROLL
  for (int k = lane * 8; k < K; k += 256) {
    float a[TOKENS][8], b[EXPERTS][8];
#pragma unroll
    for (int m = 0; m < TOKENS; ++m) load8(x[m] + k, a[m]);
#pragma unroll
    for (int e = 0; e < EXPERTS; ++e) load8(w[e] + k, b[e]);
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int e = 0; e < EXPERTS; ++e) {
        const double u = FAST ? widened(b[e][i]) : b[e][i];
#pragma unroll
        for (int m = 0; m < TOKENS; ++m) t[i % CHAINS][m][e] = fma(static_cast<double>(a[m][i]), u, t[i % CHAINS][m][e]);
        if (FAST && i % 2 == 0) finite = f2_fma(f2_pack(b[e][i], b[e][i + 1]), 0ull, finite);
      }
  }
#pragma unroll
  for (int m = 0; m < TOKENS; ++m)
#pragma unroll
    for (int e = 0; e < EXPERTS; ++e) {
      double v = t[0][m][e] + t[1][m][e];
      if (CHAINS == 4) v += t[CHAINS - 2][m][e] + t[CHAINS - 1][m][e];
      s[m][e] = FAST ? v * WIDENED : v;
    }
}
// Widened products underflow below 2^-178, and infinities and NaNs cannot be widened: a sum that this can have touched (by
// more than 2^-47 of it) is made again with converted weights. The same additions in the same order: equal rows have
// equal sums.
template <int CHAINS, int TOKENS, int EXPERTS, typename T>
__device__ __forceinline__ void route_dots(const T* const (&x)[TOKENS], const T* const (&w)[EXPERTS], int K, int lane,
                                           double (&s)[TOKENS][EXPERTS]) {
  f32x2 finite = 0ull;
  route_columns<true, CHAINS, TOKENS, EXPERTS>(x, w, K, lane, s, finite);
  float z0, z1;
  f2_unpack(finite, z0, z1);
  bool again = z0 + z1 != 0.f;
#pragma unroll
  for (int m = 0; m < TOKENS; ++m) {
    bool small = false;
#pragma unroll
    for (int e = 0; e < EXPERTS; ++e) small |= fabs(s[m][e]) < 0x1p-100;
    if (small)  // unless x is zero there: a row of padding
      for (int k = lane * 8; k < K && !again; k += 256) {
        const uint4 v = *reinterpret_cast<const uint4*>(x[m] + k);
        again = ((v.x | v.y | v.z | v.w) & 0x7fff7fffu) != 0u;
      }
  }
  if (__any_sync(0xffffffffu, again)) route_columns<false, CHAINS, TOKENS, EXPERTS>(x, w, K, lane, s, finite);
}
// PER: experts per lane of the selecting warp. TOKENS: tokens of a cluster, which share the loads and the widening of the
// router's rows.
// Four sums a product where latency counts, two where more blocks per SM do (64 tokens: 64 x 2048 7.4 us with four, 8.2
// with two; 512 x 4096 73 and 57).
template <typename T, int PER, int TOKENS>
__global__ void __launch_bounds__(ROUTE_THREADS)
moe_route_kernel(const RouteArgs args) {
  constexpr int CHAINS = TOKENS == 1 && PER <= 4 ? 4 : 2;
  __shared__ double shared_logits[TOKENS][32 * PER];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint32_t rank, size;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int first = static_cast<int>(blockIdx.x / size) * TOKENS;
  pdl_launch_dependents();
  cluster_sync_all();  // the first block's shared memory is written below: it has to be there
  pdl_wait();
  const T* x[TOKENS];
#pragma unroll
  for (int m = 0; m < TOKENS; ++m)  // (a token behind the last one is the last one again)
    x[m] = static_cast<const T*>(args.x) + (first + m < args.M ? first + m : args.M - 1) * args.ldx;
  const uint32_t dst0 = mapa_shared(smem_u32(shared_logits), 0);
  // experts warp-major over the cluster, two at a time: they share the loads of x
  const int warps = size * (ROUTE_THREADS / 32);
  auto put = [&](double v, int m, int e) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(dst0 + 8u * (m * 32 * PER + e)), "d"(v) : "memory");
  };
  for (int e = rank * (ROUTE_THREADS / 32) + warp; e < args.E; e += 2 * warps) {
    const T* const w0 = static_cast<const T*>(args.w) + static_cast<long long>(e) * args.K;
    if (e + warps < args.E) {
      const T* const w[2] = {w0, w0 + static_cast<long long>(warps) * args.K};
      double s[TOKENS][2];
      route_dots<CHAINS, TOKENS, 2>(x, w, args.K, lane, s);
#pragma unroll
      for (int m = 0; m < TOKENS; ++m) {
        put(s[m][0], m, e);
        put(s[m][1], m, e + warps);
      }
    } else {
      const T* const w[1] = {w0};
      double s[TOKENS][1];
      route_dots<CHAINS, TOKENS, 1>(x, w, args.K, lane, s);
#pragma unroll
      for (int m = 0; m < TOKENS; ++m) put(s[m][0], m, e);
    }
  }
  __syncwarp();
  cluster_sync_all();
  const int token = first + warp;  // of the first block, a warp for each token
  if (rank != 0 || warp >= TOKENS || token >= args.M) return;
  const double* const logits = shared_logits[warp];
  unsigned long long key[PER];
  float ex[PER];
  double top = -INFINITY;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    const double l = e < args.E ? logits[e] : 0.0;
    key[i] = e < args.E ? sort_key(l, e) : 0ull;
    if (e < args.E && (l > top || l != l)) top = l;  // a NaN stays the maximum and makes every weight of the token NaN
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double v = __shfl_xor_sync(0xffffffffu, top, o);
    if (v > top || v != v) top = v;
  }
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = i * 32 + lane;
    ex[i] = e < args.E ? expf(static_cast<float>(logits[e] - top)) : 0.f;
    sum += ex[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  float mine = 0.f, chosen = 0.f;  // lane j keeps choice j
  int id = 0;
  for (int j = 0; j < args.top_k; ++j) {
    unsigned long long best = key[0];
#pragma unroll
    for (int i = 1; i < PER; ++i) best = key[i] > best ? key[i] : best;
    const uint32_t hi = static_cast<uint32_t>(best >> 32);
    const uint32_t mhi = __reduce_max_sync(0xffffffffu, hi);
    const uint32_t mlo = __reduce_max_sync(0xffffffffu, hi == mhi ? static_cast<uint32_t>(best) : 0u);
    const unsigned long long win = (static_cast<unsigned long long>(mhi) << 32) | mlo;
    const int e = 511 - static_cast<int>(mlo & 511u);
    float w = 0.f;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (key[i] == win) {  // no two keys are equal: the index is in them
        w = ex[i];
        key[i] = 0ull;
      }
    w = __shfl_sync(0xffffffffu, w, e & 31);
    chosen += w;
    if (lane == j) {
      mine = w;
      id = e;
    }
  }
  if (lane < args.top_k) {
    args.ids[token * args.top_k + lane] = id;
    args.weights[token * args.top_k + lane] = mine / (args.renormalize ? chosen : sum);
  }
}

}  // namespace gmlp
