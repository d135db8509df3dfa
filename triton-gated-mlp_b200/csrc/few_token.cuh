// Pieces shared by the few-token (M <= 64) weight-streaming kernels on 4-bit weights (w4_stream.cuh) and on
// mixtures of experts (moe_stream.cuh): which experts a call streams, how the partial sums of a row tile
// that several CTAs worked on are joined, and the epilogues.
//
// Mixture of experts. Every kernel of the layer derives the set of experts that at least one token chose from
// the routing table itself (at most 64 x 32 entries), in ascending order: "active" experts a = 0 .. n-1. The
// gate/up kernel streams the rows of the active experts only and writes, for every active expert and EVERY
// token, the hidden row scaled by the token's weight for that expert, zero where the token did not choose it:
//   H[a][t][:] = f(t, a) * act(x_t Wg_a^T) * (x_t Wu_a^T),   f = w(t, a) / wmax(t)
// The weighted sum over a token's experts then is one long reduction over (expert, column) in the down kernel,
//   y_t = wmax(t) * sum_a H[a][t][:] . Wd_a^T
// so that it needs no gather, no permutation, no atomics and no pass that adds partial outputs. The zeros cost a
// write and an L2 read of n x T x N hidden values, about 1 % of the weight bytes (T = 64, 128 experts of
// 2048 x 768: 12.6 MB against 1.2 GB). Dividing by the token's largest weight keeps H in the range of 16-bit
// values whatever the scale of the weights (fp16 would lose bits to subnormals for weights of 1e-2).
#pragma once
#include "decode_stream.cuh"

namespace gmlp {

constexpr int FEW_MAX_TOKENS = 64;
constexpr int MOE_MAX_EXPERTS = 512;
constexpr int MOE_MAX_TOPK = 32;

struct MoeTable {
  const int* ids;        // [M, top_k]; null: a dense call (one "expert", weight 1). Entries outside [0, experts) are skipped
  const float* weights;  // [M, top_k]
  int top_k;
  int experts;
};

struct MoeShared {
  uint32_t seen[MOE_MAX_EXPERTS / 32];
  uint16_t list[MOE_MAX_EXPERTS];  // active experts, ascending
  int n;
  float wmax[FEW_MAX_TOKENS];  // largest |weight| of the token's valid choices; 1 for a dense call
  float f[FEW_MAX_TOKENS];     // this tile's expert: w(t, e) / wmax(t)
  int hit[FEW_MAX_TOKENS];     // this tile's expert was chosen by the token
};

// All threads of the block; ends with a barrier.
__device__ __forceinline__ void moe_collect(const MoeTable& t, int M, MoeShared& s) {
  const int tid = threadIdx.x;
  if (t.ids == nullptr) {
    if (tid == 0) {
      s.n = 1;
      s.list[0] = 0;
    }
    __syncthreads();
    return;
  }
  for (int i = tid; i < MOE_MAX_EXPERTS / 32; i += blockDim.x) s.seen[i] = 0u;
  __syncthreads();
  for (int i = tid; i < M * t.top_k; i += blockDim.x) {
    const int e = t.ids[i];
    if (static_cast<unsigned>(e) < static_cast<unsigned>(t.experts)) atomicOr(&s.seen[e >> 5], 1u << (e & 31));
  }
  for (int m = tid; m < M; m += blockDim.x) {
    float w = 0.f;
    for (int j = 0; j < t.top_k; ++j) {
      if (static_cast<unsigned>(t.ids[m * t.top_k + j]) >= static_cast<unsigned>(t.experts)) continue;
      const float a = fabsf(t.weights[m * t.top_k + j]);
      w = (a > w || a != a) ? a : w;  // a NaN stays: it belongs in the token's output
    }
    s.wmax[m] = w;
  }
  __syncthreads();
  if (tid < 32) {
    const uint32_t word = tid < MOE_MAX_EXPERTS / 32 ? s.seen[tid] : 0u;
    int before = __popc(word);
    const int own = before;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, before, o);
      if (tid >= o) before += v;
    }
    if (tid == 31) s.n = before;
    int at = before - own;
    for (uint32_t w = word; w != 0u; w &= w - 1u)
      s.list[at++] = static_cast<uint16_t>(tid * 32 + __ffs(static_cast<int>(w)) - 1);
  }
  __syncthreads();
}

// f and hit of expert `e`, by threads 0 .. 63 of the epilogue; the caller puts a barrier behind it.
__device__ __forceinline__ void moe_factors(const MoeTable& t, int M, int e, int ep_tid, MoeShared& s) {
  if (ep_tid >= M) return;
  float w = 0.f;
  int hit = 0;
  for (int j = 0; j < t.top_k; ++j)
    if (t.ids[ep_tid * t.top_k + j] == e) {
      w += t.weights[ep_tid * t.top_k + j];  // the same expert twice in a token adds
      hit = 1;
    }
  const float top = s.wmax[ep_tid];
  s.f[ep_tid] = top == 0.f ? 0.f : w / top;
  s.hit[ep_tid] = hit;
}

// Gate activations at fp32 accuracy (the GEMM epilogues use tanh.approx, whose 2^-11 is as large as fp16's own
// rounding; here the epilogue runs once per 128 x 64 outputs and costs nothing).
template <int ACT>
__device__ __forceinline__ float act_fine(float x) {
  if (ACT == ACT_SILU) return __fdividef(x, 1.0f + __expf(-x));
  if (ACT == ACT_RELU) return x < 0.0f ? 0.0f : x;  // a NaN stays one
  if (ACT == ACT_GELU) return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
  if (ACT == ACT_SIGMOID) return __fdividef(1.0f, 1.0f + __expf(-x));
  if (ACT == ACT_TANH) return tanhf(x);
  if (ACT == ACT_LEAKY_RELU) return x > 0.0f ? x : 0.01f * x;
  return x;
}

// One weight row of the gate/up kernel: hidden values of tokens col0 .. col0 + COLS - 1 (those below M).
template <int ACT, int COLS, typename T>
__device__ __forceinline__ void store_hidden_act(T* po, long long ld, int M, int col0, const float* gate,
                                                 const float* up, float b0, float b1, const MoeShared* moe) {
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    const int m = col0 + c;
    if (m < M) {
      float h = act_fine<ACT>(gate[c] + b0) * (up[c] + b1);
      if (moe != nullptr) h = moe->hit[m] ? h * moe->f[m] : 0.f;
      po[static_cast<long long>(m) * ld] = static_cast<T>(h);
    }
  }
}
template <int COLS, typename T>
__device__ __forceinline__ void store_hidden(int act, T* po, long long ld, int M, int col0, const float* gate,
                                             const float* up, float b0, float b1, const MoeShared* moe) {
  switch (act) {  // outside the unrolled token loop: one body per activation, not COLS switches
    case ACT_SILU: store_hidden_act<ACT_SILU, COLS>(po, ld, M, col0, gate, up, b0, b1, moe); break;
    case ACT_NONE: store_hidden_act<ACT_NONE, COLS>(po, ld, M, col0, gate, up, b0, b1, moe); break;
    case ACT_RELU: store_hidden_act<ACT_RELU, COLS>(po, ld, M, col0, gate, up, b0, b1, moe); break;
    case ACT_GELU: store_hidden_act<ACT_GELU, COLS>(po, ld, M, col0, gate, up, b0, b1, moe); break;
    case ACT_SIGMOID: store_hidden_act<ACT_SIGMOID, COLS>(po, ld, M, col0, gate, up, b0, b1, moe); break;
    case ACT_TANH: store_hidden_act<ACT_TANH, COLS>(po, ld, M, col0, gate, up, b0, b1, moe); break;
    default: store_hidden_act<ACT_LEAKY_RELU, COLS>(po, ld, M, col0, gate, up, b0, b1, moe); break;
  }
}
// One weight row of a plain product: out[m] = v[m] (* wmax[m]) + bias + residual[m].
template <int COLS, typename T>
__device__ __forceinline__ void store_product(T* po, const T* pr, long long ld, int M, int col0, const float* v,
                                              float bias, const MoeShared* moe) {
#pragma unroll
  for (int c = 0; c < COLS; ++c) {
    const int m = col0 + c;
    if (m < M) {
      float o = (moe != nullptr ? v[c] * moe->wmax[m] : v[c]) + bias;
      if (pr) o += static_cast<float>(pr[static_cast<long long>(m) * ld]);
      po[static_cast<long long>(m) * ld] = static_cast<T>(o);
    }
  }
}

// ---- stream-K: the units [u_begin, u_end) of a CTA, cut at row tile borders into segments ----
struct Segment {
  long long tile, begin, end;  // row tile, and this CTA's units of it
  long long tile_begin, tile_end;
};
__device__ __forceinline__ Segment segment_at(long long u, long long u_end, long long per_tile) {
  Segment s;
  s.tile = u / per_tile;
  s.begin = u;
  s.tile_begin = s.tile * per_tile;
  s.tile_end = s.tile_begin + per_tile;
  s.end = s.tile_end < u_end ? s.tile_end : u_end;
  return s;
}

struct Split {
  long long total;  // units of the launch
  long long ctas;   // CTAs that have units (at most one per unit)
  float* slots;     // [ctas][NT][COLS_ALL / 4][128] float4: a CTA's partial row tile
  int* counters;    // [row tiles]: units whose partial sums are in the slots; zero before and after the launch
  int* status;
  volatile int* abortp;
  uint32_t ring;    // shared memory free for staging while a CTA finishes its last segment
  int ring_pieces;  // 16-byte pieces per thread that the ring holds
};

enum : int { SETTLE_ABORT = 0, SETTLE_EMIT = 1, SETTLE_SENT = 2 };

// Joins a row tile's partial sums. Called by all THREADS epilogue threads (a multiple of 128: thread = weight row
// `row` of the tile, column group of COLS tokens starting at col0) with this CTA's sums of segment `s`.
// A tile that was not cut is complete. Of a cut tile the CTA that holds the first units is the owner: for it
// the tile is the last thing it works on, while the others met it first and published their part before. It
// waits (bounded) until all other units are counted, adds the parts in CTA order (the result does not depend
// on arrival) and clears the counter. Only the float4 columns below M travel: with one token that is a
// quarter of a 16-column tile.
template <int NT, int COLS, int COLS_ALL, int THREADS>
__device__ __forceinline__ int settle_segment(float (&v)[NT][COLS], const Segment& s, const Split& sp, int M,
                                              int col0, int row, int ep_tid) {
  // vote: all epilogue threads leave the same way even if the abort flag flips between their reads
  if (named_bar_or(1, THREADS, *sp.abortp != 0)) return SETTLE_ABORT;
  const bool first = s.begin == s.tile_begin;
  if (first && s.end == s.tile_end) return SETTLE_EMIT;
  constexpr long long SLOT4 = static_cast<long long>(NT) * (COLS_ALL / 4) * 128;
  const int left = M - col0;
  const int nq = left <= 0 ? 0 : ((left < COLS ? left : COLS) + 3) / 4;
  if (!first) {
    float4* const slot = reinterpret_cast<float4*>(sp.slots) + blockIdx.x * SLOT4;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < COLS / 4; ++i)
        if (i < nq)
          slot[(t * (COLS_ALL / 4) + col0 / 4 + i) * 128 + row] =
              make_float4(v[t][4 * i], v[t][4 * i + 1], v[t][4 * i + 2], v[t][4 * i + 3]);
    __threadfence();
    named_bar_sync(1, THREADS);
    if (ep_tid == 0) atomicAdd(sp.counters + s.tile, static_cast<int>(s.end - s.begin));
    return SETTLE_SENT;
  }
  if (ep_tid == 0) {
    const int need = static_cast<int>(s.tile_end - s.end);
    const volatile int* cnt = sp.counters + s.tile;
    const long long t0 = clock64();
    while (*cnt != need) {
      if (*sp.abortp != 0 || clock64() - t0 > WAIT_LIMIT_CYCLES) {
        *sp.abortp = 1;
        atomicCAS(sp.status, 0, GMLP_DEV_TIMEOUT_EPILOGUE);
        break;
      }
      __nanosleep(32);
    }
    __threadfence();
  }
  if (named_bar_or(1, THREADS, *sp.abortp != 0)) return SETTLE_ABORT;
  const long long c_first = ((s.tile_begin + 1) * sp.ctas - 1) / sp.total;
  const long long c_last = (s.tile_end * sp.ctas - 1) / sp.total;
  const int per = NT * nq;  // pieces of one contributor and thread
  if (per > 0) {
    const int batch = sp.ring_pieces / per;  // contributors fetched per round trip
    auto stage = [&](int k) { return sp.ring + static_cast<uint32_t>(k * THREADS + ep_tid) * 16u; };
    for (long long cb = c_first + 1; cb <= c_last; cb += batch) {
      const long long ce = cb + batch - 1 < c_last ? cb + batch - 1 : c_last;
      int k = 0;
      for (long long c = cb; c <= ce; ++c) {
        const float4* slot = reinterpret_cast<const float4*>(sp.slots) + c * SLOT4;
#pragma unroll
        for (int t = 0; t < NT; ++t)
          for (int i = 0; i < nq; ++i, ++k)
            cp_async_16(stage(k), slot + (t * (COLS_ALL / 4) + col0 / 4 + i) * 128 + row);
      }
      cp_async_wait_all();
      k = 0;
      for (long long c = cb; c <= ce; ++c) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int i = 0; i < COLS / 4; ++i)
            if (i < nq) {
              const float4 q = ld_shared_f4(stage(k++));
              v[t][4 * i] += q.x;
              v[t][4 * i + 1] += q.y;
              v[t][4 * i + 2] += q.z;
              v[t][4 * i + 3] += q.w;
            }
      }
    }
  }
  if (ep_tid == 0) sp.counters[s.tile] = 0;  // ready for the next call
  return SETTLE_EMIT;
}

// Bounded wait that looks at no abort flag: a thread that gives up uses it to see its own copies in flight land
// (or a last commit arrive) before its CTA leaves.
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait_suspend(bar, parity, 4000u))
    if (clock64() - t0 > 40000000LL) return;
}

}  // namespace gmlp
