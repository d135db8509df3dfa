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
  uint32_t* const top = reinterpret_cast<uint32_t*>(s.wmax);  // magnitudes as integers: the same order, NaN on top
  for (int i = tid; i < MOE_MAX_EXPERTS / 32; i += blockDim.x) s.seen[i] = 0u;
  for (int i = tid; i < FEW_MAX_TOKENS; i += blockDim.x) top[i] = 0u;
  __syncthreads();
  for (int i = tid; i < M * t.top_k; i += blockDim.x) {  // all entries at once: a token's own would be a chain of loads
    const int e = __ldcg(t.ids + i);  // (past L1: the kernel may have started before this SM saw the table last)
    const uint32_t w = __float_as_uint(__ldcg(t.weights + i)) & 0x7fffffffu;
    if (static_cast<unsigned>(e) < static_cast<unsigned>(t.experts)) {
      atomicOr(&s.seen[e >> 5], 1u << (e & 31));
      atomicMax(&top[i / t.top_k], w);  // a NaN belongs in the token's output
    }
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
#pragma unroll 8
  for (int j = 0; j < t.top_k; ++j) {
    const float x = __ldcg(t.weights + ep_tid * t.top_k + j);
    if (__ldcg(t.ids + ep_tid * t.top_k + j) == e) {
      w += x;  // the same expert twice in a token adds
      hit = 1;
    }
  }
  const float top = s.wmax[ep_tid];
  s.f[ep_tid] = top == 0.f ? 0.f : w / top;
  s.hit[ep_tid] = hit;
}

// ---- stream-K: the launch's units in row-tile-major order, cut into one contiguous range per CTA; a range is cut at row
// tile borders into segments. All in 32 bits (the host refuses larger calls): a 64-bit division is a hundred
// instructions, and a single warp at the start of a kernel takes a microsecond for four of them. ----
struct Cut {
  int total;      // units of the launch
  int grain;      // units that are not cut apart: 1, or a whole row tile where that is short
  int ctas;       // CTAs that have units (at most one per grain)
  int each, odd;  // grains per CTA; the first `odd` CTAs have one more
};
__host__ __device__ __forceinline__ Cut make_cut(int total, int grain, int grid) {
  Cut c;
  const int grains = grain == 1 ? total : total / grain;  // (a tile is the grain: total is a multiple)
  c.total = total;
  c.grain = grain;
  c.ctas = grains < grid ? grains : grid;
  c.each = c.ctas > 0 ? grains / c.ctas : 0;
  c.odd = grains - c.each * c.ctas;
  return c;
}
__device__ __forceinline__ int cut_start(const Cut& c, int cta) {
  return cta >= c.ctas ? c.total : (cta * c.each + (cta < c.odd ? cta : c.odd)) * c.grain;
}
__device__ __forceinline__ int cut_owner(const Cut& c, int unit) {  // the CTA that has the unit; only where tiles are cut
  const int big = c.odd * (c.each + 1);
  return unit < big ? unit / (c.each + 1) : c.odd + (unit - big) / c.each;
}
// Joining the parts of a tile takes some 6,000 clocks after its last unit (publish, see the others' parts, fetch them). Where
// one CTA streams the whole tile in less, tiles stay whole (device time with and without that rule: 4-bit MLP, 3 tokens,
// K=512, N=896, 10.4 against 13.1 us; 18 experts of 576 x 320, 5 tokens, top 3, with the router, 23.5 against 25.6).
constexpr int JOIN_CLOCKS = 6000;
__host__ __device__ __forceinline__ int cut_grain(int per_tile, int unit_clocks) {
  return per_tile > 0 && per_tile <= JOIN_CLOCKS / unit_clocks ? per_tile : 1;
}

// A warp's 32 lanes (rows) of COLS 32-bit columns.
template <int COLS>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t* r) {
  if constexpr (COLS == 4) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(taddr)
                 : "memory");
  } else {
#pragma unroll
    for (int c = 0; c < COLS; c += 8)
      asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                   : "=r"(r[c]), "=r"(r[c + 1]), "=r"(r[c + 2]), "=r"(r[c + 3]), "=r"(r[c + 4]), "=r"(r[c + 5]),
                     "=r"(r[c + 6]), "=r"(r[c + 7])
                   : "r"(taddr + c)
                   : "memory");
  }
}
struct Segment {
  int tile, begin, end;  // row tile, and this CTA's units of it
  int tile_begin, tile_end;
};
__device__ __forceinline__ Segment segment_at(int u, int u_end, int per_tile) {
  Segment s;
  s.tile = u / per_tile;
  s.begin = u;
  s.tile_begin = s.tile * per_tile;
  s.tile_end = s.tile_begin + per_tile;
  s.end = s.tile_end < u_end ? s.tile_end : u_end;
  return s;
}

// ---- end of a segment: sums to a slot, from there to the output ----
// A CTA's sums of a row tile go to a slot in global memory (L2), [NT][COLS_ALL / 4][128] float4 = four tokens of one
// weight row, and from there through the epilogue to the output, in a loop of a few hundred instructions. (Straight
// from the registers the epilogue is unrolled over all of a thread's tokens, 10 KB of code that run once per tile:
// fetching it took 9,500 clocks at 64 tokens.) A tile whose units lie in several CTAs is finished by all of them together:
// each publishes its part as soon as it has it, and when it is through with its units it waits (bounded) for the
// others' parts and finishes an equal share of the tile's rows and tokens, adding the parts in CTA order (the result does
// not depend on arrival). (With one owner per tile that fetched all parts, 64 tokens and 9 CTAs per tile, the owner
// alone took 26,000 clocks.) A CTA waits only after it has published everything it owes, and not for long: other CTAs
// of the launch may not have an SM yet (another stream's kernel, or another launch of this one, may hold them), and two
// launches whose CTAs kept their SMs until all of their own had come could stop one another. A CTA that has waited
// GIVE_UP_CLOCKS leaves its share to those that come later; the last one to come never waits.
// Only the float4 columns below M travel: with one token that is a quarter of a 16-column tile.
// Counter word of a tile, ten bits each: parts published, CTAs that gave up waiting (only while parts are missing), CTAs
// that have seen all parts; the last of those clears it.
constexpr int COUNT_LEFT = 1 << 10, COUNT_SEEN = 1 << 20, COUNT_MASK = (1 << 10) - 1;
constexpr long long GIVE_UP_CLOCKS = 100000;  // 50 us; in an undisturbed call parts come within 10
struct Join {
  int first, last;   // CTAs that have parts of the tile
  int mine, shares;  // this CTA finishes share `mine` of `shares`; none below 0
};
struct Split {
  Cut cut;
  int M;
  float4* slots;  // [2 * CTAs]: slot 2c holds CTA c's part of the tile it starts in the middle of, 2c + 1 any other
  int* counters;  // [row tiles]; zero before and after the launch
  volatile int* abortp;
};
__device__ __forceinline__ int ld_acquire(const int* p) {
  int v;
  asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ void red_release(int* p, int v) {
  asm volatile("red.release.gpu.global.add.s32 [%0], %1;" ::"l"(p), "r"(v) : "memory");
}
__device__ __forceinline__ int slot_of(const Cut& c, int cta, int tile_begin) {
  return 2 * cta + (cut_start(c, cta) > tile_begin ? 0 : 1);
}

// All THREADS epilogue threads: thread = weight row `row` of NT tiles, COLS of the COLS_ALL token columns from col0 on.
template <int NT, int COLS, int COLS_ALL, int THREADS>
__device__ __forceinline__ void publish_segment(const float (&v)[NT][COLS], const Segment& s, const Split& sp, int col0,
                                                int row, int ep_tid) {
  const int left = sp.M - col0;
  const int nq = left <= 0 ? 0 : ((left < COLS ? left : COLS) + 3) / 4;
  float4* const slot = sp.slots + static_cast<long long>(slot_of(sp.cut, blockIdx.x, s.tile_begin)) * (NT * COLS_ALL / 4 * 128);
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < COLS / 4; ++i)
      if (i < nq)
        slot[(t * (COLS_ALL / 4) + col0 / 4 + i) * 128 + row] =
            make_float4(v[t][4 * i], v[t][4 * i + 1], v[t][4 * i + 2], v[t][4 * i + 3]);
  named_bar_sync(1, THREADS);
  if (s.begin != s.tile_begin || s.end != s.tile_end) {
    // one thread's release covers the block's stores, which the barrier put before it (256 threads that each
    // waited for their own held up the sums behind them for 2,000 to 9,000 clocks while HBM was busy)
    if (ep_tid == 0) red_release(sp.counters + s.tile, 1);
  }
}

__device__ __forceinline__ float4 plus(const float4& a, const float4& b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
// This CTA's share of a tile whose parts are in the slots: emit(t, row, i, sums) for four tokens 4i .. 4i + 3 of a row, with
// JOINT over both tiles at once (emit(0, row, i, gate, up)). ITEMS of a thread are worked on together.
template <int NT, bool JOINT, int COLS_ALL, int THREADS, int ITEMS, typename Emit>
__device__ __forceinline__ void finish_tile(int tile_begin, const Join& join, const Split& sp, int ep_tid, Emit emit) {
  constexpr int SLOT4 = NT * COLS_ALL / 4 * 128;
  const int nq = (sp.M + 3) / 4, first = join.first, parts = join.last - first + 1;
  const int items = (JOINT ? 1 : NT) * nq * 128;
  const int share = (items + join.shares - 1) / join.shares;
  const int lo = share * join.mine, hi = lo + share < items ? lo + share : items;
  const float4* const s0 = sp.slots + static_cast<long long>(slot_of(sp.cut, first, tile_begin)) * SLOT4;
  const float4* const s1 = sp.slots + (2LL * first + 2) * SLOT4;  // the others start in the middle of the tile
  const int per_t = nq * 128;
  constexpr int UP = COLS_ALL / 4 * 128;  // from a gate value to its up value
#pragma unroll 1
  for (int it0 = lo + ep_tid; it0 < hi; it0 += THREADS * ITEMS) {
    float4 a[ITEMS], b[ITEMS];
    int at[ITEMS];
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {  // the items' loads go out together
      const int it = it0 + n * THREADS;
      const int t = (!JOINT && it >= per_t) ? 1 : 0;
      at[n] = t * (COLS_ALL / 4 * 128) + (it - t * per_t);
      if (it < hi) {
        a[n] = __ldcg(s0 + at[n]);
        if (JOINT) b[n] = __ldcg(s0 + at[n] + UP);
      }
    }
    const float4* s = s1;
    // up to BATCH parts of an item on their way at a time, added in CTA order
    constexpr int BATCH = ITEMS > 1 ? 1 : (JOINT ? 4 : 8);
#pragma unroll 1
    for (int c = 1; c < parts; c += BATCH, s += 2 * SLOT4 * BATCH) {
      float4 q[ITEMS][BATCH], r[ITEMS][BATCH];
#pragma unroll
      for (int n = 0; n < ITEMS; ++n)
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
          if (it0 + n * THREADS < hi && c + k < parts) {
            q[n][k] = __ldcg(s + 2 * SLOT4 * k + at[n]);
            if (JOINT) r[n][k] = __ldcg(s + 2 * SLOT4 * k + at[n] + UP);
          }
#pragma unroll
      for (int n = 0; n < ITEMS; ++n)
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
          if (it0 + n * THREADS < hi && c + k < parts) {
            a[n] = plus(a[n], q[n][k]);
            if (JOINT) b[n] = plus(b[n], r[n][k]);
          }
    }
#pragma unroll
    for (int n = 0; n < ITEMS; ++n) {
      const int it = it0 + n * THREADS;
      const int t = (!JOINT && it >= per_t) ? 1 : 0;
      if (it < hi) emit(t, (it - t * per_t) & 127, (it - t * per_t) >> 7, a[n], b[n]);
    }
  }
}

// Gate activations at fp32 accuracy (the GEMM epilogues use tanh.approx, whose 2^-11 is as large as fp16's own
// rounding; here the epilogue is a small part of the work).
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
template <int ACT>
__device__ __forceinline__ void hidden4(float (&h)[4], const float4& g, const float4& u, float bg, float bu) {
  h[0] = act_fine<ACT>(g.x + bg) * (u.x + bu);
  h[1] = act_fine<ACT>(g.y + bg) * (u.y + bu);
  h[2] = act_fine<ACT>(g.z + bg) * (u.z + bu);
  h[3] = act_fine<ACT>(g.w + bg) * (u.w + bu);
}
// Four tokens' factors, 1 without any.
__device__ __forceinline__ float4 token_factors(const float* rs, int M, int i) {
  float4 r = make_float4(1.f, 1.f, 1.f, 1.f);
  if (rs != nullptr) {
    r.x = rs[4 * i];
    if (4 * i + 1 < M) r.y = rs[4 * i + 1];
    if (4 * i + 2 < M) r.z = rs[4 * i + 2];
    if (4 * i + 3 < M) r.w = rs[4 * i + 3];
  }
  return r;
}
__device__ __forceinline__ float4 times(const float4& a, const float4& b) {
  return make_float4(a.x * b.x, a.y * b.y, a.z * b.z, a.w * b.w);
}
// Four tokens of a hidden row: act(gate + bg) * (up + bu), on experts times the token's factor, or 0. rs: [M] factors on
// the sums, or null.
template <typename T>
__device__ __forceinline__ void emit_hidden(T* po, long long ld, int M, int i, float4 gate, float4 up, const float* rs,
                                            float bg, float bu, int act, const MoeShared* moe) {
  const float4 r = token_factors(rs, M, i);
  gate = times(gate, r);
  up = times(up, r);
  float h[4];
  switch (act) {
    case ACT_SILU: hidden4<ACT_SILU>(h, gate, up, bg, bu); break;
    case ACT_NONE: hidden4<ACT_NONE>(h, gate, up, bg, bu); break;
    case ACT_RELU: hidden4<ACT_RELU>(h, gate, up, bg, bu); break;
    case ACT_GELU: hidden4<ACT_GELU>(h, gate, up, bg, bu); break;
    case ACT_SIGMOID: hidden4<ACT_SIGMOID>(h, gate, up, bg, bu); break;
    case ACT_TANH: hidden4<ACT_TANH>(h, gate, up, bg, bu); break;
    default: hidden4<ACT_LEAKY_RELU>(h, gate, up, bg, bu); break;
  }
  po += static_cast<long long>(4 * i) * ld;
#pragma unroll
  for (int k = 0; k < 4; ++k, po += ld) {
    const int m = 4 * i + k;
    if (m < M) {
      if (moe != nullptr) h[k] = moe->hit[m] ? h[k] * moe->f[m] : 0.f;
      *po = static_cast<T>(h[k]);
    }
  }
}
// Four tokens of an output row: v (* rs) (* wmax) + bias + residual.
template <typename T>
__device__ __forceinline__ void emit_product(T* po, const T* pr, long long ld, int M, int i, float4 v, const float* rs,
                                             float bias, const MoeShared* moe) {
  v = times(v, token_factors(rs, M, i));
  const float a[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int m = 4 * i + k;
    if (m < M) {
      float o = (moe != nullptr ? a[k] * moe->wmax[m] : a[k]) + bias;
      if (pr) o += static_cast<float>(pr[static_cast<long long>(m) * ld]);
      po[static_cast<long long>(m) * ld] = static_cast<T>(o);
    }
  }
}

// The end of a segment and of a CTA's units, shared by the stream kernels. `emit_tile(tile, tile_begin, join)` finishes
// this CTA's share of a tile from the slots.
struct Pending {
  int tile[2];
  int n = 0;
};
template <int NT, int COLS, int COLS_ALL, int THREADS, typename EmitTile>
__device__ __forceinline__ bool end_segment(const float (&v)[NT][COLS], const Segment& s, const Split& sp, int col0, int row,
                                            int ep_tid, Pending& pending, EmitTile emit_tile) {
  // vote: all epilogue threads leave the same way even if the abort flag flips between their reads
  if (named_bar_or(1, THREADS, *sp.abortp != 0)) return false;
  publish_segment<NT, COLS, COLS_ALL, THREADS>(v, s, sp, col0, row, ep_tid);
  if (s.begin == s.tile_begin && s.end == s.tile_end)
    emit_tile(s.tile, s.tile_begin, Join{static_cast<int>(blockIdx.x), static_cast<int>(blockIdx.x), 0, 1});
  else
    pending.tile[pending.n++] = s.tile;
  return true;
}
template <int THREADS, typename EmitTile>
__device__ __forceinline__ void end_units(const Pending& pending, int per_tile, const Split& sp, int ep_tid,
                                          EmitTile emit_tile) {
  __shared__ int shared_mine[2], shared_shares[2];
  if (pending.n == 0) return;
  int first[2], last[2];  // CTAs that have parts of the tile
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const int begin = pending.tile[p < pending.n ? p : 0] * per_tile;
    // this CTA is the last one of a tile that it met first, and the first of one that it ends in the middle of
    const bool tail = begin < cut_start(sp.cut, blockIdx.x);
    const bool ends = cut_start(sp.cut, blockIdx.x + 1) >= begin + per_tile;
    first[p] = tail ? cut_owner(sp.cut, begin) : static_cast<int>(blockIdx.x);
    last[p] = ends ? static_cast<int>(blockIdx.x) : cut_owner(sp.cut, begin + per_tile - 1);
  }
  // thread 0 waits for the parts of the first tile, thread 32 for those of the second
  const int k = ep_tid >> 5;
  const bool waiter = (ep_tid & 31) == 0 && k < pending.n;
  int* const counter = sp.counters + (k == 0 ? pending.tile[0] : pending.tile[1]);
  bool leave = false;  // this thread has still to count itself among those that have seen all parts
  int shares = 0;
  if (waiter) {
    const int my_first = k == 0 ? first[0] : first[1];
    const int parts = (k == 0 ? last[0] : last[1]) - my_first + 1;
    int mine = static_cast<int>(blockIdx.x) - my_first, v;
    shares = parts;
    const long long t0 = clock64();
    while (((v = ld_acquire(counter)) & COUNT_MASK) != parts) {
      // (the exchange fails when a part has come since)
      if (*sp.abortp != 0 || (clock64() - t0 > GIVE_UP_CLOCKS && atomicCAS(counter, v, v + COUNT_LEFT) == v)) {
        mine = -1;
        break;
      }
    }
    if (mine >= 0) {
      const int left = v / COUNT_LEFT & COUNT_MASK;
      shares -= left;
      leave = left == 0;
      if (left > 0) {  // the shares go to those that are here, in the order in which they ask
        mine = atomicAdd(counter, COUNT_SEEN) / COUNT_SEEN;
        if (mine == shares - 1) *counter = 0;
      }
    }
    shared_mine[k] = mine;
    shared_shares[k] = shares;
  }
  if (named_bar_or(1, THREADS, *sp.abortp != 0)) return;
#pragma unroll 1
  for (int p = 0; p < pending.n; ++p) {
    const int tile = p == 0 ? pending.tile[0] : pending.tile[1];
    const Join join{p == 0 ? first[0] : first[1], p == 0 ? last[0] : last[1], shared_mine[p], shared_shares[p]};
    if (join.mine >= 0) emit_tile(tile, tile * per_tile, join);
  }
  // the last CTA to have seen all parts leaves the counter ready for the next call
  if (leave && atomicAdd(counter, COUNT_SEEN) / COUNT_SEEN == shares - 1) *counter = 0;
}

// Bounded wait that looks at no abort flag: a thread that gives up uses it to see its own copies in flight land
// (or a last commit arrive) before its CTA leaves.
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait_suspend(bar, parity, 4000u))
    if (clock64() - t0 > 40000000LL) return;
}

}  // namespace gmlp
