// Host side of the few-token kernels that several translation units share: launches of the stream kernels.
#pragma once
#include <algorithm>
#include <cstring>

#include "host_util.h"
#include "w4_stream.cuh"

namespace gmlp {

// ---------------------------------------------------------------- launching --
// Launches a kernel with programmatic stream serialization where `dependent`, in clusters where `cluster` > 1.
inline int launch_few_args(const void* kfn, unsigned grid, unsigned threads, size_t smem, bool dependent,
                           cudaStream_t stream, void** args, int cluster) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  if (dependent) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[cfg.numAttrs].val.clusterDim.y = 1;
    attr[cfg.numAttrs++].val.clusterDim.z = 1;
  }
  const cudaError_t e = cudaLaunchKernelExC(&cfg, kfn, args);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(GMLP_ERR_LAUNCH, "kernel launch: %s", cudaGetErrorString(e));
  }
  return GMLP_OK;
}
template <typename A>
int launch_few(void (*kfn)(const A), unsigned grid, unsigned threads, size_t smem, bool dependent, cudaStream_t stream,
               A a, int cluster = 1) {
  void* args[] = {&a};
  return launch_few_args(reinterpret_cast<const void*>(kfn), grid, threads, smem, dependent, stream, args, cluster);
}
template <typename Maps, typename A>
int launch_few(void (*kfn)(const Maps, const A), unsigned grid, unsigned threads, size_t smem, bool dependent,
               cudaStream_t stream, Maps m, A a) {
  void* args[] = {&m, &a};
  return launch_few_args(reinterpret_cast<const void*>(kfn), grid, threads, smem, dependent, stream, args, 1);
}

// One 4-bit weight matrix (of one or of all experts).
struct W4Matrix {
  const void* q;
  const void* scale;
  const void* zero;
};

// Token columns of the 4-bit kernels.
inline int w4_mt(int64_t M) { return M <= 8 ? 8 : (M <= 16 ? 16 : (M <= 32 ? 32 : 64)); }

// What every instantiation of the 4-bit stream kernel is launched with.
struct W4Call {
  int dtype;
  int64_t M, rows, cols, experts, R;
  int group;
  W4Matrix w0, w1;
  const void* x;  // up to W4_FUSED_TOKENS tokens: the activations, of pitch ldx; else their terms:
  int64_t ldx;
  const void *t8, *meta, *rowscale;
  const void *bias0, *bias1, *residual;
  void* out;
  float* slots;
  int* counters;
  int act;
  bool dependent, early;
  MoeTable moe;
  int64_t max_units;
  cudaStream_t stream;
};

template <int MT, bool DUAL, typename T, int GSHIFT, bool FUSED>
int launch_w4_t(const DeviceInfo* dev, const W4Call& c) {
  using Conf = W4Conf<MT, GSHIFT, FUSED>;
  if (c.max_units > 0x7fffffffLL) return fail(GMLP_ERR_SHAPE, "the call has more than 2^31 units of work");
  W4Maps m;
  int rc;
  if ((rc = encode_map(&m.w0, c.w0.q, c.cols / 2, c.experts * c.rows, c.cols / 2, 128, 128, DTYPE_U8))) return rc;
  m.w1 = m.w0;
  if (DUAL && (rc = encode_map(&m.w1, c.w1.q, c.cols / 2, c.experts * c.rows, c.cols / 2, 128, 128, DTYPE_U8))) return rc;
  m.x = m.w0;
  if (!FUSED && (rc = encode_map(&m.x, c.t8, c.cols, W4_TERMS * c.R, c.cols, 128, MT, DTYPE_U8))) return rc;
  // Scales and zeros as TMA boxes of the unit's groups where their rows are aligned, else row by row in 16-byte blocks, one copy
  // for each (tile, group) and array. Device time, boxes against rows: 131072 x 4096, 8 tokens 56 against 61 us; K=8192,
  // N=28672 MLP of one token 70 against 72, of 64 tokens 164 against 175.
  const bool wide = c.rows % 16 == 0 && aligned16(c.w0.scale) && aligned16(c.w1.scale) && aligned16(c.w0.zero) &&
                    aligned16(c.w1.zero);
  m.s0 = m.s1 = m.z0 = m.z1 = m.w0;
  if (wide) {
    const int64_t lines = c.experts * (c.cols / c.group);
    const uint32_t box = Conf::GPU;
    if ((rc = encode_map(&m.s0, c.w0.scale, c.rows, lines, c.rows, 128, box, c.dtype, 0))) return rc;
    if (DUAL && (rc = encode_map(&m.s1, c.w1.scale, c.rows, lines, c.rows, 128, box, c.dtype, 0))) return rc;
    if (c.w0.zero && (rc = encode_map(&m.z0, c.w0.zero, c.rows, lines, c.rows, 128, box, DTYPE_U8, 0))) return rc;
    if (DUAL && c.w1.zero && (rc = encode_map(&m.z1, c.w1.zero, c.rows, lines, c.rows, 128, box, DTYPE_U8, 0))) return rc;
  }
  W4Args a;
  memset(&a, 0, sizeof(a));
  a.M = static_cast<int>(c.M);
  a.rows = static_cast<int>(c.rows);
  a.kbt = static_cast<int>((c.cols + W4_UNIT_COLS - 1) / W4_UNIT_COLS);
  a.groups = static_cast<int>(c.cols / c.group);
  a.R = c.R;
  a.x = c.x;
  a.ldx = c.ldx;
  a.cols = static_cast<int>(c.cols);
  a.status = dev->status_ptr;
  a.meta = static_cast<const float*>(c.meta);
  a.rowscale = static_cast<const float*>(c.rowscale);
  a.scale0 = static_cast<const uint16_t*>(c.w0.scale);
  a.scale1 = static_cast<const uint16_t*>(c.w1.scale);
  a.zero0 = static_cast<const uint8_t*>(c.w0.zero);
  a.zero1 = static_cast<const uint8_t*>(c.w1.zero);
  a.bias0 = c.bias0;
  a.bias1 = c.bias1;
  a.residual = c.residual;
  a.out = c.out;
  a.slots = c.slots;
  a.counters = c.counters;
  a.act = c.act;
  a.wide = wide ? 1 : 0;
  a.early = c.early ? 1 : 0;
  a.moe = c.moe;
  const int grid = static_cast<int>(c.max_units < dev->sm_count ? c.max_units : dev->sm_count);
  if (c.moe.ids == nullptr) a.cut = make_cut(static_cast<int>(c.max_units), cut_grain(a.kbt, W4_UNIT_CLOCKS), grid);
  auto kfn = w4_stream_kernel<MT, DUAL, T, GSHIFT, FUSED>;
  static std::atomic<uint64_t> attr_done{0};
  if ((rc = ensure_smem_attr(kfn, Conf::SMEM, attr_done))) return rc;
  return launch_few(kfn, grid, Conf::THREADS, Conf::SMEM, c.dependent, c.stream, m, a);
}
template <int GSHIFT, bool DUAL, typename T>
int launch_w4_type(const DeviceInfo* dev, const W4Call& c) {
  if (c.M <= W4_FUSED_TOKENS) return launch_w4_t<8, DUAL, T, GSHIFT, true>(dev, c);
  switch (w4_mt(c.M)) {
    case 8: return launch_w4_t<8, DUAL, T, GSHIFT, false>(dev, c);
    case 16: return launch_w4_t<16, DUAL, T, GSHIFT, false>(dev, c);
    case 32: return launch_w4_t<32, DUAL, T, GSHIFT, false>(dev, c);
    default: return launch_w4_t<64, DUAL, T, GSHIFT, false>(dev, c);
  }
}
template <int GSHIFT>
int launch_w4_group(const DeviceInfo* dev, const W4Call& c, bool dual) {
  if (c.dtype == GMLP_BF16)
    return dual ? launch_w4_type<GSHIFT, true, __nv_bfloat16>(dev, c) : launch_w4_type<GSHIFT, false, __nv_bfloat16>(dev, c);
  return dual ? launch_w4_type<GSHIFT, true, __half>(dev, c) : launch_w4_type<GSHIFT, false, __half>(dev, c);
}
// One translation unit each (w4_g32.cu, w4_g64.cu, w4_g128.cu): they compile side by side.
int launch_w4_g32(const DeviceInfo* dev, const W4Call& c, bool dual);
int launch_w4_g64(const DeviceInfo* dev, const W4Call& c, bool dual);
int launch_w4_g128(const DeviceInfo* dev, const W4Call& c, bool dual);

}  // namespace gmlp
