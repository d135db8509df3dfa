// C ABI of the few-token operators on 4-bit weights and on mixtures of experts (declared in include/gmlp.h):
// argument checks, tensor maps and launches. No torch types, no allocation, no CPU path.
#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstring>

#include "../../include/gmlp.h"
#include "host_util.h"
#include "few_token_host.cuh"
#include "moe_stream.cuh"

namespace gmlp {

// ----------------------------------------------------------------- scratch --
// [slots][counters of the first kernel][counters of the second]. The slots take the size of a 64-token call whatever the
// call is, so that the counters, which have to be zero between calls, lie behind them for every shape and calls of
// different shapes can follow one another on one buffer.
// two slots per CTA, each two tiles of 128 rows
static size_t slots_bytes(int ctas) { return static_cast<size_t>(ctas) * 2 * 2 * 128 * FEW_MAX_TOKENS * sizeof(float); }
struct FewLayout {
  size_t counters1_off, counters2_off, total;
};
static FewLayout few_layout(int64_t K, int64_t N, int64_t experts, int ctas) {
  FewLayout l;
  l.counters1_off = slots_bytes(ctas);
  l.counters2_off =
      l.counters1_off + align_up(static_cast<size_t>((N + 127) / 128) * static_cast<size_t>(experts) * sizeof(int), 256);
  l.total = l.counters2_off + align_up(static_cast<size_t>((K + 127) / 128) * sizeof(int), 256);
  return l;
}
static int mpad_of(int64_t M) { return M <= 16 ? 16 : (M <= 32 ? 32 : 64); }

static int check_w4(const W4Matrix& w) {
  if (!w.q || !w.scale) return fail(GMLP_ERR_ARG, "NULL 4-bit weight or scale");
  if (!aligned16(w.q)) return fail(GMLP_ERR_ALIGN, "4-bit weights must be 16-byte aligned");
  if (((reinterpret_cast<uintptr_t>(w.scale) | reinterpret_cast<uintptr_t>(w.zero)) & 3u) != 0)
    return fail(GMLP_ERR_ALIGN, "scales and zeros must be 4-byte aligned");
  return GMLP_OK;
}
static int check_group(int32_t group, int64_t cols) {
  if (group != 32 && group != 64 && group != 128)
    return fail(GMLP_ERR_SHAPE, "group size %d: supported are 32, 64 and 128", group);
  if (cols % group != 0)
    return fail(GMLP_ERR_SHAPE, "%lld columns are no multiple of the group size %d", static_cast<long long>(cols), group);
  return GMLP_OK;
}

// Work buffer of a 4-bit call: [hidden state][activation terms][group sums][token factors]. The terms of x and, later, of the
// hidden state take turns in one place; up to W4_FUSED_TOKENS tokens there is only the hidden state.
struct W4Work {
  size_t t8_off, meta_off, row_off, total;
};
static size_t w4_t8_bytes(int64_t rows, int64_t cols) { return static_cast<size_t>(W4_TERMS) * rows * cols; }
// K columns of x (M rows); N columns of h (active * M rows), N = 0 for a plain product
static W4Work w4_work(int64_t M, int64_t K, int64_t N, int64_t active, int group) {
  W4Work w;
  w.t8_off = align_up(static_cast<size_t>(active * M * N) * 2, 256);
  w.meta_off = w.row_off = w.total = std::max<size_t>(w.t8_off, 16);
  if (M <= W4_FUSED_TOKENS) return w;
  w.meta_off = w.t8_off + align_up(std::max(w4_t8_bytes(M, K), w4_t8_bytes(active * M, N)), 256);
  const int64_t k_units = (K + W4_UNIT_COLS - 1) / W4_UNIT_COLS, n_units = (N + W4_UNIT_COLS - 1) / W4_UNIT_COLS;
  w.row_off = w.meta_off + static_cast<size_t>(std::max(k_units, active * n_units)) * (W4_UNIT_COLS / group) * w4_mt(M) *
                               sizeof(float);
  w.total = w.row_off + FEW_MAX_TOKENS * sizeof(float);
  return w;
}

// Activations as e5m2 terms (see w4_stream.cuh).
static int launch_split(int64_t M, int64_t R, int64_t cols, int64_t ldx, int group, int dtype, const void* x, char* work,
                        const W4Work& w, const MoeTable& moe, bool dependent, cudaStream_t stream) {
  W4SplitArgs a;
  a.x = x;
  a.ldx = ldx;
  a.R = R;
  a.M = static_cast<int>(M);
  a.MT = w4_mt(M);
  a.cols = static_cast<int>(cols);
  a.gshift = group == 32 ? 0 : (group == 64 ? 1 : 2);
  a.t8 = reinterpret_cast<uint8_t*>(work + w.t8_off);
  a.meta = reinterpret_cast<float*>(work + w.meta_off);
  a.rowscale = reinterpret_cast<float*>(work + w.row_off);
  a.dependent = dependent ? 1 : 0;
  a.moe = moe;
  const unsigned grid = static_cast<unsigned>(M) * W4_SPLIT_CLUSTER;
  return dtype == GMLP_BF16
             ? launch_few(w4_split_kernel<__nv_bfloat16>, grid, W4_SPLIT_THREADS, 0, dependent, stream, a, W4_SPLIT_CLUSTER)
             : launch_few(w4_split_kernel<__half>, grid, W4_SPLIT_THREADS, 0, dependent, stream, a, W4_SPLIT_CLUSTER);
}

static int launch_w4(const DeviceInfo* dev, const W4Call& c, bool dual) {
  return c.group == 32 ? launch_w4_g32(dev, c, dual)
                       : (c.group == 64 ? launch_w4_g64(dev, c, dual) : launch_w4_g128(dev, c, dual));
}

template <int MPAD, bool DUAL, typename T>
static int launch_moe_t(const DeviceInfo* dev, int dtype, int64_t M, int64_t rows, int64_t cols, int64_t experts,
                        const void* w0, const void* w1, const void* x, int64_t ldx, int64_t x_rows,
                        const void* residual, void* out, float* slots, int* counters, int act, bool early,
                        const MoeTable& moe, int64_t grid_units, cudaStream_t stream) {
  if (grid_units > 0x7fffffffLL) return fail(GMLP_ERR_SHAPE, "the call has more than 2^31 units of work");
  CUtensorMap m0, m1, mx;
  int rc;
  if ((rc = encode_map(&m0, w0, cols, experts * rows, cols, 64, 128, dtype))) return rc;
  m1 = m0;
  if (DUAL && (rc = encode_map(&m1, w1, cols, experts * rows, cols, 64, 128, dtype))) return rc;
  if ((rc = encode_map(&mx, x, cols, x_rows, ldx, 64, MPAD, dtype))) return rc;
  MoeArgs a;
  memset(&a, 0, sizeof(a));
  a.M = static_cast<int>(M);
  a.rows = static_cast<int>(rows);
  a.kbt = static_cast<int>(cols / 64);
  a.idesc = make_idesc_f16(128, MPAD, dtype == GMLP_BF16 ? 1 : 0, false, false);
  a.status = dev->status_ptr;
  a.residual = residual;
  a.out = out;
  a.slots = slots;
  a.counters = counters;
  a.act = act;
  a.early = early ? 1 : 0;
  a.moe = moe;
  const int grid = static_cast<int>(grid_units < dev->sm_count ? grid_units : dev->sm_count);
  auto kfn = moe_stream_kernel<MPAD, DUAL, T>;
  constexpr size_t smem = moe_smem_bytes<MPAD, DUAL>();
  static std::atomic<uint64_t> attr_done{0};
  if ((rc = ensure_smem_attr(kfn, smem, attr_done))) return rc;
  return launch_few(kfn, grid, MOE_THREADS, smem, true, stream, MoeMaps{m0, m1, mx}, a);
}
template <bool DUAL, typename... Args>
static int launch_moe(int mpad, int dtype, const DeviceInfo* dev, Args... args) {
  const bool bf = dtype == GMLP_BF16;
  if (mpad == 16)
    return bf ? launch_moe_t<16, DUAL, __nv_bfloat16>(dev, dtype, args...)
              : launch_moe_t<16, DUAL, __half>(dev, dtype, args...);
  if (mpad == 32)
    return bf ? launch_moe_t<32, DUAL, __nv_bfloat16>(dev, dtype, args...)
              : launch_moe_t<32, DUAL, __half>(dev, dtype, args...);
  return bf ? launch_moe_t<64, DUAL, __nv_bfloat16>(dev, dtype, args...)
            : launch_moe_t<64, DUAL, __half>(dev, dtype, args...);
}

template <typename T, int TOKENS>
static int launch_route(const RouteArgs& a, int cluster, cudaStream_t st) {
  const unsigned grid = static_cast<unsigned>((a.M + TOKENS - 1) / TOKENS * cluster);
  if (a.E <= 32) return launch_few(moe_route_kernel<T, 1, TOKENS>, grid, ROUTE_THREADS, 0, true, st, a, cluster);
  if (a.E <= 128) return launch_few(moe_route_kernel<T, 4, TOKENS>, grid, ROUTE_THREADS, 0, true, st, a, cluster);
  return launch_few(moe_route_kernel<T, 16, TOKENS>, grid, ROUTE_THREADS, 0, true, st, a, cluster);
}

static int check_few(const gmlp_problem_t* p, const char* what) {
  int rc;
  if ((rc = check_problem(p))) return rc;
  if (p->dtype != GMLP_BF16 && p->dtype != GMLP_FP16) return fail(GMLP_ERR_DTYPE, "%s takes bf16 or fp16", what);
  if (p->M > FEW_MAX_TOKENS)
    return fail(GMLP_ERR_SHAPE, "%s takes at most 64 tokens, got %lld", what, static_cast<long long>(p->M));
  if (p->dropout_p != 0.0f) return fail(GMLP_ERR_ARG, "%s is inference only: dropout_p must be 0", what);
  return GMLP_OK;
}
static int check_experts(const gmlp_problem_t* p, int32_t experts, int32_t top_k, const void* ids, const void* weights) {
  if (experts < 1 || experts > MOE_MAX_EXPERTS)
    return fail(GMLP_ERR_SHAPE, "%d experts: 1 to %d are supported", experts, MOE_MAX_EXPERTS);
  if (top_k < 1 || top_k > MOE_MAX_TOPK || top_k > experts)
    return fail(GMLP_ERR_SHAPE, "top_k=%d: 1 to min(%d, experts) are supported", top_k, MOE_MAX_TOPK);
  if (static_cast<int64_t>(experts) * p->N > 0x7ffffe00LL || static_cast<int64_t>(experts) * p->K > 0x7ffffe00LL)
    return fail(GMLP_ERR_SHAPE, "experts * rows exceeds 32-bit tile coordinates");
  if (!ids || !weights) return fail(GMLP_ERR_ARG, "NULL routing table");
  if ((reinterpret_cast<uintptr_t>(ids) & 3u) != 0 || (reinterpret_cast<uintptr_t>(weights) & 3u) != 0)
    return fail(GMLP_ERR_ALIGN, "the routing table must be 4-byte aligned");
  return GMLP_OK;
}
static int64_t max_active(const gmlp_problem_t* p, int32_t experts, int32_t top_k) {
  return std::min<int64_t>(experts, p->M * top_k);
}

}  // namespace gmlp

using namespace gmlp;

extern "C" {

static int scratch_ctas() {
  const DeviceInfo* dev;
  return device_info(&dev) == GMLP_OK ? dev->sm_count : 256;  // without a device: an upper bound on the SM count
}
size_t gmlp_few_scratch_bytes(int64_t K, int64_t N, int32_t experts) {
  if (K <= 0 || N <= 0 || experts <= 0 || experts > MOE_MAX_EXPERTS) return 0;
  return few_layout(K, N, experts, scratch_ctas()).total;
}
size_t gmlp_few_scratch_counters(void) { return slots_bytes(scratch_ctas()); }

int gmlp_capture_id(void* stream, uint64_t* id) {
  if (!id) return fail(GMLP_ERR_ARG, "NULL id");
  *id = 0;
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long v = 0;
  const cudaError_t e = cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &v);
  if (e != cudaSuccess) return fail(GMLP_ERR_LAUNCH, "cudaStreamGetCaptureInfo: %s", cudaGetErrorString(e));
  if (status != cudaStreamCaptureStatusNone) *id = v;
  return GMLP_OK;
}

size_t gmlp_w4_work_bytes(int64_t M, int64_t K, int64_t N, int32_t experts, int32_t group, int32_t dtype) {
  if (M <= 0 || M > FEW_MAX_TOKENS || K <= 0 || N < 0 || experts <= 0 || (group != 32 && group != 64 && group != 128))
    return 0;
  return w4_work(M, K, N, experts, group).total;
}

int gmlp_w4_linear(int64_t M, int64_t rows, int64_t cols, int32_t group, int32_t dtype, const void* x, int64_t ldx,
                   const void* w4, const void* scale, const void* zero, const void* bias, const void* residual,
                   void* y, void* work, size_t work_bytes, void* scratch, size_t scratch_bytes, uint32_t tuning,
                   void* stream) {
  int rc;
  if (dtype != GMLP_BF16 && dtype != GMLP_FP16) return fail(GMLP_ERR_DTYPE, "the 4-bit product takes bf16 or fp16");
  if (M < 1 || M > FEW_MAX_TOKENS)
    return fail(GMLP_ERR_SHAPE, "the 4-bit product takes 1 to 64 tokens, got %lld", static_cast<long long>(M));
  if (rows < 1 || cols < 1 || rows > 0x7ffffe00LL || cols > 0x7ffffe00LL)
    return fail(GMLP_ERR_SHAPE, "rows=%lld cols=%lld out of range", static_cast<long long>(rows),
                static_cast<long long>(cols));
  if ((rc = check_group(group, cols))) return rc;
  const W4Matrix w{w4, scale, zero};
  if ((rc = check_w4(w))) return rc;
  if ((rc = check_ptrs({x, y, work, scratch}))) return rc;
  if (ldx < cols || (ldx % 8) != 0) return fail(GMLP_ERR_ALIGN, "row pitch of x must be a multiple of 8 and >= cols");
  const DeviceInfo* dev;
  if ((rc = device_info(&dev))) return rc;
  const FewLayout l = few_layout(rows, rows, 1, dev->sm_count);
  if (scratch_bytes < l.total)
    return fail(GMLP_ERR_SCRATCH, "scratch holds %zu bytes, %zu needed", scratch_bytes, l.total);
  const W4Work ww = w4_work(M, cols, 0, 1, group);
  if (work_bytes < ww.total) return fail(GMLP_ERR_SCRATCH, "work holds %zu bytes, %zu needed", work_bytes, ww.total);
  char* const wk = static_cast<char*>(work);
  char* const sc = static_cast<char*>(scratch);
  const bool dep = (tuning & (1u << 26)) == 0;  // GMLP_TUNE_ORDINARY_LAUNCH
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool split = M > W4_FUSED_TOKENS;
  if (split && (rc = launch_split(M, M, cols, ldx, group, dtype, x, wk, ww, MoeTable{nullptr, nullptr, 0, 0}, dep, st)))
    return rc;
  W4Call c;
  memset(&c, 0, sizeof(c));
  c.dtype = dtype;
  c.M = M;
  c.rows = rows;
  c.cols = cols;
  c.experts = 1;
  c.R = M;
  c.group = group;
  c.w0 = c.w1 = w;
  c.x = x;
  c.ldx = ldx;
  c.t8 = wk + ww.t8_off;
  c.meta = wk + ww.meta_off;
  c.rowscale = wk + ww.row_off;
  c.bias0 = bias;
  c.residual = residual;
  c.out = y;
  c.slots = reinterpret_cast<float*>(sc);
  c.counters = reinterpret_cast<int*>(sc + l.counters1_off);
  c.dependent = split || dep;
  c.early = true;
  c.max_units = ((rows + 255) / 256) * ((cols + W4_UNIT_COLS - 1) / W4_UNIT_COLS);
  c.stream = st;
  return launch_w4(dev, c, false);
}

// Both halves of a gated MLP on 4-bit weights, dense (moe.ids == NULL) or over experts.
static int mlp_w4(const gmlp_problem_t* p, int32_t group, int64_t experts, const MoeTable& moe, int64_t active,
                  const void* x, const W4Matrix& g, const void* b_gate, const W4Matrix& u, const void* b_up,
                  const W4Matrix& d, const void* b_down, const void* residual, void* y, void* work, size_t work_bytes,
                  void* scratch, size_t scratch_bytes, void* stream) {
  int rc;
  if ((rc = check_group(group, p->K))) return rc;
  if ((rc = check_group(group, p->N))) return rc;
  if ((rc = check_w4(g)) || (rc = check_w4(u)) || (rc = check_w4(d))) return rc;
  if ((g.zero == nullptr) != (u.zero == nullptr))
    return fail(GMLP_ERR_ARG, "gate and up weights must both have zeros or both have none");
  if ((rc = check_ptrs({x, y, work, scratch}))) return rc;
  const DeviceInfo* dev;
  if ((rc = device_info(&dev))) return rc;
  const FewLayout l = few_layout(p->K, p->N, active, dev->sm_count);
  if (scratch_bytes < l.total)
    return fail(GMLP_ERR_SCRATCH, "scratch holds %zu bytes, %zu needed", scratch_bytes, l.total);
  const W4Work ww = w4_work(p->M, p->K, p->N, active, group);
  if (work_bytes < ww.total) return fail(GMLP_ERR_SCRATCH, "work holds %zu bytes, %zu needed", work_bytes, ww.total);
  char* const wk = static_cast<char*>(work);
  char* const sc = static_cast<char*>(scratch);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool sparse = moe.ids != nullptr;
  const bool dep = sparse || (p->tuning & (1u << 26)) == 0;  // GMLP_TUNE_ORDINARY_LAUNCH
  const int64_t k_units = (p->K + W4_UNIT_COLS - 1) / W4_UNIT_COLS, n_units = (p->N + W4_UNIT_COLS - 1) / W4_UNIT_COLS;
  const bool split = p->M > W4_FUSED_TOKENS;
  if (split && (rc = launch_split(p->M, p->M, p->K, p->K, group, p->dtype, x, wk, ww, MoeTable{nullptr, nullptr, 0, 0}, dep, st)))
    return rc;
  W4Call c;
  memset(&c, 0, sizeof(c));
  c.dtype = p->dtype;
  c.M = p->M;
  c.experts = experts;
  c.group = group;
  c.t8 = wk + ww.t8_off;
  c.meta = wk + ww.meta_off;
  c.rowscale = wk + ww.row_off;
  c.slots = reinterpret_cast<float*>(sc);
  c.act = p->act;
  c.moe = moe;
  c.stream = st;
  c.rows = p->N;
  c.cols = p->K;
  c.R = p->M;
  c.x = x;
  c.ldx = p->K;
  c.w0 = g;
  c.w1 = u;
  c.bias0 = b_gate;
  c.bias1 = b_up;
  c.out = wk;
  c.counters = reinterpret_cast<int*>(sc + l.counters1_off);
  c.dependent = split || dep;
  c.early = !sparse;
  c.max_units = active * ((p->N + 127) / 128) * k_units;
  if ((rc = launch_w4(dev, c, true))) return rc;
  if (split && (rc = launch_split(p->M, active * p->M, p->N, p->N, group, p->dtype, wk, wk, ww, moe, true, st)))
    return rc;
  c.rows = p->K;
  c.cols = p->N;
  c.R = active * p->M;
  c.x = wk;
  c.ldx = p->N;
  c.w0 = c.w1 = d;
  c.bias0 = b_down;
  c.bias1 = nullptr;
  c.residual = residual;
  c.out = y;
  c.counters = reinterpret_cast<int*>(sc + l.counters2_off);
  c.dependent = true;
  c.early = true;
  c.max_units = active * ((p->K + 255) / 256) * n_units;
  return launch_w4(dev, c, false);
}

int gmlp_decode_fwd_w4(const gmlp_problem_t* p, int32_t group, const void* x, const void* w_gate4,
                       const void* w_gate_scale, const void* w_gate_zero, const void* b_gate, const void* w_up4,
                       const void* w_up_scale, const void* w_up_zero, const void* b_up, const void* w_down4,
                       const void* w_down_scale, const void* w_down_zero, const void* b_down, const void* residual,
                       void* y, void* work, size_t work_bytes, void* scratch, size_t scratch_bytes, void* stream) {
  int rc;
  if ((rc = check_few(p, "the 4-bit decode path"))) return rc;
  return mlp_w4(p, group, 1, MoeTable{nullptr, nullptr, 0, 0}, 1, x, {w_gate4, w_gate_scale, w_gate_zero}, b_gate,
                {w_up4, w_up_scale, w_up_zero}, b_up, {w_down4, w_down_scale, w_down_zero}, b_down, residual, y, work,
                work_bytes, scratch, scratch_bytes, stream);
}

int gmlp_moe_decode_fwd_w4(const gmlp_problem_t* p, int32_t group, int32_t experts, int32_t top_k, const void* x,
                           const int32_t* ids, const float* weights, const void* w_gate4, const void* w_gate_scale,
                           const void* w_gate_zero, const void* w_up4, const void* w_up_scale, const void* w_up_zero,
                           const void* w_down4, const void* w_down_scale, const void* w_down_zero,
                           const void* residual, void* y, void* work, size_t work_bytes, void* scratch,
                           size_t scratch_bytes, void* stream) {
  int rc;
  if ((rc = check_few(p, "the mixture-of-experts decode path"))) return rc;
  if ((rc = check_experts(p, experts, top_k, ids, weights))) return rc;
  return mlp_w4(p, group, experts, MoeTable{ids, weights, top_k, experts}, max_active(p, experts, top_k), x,
                {w_gate4, w_gate_scale, w_gate_zero}, nullptr, {w_up4, w_up_scale, w_up_zero}, nullptr,
                {w_down4, w_down_scale, w_down_zero}, nullptr, residual, y, work, work_bytes, scratch, scratch_bytes,
                stream);
}

int gmlp_moe_decode_fwd(const gmlp_problem_t* p, int32_t experts, int32_t top_k, const void* x, const int32_t* ids,
                        const float* weights, const void* w_gate, const void* w_up, const void* w_down,
                        const void* residual, void* h, void* y, void* scratch, size_t scratch_bytes, void* stream) {
  int rc;
  if ((rc = check_few(p, "the mixture-of-experts decode path"))) return rc;
  if ((p->K % 64) != 0 || (p->N % 64) != 0)
    return fail(GMLP_ERR_SHAPE, "the mixture-of-experts decode path needs K and N multiples of 64");
  if ((rc = check_experts(p, experts, top_k, ids, weights))) return rc;
  if ((rc = check_ptrs({x, w_gate, w_up, w_down, h, y, scratch}))) return rc;
  const DeviceInfo* dev;
  if ((rc = device_info(&dev))) return rc;
  const int64_t active = max_active(p, experts, top_k);
  const FewLayout l = few_layout(p->K, p->N, active, dev->sm_count);
  if (scratch_bytes < l.total)
    return fail(GMLP_ERR_SCRATCH, "scratch holds %zu bytes, %zu needed", scratch_bytes, l.total);
  char* sc = static_cast<char*>(scratch);
  float* slots = reinterpret_cast<float*>(sc);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const MoeTable moe{ids, weights, top_k, experts};
  rc = launch_moe<true>(mpad_of(p->M), p->dtype, dev, p->M, p->N, p->K, static_cast<int64_t>(experts), w_gate, w_up, x, p->K,
                        p->M, static_cast<const void*>(nullptr), h, slots, reinterpret_cast<int*>(sc + l.counters1_off), p->act, false,
                        moe, active * ((p->N + 127) / 128) * (p->K / 64), st);
  if (rc) return rc;
  return launch_moe<false>(mpad_of(p->M), p->dtype, dev, p->M, p->K, p->N, static_cast<int64_t>(experts), w_down,
                           static_cast<const void*>(nullptr), static_cast<const void*>(h), p->N, active * p->M,
                           residual, y, slots, reinterpret_cast<int*>(sc + l.counters2_off), p->act, true, moe,
                           active * ((p->K + 127) / 128) * (p->N / 64), st);
}

int gmlp_moe_route(int64_t M, int64_t K, int32_t experts, int32_t top_k, int32_t renormalize, int32_t dtype,
                   const void* x, int64_t ldx, const void* w_router, int32_t* ids, float* weights, void* stream) {
  int rc;
  if (dtype != GMLP_BF16 && dtype != GMLP_FP16) return fail(GMLP_ERR_DTYPE, "the router takes bf16 or fp16");
  if (M < 1 || M > 0xffffffLL || K < 1 || K > 0x7ffffe00LL || (K % 8) != 0)
    return fail(GMLP_ERR_SHAPE,
                "the router needs 1 <= M < 2^24 and K a positive multiple of 8 below 2^31 - 511; got M=%lld K=%lld",
                static_cast<long long>(M), static_cast<long long>(K));
  if (experts < 1 || experts > MOE_MAX_EXPERTS)
    return fail(GMLP_ERR_SHAPE, "%d experts: 1 to %d are supported", experts, MOE_MAX_EXPERTS);
  if (top_k < 1 || top_k > MOE_MAX_TOPK || top_k > experts)
    return fail(GMLP_ERR_SHAPE, "top_k=%d: 1 to min(%d, experts) are supported", top_k, MOE_MAX_TOPK);
  if ((rc = check_ptrs({x, w_router}))) return rc;
  if (ldx < K || (ldx % 8) != 0) return fail(GMLP_ERR_ALIGN, "row pitch of x must be a multiple of 8 and >= K");
  if (!ids || !weights) return fail(GMLP_ERR_ARG, "NULL routing table");
  if ((reinterpret_cast<uintptr_t>(ids) & 3u) != 0 || (reinterpret_cast<uintptr_t>(weights) & 3u) != 0)
    return fail(GMLP_ERR_ALIGN, "the routing table must be 4-byte aligned");
  const DeviceInfo* dev;
  if ((rc = device_info(&dev))) return rc;
  RouteArgs a;
  a.x = x;
  a.w = w_router;
  a.ldx = ldx;
  a.M = static_cast<int>(M);
  a.K = static_cast<int>(K);
  a.E = experts;
  a.top_k = top_k;
  a.renormalize = renormalize ? 1 : 0;
  a.ids = ids;
  a.weights = weights;
  // A warp takes two experts at a time, or one where there are SMs for it (32 experts x 4096, 32 tokens: 6.7 us against 7.4);
  // up to eight blocks a token.
  int cluster = 1;
  while (cluster < 8 && (cluster * 2 * (ROUTE_THREADS / 32) < experts ||
                         (cluster * (ROUTE_THREADS / 32) < experts && M * cluster * 2 <= dev->sm_count)))
    cluster *= 2;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = dtype == GMLP_BF16;
  // Two tokens a cluster where there are enough blocks either way (2048 tokens, 128 x 2048: 175 us against 229 with one; 64
  // tokens, 512 x 4096, three to four blocks an SM: 74 against 57).
  if (M * cluster > 8 * dev->sm_count)
    return bf ? launch_route<__nv_bfloat16, 2>(a, cluster, st) : launch_route<__half, 2>(a, cluster, st);
  return bf ? launch_route<__nv_bfloat16, 1>(a, cluster, st) : launch_route<__half, 1>(a, cluster, st);
}

}  // extern "C"
