// Host-side helpers of the C ABI that more than one translation unit uses: error text, device
// information, tensor-map encoding and launch attributes. Defined in gmlp_api.cu.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <initializer_list>

#include "../../include/gmlp.h"

namespace gmlp {

// Stores the calling thread's error text and returns `code`.
int fail(int code, const char* fmt, ...);

struct DeviceInfo {
  std::atomic<bool> ready{false};
  int sm_count = 0;
  int cc_major = 0;
  int* status_ptr = nullptr;  // device word that kernels which give up a bounded wait write
};
// The current device's entry; also binds its primary context to the calling thread.
int device_info(const DeviceInfo** out);

constexpr int DTYPE_U8 = 100;  // internal: one-byte elements (e4m3 and packed 4-bit operands)
int encode_map(CUtensorMap* m, const void* base, int64_t inner, int64_t outer, int64_t pitch_elems,
               uint32_t box_inner, uint32_t box_outer, int dtype, int swizzle_bytes = 128);

int check_problem(const gmlp_problem_t* p);
int check_ptrs(std::initializer_list<const void*> ps);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }
inline size_t align_up(size_t v, size_t a) { return (v + a - 1) / a * a; }

// cudaFuncSetAttribute(MaxDynamicSharedMemorySize) once per (kernel, device) instead of
// before every launch.
template <typename K>
int ensure_smem_attr(K kfn, size_t smem, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (done.load(std::memory_order_acquire) & bit) return GMLP_OK;
  const cudaError_t e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             static_cast<int>(smem));
  if (e != cudaSuccess)
    return fail(GMLP_ERR_LAUNCH, "cudaFuncSetAttribute: %s", cudaGetErrorString(e));
  done.fetch_or(bit, std::memory_order_release);
  return GMLP_OK;
}

}  // namespace gmlp
