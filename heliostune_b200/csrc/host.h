// Host-side helpers the C ABI's source files share: errors, per-device state, shared-memory
// limits and TMA tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/heliostune_b200.h"

namespace hst {

// Stores the calling thread's error message (hst_last_error) and returns `code`.
int fail(int code, const char* fmt, ...);

#define HST_CUDA(call)                                                                   \
  do {                                                                                   \
    cudaError_t err_ = (call);                                                           \
    if (err_ != cudaSuccess)                                                             \
      return fail(HST_ERR_CUDA, "%s failed: %s", #call, cudaGetErrorString(err_));       \
  } while (0)

#define HST_TRY(call)          \
  do {                                \
    int rc_ = (call);                 \
    if (rc_ != HST_OK) return rc_;    \
  } while (0)

constexpr int kMaxDevices = 64;
constexpr int kMaxDynamicSmem = 232448;  // 227 KB per CTA on sm_100
constexpr int kSmemPerSm = 233472;       // 228 KB per SM
constexpr int kSmemReservedPerCta = 1024;

struct DeviceState {
  std::atomic<bool> ready{false};
  int sm_count = 0;
  int* status = nullptr;
};

// State of the current device.
int device_state(DeviceState** out);

// Raises the dynamic shared-memory limit of a kernel once per device.
template <typename Kernel>
int allow_smem(Kernel kernel, std::atomic<uint64_t>& done_mask) {
  int dev = 0;
  HST_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << dev;
  if (!(done_mask.load(std::memory_order_acquire) & bit)) {
    HST_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  kMaxDynamicSmem));
    done_mask.fetch_or(bit, std::memory_order_release);
  }
  return HST_OK;
}

// A tiled tensor map of `rank` (2 or 3) dimensions, innermost first, with the 128-byte swizzle;
// strides (bytes) of every dimension but the innermost.
int encode_tiled(CUtensorMap* map, CUtensorMapDataType type, uint32_t rank, const void* base,
                 const uint64_t* dims, const uint64_t* strides_bytes, const uint32_t* box);

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return cdiv(a, b) * b; }

}  // namespace hst
