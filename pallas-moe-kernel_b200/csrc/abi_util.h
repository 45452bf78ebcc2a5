// What the ABI's translation units share: the calling thread's error text,
// per-device facts, and the routing limits.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstddef>

#include "../../include/moe_b200.h"

namespace moe {

extern thread_local char t_err[512];

// Sets the calling thread's error text and returns `code`.
int fail(int code, const char* fmt, ...);

#define MOE_CUDA_TRY(expr)                                                                   \
  do {                                                                                       \
    cudaError_t _e = (expr);                                                                 \
    if (_e != cudaSuccess) return fail(MOE_ERR_CUDA, "%s: %s", #expr, cudaGetErrorString(_e)); \
  } while (0)

struct DevInfo {
  CUcontext ctx = nullptr;  // context the entries below belong to
  int sms = 0;
  int* status = nullptr;  // device address of g_status on this device
  bool attr_set[46] = {};
  int pairs[30] = {};  // co-resident CTA pairs per pair-kernel variant (0 = not queried)
};

// The current device's ordinal and facts; fails on a device that is not sm_100.
int device_info(int* dev_out, DevInfo** info);

inline size_t align256(size_t v) { return (v + 255) & ~size_t(255); }

constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxK = 16;

}  // namespace moe
