// What the sources of the C ABI share: the calling thread's error detail, and the device.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <mutex>

namespace mqk {

// Sets the thread's error detail and returns `status`.
int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// Clears it and returns MQK_OK.
int ok();
// MQK_OK, or MQK_ERR_HIP with the error's name.
int hip_status(hipError_t err, const char* what);

// Compute units and XCDs of the current device.
struct Topology {
  int cus = 256;
  int xcds = 8;
};
Topology device_topology();

// Option "attn_split" (attn_api.hip).
extern std::atomic<int64_t> g_attn_split, g_attn_parts;

// Held over the launches of a call that hand data on in `workspace` (mqk_api.hip).
std::unique_lock<std::recursive_mutex> handover_lock(const void* workspace);

}  // namespace mqk
