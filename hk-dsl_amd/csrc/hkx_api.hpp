// What the C ABI's translation units share: the thread's last error message (hkx_api.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace hkx {

// The message of a refused call; returns `code`.
int api_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// Forgets the last message: at the start of every call.
void api_clear();
// HKX_OK, or HKX_ERR_LAUNCH with the runtime's words.
int api_launched(hipError_t e, const char* what);
// The current device's CUs.
int api_cus();

inline bool api_aligned(const void* p, size_t a) { return (uintptr_t)p % a == 0; }

}  // namespace hkx
