// What the translation units that hold C ABI entries share: error reporting (the message of miw_last_error) and the device
// that miw_init chose.  Defined in capi.hip.
#pragma once
#include <hip/hip_runtime.h>

namespace miw {

int api_fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
int api_hip_fail(hipError_t e, const char *what);
bool api_initialized();
int api_cu_count();

}  // namespace miw
