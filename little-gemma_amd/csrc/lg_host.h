// lg_host.h — what the translation units of liblg_hip.so share on the host side: the error text of a call.
#pragma once
#include <hip/hip_runtime.h>

// Keeps the message for lg_hip_last_error() of this thread and returns `code`.
__attribute__((visibility("hidden"), format(printf, 2, 3))) int lg_fail(int code, const char *fmt, ...);

#define LG_TRY(expr) do { hipError_t e_ = (expr); if (e_ != hipSuccess) \
    return lg_fail(-100 - (int)e_, "%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, __LINE__); } while (0)
