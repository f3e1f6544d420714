// Host-side helpers shared by the library's translation units: the error message of the calling thread, argument
// checks, small integer arithmetic.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/plconvlstm.h"

#define PLC_HIDDEN __attribute__((visibility("hidden")))

// stores the message plc_last_error() returns on this thread and gives `code` back
PLC_HIDDEN int plc_fail(int code, const char* fmt, ...);

#define PLC_HIP(expr)                                                                         \
    do {                                                                                      \
        hipError_t e_ = (expr);                                                               \
        if (e_ != hipSuccess) return plc_fail(PLC_EHIP, "%s: %s", #expr, hipGetErrorString(e_)); \
    } while (0)

#define PLC_REQUIRE(cond, ...)                              \
    do {                                                    \
        if (!(cond)) return plc_fail(PLC_EINVAL, __VA_ARGS__); \
    } while (0)

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
static inline size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }
static inline int cdiv(int a, int b) { return (a + b - 1) / b; }
