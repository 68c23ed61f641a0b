// entry_checks.h -- what the C entries of op-level launches check and how they
// report: no exception passes a C caller, rows and alignment, shared memory of
// arguments, the stream's device.  Host code of one translation unit each.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "oi.h"
#include "oi_kernels.h"

namespace oi {

namespace {

// C callers must see no exception: a message that cannot be built is left out.
int err(int code, const char *what, const std::string &msg) noexcept {
    try {
        return set_error(code, (std::string(what) + ": " + msg).c_str());
    } catch (...) {
        return code;
    }
}
template <class F>
int guarded(F f) noexcept {
    try {
        return f();
    } catch (...) {
        return OI_E_NOMEM;  // std::string is all that allocates here
    }
}

int launched(hipError_t e, const char *what) {
    return e == hipSuccess ? OI_OK : err(OI_E_DEVICE, what, hipGetErrorString(e));
}

bool aligned(const void *p, size_t n) { return (uintptr_t)p % n == 0; }
bool type_ok(int32_t t) { return t == OI_TYPE_F32 || t == OI_TYPE_F16; }
int64_t size_of(int32_t t) { return t == OI_TYPE_F16 ? 2 : 4; }
// rows of `len` elements, `stride` apart, read and written 16 bytes at a time
bool rows_ok(const void *p, int32_t type, int64_t stride, int64_t len) {
    return aligned(p, 16) && stride >= len && stride <= ((int64_t)1 << 40) && stride * size_of(type) % 16 == 0;
}
const char *const BAD_ROWS = "rows must be 16-byte aligned, a stride at least a row and a multiple of 16 bytes";

// A kernel is launched on the current device: a stream of another one is refused.
int stream_ok(void *stream, const char *what) {
    if (!stream) return OI_OK;
    int cur = -1;
    hipDevice_t dev = -1;
    if (hipGetDevice(&cur) != hipSuccess) return err(OI_E_DEVICE, what, "no current HIP device");
    if (hipStreamGetDevice((hipStream_t)stream, &dev) != hipSuccess) {
        (void)hipGetLastError();
        return OI_OK;  // the legacy and per-thread default streams are the current device's
    }
    if ((int)dev != cur) return err(OI_E_ARG, what, "the stream belongs to another device than the current one");
    return OI_OK;
}

// n pieces of `len` bytes, `stride` apart
struct Span {
    const void *p;
    int64_t len, n = 1, stride = 0;
};
// Whether any two pieces may meet: equal strides are looked at within one stride (q, k and v
// in one row of a projection lie between each other), others as a whole.
bool overlap(const Span &a, const Span &b) {
    if (!a.p || !b.p) return false;
    const __int128 x = (uintptr_t)a.p, y = (uintptr_t)b.p;  // n * stride may pass 64 bits
    if (x >= y + (__int128)(b.n - 1) * b.stride + b.len || y >= x + (__int128)(a.n - 1) * a.stride + a.len) return false;
    if (a.n == 1 || b.n == 1 || a.stride != b.stride) return true;
    const int64_t s = a.stride, by = (int64_t)((y - x) % s), r = by < 0 ? by + s : by;  // b's place behind a piece of a
    return r < a.len || s - r < b.len;
}

}  // namespace

}  // namespace oi
