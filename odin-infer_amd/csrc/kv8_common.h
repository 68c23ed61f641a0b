// kv8_common.h -- device helpers of the 8-bit cache kernels.
#pragma once
#include "device_common.h"
#include "kv8.h"

namespace oi {

typedef float f32x4 __attribute__((ext_vector_type(4)));

static __device__ __forceinline__ int kv8_past(const Kv8Past &p, int n, int cap) {
    return p.dev ? min(max(*p.dev, 0), cap - n) : p.past;
}
// An exponent as stored; memory that was never written may hold any byte.
static __device__ __forceinline__ int kv8_exp(int8_t e) { return min(max((int)e, KV8_EMIN), KV8_EMAX); }
// 2^e, e within the normal exponents
static __device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }

}  // namespace oi
