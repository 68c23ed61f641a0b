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
// f32 -> f16 of what is made of cached values: these go to 127 * 2^10, twice f16's largest
// number, which stands for all beyond it (an f16 value that the block's step rounds up to
// 65536 is one); NaN stays NaN
static __device__ __forceinline__ uint16_t f2h_top(float f) {
    return f2h(f != f ? f : __builtin_amdgcn_fmed3f(f, -65504.f, 65504.f));
}

}  // namespace oi
