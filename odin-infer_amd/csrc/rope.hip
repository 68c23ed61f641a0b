// rope.hip -- RMS norm of the q and k heads and their rotation by positions of
// three axes (time, height, width).
//
// Pair (i, i + rotary / 2) of a head turns by pos[axis(i)] * inv_freq[i]; text
// has one number on all three axes.  The angle is formed in 64 bits and reduced
// to [-pi/4, pi/4] there, since in 32 a position of 10^5 leaves it 2^-8 off;
// sine and cosine of the remainder are 32-bit.  One workgroup takes a token (a
// few heads of it where tokens are few): the angles are formed once for all its
// heads, then a wave takes a head at a time.  2311 tokens of 16 + 2 heads of 256 to
// f16 (64 MB) 18 us, bound by memory (about 6.5 us + bytes / 7 TB/s); a single token
// of 32 + 8 heads 3.6 us, the chain of load, norm and store.

#include "device_common.h"
#include "kv8.h"

namespace oi {

namespace {

constexpr int ROPE_MAX_HALF = 128;

__device__ __forceinline__ int rope_axis(const RopeArgs &a, int i) {
    if (a.interleaved) {
        const int ax = i % 3;
        return i < 3 * a.sec[ax] ? ax : 0;
    }
    return i < a.sec[0] ? 0 : i < a.sec[0] + a.sec[1] ? 1 : 2;
}

// cos and sin of pos * freq: k quarter turns taken off in 64 bits
__device__ __forceinline__ void turn(int pos, float freq, float &c, float &s) {
    const double ang = (double)pos * (double)freq;
    const double k = rint(ang * 0.63661977236758134308);
    double r = fma(-k, 1.57079632679489655800, ang);
    r = fma(-k, 6.12323399573676603587e-17, r);
    const int quad = (int)(k - 4.0 * floor(k * 0.25));
    float c0, s0;
    sincosf((float)r, &s0, &c0);
    c = quad == 0 ? c0 : quad == 1 ? -s0 : quad == 2 ? -c0 : s0;
    s = quad == 0 ? s0 : quad == 1 ? c0 : quad == 2 ? -s0 : -c0;
}

template <int E>
__device__ __forceinline__ void load_row(const void *p, int64_t at, bool f16, float (&x)[E]) {
    if (f16) {
        const uint16_t *h = (const uint16_t *)p + at;
        if constexpr (E == 2) {
            const uint32_t w = *(const uint32_t *)h;
            x[0] = h2f(w & 0xFFFFu);
            x[1] = h2f(w >> 16);
        } else {
            const u32x2 w = *(const u32x2 *)h;
            x[0] = h2f(w.x & 0xFFFFu);
            x[1] = h2f(w.x >> 16);
            x[2] = h2f(w.y & 0xFFFFu);
            x[3] = h2f(w.y >> 16);
        }
        return;
    }
    const float *f = (const float *)p + at;
    if constexpr (E == 2) {
        const float2 w = *(const float2 *)f;
        x[0] = w.x;
        x[1] = w.y;
    } else {
        const float4 w = *(const float4 *)f;
        x[0] = w.x;
        x[1] = w.y;
        x[2] = w.z;
        x[3] = w.w;
    }
}

template <int E>
__device__ __forceinline__ void store_row(void *p, int64_t at, bool f16, const float (&x)[E]) {
    if (f16) {
        uint16_t *h = (uint16_t *)p + at;
        uint32_t w[E / 2];
#pragma unroll
        for (int e = 0; e < E / 2; e++) w[e] = f2h(x[2 * e]) | (uint32_t)f2h(x[2 * e + 1]) << 16;
        if constexpr (E == 2) *(uint32_t *)h = w[0];
        else *(u32x2 *)h = u32x2{w[0], w[1]};
        return;
    }
    float *f = (float *)p + at;
    if constexpr (E == 2) *(float2 *)f = make_float2(x[0], x[1]);
    else *(float4 *)f = make_float4(x[0], x[1], x[2], x[3]);
}

template <int HD>
__global__ __launch_bounds__(WG) void rope_axes_kernel(RopeArgs a, int per) {
    constexpr int E = HD / WAVE;
    __shared__ float cs[ROPE_MAX_HALF], sn[ROPE_MAX_HALF];
    __shared__ __attribute__((aligned(16))) float row[WG / WAVE][HD];
    const int t = blockIdx.x, tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int half = a.rotary / 2, heads = a.n_heads + a.n_kv;
    const int h0 = blockIdx.y * per, h1 = min(h0 + per, heads);
    auto load = [&](int h, float (&x)[E]) {
        if (h < a.n_heads) load_row<E>(a.q, t * a.q_stride + h * a.q_head + E * lane, a.in_f16, x);
        else load_row<E>(a.k, t * a.k_stride + (int64_t)(h - a.n_heads) * HD + E * lane, a.in_f16, x);
    };
    // the next head is requested before this one is worked on, the first before the angles
    float x[E], next[E];
    int h = h0 + wave;
    if (h < h1) load(h, next);
    if (tid < half) turn(a.pos[(int64_t)rope_axis(a, tid) * a.n + t], a.inv_freq[tid], cs[tid], sn[tid]);
    __syncthreads();
    for (; h < h1; h += WG / WAVE) {
        const bool is_q = h < a.n_heads;
        float y[E];
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = next[e];
        if (h + WG / WAVE < h1) load(h + WG / WAVE, next);
        const float *w = is_q ? a.q_norm : a.k_norm;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < E; e++) ss += x[e] * x[e];
            const float inv = 1.0f / sqrtf(wave_sum(ss) / (float)HD + a.eps);
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = w[E * lane + e] * (inv * x[e]);
        }
#pragma unroll
        for (int e = 0; e < E; e++) row[wave][E * lane + e] = x[e];
        __builtin_amdgcn_wave_barrier();  // this wave's row only: DS operations of one wave complete in order
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int d = E * lane + e;
            y[e] = x[e];
            if (d < half) y[e] = x[e] * cs[d] - row[wave][d + half] * sn[d];
            else if (d < 2 * half) y[e] = row[wave][d - half] * sn[d - half] + x[e] * cs[d - half];
        }
        __builtin_amdgcn_wave_barrier();
        if (is_q) store_row<E>(a.qo, t * a.qo_stride + (int64_t)h * HD + E * lane, a.out_f16, y);
        else store_row<E>(a.ko, t * a.ko_stride + (int64_t)(h - a.n_heads) * HD + E * lane, a.out_f16, y);
    }
}

}  // namespace

hipError_t launch_rope_axes(const RopeArgs &a, hipStream_t st) {
    const int heads = a.n_heads + a.n_kv, per = a.n >= 256 ? heads : 4;
    const dim3 grid((unsigned)a.n, (unsigned)((heads + per - 1) / per));
    if (a.hd == 128) hipLaunchKernelGGL(rope_axes_kernel<128>, grid, dim3(WG), 0, st, a, per);
    else if (a.hd == 256) hipLaunchKernelGGL(rope_axes_kernel<256>, grid, dim3(WG), 0, st, a, per);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace oi
