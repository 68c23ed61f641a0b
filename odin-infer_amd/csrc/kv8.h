// kv8.h -- the 8-bit K/V cache and the rotation of q and k: kernel arguments
// and launches shared by kv8.cpp (the C entries), kv8.hip, kv8_attn.hip and
// rope.hip.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace oi {

constexpr int KV8_TILE = 64;                 // slots of a V tile, of a wave's step
constexpr int KV8_EMIN = -24, KV8_EMAX = 10;  // exponents of a block's scale 2^e

// One cache buffer in its parts.
struct Kv8 {
    int8_t *kc;  // [n_kv][cap][hd]
    int8_t *vc;  // [n_kv][cap / 64][hd][64]
    int8_t *ke;  // [n_kv][cap / block]
    int8_t *ve;
    int32_t n_kv, hd, cap, lb;  // lb: log2(block)
};

// slots in use before a call: `past`, or *past_dev (clamped to what fits) where set
struct Kv8Past {
    int32_t past;
    const int32_t *dev;
};

struct Kv8AppendArgs {
    Kv8 c;
    const void *x[2];     // K and V rows of the first token, f32 or f16
    int64_t stride[2];    // elements from a token to the next
    int32_t f16, n;
    Kv8Past past;
};
hipError_t launch_kv8_append(const Kv8AppendArgs &a, hipStream_t st);

struct Kv8ReadArgs {
    Kv8 c;
    void *out[2];  // [n_kv][n][hd]
    int32_t f16, slot0, n;
};
hipError_t launch_kv8_read(const Kv8ReadArgs &a, hipStream_t st);

struct Kv8AttnArgs {
    Kv8 c;
    const void *q;        // token t's heads at q + t * q_stride
    int64_t q_stride, out_stride;
    void *out;
    float scale;          // of q . k, times log2(e)
    int32_t f16, n, n_heads, group;
    uint32_t magic;       // ceil(2^32 / group), 0 for a group of 1
    Kv8Past past;
    float *mass;          // [n_kv][cap] or null
    float *part;          // [n * n_heads][splits][hd], where splits > 1: the splits' o
    float4 *ml;           // [n * n_heads][splits]: their m, l of the products' weights, l of the exact ones
    float2 *norm;         // [n * n_heads], where mass is set: m and 2^15 / l of a row
    // few rows with mass: every weight as it was formed [n_kv][save_units][4][rows][16]
    // and its row's maximum then [n_kv][save_units][rows]; null otherwise
    float *save, *save_m;
    int32_t save_units, splits;
    // many rows with mass: splits of the rows, and where msplits > 1 their sums [msplits][n_kv][msum_slots]
    float *msum;
    int32_t msum_slots, msplits;
};
// splits over the slots for a call that sees at most `end` of them, and the workspace that they take
int kv8_attn_splits(int n_kv, int group, int n, int end, int hd, bool f16);
bool kv8_attn_saves(int group, int n);
int kv8_mass_splits(int n_kv, int group, int n, int end, int hd);
size_t kv8_attn_workspace(int n_heads, int group, int n, int end, int hd, int splits, bool mass);
size_t kv8_attn_workspace_most(int n_heads, int group, int n, int cap, int hd);  // at any length, with mass
hipError_t launch_kv8_attn(const Kv8AttnArgs &a, hipStream_t st);

struct Kv8EvictArgs {
    Kv8 src, dst;
    const float *mass;
    const int32_t *pos;
    float *dst_mass;
    int32_t *dst_pos, *kept;  // kept [n_kv][keep]
    int32_t n, keep, first, last;
};
hipError_t launch_kv8_evict(const Kv8EvictArgs &a, hipStream_t st);

struct RopeArgs {
    const void *q, *k;
    void *qo, *ko;
    int64_t q_stride, q_head, k_stride, qo_stride, ko_stride;
    const int32_t *pos;              // [3][n]
    const float *inv_freq;           // [rotary / 2]
    const float *q_norm, *k_norm;    // [hd] or null
    float eps;
    int32_t n, n_heads, n_kv, hd, rotary, sec[3], interleaved, in_f16, out_f16;
};
hipError_t launch_rope_axes(const RopeArgs &a, hipStream_t st);

}  // namespace oi
