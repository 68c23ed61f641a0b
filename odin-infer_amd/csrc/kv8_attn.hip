// kv8_attn.hip -- attention over the 8-bit K/V cache.
//
// Token i of the call sees slots 0 .. past + i.  With K_j = a_j 2^k(j) and
// V_j = b_j 2^v(j) (bytes a, b; exponents per block of slots), scores in base 2:
//   t_j = (q . a_j) 2^k(j) scale log2(e) + v(j)
//   p_j = 2^(t_j - m + 15),  m the running maximum of t over the row
//   o = sum p_j b_j,   l = sum p_j 2^-v(j),   out = o / l
// V's exponent sits in the softmax exponent, so the weight that multiplies the
// bytes of V never passes 2^15 whatever the blocks' steps, and l takes it out
// again exactly (a power of two).  m, l and o are 32-bit.  The matrix products
// take f16 operands: a and b are exact there; q and p of an f32 call are each
// the sum of two halves (22 bits, q scaled by a power of two per row), of an
// f16 call q is exact and p is rounded once to 11 bits (the size of the output's
// own rounding).  2^15 is where the largest weight sits in f16: a weight keeps
// all its bits down to 2^-29 of it and is lost below 2^-40.

#include "kv8_common.h"

namespace oi {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int T = KV8_TILE;
constexpr float NEG = -3.402823466e38f;  // the running maximum before any slot
constexpr float PSCALE = 15.f;

// 8 signed bytes as halves: byte ^ 128 behind 0x64 is 1024 + 128 + byte
__device__ __forceinline__ f16x8 bytes_h(uint32_t lo, uint32_t hi) {
    const f16x2 bias = {(_Float16)1152.f, (_Float16)1152.f};
    const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u, k = 0x64646464u;
    const f16x2 w0 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(k, a, 0x04010400u)) - bias;
    const f16x2 w1 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(k, a, 0x04030402u)) - bias;
    const f16x2 w2 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(k, b, 0x04010400u)) - bias;
    const f16x2 w3 = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(k, b, 0x04030402u)) - bias;
    return f16x8{w0.x, w0.y, w1.x, w1.y, w2.x, w2.y, w3.x, w3.y};
}

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// over the four lanes of a column (xor 16 and 32)
__device__ __forceinline__ float col_max(float v) {
    v = fmaxf(v, __shfl_xor(v, 16, WAVE));
    return fmaxf(v, __shfl_xor(v, 32, WAVE));
}
__device__ __forceinline__ float col_sum(float v) {
    v += __shfl_xor(v, 16, WAVE);
    return v + __shfl_xor(v, 32, WAVE);
}

// 16 rows of q as the products' second operand: lane (column c, group g) holds
// dimensions 64 k + 16 g + 8 h + 0..7 of row c, the order in which its 16-byte
// loads of K fall.  f32 rows: two halves of q 2^-e, e the row's exponent.
template <int HD, bool F16>
struct QTile {
    static constexpr int NF = HD / 32;
    f16x8 hi[NF], lo[F16 ? 1 : NF];
    int e = 0;

    __device__ __forceinline__ void load(const void *q, int64_t at, int g, bool ok) {
        if constexpr (F16) {
            const u32x4 z = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const int d = 64 * (f / 2) + 16 * g + 8 * (f & 1);
                hi[f] = __builtin_bit_cast(f16x8, ok ? *(const u32x4 *)((const uint16_t *)q + at + d) : z);
            }
        } else {
            float x[NF][8];
            float amax = 0.f;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const int d = 64 * (f / 2) + 16 * g + 8 * (f & 1);
                const float4 *p = (const float4 *)((const float *)q + at + d), z = make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 u = ok ? p[0] : z, w = ok ? p[1] : z;
                x[f][0] = u.x; x[f][1] = u.y; x[f][2] = u.z; x[f][3] = u.w;
                x[f][4] = w.x; x[f][5] = w.y; x[f][6] = w.z; x[f][7] = w.w;
#pragma unroll
                for (int i = 0; i < 8; i++) amax = fmaxf(amax, fabsf(x[f][i]));
            }
            amax = col_max(amax);
            e = amax > 0.f ? (int)(__float_as_uint(amax) >> 23) - 127 - 14 : 0;
#pragma unroll
            for (int f = 0; f < NF; f++)
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float y = ldexpf(x[f][i], -e);
                    const _Float16 h = (_Float16)y;
                    hi[f][i] = h;
                    lo[f][i] = (_Float16)(y - (float)h);
                }
        }
    }
};

// Where row r (of a kv head's n * group rows, token-major) has its head in q or out
__device__ __forceinline__ int64_t row_at(int r, int group, int kvh, int64_t stride, int hd) {
    return (int64_t)(r / group) * stride + (int64_t)(kvh * group + r % group) * hd;
}

// A wave takes a unit of 64 slots at a time for 16 rows of one kv head (the
// (token, query head) pairs that share it), four waves a workgroup, alternate
// units.  Scores are formed transposed, K the first operand: a lane then holds
// 16 scores of one row, and with K's rows taken in the order
//   operand row 4 g' + i of tile t  <-  slot 16 g' + 4 t + i
// these are slots 16 g .. 16 g + 15, of one block and exactly those whose
// weights the lane supplies to the second product: nothing crosses lanes but
// the row maximum.  K and V go from memory to the operand registers without
// LDS, 16 bytes a lane; K of the next unit is requested when this unit's scores
// are done, V when its product is.  The waves' results meet in LDS.
template <int HD, bool F16>
__global__ __launch_bounds__(WG) void kv8_rows_kernel(Kv8AttnArgs a) {
    constexpr int NK = HD / 64, ND = HD / 16, PD = HD + 4;
    __shared__ __attribute__((aligned(16))) float so[4][16][PD];
    __shared__ float sm[4][16], sl[4][16];
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int c = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x, rt = blockIdx.y, split = blockIdx.z;
    const int rows = a.n * a.group, past = kv8_past(a.past, a.n, a.c.cap);
    const int row = rt * 16 + c;
    const bool ok = row < rows;
    const int rr = min(row, rows - 1);
    const int limit = past + rr / a.group + 1;  // slots that this row sees
    const int first_limit = past + (rt * 16) / a.group + 1;
    const int last_limit = past + min(rt * 16 + 15, rows - 1) / a.group + 1;
    const int units = (last_limit + T - 1) / T;
    const int per = (units + a.splits * 4 - 1) / (a.splits * 4) * 4;
    const int u0 = split * per, u1 = min(u0 + per, units);
    QTile<HD, F16> q;
    q.load(a.q, row_at(rr, a.group, kvh, a.q_stride, HD), g, ok);

    const int8_t *kb = a.c.kc + (size_t)kvh * a.c.cap * HD;
    const int8_t *vb = a.c.vc + (size_t)kvh * a.c.cap * HD;
    const int8_t *ke = a.c.ke + (size_t)kvh * (a.c.cap >> a.c.lb);
    const int8_t *ve = a.c.ve + (size_t)kvh * (a.c.cap >> a.c.lb);
    const int krow = 16 * (c >> 2) + (c & 3);
    u32x4 kr[4][NK], vr[ND];
    int kexp = 0, vexp = 0;
    auto load_k = [&](int u) {
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int k = 0; k < NK; k++)
                kr[t][k] = ldg_nt((const u32x4 *)(kb + (size_t)(u * T + krow + 4 * t) * HD + 64 * k + 16 * g));
        kexp = ke[(u * T + 16 * g) >> a.c.lb];
        vexp = ve[(u * T + 16 * g) >> a.c.lb];
    };
    auto load_v = [&](int u) {
#pragma unroll
        for (int d = 0; d < ND; d++)
            vr[d] = ldg_nt((const u32x4 *)(vb + ((size_t)u * HD + 16 * d + c) * T + 16 * g));
    };
    float m = NEG, l = 0.f;
    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    int u = u0 + wave;
    if (u < u1) {
        load_k(u);
        load_v(u);
    }
    for (; u < u1; u += 4) {
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) {
            s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < NK; k++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const f16x8 w = bytes_h(kr[t][k][2 * h], kr[t][k][2 * h + 1]);
                    s[t] = mfma(w, q.hi[2 * k + h], s[t]);
                    if constexpr (!F16) s[t] = mfma(w, q.lo[2 * k + h], s[t]);
                }
        }
        const float mul = ldexpf(a.scale, kv8_exp((int8_t)kexp) + q.e);
        const int ev = kv8_exp((int8_t)vexp);
        if (u + 4 < u1) load_k(u + 4);
        const int p0 = u * T + 16 * g;  // the lane's first slot
        const bool edge = u * T + T > first_limit;
        float top = NEG;
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[t][i] = fmaf(s[t][i], mul, (float)ev);
                if (edge && p0 + 4 * t + i >= limit) s[t][i] = -INFINITY;
                top = fmaxf(top, s[t][i]);
            }
        top = col_max(top);
        const float m1 = fmaxf(m, top), alpha = exp2f(m - m1);
        float sum = 0.f;
        f16x8 ph[2], pl[2];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = exp2f(s[t][i] - m1 + PSCALE);
                sum += p;
                const _Float16 h = (_Float16)p;
                ph[t / 2][4 * (t & 1) + i] = h;
                if constexpr (!F16) pl[t / 2][4 * (t & 1) + i] = (_Float16)(p - (float)h);
            }
        m = m1;
        l = l * alpha + sum * pow2i(-ev);
#pragma unroll
        for (int d = 0; d < ND; d++) {
            o[d] *= alpha;
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const f16x8 w = bytes_h(vr[d][2 * h], vr[d][2 * h + 1]);
                o[d] = mfma(w, ph[h], o[d]);
                if constexpr (!F16) o[d] = mfma(w, pl[h], o[d]);
            }
        }
        if (u + 4 < u1) load_v(u + 4);
    }
    l = col_sum(l);
#pragma unroll
    for (int d = 0; d < ND; d++) *(f32x4 *)&so[wave][c][16 * d + 4 * g] = o[d];
    if (g == 0) {
        sm[wave][c] = m;
        sl[wave][c] = l;
    }
    __syncthreads();
    const int n_rows = min(16, rows - rt * 16);
    for (int i = tid; i < n_rows * HD; i += WG) {
        const int r = i / HD, d = i % HD;
        const float M = fmaxf(fmaxf(sm[0][r], sm[1][r]), fmaxf(sm[2][r], sm[3][r]));
        float O = 0.f, L = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = exp2f(sm[w][r] - M);
            O += so[w][r][d] * f;
            L += sl[w][r] * f;
        }
        const int gr = rt * 16 + r, head = kvh * a.group + gr % a.group;
        const size_t id = (size_t)(gr / a.group) * a.n_heads + head;
        float *pt = a.part + ((size_t)split * a.n * a.n_heads + id) * (HD + 2);
        pt[d] = O;
        if (d == 0) {
            pt[HD] = M;
            pt[HD + 1] = L;
        }
    }
}

// One wave-multiple of threads per (token, query head): the splits' weights,
// their sum, out = o / l; and the row's base-2 log of the sum of weights.
template <int HD, bool F16>
__global__ __launch_bounds__(HD) void kv8_merge_kernel(Kv8AttnArgs a) {
    const int id = blockIdx.x, d = threadIdx.x;
    const size_t step = (size_t)a.n * a.n_heads * (HD + 2);
    const float *pt = a.part + (size_t)id * (HD + 2);
    float M = NEG;
    for (int s = 0; s < a.splits; s++) M = fmaxf(M, pt[s * step + HD]);
    float O = 0.f, L = 0.f;
    for (int s = 0; s < a.splits; s++) {
        const float f = exp2f(pt[s * step + HD] - M);
        O += pt[s * step + d] * f;
        L += pt[s * step + HD + 1] * f;
    }
    const float y = O / L;
    const int64_t at = (int64_t)(id / a.n_heads) * a.out_stride + (int64_t)(id % a.n_heads) * HD + d;
    if constexpr (F16) ((uint16_t *)a.out)[at] = f2h(y);
    else ((float *)a.out)[at] = y;
    if (d == 0 && a.lse) a.lse[id] = M + log2f(L) - PSCALE;
}

// The weight that every slot receives from the call's rows, summed in f32 over
// all of them: scores formed again from K (half of the cache) and each row's
// log-sum.  A workgroup owns a unit of 64 slots, or four where one tile of rows
// is all there is; its waves take alternate row tiles and meet in LDS, so every
// sum is in a fixed order.
template <int HD, bool F16>
__global__ __launch_bounds__(WG) void kv8_mass_kernel(Kv8AttnArgs a, int upw) {
    constexpr int NK = HD / 64;
    __shared__ float sum[4][T];
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int c = lane & 15, g = lane >> 4, kvh = blockIdx.x;
    const int rows = a.n * a.group, past = kv8_past(a.past, a.n, a.c.cap), end = past + a.n;
    const int u = blockIdx.y * upw + (upw > 1 ? wave : 0);
    const bool have = u * T < end;
    const int8_t *kb = a.c.kc + (size_t)kvh * a.c.cap * HD;
    const int krow = 16 * (c >> 2) + (c & 3);
    float acc[4][4];
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[t][i] = 0.f;
    if (have) {
        u32x4 kr[4][NK];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int k = 0; k < NK; k++)
                kr[t][k] = *(const u32x4 *)(kb + (size_t)(u * T + krow + 4 * t) * HD + 64 * k + 16 * g);
        const int kexp = kv8_exp(a.c.ke[(size_t)kvh * (a.c.cap >> a.c.lb) + ((u * T + 16 * g) >> a.c.lb)]);
        // the first row that sees a slot of this unit
        const int tok0 = max(0, u * T - past), rt0 = tok0 * a.group / 16;
        for (int rt = rt0 + (upw > 1 ? 0 : wave); rt * 16 < rows; rt += upw > 1 ? 1 : 4) {
            const int row = rt * 16 + c, rr = min(row, rows - 1);
            const bool ok = row < rows;
            const int limit = ok ? past + rr / a.group + 1 : 0;
            QTile<HD, F16> q;
            q.load(a.q, row_at(rr, a.group, kvh, a.q_stride, HD), g, ok);
            const float lse = a.lse[(size_t)(rr / a.group) * a.n_heads + kvh * a.group + rr % a.group];
            const float mul = ldexpf(a.scale, kexp + q.e);
#pragma unroll
            for (int t = 0; t < 4; t++) {
                f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < NK; k++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const f16x8 w = bytes_h(kr[t][k][2 * h], kr[t][k][2 * h + 1]);
                        s = mfma(w, q.hi[2 * k + h], s);
                        if constexpr (!F16) s = mfma(w, q.lo[2 * k + h], s);
                    }
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (u * T + 16 * g + 4 * t + i < limit) acc[t][i] += exp2f(fmaf(s[i], mul, -lse));
            }
        }
    }
#pragma unroll
    for (int t = 0; t < 4; t++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float v = lane_group_sum(acc[t][i], 16);
            if (c == 0) sum[wave][16 * g + 4 * t + i] = v;
        }
    __syncthreads();
    if (upw > 1) {
        const int s = u * T + lane;
        if (s < end) {
            float *m = a.mass + (size_t)kvh * a.c.cap + s;
            *m = s < past ? *m + sum[wave][lane] : sum[wave][lane];
        }
    } else if (tid < T) {
        const int s = u * T + tid;
        if (s < end) {
            const float v = (sum[0][tid] + sum[1][tid]) + (sum[2][tid] + sum[3][tid]);
            float *m = a.mass + (size_t)kvh * a.c.cap + s;
            *m = s < past ? *m + v : v;
        }
    }
}

}  // namespace

int kv8_attn_splits(int n_kv, int group, int n, int end) {
    const int64_t units = (end + T - 1) / T, tiles = ((int64_t)n * group + 15) / 16 * n_kv;
    int64_t s = (units + 3) / 4;  // a unit per wave
    const int64_t want = (768 + tiles - 1) / tiles;
    if (s > want) s = want;
    return s < 1 ? 1 : (int)s;
}

size_t kv8_attn_workspace(int n_heads, int n, int hd, int splits) {
    return (size_t)n * n_heads * ((size_t)splits * (hd + 2) + 1) * 4;
}

hipError_t launch_kv8_attn(const Kv8AttnArgs &a, hipStream_t st) {
    const int rows = a.n * a.group;
    const dim3 g1((unsigned)a.c.n_kv, (unsigned)((rows + 15) / 16), (unsigned)a.splits);
    const dim3 g2((unsigned)(a.n * a.n_heads));
    const int end = a.past.dev ? a.c.cap : a.past.past + a.n, units = (end + T - 1) / T;
    const int upw = rows <= 16 ? 4 : 1;
    const dim3 g3((unsigned)a.c.n_kv, (unsigned)((units + upw - 1) / upw));
    auto go = [&](auto k1, auto k2, auto k3) {
        hipLaunchKernelGGL(k1, g1, dim3(WG), 0, st, a);
        hipLaunchKernelGGL(k2, g2, dim3((unsigned)a.c.hd), 0, st, a);
        if (a.mass) hipLaunchKernelGGL(k3, g3, dim3(WG), 0, st, a, upw);
    };
    if (a.c.hd == 128) {
        if (a.f16) go(kv8_rows_kernel<128, true>, kv8_merge_kernel<128, true>, kv8_mass_kernel<128, true>);
        else go(kv8_rows_kernel<128, false>, kv8_merge_kernel<128, false>, kv8_mass_kernel<128, false>);
    } else if (a.c.hd == 256) {
        if (a.f16) go(kv8_rows_kernel<256, true>, kv8_merge_kernel<256, true>, kv8_mass_kernel<256, true>);
        else go(kv8_rows_kernel<256, false>, kv8_merge_kernel<256, false>, kv8_mass_kernel<256, false>);
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace oi
