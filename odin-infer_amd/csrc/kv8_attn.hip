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
// f16 call q is exact.  Its p is the sum of two halves where at most 8 rows share a
// kv head (half of a product's columns are free for the second; the error of one
// token over 37000 slots is then that of the output's rounding, 1.7e-4, and was
// 2.9e-4, in the same time), with more rows rounded once to 11 bits (2.2e-4 against
// 2.0e-4; a second product each would cost a third of the rate).
// 2^15 is where the row's largest p sits in f16: another keeps all its bits down to
// 2^-29 of it and is lost below 2^-40, from o, where both count with their blocks'
// steps.  A slot loses less than 2^-30 of half the step of the largest one's block, which
// storing that one's V may have cost (2^-24 in the prompt's f16 form).
// In l they count without the steps: a slot in a block of small V (of zeros, step 2^-24)
// may hold most of the row's weight while its p is far below f16's numbers.  So l is
// the sum of p before the rounding, but for 11-bit weights where V's steps are near
// each other: there it is the sum of the rounded p (a weight that dominates loses
// nothing, 2.1e-4 against 2.8e-4), near as stated at NEAR_SUM and NEAR_EXP.
// The mass takes the sum of p before the rounding.

#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "kv8_common.h"

namespace oi {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr int T = KV8_TILE;
constexpr float NEG = -3.402823466e38f;  // the running maximum before any slot
constexpr float PSCALE = 15.f;
// Where l takes rounded weights.  Half a subnormal of f16 is 2^-25.
// Rows kernel: a lane's 16 slots, of one block, where their sum is at least this: what
// subnormals lose is below 2^-18 of it.
constexpr float NEAR_SUM = 0.125f;
// Prompt kernel: a unit whose exponents of V are all up to this far below the largest so
// far: the slot with the largest score then has put 2^(7 - that largest) or more into l,
// and a subnormal loses 2^-28 of that at most.
constexpr float NEAR_EXP = 4.f;

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

// v of the lanes 16 and 32 away, by register swaps between halves and rows of 16
template <class F>
__device__ __forceinline__ float col_reduce(float v, F f) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// over the four lanes of a column (16 and 32 apart)
__device__ __forceinline__ float col_max(float v) {
    return col_reduce(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float col_sum(float v) {
    return col_reduce(v, [](float a, float b) { return a + b; });
}
// v and that of the column 8 away.  By value: __builtin_bit_cast of a vector's
// element (inside OI_DPP) takes the vector's first one.
__device__ __forceinline__ float half_sum(float v) { return v + OI_DPP(v, 0x128); }
// the sum of 8 halves in f32, one mixed multiply-add each (v_dot2_f32_f16 took 3% more of a prompt)
__device__ __forceinline__ float sum8(f16x8 p) {
    float lo = 0.f, hi = 0.f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = __builtin_bit_cast(uint32_t, f16x2{p[2 * i], p[2 * i + 1]});
        asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel_hi:[1,0,0]" : "+v"(lo) : "v"(w));
        asm("v_fma_mix_f32 %0, %1, 1.0, %0 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "+v"(hi) : "v"(w));
    }
    return lo + hi;
}
// 2^x; results below the normal numbers are 0
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// How a tile of rows lies in the 16 columns of the products' second operand.
enum {
    ROWS_F16 = 0,   // 16 rows of an f16 q
    ROWS_F32 = 1,   // 16 rows of an f32 q, two operands each (upper and lower half)
    ROWS_PACK = 2,  // 8 rows of an f32 q: upper halves in columns 0..7, lower halves in 8..15, one product for both
    ROWS_F16_PACK = 3,  // 8 rows of an f16 q, twice; only the weights p are packed so
};
constexpr bool rows_packed(int mode) { return mode == ROWS_PACK || mode == ROWS_F16_PACK; }
constexpr bool rows_f16(int mode) { return mode == ROWS_F16 || mode == ROWS_F16_PACK; }
constexpr int tile_rows(int mode) { return rows_packed(mode) ? 8 : 16; }

// A tile of q as that operand: lane (column c, group g) holds dimensions
// 64 k + 16 g + 8 h + 0..7 of its row, the order in which its 16-byte loads of K
// fall.  f32 rows are made into two halves of q 2^-e (e the row's exponent) by the
// workgroup together, a row by 256 / R threads, and pass through LDS: each wave
// for itself took 1.8 us more at head_dim 256, in one long run of instructions.  A
// negative scale turns q's sign, so that the largest score is that of the largest product.
template <int HD, int MODE>
struct QTile {
    static constexpr int NF = HD / 32, R = tile_rows(MODE);
    static constexpr bool F16 = rows_f16(MODE), TWO = MODE == ROWS_F32;
    static constexpr int TPR = WG / R, EL = HD / TPR;  // f32: threads of a row, elements of a thread
    struct Lds {
        f16x8 half[2][R][HD / 8];  // upper, lower; piece j of row r at j ^ (r & 7)
        int e[R];
    };
    f16x8 hi[NF], lo[TWO ? NF : 1];
    int e = 0;
    u32x4 raw[F16 ? NF : EL / 4];

    // f16: the loads of row `at`, this lane's; f32: `at` is the row of thread tid / TPR
    __device__ __forceinline__ void fetch(const void *q, int64_t at, int tid) {
        if constexpr (F16) {
            const int g = (tid & (WAVE - 1)) >> 4;
#pragma unroll
            for (int f = 0; f < NF; f++)
                raw[f] = *(const u32x4 *)((const uint16_t *)q + at + 64 * (f / 2) + 16 * g + 8 * (f & 1));
        } else {
#pragma unroll
            for (int i = 0; i < EL / 4; i++)
                raw[i] = *(const u32x4 *)((const float *)q + at + tid % TPR * EL + 4 * i);
        }
    }
    // f32: the halves into LDS (a barrier follows)
    __device__ __forceinline__ void split(Lds &lds, int tid, bool neg) {
        if constexpr (!F16) {
            const int r = tid / TPR, j = tid % TPR;
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < EL / 4; i++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const uint32_t bits = raw[i][k];
                    amax = fmaxf(amax, fabsf(__uint_as_float(bits)));
                }
            amax = fmaxf(amax, OI_DPP(amax, 0xB1));
            amax = fmaxf(amax, OI_DPP(amax, 0x4E));
            amax = fmaxf(amax, OI_DPP(amax, 0x141));
            amax = fmaxf(amax, OI_DPP(amax, 0x140));
            if constexpr (TPR == 32) {
                const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(amax), __float_as_uint(amax), false, false);
                amax = fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]));
            }
            const int ex = amax > 0.f ? (int)(__float_as_uint(amax) >> 23) - 127 - 14 : 0;
            uint32_t h[EL / 2], l[EL / 2];
#pragma unroll
            for (int i = 0; i < EL / 2; i++) {
                f16x2 th, tl;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const uint32_t bits = raw[i / 2][2 * (i & 1) + k];
                    const float x = __uint_as_float(bits), y = ldexpf(neg ? -x : x, -ex);
                    const _Float16 t = (_Float16)y;
                    th[k] = t;
                    tl[k] = (_Float16)(y - (float)t);
                }
                h[i] = __builtin_bit_cast(uint32_t, th);
                l[i] = __builtin_bit_cast(uint32_t, tl);
            }
            // pieces of 8 elements; a thread of 4 elements writes half of one
            constexpr int W = EL < 8 ? EL / 2 : 4;  // words of a piece per thread
#pragma unroll
            for (int i = 0; i < (EL + 7) / 8; i++) {
                const int el = j * EL + 8 * i;
                uint32_t *ph = (uint32_t *)&lds.half[0][r][(el / 8) ^ (r & 7)] + el % 8 / 2,
                         *pl = (uint32_t *)&lds.half[1][r][(el / 8) ^ (r & 7)] + el % 8 / 2;
#pragma unroll
                for (int k = 0; k < W; k++) {
                    ph[k] = h[4 * i + k];
                    pl[k] = l[4 * i + k];
                }
            }
            if (j == 0) lds.e[r] = ex;
        }
    }
    // the operands, zero with ok = false
    __device__ __forceinline__ void make(const Lds &lds, int tid, bool ok, bool neg) {
        const int c = tid & 15, g = (tid & (WAVE - 1)) >> 4;
        if constexpr (F16) {
            const uint32_t sign = neg ? 0x80008000u : 0u;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                u32x4 w;
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = ok ? raw[f][i] ^ sign : 0u;
                hi[f] = __builtin_bit_cast(f16x8, w);
            }
        } else {
            const int r = c % R;
            e = lds.e[r];
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const int at = (8 * (f / 2) + 2 * g + (f & 1)) ^ (r & 7);
                hi[f] = lds.half[TWO ? 0 : c / R][r][at];
                if constexpr (TWO) lo[f] = lds.half[1][r][at];
            }
        }
    }
};

// One tile of 16 slots of raw K times the rows
template <int HD, int MODE>
__device__ __forceinline__ f32x4 scores(const u32x4 (&kr)[HD / 64], const QTile<HD, MODE> &q) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < HD / 64; k++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const f16x8 w = bytes_h(kr[k][2 * h], kr[k][2 * h + 1]);
            s = mfma(w, q.hi[2 * k + h], s);
            if constexpr (MODE == ROWS_F32) s = mfma(w, q.lo[2 * k + h], s);
        }
    if constexpr (MODE == ROWS_PACK)
#pragma unroll
        for (int i = 0; i < 4; i++) s[i] = half_sum(s[i]);
    return s;
}

// The token of row r of a kv head's n * group rows (token-major): r / group by a
// multiplication (magic = ceil(2^32 / group), exact while r * group < 2^32)
__device__ __forceinline__ int row_token(const Kv8AttnArgs &a, int r) {
    return a.magic ? (int)__umulhi((uint32_t)r, a.magic) : r;
}
// where the row's head lies in q or out, and its place among the n * n_heads rows
__device__ __forceinline__ int64_t row_at(const Kv8AttnArgs &a, int r, int kvh, int64_t stride, int hd) {
    const int t = row_token(a, r);
    return t * stride + (int64_t)(kvh * a.group + r - t * a.group) * hd;
}
__device__ __forceinline__ size_t row_id(const Kv8AttnArgs &a, int r, int kvh) {
    const int t = row_token(a, r);
    return (size_t)t * a.n_heads + kvh * a.group + r - t * a.group;
}

// A wave takes a unit of 64 slots at a time for 16 rows of one kv head (the
// (token, query head) pairs that share it), the waves of a workgroup alternate
// units.  Scores are formed transposed, K the first operand: a lane then holds
// 16 scores of one row, and with K's rows taken in the order
//   operand row 4 g' + i of tile t  <-  slot 16 g' + 4 t + i
// these are slots 16 g .. 16 g + 15, of one block and exactly those whose
// weights the lane supplies to the second product: nothing crosses lanes but
// the row maximum.  K and V go from memory to the operand registers without
// LDS, 16 bytes a lane; K of the next unit is requested when this unit's scores
// are done, V when its product is.  The waves' results meet in LDS.  The running
// maximum is raised to whole numbers: the rescaling is exact then, and so is the
// sum of V's exponent, the maximum and the offset in front of the exponential.
// Long caches are bound by memory: 100004 slots of 4 kv heads of 128 (102 MB)
// 22 us, where a read of that size by itself takes about 6.5 us + bytes / 7 TB/s;
// short ones by one wave's chain of loads, products and the merge: 1031 slots
// 7 us.  SAVE (26 us) leaves the weights for the mass.
template <int HD, int MODE, bool SAVE>
__global__ __launch_bounds__(WG) void kv8_rows_kernel(Kv8AttnArgs a) {
    constexpr int NW = WG / WAVE, NK = HD / 64, ND = HD / 16, PD = HD + 4, R = tile_rows(MODE), TPR = WG / R;
    constexpr bool F16 = rows_f16(MODE), PACK = rows_packed(MODE), ROUND = F16 && !PACK;  // ROUND: p in 11 bits
    __shared__ __attribute__((aligned(16))) union {
        float o[NW][R][PD];
        typename QTile<HD, MODE>::Lds q;
    } lds;
    __shared__ float sm[NW][R], sl[NW][R], sx[NW][R];
    auto &so = lds.o;
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int c = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x, rt = blockIdx.y, split = blockIdx.z;
    const int rows = a.n * a.group, past = kv8_past(a.past, a.n, a.c.cap);
    const int row = rt * R + c % R;
    const bool ok = row < rows, lower = c >= R;
    const int rr = min(row, rows - 1);
    const int limit = past + row_token(a, rr) + 1;  // slots that this row sees
    const int first_limit = past + row_token(a, rt * R) + 1;
    const int last_limit = past + row_token(a, min(rt * R + R - 1, rows - 1)) + 1;
    const int units = (last_limit + T - 1) / T;
    const int u0 = (int)((int64_t)split * units / a.splits), u1 = (int)((int64_t)(split + 1) * units / a.splits);
    const bool neg = a.scale < 0.f;
    QTile<HD, MODE> q;
    q.fetch(a.q, row_at(a, F16 ? rr : min(rt * R + tid / TPR, rows - 1), kvh, a.q_stride, HD), tid);

    const int krow = 16 * (c >> 2) + (c & 3);
    const int8_t *kb = a.c.kc + (size_t)kvh * a.c.cap * HD + krow * HD + 16 * g;
    const int8_t *vb = a.c.vc + (size_t)kvh * a.c.cap * HD + c * T + 16 * g;
    const int8_t *ke = a.c.ke + (size_t)kvh * (a.c.cap >> a.c.lb);
    const int8_t *ve = a.c.ve + (size_t)kvh * (a.c.cap >> a.c.lb);
    u32x4 kr[4][NK], vr[ND];
    int kexp = 0, vexp = 0;
    auto load_k = [&](int u) {
        const int8_t *p = kb + (size_t)u * (T * HD);
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int k = 0; k < NK; k++) kr[t][k] = *(const u32x4 *)(p + 4 * t * HD + 64 * k);
        kexp = ke[(u * T + 16 * g) >> a.c.lb];
        vexp = ve[(u * T + 16 * g) >> a.c.lb];
    };
    auto load_v = [&](int u) {
        const int8_t *p = vb + (size_t)u * (T * HD);
#pragma unroll
        for (int d = 0; d < ND; d++) vr[d] = *(const u32x4 *)(p + 16 * d * T);
    };
    float m = NEG, l = 0.f, lx = 0.f;  // lx: of the weights before their rounding to f16
    f32x4 o[ND];
#pragma unroll
    for (int d = 0; d < ND; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    int u = u0 + wave;
    if (u < u1) {
        load_k(u);
        load_v(u);
    }
    if constexpr (!F16) {
        q.split(lds.q, tid, neg);
        __syncthreads();
    }
    q.make(lds.q, tid, ok, neg);
    const float scale = fabsf(a.scale);
    for (; u < u1; u += NW) {
        f32x4 s[4];
#pragma unroll
        for (int t = 0; t < 4; t++) s[t] = scores<HD, MODE>(kr[t], q);
        const float mul = fmaxf(ldexpf(scale, kv8_exp((int8_t)kexp) + q.e), FLT_MIN);  // above 0: -inf stays -inf
        const int ev = kv8_exp((int8_t)vexp);
        if (u + NW < u1) load_k(u + NW);
        if (u * T + T > first_limit) {  // some row does not see all of the unit
            const int p0 = u * T + 16 * g;
#pragma unroll
            for (int t = 0; t < 4; t++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (p0 + 4 * t + i >= limit) s[t][i] = -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) top = fmaxf(top, s[t][i]);
        top = col_max(fmaf(top, mul, (float)ev));
        const float m1 = fmaxf(m, ceilf(top)), bias = (float)ev - m1 + (ROUND ? PSCALE : 0.f);
        float sum = 0.f;
        f16x8 ph[2], pl[2];
        f32x4 w[SAVE ? 4 : 1];
#pragma unroll
        for (int t = 0; t < 4; t++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float p = ex2(fmaf(s[t][i], mul, bias)) * (ROUND ? 1.f : 32768.f);
                if constexpr (SAVE) w[t][i] = p;
                sum += p;
                const _Float16 h = (_Float16)p;
                ph[t / 2][4 * (t & 1) + i] = h;
                if constexpr (!ROUND) pl[t / 2][4 * (t & 1) + i] = (_Float16)(p - (float)h);
            }
        if constexpr (SAVE) {
            // weights without V's exponent, for the mass, and the maximum that they go by; slot
            // 16 g + 4 t + i of a row at 16 (t rows + row) + 4 g + i: each store is contiguous
            const size_t at = ((size_t)kvh * a.save_units + u) * rows;
            const float un = pow2i(-ev);
            if (c < min(R, rows)) {
#pragma unroll
                for (int t = 0; t < 4; t++) *(f32x4 *)(a.save + at * T + 16 * (t * rows + c) + 4 * g) = w[t] * un;
                if (g == 0) a.save_m[at + c] = m1;
            }
        }
        if constexpr (PACK) {
            ph[0] = lower ? pl[0] : ph[0];
            ph[1] = lower ? pl[1] : ph[1];
        }
        if (__any(m1 != m)) {  // a row's maximum rose
            const float alpha = ex2(m - m1);
            l *= alpha;
            lx *= alpha;
#pragma unroll
            for (int d = 0; d < ND; d++) o[d] *= alpha;
            m = m1;
        }
        lx += sum * pow2i(-ev);
        if constexpr (ROUND) {
            const float rounded = sum8(ph[0]) + sum8(ph[1]);
            l += (rounded >= NEAR_SUM ? rounded : sum) * pow2i(-ev);
        }
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const f16x8 w = bytes_h(vr[d][2 * h], vr[d][2 * h + 1]);
                o[d] = mfma(w, ph[h], o[d]);
                if constexpr (MODE == ROWS_F32) o[d] = mfma(w, pl[h], o[d]);
            }
        if (u + NW < u1) load_v(u + NW);
    }
    // the four waves' results in LDS; their weights once per row, then the sum
    lx = col_sum(lx);
    l = ROUND ? col_sum(l) : lx;
    if constexpr (PACK)
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) o[d][i] = half_sum(o[d][i]);
    if constexpr (!F16) __syncthreads();  // every wave has read q
    if (!lower) {
#pragma unroll
        for (int d = 0; d < ND; d++) *(f32x4 *)&so[wave][c][16 * d + 4 * g] = o[d];
        if (g == 0) {
            sm[wave][c] = m;
            sl[wave][c] = l;
            sx[wave][c] = lx;
        }
    }
    __syncthreads();
    const int r = tid / TPR, gr = rt * R + r;  // TPR threads a row from here on
    if (gr >= rows) return;
    float M = NEG, W[NW], L = 0.f, X = 0.f;
#pragma unroll
    for (int w = 0; w < NW; w++) M = fmaxf(M, sm[w][r]);
#pragma unroll
    for (int w = 0; w < NW; w++) {
        W[w] = ex2(sm[w][r] - M);
        L += sl[w][r] * W[w];
        X += sx[w][r] * W[w];
    }
    const size_t id = row_id(a, gr, kvh);
    const bool last = a.splits == 1;
    const float inv = last ? 1.f / L : 1.f;
#pragma unroll
    for (int d = 4 * (tid % TPR); d < HD; d += 4 * TPR) {
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; w++) y += *(const f32x4 *)&so[w][r][d] * W[w];
        y *= inv;
        if (!last) {
            *(f32x4 *)(a.part + (id * a.splits + split) * HD + d) = y;
        } else {
            const int64_t at = row_at(a, gr, kvh, a.out_stride, HD) + d;
            if constexpr (F16)
                *(u32x2 *)((uint16_t *)a.out + at) =
                    u32x2{f2h_top(y[0]) | (uint32_t)f2h_top(y[1]) << 16, f2h_top(y[2]) | (uint32_t)f2h_top(y[3]) << 16};
            else
                *(f32x4 *)((float *)a.out + at) = y;
        }
    }
    if (tid % TPR == 0) {
        a.ml[id * a.splits + split] = make_float4(M, L, X, 0.f);
        if (last && a.norm) a.norm[id] = make_float2(M, 32768.f / X);
    }
}

// Merge of the splits of one (token, query head): the first values of every
// thread are requested together with the (m, l) pairs, one memory round trip for
// up to MS * 8 splits; the weights 2^(m - M) are formed once, in LDS.
constexpr int MW = 512, MPRE = 8;  // threads; splits per thread in the first round trip
constexpr int KV8_MAX_SPLITS = 1024;
template <int HD>
struct MergeLds {
    static constexpr int LPR = HD / 4, MS = MW / LPR;  // lanes of a row, splits at a time
    float wt[KV8_MAX_SPLITS];
    __attribute__((aligned(16))) float red[MS][HD];
    float wmax[MW / WAVE], wsum[MW / WAVE], wsumx[MW / WAVE];
};
template <int HD, bool F16>
__device__ __forceinline__ void merge_row(const Kv8AttnArgs &a, int token, int head, MergeLds<HD> &lds) {
    constexpr int LPR = MergeLds<HD>::LPR, MS = MergeLds<HD>::MS;
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE, S = a.splits;
    const size_t id = (size_t)token * a.n_heads + head;
    const int col = tid % LPR, s0 = tid / LPR;
    const float *pt = a.part + id * S * HD + 4 * col;
    const float4 *ml = a.ml + id * S;
    f32x4 pre[MPRE];
    float4 mine[2];
#pragma unroll
    for (int k = 0; k < 2; k++) mine[k] = tid + k * MW < S ? ml[tid + k * MW] : make_float4(NEG, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < MPRE; k++) {
        const int s = s0 + k * MS;
        pre[k] = s < S ? *(const f32x4 *)(pt + (size_t)s * HD) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float m = wave_max_all(fmaxf(mine[0].x, mine[1].x));
    if (lane == 0) lds.wmax[wave] = m;
    __syncthreads();
    float M = lds.wmax[0];
#pragma unroll
    for (int w = 1; w < MW / WAVE; w++) M = fmaxf(M, lds.wmax[w]);
    float L = 0.f, X = 0.f;
#pragma unroll
    for (int k = 0; k < 2; k++) {
        const float f = ex2(mine[k].x - M);
        if (tid + k * MW < S) lds.wt[tid + k * MW] = f;
        L += mine[k].y * f;
        X += mine[k].z * f;
    }
    L = wave_sum(L);
    X = wave_sum(X);
    if (lane == 0) {
        lds.wsum[wave] = L;
        lds.wsumx[wave] = X;
    }
    __syncthreads();
    L = X = 0.f;
#pragma unroll
    for (int w = 0; w < MW / WAVE; w++) {
        L += lds.wsum[w];
        X += lds.wsumx[w];
    }
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < MPRE; k++)
        if (s0 + k * MS < S) y += pre[k] * lds.wt[s0 + k * MS];
#pragma unroll 4
    for (int s = s0 + MPRE * MS; s < S; s += MS) y += *(const f32x4 *)(pt + (size_t)s * HD) * lds.wt[s];
    *(f32x4 *)&lds.red[s0][4 * col] = y;
    __syncthreads();
    if (tid < HD) {
        float v = 0.f;
#pragma unroll
        for (int k = 0; k < MS; k++) v += lds.red[k][tid];
        v /= L;
        const int64_t at = token * a.out_stride + (int64_t)head * HD + tid;
        if constexpr (F16) ((uint16_t *)a.out)[at] = f2h_top(v);
        else ((float *)a.out)[at] = v;
    }
    if (tid == 0 && a.norm) a.norm[id] = make_float2(M, 32768.f / X);
}
template <int HD, bool F16>
__global__ __launch_bounds__(MW) void kv8_merge_kernel(Kv8AttnArgs a) {
    __shared__ MergeLds<HD> lds;
    merge_row<HD, F16>(a, blockIdx.y, blockIdx.x, lds);
}

// Merge of a few splits of many rows: four dimensions a thread, WG * 4 / HD rows a
// workgroup (a workgroup per row took 30 us for two splits of 16000 rows, this 9;
// for 11 splits of 768 rows it is the other way, 5 us against 8).
constexpr int MERGE_FEW = 16;
template <int HD, bool F16>
__global__ __launch_bounds__(WG) void kv8_merge_many_kernel(Kv8AttnArgs a) {
    constexpr int LPR = HD / 4, RPW = WG / LPR;
    const int h = blockIdx.x * RPW + threadIdx.x / LPR, d = threadIdx.x % LPR * 4, S = a.splits;
    if (h >= a.n_heads) return;
    const size_t id = (size_t)blockIdx.y * a.n_heads + h;
    const float4 *ml = a.ml + id * S;
    const float *pt = a.part + id * S * HD + d;
    float M = NEG, L = 0.f, X = 0.f;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < S; s++) M = fmaxf(M, ml[s].x);
    for (int s = 0; s < S; s++) {
        const float f = ex2(ml[s].x - M);
        L += ml[s].y * f;
        X += ml[s].z * f;
        y += *(const f32x4 *)(pt + (size_t)s * HD) * f;
    }
    y *= 1.f / L;
    const int64_t at = blockIdx.y * a.out_stride + (int64_t)h * HD + d;
    if constexpr (F16)
        *(u32x2 *)((uint16_t *)a.out + at) =
            u32x2{f2h_top(y[0]) | (uint32_t)f2h_top(y[1]) << 16, f2h_top(y[2]) | (uint32_t)f2h_top(y[3]) << 16};
    else
        *(f32x4 *)((float *)a.out + at) = y;
    if (d == 0 && a.norm) a.norm[id] = make_float2(M, 32768.f / X);
}

// ------------------------------------------------------------- prompts --

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// v of the lane 32 away
template <class F>
__device__ __forceinline__ float half_reduce(float v, F f) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// 32 rows of q in the second operand of 32x32x16 products, lane (column c, half
// h): dimensions 16 f + 8 h + 0..7 of row c; an f32 row as two halves of q 2^-e.
template <int HD, bool F16>
struct QRows {
    static constexpr int NF = HD / 16;
    f16x8 hi[NF], lo[F16 ? 1 : NF];
    int e = 0;

    __device__ __forceinline__ void load(const void *q, int64_t at, int h, bool ok, bool neg) {
        if constexpr (F16) {
            const uint32_t sign = neg ? 0x80008000u : 0u;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                u32x4 w = *(const u32x4 *)((const uint16_t *)q + at + 16 * f + 8 * h);
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = ok ? w[i] ^ sign : 0u;
                hi[f] = __builtin_bit_cast(f16x8, w);
            }
        } else {
            const float *p = (const float *)q + at + 8 * h;
            float amax = 0.f;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const f32x4 u = *(const f32x4 *)(p + 16 * f), w = *(const f32x4 *)(p + 16 * f + 4);
#pragma unroll
                for (int i = 0; i < 4; i++) amax = fmaxf(amax, fmaxf(fabsf(u[i]), fabsf(w[i])));
            }
            amax = half_reduce(amax, [](float a, float b) { return fmaxf(a, b); });
            e = ok && amax > 0.f ? (int)(__float_as_uint(amax) >> 23) - 127 - 14 : 0;
#pragma unroll
            for (int f = 0; f < NF; f++) {  // read again: the row is in cache, its registers are not free
                const f32x4 u = *(const f32x4 *)(p + 16 * f), w = *(const f32x4 *)(p + 16 * f + 4);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x = i < 4 ? u[i & 3] : w[i & 3];
                    const float y = ok ? ldexpf(neg ? -x : x, -e) : 0.f;
                    const _Float16 t = (_Float16)y;
                    hi[f][i] = t;
                    lo[f][i] = (_Float16)(y - (float)t);
                }
            }
        }
    }
};

// A unit of 64 slots, K and V as halves in LDS, in 16-byte pieces (8 values).
// Lanes read equal pieces of neighbouring rows, sixteen at a time over the 64
// banks (256 bytes): a K row of 256 or 512 bytes has its piece j at j ^ (r & 15),
// V rows of 128 bytes, two to a round of the banks, at j ^ (r / 2 & 7).  (With r & 7
// for both, 46% of the LDS cycles were conflicts.)  K row r holds the slot with bits 2 and 3 of r
// exchanged: the products then leave a lane the scores of slots 8 h + 0..7 of
// each 16, those whose weights it supplies to the product with V.
template <int HD, int NT, bool F16>
struct Stage {
    static constexpr int N = T * HD / 16 / NT;  // 16-byte pieces of codes per thread
    u32x4 k[N], v[N];
    int8_t e;  // thread 4 w + b: of K (w = 0) or V (w = 1), slots 16 b ..
    float vmax = KV8_EMIN;  // V's threads: the largest exponent so far
    __device__ __forceinline__ void load(const int8_t *kb, const int8_t *vb, const int8_t *ke, const int8_t *ve, int lb,
                                         int u, int tid) {
        if (tid < 8) e = (tid < 4 ? ke : ve)[(u * T + 16 * (tid & 3)) >> lb];
        const u32x4 *kp = (const u32x4 *)(kb + (size_t)u * (T * HD)), *vp = (const u32x4 *)(vb + (size_t)u * (T * HD));
#pragma unroll
        for (int i = 0; i < N; i++) {
            k[i] = kp[tid + i * NT];
            v[i] = vp[tid + i * NT];
        }
    }
    // unit u.  es: K's steps, V's exponents and, for f16 rows, 2^-v of V's exponents or, where one of
    // them is more than NEAR_EXP below the largest so far, 0.  Bytes behind the `end` slots in use count for nothing.
    __device__ __forceinline__ void store(f16x8 *ks, f16x8 *vs, float *es, int u, int end, int tid) {
        if (tid < 8) es[tid] = tid < 4 ? pow2i(kv8_exp(e)) : (float)kv8_exp(e);
        if constexpr (F16)
            if (tid < 8) {
                const int x = kv8_exp(e);
                const bool used = u * T + 16 * (tid & 3) < end;
                float lo = used ? (float)x : (float)KV8_EMAX, hi = used ? (float)x : (float)KV8_EMIN;
                lo = fminf(lo, OI_DPP(lo, 0xB1));
                hi = fmaxf(hi, OI_DPP(hi, 0xB1));
                lo = fminf(lo, OI_DPP(lo, 0x4E));
                vmax = fmaxf(vmax, fmaxf(hi, OI_DPP(hi, 0x4E)));
                if (tid >= 4) es[tid + 4] = lo < vmax - NEAR_EXP ? 0.f : pow2i(-x);
            }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int at = tid + i * NT;
            const int s = at / (HD / 16), j = at % (HD / 16) * 2;
            const int r = (s & ~12) | (s & 4) << 1 | (s & 8) >> 1;
            ks[r * (HD / 8) + (j ^ (r & 15))] = bytes_h(k[i][0], k[i][1]);
            ks[r * (HD / 8) + ((j + 1) ^ (r & 15))] = bytes_h(k[i][2], k[i][3]);
            const int d = at / 4, m = at % 4 * 2;
            vs[d * 8 + (m ^ (d >> 1 & 7))] = bytes_h(v[i][0], v[i][1]);
            vs[d * 8 + ((m + 1) ^ (d >> 1 & 7))] = bytes_h(v[i][2], v[i][3]);
        }
    }
};

// Many rows: a workgroup of NW waves takes 32 NW / DS rows of one kv head, a wave
// 32 of them (all their dimensions, or half of them beside another wave with DS =
// 2, both of which form the scores), and the units one after another, turned into
// halves in LDS once for all its rows (two buffers: the next unit is requested
// before and stored after this one's products).  Scores transposed as above, on
// 32x32x16 products, for half a unit at a time.  f16 rows rescale o only when a
// maximum rises by more than 2^7: their weights then reach 2^15 at most, from 2^8
// (a p keeps its bits down to 2^-22 of the largest and is lost from o below 2^-33,
// 2^17 of which are below the output's rounding; l as stated above.  A unit whose V
// lies far apart forms its exponentials twice: 375 us where every unit does).
// 2047 tokens of 32 heads of 128 over 8 at 8048 slots: 304 us in f16 (776 TFLOP/s;
// 314 with the sums that the mass needs), 477 in f32 (twice the products); 1000 tokens
// of 16 heads of 256 over 2 at 5000 slots: 147 us in f16 (500 TFLOP/s), 317 in f32
// (233).  Vector instructions fill 64% of its cycles (softmax, and the bytes'
// conversion for 256 rows), the matrix units 41%, at the 1.8 GHz that the card
// holds under them.  Measured and not kept: 64 rows a wave (one wave a SIMD, 428);
// the waves of a SIMD half a unit apart with three buffers (311); a raised wave
// priority around the products (f16 the same, f32 600).
template <int HD, bool F16, int NW, int DS, bool NORM>
__global__ __launch_bounds__(NW *WAVE, HD == 128 ? 2 : 1) void kv8_prompt_kernel(Kv8AttnArgs a) {
    constexpr int NF = HD / 16, DT = HD / 32 / DS, R = 32 * NW / DS;
    constexpr bool AHEAD = HD == 128;  // registers left to request operands from LDS ahead of their use
    constexpr float PS = F16 ? 8.f : PSCALE, LAZY = F16 ? 7.f : 0.f;
    __shared__ __attribute__((aligned(16))) f16x8 lds[2][2][T * HD / 8];  // [buffer][K, V]
    __shared__ __attribute__((aligned(16))) float es[2][F16 ? 12 : 8];  // per 16 slots, as Stage::store leaves them
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int c = lane & 31, h = lane >> 5;
    const int kvh = blockIdx.x, rt = gridDim.y - 1 - blockIdx.y, split = blockIdx.z;  // the longest first
    const int rows = a.n * a.group, past = kv8_past(a.past, a.n, a.c.cap);
    const int row0 = rt * R + wave / DS * 32, d0 = wave % DS * DT;  // my rows, my first tile of 32 dimensions
    const int units = (past + row_token(a, min(rt * R + R - 1, rows - 1)) + T) / T;
    const int u0 = (int)((int64_t)split * units / a.splits), u1 = (int)((int64_t)(split + 1) * units / a.splits);
    const int mine = row0 < rows ? past + row_token(a, min(row0 + 31, rows - 1)) + 1 : 0;  // slots my rows see
    const int first_limit = past + row_token(a, row0) + 1;
    const int r = row0 + c, rr = min(r, rows - 1), limit = past + row_token(a, rr) + 1;
    QRows<HD, F16> q;
    q.load(a.q, row_at(a, rr, kvh, a.q_stride, HD), h, r < rows, a.scale < 0.f);
    const int8_t *kb = a.c.kc + (size_t)kvh * a.c.cap * HD, *vb = a.c.vc + (size_t)kvh * a.c.cap * HD;
    const int8_t *ke = a.c.ke + (size_t)kvh * (a.c.cap >> a.c.lb);
    const int8_t *ve = a.c.ve + (size_t)kvh * (a.c.cap >> a.c.lb);
    const float scale = fabsf(a.scale);
    float m = NEG, l = 0.f, lx = 0.f;  // lx: of the weights before their rounding to f16 (f32 rows, and NORM)
    f32x16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) o[d][i] = 0.f;
    Stage<HD, NW * WAVE, F16> st;
    if (u0 < u1) {
        st.load(kb, vb, ke, ve, a.c.lb, u0, tid);
        st.store(lds[0][0], lds[0][1], es[0], u0, past + a.n, tid);
    }
    __syncthreads();
    for (int u = u0; u < u1; u++) {
        const int buf = (u - u0) & 1;
        const f16x8 *kt = lds[buf][0], *vt = lds[buf][1];
        if (u + 1 < u1) st.load(kb, vb, ke, ve, a.c.lb, u + 1, tid);
        if (u * T < mine) {
            const f32x4 kmul = *(const f32x4 *)&es[buf][0] * scale, ev = *(const f32x4 *)&es[buf][4];
            // 2^-v, or 0 in a far unit, whose weights are summed before their rounding
            f32x4 un;
            bool far = false;
            if constexpr (F16) {
                un = *(const f32x4 *)&es[buf][8];
                far = __builtin_amdgcn_readfirstlane(__float_as_int(un[0])) == 0;
            }
            auto k_at = [&](int x, int f) { return kt[(32 * x + c) * (HD / 8) + ((2 * f + h) ^ (c & 15))]; };
            auto v_at = [&](int x, int b, int d) {
                return vt[(32 * (d0 + d) + c) * 8 + ((4 * x + 2 * b + h) ^ (c >> 1 & 7))];
            };
            f16x8 kf[AHEAD ? NF : 1], vf[AHEAD ? DT : 1][2];
            if constexpr (AHEAD)
#pragma unroll
                for (int f = 0; f < NF; f++) kf[f] = k_at(0, f);
            // 32 slots: two groups of 16 with an exponent each
#pragma unroll
            for (int x = 0; x < 2; x++) {
                f32x16 s;
#pragma unroll
                for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
                for (int f = 0; f < NF; f++) {
                    const f16x8 w = AHEAD ? kf[AHEAD ? f : 0] : k_at(x, f);
                    s = mfma32(w, q.hi[f], s);
                    if constexpr (!F16) s = mfma32(w, q.lo[f], s);
                }
                // V of this half is requested before the softmax, K of the next half before V's products
                if constexpr (AHEAD) {
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int b = 0; b < 2; b++) vf[d][b] = v_at(x, b, d);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (u * T + 32 * x + 32 > first_limit) {
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (u * T + 32 * x + 16 * (i / 8) + 8 * h + i % 8 >= limit) s[i] = -INFINITY;
                }
                f16x8 ph[2], pl[2];
                float mul[2], top = -INFINITY;
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    mul[b] = fmaxf(F16 ? kmul[2 * x + b] : ldexpf(kmul[2 * x + b], q.e), FLT_MIN);
                    float t8 = s[8 * b];
#pragma unroll
                    for (int i = 1; i < 8; i++) t8 = fmaxf(t8, s[8 * b + i]);
                    top = fmaxf(top, fmaf(t8, mul[b], ev[2 * x + b]));
                }
                top = half_reduce(top, [](float y, float z) { return fmaxf(y, z); });
                if (__any(top > m + LAZY) || far) {
                    const float m1 = fmaxf(m, ceilf(top)), alpha = ex2(m - m1);
                    m = m1;
                    l *= alpha;
                    lx *= alpha;
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int i = 0; i < 16; i++) o[d][i] *= alpha;
                    if (far)
#pragma unroll
                        for (int b = 0; b < 2; b++) {
                            const float bias = ev[2 * x + b] - m + PS;
                            float sum = 0.f;
#pragma unroll
                            for (int i = 0; i < 8; i++) sum += ex2(fmaf(s[8 * b + i], mul[b], bias));
                            sum *= pow2i(-(int)ev[2 * x + b]);
                            l += sum;
                            lx += sum;
                        }
                }
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const float bias = ev[2 * x + b] - m + (F16 ? PS : 0.f);
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float p = ex2(fmaf(s[8 * b + i], mul[b], bias)) * (F16 ? 1.f : 32768.f);
                        sum += p;
                        const _Float16 t = (_Float16)p;
                        ph[b][i] = t;
                        if constexpr (!F16) pl[b][i] = (_Float16)(p - (float)t);
                    }
                    if constexpr (F16) l = fmaf(sum8(ph[b]), un[2 * x + b], l);
                    if constexpr (!F16 || NORM) lx = fmaf(sum, F16 ? un[2 * x + b] : pow2i(-(int)ev[2 * x + b]), lx);
                }
                if constexpr (AHEAD)
                    if (x == 0) {
#pragma unroll
                        for (int f = 0; f < NF; f++) kf[f] = k_at(1, f);
                    }
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        const f16x8 w = AHEAD ? vf[AHEAD ? d : 0][b] : v_at(x, b, d);
                        o[d] = mfma32(w, ph[b], o[d]);
                        if constexpr (!F16) o[d] = mfma32(w, pl[b], o[d]);
                    }
            }
        }
        if (u + 1 < u1) st.store(lds[buf ^ 1][0], lds[buf ^ 1][1], es[buf ^ 1], u + 1, past + a.n, tid);
        __syncthreads();
    }
    constexpr float UP = F16 ? 128.f : 1.f;  // 2^(PSCALE - PS): results leave at 2^15 as from the other kernel
    lx = half_reduce(lx, [](float x, float y) { return x + y; }) * UP;
    l = F16 ? half_reduce(l, [](float x, float y) { return x + y; }) * UP : lx;
    if (r >= rows) return;
    const size_t id = row_id(a, r, kvh);
    const bool last = a.splits == 1;
    const float inv = last ? UP / l : UP;
    const int64_t to = row_at(a, r, kvh, a.out_stride, HD);
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int dim = 32 * (d0 + d) + 8 * i + 4 * h;
            const f32x4 y = {o[d][4 * i] * inv, o[d][4 * i + 1] * inv, o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv};
            if (!last)
                *(f32x4 *)(a.part + (id * a.splits + split) * HD + dim) = y;
            else if constexpr (F16)
                *(u32x2 *)((uint16_t *)a.out + to + dim) =
                    u32x2{f2h_top(y[0]) | (uint32_t)f2h_top(y[1]) << 16, f2h_top(y[2]) | (uint32_t)f2h_top(y[3]) << 16};
            else
                *(f32x4 *)((float *)a.out + to + dim) = y;
        }
    if (h == 0 && d0 == 0) {
        if (!last) a.ml[id * a.splits + split] = make_float4(m, l, lx, 0.f);
        else if (NORM) a.norm[id] = make_float2(m, 32768.f / lx);
    }
}

// The weight that every slot receives from the call's rows, summed in f32 over
// all of them: scores formed again from K (half of the cache), 2^(t - m) times
// 2^15 / l of the row.  Every sum is in a fixed order.
//
// One tile of rows (decode): the rows kernel has left every weight relative to
// its row's maximum so far, and that maximum (an integer, so what is left to
// multiply is an exact power of two and the row's 2^15 / l).  The workgroups before
// `merges` merge a (token, query head) each; of the others a wave takes unit after
// unit, a slot per lane.  Both read the splits' (m, l) by themselves, so one launch
// does for both.  A slot takes nothing from rows that do not see it, not 0 times their
// 1 / l either (NaN of a row that holds NaN).  At 100004 slots of 4 kv heads 8 us
// (scores formed again from K: 18; reads of 2 KB a unit instead of 8).
constexpr int FEW_MASS_ROWS = 16;
template <int HD, bool F16>
__global__ __launch_bounds__(MW) void kv8_mass_few_kernel(Kv8AttnArgs a, int merges) {
    constexpr int NW = MW / WAVE, R = FEW_MASS_ROWS, AHEAD = 4;
    __shared__ union {
        MergeLds<HD> merge;
        float2 norm[R];
    } lds;
    if ((int)blockIdx.x < merges) {
        const int token = blockIdx.x / a.n_heads;
        merge_row<HD, F16>(a, token, blockIdx.x - token * a.n_heads, lds.merge);
        return;
    }
    const int at = blockIdx.x - merges, kvh = at % a.c.n_kv, nth = at / a.c.n_kv;
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int rows = a.n * a.group, past = kv8_past(a.past, a.n, a.c.cap), end = past + a.n;
    const int units = (end + T - 1) / T, step = (gridDim.x - merges) / a.c.n_kv * NW;
    // the rows' m and 1 / l (the weights' 2^15 is in both): a wave per row over its splits
    for (int r = wave; r < rows; r += NW) {
        const float4 *ml = a.ml + row_id(a, r, kvh) * a.splits;
        float M = NEG, L = 0.f;
        for (int s = lane; s < a.splits; s += WAVE) {
            const float4 x = ml[s];
            const float m1 = fmaxf(M, x.x);
            L = L * ex2(M - m1) + x.z * ex2(x.x - m1);
            M = m1;
        }
        const float all = wave_max_all(M);
        L = wave_sum(L * ex2(M - all));
        if (lane == 0) lds.norm[r] = make_float2(all, 1.f / L);
    }
    __syncthreads();
    const float2 norm = lds.norm[min(lane, rows - 1)];
    float *mass = a.mass + (size_t)kvh * a.c.cap;
    for (int u = nth * NW + wave; u < units; u += step) {
        const size_t from = ((size_t)kvh * a.save_units + u) * rows;
        const int s = u * T + lane;
        const float *w = a.save + from * T + 16 * ((lane >> 2 & 3) * rows) + 4 * (lane >> 4) + (lane & 3);
        const float had = s < past ? mass[s] : 0.f;
        const float f = ex2(a.save_m[from + min(lane, rows - 1)] - norm.x) * norm.y;  // lane r: of row r
        float sum = 0.f;
        for (int r0 = 0; r0 < rows; r0 += AHEAD) {
            float x[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) x[i] = w[min(r0 + i, rows - 1) * 16];
#pragma unroll
            for (int i = 0; i < AHEAD; i++)
                if (r0 + i < rows && row_token(a, r0 + i) >= s - past) sum = fmaf(x[i], lane_value(f, r0 + i), sum);
        }
        if (s < end) mass[s] = had + sum;
    }
}

// Many rows: a workgroup owns 64 X slots, a wave 32 X of them (K in its operand
// registers, converted once) and every other 32 rows of the tiles of 64 rows of q
// that pass through LDS (two buffers).  The sums over rows stay in registers; at
// the end they cross the lanes and meet, two waves a slot, in LDS.  Where slots are
// too few to fill the card, the rows are split over workgroups too, whose sums a
// second launch adds (1000 rows of 16 heads of 2 kv heads at 5000 slots, head_dim
// 256: 168 us in one split, 96 in three).  2047 tokens of 32 heads at 8048 slots:
// 192 us, 613 TFLOP/s; 54% of its cycles are vector instructions (an exponential
// and two multiply-adds a score), 32% the matrix units.
template <int HD, bool F16, int X>
__global__ __launch_bounds__(WG, 2) void kv8_mass_kernel(Kv8AttnArgs a) {
    constexpr int NF = HD / 16, QR = 64, PC = F16 ? 1 : 2, TPR = WG / QR, EL = HD / TPR, WS = 32 * X, GS = 2 * WS;
    __shared__ __attribute__((aligned(16))) f16x8 qs[2][PC][QR * HD / 8];
    __shared__ float qmul[2][QR], sum[2][GS];
    __shared__ float2 qnorm[2][QR];
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int c = lane & 31, h = lane >> 5, kvh = blockIdx.x % a.c.n_kv, blk = blockIdx.x / a.c.n_kv;
    const int s0 = blk * GS + (wave & 1) * WS;
    const int rows = a.n * a.group, past = kv8_past(a.past, a.n, a.c.cap), end = past + a.n;
    if (blk * GS >= end) return;
    // the tile's rows into registers, four threads a row, then as halves into LDS
    const int qr = tid / TPR, qj = tid % TPR;
    u32x4 raw[F16 ? EL / 8 : EL / 4];
    float2 raw_norm = make_float2(0.f, 0.f);
    auto fetch = [&](int t0) {
        const int r = min(t0 + qr, rows - 1);
        const int64_t at = row_at(a, r, kvh, a.q_stride, HD) + qj * EL;
#pragma unroll
        for (int i = 0; i < (F16 ? EL / 8 : EL / 4); i++)
            raw[i] = F16 ? *(const u32x4 *)((const uint16_t *)a.q + at + 8 * i)
                         : *(const u32x4 *)((const float *)a.q + at + 4 * i);
        raw_norm = a.norm[row_id(a, r, kvh)];
    };
    auto store = [&](int b) {
        int e = 0;
        if constexpr (F16) {
#pragma unroll
            for (int i = 0; i < EL / 8; i++)
                qs[b][0][qr * (HD / 8) + ((qj * (EL / 8) + i) ^ (qr & 15))] = __builtin_bit_cast(f16x8, raw[i]);
        } else {
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < EL / 4; i++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float x = __uint_as_float(raw[i][k]);
                    amax = fmaxf(amax, fabsf(x));
                }
            amax = fmaxf(amax, OI_DPP(amax, 0xB1));
            amax = fmaxf(amax, OI_DPP(amax, 0x4E));
            e = amax > 0.f ? (int)(__float_as_uint(amax) >> 23) - 127 - 14 : 0;
#pragma unroll
            for (int i = 0; i < EL / 8; i++) {
                f16x8 hi, lo;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const uint32_t bits = raw[2 * i + k / 4][k & 3];
                    const float y = ldexpf(__uint_as_float(bits), -e);
                    const _Float16 t = (_Float16)y;
                    hi[k] = t;
                    lo[k] = (_Float16)(y - (float)t);
                }
                const int at = qr * (HD / 8) + ((qj * (EL / 8) + i) ^ (qr & 15));
                qs[b][0][at] = hi;
                qs[b][PC - 1][at] = lo;
            }
        }
        if (qj == 0) {
            qmul[b][qr] = ldexpf(a.scale, e);
            qnorm[b][qr] = raw_norm;
        }
    };
    // K: row c of each half unit; its 16-byte loads supply two operands, dimensions 32 m + 16 h + 0..7 and + 8..15
    f16x8 kf[X][NF];
    const int8_t *kb = a.c.kc + (size_t)kvh * a.c.cap * HD;
    const bool have = s0 < a.c.cap;
    const int s_at = have ? s0 : 0;
#pragma unroll
    for (int x = 0; x < X; x++)
#pragma unroll
        for (int m = 0; m < NF / 2; m++) {
            const u32x4 w = *(const u32x4 *)(kb + (size_t)(s_at + 32 * x + c) * HD + 32 * m + 16 * h);
            kf[x][2 * m] = bytes_h(w[0], w[1]);
            kf[x][2 * m + 1] = bytes_h(w[2], w[3]);
        }
    float step[2 * X];
    const int8_t *ke = a.c.ke + (size_t)kvh * (a.c.cap >> a.c.lb);
#pragma unroll
    for (int b = 0; b < 2 * X; b++) step[b] = pow2i(kv8_exp(ke[(s_at + 16 * b) >> a.c.lb]));
    float acc[X][16];
#pragma unroll
    for (int x = 0; x < X; x++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[x][i] = 0.f;
    // from the tile of rows that first sees one of the slots, this split's part of the tiles
    const int first = max(0, blk * GS - past) * a.group / QR, tiles = (rows + QR - 1) / QR - first;
    const int from = (first + (int)((int64_t)blockIdx.y * tiles / gridDim.y)) * QR,
              to = (first + (int)((int64_t)(blockIdx.y + 1) * tiles / gridDim.y)) * QR;
    if (from < to) {
        fetch(from);
        store(0);
    }
    __syncthreads();
    for (int t0 = from, b = 0; t0 < to; t0 += QR, b ^= 1) {
        if (t0 + QR < to) fetch(t0 + QR);
        const int lr = 32 * (wave >> 1) + c, r = t0 + lr;  // my column's row
        const int r_last = min(t0 + 32 * (wave >> 1) + 31, rows - 1);
        if (s0 < past + row_token(a, r_last) + 1 && t0 + 32 * (wave >> 1) < rows) {
            const int limit = r < rows ? past + row_token(a, r) + 1 : 0;
            const float qm = qmul[b][lr];
            const float2 norm = qnorm[b][lr];
            const bool edge = s0 + WS > past + row_token(a, t0 + 32 * (wave >> 1)) + 1 || t0 + QR > rows;
            f32x16 s[X];
#pragma unroll
            for (int x = 0; x < X; x++)
#pragma unroll
                for (int i = 0; i < 16; i++) s[x][i] = 0.f;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const int at = lr * (HD / 8) + ((4 * (f / 2) + 2 * h + (f & 1)) ^ (lr & 15));
                const f16x8 hi = qs[b][0][at], lo = qs[b][PC - 1][at];
#pragma unroll
                for (int x = 0; x < X; x++) {
                    s[x] = mfma32(kf[x][f], hi, s[x]);
                    if constexpr (!F16) s[x] = mfma32(kf[x][f], lo, s[x]);
                }
            }
#pragma unroll
            for (int x = 0; x < X; x++) {
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float p = ex2(fmaf(s[x][i], step[2 * x + i / 8] * qm, -norm.x)) * norm.y;
                        acc[x][i] += s0 + 32 * x + 8 * (i / 4) + 4 * h + i % 4 < limit ? p : 0.f;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        acc[x][i] = fmaf(ex2(fmaf(s[x][i], step[2 * x + i / 8] * qm, -norm.x)), norm.y, acc[x][i]);
                }
            }
        }
        if (t0 + QR < to) store(b ^ 1);
        __syncthreads();
    }
#pragma unroll
    for (int x = 0; x < X; x++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            float v = lane_group_sum(acc[x][i], 16);
            const auto w = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
            v = __uint_as_float(w[0]) + __uint_as_float(w[1]);
            if (c == 0) sum[wave >> 1][(wave & 1) * WS + 32 * x + 8 * (i / 4) + 4 * h + i % 4] = v;
        }
    __syncthreads();
    const int s = blk * GS + tid;
    if (tid < GS && s < end) {
        const float v = sum[0][tid] + sum[1][tid];
        if (gridDim.y > 1) {
            a.msum[((size_t)blockIdx.y * a.c.n_kv + kvh) * a.msum_slots + s] = v;
            return;
        }
        float *m = a.mass + (size_t)kvh * a.c.cap + s;
        *m = s < past ? *m + v : v;
    }
}
// the row splits' sums, in order
__global__ __launch_bounds__(WG) void kv8_mass_sum_kernel(Kv8AttnArgs a, int splits) {
    const int past = kv8_past(a.past, a.n, a.c.cap), s = blockIdx.x * WG + threadIdx.x, kvh = blockIdx.y;
    if (s >= past + a.n) return;
    float v = 0.f;
    for (int y = 0; y < splits; y++) v += a.msum[((size_t)y * a.c.n_kv + kvh) * a.msum_slots + s];
    float *m = a.mass + (size_t)kvh * a.c.cap + s;
    *m = s < past ? *m + v : v;
}

}  // namespace

constexpr int CUS = 256;

// Whether rows go by 16 over many splits (kv8_rows_kernel) or by 128 and 256 with
// units converted once for all of them (kv8_prompt_kernel).  Always the former
// where a tile of rows is all; else up to 512 rows while tiles of 16 rows x units
// stay below a bound, both measured at 24 to 480 rows and 500 to 30000 slots:
//   head_dim 128  f32 20000: 45 us against 49, 37700: 90 / 70
//                 f16  7500: 23 / 26 (24 rows), 3960: 22 / 25 (240), 3020: 20 / 17 (96), 20000: 40 / 33
//   head_dim 256  f32  3840: 43 / 55   f16 1020: 21 / 26, 1510: 27 / 25, 2810: 38 / 24
static int64_t most_by_sixteen(int hd, bool f16) { return hd == 128 ? (f16 ? 8000 : 24000) : (f16 ? 2000 : 5000); }
static bool by_sixteen(int hd, bool f16, int n_kv, int64_t rows, int64_t units) {
    return rows <= 16 || (rows <= 512 && (rows + 15) / 16 * n_kv * units <= most_by_sixteen(hd, f16));
}

// The prompt kernel's workgroups: 8 waves where they fill the card's CUs (a unit is
// converted for 256 rows at a time), 4 waves, two to a CU, otherwise; for head_dim
// 256 the registers of f16 rows allow 8 waves in pairs that share 32 rows and hold
// half of the dimensions each, those of f32 rows 4 waves.
struct PromptPlan {
    int waves, rows, resident;  // of a workgroup; workgroups at a time
};
static PromptPlan prompt_plan(int hd, bool f16, int n_kv, int64_t rows) {
    if (hd == 256) return {f16 ? 8 : 4, 128, CUS};
    if ((rows + 255) / 256 * n_kv >= CUS) return {8, 256, CUS};
    return {4, 128, 2 * CUS};
}

int kv8_attn_splits(int n_kv, int group, int n, int end, int hd, bool f16) {
    const int64_t units = (end + T - 1) / T, rows = (int64_t)n * group;
    if (n > 65535) return 1;  // the merge's grid
    if (by_sixteen(hd, f16, n_kv, rows, units)) {
        // a unit per wave, up to two workgroups a CU (one for head_dim 256, whose registers leave room for one)
        const int64_t tiles = (rows + 15) / 16 * n_kv, room = hd == 128 ? 2 * CUS : CUS, most = (room + tiles - 1) / tiles;
        return (int)std::max<int64_t>(1, std::min((units + 3) / 4, most));
    }
    // The least of rounds * (units of a split + 3 for its beginning and end) + the
    // merge (a launch, and the splits' f32 results out and in), in units of one
    // tile's step (about 2.7 us)
    const PromptPlan p = prompt_plan(hd, f16, n_kv, rows);
    const int64_t tiles = (rows + p.rows - 1) / p.rows * n_kv;
    const double merge = (double)rows * n_kv * hd * 8 / 5e6 / 2.7;
    int best = 1;
    double least = 1e30;
    for (int64_t s = 1; s <= 256 && s <= (units + 1) / 2; s++) {
        const double c = (double)((tiles * s + p.resident - 1) / p.resident) * ((double)units / s + 3) +
                         (s > 1 ? 2 + merge * s : 0);
        if (c < least) {
            least = c;
            best = (int)s;
        }
    }
    return best;
}

bool kv8_attn_saves(int group, int n) { return (int64_t)n * group <= FEW_MASS_ROWS; }

// slots of a workgroup of the mass of many rows: 64 of K a wave, 32 where a row is twice as long
static int mass_slots(int hd) { return hd == 128 ? 128 : 64; }

// Splits of the rows for the mass of many rows: workgroups for two a CU, but a
// dozen tiles of 64 rows each
int kv8_mass_splits(int n_kv, int group, int n, int end, int hd) {
    const int64_t wgs = ((int64_t)end + mass_slots(hd) - 1) / mass_slots(hd) * n_kv, tiles = ((int64_t)n * group + 63) / 64;
    return (int)std::max<int64_t>(1, std::min((2 * CUS + wgs / 2) / wgs, tiles / 12));
}

size_t kv8_attn_workspace(int n_heads, int group, int n, int end, int hd, int splits, bool mass) {
    const size_t rows = (size_t)n * n_heads, units = ((size_t)end + T - 1) / T;
    const size_t saved = mass && kv8_attn_saves(group, n) ? rows * units * T + (rows * units + 3) / 4 * 4 : 0;
    const int n_kv = n_heads / group, ms = mass && !kv8_attn_saves(group, n) ? kv8_mass_splits(n_kv, group, n, end, hd) : 1;
    const size_t sums = ms > 1 ? (size_t)ms * n_kv * end : 0;
    return (saved + rows * ((splits > 1 ? (size_t)splits * hd : 0) + 4 * (size_t)splits + 2) + sums) * 4;
}

// What a call of n tokens may need at any length up to the capacity.  The splits over
// the slots grow with the length in either form (more units to share out), but may
// fall where the form changes; the mass's row splits fall as its slots fill the card,
// in steps, just before which their sums take the most.
size_t kv8_attn_workspace_most(int n_heads, int group, int n, int cap, int hd) {
    const int n_kv = n_heads / group;
    const int64_t rows = (int64_t)n * group, units = cap / T;
    int splits = 1;
    for (const bool f16 : {false, true}) {
        splits = std::max(splits, kv8_attn_splits(n_kv, group, n, cap, hd, f16));
        const int64_t last = std::min(units, most_by_sixteen(hd, f16) / ((rows + 15) / 16 * n_kv));
        if (last > 0) splits = std::max(splits, kv8_attn_splits(n_kv, group, n, (int)(last * T), hd, f16));
    }
    size_t sums = 0;
    if (!kv8_attn_saves(group, n))
        for (int64_t end = mass_slots(hd), e = 0; e < cap; end += mass_slots(hd)) {
            e = std::min<int64_t>(end, cap);
            const int ms = kv8_mass_splits(n_kv, group, n, (int)e, hd);
            if (ms == 1) break;  // and at every greater length
            sums = std::max(sums, (size_t)ms * n_kv * e * 4);
        }
    const size_t all = kv8_attn_workspace(n_heads, group, n, cap, hd, splits, true);
    return std::max(all, kv8_attn_workspace(n_heads, group, n, cap, hd, splits, false) + sums);
}

namespace {

template <int HD, int MODE>
void launch(const Kv8AttnArgs &a, hipStream_t st) {
    constexpr int R = tile_rows(MODE);
    constexpr bool F16 = rows_f16(MODE);
    const int rows = a.n * a.group;
    const int end = a.past.dev ? a.c.cap : a.past.past + a.n, units = (end + T - 1) / T;
    const dim3 merge_grid((unsigned)a.n_heads, (unsigned)a.n);
    if (by_sixteen(HD, F16, a.c.n_kv, rows, units)) {
        const dim3 grid((unsigned)a.c.n_kv, (unsigned)((rows + R - 1) / R), (unsigned)a.splits);
        if (a.save) hipLaunchKernelGGL((kv8_rows_kernel<HD, MODE, true>), grid, dim3(WG), 0, st, a);
        else hipLaunchKernelGGL((kv8_rows_kernel<HD, MODE, false>), grid, dim3(WG), 0, st, a);
    } else if constexpr (!rows_packed(MODE)) {  // (at most 8 rows always go by 16)
        const PromptPlan p = prompt_plan(HD, F16, a.c.n_kv, rows);
        const dim3 grid((unsigned)a.c.n_kv, (unsigned)((rows + p.rows - 1) / p.rows), (unsigned)a.splits);
        auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3((unsigned)(p.waves * WAVE)), 0, st, a); };
        auto by_norm = [&](auto norm) {
            constexpr bool N = decltype(norm)::value;
            if constexpr (HD == 128)
                p.waves == 8 ? go(kv8_prompt_kernel<HD, F16, 8, 1, N>) : go(kv8_prompt_kernel<HD, F16, 4, 1, N>);
            else if constexpr (F16) go(kv8_prompt_kernel<HD, F16, 8, 2, N>);
            else go(kv8_prompt_kernel<HD, F16, 4, 1, N>);
        };
        if (a.norm) by_norm(std::integral_constant<bool, true>{});
        else by_norm(std::integral_constant<bool, false>{});
    }
    if (a.save) {
        const int merges = a.splits > 1 ? a.n * a.n_heads : 0;
        const int wgs = std::max(1, std::min((units + 7) / 8, 2 * CUS / a.c.n_kv)) * a.c.n_kv;
        hipLaunchKernelGGL((kv8_mass_few_kernel<HD, F16>), dim3((unsigned)(merges + wgs)), dim3(MW), 0, st, a, merges);
        return;
    }
    if (a.splits > 1 && a.splits <= MERGE_FEW && a.n * a.n_heads >= (a.splits <= 4 ? 512 : 4096)) {
        constexpr int RPW = WG * 4 / HD;
        hipLaunchKernelGGL((kv8_merge_many_kernel<HD, F16>),
                           dim3((unsigned)((a.n_heads + RPW - 1) / RPW), (unsigned)a.n), dim3(WG), 0, st, a);
    } else if (a.splits > 1) {
        hipLaunchKernelGGL((kv8_merge_kernel<HD, F16>), merge_grid, dim3(MW), 0, st, a);
    }
    if (!a.mass) return;
    if constexpr (!rows_packed(MODE)) {
        constexpr int X = HD == 128 ? 2 : 1;
        hipLaunchKernelGGL((kv8_mass_kernel<HD, F16, X>),
                           dim3((unsigned)a.c.n_kv * ((end + 64 * X - 1) / (64 * X)), (unsigned)a.msplits), dim3(WG), 0, st,
                           a);
        if (a.msplits > 1)
            hipLaunchKernelGGL(kv8_mass_sum_kernel, dim3((unsigned)((end + WG - 1) / WG), (unsigned)a.c.n_kv), dim3(WG), 0,
                               st, a, a.msplits);
    }
}

}  // namespace

hipError_t launch_kv8_attn(const Kv8AttnArgs &a, hipStream_t st) {
    const bool pack = a.n * a.group <= 8;
    const int mode = a.f16 ? (pack ? ROWS_F16_PACK : ROWS_F16) : pack ? ROWS_PACK : ROWS_F32;
    auto by_mode = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (mode == ROWS_F16) launch<HD, ROWS_F16>(a, st);
        else if (mode == ROWS_F16_PACK) launch<HD, ROWS_F16_PACK>(a, st);
        else if (mode == ROWS_PACK) launch<HD, ROWS_PACK>(a, st);
        else launch<HD, ROWS_F32>(a, st);
    };
    if (a.c.hd == 128) by_mode(std::integral_constant<int, 128>{});
    else if (a.c.hd == 256) by_mode(std::integral_constant<int, 256>{});
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace oi
