// paged_attn.hip -- attention over the paged f16 cache: the newest tokens of many
// sequences, and packed prompts.
//
// Token j of a sequence's n sees slots 0 .. len - n + j.  Scores in base 2:
//   t_s = (q . K_s) scale log2(e),  p_s = 2^(t_s - m + 15),  m the running maximum
//   o = sum p_s V_s,   l = sum p_s,   out = o / l  (0 where a row sees nothing)
// m, l and o are 32-bit.  The matrix products take f16 operands: K and V are exact
// there; an f32 q is the sum of two halves (22 bits, scaled by a power of two per
// row), an f16 q exact.  Weights are the sum of two halves (22 bits) but for f16
// prompts, whose outputs hold no more than 11 bits: there p is rounded once and l is
// the sum of the rounded weights.  2^15 is where the row's largest p sits in f16:
// another keeps all its bits down to 2^-29 of it and is lost below 2^-40 (f16 prompts:
// 2^-22 and 2^-33).  Cached values are finite (the append sees to it): a slot that a
// row does not see has weight 0, and slots past a sequence's end count as zeros.
//
// Work is shared out on the device, since the lengths are there: every tile of rows
// of every kv head and sequence has a cost (its units of slots, and something for
// itself), the tiles lie one behind the other, and each workgroup (worker) takes an
// equal stretch of their sum.  A tile that a border falls into leaves partial results
// of both sides (a worker has at most two such, its first and its last) that a second
// launch joins.  A border near a tile's end moves there.  So one long sequence among
// short ones keeps the whole card busy, and the grid and the workspace do not depend on
// lengths: a captured call serves all of them.

#include <cfloat>

#include "device_common.h"
#include "paged.h"

namespace oi {

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef const __attribute__((address_space(4))) int32_t *ScalarInts;  // read through the scalar cache

constexpr float NEG = -3.402823466e38f;  // the running maximum before any slot
constexpr int TU = 32;                   // slots of a unit of the tokens kernel
constexpr int PU = 64;                   // of the prompts kernel

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ int seq_len(const PagedAttnArgs &a, int s) {
    return (int)min((int64_t)max(a.lens[s], 0), (int64_t)a.stride << a.c.lp);
}
// The token of row r of a sequence and kv head (token-major): r / group by a
// multiplication (exact while r * group < 2^32)
__device__ __forceinline__ int row_token(const PagedAttnArgs &a, int r) {
    return a.magic ? (int)__umulhi((uint32_t)r, a.magic) : r;
}
// where row r's head lies in q or out; base: the sequence's first token
__device__ __forceinline__ int64_t row_at(const PagedAttnArgs &a, int base, int r, int head, int64_t stride) {
    const int t = row_token(a, r);
    return (int64_t)(base + t) * stride + (int64_t)(head * a.group + r - t * a.group) * a.c.hd;
}
// a table's entry as a page that the pool has
__device__ __forceinline__ int page_ok(const PagedAttnArgs &a, int id) {
    return (int)min((uint32_t)id, (uint32_t)a.c.n_pages - 1u);
}

// ------------------------------------------------------------- sharing out --

// x / y of numbers below 2^53 (y > 0)
__device__ __forceinline__ int64_t quot(int64_t x, int64_t y) {
    int64_t q = (int64_t)((double)x / (double)y);
    if (q * y > x) q--;
    else if ((q + 1) * y <= x) q++;
    return q;
}

// The tiles of a sequence and their costs.  Tokens: `tiles` alike.  Prompts: a tile
// of R rows more sees R / group slots more, and costs are slots times the group.
struct SeqWork {
    int len, tokens, tiles;
    int64_t first, step;  // a tile's cost: first + t * step
    __device__ __forceinline__ int64_t upto(int64_t t) const { return t * first + step * (t * (t - 1) / 2); }
};
struct TokensWork {
    static constexpr int OWN = 1, LEAST = 4, PARTS = 256;  // a tile's own cost, a worker's least, a tile's most parts
    __device__ static __forceinline__ SeqWork of(const PagedAttnArgs &a, int s) {
        SeqWork w;
        w.len = seq_len(a, s);
        w.tokens = a.n_q;
        w.tiles = (a.n_q * a.group + 15) / 16;
        w.first = (w.len + TU - 1) / TU + OWN;
        w.step = 0;
        return w;
    }
    __device__ static __forceinline__ int64_t unit(const PagedAttnArgs &) { return 1; }
    __device__ static __forceinline__ int units(const PagedAttnArgs &, const SeqWork &w, int) {
        return (w.len + TU - 1) / TU;
    }
};
template <int R>
struct PromptsWork {
    static constexpr int OWN = 1, LEAST = 4, PARTS = 128;
    __device__ static __forceinline__ SeqWork of(const PagedAttnArgs &a, int s) {
        SeqWork w;
        const int r0 = min(max(a.starts[s], 0), a.n_rows), r1 = min(max(a.starts[s + 1], r0), a.n_rows);
        w.len = seq_len(a, s);
        w.tokens = r1 - r0;
        w.tiles = (int)(((int64_t)w.tokens * a.group + R - 1) / R);
        w.first = (int64_t)a.group * (max(w.len - w.tokens, 0) + OWN * PU) + R;
        w.step = R;
        return w;
    }
    __device__ static __forceinline__ int64_t unit(const PagedAttnArgs &a) { return (int64_t)a.group * PU; }
    __device__ static __forceinline__ int units(const PagedAttnArgs &a, const SeqWork &w, int tile) {
        const int last = row_token(a, min(tile * R + R, w.tokens * a.group) - 1);
        return (max(w.len - w.tokens + last + 1, 0) + PU - 1) / PU;
    }
};

// The border at x of the whole cost: sequence s holds it, x less the sequences before.
template <class W>
__device__ PagedAt border(const PagedAttnArgs &a, int s, int64_t x, int64_t share) {
    const SeqWork w = W::of(a, s);
    const int64_t one = w.upto(w.tiles), u1 = W::unit(a);
    int head = (int)quot(x, one);
    x -= head * one;
    // the last tile with upto(t) <= x
    int64_t t;
    if (w.step == 0) {
        t = quot(x, w.first);
    } else {
        const double b = (double)w.first - 0.5 * w.step;
        t = (int64_t)((sqrt(b * b + 2.0 * w.step * x) - b) / w.step);
        t = min(max(t, (int64_t)0), (int64_t)w.tiles - 1);
        while (t > 0 && w.upto(t) > x) t--;
        while (t + 1 < w.tiles && w.upto(t + 1) <= x) t++;
    }
    const int64_t in = x - w.upto(t), cost = w.first + t * w.step, own = W::OWN * u1;
    const int units = W::units(a, w, (int)t);
    int u = in <= own ? 0 : (int)quot((in - own) * units, cost - own);
    const int near = (int)quot(share, 8 * u1);
    int tile = (int)t;
    if (u <= near) {
        u = 0;
    } else if (units - u <= near) {
        u = 0;
        if (++tile == w.tiles) {
            tile = 0;
            if (++head == a.c.n_kv) {
                head = 0;
                s++;
            }
        }
    }
    return {s, head, tile, u};
}

struct ShareLds {
    int64_t sum[WG / WAVE];
    int64_t most[WG / WAVE];
    PagedAt at[2];
};
// Worker's stretch, [at[0], at[1]); the number of workers used is returned.  All WG
// threads take part; each sums a run of neighbouring sequences.  `spread`: neighbouring
// workers go to one XCD (blocks are dealt to the 8 in turn), whose cache then holds
// what they share.
template <class W, bool SPREAD>
__device__ int share_out(const PagedAttnArgs &a, ShareLds &lds, int &worker) {
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int per = (a.n_seqs + WG - 1) / WG, s0 = min(tid * per, a.n_seqs), s1 = min(s0 + per, a.n_seqs);
    int64_t sum = 0, most = 0;
    for (int s = s0; s < s1; s++) {
        const SeqWork w = W::of(a, s);
        sum += w.upto(w.tiles) * a.c.n_kv;
        if (w.tiles) most = max(most, w.first + (w.tiles - 1) * w.step);
    }
    int64_t run = sum;
#pragma unroll
    for (int d = 1; d < WAVE; d *= 2) {
        const int64_t o = __shfl_up(run, d);
        if (lane >= d) run += o;
        most = max(most, (int64_t)__shfl_xor(most, d));
    }
    if (lane == WAVE - 1) {
        lds.sum[wave] = run;
        lds.most[wave] = most;
    }
    if (tid < 2) lds.at[tid] = {a.n_seqs, 0, 0, 0};
    __syncthreads();
    int64_t before = 0, total = 0;
    most = 0;
#pragma unroll
    for (int w = 0; w < WG / WAVE; w++) {
        const int64_t x = lds.sum[w];
        before += w < wave ? x : 0;
        total += x;
        most = max(most, lds.most[w]);
    }
    run += before - sum;  // the sequences before this thread's
    int64_t share = quot(total + a.workers - 1, a.workers);
    share = max(share, max(W::LEAST * W::unit(a), quot(most + W::PARTS - 1, (int64_t)W::PARTS)));
    const int used = (int)quot(total + share - 1, share);
    const int each = (used + 7) / 8, b = blockIdx.x;
    worker = SPREAD ? (b / 8 < each ? (b & 7) * each + b / 8 : used) : b;
    if (worker < used) {
#pragma unroll
        for (int k = 0; k < 2; k++) {
            int64_t x = (worker + k) * share;
            if (x < run || x >= run + sum) continue;  // past the end of all: as set
            x -= run;
            for (int s = s0; s < s1; s++) {
                const SeqWork w = W::of(a, s);
                const int64_t c = w.upto(w.tiles) * a.c.n_kv;
                if (x < c) {
                    lds.at[k] = border<W>(a, s, x, share);
                    break;
                }
                x -= c;
            }
        }
    }
    __syncthreads();
    return used;
}
// the same in every lane, in scalar registers
__device__ __forceinline__ PagedAt uniform(const PagedAt &x) {
    return {__builtin_amdgcn_readfirstlane(x.seq), __builtin_amdgcn_readfirstlane(x.head),
            __builtin_amdgcn_readfirstlane(x.tile), __builtin_amdgcn_readfirstlane(x.u)};
}
__device__ __forceinline__ bool same_tile(const PagedAt &x, const PagedAt &y) {
    return x.seq == y.seq && x.head == y.head && x.tile == y.tile;
}

// What a worker leaves for the join beside its results: where it begins and, where both
// borders of its stretch fall on one unit inside a tile, that its part is empty.
__device__ __forceinline__ void leave_border(const PagedAttnArgs &a, int worker, const PagedAt &begin, const PagedAt &end) {
    if (threadIdx.x == 0) a.at[worker] = begin;
    if (begin.u > 0 && same_tile(begin, end) && begin.u == end.u)
        for (int r = threadIdx.x; r < a.part_rows; r += WG) a.ml[(size_t)worker * 2 * a.part_rows + r] = make_float2(NEG, 0.f);
}

// Calls f(w, at, units, u0, u1) for each piece of the stretch (at.u unused).
template <class W, class F>
__device__ __forceinline__ void each_piece(const PagedAttnArgs &a, PagedAt at, const PagedAt end, F f) {
    while (at.seq < end.seq || (at.seq == end.seq && (at.head < end.head || (at.head == end.head &&
                               (at.tile < end.tile || (at.tile == end.tile && at.u < end.u)))))) {
        const SeqWork w = W::of(a, at.seq);
        if (w.tiles) {
            const int units = W::units(a, w, at.tile);
            f(w, at, units, at.u, same_tile(at, end) ? end.u : units);
        }
        at.u = 0;
        if (++at.tile >= w.tiles) {
            at.tile = 0;
            if (!w.tiles || ++at.head == a.c.n_kv) {
                at.head = 0;
                at.seq++;
            }
        }
    }
}

// --------------------------------------------------------------- operands --

__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// v of the lane 32 away
template <class F>
__device__ __forceinline__ float half_reduce(float v, F f) {
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// of the lanes 16 and 32 away
template <class F>
__device__ __forceinline__ float col_reduce(float v, F f) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return half_reduce(f(__uint_as_float(a[0]), __uint_as_float(a[1])), f);
}
struct Max {
    __device__ __forceinline__ float operator()(float x, float y) const { return fmaxf(x, y); }
};
struct Add {
    __device__ __forceinline__ float operator()(float x, float y) const { return x + y; }
};

// Rows of q as the second operand of a product: the lane's NF pieces of 8 dimensions
// of its row, PART apart.  An f32 row is two halves of q 2^-e, e the row's exponent,
// over the lanes that hold it (reduce).  A negative scale turns q's sign, so that the
// largest score is that of the largest product.
template <int NF, int PART, bool F16>
struct QPieces {
    f16x8 hi[NF], lo[F16 ? 1 : NF];
    int e = 0;
    template <class R>
    __device__ __forceinline__ void load(const void *q, int64_t at, bool ok, bool neg, R reduce) {
        if constexpr (F16) {
            const uint32_t sign = neg ? 0x80008000u : 0u;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                u32x4 w = *(const u32x4 *)((const uint16_t *)q + at + PART * f);
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = ok ? w[i] ^ sign : 0u;
                hi[f] = __builtin_bit_cast(f16x8, w);
            }
        } else {
            const float *p = (const float *)q + at;
            float amax = 0.f;
#pragma unroll
            for (int f = 0; f < NF; f++) {
                const f32x4 u = *(const f32x4 *)(p + PART * f), w = *(const f32x4 *)(p + PART * f + 4);
#pragma unroll
                for (int i = 0; i < 4; i++) amax = fmaxf(amax, fmaxf(fabsf(u[i]), fabsf(w[i])));
            }
            amax = reduce(amax);
            e = ok && amax > 0.f ? (int)(__float_as_uint(amax) >> 23) - 127 - 14 : 0;
#pragma unroll
            for (int f = 0; f < NF; f++) {  // read again: the row is in cache, its registers are not free
                const f32x4 u = *(const f32x4 *)(p + PART * f), w = *(const f32x4 *)(p + PART * f + 4);
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

__device__ __forceinline__ void store_out(void *out, bool f16, int64_t at, f32x4 y) {
    if (f16) {
        *(u32x2 *)((uint16_t *)out + at) =
            u32x2{f2h(y[0]) | (uint32_t)f2h(y[1]) << 16, f2h(y[2]) | (uint32_t)f2h(y[3]) << 16};
    } else {
        *(f32x4 *)((float *)out + at) = y;
    }
}
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }

// ----------------------------------------------------------------- tokens --

// A worker's four waves take units of 32 slots in turn for 16 rows (the (token, query
// head) pairs of a kv head).  Scores are formed transposed, K the first operand; with
// K's rows taken in the order
//   operand row 4 g' + i of tile t  <-  slot 8 g' + 4 t + i
// a lane (column c, group g) holds its row's scores of slots 8 g .. 8 g + 7, those
// whose weights it supplies to the product with V: nothing crosses lanes but the row
// maximum.  V lies in eights of slots, so both go from memory to the operand registers
// 16 bytes a lane without LDS; K of the next unit is requested when this one's scores
// are done, V when its product is, pages one unit ahead of both.  The maximum is raised
// to whole numbers, so rescaling is exact.
template <int HD, bool F16>
__global__ __launch_bounds__(WG) void paged_tokens_kernel(PagedAttnArgs a) {
    constexpr int NW = WG / WAVE, NK = HD / 32, ND = HD / 16, PD = HD + 4, R = 16, TPR = WG / R;
    __shared__ __attribute__((aligned(16))) float so[NW][R][PD];
    __shared__ float sm[NW][R], sl[NW][R];
    __shared__ ShareLds share;
    int worker;
    const int used = share_out<TokensWork, false>(a, share, worker);
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    if (blockIdx.x == 0 && tid == 0) a.at[a.workers] = {used, 0, 0, 0};
    if (worker >= used) return;
    const PagedAt begin = uniform(share.at[0]), end = uniform(share.at[1]);
    leave_border(a, worker, begin, end);
    const int c = lane & 15, g = lane >> 4, lp = a.c.lp, P = 1 << lp;
    const bool neg = a.scale < 0.f;
    const float scale = fabsf(a.scale);
    const int kslot = 8 * (c >> 2) + (c & 3);  // of tile 0; 4 more in tile 1
    const size_t page_elems = ((size_t)a.c.n_kv << lp) * HD;

    each_piece<TokensWork>(a, begin, end, [&](const SeqWork &w, const PagedAt &at, int units, int u0, int u1) {
        const int rows = a.n_q * a.group, rt = at.tile, len = w.len;
        const int row = rt * R + c, rr = min(row, rows - 1);
        const int limit = len - a.n_q + row_token(a, rr) + 1;  // slots that this row sees
        const int first_limit = len - a.n_q + row_token(a, rt * R) + 1;
        const int32_t *table = a.table + (int64_t)at.seq * a.stride;
        const uint16_t *kb = a.c.k + ((size_t)at.head << lp) * HD + 8 * g;
        const uint16_t *vb = a.c.v + ((size_t)at.head << lp) * HD + 8 * c;
        const int last_page = max(len - 1, 0) >> lp;
        u32x4 kr[2][NK], vr[ND];
        int kp = 0, vp = 0, kn = 0, vn = 0;  // pages of the unit at hand and of the next
        auto pages = [&](int u, int &k, int &v) {
            k = table[min((u * TU + (kslot & ~7)) >> lp, last_page)];
            v = table[min((u * TU + 8 * g) >> lp, last_page)];
        };
        auto load_k = [&](int u) {
            const uint16_t *p = kb + page_ok(a, kp) * page_elems + (size_t)((u * TU + kslot) & (P - 1)) * HD;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int f = 0; f < NK; f++) kr[t][f] = *(const u32x4 *)(p + 4 * t * HD + 32 * f);
        };
        auto load_v = [&](int u, int page) {
            const uint16_t *p = vb + page_ok(a, page) * page_elems + (size_t)((u * TU + 8 * g) & (P - 1)) * HD;
#pragma unroll
            for (int d = 0; d < ND; d++) vr[d] = *(const u32x4 *)(p + 16 * d * 8);
        };
        float m = NEG, l = 0.f;
        f32x4 o[ND];
#pragma unroll
        for (int d = 0; d < ND; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
        int u = u0 + wave;
        if (u < u1) {
            pages(u, kp, vp);
            if (u + NW < u1) pages(u + NW, kn, vn);
        }
        QPieces<NK, 32, F16> q;
        q.load(a.q, row_at(a, at.seq * a.n_q, rr, at.head, a.q_stride) + 8 * g, row < rows, neg,
               [](float x) { return col_reduce(x, Max()); });
        if (u < u1) {
            load_k(u);
            load_v(u, vp);
        }
        const float mul = fmaxf(ldexpf(scale, q.e), FLT_MIN);  // above 0: -inf stays -inf
        for (; u < u1; u += NW) {
            f32x4 s[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                s[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int f = 0; f < NK; f++) {
                    const f16x8 k = __builtin_bit_cast(f16x8, kr[t][f]);
                    s[t] = mfma(k, q.hi[f], s[t]);
                    if constexpr (!F16) s[t] = mfma(k, q.lo[f], s[t]);
                }
            }
            kp = kn;
            if (u + NW < u1) load_k(u + NW);
            const int p0 = u * TU + 8 * g;  // the slot of s[0][0]
            if (u * TU + TU > first_limit) {  // some row does not see all of the unit
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (p0 + 4 * t + i >= limit) s[t][i] = -INFINITY;
            }
            float top = s[0][0];
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, s[t][i]);
            top = col_reduce(top * mul, Max());
            const float m1 = fmaxf(m, ceilf(top));
            f16x8 ph, pl;
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float p = ex2(fmaf(s[t][i], mul, -m1)) * 32768.f;
                    sum += p;
                    const _Float16 h = (_Float16)p;
                    ph[4 * t + i] = h;
                    pl[4 * t + i] = (_Float16)(p - (float)h);
                }
            if (__any(m1 != m)) {  // a row's maximum rose
                const float alpha = ex2(m - m1);
                l *= alpha;
#pragma unroll
                for (int d = 0; d < ND; d++) o[d] *= alpha;
                m = m1;
            }
            l += sum;
            if (u * TU + TU > len) {  // bytes behind the sequence's end count for nothing
                u32x4 keep;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    keep[i] = (p0 + 2 * i < len ? 0xFFFFu : 0u) | (p0 + 2 * i + 1 < len ? 0xFFFF0000u : 0u);
#pragma unroll
                for (int d = 0; d < ND; d++) vr[d] &= keep;
            }
#pragma unroll
            for (int d = 0; d < ND; d++) {
                const f16x8 v = __builtin_bit_cast(f16x8, vr[d]);
                o[d] = mfma(v, ph, o[d]);
                o[d] = mfma(v, pl, o[d]);
            }
            if (u + NW < u1) {
                load_v(u + NW, vn);
                if (u + 2 * NW < u1) pages(u + 2 * NW, kn, vn);
            }
        }
        // the four waves' results meet in LDS
        l = col_reduce(l, Add());
#pragma unroll
        for (int d = 0; d < ND; d++) *(f32x4 *)&so[wave][c][16 * d + 4 * g] = o[d];
        if (g == 0) {
            sm[wave][c] = m;
            sl[wave][c] = l;
        }
        __syncthreads();
        const int r = tid / TPR, gr = rt * R + r;  // TPR threads a row from here on
        if (gr < rows) {
            float M = NEG, wt[NW], L = 0.f;
#pragma unroll
            for (int k = 0; k < NW; k++) M = fmaxf(M, sm[k][r]);
#pragma unroll
            for (int k = 0; k < NW; k++) {
                wt[k] = ex2(sm[k][r] - M);
                L += sl[k][r] * wt[k];
            }
            const bool whole = u0 == 0 && u1 == units;
            const size_t slot = ((size_t)worker * 2 + (u0 == 0)) * a.part_rows + r;
            const float inv = whole ? inverse(L) : 1.f;
            const int64_t to = row_at(a, at.seq * a.n_q, gr, at.head, a.out_stride);
#pragma unroll
            for (int d = 4 * (tid % TPR); d < HD; d += 4 * TPR) {
                f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < NW; k++) y += *(const f32x4 *)&so[k][r][d] * wt[k];
                y *= inv;
                if (whole) store_out(a.out, F16, to + d, y);
                else *(f32x4 *)(a.part + slot * HD + d) = y;
            }
            if (!whole && tid % TPR == 0) a.ml[slot] = make_float2(M, L);
        }
        __syncthreads();  // LDS is read before the next piece is written there
    });
}

// ------------------------------------------------------------------- join --

// The parts of a tile that the border behind worker w cuts first: part 1 of w, then
// part 0 of the workers after it while they begin inside the tile.  A workgroup takes
// `JR` of its rows.
constexpr int JR = 8;
template <class W, int HD, int R>
__global__ __launch_bounds__(WG) void paged_join_kernel(PagedAttnArgs a) {
    constexpr int LPR = HD / 4, MS = WG / LPR;  // lanes of a row, parts at a time
    __shared__ int parts;
    __shared__ __attribute__((aligned(16))) float red[MS][HD];
    __shared__ float redl[MS], redm[MS];
    const int w = blockIdx.x, tid = threadIdx.x, used = a.at[a.workers].seq;
    if (w + 1 >= used) return;
    const PagedAt at = a.at[w + 1], prev = a.at[w];
    if (at.u == 0 || (same_tile(at, prev) && prev.u > 0)) return;
    const SeqWork sw = W::of(a, at.seq);
    const int rows = min(sw.tokens * a.group - at.tile * R, R), r0 = blockIdx.y * JR;
    if (r0 >= rows) return;
    if (tid == 0) parts = 1;
    __syncthreads();
    int n = 0;
    for (int k = w + 1 + tid; k < used; k += WG) {
        const PagedAt x = a.at[k];
        if (!same_tile(x, at) || x.u == 0) break;
        n++;
    }
    if (n) atomicAdd(&parts, n);
    __syncthreads();
    n = parts;
    const int base = a.starts ? min(max(a.starts[at.seq], 0), a.n_rows) : at.seq * a.n_q;
    const int col = tid % LPR, k0 = tid / LPR;
    for (int r = r0; r < min(r0 + JR, rows); r++) {
        float M = NEG, L = 0.f;
        f32x4 y = {0.f, 0.f, 0.f, 0.f};
        for (int k = k0; k < n; k += MS) {
            const size_t slot = ((size_t)(w + k) * 2 + (k == 0)) * a.part_rows + r;
            const float2 ml = a.ml[slot];
            f32x4 p = *(const f32x4 *)(a.part + slot * HD + 4 * col);
            if (ml.y == 0.f) p = f32x4{0.f, 0.f, 0.f, 0.f};  // saw nothing, or an empty part that nobody wrote
            const float m1 = fmaxf(M, ml.x), f0 = ex2(M - m1), f1 = ex2(ml.x - m1);
            L = L * f0 + ml.y * f1;
            y = y * f0 + p * f1;
            M = m1;
        }
        *(f32x4 *)&red[k0][4 * col] = y;
        if (col == 0) {
            redl[k0] = L;
            redm[k0] = M;
        }
        __syncthreads();
        if (tid < LPR) {
            M = NEG;
#pragma unroll
            for (int k = 0; k < MS; k++) M = fmaxf(M, redm[k]);
            L = 0.f;
            y = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < MS; k++) {
                const float f = ex2(redm[k] - M);
                L += redl[k] * f;
                y += *(const f32x4 *)&red[k][4 * col] * f;
            }
            store_out(a.out, a.f16, row_at(a, base, at.tile * R + r, at.head, a.out_stride) + 4 * col, y * inverse(L));
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- prompts --

__device__ __forceinline__ float sum8(f16x8 p, float to) {
    const f16x2 one = {(_Float16)1.f, (_Float16)1.f};
#pragma unroll
    for (int i = 0; i < 4; i++) to = __builtin_amdgcn_fdot2(f16x2{p[2 * i], p[2 * i + 1]}, one, to, false);
    return to;
}

template <int HD, bool F16>
struct PromptShape {
    static constexpr int NW = 4, R = 32 * NW;  // waves, rows
    static constexpr int SLOTS = HD == 128 ? 64 : 32;  // of a staged step
    static constexpr int PER_CU = HD == 256 && !F16 ? 1 : 2;
};

// A worker of NW waves takes tiles of 32 NW rows of one kv head, a wave 32 of them,
// and the tile's slots step after step through two buffers in LDS, filled straight from
// memory while the other is worked on.  Scores transposed, on 32x32x16 products.  K's
// piece j (8 dimensions) of LDS row r lies at j ^ (r & 15), and row r holds the slot with
// bits 2 and 3 of r exchanged: the products then leave a lane the scores of slots 8 h +
// 0..7 of each 16, those whose weights it supplies to the product with V; V's pieces (8
// slots of a dimension) lie as in the cache.  Either way sixteen lanes read all banks
// once.  f16 rows rescale o only when a maximum rises by more than 2^7: their weights
// then reach 2^15 at most, from 2^8.
template <int HD, bool F16>
__global__ __launch_bounds__(WG, (PromptShape<HD, F16>::PER_CU)) void paged_prompts_kernel(PagedAttnArgs a) {
    using S = PromptShape<HD, F16>;
    constexpr int NF = HD / 16, DT = HD / 32, R = S::R, ST = S::SLOTS, X = ST / 32;
    constexpr int PIECES = ST * HD / 8;           // of K, and of V, in a step
    constexpr int CH = PIECES / WAVE / S::NW;     // a wave's stretches of 64 pieces, of each
    constexpr int RPC = WAVE / (HD / 8);          // K rows of a stretch
    constexpr float PS = F16 ? 8.f : 15.f, LAZY = F16 ? 7.f : 0.f;
    using W = PromptsWork<R>;
    static_assert(S::NW * WAVE == WG, "the sharing out takes WG threads");
    __shared__ __attribute__((aligned(16))) f16x8 lds[2][2][PIECES];  // [buffer][K, V]
    __shared__ ShareLds share;
    int worker;
    const int used = share_out<W, true>(a, share, worker);
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    if (blockIdx.x == 0 && tid == 0) a.at[a.workers] = {used, 0, 0, 0};
    if (worker >= used) return;
    const PagedAt begin = uniform(share.at[0]), end = uniform(share.at[1]);
    leave_border(a, worker, begin, end);
    const int c = lane & 31, h = lane >> 5, lp = a.c.lp, P = 1 << lp;
    const float scale = fabsf(a.scale);
    const size_t page_elems = ((size_t)a.c.n_kv << lp) * HD;
    // a lane's place in the sources of its stretches: stretch i of a wave is number i NW + wave
    uint32_t ksrc[CH];
#pragma unroll
    for (int i = 0; i < CH; i++) {
        const int r = ((i * S::NW + wave) * RPC + lane / (HD / 8)) & 15, j = lane % (HD / 8);
        const int s16 = (r & 3) | (r & 4) << 1 | (r & 8) >> 1;
        ksrc[i] = (uint32_t)(s16 * HD + 8 * (j ^ r)) * 2;
    }

    each_piece<W>(a, begin, end, [&](const SeqWork &w, const PagedAt &at, int units, int u0, int u1) {
        const int rows = w.tokens * a.group, past = w.len - w.tokens;
        const int base = min(max(a.starts[at.seq], 0), a.n_rows);
        const int row0 = at.tile * R + wave * 32;  // my rows
        const int r = row0 + c, rr = min(r, rows - 1), limit = past + row_token(a, rr) + 1;
        const int mine = row0 < rows ? past + row_token(a, min(row0 + 31, rows - 1)) + 1 : 0;  // slots my rows see
        const int first_limit = past + row_token(a, min(row0, rows - 1)) + 1;
        const int s_end = min(u1 * PU, units * PU), s_begin = u0 * PU;
        const int last_page = max(w.len - 1, 0) >> lp;
        const ScalarInts table = (ScalarInts)(uintptr_t)(a.table + (int64_t)at.seq * a.stride);
        const uint16_t *kb = a.c.k + ((size_t)at.head << lp) * HD, *vb = a.c.v + ((size_t)at.head << lp) * HD;
        auto fetch = [&](int s0, int buf) {  // slots s0 .. s0 + ST - 1
#pragma unroll
            for (int i = 0; i < CH; i++) {
                const int st = i * S::NW + wave;
                {
                    const int s = s0 + (st * RPC & ~15);
                    const int page = page_ok(a, table[min(s >> lp, last_page)]);
                    const char *src = (const char *)(kb + page * page_elems + (size_t)(s & (P - 1)) * HD) + ksrc[i];
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(uintptr_t)src,
                                                     (__attribute__((address_space(3))) void *)&lds[buf][0][st * WAVE], 16,
                                                     0, 0);
                }
                {
                    const int e = st / (HD / WAVE), s = s0 + 8 * e;
                    const int page = page_ok(a, table[min(s >> lp, last_page)]);
                    const uint16_t *src = vb + page * page_elems + (size_t)(s & (P - 1)) * HD +
                                          (st % (HD / WAVE) * WAVE + lane) * 8;
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(uintptr_t)src,
                                                     (__attribute__((address_space(3))) void *)&lds[buf][1][st * WAVE], 16,
                                                     0, 0);
                }
            }
        };
        float m = NEG, l = 0.f;
        f32x16 o[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = 0.f;
        if (s_begin < s_end) fetch(s_begin, 0);
        QPieces<NF, 16, F16> q;
        q.load(a.q, row_at(a, base, rr, at.head, a.q_stride) + 8 * h, r < rows, a.scale < 0.f,
               [](float x) { return half_reduce(x, Max()); });
        const float mul = fmaxf(ldexpf(scale, q.e), FLT_MIN);
        int buf = 0;
        for (int s0 = s_begin; s0 < s_end; s0 += ST, buf ^= 1) {
            // this step has arrived, and every wave is done with the other buffer
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (s0 + ST < s_end) fetch(s0 + ST, buf ^ 1);
            if (s0 >= mine) continue;
            const f16x8 *kt = lds[buf][0], *vt = lds[buf][1];
#pragma unroll
            for (int x = 0; x < X; x++) {
                f32x16 s;
#pragma unroll
                for (int i = 0; i < 16; i++) s[i] = 0.f;
#pragma unroll
                for (int f = 0; f < NF; f++) {
                    const f16x8 k = kt[(32 * x + c) * (HD / 8) + ((2 * f + h) ^ (c & 15))];
                    s = mfma32(k, q.hi[f], s);
                    if constexpr (!F16) s = mfma32(k, q.lo[f], s);
                }
                const int p0 = s0 + 32 * x;
                if (p0 + 32 > first_limit) {
#pragma unroll
                    for (int i = 0; i < 16; i++)
                        if (p0 + 16 * (i / 8) + 8 * h + i % 8 >= limit) s[i] = -INFINITY;
                }
                float top = s[0];
#pragma unroll
                for (int i = 1; i < 16; i++) top = fmaxf(top, s[i]);
                top = half_reduce(top * mul, Max());
                if (__any(top > m + LAZY)) {
                    const float m1 = fmaxf(m, ceilf(top)), alpha = ex2(m - m1);
                    m = m1;
                    l *= alpha;
#pragma unroll
                    for (int d = 0; d < DT; d++)
#pragma unroll
                        for (int i = 0; i < 16; i++) o[d][i] *= alpha;
                }
                f16x8 ph[2], pl[2];
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float p = F16 ? ex2(fmaf(s[8 * b + i], mul, PS - m))
                                            : ex2(fmaf(s[8 * b + i], mul, -m)) * 32768.f;
                        const _Float16 t = (_Float16)p;
                        ph[b][i] = t;
                        if constexpr (!F16) {
                            sum += p;
                            pl[b][i] = (_Float16)(p - (float)t);
                        }
                    }
                    if constexpr (F16) l = sum8(ph[b], l);
                    else l += sum;
                }
                const bool tail = p0 + 32 > w.len;  // bytes behind the sequence's end count for nothing
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    u32x4 keep;
                    if (tail) {
                        const int s8 = p0 + 16 * b + 8 * h;
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            keep[i] = (s8 + 2 * i < w.len ? 0xFFFFu : 0u) | (s8 + 2 * i + 1 < w.len ? 0xFFFF0000u : 0u);
                    }
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        f16x8 v = vt[(4 * x + 2 * b + h) * HD + 32 * d + c];
                        if (tail) v = __builtin_bit_cast(f16x8, __builtin_bit_cast(u32x4, v) & keep);
                        o[d] = mfma32(v, ph[b], o[d]);
                        if constexpr (!F16) o[d] = mfma32(v, pl[b], o[d]);
                    }
                }
            }
        }
        constexpr float UP = F16 ? 128.f : 1.f;
        l = half_reduce(l, Add()) * UP;
        if (r < rows) {
            const bool whole = u0 == 0 && u1 == units;
            const size_t slot = ((size_t)worker * 2 + (u0 == 0)) * a.part_rows + wave * 32 + c;
            const float inv = whole ? UP * inverse(l) : UP;
            const int64_t to = row_at(a, base, r, at.head, a.out_stride);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int dim = 32 * d + 8 * i + 4 * h;
                    const f32x4 y = {o[d][4 * i] * inv, o[d][4 * i + 1] * inv, o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv};
                    if (whole) store_out(a.out, F16, to + dim, y);
                    else *(f32x4 *)(a.part + slot * HD + dim) = y;
                }
            if (!whole && h == 0) a.ml[slot] = make_float2(m, l);
        }
        // the buffers are read before the next piece fills them
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    });
}

template <int HD, bool F16>
void prompts(const PagedAttnArgs &a, hipStream_t st) {
    constexpr int R = PromptShape<HD, F16>::R;
    hipLaunchKernelGGL((paged_prompts_kernel<HD, F16>), dim3((unsigned)a.workers), dim3(WG), 0, st, a);
    hipLaunchKernelGGL((paged_join_kernel<PromptsWork<R>, HD, R>), dim3((unsigned)a.workers - 1, (unsigned)((a.part_rows + JR - 1) / JR)),
                       dim3(WG), 0, st, a);
}
template <int HD>
void tokens(const PagedAttnArgs &a, hipStream_t st) {
    if (a.f16) hipLaunchKernelGGL((paged_tokens_kernel<HD, true>), dim3((unsigned)a.workers), dim3(WG), 0, st, a);
    else hipLaunchKernelGGL((paged_tokens_kernel<HD, false>), dim3((unsigned)a.workers), dim3(WG), 0, st, a);
    hipLaunchKernelGGL((paged_join_kernel<TokensWork, HD, 16>), dim3((unsigned)a.workers - 1, (unsigned)((a.part_rows + JR - 1) / JR)),
                       dim3(WG), 0, st, a);
}

constexpr int CUS = 256;

}  // namespace

int paged_tokens_workers(int hd) { return hd == 128 ? 3 * CUS : 2 * CUS; }
int paged_prompts_workers(int hd, bool f16) { return hd == 256 && !f16 ? CUS : 2 * CUS; }
int paged_prompts_tile(int hd, bool f16) {
    return hd == 128 ? (f16 ? PromptShape<128, true>::R : PromptShape<128, false>::R)
                     : (f16 ? PromptShape<256, true>::R : PromptShape<256, false>::R);
}

hipError_t launch_paged_tokens(const PagedAttnArgs &a, hipStream_t st) {
    if (a.c.hd == 128) tokens<128>(a, st);
    else if (a.c.hd == 256) tokens<256>(a, st);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}
hipError_t launch_paged_prompts(const PagedAttnArgs &a, hipStream_t st) {
    if (a.c.hd == 128 && a.f16) prompts<128, true>(a, st);
    else if (a.c.hd == 128) prompts<128, false>(a, st);
    else if (a.c.hd == 256 && a.f16) prompts<256, true>(a, st);
    else if (a.c.hd == 256) prompts<256, false>(a, st);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace oi
