// paged_attn.hip -- attention over the paged f16 cache: the newest tokens of many
// sequences, and packed prompts.
//
// Token j of a sequence's n sees slots 0 .. len - n + j.  Scores in base 2:
//   t_s = (q . K_s) scale log2(e),  p_s = 2^(t_s - m + 15),  m the running maximum
//   o = sum p_s V_s,   l = sum p_s,   out = o / l  (0 where a row sees nothing)
// m, l and o are 32-bit.  The matrix products take f16 operands: K and V are exact
// there; an f32 q is the sum of two halves (22 bits, scaled by a power of two per
// row), an f16 q exact.  Weights are the sum of two halves (22 bits) but for packed f16
// prompts, whose outputs hold no more than 11 bits: there p is rounded once and l is
// the sum of the rounded weights (with two halves 385 GFLOP of such prompts take 631 us, not 489, and are off by
// 2.0e-4 of their size, not 2.2e-4; a caller with use for them makes an F32 call).
// f16 numbers end at steps of 2^-24, so a weight is off by up to 2^-25 beside its bits, and lost below that.
// Tokens: the row's largest p is 2^14 to 2^15, so 2^-39 of it.  Prompts leave room above the maximum, so that few
// rises of it rescale o: the largest p is from 2^(PS - 1) on, PS 6 in f16 (2^-30: 2^17 such slots make a quarter of an
// output's rounding; 3 is 0.6% faster at head_dim 128, 3.5% at 256, and ends at 2^-27), 12 in f32 (2^-36: 2^17 make
// 2e-6, as much as an f32 sum of them may be off by; 9 is 4% faster and ends at 2^-33), 9 for tokens of f16
// rows (2^-33).  Cached values are finite (the append sees to it): a slot that a
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

#include <algorithm>
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
// A score's exponent is one multiply-add, its product with the row's factor not rounded, while a maximum is a
// rounded product: in a row whose largest score is FAR or more in base 2 (below it they differ by 2^-3 at most)
// they may lie powers of two apart, its weights all past f16 or all below it.  An f32 row's factor is a power of
// two, its products exact; an f16 row weighs such scores by their distance from the largest.
constexpr float FAR = 4194304.f;
__device__ __forceinline__ bool is_far(float top) { return fabsf(top) >= FAR && fabsf(top) <= FLT_MAX; }
constexpr int TU = 32;                   // slots of a unit of the tokens kernel
constexpr int PU = 64;                   // of the prompts kernel

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// a sequence's number in one of the call's arrays, through the scalar cache where all lanes ask for the same
template <bool SCALAR>
__device__ __forceinline__ int number(const int32_t *p, int s) {
    if constexpr (SCALAR) return ((ScalarInts)(uintptr_t)p)[__builtin_amdgcn_readfirstlane(s)];
    else return p[s];
}
template <bool SCALAR>
__device__ __forceinline__ int seq_len(const PagedAttnArgs &a, int s) {
    return min(max(number<SCALAR>(a.lens, s), 0), a.cap);
}
// All of the call's arguments asked for at once: a line of them at a time, where each is first
// used, they take a chain of misses.
__device__ __forceinline__ void ask(const PagedAttnArgs &a) {
    asm volatile("" ::"s"(a.c.k), "s"(a.c.v), "s"(a.q), "s"(a.out), "s"(a.q_stride), "s"(a.out_stride), "s"(a.scale));
    asm volatile("" ::"s"(a.magic), "s"(a.n_rows), "s"(a.starts), "s"(a.lens), "s"(a.table), "s"(a.stride), "s"(a.workers),
                 "s"(a.tile_units), "s"(a.at), "s"(a.ml), "s"(a.part));
}
// The token of row r of a sequence and kv head (token-major): r / group by a
// multiplication (exact while r * group < 2^32)
__device__ __forceinline__ int row_token(const PagedAttnArgs &a, int r) {
    return a.magic ? (int)__umulhi((uint32_t)r, a.magic) : r;
}
// A sequence's first token in q and out: starts[s], or n_q of each where there are no starts.
template <bool SCALAR>
__device__ __forceinline__ int first_token(const PagedAttnArgs &a, int s) {
    return a.starts ? min(max(number<SCALAR>(a.starts, s), 0), a.n_rows) : s * a.n_q;
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

// The tiles of a sequence and their costs, in units of slots (f32: a sum that f32 does not
// hold to the unit moves borders by as much, alike for both workers at one).
// Tokens: one tile.
struct TokensWork {
    // a worker's least, a tile's most parts; see border()
    static constexpr int LEAST = 4, PARTS = 256, NEAR = 2, SHORT = 0;
    // A tile's own cost (its rows of q, the waves' results joined; 48 sequences 62 us with 1, 54
    // with 4, 57 with 8)
    static constexpr float OWN = 4.f;
    static constexpr int tiles = 1;
    int len;
    float cost;
    template <bool SCALAR>
    __device__ static __forceinline__ TokensWork of(const PagedAttnArgs &a, int s) {
        TokensWork w;
        w.len = seq_len<SCALAR>(a, s);
        w.cost = (float)((w.len + TU - 1) / TU) + OWN;
        return w;
    }
    __device__ __forceinline__ float all() const { return cost; }
    __device__ __forceinline__ float most() const { return cost; }
    __device__ __forceinline__ int units(const PagedAttnArgs &, int) const { return (len + TU - 1) / TU; }
    // the tile that x falls into, and the unit there
    __device__ __forceinline__ int find(const PagedAttnArgs &a, float x, int &u) const {
        u = min((int)max(x - OWN, 0.f), units(a, 0));
        return 0;
    }
};
// Prompts: a tile of R rows more sees R / group slots more.
struct PromptsWork {
    static constexpr int R = 128, LEAST = 4, PARTS = 128, NEAR = 8, SHORT = 6;
    static constexpr float OWN = 4.f;  // nine short prompts 28 us with 1, 18 with 2 to 6
    int len, tokens, tiles;
    float first, step;  // of tile 0, and what each further one costs more
    template <bool SCALAR>
    __device__ static __forceinline__ PromptsWork of(const PagedAttnArgs &a, int s) {
        PromptsWork w;
        const int r0 = first_token<SCALAR>(a, s), r1 = max(first_token<SCALAR>(a, s + 1), r0);
        w.len = seq_len<SCALAR>(a, s);
        w.tokens = r1 - r0;
        w.tiles = (int)(((uint32_t)w.tokens * (uint32_t)a.group + R - 1) / R);  // rows stay below 2^32
        w.step = a.tile_units;
        w.first = (float)max(w.len - w.tokens, 0) * (1.f / PU) + OWN + w.step;
        return w;
    }
    __device__ __forceinline__ float upto(float t) const { return t * (first + 0.5f * step * (t - 1.f)); }
    __device__ __forceinline__ float all() const { return upto((float)tiles); }
    __device__ __forceinline__ float most() const { return tiles ? first + (float)(tiles - 1) * step : 0.f; }
    __device__ __forceinline__ int units(const PagedAttnArgs &a, int tile) const {
        const int last = row_token(a, min(tile * R + R, tokens * a.group) - 1);
        return (max(len - tokens + last + 1, 0) + PU - 1) / PU;
    }
    __device__ __forceinline__ int find(const PagedAttnArgs &a, float x, int &u) const {
        // upto(t) = x solved, of its two forms the one that does not cancel
        const float b = first - 0.5f * step;
        const int t = min((int)(2.f * x / (b + sqrtf(b * b + 2.f * step * x))), tiles - 1);
        const int n = units(a, t);
        const float in = x - upto((float)t) - OWN, cost = first + (float)t * step - OWN;
        u = min((int)(max(in, 0.f) / cost * (float)n), n);
        return t;
    }
};

// Sums over the lanes up to each, and a lane's value for all.
__device__ __forceinline__ float scan_lanes(float v) {
#define OI_SCAN(ctrl, rows) \
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), ctrl, rows, 0xF, false))
    OI_SCAN(0x111, 0xF);  // rows of 16: 1, 2, 4, 8 lanes back
    OI_SCAN(0x112, 0xF);
    OI_SCAN(0x114, 0xF);
    OI_SCAN(0x118, 0xF);
    OI_SCAN(0x142, 0xA);  // the last lane of rows 0 and 2 to the row behind
    OI_SCAN(0x143, 0xC);  // lane 31 to rows 2 and 3
#undef OI_SCAN
    return v;
}

// The border at x of the whole cost, given each lane's sum of `per` neighbouring sequences
// (own) and that of the lanes up to it (run); x at or behind the end of all is that end.  It
// rises with x, as every step of it does, so workers' stretches cover each unit once, wherever
// rounding puts the borders.  Within NEAR units of a tile's end (an eighth of a share, if that is
// less) it moves there; in a tile of at most SHORT units from up to half a share, since each
// part costs what a tile costs by itself, and the join.  Against an eighth throughout, 45 calls of 1 to 64 prompts
// of 5 to 1000 tokens, some behind caches, take 0.96 of the time in the mean: 0.76 to 0.86 where a few prompts of 100
// to 300 tokens meet, 1.13 at worst (12 prompts of 30 to 600 at head_dim 256, 47 -> 53 us; a step of 12 sequences 23.4 ->
// 22.4, another 16.8 -> 18.4).  Fractions that fall with a tile's length in place of the step (3 to 8 units over it)
// are the same in the mean (0.996 to 1.000 of this) and 0.82 to 1.13 of it in single calls.
template <class W>
__device__ PagedAt border(const PagedAttnArgs &a, float x, float share, float own, float run, int per) {
    const int lane = __lane_id();
    unsigned long long hit = __ballot(x < run && own > 0.f);
    if (!hit) return {a.n_seqs, 0, 0, 0};
    int at = __ffsll(hit) - 1;
    x = max(x - (lane_value(run, at) - lane_value(own, at)), 0.f);
    int s = at * per;
    if (per > 1) {  // these sequences, a lane each
        const int s1 = min(s + per, a.n_seqs);
        int last = s;  // with tiles, so far: rounding may leave x behind them all
        for (; s < s1; s += WAVE) {
            const float c = s + lane < s1 ? W::template of<false>(a, min(s + lane, s1 - 1)).all() * (float)a.c.n_kv : 0.f;
            const float r = scan_lanes(c);
            hit = __ballot(x < r && c > 0.f);
            if (hit) {
                at = __ffsll(hit) - 1;
                x = max(x - (lane_value(r, at) - lane_value(c, at)), 0.f);
                last = s + at;
                break;
            }
            hit = __ballot(c > 0.f);
            if (hit) last = s + 63 - __clzll(hit);
            x -= lane_value(r, WAVE - 1);
        }
        if (s >= s1) x = FLT_MAX;
        s = last;
    }
    s = __builtin_amdgcn_readfirstlane(s);
    const W w = W::template of<true>(a, s);
    const float one = w.all();
    int head = min((int)min(x / one, 2e9f), a.c.n_kv - 1), u;
    int tile = w.find(a, min(max(x - (float)head * one, 0.f), one), u);
    const int units = w.units(a, tile);
    const int near = (int)min(share * (units <= W::SHORT ? 0.5f : 0.125f), (float)W::NEAR);
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
    return {__builtin_amdgcn_readfirstlane(s), __builtin_amdgcn_readfirstlane(head), __builtin_amdgcn_readfirstlane(tile),
            __builtin_amdgcn_readfirstlane(u)};
}

// A worker's stretch, [begin, end); the number of workers used is returned (this one is
// idle if it is not below).  Every wave does it for itself, without LDS: a lane sums a run
// of neighbouring sequences.  Neighbouring workers go to one XCD (blocks are dealt to the
// 8 in turn), whose cache then holds what they share.
template <class W>
__device__ int share_out(const PagedAttnArgs &a, int &worker, PagedAt &begin, PagedAt &end) {
    const int lane = __lane_id(), per = (a.n_seqs + WAVE - 1) / WAVE;
    const int s0 = min(lane * per, a.n_seqs), s1 = min(s0 + per, a.n_seqs);
    float own = 0.f, most = 0.f;
    for (int s = s0; s < s1; s++) {
        const W w = W::template of<false>(a, s);
        own += w.all() * (float)a.c.n_kv;
        most = max(most, w.most());
    }
    const float run = scan_lanes(own), total = lane_value(run, WAVE - 1);
    const float share = max(max(total / (float)a.workers, (float)W::LEAST), wave_max_all(most) / (float)W::PARTS);
    const int used = __builtin_amdgcn_readfirstlane(min((int)ceilf(total / share), a.workers));
    const int each = (used + 7) / 8, b = blockIdx.x;
    worker = b / 8 < each ? (b & 7) * each + b / 8 : used;
    if (worker < used) {
        begin = border<W>(a, (float)worker * share, share, own, run, per);
        end = {a.n_seqs, 0, 0, 0};
        if (worker + 1 < used) end = border<W>(a, (float)(worker + 1) * share, share, own, run, per);
    }
    return used;
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
        const W w = W::template of<true>(a, at.seq);
        if (w.tiles) {
            const int units = w.units(a, at.tile);
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
// of its row, PART apart.  An f32 row is two halves of q f 2^-e, e the row's exponent,
// over the lanes that hold it (reduce), f the scale's fraction (1/2 to 1): what is left for the scores is a
// power of two.  A negative scale turns q's sign, so that the largest score is that of the largest product.
template <int NF, int PART, bool F16>
struct QPieces {
    f16x8 hi[NF], lo[F16 ? 1 : NF];
    int e = 0;
    template <class R>
    __device__ __forceinline__ void load(const void *q, int64_t at, bool ok, float scale, R reduce) {
        if constexpr (F16) {
            const uint32_t sign = scale < 0.f ? 0x80008000u : 0u;
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
            // f 2^-e as two factors that f32 holds; 0 for no row
            const float s0 = ok ? ldexpf(__builtin_amdgcn_frexp_mantf(scale), -e / 2) : 0.f, s1 = ldexpf(1.f, -e - -e / 2);
#pragma unroll
            for (int f = 0; f < NF; f++) {  // read again: the row is in cache, its registers are not free
                const f32x4 u = *(const f32x4 *)(p + PART * f), w = *(const f32x4 *)(p + PART * f + 4);
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const float x = i < 4 ? u[i & 3] : w[i & 3];
                    const float y = x * s0 * s1;
                    const _Float16 t = (_Float16)y;
                    hi[f][i] = t;
                    lo[f][i] = (_Float16)(y - (float)t);
                }
            }
        }
    }
    // what its products are to be multiplied by, above 0: -inf stays -inf
    __device__ __forceinline__ float factor(float scale) const {
        return fmaxf(F16 ? fabsf(scale) : ldexpf(1.f, __builtin_amdgcn_frexp_expf(scale) + e), FLT_MIN);
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
// Memory bounds it: 48 sequences of up to 9001 slots of 8 heads of 128 (320 MB) 54.6 us, 5.9
// TB/s; 3 of up to 120001 of 2 heads of 256 (456 MB) 74.6 us, 6.1; where a large nontemporal read
// makes 7.0.  A sequence of 1031 slots takes 6.6 us, a chain of misses: numbers, page ids, K, V.  More
// than 16 rows go to a wave two tiles at a time where registers allow, then to groups of waves that read
// the same slots (24 drafts of 5 tokens, 53 MB, 20.4 us); more than 64 to the prompts' kernel.  Three
// workgroups a CU spill registers (131 us against 122 where two hold all); so do four tiles a wave.
template <int HD>
struct TokensShape {
    static constexpr int PER_CU = HD == 128 ? 2 : 1;  // workgroups of a CU
};
template <int HD, bool F16, int NT, bool GROUPS>
__global__ __launch_bounds__(WG, TokensShape<HD>::PER_CU) void paged_tokens_kernel(PagedAttnArgs a) {
    constexpr int NW = WG / WAVE, NK = HD / 32, ND = HD / 16, PD = HD + 4;
    using W = TokensWork;
    __shared__ __attribute__((aligned(16))) float so[NW][16][PD];
    __shared__ float sm[NW][16], sl[NW][16];
    ask(a);
    int worker;
    PagedAt begin, end;
    const int used = share_out<W>(a, worker, begin, end);
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    if (blockIdx.x == 0 && tid == 0) a.at[a.workers] = {used, 0, 0, 0};
    if (worker >= used) return;
    leave_border(a, worker, begin, end);
    const int c = lane & 15, g = lane >> 4, lp = a.c.lp, P = 1 << lp;
    const int kslot = 8 * (c >> 2) + (c & 3);  // of a product's first 16 slots; 4 more in its second
    const size_t page_elems = ((size_t)a.c.n_kv << lp) * HD;
    const int rows = a.n_q * a.group;
    const int lg = GROUPS ? a.groups : 0, ng = 1 << lg;  // groups of waves
    const int group = wave & (ng - 1), turn = wave >> lg, step = NW >> lg;

    each_piece<W>(a, begin, end, [&](const W &w, const PagedAt &at, int units, int u0, int u1) {
        const int row0 = 16 * NT * group;
        const int len = w.len, seen0 = len - a.n_q + 1;  // slots that the first token sees
        const int first_limit = seen0 + row_token(a, min(row0, rows - 1));
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
        // Read once, by one wave, K and V pass the caches by (48 sequences of 320 MB 61 -> 54 us); the
        // groups' waves find them there (drafts of 24 sequences 21 us, 25 the other way).
        auto once = [](const uint16_t *p) {
            if constexpr (GROUPS) return *(const u32x4 *)p;
            else return ldg_nt((const u32x4 *)p);
        };
        auto load_k = [&](int u) {
            const uint16_t *p = kb + page_ok(a, kp) * page_elems + (size_t)((u * TU + kslot) & (P - 1)) * HD;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int f = 0; f < NK; f++) kr[t][f] = once(p + 4 * t * HD + 32 * f);
        };
        auto load_v = [&](int u, int page) {
            const uint16_t *p = vb + page_ok(a, page) * page_elems + (size_t)((u * TU + 8 * g) & (P - 1)) * HD;
#pragma unroll
            for (int d = 0; d < ND; d++) vr[d] = once(p + 16 * d * 8);
        };
        float m[NT], l[NT], mul[NT];
        int limit[NT];  // slots that this lane's rows see
        f32x4 o[NT][ND];
        int u = row0 < rows ? u0 + turn : u1;
        if (u < u1) {
            pages(u, kp, vp);
            if (u + step < u1) pages(u + step, kn, vn);
        }
        QPieces<NK, 32, F16> q[NT];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int row = row0 + 16 * n + c, rr = min(row, rows - 1);
            limit[n] = seen0 + row_token(a, rr);
            q[n].load(a.q, row_at(a, at.seq * a.n_q, rr, at.head, a.q_stride) + 8 * g, row < rows, a.scale,
                      [](float x) { return col_reduce(x, Max()); });
            mul[n] = q[n].factor(a.scale);
            m[n] = NEG;
            l[n] = 0.f;
#pragma unroll
            for (int d = 0; d < ND; d++) o[n][d] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (u < u1) {
            load_k(u);
            load_v(u, vp);
        }
        for (; u < u1; u += step) {
            f32x4 s[NT][2];
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int t = 0; t < 2; t++) s[n][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int f = 0; f < NK; f++) {
                    const f16x8 k = __builtin_bit_cast(f16x8, kr[t][f]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        s[n][t] = mfma(k, q[n].hi[f], s[n][t]);
                        if constexpr (!F16) s[n][t] = mfma(k, q[n].lo[f], s[n][t]);
                    }
                }
            kp = kn;
            if (u + step < u1) load_k(u + step);
            const int p0 = u * TU + 8 * g;  // the slot of s[n][0][0]
            f16x8 ph[NT], pl[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                if (u * TU + TU > first_limit) {  // some row does not see all of the unit
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (p0 + 4 * t + i >= limit[n]) s[n][t][i] = -INFINITY;
                }
                float top = s[n][0][0];
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) top = fmaxf(top, s[n][t][i]);
                const float most = col_reduce(top, Max());
                top = most * mul[n];
                const float m1 = fmaxf(m[n], ceilf(top));
                float bias = -m1;
                if (F16 && __builtin_expect(__any(is_far(top)), 0)) {
                    const float from = is_far(top) ? most : 0.f;
                    if (is_far(top)) bias = top - m1;
#pragma unroll
                    for (int t = 0; t < 2; t++)
#pragma unroll
                        for (int i = 0; i < 4; i++) s[n][t][i] -= from;
                }
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const float p = ex2(fmaf(s[n][t][i], mul[n], bias)) * 32768.f;
                        sum += p;
                        const _Float16 h = (_Float16)p;
                        ph[n][4 * t + i] = h;
                        pl[n][4 * t + i] = (_Float16)(p - (float)h);
                    }
                if (__any(m1 != m[n])) {  // a row's maximum rose
                    const float alpha = ex2(m[n] - m1);
                    l[n] *= alpha;
#pragma unroll
                    for (int d = 0; d < ND; d++) o[n][d] *= alpha;
                    m[n] = m1;
                }
                l[n] += sum;
            }
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
#pragma unroll
                for (int n = 0; n < NT; n++) o[n][d] = mfma(v, ph[n], o[n][d]);
#pragma unroll
                for (int n = 0; n < NT; n++) o[n][d] = mfma(v, pl[n], o[n][d]);
            }
            if (u + step < u1) {
                load_v(u + step, vn);
                if (u + 2 * step < u1) pages(u + 2 * step, kn, vn);
            }
        }
        // the waves' results meet in LDS, 16 rows of each group at a time
        const bool whole = u0 == 0 && u1 == units;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            if (n > 0 && 16 * n >= rows) break;
            const float ls = col_reduce(l[n], Add());
#pragma unroll
            for (int d = 0; d < ND; d++) *(f32x4 *)&so[wave][c][16 * d + 4 * g] = o[n][d];
            if (g == 0) {
                sm[wave][c] = m[n];
                sl[wave][c] = ls;
            }
            __syncthreads();
            // a group's rows over its `step` waves, 4 step threads a row
            const int tpr = 16 >> lg, tr = tid & ((WG >> lg) - 1), r = tr >> (4 - lg), sg = tid >> (8 - lg);
            const int row = 16 * (NT * sg + n) + r;
            if (row < rows) {
                float M = NEG, wt[NW], L = 0.f;
#pragma unroll
                for (int k = 0; k < NW; k++)
                    if (k < step) M = fmaxf(M, sm[sg + k * ng][r]);
#pragma unroll
                for (int k = 0; k < NW; k++)
                    if (k < step) {
                        wt[k] = ex2(sm[sg + k * ng][r] - M);
                        L += sl[sg + k * ng][r] * wt[k];
                    }
                const size_t slot = ((size_t)worker * 2 + (u0 == 0)) * a.part_rows + row;
                const float inv = whole ? inverse(L) : 1.f;
                const int64_t to = row_at(a, at.seq * a.n_q, row, at.head, a.out_stride);
                for (int d = 4 * (tr & (tpr - 1)); d < HD; d += 4 * tpr) {
                    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int k = 0; k < NW; k++)
                        if (k < step) y += *(const f32x4 *)&so[sg + k * ng][r][d] * wt[k];
                    y *= inv;
                    if (whole) store_out(a.out, F16, to + d, y);
                    else *(f32x4 *)(a.part + slot * HD + d) = y;
                }
                if (!whole && (tr & (tpr - 1)) == 0) a.ml[slot] = make_float2(M, L);
            }
            __syncthreads();  // LDS is read before it is written again
        }
    });
}

// ------------------------------------------------------------------- join --

// The parts of a tile that the border behind worker w cuts first: part 1 of w, then
// part 0 of the workers after it while they begin inside the tile.
__device__ __forceinline__ bool first_cut(const PagedAt &at, const PagedAt &prev) {
    return at.u > 0 && !(same_tile(at, prev) && prev.u > 0);
}

// One row of n parts, a workgroup's work: (m, l) and the first results of every thread are
// requested together.
constexpr int JOIN_MOST = 512, JPRE = 8;  // parts of a tile; of a thread in the first round trip
template <int HD>
struct JoinLds {
    static constexpr int LPR = HD / 4, MS = WG / LPR;  // lanes of a row, parts at a time
    float wt[JOIN_MOST];
    __attribute__((aligned(16))) float red[MS][HD];
    float wmax[WG / WAVE], wsum[WG / WAVE];
};
// part 1 of worker w, then part 0 of those behind it
__device__ __forceinline__ size_t part_at(const PagedAttnArgs &a, int w, int k, int r) {
    return ((size_t)(w + k) * 2 + (k == 0)) * a.part_rows + r;
}
template <int HD>
__device__ __forceinline__ void join_row(const PagedAttnArgs &a, int w, int n, int r, int64_t to, JoinLds<HD> &lds) {
    constexpr int LPR = JoinLds<HD>::LPR, MS = JoinLds<HD>::MS, KP = JOIN_MOST / WG;
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE, col = tid % LPR, k0 = tid / LPR;
    float2 ml[KP];
    f32x4 pre[JPRE];
#pragma unroll
    for (int i = 0; i < KP; i++) ml[i] = tid + i * WG < n ? a.ml[part_at(a, w, tid + i * WG, r)] : make_float2(NEG, 0.f);
#pragma unroll
    for (int i = 0; i < JPRE; i++) {
        const int k = k0 + i * MS;
        pre[i] = k < n ? *(const f32x4 *)(a.part + part_at(a, w, k, r) * HD + 4 * col) : f32x4{0.f, 0.f, 0.f, 0.f};
    }
    float m = NEG;
#pragma unroll
    for (int i = 0; i < KP; i++) m = fmaxf(m, ml[i].x);
    m = wave_max_all(m);
    if (lane == 0) lds.wmax[wave] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WG / WAVE; i++) m = fmaxf(m, lds.wmax[i]);
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < KP; i++) {
        const float f = ex2(ml[i].x - m);
        // 0 for a part that saw nothing (an empty one has no results to read)
        if (tid + i * WG < n) lds.wt[tid + i * WG] = ml[i].y == 0.f ? 0.f : f;
        l += ml[i].y * f;
    }
    l = wave_sum(l);
    if (lane == 0) lds.wsum[wave] = l;
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (int i = 0; i < WG / WAVE; i++) l += lds.wsum[i];
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < JPRE; i++) {
        const float f = k0 + i * MS < n ? lds.wt[k0 + i * MS] : 0.f;
        if (f != 0.f) y += pre[i] * f;
    }
#pragma unroll 8
    for (int k = k0 + JPRE * MS; k < n; k += MS) {
        const f32x4 p = *(const f32x4 *)(a.part + part_at(a, w, k, r) * HD + 4 * col);
        const float f = lds.wt[k];
        if (f != 0.f) y += p * f;
    }
    *(f32x4 *)&lds.red[k0][4 * col] = y;
    __syncthreads();
    if (tid < LPR) {
#pragma unroll
        for (int k = 1; k < MS; k++) y += *(const f32x4 *)&lds.red[k][4 * col];
        store_out(a.out, a.f16, to + 4 * col, y * inverse(l));
    }
}
// RT rows a thread, RT WG * 4 / HD of them apart from each other, four dimensions a thread;
// at(r): where row r goes
template <int HD, int RT, class F>
__device__ __forceinline__ void join_rows(const PagedAttnArgs &a, int w, int n, int r0, int rows, F at) {
    constexpr int LPR = HD / 4, RPW = WG / LPR, B = RT == 1 ? 8 : 2;
    const int col = threadIdx.x % LPR, r1 = r0 + threadIdx.x / LPR;
    float M[RT], L[RT];
    f32x4 y[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) {
        M[t] = NEG;
        L[t] = 0.f;
        y[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int k0 = 0; k0 < n; k0 += B) {
        float2 ml[RT][B];
        f32x4 p[RT][B];
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int i = 0; i < B; i++) {
                const size_t slot = part_at(a, w, min(k0 + i, n - 1), min(r1 + t * RPW, rows - 1));
                ml[t][i] = a.ml[slot];
                p[t][i] = *(const f32x4 *)(a.part + slot * HD + 4 * col);
            }
#pragma unroll
        for (int t = 0; t < RT; t++)
#pragma unroll
            for (int i = 0; i < B; i++) {
                if (k0 + i >= n || ml[t][i].y == 0.f) continue;  // saw nothing: an empty part has no results
                const float m1 = fmaxf(M[t], ml[t][i].x), f0 = ex2(M[t] - m1), f1 = ex2(ml[t][i].x - m1);
                L[t] = L[t] * f0 + ml[t][i].y * f1;
                y[t] = y[t] * f0 + p[t][i] * f1;
                M[t] = m1;
            }
    }
#pragma unroll
    for (int t = 0; t < RT; t++)
        if (r1 + t * RPW < rows) store_out(a.out, a.f16, at(r1 + t * RPW) + 4 * col, y[t] * inverse(L[t]));
}

// Tokens.  BY_TILE: a workgroup per tile (there are few) looks for the borders in it;
// otherwise one per border.  ROWS: 1, or those that a workgroup takes at once where there are
// many (3840 workgroups of a row each took 9 us for drafts of 24 sequences, 6.7 this way; 64 rows of 130000
// slots beside 63 sequences of 100: the call 72 us, 114 with tiles of many parts a row after the other).  A chain of
// three misses: borders, (m, l) with the results, out; 3.8 us for one sequence, 4.7 for 48.
template <int HD, bool BY_TILE, int ROWS>
__global__ __launch_bounds__(WG, 4) void paged_join_kernel(PagedAttnArgs a) {
    constexpr int NB = JOIN_MOST / WG;  // borders of a thread
    static_assert(TokensWork::PARTS + 2 <= JOIN_MOST && 2 * 256 <= JOIN_MOST, "a tile's parts, and all workers, fit");
    __shared__ JoinLds<HD> lds;
    __shared__ int count[WG / WAVE], least[WG / WAVE];
    const int r0 = blockIdx.y * ROWS, tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int used = a.at[a.workers].seq;
    PagedAt at;
    int w0 = blockIdx.x;  // the border looked at first is w0 + 1
    if constexpr (BY_TILE) {
        const int seq = (int)((uint32_t)blockIdx.x / (uint32_t)a.c.n_kv);
        at = {seq, (int)blockIdx.x - seq * a.c.n_kv, 0, 0};
        w0 = 0;
    } else {
        at = a.at[w0 + 1];
        const PagedAt prev = a.at[w0];
        if (w0 + 1 >= used || !first_cut(at, prev)) return;
    }
    const int rows = a.n_q * a.group;
    if (r0 >= rows) return;
    // borders inside the tile are neighbours
    int n = 0, first = INT32_MAX;
#pragma unroll
    for (int i = 0; i < NB; i++) {
        const int k = w0 + 1 + tid + i * WG;
        const PagedAt x = k < a.workers ? a.at[k] : PagedAt{-1, 0, 0, 0};
        const unsigned long long in = __ballot(k < used && same_tile(x, at) && x.u > 0);
        n += __popcll(in);
        if (in) first = min(first, k - lane + __ffsll(in) - 1);
    }
    if (lane == 0) {
        count[wave] = n;
        least[wave] = first;
    }
    __syncthreads();
    n = 0;
#pragma unroll
    for (int i = 0; i < WG / WAVE; i++) {
        n += count[i];
        first = min(first, least[i]);
    }
    if (n == 0) return;
    n++;
    const int w = first - 1;
    auto to = [&](int r) { return row_at(a, at.seq * a.n_q, r, at.head, a.out_stride); };
    if constexpr (ROWS == 1) join_row<HD>(a, w, n, r0, to(r0), lds);
    else join_rows<HD, ROWS * HD / 4 / WG>(a, w, n, r0, min(rows, r0 + ROWS), to);
}

// Prompts: a workgroup per border, RT rows a thread: 14703 packed rows, two parts to a tile, 11.3
// us with four, 16.7 with one; few tiles of many parts 20.7 and 12.1.
template <int HD, int RT>
__global__ __launch_bounds__(WG) void paged_join_rows_kernel(PagedAttnArgs a) {
    constexpr int R = PromptsWork::R, ROWS = WG * 4 / HD * RT;
    const int w = blockIdx.x, lane = threadIdx.x & (WAVE - 1), r0 = blockIdx.y * ROWS;
    const int used = a.at[a.workers].seq;
    const PagedAt at = a.at[w + 1], prev = a.at[w];
    const PagedAt next = w + 1 + lane < a.workers ? a.at[w + 1 + lane] : PagedAt{-1, 0, 0, 0};
    if (w + 1 >= used || !first_cut(at, prev)) return;
    const PromptsWork sw = PromptsWork::of<true>(a, at.seq);
    const int rows = min(sw.tokens * a.group - at.tile * R, R);
    if (r0 >= rows) return;
    // neighbours all: 1 and those of the next 64 that begin inside the tile, and so on
    int n = 1 + __popcll(__ballot(w + 1 + lane < used && same_tile(next, at) && next.u > 0));
    for (int k = w + 1 + WAVE; n == k - w && k < used; k += WAVE) {
        const PagedAt x = k + lane < used ? a.at[k + lane] : PagedAt{-1, 0, 0, 0};
        n += __popcll(__ballot(same_tile(x, at) && x.u > 0));
    }
    const int base = first_token<true>(a, at.seq);
    join_rows<HD, RT>(a, w, n, r0, rows,
                           [&](int r) { return row_at(a, base, at.tile * R + r, at.head, a.out_stride); });
}

// ---------------------------------------------------------------- prompts --

// Workgroups of a CU, as registers and LDS allow.
template <int HD, bool F16>
struct PromptsShape {
    static constexpr int PER_CU = HD == 128 && F16 ? 2 : 1;
};
constexpr int PR = PromptsWork::R;  // rows of a tile

// A worker of four waves takes tiles of 128 rows of one kv head, a wave 32 of them, and the
// tile's slots 64 at a time through two buffers of K and two of V in LDS, filled straight from
// memory (K a step ahead of V) while the others are worked on.  Scores transposed, on 32x32x16
// products.  K's piece j (8 dimensions) of LDS row r lies at j ^ (r & 15), and row r holds the
// slot with bits 2 and 3 of r exchanged: the products then leave a lane the scores of slots 8 h +
// 0..7 of each 16, those whose weights it supplies to the product with V; V's pieces (8 slots of
// a dimension) lie as in the cache.  Either way sixteen lanes read all banks once.
// A wave's work is a pipeline over halves of 32 slots: while the vector units turn half i's
// scores to weights, the matrix units form half i + 1's scores and the products of half i -
// 1's weights with V.  A row's maximum is raised only when another is more than 2^LAZY above it
// (weights then reach 2^15 at most, from 2^PS), and o follows after the products that go by the
// old one.
// Packed f16 prompts of 900 to 5003 tokens, 32 heads of 128 over 8 (385 GFLOP): 478 to 505 us, 760
// to 805 TFLOP/s; four of 8000 tokens 866; at head_dim 256 (378 GFLOP) 565 us; f32 rows there, two products for
// each (110 GFLOP), 271 to 282 us.  Matrix and vector units are both busy in 4 of 10 cycles: a wave issues in order, and
// two waves a SIMD do not fill each other's gaps (16 products alone 225 ns, beside their softmax
// 433 in a loop of nothing else, 600 here).  Where pages are read once or twice, their misses add a
// tenth to two (two times 50 tokens behind 40000 slots 121 us, 99 with pages in cache).
// Measured and left: 64 rows a wave (700 us against 565), eight waves on 256 rows (the same, long ones 5%
// slower), pieces of LDS read 6 or 8 ahead (the same), lines of the step after next touched ahead of
// their fetch (10% slower), a half's first pieces read before the fetches are issued (f16 at head_dim
// 256 5% slower), waves' priorities (the same), no pipeline (f16 the same, f32 slower).  Scalar registers: 30 to 33
// spill into lanes of a vector one; vector registers only at head_dim 256 in f32 (8), outside the products.
// TWO: weights as two halves (all but packed f16 prompts).
template <int HD, bool F16, bool TWO>
__global__ __launch_bounds__(WG, (PromptsShape<HD, F16>::PER_CU)) void paged_prompts_kernel(PagedAttnArgs a) {
    constexpr int NW = WG / WAVE, NF = HD / 16, DT = HD / 32;
    constexpr int PIECES = PU * HD / 8;     // of K, and of V, in a step
    constexpr int CH = PIECES / WAVE / NW;  // a wave's stretches of 64 pieces, of each
    static_assert(CH * WAVE == 2 * HD, "sixteen slots");
    constexpr int RPC = WAVE / (HD / 8);    // K rows of a stretch
    // room for a rise of the maximum and for small weights share f16's range: see above
    constexpr float PS = !TWO ? 6.f : F16 ? 9.f : 12.f, LAZY = 15.f - PS;
    using W = PromptsWork;
    __shared__ __attribute__((aligned(16))) f16x8 kl[2][PIECES], vl[2][PIECES];
    ask(a);
    int worker;
    PagedAt begin, end;
    const int used = share_out<W>(a, worker, begin, end);
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    if (blockIdx.x == 0 && tid == 0) a.at[a.workers] = {used, 0, 0, 0};
    if (worker >= used) return;
    leave_border(a, worker, begin, end);
    const int c = lane & 31, h = lane >> 5, lp = a.c.lp, P = 1 << lp;
    const uint32_t page_bytes = ((uint32_t)a.c.n_kv << lp) * HD * 2;
    // A wave brings the sixteen slots of its number, in CH stretches: a lane's place there.
    uint32_t ksrc[CH], vsrc[CH];
#pragma unroll
    for (int i = 0; i < CH; i++) {
        const int r = i * RPC + lane / (HD / 8), j = lane % (HD / 8);
        const int s16 = (r & 3) | (r & 4) << 1 | (r & 8) >> 1;
        ksrc[i] = (uint32_t)(s16 * HD + 8 * (j ^ r)) * 2;
        vsrc[i] = (uint32_t)(i * WAVE + lane) * 16;
    }

    each_piece<W>(a, begin, end, [&](const W &w, const PagedAt &at, int units, int u0, int u1) {
        const int rows = w.tokens * a.group, past = w.len - w.tokens;
        const int base = first_token<true>(a, at.seq);
        const int row0 = at.tile * PR + wave * 32, r = row0 + c, rr = min(r, rows - 1);  // my rows
        const int s_end = u1 * PU;
        const int mine = row0 < rows ? past + row_token(a, min(row0 + 32, rows) - 1) + 1 : 0;  // slots my rows see
        const int first_limit = min(past + row_token(a, min(row0, rows - 1)) + 1, s_end);
        const int limit = min(past + row_token(a, rr) + 1, s_end);
        const int last_page = max(w.len - 1, 0) >> lp;
        const ScalarInts table = (ScalarInts)(uintptr_t)(a.table + (int64_t)at.seq * a.stride);
        const char *kb = (const char *)(a.c.k + ((size_t)at.head << lp) * HD),
                   *vb = (const char *)(a.c.v + ((size_t)at.head << lp) * HD);
        // My sixteen slots of a step lie within a page (one to look up in place of four: 8000 tokens 2.5%
        // faster, f32 at head_dim 256 4%): the page, and where they begin (K and V at the
        // same place of their halves of the cache), in bytes.
        auto look_up = [&](int u) { return table[min((u * PU + 16 * wave) >> lp, last_page)]; };
        auto place = [&](int u, int page) {
            return (uint64_t)(uint32_t)page_ok(a, page) * page_bytes + (uint32_t)(((u * PU + 16 * wave) & (P - 1)) * HD * 2);
        };
        auto fetch = [&](const char *from, uint64_t at, const uint32_t (&src)[CH], f16x8 *to) {
            const char *x = from + at;
            asm volatile("" : "+s"(x));  // a scalar address, the lane's 32-bit place behind it
#pragma unroll
            for (int i = 0; i < CH; i++)
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(uintptr_t)(x + src[i]),
                                                 (__attribute__((address_space(3))) void *)(to + (wave * CH + i) * WAVE), 16, 0,
                                                 0);
        };
        // what this wave asked for has arrived and what it read is in registers; then all waves
        auto meet = [&]() {
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        // ahead of their use: where the next steps of V and of K lie, and the page of the one after
        uint64_t vp = place(u0, look_up(u0)), kp = place(u0 + 1, look_up(u0 + 1));
        int ahead = look_up(u0 + 2);
        auto go_on = [&](int u) {
            vp = kp;
            kp = place(u, ahead);
            ahead = look_up(u + 1);
        };
        if (u0 < u1) fetch(kb, vp, ksrc, kl[u0 & 1]);
        QPieces<NF, 16, F16> q;
        q.load(a.q, row_at(a, base, rr, at.head, a.q_stride) + 8 * h, r < rows, a.scale,
               [](float x) { return half_reduce(x, Max()); });
        const float mul = q.factor(a.scale);
        float m = NEG, l = 0.f;
        f32x16 o[DT];
#pragma unroll
        for (int d = 0; d < DT; d++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[d][i] = 0.f;
        // The softmax of a half in steps: the maximum of score pairs, the rows' new maxima, weights of a
        // pair.  Rows rise together, so that one that climbs takes the others along and few halves
        // rise at all; alpha: what o is to be multiplied by then.
        // high: what a score is to pass for that; most: the row's largest score before its factor.
        float top = 0.f, most = 0.f, alpha = 1.f, bias = 0.f, high = NEG, sum = 0.f;  // sum: of the half's weights
        bool rise = false;
        auto higher = [&](const f32x16 &s, int i) {
            top = i == 0 ? fmaxf(s[0], s[1]) : fmaxf(fmaxf(top, s[2 * i]), s[2 * i + 1]);
        };
        auto highest = [&]() {
            most = half_reduce(top, Max());
            top = most * mul;
        };
        auto turn = [&](f32x16 &s) {
            rise = __any(top > high);
            // a branch where registers allow (f32 rows at head_dim 256 take 310 us with it, 278 without; at 128 426
            // and 429, f16 rows at 256 545 and 550)
            if ((HD == 128 || F16) && __builtin_expect(!rise, 1)) return;
            const float m1 = rise ? fmaxf(m, ceilf(top)) : m;
            alpha = ex2(m - m1);
            m = m1;
            l *= alpha;
            // a far maximum has no room for PS or LAZY beside it
            const bool near = fabsf(m1) < FAR;
            bias = (near ? PS : 0.f) - m1;
            high = near ? m1 + LAZY : F16 ? NEG : m1;
            if (F16 && __builtin_expect(rise, 0)) {
                if (__any(is_far(top))) {  // every half of such a row comes by here
                    const float from = is_far(top) ? most : 0.f;
                    if (is_far(top)) bias = top - m1;
#pragma unroll
                    for (int i = 0; i < 16; i++) s[i] -= from;
                }
            }
        };
        auto weigh = [&](const f32x16 &s, f16x8 (&ph)[2], f16x8 (&pl)[2], int i) {
            f16x2 hi, lo;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const float p = ex2(fmaf(s[2 * i + k], mul, bias));
                hi[k] = (_Float16)p;
                if constexpr (TWO) {
                    sum = i + k == 0 ? p : sum + p;
                    lo[k] = (_Float16)(p - (float)hi[k]);
                }
            }
            if constexpr (!TWO) sum = __builtin_amdgcn_fdot2(hi, f16x2{(_Float16)1.f, (_Float16)1.f}, i == 0 ? 0.f : sum, false);
            if (i == 7) l += sum;
            asm volatile("" : "+v"(hi), "+v"(sum));  // here, not where it is used
            if constexpr (TWO) asm volatile("" : "+v"(lo));
#pragma unroll
            for (int k = 0; k < 2; k++) {
                ph[i / 4][2 * (i % 4) + k] = hi[k];
                if constexpr (TWO) pl[i / 4][2 * (i % 4) + k] = lo[k];
            }
        };
        auto k_piece = [&](const f16x8 *kt, int x, int f) { return kt[(32 * x + c) * (HD / 8) + ((2 * f + h) ^ (c & 15))]; };
        auto score = [&](const f16x8 &k, int f, f32x16 &s) {
            if (f == 0) {
#pragma unroll
                for (int i = 0; i < 16; i++) s[i] = 0.f;
            }
            s = mfma32(k, q.hi[f], s);
            if constexpr (!F16) s = mfma32(k, q.lo[f], s);
        };
        // o in the registers that only the matrix units use, where the others do not hold it
        auto pin = [&]() {
            if constexpr (PromptsShape<HD, F16>::PER_CU == 1)
#pragma unroll
                for (int d = 0; d < DT; d++) asm volatile("" : "+a"(o[d]));
        };
        // Half a step of the pipeline: weights p1 of the scores s0, the next scores s1 from half x of the K
        // buffer, the products of the former weights p0 with half x of the V buffer.  Pieces of K, then of
        // V come from LDS AHEAD of their use, and the vector units' work lies between their products in
        // the order written here.
        auto half = [&](const f16x8 *kt, const f16x8 *vt, int x, f32x16 &s0, f32x16 &s1, const f16x8 (&ph0)[2],
                        const f16x8 (&pl0)[2], f16x8 (&ph1)[2], f16x8 (&pl1)[2]) {
            constexpr int N = NF + 2 * DT, AHEAD = 4, CLIMB = N / 4, STEP = N / 16;
            static_assert(CLIMB + 2 + 7 * STEP < N, "all weights are formed");
            f16x8 w[N];
            auto read = [&](int j) {
                if (j < NF) w[j] = k_piece(kt, x, j);
                else w[j] = vt[(4 * x + 2 * ((j - NF) / DT) + h) * HD + 32 * ((j - NF) % DT) + c];
            };
#pragma unroll
            for (int j = 0; j < AHEAD; j++) read(j);
#pragma unroll
            for (int j = 0; j < N; j++) {
                if (j + AHEAD < N) read(j + AHEAD);
                if (j < NF) {
                    score(w[j], j, s1);
                } else {
                    const int i = (j - NF) / DT, d = (j - NF) % DT;
                    o[d] = mfma32(w[j], ph0[i], o[d]);
                    if constexpr (TWO) o[d] = mfma32(w[j], pl0[i], o[d]);
                }
                if (j < CLIMB) {
#pragma unroll
                    for (int i = 8 * j / CLIMB; i < 8 * (j + 1) / CLIMB; i++) higher(s0, i);
                } else if (j == CLIMB) {
                    highest();
                } else if (j == CLIMB + 1) {
                    turn(s0);
                } else if ((j - CLIMB - 2) % STEP == 0 && (j - CLIMB - 2) / STEP < 8) {
                    weigh(s0, ph1, pl1, (j - CLIMB - 2) / STEP);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if (__builtin_expect(rise, 0)) {
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int i = 0; i < 16; i++) o[d][i] *= alpha;
            }
            pin();
        };
        // some row does not see all of the half
        auto hide = [&](f32x16 &s, int p0) {
            if (__builtin_expect(p0 + 32 > first_limit, 0)) {
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (p0 + 16 * (i / 8) + 8 * h + i % 8 >= limit) s[i] = -INFINITY;
            }
        };
        // step u: V of it and K of the next are here, the other two buffers free
        auto stage = [&](int u) {
            meet();
            if (u + 1 < u1) fetch(vb, vp, vsrc, vl[(u + 1) & 1]);
            if (u + 2 < u1) fetch(kb, kp, ksrc, kl[u & 1]);
            go_on(u + 3);
            if (__builtin_expect(u * PU + PU > w.len, 0)) {  // bytes behind the sequence's end count for nothing
                for (int i = tid; i < PIECES; i += WG) {
                    const int s8 = u * PU + 8 * (i / HD);
                    u32x4 keep;
#pragma unroll
                    for (int k = 0; k < 4; k++)
                        keep[k] = (s8 + 2 * k < w.len ? 0xFFFFu : 0u) | (s8 + 2 * k + 1 < w.len ? 0xFFFF0000u : 0u);
                    f16x8 &v = vl[u & 1][i];
                    v = __builtin_bit_cast(f16x8, __builtin_bit_cast(u32x4, v) & keep);
                }
                meet();
            }
        };
        if (u0 < u1) {
            meet();
            fetch(vb, vp, vsrc, vl[u0 & 1]);
            if (u0 + 1 < u1) fetch(kb, kp, ksrc, kl[(u0 + 1) & 1]);
            go_on(u0 + 2);
        }
        if (mine <= u0 * PU) {  // my rows see nothing here; this wave fetches for the others
            for (int u = u0; u < u1; u++) stage(u);
        } else {
            f32x16 s0, s1;
            f16x8 ph0[2], pl0[2], ph1[2], pl1[2];
#pragma unroll
            for (int f = 0; f < NF; f++) score(k_piece(kl[u0 & 1], 0, f), f, s0);
            hide(s0, u0 * PU);
#pragma unroll
            for (int i = 0; i < 8; i++) higher(s0, i);
            highest();
            turn(s0);  // o is 0
#pragma unroll
            for (int i = 0; i < 8; i++) weigh(s0, ph0, pl0, i);
#pragma unroll
            for (int f = 0; f < NF; f++) score(k_piece(kl[u0 & 1], 1, f), f, s1);
            pin();
            // the last half's scores are of no step (K's buffer holds an older one): hidden, they weigh nothing
            for (int u = u0; u < u1; u++) {
                stage(u);
                const f16x8 *kt = kl[(u + 1) & 1], *vt = vl[u & 1];
                hide(s1, u * PU + 32);
                half(kt, vt, 0, s1, s0, ph0, pl0, ph1, pl1);
                hide(s0, u * PU + PU);
                half(kt, vt, 1, s0, s1, ph1, pl1, ph0, pl0);
            }
        }
        const bool whole = u0 == 0 && u1 == units;
        l = half_reduce(l, Add());
        if (r < rows) {
            const size_t slot = ((size_t)worker * 2 + (u0 == 0)) * a.part_rows + wave * 32 + c;
            const float inv = whole ? inverse(l) : 1.f;
            const int64_t to = row_at(a, base, r, at.head, a.out_stride);
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int dim = 32 * d + 8 * i + 4 * h;
                    const f32x4 y = f32x4{o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]} * inv;
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

constexpr int CUS = 256;

unsigned groups_of(int n, int size) { return (unsigned)((n + size - 1) / size); }

template <int HD, bool F16>
void prompts(const PagedAttnArgs &a, hipStream_t st) {
    if (F16 && a.starts)  // packed; a tokens call has none
        hipLaunchKernelGGL((paged_prompts_kernel<HD, F16, !F16>), dim3((unsigned)a.workers), dim3(WG), 0, st, a);
    else
        hipLaunchKernelGGL((paged_prompts_kernel<HD, F16, true>), dim3((unsigned)a.workers), dim3(WG), 0, st, a);
    // about as many tiles as workers: two parts each, four rows a thread; few tiles: many parts
    constexpr int RT = 4, ROWS = WG * 4 / HD;
    const int64_t tiles = ((int64_t)a.n_rows * a.group / PR + a.n_seqs) * a.c.n_kv;
    if (2 * tiles > a.workers)
        hipLaunchKernelGGL((paged_join_rows_kernel<HD, RT>), dim3((unsigned)a.workers - 1, groups_of(a.part_rows, ROWS * RT)),
                           dim3(WG), 0, st, a);
    else
        hipLaunchKernelGGL((paged_join_rows_kernel<HD, 1>), dim3((unsigned)a.workers - 1, groups_of(a.part_rows, ROWS)), dim3(WG),
                           0, st, a);
}
template <int HD, bool BY_TILE>
void join_tokens(const PagedAttnArgs &a, int n, hipStream_t st) {
    constexpr int ROWS = WG * 4 / HD;
    if ((int64_t)n * a.part_rows <= 4 * CUS)
        hipLaunchKernelGGL((paged_join_kernel<HD, BY_TILE, 1>), dim3((unsigned)n, (unsigned)a.part_rows), dim3(WG), 0, st, a);
    else
        hipLaunchKernelGGL((paged_join_kernel<HD, BY_TILE, ROWS>), dim3((unsigned)n, groups_of(a.part_rows, ROWS)), dim3(WG), 0,
                           st, a);
}
template <int HD, bool F16, int NT>
void tokens(const PagedAttnArgs &a, hipStream_t st) {
    constexpr bool MORE = !(HD == 128 && F16 && NT == 1);  // than 16 NT rows, as tokens_tiles has it
    if (MORE && a.groups)
        hipLaunchKernelGGL((paged_tokens_kernel<HD, F16, NT, MORE>), dim3((unsigned)a.workers), dim3(WG), 0, st, a);
    else
        hipLaunchKernelGGL((paged_tokens_kernel<HD, F16, NT, false>), dim3((unsigned)a.workers), dim3(WG), 0, st, a);
    const int64_t items = (int64_t)a.n_seqs * a.c.n_kv;
    if (items < a.workers) join_tokens<HD, true>(a, (int)items, st);
    else join_tokens<HD, false>(a, a.workers - 1, st);
}

}  // namespace

// 16 rows of a wave (twice where registers allow) and, as a power of two, its workgroup's groups of
// waves, which read the same slots for other rows
static int tokens_tiles(int hd, int rows, bool f16) { return hd == 128 && f16 && rows > 16 ? 2 : 1; }
int paged_tokens_groups(int hd, int rows, bool f16) {
    const int r = 16 * tokens_tiles(hd, rows, f16);
    return rows <= r ? 0 : rows <= 2 * r ? 1 : 2;
}
int paged_tokens_workers(int hd) {
    return CUS * (hd == 128 ? TokensShape<128>::PER_CU : TokensShape<256>::PER_CU);
}
int paged_prompts_workers(int hd, bool f16) {
    return CUS * (hd == 128 ? (f16 ? PromptsShape<128, true>::PER_CU : PromptsShape<128, false>::PER_CU)
                            : (f16 ? PromptsShape<256, true>::PER_CU : PromptsShape<256, false>::PER_CU));
}
int paged_prompts_rows() { return PR; }

hipError_t launch_paged_tokens(const PagedAttnArgs &a, hipStream_t st) {
    const int nt = tokens_tiles(a.c.hd, a.n_q * a.group, a.f16);
    if (a.c.hd == 128 && a.f16 && nt == 2) tokens<128, true, 2>(a, st);
    else if (a.c.hd == 128 && a.f16) tokens<128, true, 1>(a, st);
    else if (a.c.hd == 128) tokens<128, false, 1>(a, st);
    else if (a.c.hd == 256 && a.f16) tokens<256, true, 1>(a, st);
    else if (a.c.hd == 256) tokens<256, false, 1>(a, st);
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
