// kv8.hip -- the 8-bit K/V cache: append, read, eviction.
//
// value = c 2^e: a signed byte c per value, an exponent e per (kv head, block of
// slots), apart for K and V.  With a power of two as the step, x 2^-e is exact
// and one rounding (half to even) makes the byte; when a later token raises the
// exponent of a partly filled block, its earlier codes are shifted down and
// rounded again, by at most half the new step each time.  As the step at least
// doubles, these sum to less than one final step, however many appends it took.
// The step is 1.44 times that of amax / 127 on average.
//
// V lies transposed in tiles of 64 slots, [hd][64], the order in which the
// matrix product P V takes it (kv8_attn.hip).

#include <type_traits>

#include "kv8_common.h"

namespace oi {

namespace {

constexpr int T = KV8_TILE;

// the least e in [EMIN, EMAX] with amax <= 127 * 2^e: 127 = 1.984375 * 2^6
__device__ __forceinline__ int exp_for(float amax) {
    const uint32_t b = __float_as_uint(amax);
    const int e = (int)(b >> 23) - 127 - 6 + ((b & 0x7FFFFFu) > 0x7E0000u ? 1 : 0);
    return min(max(e, KV8_EMIN), KV8_EMAX);
}
// half to even; NaN is stored as 0, what lies past the largest block's range as +-127
__device__ __forceinline__ int code_of(float x, float inv) {
    const float r = rintf(x * inv);
    return r == r ? (int)fminf(fmaxf(r, -127.f), 127.f) : 0;
}
// a code whose exponent rises by d >= 0
__device__ __forceinline__ int shift_code(int c, float down) { return (int)rintf((float)c * down); }

__device__ __forceinline__ int byte_of(uint32_t w, int j) { return (int)(int8_t)(w >> (8 * j)); }
__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)(d & 255) << 24;
}

// One workgroup per (64-slot unit that the new tokens touch, kv head, K or V),
// wave w its slots 16 w .. 16 w + 15, a lane 4 dimensions of every row it
// loads.  All rows are requested at once; the largest finite magnitudes of the
// waves of a block meet in LDS, K codes go out from registers, V codes through an
// LDS tile that is read by columns.  8001 tokens of 8 heads of 128 from f16 (49 MB)
// 14 us, bound by memory behind one chain of load, maximum and store; one token
// 5.3 us, that chain.
template <int HD, bool F16>
__global__ __launch_bounds__(WG) void kv8_append_kernel(Kv8AppendArgs a) {
    constexpr int RPL = WAVE * 4 / HD, NR = 16 / RPL;  // rows of one load of the wave, loads
    __shared__ __attribute__((aligned(16))) uint32_t tile[T][HD / 4];
    __shared__ float wmax[4];
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int past = kv8_past(a.past, a.n, a.c.cap), end = past + a.n;
    const int unit = past / T + (int)blockIdx.x, kvh = blockIdx.y, which = blockIdx.z;
    if (unit * T >= end) return;
    const int s0 = unit * T + 16 * wave, col = lane % (HD / 4), r0 = lane / (HD / 4);
    const int64_t stride = a.stride[which];
    const int blk = s0 >> a.c.lb, b0 = blk << a.c.lb;
    int8_t *ep = (which ? a.c.ve : a.c.ke) + (size_t)kvh * (a.c.cap >> a.c.lb) + blk;
    const bool old = b0 < past;  // the block holds earlier slots
    // what the call may have to keep is requested with the new rows: the exponent, and V's
    // pieces of 16 slots that are not all new
    const int8_t e_was = old ? *ep : 0;
    const bool whole = s0 >= past && s0 + 16 <= end, any = s0 < end && s0 + 16 > past;
    u32x4 vp[HD / WAVE];
    u32x4 *const vat = (u32x4 *)(a.c.vc + (((size_t)kvh * (a.c.cap / T) + unit) * HD + lane) * T + 16 * wave);
    if (which && !whole && (any || (old && s0 < past)))
#pragma unroll
        for (int k = 0; k < HD / WAVE; k++) vp[k] = vat[k * WAVE * T / 16];
    float x[NR][4];
#pragma unroll
    for (int j = 0; j < NR; j++) {
        const int s = s0 + j * RPL + r0;
        const bool in = s >= past && s < end;
        const int64_t at = (int64_t)(in ? s - past : 0) * stride + (int64_t)kvh * HD + 4 * col;
        if constexpr (F16) {
            const u32x2 w = in ? *(const u32x2 *)((const uint16_t *)a.x[which] + at) : u32x2{0u, 0u};
            x[j][0] = h2f(w.x & 0xFFFFu);
            x[j][1] = h2f(w.x >> 16);
            x[j][2] = h2f(w.y & 0xFFFFu);
            x[j][3] = h2f(w.y >> 16);
        } else {
            const float4 w = in ? *(const float4 *)((const float *)a.x[which] + at) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[j][0] = w.x;
            x[j][1] = w.y;
            x[j][2] = w.z;
            x[j][3] = w.w;
        }
    }
    float amax = 0.f;
#pragma unroll
    for (int j = 0; j < NR; j++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const float m = fabsf(x[j][e]);
            amax = fmaxf(amax, m < INFINITY ? m : 0.f);
        }
    amax = wave_max_all(amax);
    if (lane == 0) wmax[wave] = amax;
    __syncthreads();
    const int nw = 1 << (a.c.lb - 4), w0 = wave & ~(nw - 1);  // waves of this block, its first
    for (int w = 0; w < nw; w++) amax = fmaxf(amax, wmax[w0 + w]);
    int e = exp_for(amax), e_old = e;
    if (old) {
        e_old = kv8_exp(e_was);
        e = max(e, e_old);
    }
    const bool touched = b0 < end && b0 + (1 << a.c.lb) > past;
    const float inv = pow2i(-e), down = pow2i(e_old - e);
    uint32_t q[NR];
#pragma unroll
    for (int j = 0; j < NR; j++)
        q[j] = pack4(code_of(x[j][0], inv), code_of(x[j][1], inv), code_of(x[j][2], inv), code_of(x[j][3], inv));
    const bool requant = old && e > e_old;
    if (which == 0) {
        uint32_t *kc = (uint32_t *)(a.c.kc + ((size_t)kvh * a.c.cap + s0) * HD) + lane;
#pragma unroll
        for (int j = 0; j < NR; j++) {
            const int s = s0 + j * RPL + r0;
            uint32_t *p = kc + j * WAVE;
            if (s >= past && s < end) *p = q[j];
            else if (requant && s < past && s >= b0) {
                const uint32_t w = *p;
                *p = pack4(shift_code(byte_of(w, 0), down), shift_code(byte_of(w, 1), down),
                           shift_code(byte_of(w, 2), down), shift_code(byte_of(w, 3), down));
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < NR; j++) tile[16 * wave + j * RPL + r0][col] = q[j];
        __builtin_amdgcn_wave_barrier();  // this wave's 16 rows only
        // 16 slots of a dimension: one 16-byte piece of its row
        if (any || (requant && s0 < past)) {
            const uint8_t *tb = (const uint8_t *)&tile[16 * wave][0];
#pragma unroll
            for (int k = 0; k < HD / WAVE; k++) {
                const int d = lane + k * WAVE;
                u32x4 w = whole ? u32x4{0u, 0u, 0u, 0u} : vp[k];
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    uint32_t r = 0;
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int s = s0 + 4 * c + i;
                        const int was = byte_of(w[c], i);
                        const int v = s >= past && s < end ? (int)tb[(4 * c + i) * HD + d]
                                      : requant && s < past ? shift_code(was, down) : was;
                        r |= (uint32_t)(v & 255) << (8 * i);
                    }
                    w[c] = r;
                }
                vat[k * WAVE * T / 16] = w;
            }
        }
    }
    if (touched && lane == 0 && wave == w0) *ep = (int8_t)e;
}

// One workgroup per (64 slots, kv head, K or V): codes times their block's
// step.  K as it lies, V through an LDS tile read by columns.  Bound by memory:
// 40001 slots of 8 heads of 128 to f32 (410 MB) 59 us, 6.9 TB/s (f32 values stored
// past the caches; 72 us through them).
template <int HD, bool F16>
__global__ __launch_bounds__(WG) void kv8_read_kernel(Kv8ReadArgs a) {
    __shared__ __attribute__((aligned(16))) uint32_t tile[HD][T / 4 + 1];
    const int tid = threadIdx.x, kvh = blockIdx.y, which = blockIdx.z, end = a.slot0 + a.n;
    const int unit = a.slot0 / T + (int)blockIdx.x;
    const int8_t *ep = (which ? a.c.ve : a.c.ke) + (size_t)kvh * (a.c.cap >> a.c.lb);
    if (which) {
        const uint32_t *vc = (const uint32_t *)(a.c.vc + ((size_t)kvh * (a.c.cap / T) + unit) * HD * T);
#pragma unroll
        for (int k = 0; k < HD * T / 4 / WG; k++) {
            const int i = tid + k * WG;
            tile[i / (T / 4)][i % (T / 4)] = vc[i];
        }
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < HD * T / 4 / WG; k++) {
        const int i = tid + k * WG, r = i / (HD / 4), col = i % (HD / 4), s = unit * T + r;
        if (s < a.slot0 || s >= end) continue;
        const float step = pow2i(kv8_exp(ep[s >> a.c.lb]));
        int c[4];
        if (which) {
#pragma unroll
            for (int e = 0; e < 4; e++) c[e] = ((const int8_t *)&tile[4 * col + e][0])[r];
        } else {
            const uint32_t w = *((const uint32_t *)(a.c.kc + ((size_t)kvh * a.c.cap + s) * HD) + col);
#pragma unroll
            for (int e = 0; e < 4; e++) c[e] = byte_of(w, e);
        }
        const size_t at = ((size_t)kvh * a.n + (s - a.slot0)) * HD + 4 * col;
        const float y[4] = {(float)c[0] * step, (float)c[1] * step, (float)c[2] * step, (float)c[3] * step};
        if constexpr (F16)
            *(u32x2 *)((uint16_t *)a.out[which] + at) =
                u32x2{f2h_top(y[0]) | (uint32_t)f2h_top(y[1]) << 16, f2h_top(y[2]) | (uint32_t)f2h_top(y[3]) << 16};
        else
            __builtin_nontemporal_store(f32x4{y[0], y[1], y[2], y[3]}, (f32x4 *)((float *)a.out[which] + at));
    }
}

// ------------------------------------------------------------- eviction --

constexpr int EV = 1024;  // threads of the selection

// Slot s's mass as an unsigned key of the same order, -0 as 0: infinities are
// 0x007FFFFF and 0xFF800000, NaN is 1.  A slot that stays in any case (the first,
// the last) has a key above them all, one past the end the key 0.
__device__ __forceinline__ uint32_t slot_key(float m, int s, const Kv8EvictArgs &a) {
    const uint32_t b = __float_as_uint(m == 0.f ? 0.f : m);
    uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    k = m == m ? k : 1u;
    k = s < a.first || s >= a.n - a.last ? 0xFFFFFFFFu : k;
    return s < a.n ? k : 0u;
}

// Sum of v over the threads before this one; the total in *all.  ws: EV / 64 words.
__device__ __forceinline__ uint32_t block_before(uint32_t v, uint32_t *ws, uint32_t *all) {
    const int lane = threadIdx.x & (WAVE - 1), wave = threadIdx.x / WAVE;
    uint32_t s = v;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const uint32_t u = __shfl_up(s, o, WAVE);
        if (lane >= o) s += u;
    }
    __syncthreads();  // ws is free
    if (lane == WAVE - 1) ws[wave] = s;
    __syncthreads();
    uint32_t before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < EV / WAVE; w++) {
        const uint32_t t = ws[w];
        before += w < wave ? t : 0u;
        total += t;
    }
    *all = total;
    return s - v + before;
}

// One workgroup per kv head, a thread four neighbouring slots of every 4096.  The
// keep-th largest key is found digit by digit (11, 11 and 10 bits from the top; a
// first digit of the exponent and two more bits spreads the masses over many
// counters) with counts in LDS.  Keys of the first digit's border go to a list in
// LDS, so the other digits need no pass over the slots; only where too many share
// it (more than EV_LIST) they take one each.  Then the slots that stay are counted
// per wave, the counts summed up, and each finds its place; of equal keys at the
// border the lowest slots stay.  Bound by its instructions on one CU, three passes
// over the slots: 27 us for 40960, 9 us for 4096 (three digits with a pass each and
// slots one at a time took 45; the masses held in registers from one pass to the next
// in unrolled loops, 37 and 18: they spill, and the code is fetched for a single use).
constexpr int EV_TILE = 4 * EV, EV_CH = 64, EV_LIST = 8192;  // slots of a chunk; chunks counted at a time; the list
__global__ __launch_bounds__(EV) void kv8_select_kernel(Kv8EvictArgs a) {
    constexpr int NW = EV / WAVE;
    __shared__ uint32_t hist[2048], cnt[EV_CH * NW], tcnt[EV_CH * NW], list[EV_LIST], ws[NW];
    __shared__ uint32_t s_bin, s_left, s_ties, s_listed;
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE, kvh = blockIdx.x;
    const float *mass = a.mass + (size_t)kvh * a.src.cap;
    int32_t *kept = a.kept + (size_t)kvh * a.keep;
    const int chunks = (a.n + EV_TILE - 1) / EV_TILE;
    // f(chunk - ch0, first slot, keys) for the thread's four slots of chunks ch0 .. ch0 + nch - 1
    auto each = [&](int ch0, int nch, auto f) {
        constexpr int B = 4;
        for (int i0 = 0; i0 < nch; i0 += B) {
            f32x4 x[B];
#pragma unroll
            for (int i = 0; i < B; i++)
                x[i] = *(const f32x4 *)(mass + min((ch0 + i0 + i) * EV_TILE + 4 * tid, a.src.cap - 4));
#pragma unroll
            for (int i = 0; i < B; i++) {
                if (i0 + i >= nch) continue;
                const int s = (ch0 + i0 + i) * EV_TILE + 4 * tid;
                uint32_t k[4];
#pragma unroll
                for (int j = 0; j < 4; j++) k[j] = slot_key(x[i][j], s + j, a);
                f(i0 + i, s, k);
            }
        }
    };
    // kept: keys above `border`, and `need` of the `ties` equal to it
    uint32_t border = 0, need = (uint32_t)a.keep, ties = 0, all;
    // the digit of `bits` bits at `sh`: the largest counter with at least `need` keys in it and above
    auto digit = [&](int sh, int bits) {
        __syncthreads();
        const int top = (1 << bits) - 1 - 2 * tid;  // counters in falling order, two a thread
        const uint32_t c0 = top >= 0 ? hist[top] : 0, c1 = top >= 0 ? hist[top - 1] : 0;
        const uint32_t before = block_before(c0 + c1, ws, &all);
        if (before < need && before + c0 >= need) {
            s_bin = (uint32_t)top;
            s_left = need - before;
            s_ties = c0;
        } else if (before + c0 < need && before + c0 + c1 >= need) {
            s_bin = (uint32_t)(top - 1);
            s_left = need - before - c0;
            s_ties = c1;
        }
        __syncthreads();
        border |= s_bin << sh;
        need = s_left;
        ties = s_ties;
        hist[tid] = 0;
        hist[tid + EV] = 0;
        __syncthreads();
    };
    hist[tid] = 0;
    hist[tid + EV] = 0;
    cnt[tid] = 0;
    if (tid == 0) s_listed = 0;
    __syncthreads();
    each(0, chunks, [&](int, int, const uint32_t (&k)[4]) {
#pragma unroll
        for (int j = 0; j < 4; j++) atomicAdd(&hist[k[j] >> 21], 1u);
    });
    digit(21, 11);
    bool counted = false;
    if (chunks <= EV_CH && ties <= EV_LIST) {
        const uint32_t head = border >> 21;
        each(0, chunks, [&](int i, int, const uint32_t (&k)[4]) {
            uint32_t above = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                above += (uint32_t)__popcll(__ballot(k[j] >> 21 > head));
                if (k[j] >> 21 == head) list[atomicAdd(&s_listed, 1u)] = (k[j] & 0x1FFFFFu) << 10 | (uint32_t)(i * NW + wave);
            }
            if (lane == 0) cnt[i * NW + wave] = above;
        });
        __syncthreads();
        const uint32_t listed = s_listed;
        for (uint32_t i = tid; i < listed; i += EV) atomicAdd(&hist[list[i] >> 20], 1u);
        digit(10, 11);
        for (uint32_t i = tid; i < listed; i += EV)
            if (list[i] >> 20 == ((border >> 10) & 0x7FFu)) atomicAdd(&hist[(list[i] >> 10) & 0x3FFu], 1u);
        digit(0, 10);
        counted = ties <= need;
        if (counted)
            for (uint32_t i = tid; i < listed; i += EV)
                if (list[i] >> 10 >= (border & 0x1FFFFFu)) atomicAdd(&cnt[list[i] & 0x3FFu], 1u);
        __syncthreads();
    } else {
        for (int pass = 1; pass < 3; pass++) {
            const int sh = pass == 1 ? 10 : 0, bits = pass == 1 ? 11 : 10;
            const uint32_t head = border >> (sh + bits), mask = (1u << bits) - 1;
            each(0, chunks, [&](int, int, const uint32_t (&k)[4]) {
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (k[j] >> (sh + bits) == head) atomicAdd(&hist[(k[j] >> sh) & mask], 1u);
            });
            digit(sh, bits);
        }
    }
    uint32_t base = 0, tie_base = 0;
    auto before_me = [&](unsigned long long b, uint32_t from) {
        return __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, from));
    };
    auto place = [&](auto ranked) {  // ranked: some of the ties go
        constexpr bool RANK = decltype(ranked)::value;
        for (int ch0 = 0; ch0 < chunks; ch0 += EV_CH) {
            const int nch = min(EV_CH, chunks - ch0);
            if (!counted) {
                each(ch0, nch, [&](int i, int, const uint32_t (&k)[4]) {
                    uint32_t n = 0, t = 0;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        n += (uint32_t)__popcll(__ballot(RANK ? k[j] > border : k[j] >= border));
                        if constexpr (RANK) t += (uint32_t)__popcll(__ballot(k[j] == border));
                    }
                    if (lane == 0) {
                        cnt[i * NW + wave] = n;
                        if constexpr (RANK) tcnt[i * NW + wave] = t;
                    }
                });
                __syncthreads();
            }
            uint32_t mine = tid < nch * NW ? cnt[tid] : 0, tie_all = 0;
            if constexpr (RANK) {
                const uint32_t t = tid < nch * NW ? tcnt[tid] : 0, ranks = tie_base + block_before(t, ws, &tie_all);
                mine += ranks >= need ? 0u : min(t, need - ranks);
                tcnt[tid] = ranks;
            }
            const uint32_t before = base + block_before(mine, ws, &all);
            cnt[tid] = before;
            __syncthreads();
            each(ch0, nch, [&](int i, int s, const uint32_t (&k)[4]) {
                bool on[4];
                if constexpr (RANK) {
                    uint32_t r = tcnt[i * NW + wave];
#pragma unroll
                    for (int j = 0; j < 4; j++) r = before_me(__ballot(k[j] == border), r);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        on[j] = k[j] > border || (k[j] == border && r < need);
                        r += k[j] == border;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) on[j] = k[j] >= border;
                }
                uint32_t at = cnt[i * NW + wave];
#pragma unroll
                for (int j = 0; j < 4; j++) at = before_me(__ballot(on[j]), at);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (on[j] && at < (uint32_t)a.keep) kept[at++] = s + j;
            });
            base += all;
            tie_base += tie_all;
            __syncthreads();  // the counts are free
        }
    };
    if (ties <= need) place(std::integral_constant<bool, false>{});
    else place(std::integral_constant<bool, true>{});
}

// One workgroup per (64 kept slots, kv head, K or V): the codes of the slots in
// `kept`, brought to the exponent that their new block needs (a left shift is
// exact, a right shift rounds half to even; most need none), from registers to
// registers.  K rows are read where they lie, 16 bytes a thread.  Of V a slot is a
// byte column: the lanes of a wave are the 64 slots of one dimension, which lie in
// a few neighbouring 64-byte rows.  Bound by memory: K reads what is kept, V every
// row that holds a kept slot.  21 us for 8192 of 40960 slots of 8 heads of 128
// (with V's tiles brought through LDS 49, four dimensions a wave 27).
template <int HD>
__global__ __launch_bounds__(WG) void kv8_gather_kernel(Kv8EvictArgs a) {
    constexpr int PPR = HD / 16, NP = T * PPR / WG, NV = HD * T / WG;  // K: 16-byte pieces of a row, of a thread; V: bytes of a thread
    __shared__ int slot[T], es[T], mx[T], be[4], up[T];
    const int tid = threadIdx.x;
    const int unit = blockIdx.x, kvh = blockIdx.y, which = blockIdx.z, n = min(T, a.keep - unit * T);
    const int8_t *ep = (which ? a.src.ve : a.src.ke) + (size_t)kvh * (a.src.cap >> a.src.lb);
    if (tid < T) {
        const int s = a.kept[(size_t)kvh * a.keep + unit * T + min(tid, n - 1)];
        slot[tid] = s;
        mx[tid] = 0;
        es[tid] = kv8_exp(ep[s >> a.src.lb]);
        if (tid < n && which == 0) {
            const size_t to = (size_t)kvh * a.dst.cap + unit * T + tid, from = (size_t)kvh * a.src.cap + s;
            a.dst_mass[to] = a.mass[from];
            if (a.dst_pos) a.dst_pos[to] = a.pos[from];
        }
    }
    __syncthreads();
    u32x4 w[NP];
    int8_t v[NV];
    const int vr = tid % T, vd = tid / T;  // V: my slot, my first dimension
    if (which == 0) {
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const int i = tid + k * WG;
            w[k] = *((const u32x4 *)(a.src.kc + ((size_t)kvh * a.src.cap + slot[i / PPR]) * HD) + i % PPR);
        }
#pragma unroll
        for (int k = 0; k < NP; k++) {
            int x = 0;
#pragma unroll
            for (int c = 0; c < 4; c++)
#pragma unroll
                for (int j = 0; j < 4; j++) x = max(x, abs(byte_of(w[k][c], j)));
            atomicMax(&mx[(tid + k * WG) / PPR], x);
        }
    } else {
        const int s = slot[vr];
        const int8_t *from = a.src.vc + ((size_t)kvh * a.src.cap + (s & ~(T - 1))) * HD + vd * T + (s & (T - 1));
#pragma unroll
        for (int k = 0; k < NV; k++) v[k] = from[k * (WG / T) * T];
        int big = 0;
#pragma unroll
        for (int k = 0; k < NV; k++) big = max(big, abs((int)v[k]));
        atomicMax(&mx[vr], big);
    }
    __syncthreads();
    const int B = 1 << a.dst.lb;
    if (tid < T / B && tid * B < n) {
        int e = KV8_EMIN;
        for (int r = tid * B; r < min((tid + 1) * B, n); r++)
            if (mx[r]) e = max(e, es[r] + (31 - __clz(mx[r])) - 6);
        be[tid] = e;
        (which ? a.dst.ve : a.dst.ke)[(size_t)kvh * (a.dst.cap >> a.dst.lb) + ((unit * T) >> a.dst.lb) + tid] = (int8_t)e;
    }
    __syncthreads();
    if (tid < T) up[tid] = tid < n ? es[tid] - be[tid >> a.dst.lb] : 0;
    __syncthreads();
    auto moved = [](int c, int by) { return (int)rintf(ldexpf((float)c, by)); };
    if (which == 0) {
        u32x4 *dst = (u32x4 *)(a.dst.kc + ((size_t)kvh * a.dst.cap + unit * T) * HD);
#pragma unroll
        for (int k = 0; k < NP; k++) {
            const int i = tid + k * WG, by = up[i / PPR];
            if (i / PPR >= n) continue;
            if (by)
#pragma unroll
                for (int c = 0; c < 4; c++)
                    w[k][c] = pack4(moved(byte_of(w[k][c], 0), by), moved(byte_of(w[k][c], 1), by),
                                    moved(byte_of(w[k][c], 2), by), moved(byte_of(w[k][c], 3), by));
            dst[i] = w[k];
        }
        return;
    }
    if (vr >= n) return;
    int8_t *dst = a.dst.vc + ((size_t)kvh * a.dst.cap + unit * T) * HD + vd * T + vr;
    const int by = up[vr];
#pragma unroll
    for (int k = 0; k < NV; k++) dst[k * (WG / T) * T] = (int8_t)(by ? moved(v[k], by) : v[k]);
}

}  // namespace

hipError_t launch_kv8_append(const Kv8AppendArgs &a, hipStream_t st) {
    // with the length on the device the new tokens may begin anywhere in a unit
    const int first = a.past.dev ? T - 1 : a.past.past % T;
    const dim3 grid((unsigned)((first + a.n + T - 1) / T), (unsigned)a.c.n_kv, 2u);
    auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(WG), 0, st, a); };
    if (a.c.hd == 128) a.f16 ? go(kv8_append_kernel<128, true>) : go(kv8_append_kernel<128, false>);
    else if (a.c.hd == 256) a.f16 ? go(kv8_append_kernel<256, true>) : go(kv8_append_kernel<256, false>);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_kv8_read(const Kv8ReadArgs &a, hipStream_t st) {
    const dim3 grid((unsigned)((a.slot0 % T + a.n + T - 1) / T), (unsigned)a.c.n_kv, 2u);
    auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, dim3(WG), 0, st, a); };
    if (a.c.hd == 128) a.f16 ? go(kv8_read_kernel<128, true>) : go(kv8_read_kernel<128, false>);
    else if (a.c.hd == 256) a.f16 ? go(kv8_read_kernel<256, true>) : go(kv8_read_kernel<256, false>);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

hipError_t launch_kv8_evict(const Kv8EvictArgs &a, hipStream_t st) {
    hipLaunchKernelGGL(kv8_select_kernel, dim3((unsigned)a.src.n_kv), dim3(EV), 0, st, a);
    const dim3 grid((unsigned)((a.keep + T - 1) / T), (unsigned)a.src.n_kv, 2u);
    if (a.src.hd == 128) hipLaunchKernelGGL(kv8_gather_kernel<128>, grid, dim3(WG), 0, st, a);
    else if (a.src.hd == 256) hipLaunchKernelGGL(kv8_gather_kernel<256>, grid, dim3(WG), 0, st, a);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}

}  // namespace oi
