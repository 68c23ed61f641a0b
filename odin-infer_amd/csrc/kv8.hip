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
// LDS tile that is read by columns.  Memory bound on prompts.
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
    const int blk = s0 >> a.c.lb, b0 = blk << a.c.lb;
    int8_t *ep = (which ? a.c.ve : a.c.ke) + (size_t)kvh * (a.c.cap >> a.c.lb) + blk;
    int e = exp_for(amax), e_old = e;
    const bool old = b0 < past;  // the block holds earlier slots
    if (old) {
        e_old = kv8_exp(*ep);
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
        const bool whole = s0 >= past && s0 + 16 <= end;
        const bool any = s0 < end && s0 + 16 > past;
        if (any || (requant && s0 < past)) {
            const uint8_t *tb = (const uint8_t *)&tile[16 * wave][0];
#pragma unroll
            for (int k = 0; k < HD / WAVE; k++) {
                const int d = lane + k * WAVE;
                u32x4 *p = (u32x4 *)(a.c.vc + (((size_t)kvh * (a.c.cap / T) + unit) * HD + d) * T + 16 * wave);
                u32x4 w = whole ? u32x4{0u, 0u, 0u, 0u} : *p;
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
                *p = w;
            }
        }
    }
    __syncthreads();  // every wave of the block has read the old exponent
    if (touched && lane == 0 && wave == w0) *ep = (int8_t)e;
}

// One workgroup per (64 slots, kv head, K or V): codes times their block's
// step.  K as it lies, V through an LDS tile read by columns.
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
                u32x2{f2h(y[0]) | (uint32_t)f2h(y[1]) << 16, f2h(y[2]) | (uint32_t)f2h(y[3]) << 16};
        else
            *(float4 *)((float *)a.out[which] + at) = make_float4(y[0], y[1], y[2], y[3]);
    }
}

// ------------------------------------------------------------- eviction --

constexpr int EV = 1024;  // threads of the selection

// a mass as an unsigned key of the same order; NaN below everything, -0 as 0
__device__ __forceinline__ uint32_t mass_key(float m) {
    if (!(m == m)) return 0u;
    const uint32_t b = __float_as_uint(m == 0.f ? 0.f : m);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// inclusive scan of one value per thread over the workgroup; total in *sum
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t *ws, uint32_t *sum) {
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
#pragma unroll
    for (int o = 1; o < WAVE; o <<= 1) {
        const uint32_t u = __shfl_up(v, o, WAVE);
        if (lane >= o) v += u;
    }
    __syncthreads();  // ws is free
    if (lane == WAVE - 1) ws[wave] = v;
    __syncthreads();
    uint32_t before = 0, all = 0;
    for (int w = 0; w < EV / WAVE; w++) {
        const uint32_t t = ws[w];
        if (w < wave) before += t;
        all += t;
    }
    *sum = all;
    return v + before;
}

// One workgroup per kv head.  The m-th largest key of the middle slots is found
// digit by digit (8 bits, from the top) with a histogram in LDS; then every
// thread walks a run of slots of its own, and two scans give the ties before it
// (the lowest slots of them are kept) and its first place in the list.
__global__ __launch_bounds__(EV) void kv8_select_kernel(Kv8EvictArgs a) {
    __shared__ uint32_t hist[256], ws[EV / WAVE];
    __shared__ uint32_t s_prefix, s_need;
    const int tid = threadIdx.x, kvh = blockIdx.x;
    const float *mass = a.mass + (size_t)kvh * a.src.cap;
    const int lo = a.first, hi = a.n - a.last;  // the middle
    const uint32_t m = (uint32_t)(a.keep - a.first - a.last);
    uint32_t prefix = 0, need = m;
    if (m > 0 && (uint32_t)(hi - lo) > m) {
        for (int digit = 3; digit >= 0; digit--) {
            const int sh = 8 * digit;
            for (int i = tid; i < 256; i += EV) hist[i] = 0;
            __syncthreads();
            for (int s = lo + tid; s < hi; s += EV) {
                const uint32_t k = mass_key(mass[s]);
                if (digit == 3 || (k >> (sh + 8)) == (prefix >> (sh + 8))) atomicAdd(&hist[(k >> sh) & 255u], 1u);
            }
            __syncthreads();
            if (tid == 0) {
                uint32_t left = need;
                int b = 255;
                while (b > 0 && hist[b] < left) left -= hist[b--];
                s_prefix = prefix | (uint32_t)b << sh;
                s_need = left;
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_need;  // of the keys equal to the prefix so far, how many
        }
    } else if (m > 0) {  // all of the middle
        prefix = 0;
        need = 0xFFFFFFFFu;
    } else {
        prefix = 0xFFFFFFFFu;
        need = 0;
    }
    // a key above the prefix is kept, `need` of those equal to it
    const int per = (a.n + EV - 1) / EV, b0 = min(tid * per, a.n), b1 = min(b0 + per, a.n);
    uint32_t above = 0, ties = 0;
    for (int s = b0; s < b1; s++) {
        if (s < lo || s >= hi) {
            above++;
            continue;
        }
        const uint32_t k = mass_key(mass[s]);
        if (k > prefix) above++;
        else if (k == prefix) ties++;
    }
    uint32_t sum;
    uint32_t before = block_scan(ties, ws, &sum) - ties;
    const uint32_t mine = before >= need ? 0u : min(ties, need - before);
    uint32_t at = block_scan(above + mine, ws, &sum) - (above + mine);
    uint32_t left = mine;
    for (int s = b0; s < b1; s++) {
        bool keep = s < lo || s >= hi;
        if (!keep) {
            const uint32_t k = mass_key(mass[s]);
            if (k > prefix) keep = true;
            else if (k == prefix && left > 0) {
                keep = true;
                left--;
            }
        }
        if (keep && at < (uint32_t)a.keep) a.kept[(size_t)kvh * a.keep + at++] = s;
    }
}

// One workgroup per (64 kept slots, kv head, K or V): codes of the slots in
// `kept`, brought to the exponent that their new block needs (a left shift is
// exact, a right shift rounds half to even).  K rows are read where they lie; of
// V the source tiles between the first and the last slot come through LDS, since
// a slot is a byte column of its tile.
template <int HD>
__global__ __launch_bounds__(WG) void kv8_gather_kernel(Kv8EvictArgs a) {
    constexpr int PR = T + 4;
    __shared__ __attribute__((aligned(16))) int8_t in[HD * PR];   // a source V tile
    __shared__ __attribute__((aligned(16))) int8_t out[HD * PR];  // gathered codes [dim][slot]
    __shared__ int slot[T], need[T];
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const int unit = blockIdx.x, kvh = blockIdx.y, which = blockIdx.z, n = min(T, a.keep - unit * T);
    const int32_t *kept = a.kept + (size_t)kvh * a.keep + unit * T;
    if (tid < T) {
        const int s = kept[min(tid, n - 1)];
        slot[tid] = s;
        if (tid < n && which == 0) {
            const size_t to = (size_t)kvh * a.dst.cap + unit * T + tid, from = (size_t)kvh * a.src.cap + s;
            a.dst_mass[to] = a.mass[from];
            if (a.dst_pos) a.dst_pos[to] = a.pos[from];
        }
    }
    __syncthreads();
    const int8_t *ep = (which ? a.src.ve : a.src.ke) + (size_t)kvh * (a.src.cap >> a.src.lb);
    if (which == 0) {
        // a wave per row
        constexpr int CPL = HD / WAVE;  // codes per lane
        for (int r = wave; r < n; r += WG / WAVE) {
            const int8_t *row = a.src.kc + ((size_t)kvh * a.src.cap + slot[r]) * HD + CPL * lane;
            int mx = 0;
#pragma unroll
            for (int i = 0; i < CPL; i++) {
                const int c = row[i];
                out[r * HD + CPL * lane + i] = (int8_t)c;
                mx = max(mx, c < 0 ? -c : c);
            }
            mx = (int)wave_max_all((float)mx);
            if (lane == 0) need[r] = mx ? kv8_exp(ep[slot[r] >> a.src.lb]) + (31 - __clz(mx)) - 6 : KV8_EMIN;
        }
    } else {
        const int t0 = slot[0] / T, t1 = slot[n - 1] / T;
        for (int t = t0; t <= t1; t++) {
            const u32x4 *src = (const u32x4 *)(a.src.vc + ((size_t)kvh * (a.src.cap / T) + t) * HD * T);
            __syncthreads();  // the previous tile has been read
            for (int i = tid; i < HD * T / 16; i += WG) {
                const u32x4 w = src[i];
                uint32_t *p = (uint32_t *)(in + (i / 4) * PR + (i % 4) * 16);
#pragma unroll
                for (int c = 0; c < 4; c++) p[c] = w[c];
            }
            __syncthreads();
            for (int i = tid; i < HD * T; i += WG) {
                const int d = i / T, r = i % T, s = slot[r];
                if (r < n && s / T == t) out[d * PR + r] = in[d * PR + s % T];
            }
        }
        __syncthreads();
        if (tid < n) {
            int mx = 0;
            for (int d = 0; d < HD; d++) {
                const int c = out[d * PR + tid];
                mx = max(mx, c < 0 ? -c : c);
            }
            need[tid] = mx ? kv8_exp(ep[slot[tid] >> a.src.lb]) + (31 - __clz(mx)) - 6 : KV8_EMIN;
        }
    }
    __syncthreads();
    __shared__ int be[4];
    const int B = 1 << a.dst.lb;
    if (tid < T / B) {
        int e = KV8_EMIN;
        for (int r = tid * B; r < min((tid + 1) * B, n); r++) e = max(e, need[r]);
        be[tid] = e;
        if (tid * B < n)
            (which ? a.dst.ve : a.dst.ke)[(size_t)kvh * (a.dst.cap >> a.dst.lb) + ((unit * T) >> a.dst.lb) + tid] =
                (int8_t)e;
    }
    __syncthreads();
    for (int i = tid; i < HD * T; i += WG) {
        const int r = which ? i % T : i / HD, d = which ? i / T : i % HD;
        if (r >= n) continue;
        const int c = which ? out[d * PR + r] : out[i];
        const int up = kv8_exp(ep[slot[r] >> a.src.lb]) - be[r >> a.dst.lb];
        const int8_t v = (int8_t)rintf(ldexpf((float)c, up));
        if (which) a.dst.vc[(((size_t)kvh * (a.dst.cap / T) + unit) * HD + d) * T + r] = v;
        else a.dst.kc[((size_t)kvh * a.dst.cap + unit * T + r) * HD + d] = v;
    }
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
