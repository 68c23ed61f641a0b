// paged.hip -- pages of a pool given to sequences and taken back, the slots of
// packed rows, and the append of their K and V.

#include "device_common.h"
#include "paged.h"

namespace oi {

namespace {

constexpr int PW = 1024;  // threads of the planning workgroup, sequences that it takes at a time

// Sum over the lanes up to each (below 2^32).
__device__ __forceinline__ uint32_t scan_lanes(uint32_t v) {
#define OI_SCAN(ctrl, rows) v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, rows, 0xF, false)
    OI_SCAN(0x111, 0xF);  // rows of 16: 1, 2, 4, 8 lanes back
    OI_SCAN(0x112, 0xF);
    OI_SCAN(0x114, 0xF);
    OI_SCAN(0x118, 0xF);
    OI_SCAN(0x142, 0xA);  // the last lane of rows 0 and 2 to the row behind
    OI_SCAN(0x143, 0xC);  // lane 31 to rows 2 and 3
#undef OI_SCAN
    return v;
}
// Sum over the workgroup's threads (PW of them, below 2^25 each) up to each, and the total.
__device__ __forceinline__ int64_t scan_add(uint32_t x, uint32_t *lds, int64_t &total) {
    const int tid = threadIdx.x, lane = tid & (WAVE - 1), wave = tid / WAVE;
    const uint32_t v = scan_lanes(x);
    __syncthreads();  // the previous use of lds is complete
    if (lane == WAVE - 1) lds[wave] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PW / WAVE; w++) {
        const int64_t y = lds[w];
        before += w < wave ? y : 0;
        total += y;
    }
    return v + before;
}

// the last i < n with p[i] <= x (p rising, p[0] <= x)
__device__ __forceinline__ int last_le(const int *p, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int pages_of(int slots, int lp) { return (int)(((int64_t)slots + (1 << lp) - 1) >> lp); }
// slot number of offset `off` of a page; a page that the pool does not have gives none
__device__ __forceinline__ int slot_of(int page, int off, int lp, int n_pages) {
    return (uint32_t)page < (uint32_t)n_pages ? (page << lp) + off : -1;
}

// One workgroup: sequences PW at a time, a thread each, with running sums of rows
// and pages; then the pages of these sequences, and (MAPS) their rows, over all
// threads, the owner by bisection of the sums in LDS.  The n-th page taken is
// the list's n-th from its end.  A page of a row that is new here is looked up in
// the list, not in the table that another thread writes.  A step of 61 sequences 4.4
// us (a release of them 2.7): a chain of one load, two scans and two searches.
template <bool MAPS>
__global__ __launch_bounds__(PW) void paged_plan_kernel(PagedPlanArgs a) {
    __shared__ uint32_t red[PW / WAVE];
    __shared__ int need0[PW], row0[PW], before[PW], past0[PW], lives[PW], taken_by[PW / WAVE];
    const int tid = threadIdx.x, P = 1 << a.lp;
    const int n_free = min(max(*a.n_free, 0), a.n_pages);
    int64_t rows = 0, pages = 0;  // of the sequences so far
    int taken = 0;
    if (tid == 0) a.starts[0] = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += PW) {
        const int s = s0 + tid, m = min(PW, a.n_seqs - s0);
        const bool real = s < a.n_seqs;
        // more than all rows is as good as one more
        const int past = real ? a.past[s] : 0, fresh = real ? min(max(a.fresh[s], 0), a.n_rows + 1) : 0;
        int64_t all, all_pages;
        const int64_t end = rows + scan_add((uint32_t)fresh, red, all);
        const bool fits = real && past >= 0 && end <= a.n_rows && (int64_t)past + fresh <= (int64_t)a.stride << a.lp;
        const int have = fits ? pages_of(past, a.lp) : 0, need = fits ? pages_of(past + fresh, a.lp) - have : 0;
        const int64_t run = pages + scan_add((uint32_t)need, red, all_pages);
        const bool given = fits && (need == 0 || run <= n_free);
        // given needs are the first of the sum: a place in the list is the sum before, less what went
        // before these sequences
        need0[tid] = (int)min(run - need - pages, (int64_t)INT32_MAX);
        row0[tid] = (int)min(end - fresh, (int64_t)a.n_rows);
        before[tid] = have;
        past0[tid] = past;
        lives[tid] = given;
        const int mine = given && need ? (int)(run - pages) : 0;
        const unsigned long long takers = __ballot(mine > 0);
        const int last = takers ? __builtin_amdgcn_readlane(mine, 63 - __clzll(takers)) : 0;
        if ((tid & (WAVE - 1)) == 0) taken_by[tid / WAVE] = last;
        if (real) {
            a.lens[s] = given ? past + fresh : 0;
            a.starts[s + 1] = (int)min(end, (int64_t)a.n_rows);
        }
        __syncthreads();
        int got = 0;
#pragma unroll
        for (int w = 0; w < PW / WAVE; w++) got = max(got, taken_by[w]);
        const int top = n_free - 1 - taken;
        for (int k = tid; k < got; k += PW) {
            const int i = last_le(need0, m, k);
            a.table[(int64_t)(s0 + i) * a.stride + before[i] + k - need0[i]] = a.free_pages[top - k];
        }
        if constexpr (MAPS) {
            const int r1 = (int)min(rows + all, (int64_t)a.n_rows);
            for (int r = (int)min(rows, (int64_t)a.n_rows) + tid; r < r1; r += PW) {
                const int i = last_le(row0, m, r), j = past0[i] + r - row0[i];
                int slot = -1;
                if (lives[i]) {
                    const int pi = j >> a.lp;
                    const int page = pi < before[i] ? a.table[(int64_t)(s0 + i) * a.stride + pi]
                                                    : a.free_pages[top - (need0[i] + pi - before[i])];
                    slot = slot_of(page, j & (P - 1), a.lp, a.n_pages);
                }
                a.slots[r] = slot;
                if (a.pos)
                    for (int x = 0; x < 3; x++) a.pos[(int64_t)x * a.n_rows + r] = lives[i] ? j : 0;
            }
        }
        rows += all;
        pages += all_pages;
        taken += got;
        __syncthreads();  // the sums are read before the next sequences' are written
    }
    if constexpr (MAPS)
        for (int r = (int)min(rows, (int64_t)a.n_rows) + tid; r < a.n_rows; r += PW) {
            a.slots[r] = -1;
            if (a.pos)
                for (int x = 0; x < 3; x++) a.pos[(int64_t)x * a.n_rows + r] = 0;
        }
    if (tid == 0) *a.n_free = n_free - taken;  // every thread has read it before the first barrier
}

// The rows' maps from the sequences' starts, lengths and pages, a row a thread: a bisection's
// chain of cached loads, 4.3 us for 28700 rows of 300 sequences, with the plan's 3.9; the plan's one
// workgroup takes 29.7 for both.
__global__ __launch_bounds__(WG) void paged_maps_kernel(PagedPlanArgs a) {
    const int r = blockIdx.x * WG + threadIdx.x;
    if (r >= a.n_rows) return;
    const int s = last_le(a.starts, a.n_seqs + 1, r);  // n_seqs: behind the last row
    int slot = -1, j = 0;
    if (s < a.n_seqs && a.lens[s] > 0) {
        j = a.lens[s] - a.starts[s + 1] + r;
        slot = slot_of(a.table[(int64_t)s * a.stride + (j >> a.lp)], j & ((1 << a.lp) - 1), a.lp, a.n_pages);
    }
    a.slots[r] = slot;
    if (a.pos)
        for (int x = 0; x < 3; x++) a.pos[(int64_t)x * a.n_rows + r] = j;
}

// Pages behind the first keep slots of each sequence go back on the list, in such
// an order that a release of what the last plan took leaves the list as it was.
__global__ __launch_bounds__(PW) void paged_release_kernel(PagedReleaseArgs a) {
    __shared__ uint32_t red[PW / WAVE];
    __shared__ int sum0[PW], first[PW];
    const int tid = threadIdx.x;
    const int n_free = min(max(*a.n_free, 0), a.n_pages);
    auto span = [&](int s, int &from) {
        const int most = (int)min((int64_t)a.stride << a.lp, (int64_t)INT32_MAX);
        const int held = min(max(a.held[s], 0), most), keep = a.keep ? min(max(a.keep[s], 0), held) : 0;
        from = pages_of(keep, a.lp);
        return pages_of(held, a.lp) - from;
    };
    int64_t total = 0;
    if (a.n_seqs > PW) {
        for (int s0 = 0; s0 < a.n_seqs; s0 += PW) {
            int from;
            int64_t some;
            scan_add(s0 + tid < a.n_seqs ? (uint32_t)span(s0 + tid, from) : 0u, red, some);
            total += some;
        }
    }
    int64_t done = 0;
    for (int s0 = 0; s0 < a.n_seqs; s0 += PW) {
        const int s = s0 + tid, m = min(PW, a.n_seqs - s0);
        int from = 0, all = 0;
        if (s < a.n_seqs) all = span(s, from);
        int64_t got;
        const int64_t mine = scan_add((uint32_t)all, red, got);
        if (a.n_seqs <= PW) total = got;
        if (n_free + total > a.n_pages) return;  // more than the pool has: nothing is released
        sum0[tid] = (int)min(mine - all, (int64_t)INT32_MAX);
        first[tid] = from;
        __syncthreads();
        for (int k = tid; k < (int)got; k += PW) {
            const int i = last_le(sum0, m, k);
            a.free_pages[n_free + total - 1 - done - k] = a.table[(int64_t)(s0 + i) * a.stride + first[i] + k - sum0[i]];
        }
        done += got;
        __syncthreads();
    }
    if (tid == 0) *a.n_free = n_free + (int)total;
}

// Values as the cache holds them: nothing infinite, no NaN, so that a weight of 0
// always gives 0 times a slot's value.
__device__ __forceinline__ uint32_t stored(float x) {
    return f2h(x != x ? 0.f : __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f));
}

constexpr int APPEND_T = 8, APPEND_E = 512;  // packed rows and elements of a workgroup

// A workgroup takes 8 packed rows and 512 of their elements.  K: a wave per row,
// 16-byte stores.  V lies in eights of slots: rows whose slots are neighbours in one
// eight (a run, found from the slots alone) are written together, a whole run as one
// 16-byte piece per dimension; it belongs to the workgroup of its first row.  8353 f16
// rows of 8 heads of 128 17 us: 4.0 TB/s behind a launch's ramp, where a large copy makes 4.7.
template <bool F16>
__global__ __launch_bounds__(WG, 4) void paged_append_kernel(PagedAppendArgs a) {
    constexpr int NR = 2 * APPEND_T - 1;
    const int t0 = blockIdx.x * APPEND_T, e0 = blockIdx.y * APPEND_E, tid = threadIdx.x, lane = tid & (WAVE - 1);
    const int wave = __builtin_amdgcn_readfirstlane(tid / WAVE);
    const int row = a.c.n_kv * a.c.hd, lh = a.c.hd == 128 ? 7 : 8, P = 1 << a.c.lp;
    const int64_t most = (int64_t)a.c.n_pages << a.c.lp;
    // slots of the rows t0 - 1 .. t0 + 14
    int slot[NR + 1];
#pragma unroll
    for (int i = 0; i <= NR; i++) {
        const int t = t0 - 1 + i;
        slot[i] = t >= 0 && t < a.n ? a.slots[t] : -1;
        if (slot[i] >= most) slot[i] = -1;
    }
    const int ek = e0 + 8 * lane;
    if (ek < row) {
        uint16_t *kb = a.c.k + ((size_t)(ek >> lh) << a.c.lp) * a.c.hd + (ek & (a.c.hd - 1));
        u32x4 w[2][F16 ? 1 : 2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const int64_t t = min(t0 + wave + 4 * i, a.n - 1);
#pragma unroll
            for (int j = 0; j < (F16 ? 1 : 2); j++)
                w[i][j] = F16 ? *(const u32x4 *)((const uint16_t *)a.x[0] + t * a.stride[0] + ek)
                              : *(const u32x4 *)((const float *)a.x[0] + t * a.stride[0] + ek + 4 * j);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            int s = -1;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (wave == k) s = slot[1 + k + 4 * i];
            if (s < 0) continue;
            u32x4 h;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float lo, hi;
                if constexpr (F16) {
                    const uint32_t b = w[i][0][j];
                    lo = h2f(b & 0xFFFFu);
                    hi = h2f(b >> 16);
                } else {
                    const uint32_t bl = w[i][j / 2][2 * (j & 1)], bh = w[i][j / 2][2 * (j & 1) + 1];
                    lo = __uint_as_float(bl);
                    hi = __uint_as_float(bh);
                }
                h[j] = stored(lo) | stored(hi) << 16;
            }
            *(u32x4 *)(kb + (((size_t)(s >> a.c.lp) * a.c.n_kv << a.c.lp) + (s & (P - 1))) * a.c.hd) = h;
        }
    }
    const int ev = e0 + 2 * tid;
    if (ev >= row) return;
    uint32_t x[NR];  // two dimensions of a row each
    uint32_t raw[NR][F16 ? 1 : 2] = {};
#pragma unroll
    for (int i = 0; i < NR; i++) {
        const int t = min(t0 + i, a.n - 1);
        // this workgroup's rows at once, those past them only where they go on a run
        if (i >= APPEND_T && (slot[i + 1] < 0 || (slot[i + 1] & 7) == 0 || (slot[i + 1] & 7) < i - APPEND_T + 1)) continue;
        if constexpr (F16) {
            raw[i][0] = *(const uint32_t *)((const uint16_t *)a.x[1] + t * a.stride[1] + ev);
        } else {
            const u32x2 f = *(const u32x2 *)((const float *)a.x[1] + t * a.stride[1] + ev);
            raw[i][0] = f.x;
            raw[i][1] = f.y;
        }
    }
#pragma unroll
    for (int i = 0; i < NR; i++) {
        float lo, hi;
        if constexpr (F16) {
            lo = h2f(raw[i][0] & 0xFFFFu);
            hi = h2f(raw[i][0] >> 16);
        } else {
            lo = __uint_as_float(raw[i][0]);
            hi = __uint_as_float(raw[i][1]);
        }
        x[i] = stored(lo) | stored(hi) << 16;
    }
    uint16_t *vb = a.c.v + ((size_t)(ev >> lh) << a.c.lp) * a.c.hd + (size_t)(ev & (a.c.hd - 1)) * 8;
#pragma unroll
    for (int i = 0; i < APPEND_T; i++) {
        const int s = slot[i + 1];
        // the first row of a run: it opens an eight, or the row before is not its neighbour
        if (s < 0 || ((s & 7) != 0 && slot[i] == s - 1)) continue;
        uint16_t *p = vb + (((size_t)(s >> a.c.lp) * a.c.n_kv << a.c.lp) + (s & (P - 1) & ~7)) * a.c.hd;
        int len = 1;
#pragma unroll
        for (int k = 1; k < 8; k++)
            if (len == k && ((s + k) & 7) != 0 && slot[i + 1 + k] == s + k) len++;
        if (len == 8) {
            u32x4 d0, d1;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                d0[k] = (x[i + 2 * k] & 0xFFFFu) | x[i + 2 * k + 1] << 16;
                d1[k] = x[i + 2 * k] >> 16 | (x[i + 2 * k + 1] & 0xFFFF0000u);
            }
            *(u32x4 *)p = d0;
            *(u32x4 *)(p + 8) = d1;
        } else {
#pragma unroll
            for (int k = 0; k < 7; k++)
                if (k < len) {
                    p[(s & 7) + k] = (uint16_t)x[i + k];
                    p[(s & 7) + k + 8] = (uint16_t)(x[i + k] >> 16);
                }
        }
    }
}

// Few elements: a row a workgroup, four elements a thread, V's by 2-byte stores; the slot and the
// values are one round trip.  us (by runs), rows one of each sequence and neighbours in one, heads of 128 in f16, f32 within
// a tenth of them:
//   1 head    600 rows 2.8 (6.2), 2.9 (4.4)    1500 rows 3.7 (6.5), 3.7 (4.5)
//   2 heads   600 3.5 (6.4), 3.5 (4.7)         1500 5.2 (7.2), 5.1 (4.5)
//   8         256 4.4 (7.0), 4.1 (5.5)         300 4.8 (7.1), 4.8 (4.5)      600 7.3 (8.3), 6.9 (5.8)
//   16        64 3.6 (6.5), 3.6 (5.5)          256 6.6 (8.3), 6.0 (5.7)      600 12.0 (11.3), 11.2 (6.8)
//   32        64 4.1 (7.0), 4.6 (5.6)          256 11.2 (9.6), 9.8 (6.0)
constexpr int64_t APPEND_FEW = 1 << 18;  // elements of K
template <bool F16>
__global__ __launch_bounds__(WG) void paged_append_row_kernel(PagedAppendArgs a) {
    const int t = blockIdx.x, e = (blockIdx.y * WG + threadIdx.x) * 4;
    const int row = a.c.n_kv * a.c.hd, lh = a.c.hd == 128 ? 7 : 8, P = 1 << a.c.lp;
    if (e >= row) return;
    const int s = a.slots[t];
    uint32_t h[2][4];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        if constexpr (F16) {
            const u32x2 x = *(const u32x2 *)((const uint16_t *)a.x[w] + (int64_t)t * a.stride[w] + e);
#pragma unroll
            for (int i = 0; i < 4; i++) h[w][i] = stored(h2f((i < 2 ? x.x : x.y) >> 16 * (i & 1) & 0xFFFFu));
        } else {
            const float4 x = *(const float4 *)((const float *)a.x[w] + (int64_t)t * a.stride[w] + e);
            h[w][0] = stored(x.x);
            h[w][1] = stored(x.y);
            h[w][2] = stored(x.z);
            h[w][3] = stored(x.w);
        }
    }
    if (s < 0 || s >= (int64_t)a.c.n_pages << a.c.lp) return;
    const size_t head = (((size_t)(s >> a.c.lp) * a.c.n_kv + (e >> lh)) << a.c.lp) * a.c.hd;
    const int off = s & (P - 1), d = e & (a.c.hd - 1);
    *(u32x2 *)(a.c.k + head + (size_t)off * a.c.hd + d) = u32x2{h[0][0] | h[0][1] << 16, h[0][2] | h[0][3] << 16};
    uint16_t *v = a.c.v + head + (size_t)(off & ~7) * a.c.hd + d * 8 + (off & 7);
#pragma unroll
    for (int i = 0; i < 4; i++) v[8 * i] = (uint16_t)h[1][i];
}

}  // namespace

hipError_t launch_paged_plan(const PagedPlanArgs &a, hipStream_t st) {
    // one launch while the rows are few passes of the one workgroup; a second one takes 4 us
    if (a.n_rows <= 4096) {
        hipLaunchKernelGGL(paged_plan_kernel<true>, dim3(1), dim3(PW), 0, st, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(paged_plan_kernel<false>, dim3(1), dim3(PW), 0, st, a);
    hipLaunchKernelGGL(paged_maps_kernel, dim3((unsigned)((a.n_rows + WG - 1) / WG)), dim3(WG), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_paged_release(const PagedReleaseArgs &a, hipStream_t st) {
    hipLaunchKernelGGL(paged_release_kernel, dim3(1), dim3(PW), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t st) {
    if ((int64_t)a.n * a.c.n_kv * a.c.hd <= APPEND_FEW) {
        const dim3 grid((unsigned)a.n, (unsigned)((a.c.n_kv * a.c.hd + 4 * WG - 1) / (4 * WG)));
        if (a.f16) hipLaunchKernelGGL(paged_append_row_kernel<true>, grid, dim3(WG), 0, st, a);
        else hipLaunchKernelGGL(paged_append_row_kernel<false>, grid, dim3(WG), 0, st, a);
        return hipGetLastError();
    }
    const dim3 grid((unsigned)((a.n + APPEND_T - 1) / APPEND_T), (unsigned)((a.c.n_kv * a.c.hd + APPEND_E - 1) / APPEND_E));
    if (a.f16) hipLaunchKernelGGL(paged_append_kernel<true>, grid, dim3(WG), 0, st, a);
    else hipLaunchKernelGGL(paged_append_kernel<false>, grid, dim3(WG), 0, st, a);
    return hipGetLastError();
}

}  // namespace oi
