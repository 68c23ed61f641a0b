// paged.cpp -- C entries of the paged f16 K/V cache: argument checks, the parts of a
// pool, launches (paged.hip, paged_attn.hip).  Nothing here allocates device memory or
// waits for the device, so every launch can be captured into a graph.
#include "paged.h"

#include <algorithm>
#include <cmath>
#include <string>

#include "entry_checks.h"
#include "oi.h"
#include "oi_kernels.h"

using namespace oi;

namespace {

constexpr int32_t MAX_SEQS = 65536;
constexpr int32_t MAX_TOKENS = 1 << 24;  // rows of a call
constexpr int32_t MAX_DRAFT = 16;        // tokens of a sequence in one tokens call

int log2_page(const oi_paged_dims *d) { return d->page == 16 ? 4 : d->page == 32 ? 5 : 6; }
bool dims_ok(const oi_paged_dims *d) {
    return d && d->n_kv_heads > 0 && d->n_kv_heads <= 1024 && (d->head_dim == 128 || d->head_dim == 256) &&
           (d->page == 16 || d->page == 32 || d->page == 64) && d->n_pages > 0 &&
           d->n_pages <= (1 << 28) / d->page;
}
const char *const BAD_DIMS = "bad dims (head_dim 128 or 256, page 16, 32 or 64, n_pages * page at most 2^28)";

Paged parts(const oi_paged_dims *d, const void *cache) {
    Paged c{};
    c.n_kv = d->n_kv_heads;
    c.hd = d->head_dim;
    c.n_pages = d->n_pages;
    c.lp = log2_page(d);
    c.k = (uint16_t *)const_cast<void *>(cache);
    c.v = c.k + (size_t)d->n_pages * d->n_kv_heads * d->page * d->head_dim;
    return c;
}

bool ints_ok(std::initializer_list<const void *> ps) {
    return std::all_of(ps.begin(), ps.end(), [](const void *p) { return aligned(p, 4); });
}
// the first `n_out` of the spans share no memory with each other or with the others
bool apart(std::initializer_list<Span> spans, int n_out) {
    int i = 0;
    for (const Span &o : spans) {
        if (i == n_out) break;
        int j = 0;
        for (const Span &s : spans)
            if (j++ > i && overlap(o, s)) return false;
        i++;
    }
    return true;
}
// a table: n_seqs rows of n_entries
int table_ok(int32_t n_seqs, int32_t stride, const char *what) {
    if (n_seqs <= 0 || n_seqs > MAX_SEQS) return err(OI_E_RANGE, what, "n_seqs outside 1 .. 65536");
    if (stride <= 0 || stride > (1 << 24)) return err(OI_E_RANGE, what, "a table's row has 1 .. 2^24 entries");
    return OI_OK;
}

bool heads_ok(const oi_paged_dims *d, int32_t n_heads) {
    return n_heads > 0 && n_heads <= 4096 && n_heads % d->n_kv_heads == 0;
}

// A call's workspace: borders, (m, l) and results of partial tiles, each 16-byte aligned.
struct Workspace {
    int workers, part_rows;
    size_t ml, part, bytes;
};
Workspace workspace(int workers, int part_rows, int hd) {
    Workspace w;
    w.workers = workers;
    w.part_rows = part_rows;
    w.ml = ((size_t)workers + 1) * sizeof(PagedAt);
    w.part = (w.ml + (size_t)workers * 2 * part_rows * sizeof(float2) + 15) / 16 * 16;
    w.bytes = w.part + (size_t)workers * 2 * part_rows * hd * sizeof(float);
    return w;
}
bool tokens_fit(int32_t n_seqs, int32_t n_q) {
    return n_seqs > 0 && n_seqs <= MAX_SEQS && n_q > 0 && n_q <= MAX_DRAFT;
}
Workspace tokens_workspace(const oi_paged_dims *d, int32_t n_heads, int32_t n_q, bool f16) {
    const int rows = n_q * (n_heads / d->n_kv_heads);
    if (rows > PAGED_TOKENS_ROWS)
        return workspace(paged_prompts_workers(d->head_dim, f16), std::min(paged_prompts_rows(), rows), d->head_dim);
    return workspace(paged_tokens_workers(d->head_dim), rows, d->head_dim);
}
bool prompts_fit(const oi_paged_dims *d, int32_t n_heads, int32_t n_seqs, int32_t n_rows) {
    const int64_t g = n_heads / d->n_kv_heads;
    return n_seqs > 0 && n_seqs <= MAX_SEQS && n_rows > 0 && n_rows <= MAX_TOKENS && n_rows * g * g < ((int64_t)1 << 32);
}
Workspace prompts_workspace(const oi_paged_dims *d, int32_t n_heads, int32_t n_rows, bool f16) {
    return workspace(paged_prompts_workers(d->head_dim, f16),
                     (int)std::min<int64_t>(paged_prompts_rows(), (int64_t)n_rows * (n_heads / d->n_kv_heads)), d->head_dim);
}

float tile_units(int group) { return (float)paged_prompts_rows() / (64.f * (float)group); }

// What both attention calls have alike.  n_rows: tokens of q and out.
int attention(PagedAttnArgs &a, const char *what, const oi_paged_dims *d, const void *cache, int32_t n_heads, int32_t type,
              const void *q, int64_t q_stride, float scale, int32_t n_seqs, int64_t n_rows, const int32_t *starts,
              const int32_t *lens, const int32_t *table, int32_t stride, void *out, int64_t out_stride, void *ws,
              int64_t ws_bytes, const Workspace &w, void *stream) {
    if (int rc = table_ok(n_seqs, stride, what)) return rc;
    if (!cache || !q || !out || !ws || !lens || !table) return err(OI_E_ARG, what, "null argument");
    if (!aligned(cache, 256)) return err(OI_E_ARG, what, "the cache must be 256-byte aligned");
    if (!aligned(ws, 16)) return err(OI_E_ARG, what, "the workspace must be 16-byte aligned");
    if (!ints_ok({starts, lens, table})) return err(OI_E_ARG, what, "misaligned starts, lens or table");
    const float scale2 = (float)((double)scale * 1.4426950408889634);  // exponents are formed in base 2
    if (!std::isfinite(scale2)) return err(OI_E_ARG, what, "scale (times log2 e) is not finite");
    const int64_t row = (int64_t)n_heads * d->head_dim;
    if (!rows_ok(q, type, q_stride, row) || !rows_ok(out, type, out_stride, row)) return err(OI_E_ARG, what, BAD_ROWS);
    if (out == q && q_stride != out_stride) return err(OI_E_ARG, what, "out may be q only with the same stride");
    if (ws_bytes < (int64_t)w.bytes)
        return err(OI_E_ARG, what, "workspace of " + std::to_string(ws_bytes) + " bytes, " + std::to_string(w.bytes) +
                                       " needed");
    const int64_t group = n_heads / d->n_kv_heads, cap = (int64_t)stride * d->page;
    const int64_t es = size_of(type);
    const Span qs{q, row * es, n_rows, q_stride * es}, os{out, row * es, n_rows, out_stride * es}, wsp{ws, (int64_t)w.bytes},
        all{cache, oi_paged_bytes(d)}, ls{lens, (int64_t)n_seqs * 4}, ts{table, (int64_t)n_seqs * stride * 4},
        ss{starts, ((int64_t)n_seqs + 1) * 4};
    if (!apart({os, wsp, all, ls, ts, ss}, 2) || overlap(wsp, qs) || (out != q && overlap(os, qs)))
        return err(OI_E_ARG, what, "out or workspace overlaps another argument");
    if (int rc = stream_ok(stream, what)) return rc;
    a.c = parts(d, cache);
    a.q = q;
    a.out = out;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.scale = scale2;
    a.f16 = type == OI_TYPE_F16;
    a.group = (int)group;
    a.magic = group > 1 ? (uint32_t)((((uint64_t)1 << 32) + group - 1) / group) : 0u;
    a.n_seqs = n_seqs;
    a.n_rows = (int)n_rows;
    a.starts = starts;
    a.lens = lens;
    a.table = table;
    a.stride = stride;
    a.cap = (int)std::min<int64_t>(cap, INT32_MAX - 64);  // rounding up to units stays in range
    a.workers = w.workers;
    a.part_rows = w.part_rows;
    a.at = (PagedAt *)ws;
    a.ml = (float2 *)((char *)ws + w.ml);
    a.part = (float *)((char *)ws + w.part);
    return OI_OK;
}

}  // namespace

extern "C" {

int64_t oi_paged_bytes(const oi_paged_dims *d) {
    if (!dims_ok(d)) return 0;
    return ((int64_t)d->n_pages * d->n_kv_heads * d->page * d->head_dim * 4 + 255) / 256 * 256;
}

int oi_paged_plan_launch(const oi_paged_dims *d, int32_t n_seqs, const int32_t *n_past, const int32_t *n_new, int32_t *table,
                         int32_t table_stride, const int32_t *free_pages, int32_t *n_free, int32_t n_rows, int32_t *lens,
                         int32_t *starts, int32_t *slots, int32_t *pos, void *stream) {
    const char *const W = "paged plan";
    return guarded([&]() -> int {
        if (!dims_ok(d)) return err(OI_E_ARG, W, BAD_DIMS);
        if (int rc = table_ok(n_seqs, table_stride, W)) return rc;
        if (n_rows < 0 || n_rows > MAX_TOKENS) return err(OI_E_RANGE, W, "n_rows outside 0 .. 2^24");
        if (!n_past || !n_new || !table || !free_pages || !n_free || !lens || !starts || (n_rows && !slots))
            return err(OI_E_ARG, W, "null argument");
        if (!ints_ok({n_past, n_new, table, free_pages, n_free, lens, starts, slots, pos}))
            return err(OI_E_ARG, W, "misaligned argument");
        const int64_t n = (int64_t)n_seqs * 4, r = (int64_t)n_rows * 4;
        const Span ms{n_rows ? slots : nullptr, r}, ps{n_rows ? pos : nullptr, 3 * r};
        if (!apart({{table, n * table_stride}, {lens, n}, {starts, n + 4}, ms, ps, {n_free, 4}, {free_pages, (int64_t)d->n_pages * 4},
                    {n_past, n}, {n_new, n}}, 6))
            return err(OI_E_ARG, W, "an output overlaps another argument");
        if (int rc = stream_ok(stream, W)) return rc;
        PagedPlanArgs a{};
        a.past = n_past;
        a.fresh = n_new;
        a.table = table;
        a.free_pages = free_pages;
        a.n_free = n_free;
        a.lens = lens;
        a.starts = starts;
        a.slots = slots;
        a.pos = pos;
        a.n_seqs = n_seqs;
        a.stride = table_stride;
        a.n_rows = n_rows;
        a.n_pages = d->n_pages;
        a.lp = log2_page(d);
        return launched(launch_paged_plan(a, (hipStream_t)stream), W);
    });
}

int oi_paged_release_launch(const oi_paged_dims *d, int32_t n_seqs, const int32_t *n_held, const int32_t *n_keep,
                            const int32_t *table, int32_t table_stride, int32_t *free_pages, int32_t *n_free, void *stream) {
    const char *const W = "paged release";
    return guarded([&]() -> int {
        if (!dims_ok(d)) return err(OI_E_ARG, W, BAD_DIMS);
        if (int rc = table_ok(n_seqs, table_stride, W)) return rc;
        if (!n_held || !table || !free_pages || !n_free) return err(OI_E_ARG, W, "null argument");
        if (!ints_ok({n_held, n_keep, table, free_pages, n_free})) return err(OI_E_ARG, W, "misaligned argument");
        const int64_t n = (int64_t)n_seqs * 4;
        if (!apart({{free_pages, (int64_t)d->n_pages * 4}, {n_free, 4}, {n_held, n}, {n_keep, n}, {table, n * table_stride}}, 2))
            return err(OI_E_ARG, W, "the list or its count overlaps another argument");
        if (int rc = stream_ok(stream, W)) return rc;
        PagedReleaseArgs a{};
        a.held = n_held;
        a.keep = n_keep;
        a.table = table;
        a.free_pages = free_pages;
        a.n_free = n_free;
        a.n_seqs = n_seqs;
        a.stride = table_stride;
        a.n_pages = d->n_pages;
        a.lp = log2_page(d);
        return launched(launch_paged_release(a, (hipStream_t)stream), W);
    });
}

int oi_paged_append_launch(const oi_paged_dims *d, void *cache, int32_t type, const void *k, int64_t k_stride,
                           const void *v, int64_t v_stride, int32_t n, const int32_t *slots, void *stream) {
    const char *const W = "paged append";
    return guarded([&]() -> int {
        if (!dims_ok(d)) return err(OI_E_ARG, W, BAD_DIMS);
        if (!type_ok(type)) return err(OI_E_ARG, W, "type must be F32 or F16");
        if (!cache || !k || !v || !slots) return err(OI_E_ARG, W, "null argument");
        if (!aligned(cache, 256)) return err(OI_E_ARG, W, "the cache must be 256-byte aligned");
        if (!aligned(slots, 4)) return err(OI_E_ARG, W, "misaligned slots");
        if (n <= 0 || n > MAX_TOKENS) return err(OI_E_RANGE, W, "n outside 1 .. 2^24");
        const int64_t row = (int64_t)d->n_kv_heads * d->head_dim, es = size_of(type);
        if (!rows_ok(k, type, k_stride, row) || !rows_ok(v, type, v_stride, row)) return err(OI_E_ARG, W, BAD_ROWS);
        if (!apart({{cache, oi_paged_bytes(d)}, {k, row * es, n, k_stride * es}, {v, row * es, n, v_stride * es},
                    {slots, (int64_t)n * 4}}, 1))
            return err(OI_E_ARG, W, "the cache overlaps another argument");
        if (int rc = stream_ok(stream, W)) return rc;
        PagedAppendArgs a{};
        a.c = parts(d, cache);
        a.x[0] = k;
        a.x[1] = v;
        a.stride[0] = k_stride;
        a.stride[1] = v_stride;
        a.slots = slots;
        a.f16 = type == OI_TYPE_F16;
        a.n = n;
        return launched(launch_paged_append(a, (hipStream_t)stream), W);
    });
}

int64_t oi_paged_tokens_workspace_bytes(const oi_paged_dims *d, int32_t n_heads, int32_t n_seqs, int32_t n_q) {
    if (!dims_ok(d) || !heads_ok(d, n_heads) || !tokens_fit(n_seqs, n_q)) return 0;
    return (int64_t)std::max(tokens_workspace(d, n_heads, n_q, true).bytes, tokens_workspace(d, n_heads, n_q, false).bytes);
}

int oi_paged_tokens_launch(const oi_paged_dims *d, const void *cache, int32_t n_heads, int32_t type, const void *q,
                           int64_t q_stride, float scale, int32_t n_seqs, int32_t n_q, const int32_t *lens,
                           const int32_t *table, int32_t table_stride, void *out, int64_t out_stride, void *workspace,
                           int64_t workspace_bytes, void *stream) {
    const char *const W = "paged tokens";
    return guarded([&]() -> int {
        if (!dims_ok(d)) return err(OI_E_ARG, W, BAD_DIMS);
        if (!heads_ok(d, n_heads)) return err(OI_E_ARG, W, "n_heads must be a multiple of n_kv_heads (at most 4096)");
        if (!type_ok(type)) return err(OI_E_ARG, W, "type must be F32 or F16");
        if (!tokens_fit(n_seqs, n_q)) return err(OI_E_RANGE, W, "n_seqs outside 1 .. 65536 or n_q outside 1 .. 16");
        PagedAttnArgs a{};
        a.n_q = n_q;
        const Workspace w = tokens_workspace(d, n_heads, n_q, type == OI_TYPE_F16);
        if (int rc = attention(a, W, d, cache, n_heads, type, q, q_stride, scale, n_seqs, (int64_t)n_seqs * n_q, nullptr, lens,
                               table, table_stride, out, out_stride, workspace, workspace_bytes, w, stream))
            return rc;
        if (n_q * a.group > PAGED_TOKENS_ROWS) {
            a.tile_units = tile_units(a.group);
            return launched(launch_paged_prompts(a, (hipStream_t)stream), W);
        }
        a.groups = paged_tokens_groups(d->head_dim, n_q * a.group, a.f16);
        return launched(launch_paged_tokens(a, (hipStream_t)stream), W);
    });
}

int64_t oi_paged_prompts_workspace_bytes(const oi_paged_dims *d, int32_t n_heads, int32_t n_seqs, int32_t n_rows) {
    if (!dims_ok(d) || !heads_ok(d, n_heads) || !prompts_fit(d, n_heads, n_seqs, n_rows)) return 0;
    return (int64_t)std::max(prompts_workspace(d, n_heads, n_rows, true).bytes, prompts_workspace(d, n_heads, n_rows, false).bytes);
}

int oi_paged_prompts_launch(const oi_paged_dims *d, const void *cache, int32_t n_heads, int32_t type, const void *q,
                            int64_t q_stride, float scale, int32_t n_seqs, int32_t n_rows, const int32_t *starts,
                            const int32_t *lens, const int32_t *table, int32_t table_stride, void *out, int64_t out_stride,
                            void *workspace, int64_t workspace_bytes, void *stream) {
    const char *const W = "paged prompts";
    return guarded([&]() -> int {
        if (!dims_ok(d)) return err(OI_E_ARG, W, BAD_DIMS);
        if (!heads_ok(d, n_heads)) return err(OI_E_ARG, W, "n_heads must be a multiple of n_kv_heads (at most 4096)");
        if (!type_ok(type)) return err(OI_E_ARG, W, "type must be F32 or F16");
        if (!prompts_fit(d, n_heads, n_seqs, n_rows))
            return err(OI_E_RANGE, W, "n_seqs outside 1 .. 65536, or n_rows outside 1 .. 2^24 or times group^2 past 2^32");
        if (!starts) return err(OI_E_ARG, W, "null argument");
        PagedAttnArgs a{};
        const Workspace w = prompts_workspace(d, n_heads, n_rows, type == OI_TYPE_F16);
        if (int rc = attention(a, W, d, cache, n_heads, type, q, q_stride, scale, n_seqs, n_rows, starts, lens, table,
                               table_stride, out, out_stride, workspace, workspace_bytes, w, stream))
            return rc;
        a.tile_units = tile_units(a.group);
        return launched(launch_paged_prompts(a, (hipStream_t)stream), W);
    });
}

}  // extern "C"
