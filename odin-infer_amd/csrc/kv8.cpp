// kv8.cpp -- C entries of the 8-bit K/V cache and of the rotation of q and k:
// argument checks, the parts of a cache buffer, launches (kv8.hip, kv8_attn.hip,
// rope.hip).  Nothing here allocates device memory or waits for the device, so
// every launch can be captured into a graph.
#include "kv8.h"

#include <algorithm>
#include <cmath>
#include <string>

#include "oi.h"
#include "oi_kernels.h"

using namespace oi;

namespace {

// C callers must see no exception: a message that cannot be built is left out.
int err(int code, const char *what, const std::string &msg) noexcept {
    try {
        return set_error(code, (std::string(what) + ": " + msg).c_str());
    } catch (...) {
        return code;
    }
}
template <class F>
int guarded(F f) noexcept {
    try {
        return f();
    } catch (...) {
        return OI_E_NOMEM;  // std::string is all that allocates here
    }
}

int launched(hipError_t e, const char *what) {
    return e == hipSuccess ? OI_OK : err(OI_E_DEVICE, what, hipGetErrorString(e));
}

bool dims_ok(const oi_kv8_dims *d) {
    return d && d->n_kv_heads > 0 && d->n_kv_heads <= 1024 && (d->head_dim == 128 || d->head_dim == 256) &&
           d->capacity > 0 && d->capacity <= (1 << 28) && d->capacity % KV8_TILE == 0 &&
           (d->block == 16 || d->block == 32 || d->block == 64);
}
const char *const BAD_DIMS = "bad dims (head_dim 128 or 256, capacity a multiple of 64, block 16, 32 or 64)";

Kv8 parts(const oi_kv8_dims *d, const void *cache) {
    Kv8 c{};
    c.n_kv = d->n_kv_heads;
    c.hd = d->head_dim;
    c.cap = d->capacity;
    c.lb = d->block == 16 ? 4 : d->block == 32 ? 5 : 6;
    const size_t codes = (size_t)c.n_kv * c.cap * c.hd, exps = (size_t)c.n_kv * (c.cap / d->block);
    c.kc = (int8_t *)const_cast<void *>(cache);
    c.vc = c.kc + codes;
    c.ke = c.vc + codes;
    c.ve = c.ke + exps;
    return c;
}

bool aligned(const void *p, size_t n) { return (uintptr_t)p % n == 0; }
bool type_ok(int32_t t) { return t == OI_TYPE_F32 || t == OI_TYPE_F16; }
int64_t size_of(int32_t t) { return t == OI_TYPE_F16 ? 2 : 4; }
// rows of `len` elements, `stride` apart, read and written 16 bytes at a time
bool rows_ok(const void *p, int32_t type, int64_t stride, int64_t len) {
    return aligned(p, 16) && stride >= len && stride <= ((int64_t)1 << 40) && stride * size_of(type) % 16 == 0;
}
const char *const BAD_ROWS = "rows must be 16-byte aligned, a stride at least a row and a multiple of 16 bytes";

// A kernel is launched on the current device: a stream of another one is refused.
int stream_ok(void *stream, const char *what) {
    if (!stream) return OI_OK;
    int cur = -1;
    hipDevice_t dev = -1;
    if (hipGetDevice(&cur) != hipSuccess) return err(OI_E_DEVICE, what, "no current HIP device");
    if (hipStreamGetDevice((hipStream_t)stream, &dev) != hipSuccess) {
        (void)hipGetLastError();
        return OI_OK;  // the legacy and per-thread default streams are the current device's
    }
    if ((int)dev != cur) return err(OI_E_ARG, what, "the stream belongs to another device than the current one");
    return OI_OK;
}

constexpr int64_t MAX_ROWS = 65535 * 16;  // of a kv head in one attention call: the grid of tiles of 16

// `past` slots in use, then `n` more
int range_ok(const oi_kv8_dims *d, int32_t n, int32_t past, const int32_t *past_dev, const char *what) {
    if (n <= 0 || n > d->capacity) return err(OI_E_RANGE, what, "n=" + std::to_string(n) + " outside 1..capacity");
    if (!past_dev && (past < 0 || past > d->capacity - n))
        return err(OI_E_RANGE, what, "slots " + std::to_string(past) + "+" + std::to_string(n) +
                                         " out of range (capacity=" + std::to_string(d->capacity) + ")");
    return OI_OK;
}

// n pieces of `len` bytes, `stride` apart
struct Span {
    const void *p;
    int64_t len, n = 1, stride = 0;
};
// Whether any two pieces may meet: equal strides are looked at within one stride (q, k and v
// in one row of a projection lie between each other), others as a whole.
bool overlap(const Span &a, const Span &b) {
    if (!a.p || !b.p) return false;
    const __int128 x = (uintptr_t)a.p, y = (uintptr_t)b.p;  // n * stride may pass 64 bits
    if (x >= y + (__int128)(b.n - 1) * b.stride + b.len || y >= x + (__int128)(a.n - 1) * a.stride + a.len) return false;
    if (a.n == 1 || b.n == 1 || a.stride != b.stride) return true;
    const int64_t s = a.stride, by = (int64_t)((y - x) % s), r = by < 0 ? by + s : by;  // b's place behind a piece of a
    return r < a.len || s - r < b.len;
}

}  // namespace

extern "C" {

int64_t oi_kv8_bytes(const oi_kv8_dims *d) {
    if (!dims_ok(d)) return 0;
    const int64_t n = (int64_t)d->n_kv_heads * d->capacity;
    return (2 * n * d->head_dim + 2 * (n / d->block) + 255) / 256 * 256;
}

int oi_kv8_append_launch(const oi_kv8_dims *d, void *cache, int32_t type, const void *k, int64_t k_stride,
                         const void *v, int64_t v_stride, int32_t n, int32_t n_past, const int32_t *n_past_dev,
                         void *stream) {
    const char *const W = "kv8 append";
    return guarded([&]() -> int {
        if (!dims_ok(d)) return err(OI_E_ARG, W, BAD_DIMS);
        if (!type_ok(type)) return err(OI_E_ARG, W, "type must be F32 or F16");
        if (!cache || !k || !v) return err(OI_E_ARG, W, "null argument");
        if (!aligned(cache, 256)) return err(OI_E_ARG, W, "the cache must be 256-byte aligned");
        if (!aligned(n_past_dev, 4)) return err(OI_E_ARG, W, "misaligned n_past_dev");
        if (int rc = range_ok(d, n, n_past, n_past_dev, W)) return rc;
        const int64_t row = (int64_t)d->n_kv_heads * d->head_dim;
        if (!rows_ok(k, type, k_stride, row) || !rows_ok(v, type, v_stride, row)) return err(OI_E_ARG, W, BAD_ROWS);
        const int64_t es = size_of(type);
        const Span all{cache, oi_kv8_bytes(d)};
        if (overlap(all, {k, row * es, n, k_stride * es}) || overlap(all, {v, row * es, n, v_stride * es}))
            return err(OI_E_ARG, W, "k or v lies in the cache");
        if (overlap(all, {n_past_dev, 4})) return err(OI_E_ARG, W, "n_past_dev lies in the cache");
        if (int rc = stream_ok(stream, W)) return rc;
        Kv8AppendArgs a{};
        a.c = parts(d, cache);
        a.x[0] = k;
        a.x[1] = v;
        a.stride[0] = k_stride;
        a.stride[1] = v_stride;
        a.f16 = type == OI_TYPE_F16;
        a.n = n;
        a.past = {n_past, n_past_dev};
        return launched(launch_kv8_append(a, (hipStream_t)stream), W);
    });
}

int oi_kv8_read_launch(const oi_kv8_dims *d, const void *cache, int32_t slot0, int32_t n, int32_t type, void *k,
                       void *v, void *stream) {
    const char *const W = "kv8 read";
    return guarded([&]() -> int {
        if (!dims_ok(d)) return err(OI_E_ARG, W, BAD_DIMS);
        if (!type_ok(type)) return err(OI_E_ARG, W, "type must be F32 or F16");
        if (!cache || !k || !v) return err(OI_E_ARG, W, "null argument");
        if (!aligned(cache, 256)) return err(OI_E_ARG, W, "the cache must be 256-byte aligned");
        if (!aligned(k, 16) || !aligned(v, 16)) return err(OI_E_ARG, W, "outputs must be 16-byte aligned");
        if (int rc = range_ok(d, n, slot0, nullptr, W)) return rc;
        const int64_t bytes = (int64_t)d->n_kv_heads * n * d->head_dim * size_of(type);
        const Span all{cache, oi_kv8_bytes(d)}, ko{k, bytes}, vo{v, bytes};
        if (overlap(all, ko) || overlap(all, vo) || overlap(ko, vo)) return err(OI_E_ARG, W, "outputs overlap");
        if (int rc = stream_ok(stream, W)) return rc;
        Kv8ReadArgs a{};
        a.c = parts(d, cache);
        a.out[0] = k;
        a.out[1] = v;
        a.f16 = type == OI_TYPE_F16;
        a.slot0 = slot0;
        a.n = n;
        return launched(launch_kv8_read(a, (hipStream_t)stream), W);
    });
}

int64_t oi_kv8_attn_workspace_bytes(const oi_kv8_dims *d, int32_t n_heads, int32_t n) {
    if (!dims_ok(d) || n_heads <= 0 || n_heads > 4096 || n_heads % d->n_kv_heads || n <= 0 || n > d->capacity) return 0;
    if ((int64_t)n * (n_heads / d->n_kv_heads) > MAX_ROWS) return 0;
    return (int64_t)kv8_attn_workspace_most(n_heads, n_heads / d->n_kv_heads, n, d->capacity, d->head_dim);
}

int oi_kv8_attn_launch(const oi_kv8_dims *d, const void *cache, int32_t n_heads, int32_t type, const void *q,
                       int64_t q_stride, float scale, int32_t n, int32_t n_past, const int32_t *n_past_dev,
                       float *mass, void *out, int64_t out_stride, void *workspace, int64_t workspace_bytes,
                       void *stream) {
    const char *const W = "kv8 attention";
    return guarded([&]() -> int {
        if (!dims_ok(d)) return err(OI_E_ARG, W, BAD_DIMS);
        if (n_heads <= 0 || n_heads > 4096 || n_heads % d->n_kv_heads)
            return err(OI_E_ARG, W, "n_heads must be a multiple of n_kv_heads (at most 4096)");
        if (!type_ok(type)) return err(OI_E_ARG, W, "type must be F32 or F16");
        if (!cache || !q || !out || !workspace) return err(OI_E_ARG, W, "null argument");
        if (!aligned(cache, 256)) return err(OI_E_ARG, W, "the cache must be 256-byte aligned");
        if (!aligned(workspace, 16) || !aligned(mass, 4) || !aligned(n_past_dev, 4)) return err(OI_E_ARG, W, "misaligned workspace, mass or n_past_dev");
        if (int rc = range_ok(d, n, n_past, n_past_dev, W)) return rc;
        const float scale2 = (float)((double)scale * 1.4426950408889634);  // exponents are formed in base 2
        if (!std::isfinite(scale2)) return err(OI_E_ARG, W, "scale (times log2 e) is not finite");
        const int64_t row = (int64_t)n_heads * d->head_dim;
        if (!rows_ok(q, type, q_stride, row) || !rows_ok(out, type, out_stride, row)) return err(OI_E_ARG, W, BAD_ROWS);
        if (out == q && (q_stride != out_stride || mass))
            return err(OI_E_ARG, W, "out may be q only with the same stride and without mass");
        const int group = n_heads / d->n_kv_heads;
        if ((int64_t)n * group > MAX_ROWS) return err(OI_E_RANGE, W, "too many rows in one call");
        const int end = n_past_dev ? d->capacity : n_past + n;
        const int splits = kv8_attn_splits(d->n_kv_heads, group, n, end, d->head_dim, type == OI_TYPE_F16);
        const int64_t need = (int64_t)kv8_attn_workspace(n_heads, group, n, end, d->head_dim, splits, mass);
        if (workspace_bytes < need)
            return err(OI_E_ARG, W, "workspace of " + std::to_string(workspace_bytes) + " bytes, " +
                                        std::to_string(need) + " needed");
        const int64_t es = size_of(type);
        const Span all{cache, oi_kv8_bytes(d)}, qs{q, row * es, n, q_stride * es}, os{out, row * es, n, out_stride * es},
            ws_span{workspace, need}, ms{mass, (int64_t)d->n_kv_heads * d->capacity * 4}, past{n_past_dev, 4};
        if ((out != q && overlap(os, qs)) || overlap(os, all) || overlap(os, ws_span) || overlap(os, ms) ||
            overlap(ws_span, all) || overlap(ws_span, qs) || overlap(ws_span, ms) || overlap(ms, all) ||
            overlap(ms, qs) || overlap(past, os) || overlap(past, ws_span) || overlap(past, ms))
            return err(OI_E_ARG, W, "out, workspace or mass overlaps another argument");
        if (int rc = stream_ok(stream, W)) return rc;
        Kv8AttnArgs a{};
        a.c = parts(d, cache);
        a.q = q;
        a.q_stride = q_stride;
        a.out = out;
        a.out_stride = out_stride;
        a.scale = scale2;
        a.f16 = type == OI_TYPE_F16;
        a.n = n;
        a.n_heads = n_heads;
        a.group = group;
        a.magic = group > 1 ? (uint32_t)((((uint64_t)1 << 32) + group - 1) / group) : 0u;
        a.past = {n_past, n_past_dev};
        a.mass = mass;
        a.splits = splits;
        // the saved weights first (16-byte stores), then the splits' results
        const size_t rows = (size_t)n * n_heads, parts = rows * splits;
        float *ws = (float *)workspace;
        if (mass && kv8_attn_saves(group, n)) {
            a.save_units = (end + KV8_TILE - 1) / KV8_TILE;
            a.save = ws;
            a.save_m = ws + rows * a.save_units * KV8_TILE;
            ws = a.save_m + (rows * a.save_units + 3) / 4 * 4;
        }
        a.part = ws;
        a.ml = (float4 *)(a.part + (splits > 1 ? parts * d->head_dim : 0));
        a.norm = mass ? (float2 *)(a.ml + parts) : nullptr;
        if (mass && !a.save) {
            a.msplits = kv8_mass_splits(d->n_kv_heads, group, n, end, d->head_dim);
            a.msum_slots = end;
            a.msum = (float *)(a.norm + rows);
        }
        return launched(launch_kv8_attn(a, (hipStream_t)stream), W);
    });
}

int oi_kv8_evict_launch(const oi_kv8_dims *src_dims, const void *src, const float *src_mass, const int32_t *src_pos,
                        int32_t n, int32_t keep, int32_t n_first, int32_t n_last, const oi_kv8_dims *dst_dims,
                        void *dst, float *dst_mass, int32_t *dst_pos, int32_t *kept, void *stream) {
    const char *const W = "kv8 evict";
    return guarded([&]() -> int {
        if (!dims_ok(src_dims) || !dims_ok(dst_dims)) return err(OI_E_ARG, W, BAD_DIMS);
        if (src_dims->n_kv_heads != dst_dims->n_kv_heads || src_dims->head_dim != dst_dims->head_dim)
            return err(OI_E_ARG, W, "the caches' heads differ");
        if (!src || !src_mass || !dst || !dst_mass || !kept || !src_pos != !dst_pos)
            return err(OI_E_ARG, W, "null argument (positions come and go together)");
        if (!aligned(src, 256) || !aligned(dst, 256)) return err(OI_E_ARG, W, "a cache must be 256-byte aligned");
        if (!aligned(src_mass, 16) || !aligned(dst_mass, 4) || !aligned(src_pos, 4) || !aligned(dst_pos, 4) ||
            !aligned(kept, 4))
            return err(OI_E_ARG, W, "src_mass must be 16-byte aligned, the others 4");
        if (n <= 0 || n > src_dims->capacity || keep <= 0 || keep > n || keep > dst_dims->capacity)
            return err(OI_E_RANGE, W, "n=" + std::to_string(n) + " keep=" + std::to_string(keep) + " out of range");
        if (n_first < 0 || n_last < 0 || (int64_t)n_first + n_last > keep)
            return err(OI_E_RANGE, W, "n_first + n_last outside 0..keep");
        const int64_t h = src_dims->n_kv_heads, sm = h * src_dims->capacity * 4, dm = h * dst_dims->capacity * 4;
        const Span in[] = {{src, oi_kv8_bytes(src_dims)}, {src_mass, sm}, {src_pos, sm}},
                   to[] = {{dst, oi_kv8_bytes(dst_dims)}, {dst_mass, dm}, {dst_pos, dm}, {kept, h * keep * 4}};
        for (int i = 0; i < 4; i++) {
            for (const Span &s : in)
                if (overlap(to[i], s)) return err(OI_E_ARG, W, "the two caches overlap");
            for (int j = 0; j < i; j++)
                if (overlap(to[i], to[j])) return err(OI_E_ARG, W, "outputs overlap");
        }
        if (int rc = stream_ok(stream, W)) return rc;
        Kv8EvictArgs a{};
        a.src = parts(src_dims, src);
        a.dst = parts(dst_dims, dst);
        a.mass = src_mass;
        a.pos = src_pos;
        a.dst_mass = dst_mass;
        a.dst_pos = dst_pos;
        a.kept = kept;
        a.n = n;
        a.keep = keep;
        a.first = n_first;
        a.last = n_last;
        return launched(launch_kv8_evict(a, (hipStream_t)stream), W);
    });
}

int oi_rope_axes_launch(const oi_rope_axes_dims *d, int32_t n, const int32_t *pos, const float *inv_freq,
                        const float *q_norm, const float *k_norm, int32_t in_type, const void *q, int64_t q_stride,
                        int64_t q_head_stride, const void *k, int64_t k_stride, int32_t out_type, void *q_out,
                        int64_t q_out_stride, void *k_out, int64_t k_out_stride, void *stream) {
    const char *const W = "rope";
    return guarded([&]() -> int {
        if (!d || d->n_heads <= 0 || d->n_heads > 4096 || d->n_kv_heads <= 0 || d->n_kv_heads > 1024 ||
            (d->head_dim != 128 && d->head_dim != 256) || d->rotary_dim < 0 || d->rotary_dim > d->head_dim ||
            d->rotary_dim % 2)
            return err(OI_E_ARG, W, "bad dims (head_dim 128 or 256, rotary_dim even and at most head_dim)");
        int64_t pairs = 0;
        for (int32_t s : d->sections) {
            if (s < 0) return err(OI_E_ARG, W, "a section is negative");
            pairs += s;
        }
        if (pairs != d->rotary_dim / 2) return err(OI_E_ARG, W, "the sections' sum is not rotary_dim / 2");
        if (!(d->eps >= 0.f) || !std::isfinite(d->eps)) return err(OI_E_ARG, W, "bad eps");
        if (n <= 0 || n >= 1 << 24) return err(OI_E_RANGE, W, "n outside 1 .. 2^24 - 1");  // 256 threads each in one grid
        if (!type_ok(in_type) || !type_ok(out_type)) return err(OI_E_ARG, W, "type must be F32 or F16");
        if (!q || !k || !q_out || !k_out || (d->rotary_dim && (!pos || !inv_freq)))
            return err(OI_E_ARG, W, "null argument");
        const int64_t hd = d->head_dim, qr = (int64_t)(d->n_heads - 1) * q_head_stride + hd;
        if (q_head_stride < hd || q_head_stride > ((int64_t)1 << 32) || q_head_stride * size_of(in_type) % 16 ||
            !rows_ok(q, in_type, q_stride, qr) || !rows_ok(k, in_type, k_stride, d->n_kv_heads * hd) ||
            !rows_ok(q_out, out_type, q_out_stride, d->n_heads * hd) ||
            !rows_ok(k_out, out_type, k_out_stride, d->n_kv_heads * hd))
            return err(OI_E_ARG, W, BAD_ROWS);
        if ((q_out == q && (in_type != out_type || q_stride != q_out_stride || q_head_stride != hd)) ||
            (k_out == k && (in_type != out_type || k_stride != k_out_stride)))
            return err(OI_E_ARG, W, "in place needs the same type and strides");
        const int64_t ei = size_of(in_type), eo = size_of(out_type);
        const Span qs{q, qr * ei, n, q_stride * ei}, ks{k, d->n_kv_heads * hd * ei, n, k_stride * ei},
            qo{q_out, d->n_heads * hd * eo, n, q_out_stride * eo}, ko{k_out, d->n_kv_heads * hd * eo, n, k_out_stride * eo};
        if ((q_out != q && overlap(qo, qs)) || (k_out != k && overlap(ko, ks)) || overlap(qo, ks) || overlap(ko, qs) ||
            overlap(qo, ko))
            return err(OI_E_ARG, W, "an output overlaps another argument");
        if (d->rotary_dim)  // not read otherwise
            for (const Span &s : {Span{pos, (int64_t)n * 12}, Span{inv_freq, (int64_t)d->rotary_dim * 2}})
                if (overlap(qo, s) || overlap(ko, s)) return err(OI_E_ARG, W, "an output overlaps the positions or frequencies");
        for (const float *p : {q_norm, k_norm})
            if (overlap(qo, {p, hd * 4}) || overlap(ko, {p, hd * 4}))
                return err(OI_E_ARG, W, "an output overlaps a norm's weights");
        if (!aligned(pos, 4) || !aligned(inv_freq, 4) || !aligned(q_norm, 4) || !aligned(k_norm, 4))
            return err(OI_E_ARG, W, "misaligned positions, frequencies or norm weights");
        if (int rc = stream_ok(stream, W)) return rc;
        RopeArgs a{};
        a.q = q; a.k = k; a.qo = q_out; a.ko = k_out;
        a.q_stride = q_stride; a.q_head = q_head_stride; a.k_stride = k_stride;
        a.qo_stride = q_out_stride; a.ko_stride = k_out_stride;
        a.pos = pos; a.inv_freq = inv_freq; a.q_norm = q_norm; a.k_norm = k_norm;
        a.eps = d->eps;
        a.n = n; a.n_heads = d->n_heads; a.n_kv = d->n_kv_heads; a.hd = d->head_dim; a.rotary = d->rotary_dim;
        for (int i = 0; i < 3; i++) a.sec[i] = d->sections[i];
        a.interleaved = d->interleaved != 0;
        a.in_f16 = in_type == OI_TYPE_F16;
        a.out_f16 = out_type == OI_TYPE_F16;
        return launched(launch_rope_axes(a, (hipStream_t)stream), W);
    });
}

}  // extern "C"
