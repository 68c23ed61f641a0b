// paged.h -- the paged f16 K/V cache: kernel arguments and launches shared by
// paged.cpp (the C entries), paged.hip and paged_attn.hip.
#pragma once
#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace oi {

// One pool of pages in its parts.
struct Paged {
    uint16_t *k;  // [n_pages][n_kv][page][hd]
    uint16_t *v;  // [n_pages][n_kv][page / 8][hd][8]
    int32_t n_kv, hd, n_pages, lp;  // lp: log2(page)
};

struct PagedPlanArgs {
    const int32_t *past, *fresh;  // [n_seqs]: slots held, tokens to come
    int32_t *table;
    const int32_t *free_pages;
    int32_t *n_free, *lens, *starts, *slots, *pos;
    int32_t n_seqs, stride, n_rows, n_pages, lp;
};
hipError_t launch_paged_plan(const PagedPlanArgs &a, hipStream_t st);

struct PagedReleaseArgs {
    const int32_t *held, *keep, *table;  // keep: null for none
    int32_t *free_pages, *n_free;
    int32_t n_seqs, stride, n_pages, lp;
};
hipError_t launch_paged_release(const PagedReleaseArgs &a, hipStream_t st);

struct PagedAppendArgs {
    Paged c;
    const void *x[2];   // K and V rows, f32 or f16
    int64_t stride[2];  // elements from a row to the next
    const int32_t *slots;
    int32_t f16, n;
};
hipError_t launch_paged_append(const PagedAppendArgs &a, hipStream_t st);

// Where a worker's share of an attention call begins: unit u of a tile of rows of
// one kv head of a sequence.
struct PagedAt {
    int32_t seq, head, tile, u;
};

struct PagedAttnArgs {
    Paged c;
    const void *q;
    void *out;
    int64_t q_stride, out_stride;  // elements from a row (a token's heads) to the next
    float scale;                   // of q . k, times log2(e)
    int32_t f16, group;
    uint32_t magic;                // ceil(2^32 / group), 0 for a group of 1
    int32_t n_seqs, n_q, n_rows;   // n_q: tokens of each sequence (tokens call)
    const int32_t *starts, *lens, *table;  // starts: prompts call (null: n_q tokens of each)
    int32_t stride, cap;           // entries of a table row, and its slots
    int32_t groups;                // tokens kernel: log2 of the groups of waves
    float tile_units;              // prompts kernel: units of slots that a tile sees more than the one before
    // workspace
    int32_t workers, part_rows;    // part_rows: rows of a partial result
    PagedAt *at;                   // [workers + 1], the last: {used workers, 0, 0, 0}
    float2 *ml;                    // [workers][2][part_rows]: m, l
    float *part;                   // [workers][2][part_rows][hd]
};
// the workers of a call and the bytes that they take
int paged_tokens_workers(int hd);
// Rows of a sequence and kv head that the tokens kernel takes; more go through the prompts kernel, as if packed
// (whole calls, 24 sequences of 32 f16 heads of 128 over 4: 16 tokens, 128 rows, at 4000 slots 90 and 77 us, at 1050
// 38 and 37.5; 8 tokens, 64 rows, 62 and 61.5, 26 and 30; f32 77 and 85, 31 and 36).
constexpr int PAGED_TOKENS_ROWS = 64;
// log2 of the groups of waves, given the rows of a sequence and kv head
int paged_tokens_groups(int hd, int rows, bool f16);
int paged_prompts_workers(int hd, bool f16);
int paged_prompts_rows();  // of a tile
hipError_t launch_paged_tokens(const PagedAttnArgs &a, hipStream_t st);
hipError_t launch_paged_prompts(const PagedAttnArgs &a, hipStream_t st);

}  // namespace oi
