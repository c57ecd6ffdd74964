// Attention over pages of keys and values that requests share, and over packed prompts (internal declarations).
#pragma once

#include "dense.h"

namespace zq {

constexpr uint32_t kMaxPlanRequests = 8192;  // four words of shared memory each
constexpr uint32_t kMaxPagedDim = 512;       // of a key or value head

// ---- the plan of a step, the write of its keys and values (paged_plan.cu) ---------------------------------------------
struct PagePlanArgs {
    uint32_t pages, shift, requests, table_ld, rows;  // pages of 1 << shift tokens
    const int32_t *fresh, *lens, *span;
    int32_t *lens_out, *tables, *free, *span_out, *row_start, *pos, *places, *status;
};
int launch_page_plan(const PagePlanArgs& a, cudaStream_t st);

struct PagedWriteArgs {
    GqaShape s;
    const float* qkv;
    const float *q_norm, *k_norm;
    float eps, temp_coef, temp_every;
    const float* vmix;
    float* v_first;
    void *q, *kc, *vc;
    const int32_t *pos, *places;
    uint32_t n_places, rows;  // places of the cache
};
int launch_paged_write(const PagedWriteArgs& a, bool f32, cudaStream_t st);

// ---- attention of ragged rows (paged_attention.cu, paged_attention_tc.cu) ----------------------------------------------
// Rows row_start[i] .. row_start[i + 1] - 1 are the last tokens of request i. Over pages: it holds lens[i] tokens, token t in place
// t % page of page tables[i][t / page]; an entry outside 0 .. pages - 1 stands for a page of zeros. Packed: its tokens are its
// rows, k and v their own.
struct RaggedArgs {
    GqaShape s;
    const void *q, *k, *v;
    void* out;
    size_t q_ld, k_ld, v_ld;  // values from row to row (of a token in the cache)
    uint32_t out_pitch;
    float scale;
    const int32_t *row_start, *lens, *tables;
    uint32_t requests, rows, table_ld, shift, pages;
    uint32_t capacity;  // tokens of a request at most
    bool paged;
    // Tokens of a request up to which the kernel of few rows takes it, when another one takes the others (`rest`); 0: one form for all.
    uint32_t split;
    bool rest;
    void* work;
};
size_t ragged_work_bytes(const RaggedArgs& a, bool f32);
int launch_ragged_attention(const RaggedArgs& a, bool f32, cudaStream_t st);
// Its form on tcgen05, for requests with more than a few rows (bf16): whether it has one, its work memory.
bool ragged_tc_takes(const RaggedArgs& a);
size_t ragged_tc_work_bytes(const RaggedArgs& a);
// n_ranges: a word per row that it sets to 0, or null.
int launch_ragged_tc(const RaggedArgs& a, uint32_t* n_ranges, cudaStream_t st);

}  // namespace zq
