// A paged cache of keys and values and how a slot of a sequence is found in it.
//
//   k [pages, page, G, dim], v [pages, page, G, vdim]: bf16, innermost axis contiguous, the other strides are given (elements)
//   table [sequences, per_seq]: the page that holds the slots page * i .. of a sequence; entries behind its last page are never read for it
#pragma once

#include "common.cuh"

struct PagedArgs {
    bf16* k; int64_t k_page, k_slot, k_head;
    bf16* v; int64_t v_page, v_slot, v_head;
    const int* table; int64_t table_stride;
    int seqs, per_seq, pages, page, G, dim, vdim;
};

// The page of a slot, or -1: outside the table, or an entry that names no page of the pool.
__device__ __forceinline__ int paged_page(const PagedArgs& c, int seq, int slot) {
    const int i = slot / c.page;
    if (slot < 0 || i >= c.per_seq) return -1;
    const int page = c.table[(int64_t)seq * c.table_stride + i];
    return page >= 0 && page < c.pages ? page : -1;
}

struct PagedAppendArgs {
    PagedArgs cache;
    const bf16* qkv; int64_t qkv_stride;       // q [H, dim] | k [G, dim] | v [G, vdim] a row
    const bf16* q_norm; const bf16* k_norm;    // [dim] or null
    const float2* rot; int rot_dims, rot_rows, pairs;  // (cos, sin) [rot_rows, rot_dims / 2]
    const int* positions; const int* row_seq; const int* slots;
    bf16* q; int64_t q_stride;                 // null: only keys and values
    int rows, H;
    float eps;
    uint32_t* status;
};

struct TreeAttentionArgs {
    PagedArgs cache;
    const bf16* q; int64_t q_row, q_head;
    bf16* out; int64_t out_row, out_head;
    const int* starts; const int* lengths; const int64_t* masks;
    const float* sink;
    float* part_o; float* part_ml; int64_t parts;  // room for so many sums (vdim floats, and 2)
    int rows, H, max_rows;
    float scale;
    int clear_rest;  // rows behind the last sequence become zeros (a buffer that nobody wrote), else they stay as they are
    uint32_t* status;
};
