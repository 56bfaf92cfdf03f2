/*
 * kvrepair_step.h — one step of several requests over one paged cache: the
 * step's plan (pages, slots, positions, tree masks, attention work list, all
 * built on the GPU) and attention of its rows, new tokens or trees of drafted
 * tokens, over each request's own cache. Conventions and statuses are
 * kvrepair.h's.
 *
 * A pool is a cache tensor [1, kv_heads, n_slots, head_dim]; a page is
 * page_size consecutive slots, page p the slots p * page_size and up. Request r
 * has lengths[r] committed tokens in the cache and counts[r] new rows in this
 * step; token j of r lies in slot table[r][j / page_size] * page_size + j mod
 * page_size. The rows of a step are packed, request after request. Requests
 * may share pages of committed tokens, but not a page that the step writes.
 */
#ifndef KVREPAIR_STEP_H
#define KVREPAIR_STEP_H

#include "kvrepair.h"

#ifdef __cplusplus
extern "C" {
#endif

#define KVR_STEP_MAX_REQUESTS 4096
#define KVR_STEP_MAX_NODES 64 /* rows of one request in attention */

/* Per-request outcome of a plan (kvr_step_desc.status). */
enum kvr_step_status {
    KVR_STEP_OK = 0,
    KVR_STEP_NO_PAGES = 1,  /* the free list ended before this request's pages */
    KVR_STEP_TOO_LONG = 2,  /* its tokens do not fit its row of the table */
    KVR_STEP_INVALID = 3,   /* negative length, count outside [0, max_rows], or rows past the step's */
};

/*
 * A step's sizes, inputs and outputs. Device memory throughout; mirrored by
 * _native.StepDesc (kvr_step_desc_size guards the mirror).
 */
typedef struct kvr_step_desc {
    /* inputs */
    const int32_t* lengths;      /* [requests] */
    const int32_t* counts;       /* [requests] */
    const int32_t* parents;      /* [rows] node index within its request, -1: hangs on the cache; null: chains */
    const int32_t* free_pages;   /* [free_count] pages to hand out, in order; may be null with free_count 0 */
    const int32_t* free_start;   /* one value: the first page of free_pages to hand out; null: 0 */
    int32_t* tables;             /* [requests][table_stride], read for committed tokens, written for new pages */
    /* outputs */
    int32_t* row_starts;         /* [requests + 1] */
    int32_t* request;            /* [rows]; -1: a row of no request */
    int64_t* slots;              /* [rows]; -1: the row is not written to the cache */
    int64_t* positions;          /* [rows]; -1: as slots, and padding nodes */
    uint64_t* masks;             /* [rows] ancestors of the row and itself, one bit a node; 0: attends to nothing.
                                    null iff max_rows > KVR_STEP_MAX_NODES */
    int32_t* status;             /* [requests] kvr_step_status */
    int32_t* pages_taken;        /* one value */
    int32_t* schedule;           /* kvr_step_schedule_ints values, 32-byte aligned; null: no attention */
    /* sizes */
    int64_t n_slots;
    int64_t table_stride;
    int32_t requests;
    int32_t rows;                /* room for the packed rows */
    int32_t max_rows;            /* most rows of one request */
    int32_t page_size;           /* a power of two, at least 16 */
    int32_t table_width;         /* with a schedule, requests * (table_width * page_size / 128 + 1) <= 2^30 */
    int32_t free_count;
    int32_t q_heads;             /* of the attention; 0 with a null schedule */
    int32_t kv_heads;
} kvr_step_desc;

int64_t kvr_step_desc_size(void);

/* int32 values of a step's attention schedule (host-only), or a negative status. */
int64_t kvr_step_schedule_ints(int32_t requests, int32_t max_rows, int32_t q_heads, int32_t kv_heads);

/*
 * Build a step's plan, one launch. Of each request's tokens those past its
 * committed pages get new ones: request r needs ceil((length + count) / P) -
 * ceil(length / P) pages and takes them from free_pages in request order, its
 * table row gets them. A request that fails (status) takes none, has no slots
 * and attends to nothing; once the free list ends, every later request that
 * needs a page fails too. Rows whose page id lies outside the pool get slot -1.
 * Node t of a tree: parent -1 or a node before it; any other parent marks a
 * padding node, which like its descendants gets no slot and no mask. The same
 * inputs give the same outputs, the tables included, however often they are
 * planned. Replaces no reference call: the reference's plan is one request's
 * selected rows (src/kv_cache_repair/kernels/indexed_attention.py:42-110).
 */
int kvr_step_plan(const kvr_step_desc* d, void* stream);

/*
 * Attention of a step's rows: row t of request r attends to the request's
 * lengths[r] committed tokens and to the nodes of its mask,
 *   out[h, row] = softmax_j(scale * q[h, row] . k[h / G, slot(j)]) @ v[h / G, slot(j)],
 * G = q_heads / kv_heads. K and V hold the step's rows already. Rows without
 * weight on any key (padding nodes, failed requests) get zeros, rows of no
 * request are zeroed with zero_rest and left as they were without. Keys in
 * pages outside the pool are not attended.
 * What stands in a key that a row does not see never reaches the row, NaN and
 * infinities included. strides: {head, row, dim} of q, k, v, out; fp16 or bf16,
 * head_dim 64 or 128, unit dim strides, head and row strides multiples of 8
 * elements (out: 4), row strides at most 2^26, on 16-byte (out: 8) aligned
 * bases; a page of K or V spans less than 4 GiB. `d` as it was planned, with
 * schedule and heads; `workspace` 16-byte aligned.
 */
int64_t kvr_tree_workspace_bytes(const kvr_step_desc* d, int32_t head_dim);
int kvr_tree_attention(const void* q, const void* k, const void* v, void* out, const kvr_step_desc* d,
                       int32_t head_dim, float scale, const int64_t strides[12], int32_t zero_rest, void* workspace,
                       int64_t workspace_bytes, int32_t dtype, void* stream);

/*
 * Projections of a step's rows with a low-rank adapter of each row's own:
 *   y[m, :] = dtype(W x_m + scales[a] * up[a] (down[a] x_m)),  a = ids[m],
 * W x_m alone where ids[m] lies outside [0, n_adapters). W are 1 to 3 weights
 * [rows_i][ldw_i], rows concatenated as in kvr_linear_multi, down[i] the pool
 * [n_adapters][rank][k] and up[i] [n_adapters][rows_i][rank] of weight i, both
 * contiguous, scales fp32. Sums are fp32, rounded once; the same inputs give the
 * same bits. Any m up to 2^20; k and rank multiples of 8, rank at most 512; ldx
 * and ldw multiples of 8 elements on 16-byte aligned bases, as the pools and
 * `workspace`. More than 64 rows run on the tiled projections where k is a
 * multiple of 64, every weight's rows one of 8, ldx and ldw at most 2^21, ldy a
 * multiple of 4 and y 8-byte aligned, and 64 rows at a time otherwise. No
 * reference counterpart.
 */
int64_t kvr_adapter_linear_workspace_bytes(int32_t m, int32_t n_weights, const int32_t* rows, int32_t k,
                                           int32_t rank);
int kvr_adapter_linear(const void* x, int32_t n_weights, const void* const* w, const int32_t* rows,
                       const int64_t* ldw, const void* const* down, const void* const* up, const float* scales,
                       int32_t n_adapters, int32_t rank, const int32_t* ids, void* y, int32_t m, int32_t k,
                       int64_t ldx, int64_t ldy, void* workspace, int64_t workspace_bytes, int32_t dtype,
                       void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KVREPAIR_STEP_H */
