/*
 * kvrepair_serve.h — what stands around a step of several requests
 * (kvrepair_step.h): attention of the chunks of new tokens that its plan pages
 * in, verification of drafted tokens, and the order of the cache afterwards:
 * accepted rows moved together, requests forked, pages given back. Conventions
 * and statuses are kvrepair.h's; pools, pages and tables are kvrepair_step.h's.
 */
#ifndef KVREPAIR_SERVE_H
#define KVREPAIR_SERVE_H

#include "kvrepair_step.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Attention of a step's rows, any number a request, each after the one before:
 * row t of request r attends to the request's lengths[r] committed tokens and to
 * its new tokens 0..t,
 *   out[h, row] = softmax_j(scale * q[h, row] . k[h / G, slot(j)]) @ v[h / G, slot(j)],
 * G = q_heads / kv_heads. K and V hold the step's rows already. `d` as
 * kvr_step_plan planned it, without parents; its schedule and heads are not
 * used. kvr_chunk_schedule makes the work list of that plan, one launch, for
 * every layer's attention: kvr_chunk_schedule_ints int32 values, 32-byte
 * aligned. Probabilities are rounded to the inputs' type before they weigh V,
 * their maximum, sum and the weighted sums are fp32. Rows of failed requests get
 * zeros, rows of no request are zeroed with zero_rest and left as they were
 * without; keys in pages outside the pool are not attended, and a row none of
 * whose keys is attended gets zeros; one that attends to scores of -inf alone gets
 * NaN, as the softmax has it. What stands in a key that a row does not see never
 * reaches the row, NaN and infinities included. strides: {head, row, dim} of q, k,
 * v, out; fp16 or bf16, head_dim 64 or 128, 0 < scale < 2^127, unit dim strides,
 * head and row strides multiples of 8 elements (out: 4), row strides at most 2^26,
 * on 16-byte (out: 8) aligned bases; a page of K or V spans less than 4 GiB;
 * (rows * G / 256 + requests) * (table_width * page_size / 128 + 2) at most 2^30.
 * `workspace` 16-byte aligned.
 */
int64_t kvr_chunk_schedule_ints(const kvr_step_desc* d, int32_t q_heads, int32_t kv_heads);
int kvr_chunk_schedule(const kvr_step_desc* d, int32_t q_heads, int32_t kv_heads, int32_t* schedule, void* stream);
int64_t kvr_chunk_workspace_bytes(const kvr_step_desc* d, int32_t q_heads, int32_t kv_heads, int32_t head_dim);
int kvr_chunk_attention(const void* q, const void* k, const void* v, void* out, const kvr_step_desc* d,
                        const int32_t* schedule, int32_t q_heads, int32_t kv_heads, int32_t head_dim, float scale,
                        const int64_t strides[12], int32_t zero_rest, void* workspace, int64_t workspace_bytes,
                        int32_t dtype, void* stream);

/*
 * Verification of drafted tokens against the target's probabilities. The rows
 * of a request are the nodes of its plan (with masks); node 0 is a token that is
 * known, the others are drafts that hang on it. Row i of
 * probs [rows][vocab] is the target's distribution after node i, tokens[i] the
 * node's token, uniforms[i] the number in [0, 1) that decides among the nodes
 * that hang on it. Node 0 is kept; of those that hang on a kept node a,
 *   without draft_probs: the first, in order, with uniforms[a] < the sum of
 *     probs[a] over the tokens of those up to it (a token that an earlier one
 *     has does not count again),
 *   with draft_probs (row i: the distribution that the token after node i was
 *     drawn from): the one that hangs on it, if uniforms[a] * draft_probs[a][x] <
 *     probs[a][x]; where several hang on one node, only the first may be kept.
 * Then answers[r] is drawn from what is left after the last kept node a: probs[a]
 * without the tokens that hang on it, max(probs[a] - draft_probs[a], 0) where one
 * hangs on it, or probs[a]: the first token whose running sum exceeds draws[r] of
 * the whole; from probs[a] where nothing is left. Entries of probs that are
 * negative, infinite or NaN count as zero, and so do such differences; -1 where all
 * do. Differences are of the entries as they stand, and draft_probs[a][x] by itself
 * is what it is: an infinite or NaN one leaves nothing of its token, a negative one
 * adds to it, and a product that is NaN or +inf keeps nothing. Sums and comparisons
 * are fp64. kept[r]: rows of the request that are kept, path: their nodes, packed at
 * row_starts[r], -1 behind them. A request without rows, or whose node 0 has no
 * mask, keeps none and answers -1. Tokens outside [0, vocab) are not kept. `d`
 * as it was planned; ld, ldd: elements of a row, at least vocab; vocab at most
 * 2^30. `workspace` 16-byte aligned.
 */
int64_t kvr_verify_workspace_bytes(int32_t requests, int32_t vocab);
int kvr_verify_drafts(const float* probs, int64_t ld, const float* draft_probs, int64_t ldd, int32_t vocab,
                      const int64_t* tokens, const float* uniforms, const float* draws, const kvr_step_desc* d,
                      int32_t* kept, int32_t* path, int64_t* answers, void* workspace, int64_t workspace_bytes,
                      void* stream);

/* Pools of several layers: K and V of each, of one layout. strides and sizes in bytes. */
typedef struct kvr_pools {
    void* const* k;       /* [layers] device addresses, an array of the host */
    void* const* v;
    int64_t k_head, k_row, v_head, v_row;
    int64_t n_slots;
    int32_t layers;
    int32_t kv_heads;
    int32_t row_bytes;    /* of a token of one head, a multiple of 16 on 16-byte aligned addresses */
    int32_t page_size;
} kvr_pools;

int64_t kvr_pools_size(void);

/*
 * Of each request of a plan the rows path[row_starts[r]] .. + kept[r] (ascending
 * nodes, as kvr_verify_drafts leaves them) become the tokens behind its
 * committed ones: row path[i]'s K and V go to token lengths[r] + i's slot, in
 * all layers. A path is taken up to its first entry that is not above the one
 * before it, or no node of its request. Rows without a slot, and slots outside
 * the pool, are neither read nor written.
 */
int kvr_keep_rows(const kvr_pools* p, const kvr_step_desc* d, const int32_t* path, const int32_t* kept, void* stream);

/*
 * `count` requests that continue others: out_tables[i] gets the pages of the
 * request sources[i] and -1 behind them, out_lengths[i] its length. Full pages are shared; a
 * partly filled last page stays with the first that continues its request, each
 * later one gets a page of the free list (its next, in order) with a copy of the
 * page's tokens in all layers. sources[i] -1: an empty request. status[i] is a kvr_step_status:
 * KVR_STEP_NO_PAGES once the free list has ended, KVR_STEP_TOO_LONG where a
 * length does not fit its table, KVR_STEP_INVALID for a source outside [-1,
 * requests) or a negative length; those are empty requests too, and leave the
 * others as they are. A last page outside the pool is entered as it is, a copy of
 * nothing, and so is a page of the free list that lies outside.
 * What is written is memory of its own, apart from what is read.
 */
typedef struct kvr_fork_desc {
    const int32_t* sources;     /* [count] */
    const int32_t* lengths;     /* [requests] */
    const int32_t* tables;      /* [requests][table_stride] */
    const int32_t* free_pages;  /* [free_count]; may be null with free_count 0 */
    const int32_t* free_start;  /* one value; null: 0 */
    int32_t* out_lengths;       /* [count] */
    int32_t* out_tables;        /* [count][out_stride] */
    int32_t* status;            /* [count] */
    int32_t* pages_taken;       /* one value */
    int64_t table_stride;
    int64_t out_stride;
    int32_t count;
    int32_t requests;
    int32_t table_width;
    int32_t free_count;
} kvr_fork_desc;

int64_t kvr_fork_desc_size(void);
int kvr_fork_requests(const kvr_pools* p, const kvr_fork_desc* d, void* stream);

/*
 * The free list of a pool of n_pages pages: list[*start] .. list[n_pages - 1]
 * become, ascending, the pages that no request holds, what stands before them -1.
 * Request r holds the first ceil(lengths[r] / page_size) entries of its row of the
 * tables (all of the row where it is shorter). `workspace`: kvr_free_pages_workspace_bytes,
 * 16-byte aligned, zero before its first call; it is not to be cleared again, and
 * calls of pools of any sizes that it holds may follow one another in it.
 */
int64_t kvr_free_pages_workspace_bytes(int32_t n_pages);
int kvr_free_pages(const int32_t* lengths, const int32_t* tables, int64_t table_stride, int32_t requests,
                   int32_t table_width, int32_t page_size, int32_t n_pages, int32_t* list, int32_t* start,
                   void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KVREPAIR_SERVE_H */
