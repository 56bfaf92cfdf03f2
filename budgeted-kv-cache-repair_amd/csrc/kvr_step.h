// What a step's plan (kvr_step_plan.hip) and its attention (kvr_tree_attention.hip) share.
#pragma once

#include "kvr_internal.h"
#include "kvrepair_step.h"

namespace kvr {

// Attention work of a step. Keys are walked in steps of kStepKeys. As many
// workers as fill the CUs (per KV head and group of query rows) share all steps
// of all requests evenly; a work item is a worker's run of steps of one request.
constexpr int32_t kStepKeys = 128;
constexpr int32_t kStepCus = 256;
constexpr int32_t kStepMinPage = 16;

// Schedule (int32): header {items, split requests, units of a share, 0, ...};
// workers + 1 x {first item}, padded to 8; items x {request, first key, end key,
// partial slot or -1, length, rows that attend, first row, rows}; then the split
// requests x {worker of the first piece, pieces, rows, first row}.
constexpr int32_t kStepHeader = 8;
constexpr int32_t kStepItem = 8;
constexpr int32_t kStepSplit = 4;

__host__ __device__ constexpr int32_t step_worker_ints(int64_t workers) {
    return static_cast<int32_t>((workers + 1 + 7) / 8 * 8);
}

// Partial slot of piece p of a split request whose first piece is worker w's.
__host__ __device__ constexpr int32_t step_partial(int32_t w, int32_t p) { return p == 0 ? 2 * w + 1 : 2 * (w + p); }

// Query rows (row of the request x query head of the KV head) of one block.
inline int32_t step_group_rows(int64_t m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : m <= 128 ? 128 : 256; }

struct StepShape {
    int64_t group_rows;   // query rows of a block
    int64_t row_groups;   // blocks of a request's query rows, per KV head and item
    int64_t workers;
    int64_t items;        // room for items: one a request, and one more at each share's end
    int64_t partials;     // a worker's first and last item may be pieces of split requests
    int64_t splits;
};

inline StepShape step_shape(int32_t requests, int32_t max_rows, int32_t q_heads, int32_t kv_heads) {
    const int64_t m = static_cast<int64_t>(max_rows) * (q_heads / kv_heads);
    StepShape s;
    s.group_rows = step_group_rows(m);
    s.row_groups = ceil_div(m, s.group_rows);
    const int64_t wide = s.row_groups * kv_heads;
    // As many as give each CU one block; where the width alone is more than half of the CUs, as many
    // as two rounds of blocks hold (three up to 170, two up to 256), so that CUs left over by one round
    // have work. us a call, 170 wide with three, then 171 wide with two against one (which needs no
    // merge): one row over 4k tokens 63, 73 against 59; one row of each of 8 requests of 1k 124, 159
    // against 145; 64 rows over 4k 91, 103 against 80. 256 wide 90 against 85, 180 against 176, 125
    // against 103: above 170 one worker would do, and such widths (more than 170 KV heads, or
    // fewer with several groups of rows) are left as they are.
    s.workers = wide <= kStepCus / 2 ? kStepCus / wide : wide <= kStepCus ? 2 * kStepCus / wide : 1;
    s.items = requests + s.workers;
    s.partials = s.workers > 1 ? 2 * s.workers : 0;
    s.splits = requests < s.workers ? requests : s.workers;
    return s;
}

// Sizes of a step and the pointers that plan and attention both use (a status).
int check_step(const kvr_step_desc* d);

}  // namespace kvr
