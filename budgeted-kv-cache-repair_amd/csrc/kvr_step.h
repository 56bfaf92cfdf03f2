// What a step's plan (kvr_step_plan.hip) and its attention (kvr_tree_attention.hip) share.
#pragma once

#include "kvr_internal.h"
#include "kvrepair_step.h"

namespace kvr {

// Attention work of a step. Keys are walked in steps of kStepKeys; a work item
// is a run of whole steps of one request, for every KV head and row group.
constexpr int32_t kStepKeys = 128;
constexpr int32_t kStepCus = 256;
constexpr int32_t kStepMinPage = 16;

// Schedule (int32): header {items, split requests, steps of a chunk, 0, ...},
// then items x {request, first key, end key, partial slot or -1, length, rows
// that attend, first row, rows}, then the split requests x {request, first
// partial slot, chunks, 0}.
constexpr int32_t kStepHeader = 8;
constexpr int32_t kStepItem = 8;
constexpr int32_t kStepSplit = 4;

// Query rows (row of the request x query head of the KV head) of one block.
inline int32_t step_group_rows(int64_t m) { return m <= 16 ? 16 : m <= 32 ? 32 : m <= 64 ? 64 : m <= 128 ? 128 : 256; }

struct StepShape {
    int64_t group_rows;   // query rows of a block
    int64_t row_groups;   // blocks of a request's query rows, per KV head and item
    int64_t target;       // items that fill every CU once
    int64_t items;        // room for items
    int64_t partials;     // ... for chunks of split requests
};

inline StepShape step_shape(int32_t requests, int32_t max_rows, int32_t q_heads, int32_t kv_heads) {
    const int64_t m = static_cast<int64_t>(max_rows) * (q_heads / kv_heads);
    StepShape s;
    s.group_rows = step_group_rows(m);
    s.row_groups = ceil_div(m, s.group_rows);
    const int64_t wide = s.row_groups * kv_heads;
    s.target = wide >= kStepCus ? 1 : kStepCus / wide;
    s.items = requests + s.target;
    // chunks hold at least 1 / (2 target) of all steps, and a split request has
    // at least two: fewer than twice the 2 target shares
    s.partials = s.items < 4 * s.target ? s.items : 4 * s.target;
    return s;
}

// Sizes of a step and the pointers that plan and attention both use (a status).
int check_step(const kvr_step_desc* d);

}  // namespace kvr
