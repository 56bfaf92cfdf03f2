// A step's plan: pages, slots, positions, tree masks and the attention work
// list of several requests' rows, from their lengths, in one launch.
//
//   have_r = ceil(L_r / P)   need_r = ceil((L_r + T_r) / P) - have_r   off_r = sum_{q < r} need_q
//   table[r][have_r + j] = free[off_r + j]                    row i = start_r + t, token j = L_r + t
//   slot_i = table[r][j / P] P + j mod P      mask_i = bit t | mask of the parent
//
// What bounds it: the launch and a few dependent memory round trips. Every
// block therefore sums the requests' counts and needs by itself (at most 4096
// of them, four a thread) instead of waiting for another launch, and looks up a
// fresh page in the free list rather than in the table that another block writes.
// The sums are whole numbers, so every block's are the same.
//
// Measured (kernel alone; one that fills a value takes 2 us): one row of each of 8
// requests 4.4 us, 16 prompts of 4k to 16k rows 7.2, trees of up to 64 nodes of 256 requests
// 7.5. With an attention work list 8 to 16 (1 to 48 requests): that is the block that
// makes the list, three sums over the requests and then the items.
#include "kvr_step.h"

namespace kvr {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kMaxPerThread = KVR_STEP_MAX_REQUESTS / kPlanThreads;

struct PlanArgs {
    kvr_step_desc d;
    int32_t page_log2;
    int32_t n_pages;
    int32_t row_blocks;    // blocks before the one that makes the schedule
    int32_t workers;       // StepShape
    int32_t items;
};

struct PlanShared {
    int32_t start[KVR_STEP_MAX_REQUESTS + 1];  // first packed row of each request
    int32_t off[KVR_STEP_MAX_REQUESTS + 1];    // its first page in the free list; the schedule's: its first unit
    int32_t len[KVR_STEP_MAX_REQUESTS];        // committed tokens; -1: failed
    int64_t wave_sums[kPlanWaves];
    int32_t taken;
};

// Exclusive sums of v over the block's values in order (PT a thread); returns the total.
template <typename V, int PT>
__device__ inline V block_scan(V (&v)[PT], int64_t* wave_sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    V mine = 0;
#pragma unroll
    for (int e = 0; e < PT; ++e) {
        const V x = v[e];
        v[e] = mine;
        mine += x;
    }
    V sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const V up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    V before = sum - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        const V x = static_cast<V>(wave_sums[w]);
        if (w < wave) before += x;
        total += x;
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PT; ++e) v[e] += before;
    return total;
}

// The last of the n ascending values that is <= x (at[0] <= x).
__device__ inline int32_t last_at_most(const int32_t* at, int32_t n, int32_t x) {
    int32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const int32_t mid = (lo + hi) >> 1;
        if (at[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// The attention work list, by one block. A request of n steps of keys is n + 1
// units (one for its start), all of them in a row; each worker gets the same
// share of the units, so one that starts in a long request ends in another. Cut
// where a share ends, request r has pieces p = 0, 1, ... at workers
// (first + 1) / share + p; a share that would begin with r's second unit leaves
// the whole of r to the next worker. Piece 0 of a cut request has partial slot
// 2 worker + 1, the others, each its worker's first item, 2 worker.
template <int PT>
__device__ inline void make_schedule(const PlanArgs& a, PlanShared& s) {
    const int R = a.d.requests, tid = threadIdx.x;
    int32_t units[PT];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PT; ++e) {
        const int r = tid * PT + e;
        units[e] = 0;
        if (r < R) {
            const int32_t rows = s.start[r + 1] - s.start[r], len = s.len[r];
            if (rows > 0) units[e] = 1 + (len < 0 ? 0 : (len + rows + kStepKeys - 1) / kStepKeys);
        }
    }
    const int32_t all = block_scan(units, s.wave_sums);
    const int32_t share = all > a.workers ? (all + a.workers - 1) / a.workers : 1;
    // this thread's first unit behind its requests is the next thread's first
#pragma unroll
    for (int e = 0; e < PT; ++e)
        if (tid * PT + e <= R) s.off[tid * PT + e] = units[e];
    if (tid == 0 && R == PT * kPlanThreads) s.off[R] = all;
    __syncthreads();
    int32_t item[PT], split[PT];
#pragma unroll
    for (int e = 0; e < PT; ++e) {
        const int r = tid * PT + e;
        // one with rows and no keys, which failed, is a unit and a piece
        item[e] = 0;
        if (r < R && s.off[r + 1] > s.off[r])
            item[e] = s.off[r + 1] - s.off[r] == 1 ? 1 : (s.off[r + 1] - 1) / share - (s.off[r] + 1) / share + 1;
        split[e] = item[e] > 1;
    }
    const int32_t n_items = block_scan(item, s.wave_sums);
    const int32_t n_split = block_scan(split, s.wave_sums);
    int32_t* const first_of = a.d.schedule + kStepHeader;
    int32_t* const work = first_of + step_worker_ints(a.workers);
    int32_t* const splits = work + static_cast<int64_t>(a.items) * kStepItem;
    if (tid == 0) {
        a.d.schedule[0] = n_items;
        a.d.schedule[1] = n_split;
        a.d.schedule[2] = share;
        a.d.schedule[3] = 0;
    }
    // workers behind the last item's have none
    const int32_t used = all > 0 ? (all - 1) / share : -1;
    for (int32_t k = used + 1 + tid; k <= a.workers; k += kPlanThreads) first_of[k] = n_items;
    const int lane = tid & 63;
#pragma unroll 1
    for (int e = 0; e < PT; ++e) {
        const int r = tid * PT + e;
        const bool has = r < R && s.off[r + 1] > s.off[r];
        const int32_t from = has ? s.off[r] : 0, steps = has ? s.off[r + 1] - from - 1 : 0;
        const int32_t rows = has ? s.start[r + 1] - s.start[r] : 0, row0 = has ? s.start[r] : 0;
        const int32_t len = has ? s.len[r] : -1, keys = len < 0 ? 0 : len + rows;
        const int32_t at = (steps > 0 ? from + 1 : from) / share;
        const int32_t n = steps > 0 ? (from + steps) / share - at + 1 : 1;
        auto put = [&](int32_t i, int32_t p, int32_t n, int32_t r, int32_t at, int32_t from, int32_t steps, int32_t keys,
                       int32_t len, int32_t rows, int32_t row0) {
            int32_t* const out = work + static_cast<int64_t>(i) * kStepItem;
            const int32_t begin = p == 0 ? 0 : (at + p) * share - from - 1;
            const int32_t end = p + 1 == n ? steps : (at + p + 1) * share - from - 1;
            out[0] = r;
            out[1] = min(begin * kStepKeys, keys);
            out[2] = min(end * kStepKeys, keys);
            out[3] = n == 1 ? -1 : step_partial(at, p);
            out[4] = max(len, 0);
            out[5] = len < 0 ? 0 : rows;
            out[6] = row0;
            out[7] = rows;
        };
        if (has) {
            if (n > 1) {
                int32_t* const p = splits + static_cast<int64_t>(split[e]) * kStepSplit;
                p[0] = at;
                p[1] = n;
                p[2] = rows;
                p[3] = row0;
            }
            // it is the first item of the workers behind the item before it, up to its own
            for (int32_t k = from > 0 ? (from - 1) / share + 1 : 0; k <= at; ++k) first_of[k] = item[e];
            put(item[e], 0, n, r, at, from, steps, keys, len, rows, row0);
        }
        // the other pieces of cut requests, by the whole wave
        uint64_t cut = __ballot(has && n > 1);
        while (cut) {
            const int l = __builtin_ctzll(cut);
            cut &= cut - 1;
            const int32_t i0 = __shfl(item[e], l), n0 = __shfl(n, l), at0 = __shfl(at, l), r0 = __shfl(r, l);
            const int32_t from0 = __shfl(from, l), steps0 = __shfl(steps, l), keys0 = __shfl(keys, l);
            const int32_t len0 = __shfl(len, l), rows0 = __shfl(rows, l), first0 = __shfl(row0, l);
            for (int32_t p = 1 + lane; p < n0; p += 64) {
                first_of[at0 + p] = i0 + p;
                put(i0 + p, p, n0, r0, at0, from0, steps0, keys0, len0, rows0, first0);
            }
        }
    }
}

template <int PT>
__global__ void __launch_bounds__(kPlanThreads) step_plan_kernel(PlanArgs a) {
    __shared__ PlanShared s;
    const kvr_step_desc& d = a.d;
    const int tid = threadIdx.x;
    const int R = d.requests;
    const int32_t P = d.page_size;
    if (tid == 0) s.taken = 0;
    const int32_t skip = d.free_start ? *d.free_start : 0;
    int32_t len[PT], cnt[PT], status[PT], need[PT], off[PT];
    int64_t start[PT];
#pragma unroll
    for (int e = 0; e < PT; ++e) {
        const int r = tid * PT + e;
        len[e] = r < R ? d.lengths[r] : 0;
        cnt[e] = r < R ? d.counts[r] : 0;
        start[e] = cnt[e] > 0 ? cnt[e] : 0;
    }
    const int64_t all_rows = block_scan(start, s.wave_sums);
    const int32_t total = static_cast<int32_t>(all_rows < d.rows ? all_rows : d.rows);
#pragma unroll
    for (int e = 0; e < PT; ++e) {
        status[e] = KVR_STEP_OK;
        if (len[e] < 0 || cnt[e] < 0 || cnt[e] > d.max_rows || start[e] + cnt[e] > d.rows)
            status[e] = KVR_STEP_INVALID;
        else if (static_cast<int64_t>(len[e]) + cnt[e] > static_cast<int64_t>(d.table_width) * P)
            status[e] = KVR_STEP_TOO_LONG;
        // at most 2^30 tokens where the request fits its table
        need[e] = status[e] == KVR_STEP_OK ? ((len[e] + cnt[e] + P - 1) >> a.page_log2) - ((len[e] + P - 1) >> a.page_log2)
                                           : 0;
        off[e] = need[e];
    }
    block_scan(off, s.wave_sums);  // at most requests * table_width < 2^31
    const int32_t given = skip < 0 || skip > d.free_count ? 0 : d.free_count - skip;
#pragma unroll
    for (int e = 0; e < PT; ++e) {
        const int r = tid * PT + e;
        if (need[e] > 0) {
            if (off[e] > given - need[e])
                status[e] = KVR_STEP_NO_PAGES;
            else
                atomicMax(&s.taken, off[e] + need[e]);  // a largest value: the order is no matter
        }
        if (r < R) {
            s.start[r] = static_cast<int32_t>(start[e] < d.rows ? start[e] : d.rows);
            // past the free list's end only failed requests, or such as need none
            s.off[r] = min(off[e], given);
            s.len[r] = status[e] == KVR_STEP_OK ? len[e] : -1;
        }
    }
    if (tid == 0) s.start[R] = total;
    __syncthreads();
    if (blockIdx.x == static_cast<unsigned>(a.row_blocks)) {
        make_schedule<PT>(a, s);
        return;
    }
    if (blockIdx.x == 0) {
#pragma unroll
        for (int e = 0; e < PT; ++e) {
            const int r = tid * PT + e;
            if (r < R) {
                d.row_starts[r] = s.start[r];
                d.status[r] = status[e];
            }
        }
        if (tid == 0) {
            d.row_starts[R] = total;
            *d.pages_taken = s.taken;
        }
    }
    const int32_t* fresh = d.free_pages + skip;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kPlanThreads + tid;
    const int64_t step = static_cast<int64_t>(a.row_blocks) * kPlanThreads;
    // ---- tables: page p of those taken is the next one of the last request that starts at or before it ----
    for (int64_t p = first; p < s.taken; p += step) {
        const int32_t r = last_at_most(s.off, R, static_cast<int32_t>(p));
        const int64_t have = (static_cast<int64_t>(s.len[r]) + P - 1) >> a.page_log2;
        d.tables[r * d.table_stride + have + (p - s.off[r])] = fresh[p];
    }
    // slot of token `tok` of request r, which has `length` committed tokens
    auto slot_of = [&](int32_t r, int32_t length, int64_t tok) __attribute__((always_inline)) -> int64_t {
        const int64_t have = (static_cast<int64_t>(length) + P - 1) >> a.page_log2;
        const int64_t at = tok >> a.page_log2;
        const int32_t page = at < have ? d.tables[r * d.table_stride + at] : fresh[s.off[r] + (at - have)];
        if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.n_pages)) return -1;
        return (static_cast<int64_t>(page) << a.page_log2) + (tok & (P - 1));
    };
    const bool masks = d.masks != nullptr;
    if (!d.parents) {
        for (int64_t i = first; i < total; i += step) {
            const int32_t r = last_at_most(s.start, R, static_cast<int32_t>(i));
            const int32_t length = s.len[r];
            const int64_t t = i - s.start[r], tok = length + t;
            d.request[i] = r;
            d.slots[i] = length < 0 ? -1 : slot_of(r, length, tok);
            d.positions[i] = length < 0 ? -1 : tok;
            if (masks) d.masks[i] = length < 0 ? 0 : ~uint64_t(0) >> (63 - t);
        }
    } else {
        // a wave for each request: lane t is node t; after i rounds it knows its
        // nearest 2^i ancestors, and whether one of them is a padding node
        const int lane = tid & 63;
        for (int32_t r = blockIdx.x * kPlanWaves + (tid >> 6); r < R; r += a.row_blocks * kPlanWaves) {
            const int32_t from = s.start[r], n = s.start[r + 1] - from, length = s.len[r];
            if (length < 0) {
                for (int32_t t = lane; t < n; t += 64) {
                    d.request[from + t] = r;
                    d.slots[from + t] = d.positions[from + t] = -1;
                    d.masks[from + t] = 0;
                }
                continue;
            }
            int32_t up = lane < n ? d.parents[from + lane] : -2;
            bool lost = lane >= n || up < -1 || up >= lane;
            if (lost) up = -1;
            uint64_t mask = uint64_t(1) << lane;
#pragma unroll
            for (int i = 0; i < 6; ++i) {
                const int at = up < 0 ? lane : up;
                const uint64_t more = __shfl(mask, at);
                const bool gone = __shfl(static_cast<int>(lost), at);
                const int32_t next = __shfl(up, at);
                if (up >= 0) {
                    mask |= more;
                    lost |= gone;
                    up = next;
                }
            }
            if (lane < n) {
                d.request[from + lane] = r;
                d.slots[from + lane] = lost ? -1 : slot_of(r, length, static_cast<int64_t>(length) + lane);
                d.positions[from + lane] = lost ? -1 : static_cast<int64_t>(length) + __popcll(mask) - 1;
                d.masks[from + lane] = lost ? 0 : mask;
            }
        }
    }
    for (int64_t i = total + first; i < d.rows; i += step) {
        d.request[i] = -1;
        d.slots[i] = d.positions[i] = -1;
        if (masks) d.masks[i] = 0;
    }
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

}  // namespace

// Sizes of a step and the pointers that plan and attention both use.
int check_step(const kvr_step_desc* d) {
    if (!d) return KVR_E_NULL_POINTER;
    if (d->requests <= 0 || d->requests > KVR_STEP_MAX_REQUESTS || d->rows <= 0 || d->max_rows <= 0 ||
        d->table_width <= 0 || d->free_count < 0 || d->n_slots <= 0)
        return KVR_E_UNSUPPORTED_SHAPE;
    const int32_t P = d->page_size;
    if (P < kStepMinPage || (P & (P - 1)) || d->n_slots % P || d->n_slots / P > INT32_MAX) return KVR_E_UNSUPPORTED_SHAPE;
    // lengths, and pages in all, fit 32 bits
    if (static_cast<int64_t>(d->table_width) * P > (int64_t(1) << 30) ||
        static_cast<int64_t>(d->table_width) * d->requests > INT32_MAX)
        return KVR_E_UNSUPPORTED_SHAPE;
    if (d->table_stride < d->table_width) return KVR_E_BAD_STRIDE;
    if (!d->tables || !d->row_starts || !d->request || !d->slots || !d->positions || !d->status || !d->pages_taken)
        return KVR_E_NULL_POINTER;
    if (d->schedule) {
        if (!d->masks) return KVR_E_NULL_POINTER;
        if (d->q_heads <= 0 || d->kv_heads <= 0 || d->q_heads % d->kv_heads || d->max_rows > KVR_STEP_MAX_NODES)
            return KVR_E_UNSUPPORTED_SHAPE;
        // the units of all requests (make_schedule) fit 32 bits
        if (d->requests * (ceil_div(static_cast<int64_t>(d->table_width) * P, kStepKeys) + 1) > (int64_t(1) << 30))
            return KVR_E_UNSUPPORTED_SHAPE;
        if (!aligned(d->schedule, 32)) return KVR_E_BAD_STRIDE;
    }
    return KVR_OK;
}

}  // namespace kvr

using namespace kvr;

extern "C" int64_t kvr_step_desc_size(void) { return sizeof(kvr_step_desc); }

extern "C" int64_t kvr_step_schedule_ints(int32_t requests, int32_t max_rows, int32_t q_heads, int32_t kv_heads) {
    if (requests <= 0 || requests > KVR_STEP_MAX_REQUESTS || max_rows <= 0 || max_rows > KVR_STEP_MAX_NODES ||
        q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads)
        return KVR_E_UNSUPPORTED_SHAPE;
    const StepShape s = step_shape(requests, max_rows, q_heads, kv_heads);
    return kStepHeader + step_worker_ints(s.workers) + s.items * kStepItem + s.splits * kStepSplit;
}

extern "C" int kvr_step_plan(const kvr_step_desc* d, void* stream) {
    const int st = check_step(d);
    if (st != KVR_OK) return st;
    if (!d->lengths || !d->counts || (d->free_count > 0 && !d->free_pages)) return KVR_E_NULL_POINTER;
    if ((d->masks == nullptr) != (d->max_rows > KVR_STEP_MAX_NODES)) return KVR_E_NULL_POINTER;
    if (d->parents && !d->masks) return KVR_E_UNSUPPORTED_SHAPE;
    PlanArgs a;
    a.d = *d;
    a.page_log2 = __builtin_ctz(static_cast<unsigned>(d->page_size));
    a.n_pages = static_cast<int32_t>(d->n_slots / d->page_size);
    const int64_t per = d->parents ? ceil_div(d->requests, kPlanWaves) : ceil_div(d->rows, kPlanThreads);
    a.row_blocks = static_cast<int32_t>(per < kStepCus ? per : kStepCus);
    a.workers = a.items = 0;
    if (d->schedule) {
        const StepShape s = step_shape(d->requests, d->max_rows, d->q_heads, d->kv_heads);
        a.workers = static_cast<int32_t>(s.workers);
        a.items = static_cast<int32_t>(s.items);
    }
    const int blocks = a.row_blocks + (d->schedule ? 1 : 0);
    if (d->requests <= kPlanThreads)
        step_plan_kernel<1><<<blocks, kPlanThreads, 0, as_stream(stream)>>>(a);
    else
        step_plan_kernel<kMaxPerThread><<<blocks, kPlanThreads, 0, as_stream(stream)>>>(a);
    return launch_status();
}
