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
#include "kvr_step.h"

namespace kvr {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kPerThread = KVR_STEP_MAX_REQUESTS / kPlanThreads;

struct PlanArgs {
    kvr_step_desc d;
    int32_t page_log2;
    int32_t n_pages;
    int32_t row_blocks;    // blocks before the one that makes the schedule
    int32_t target, items; // StepShape
};

// Exclusive sums of v over the block's values in order (four a thread); the
// total in every thread.
__device__ inline int64_t block_scan(int64_t (&v)[kPerThread], int64_t* wave_sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t mine = 0;
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int64_t x = v[e];
        v[e] = mine;
        mine += x;
    }
    int64_t sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int64_t up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    int64_t before = sum - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        if (w < wave) before += wave_sums[w];
        total += wave_sums[w];
    }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) v[e] += before;
    return total;
}

// The last of the n + 1 ascending values that is <= x (at[0] <= x).
__device__ inline int32_t last_at_most(const int32_t* at, int32_t n, int32_t x) {
    int32_t lo = 0, hi = n + 1;
    while (hi - lo > 1) {
        const int32_t mid = (lo + hi) >> 1;
        if (at[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

struct PlanShared {
    int32_t start[KVR_STEP_MAX_REQUESTS + 1];  // first packed row of each request
    int32_t off[KVR_STEP_MAX_REQUESTS + 1];    // its first page in the free list
    int32_t len[KVR_STEP_MAX_REQUESTS];        // committed tokens; -1: failed
    int64_t wave_sums[kPlanWaves];
    int32_t taken;
    int32_t sums[kPlanWaves];                  // of the chunk search
    int32_t range[2];
};

// The attention work list, by one block. Chunks of `c` steps, the smallest c
// that keeps the items within their room: one item per CU slot while there are
// few requests, else one per request and that many more; never below the share
// of a CU (half of it with many requests, whose blocks come in several rounds).
__device__ inline void make_schedule(const PlanArgs& a, PlanShared& s) {
    const int R = a.d.requests, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // steps (0: no rows) of each request, over s.off, which this block needs no more
    int64_t steps[kPerThread], active[kPerThread];
    int32_t longest = 1;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int r = tid * kPerThread + e;
        steps[e] = active[e] = 0;
        if (r < R) {
            const int32_t rows = s.start[r + 1] - s.start[r], len = s.len[r];
            active[e] = rows > 0;
            if (rows > 0 && len >= 0) steps[e] = (static_cast<int64_t>(len) + rows + kStepKeys - 1) / kStepKeys;
            s.off[r] = rows > 0 ? max(1, static_cast<int32_t>(steps[e])) : 0;
            longest = max(longest, static_cast<int32_t>(steps[e]));
        }
    }
    const int64_t all = block_scan(steps, s.wave_sums);
    const int64_t live = block_scan(active, s.wave_sums);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) longest = max(longest, __shfl_xor(longest, d));
    if (lane == 0) s.sums[wave] = longest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) longest = max(longest, s.sums[w]);
    const bool few = 2 * live <= a.target;
    const int64_t room = few ? a.target : live + a.target;
    const int64_t share = few ? a.target : 2 * a.target;
    int32_t lo = static_cast<int32_t>((all + share - 1) / share);
    if (lo < 1) lo = 1;
    int32_t hi = max(longest, lo);  // one chunk a request always fits
    // each wave tries one chunk length between lo and hi at a time
    while (lo < hi) {
        __syncthreads();
        const int32_t width = (hi - lo + kPlanWaves - 1) / kPlanWaves;
        const int32_t c = min(hi, lo + wave * width);
        int64_t sum = 0;
        for (int r = lane; r < R; r += 64) sum += (s.off[r] + c - 1) / c;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) sum += __shfl_xor(sum, d);
        if (lane == 0) s.sums[wave] = sum <= room;
        __syncthreads();
        int first = kPlanWaves;
#pragma unroll
        for (int w = kPlanWaves - 1; w >= 0; --w)
            if (s.sums[w]) first = w;
        if (first == 0)
            hi = lo;
        else {
            const int32_t from = min(hi, lo + (first - 1) * width);
            const int32_t to = first < kPlanWaves ? min(hi, lo + first * width) : hi;
            lo = min(from + 1, to);
            hi = to;
        }
    }
    const int32_t c = lo;
    // items of each request, then their places; split requests and their partial slots
    int64_t items[kPerThread], part[kPerThread], split[kPerThread];
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int r = tid * kPerThread + e;
        items[e] = r < R ? (s.off[r] + c - 1) / c : 0;
        part[e] = items[e] > 1 ? items[e] : 0;
        split[e] = items[e] > 1;
    }
    const int64_t n_items = block_scan(items, s.wave_sums);
    block_scan(part, s.wave_sums);
    const int64_t n_split = block_scan(split, s.wave_sums);
    int32_t* work = a.d.schedule + kStepHeader;
    int32_t* splits = work + static_cast<int64_t>(a.items) * kStepItem;
    if (tid == 0) {
        a.d.schedule[0] = static_cast<int32_t>(n_items);
        a.d.schedule[1] = static_cast<int32_t>(n_split);
        a.d.schedule[2] = c;
        a.d.schedule[3] = 0;
    }
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int r = tid * kPerThread + e;
        if (r < R) {
            const int32_t n_steps = s.off[r], n = (n_steps + c - 1) / c;
            const int32_t rows = s.start[r + 1] - s.start[r], len = s.len[r];
            const int32_t keys = len < 0 ? 0 : len + rows;
            if (n > 1) {
                int32_t* at = splits + split[e] * kStepSplit;
                at[0] = r;
                at[1] = static_cast<int32_t>(part[e]);
                at[2] = n;
                at[3] = 0;
            }
            for (int32_t j = 0; j < n; ++j) {
                int32_t* at = work + (items[e] + j) * kStepItem;
                // chunks of nearly equal length, whole steps each
                const int32_t b = static_cast<int32_t>(static_cast<int64_t>(n_steps) * j / n) * kStepKeys;
                const int32_t end = static_cast<int32_t>(static_cast<int64_t>(n_steps) * (j + 1) / n) * kStepKeys;
                at[0] = r;
                at[1] = min(b, keys);
                at[2] = min(end, keys);
                at[3] = n > 1 ? static_cast<int32_t>(part[e]) + j : -1;
                at[4] = max(len, 0);
                at[5] = len < 0 ? 0 : rows;
                at[6] = s.start[r];
                at[7] = rows;
            }
        }
    }
}

__global__ void __launch_bounds__(kPlanThreads) step_plan_kernel(PlanArgs a) {
    __shared__ PlanShared s;
    const kvr_step_desc& d = a.d;
    const int tid = threadIdx.x;
    const int R = d.requests;
    const int32_t P = d.page_size;
    int64_t len[kPerThread], cnt[kPerThread], start[kPerThread], off[kPerThread];
    if (tid == 0) s.taken = 0;
    const int32_t skip = d.free_start ? *d.free_start : 0;
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int r = tid * kPerThread + e;
        len[e] = r < R ? d.lengths[r] : 0;
        cnt[e] = r < R ? d.counts[r] : 0;
        start[e] = cnt[e] > 0 ? cnt[e] : 0;
    }
    const int64_t all_rows = block_scan(start, s.wave_sums);
    const int32_t total = static_cast<int32_t>(all_rows < d.rows ? all_rows : d.rows);
    int32_t status[kPerThread];
    int64_t need[kPerThread];
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        status[e] = KVR_STEP_OK;
        if (len[e] < 0 || cnt[e] < 0 || cnt[e] > d.max_rows || start[e] + cnt[e] > d.rows)
            status[e] = KVR_STEP_INVALID;
        else if (len[e] + cnt[e] > static_cast<int64_t>(d.table_width) * P)
            status[e] = KVR_STEP_TOO_LONG;
        need[e] = status[e] == KVR_STEP_OK ? ((len[e] + cnt[e] + P - 1) >> a.page_log2) - ((len[e] + P - 1) >> a.page_log2)
                                           : 0;
        off[e] = need[e];
    }
    block_scan(off, s.wave_sums);
    const int64_t given = skip < 0 || skip > d.free_count ? 0 : d.free_count - skip;
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) {
        const int r = tid * kPerThread + e;
        if (need[e] > 0) {
            if (off[e] + need[e] > given)
                status[e] = KVR_STEP_NO_PAGES;
            else
                atomicMax(&s.taken, static_cast<int32_t>(off[e] + need[e]));  // a largest value: the order is no matter
        }
        if (r < R) {
            s.start[r] = static_cast<int32_t>(start[e] < d.rows ? start[e] : d.rows);
            // past the free list's end only failed requests, or such as need none
            s.off[r] = static_cast<int32_t>(off[e] < given ? off[e] : given);
            s.len[r] = status[e] == KVR_STEP_OK ? static_cast<int32_t>(len[e]) : -1;
        }
    }
    if (tid == 0) {
        s.start[R] = total;
        s.off[R] = INT32_MAX;
    }
    __syncthreads();
    if (blockIdx.x == static_cast<unsigned>(a.row_blocks)) {
        make_schedule(a, s);
        return;
    }
    if (blockIdx.x == 0) {
#pragma unroll
        for (int e = 0; e < kPerThread; ++e) {
            const int r = tid * kPerThread + e;
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
        const int32_t r = last_at_most(s.off, R - 1, static_cast<int32_t>(p));
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
            const int32_t r = last_at_most(s.start, R - 1, static_cast<int32_t>(i));
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
    return kStepHeader + s.items * kStepItem + (s.partials / 2 + 1) * kStepSplit;
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
    a.target = a.items = 0;
    if (d->schedule) {
        const StepShape s = step_shape(d->requests, d->max_rows, d->q_heads, d->kv_heads);
        a.target = static_cast<int32_t>(s.target);
        a.items = static_cast<int32_t>(s.items);
    }
    step_plan_kernel<<<a.row_blocks + (d->schedule ? 1 : 0), kPlanThreads, 0, as_stream(stream)>>>(a);
    return launch_status();
}
