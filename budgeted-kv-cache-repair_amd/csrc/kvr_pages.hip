// The order of a paged cache between steps: accepted rows moved together
// (kvr_keep_rows), requests continued as several (kvr_fork_requests), the free list
// made from what requests still hold (kvr_free_pages). Copies of bits and whole
// numbers; what bounds the copies is HBM, once there are enough of them, and a few
// dependent round trips before.
#include "kvr_internal.h"
#include "kvr_step.h"
#include "kvrepair_serve.h"

namespace kvr {
namespace {

constexpr int kMaxLayers = 64;  // of a launch: their addresses are kernel arguments

struct PoolArgs {
    char* pool[2][kMaxLayers];  // [K=0 / V=1][layer]
    int64_t head[2], row[2];    // bytes
    int64_t n_slots;
    int32_t kv_heads;
    int32_t pieces;             // 16-byte pieces of a token of one head
    int32_t page_log2;
    int32_t n_pages;
};

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_pools(const kvr_pools* p) {
    if (!p || !p->k || !p->v) return KVR_E_NULL_POINTER;
    if (p->layers <= 0 || p->kv_heads <= 0 || p->row_bytes <= 0 || p->row_bytes % 16 || p->n_slots <= 0)
        return KVR_E_UNSUPPORTED_SHAPE;
    const int32_t P = p->page_size;
    if (P < kStepMinPage || (P & (P - 1)) || p->n_slots % P || p->n_slots / P > INT32_MAX) return KVR_E_UNSUPPORTED_SHAPE;
    // pieces of a page of all heads fit 32 bits
    if (static_cast<int64_t>(p->kv_heads) * (p->row_bytes / 16) * P > INT32_MAX) return KVR_E_UNSUPPORTED_SHAPE;
    if (p->k_head <= 0 || p->k_row <= 0 || p->v_head <= 0 || p->v_row <= 0 || p->k_head % 16 || p->k_row % 16 ||
        p->v_head % 16 || p->v_row % 16)
        return KVR_E_BAD_STRIDE;
    for (int32_t l = 0; l < p->layers; ++l) {
        if (!p->k[l] || !p->v[l]) return KVR_E_NULL_POINTER;
        if (!aligned(p->k[l], 16) || !aligned(p->v[l], 16)) return KVR_E_BAD_STRIDE;
    }
    return KVR_OK;
}

// Layers [first, first + count) of checked pools.
PoolArgs pool_args(const kvr_pools* p, int32_t first, int32_t count) {
    PoolArgs a = {};
    for (int32_t l = 0; l < count; ++l) {
        a.pool[0][l] = static_cast<char*>(p->k[first + l]);
        a.pool[1][l] = static_cast<char*>(p->v[first + l]);
    }
    a.head[0] = p->k_head;
    a.head[1] = p->v_head;
    a.row[0] = p->k_row;
    a.row[1] = p->v_row;
    a.n_slots = p->n_slots;
    a.kv_heads = p->kv_heads;
    a.pieces = p->row_bytes / 16;
    a.page_log2 = __builtin_ctz(static_cast<unsigned>(p->page_size));
    a.n_pages = static_cast<int32_t>(p->n_slots / p->page_size);
    return a;
}

// ---------------------------------------------------------------------------
// Accepted rows. Row path[i] >= i becomes row i: a thread moves one 16-byte piece
// of every row, 8 rows read before 8 are written. A batch's targets lie below the sources
// of the rows behind it, so nothing is overwritten before it has been read.
// ---------------------------------------------------------------------------
constexpr int kKeepThreads = 128;
constexpr int kKeepRows = 128;  // rows whose slots are looked up at a time
constexpr int kKeepBatch = 8;

struct KeepArgs {
    PoolArgs p;
    const int32_t* row_starts;
    const int64_t* slots;
    const int64_t* positions;
    const int32_t* tables;
    int64_t table_stride;
    const int32_t* path;
    const int32_t* kept;
    int32_t table_width;
};

__global__ void __launch_bounds__(kKeepThreads) keep_rows_kernel(KeepArgs a) {
    __shared__ int64_t from[kKeepRows], to[kKeepRows];
    __shared__ int32_t s_bad;
    const int tid = threadIdx.x;
    const int32_t r = blockIdx.x, start = a.row_starts[r], rows = a.row_starts[r + 1] - start;
    int32_t n = min(a.kept[r], rows);
    if (n <= 0) return;
    const int64_t length = a.positions[start];  // node 0 is the first behind the committed tokens
    if (length < 0) return;
    const int which = blockIdx.y & 1;
    char* const pool = a.p.pool[which][blockIdx.y >> 1];
    const int64_t head = a.p.head[which], stride = a.p.row[which];
    const int32_t columns = a.p.kv_heads * a.p.pieces;
    for (int32_t base = 0; base < n; base += kKeepRows) {
        const int32_t here = min(n - base, kKeepRows);
        if (tid == 0) s_bad = here;
        __syncthreads();
        if (tid < here) {
            const int32_t i = base + tid, node = a.path[start + i];
            const int32_t before = i > 0 ? a.path[start + i - 1] : -1;
            if (node <= before || node >= rows || node < i) {
                atomicMin(&s_bad, tid);  // a smallest value: the order is no matter
            } else {
                const int64_t slot = a.slots[start + node], token = length + i, at = token >> a.p.page_log2;
                int64_t target = -1;
                if (at < a.table_width) {
                    const int32_t page = a.tables[r * a.table_stride + at];
                    if (static_cast<uint32_t>(page) < static_cast<uint32_t>(a.p.n_pages))
                        target = (static_cast<int64_t>(page) << a.p.page_log2) +
                                 (token & ((int64_t(1) << a.p.page_log2) - 1));
                }
                const bool move = node != i && slot >= 0 && slot < a.p.n_slots && target >= 0;
                from[tid] = move ? slot : -1;
                to[tid] = target;
            }
        }
        __syncthreads();
        const int32_t good = s_bad;
        for (int32_t c = tid; c < columns; c += kKeepThreads) {
            char* const column = pool + (c / a.p.pieces) * head + (c % a.p.pieces) * 16;
            for (int32_t i = 0; i < good; i += kKeepBatch) {
                u32x4 x[kKeepBatch];
#pragma unroll
                for (int b = 0; b < kKeepBatch; ++b)
                    if (i + b < good && from[i + b] >= 0)
                        x[b] = *reinterpret_cast<const u32x4*>(column + from[i + b] * stride);
#pragma unroll
                for (int b = 0; b < kKeepBatch; ++b)
                    if (i + b < good && from[i + b] >= 0) *reinterpret_cast<u32x4*>(column + to[i + b] * stride) = x[b];
            }
        }
        if (good < here) return;
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------
// Forked requests. First the new tables (every block finds all of them out by
// itself: at most 4096, four a thread), then the copies of last pages: an output whose
// last page is not its source's has one.
// ---------------------------------------------------------------------------
constexpr int kForkThreads = 1024;
constexpr int kForkMax = KVR_STEP_MAX_REQUESTS;
constexpr int kForkPer = kForkMax / kForkThreads;

struct ForkArgs {
    kvr_fork_desc d;
    int32_t page_log2;
    int32_t n_pages;
};

__global__ void __launch_bounds__(kForkThreads) fork_tables_kernel(ForkArgs a) {
    __shared__ int32_t first[kForkMax];   // the first output that continues a request
    __shared__ int32_t source[kForkMax];  // of an output that is one; -1
    __shared__ int32_t pages[kForkMax];   // its pages
    __shared__ int32_t fresh[kForkMax];   // its own last page's place in the free list; -1: none
    __shared__ int32_t wave_sums[kForkThreads / 64];
    __shared__ int32_t s_taken;
    const kvr_fork_desc& d = a.d;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t P = 1 << a.page_log2;
    for (int32_t r = tid; r < d.requests; r += kForkThreads) first[r] = INT32_MAX;
    if (tid == 0) s_taken = 0;
    __syncthreads();
    int32_t src[kForkPer], status[kForkPer], len[kForkPer];
#pragma unroll
    for (int e = 0; e < kForkPer; ++e) {
        const int32_t i = tid * kForkPer + e;
        src[e] = i < d.count ? d.sources[i] : -1;
        status[e] = KVR_STEP_OK;
        len[e] = 0;
        if (src[e] < -1 || src[e] >= d.requests) {
            status[e] = KVR_STEP_INVALID;
        } else if (src[e] >= 0) {
            len[e] = d.lengths[src[e]];
            if (len[e] < 0)
                status[e] = KVR_STEP_INVALID;
            else if (len[e] > static_cast<int64_t>(d.table_width) << a.page_log2)
                status[e] = KVR_STEP_TOO_LONG;
            else
                atomicMin(&first[src[e]], i);  // a smallest value: the order is no matter
        }
        if (status[e] != KVR_STEP_OK) {
            src[e] = -1;
            len[e] = 0;
        }
    }
    __syncthreads();
    const int32_t skip = d.free_start ? *d.free_start : 0;
    const int32_t given = skip < 0 || skip > d.free_count ? 0 : d.free_count - skip;
    int32_t need[kForkPer], mine = 0;
#pragma unroll
    for (int e = 0; e < kForkPer; ++e) {
        const int32_t i = tid * kForkPer + e;
        need[e] = 0;
        if (src[e] >= 0 && (len[e] & (P - 1)) && first[src[e]] != i) {
            const int32_t page = d.tables[src[e] * d.table_stride + (len[e] >> a.page_log2)];
            need[e] = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.n_pages);
        }
        mine += need[e];
    }
    int32_t sum = mine;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const int32_t up = __shfl_up(sum, s);
        if (lane >= s) sum += up;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    int32_t at = sum - mine;
    for (int w = 0; w < wave; ++w) at += wave_sums[w];
#pragma unroll
    for (int e = 0; e < kForkPer; ++e) {
        const int32_t i = tid * kForkPer + e;
        if (i >= d.count) break;
        int32_t place = -1;
        if (need[e]) {
            if (at < given) {
                place = at;
                atomicMax(&s_taken, at + 1);
            } else {
                status[e] = KVR_STEP_NO_PAGES;
                src[e] = -1;
                len[e] = 0;
            }
            ++at;
        }
        source[i] = src[e];
        pages[i] = (len[e] + P - 1) >> a.page_log2;
        fresh[i] = place;
        if (blockIdx.x == 0) {
            d.out_lengths[i] = len[e];
            d.status[i] = status[e];
        }
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) *d.pages_taken = s_taken;
    // the rows of the new tables, a wave each
    for (int32_t i = blockIdx.x * (kForkThreads / 64) + wave; i < d.count; i += gridDim.x * (kForkThreads / 64)) {
        const int32_t r = source[i], n = pages[i], own = fresh[i];
        for (int32_t c = lane; c < d.table_width; c += 64)
            d.out_tables[i * d.out_stride + c] = c >= n                    ? -1
                                                 : own >= 0 && c == n - 1 ? d.free_pages[skip + own]
                                                                           : d.tables[r * d.table_stride + c];
    }
}

constexpr int kCopyThreads = 256;
constexpr int kCopyRows = 64;  // of a page, a block

struct CopyArgs {
    PoolArgs p;
    const int32_t* sources;
    const int32_t* out_lengths;
    const int32_t* tables;
    const int32_t* out_tables;
    int64_t table_stride, out_stride;
};

__global__ void __launch_bounds__(kCopyThreads) fork_copy_kernel(CopyArgs a) {
    const int32_t i = blockIdx.x, len = a.out_lengths[i];
    const int32_t part = len & ((1 << a.p.page_log2) - 1), at = len >> a.p.page_log2;
    const int32_t row0 = blockIdx.z * kCopyRows, rows = min(part - row0, kCopyRows);
    if (rows <= 0) return;  // an empty request, or whole pages only
    const int32_t old = a.tables[a.sources[i] * a.table_stride + at], own = a.out_tables[i * a.out_stride + at];
    if (old == own || static_cast<uint32_t>(old) >= static_cast<uint32_t>(a.p.n_pages) ||
        static_cast<uint32_t>(own) >= static_cast<uint32_t>(a.p.n_pages))
        return;
    const int which = blockIdx.y & 1;
    char* const pool = a.p.pool[which][blockIdx.y >> 1];
    const int64_t head = a.p.head[which], stride = a.p.row[which];
    const char* const src = pool + ((static_cast<int64_t>(old) << a.p.page_log2) + row0) * stride;
    char* const dst = pool + ((static_cast<int64_t>(own) << a.p.page_log2) + row0) * stride;
    const int32_t per_head = rows * a.p.pieces, all = a.p.kv_heads * per_head;
    for (int32_t c = threadIdx.x; c < all; c += kCopyThreads) {
        const int32_t h = c / per_head, rest = c % per_head;
        const int64_t off = h * head + (rest / a.p.pieces) * stride + rest % a.p.pieces * 16;
        *reinterpret_cast<u32x4*>(dst + off) = *reinterpret_cast<const u32x4*>(src + off);
    }
}

// ---------------------------------------------------------------------------
// The free list: a byte a page says whether a request holds it (many may say so at
// once: the same value, and no atomics), groups of pages count theirs that are
// free, and each writes them behind those of the groups before it.
// ---------------------------------------------------------------------------
constexpr int kFreeThreads = 256;
constexpr int kFreeGroup = 16 * kFreeThreads;  // pages of a block: 16 bytes a thread

int64_t free_groups(int32_t n_pages) { return ceil_div(n_pages, kFreeGroup); }

__global__ void __launch_bounds__(kFreeThreads) free_clear_kernel(u32x4* used, int64_t count) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * kFreeThreads + threadIdx.x;
    if (i < count) used[i] = u32x4{0u, 0u, 0u, 0u};
}

__global__ void __launch_bounds__(kFreeThreads) free_mark_kernel(const int32_t* lengths, const int32_t* tables,
                                                                 int64_t table_stride, int32_t table_width,
                                                                 int32_t page_log2, int32_t n_pages, uint8_t* used) {
    const int32_t r = blockIdx.y, len = lengths[r];
    if (len <= 0) return;
    const int64_t have = (static_cast<int64_t>(len) + (1 << page_log2) - 1) >> page_log2;
    const int32_t n = have < table_width ? static_cast<int32_t>(have) : table_width;
    for (int32_t c = blockIdx.x * kFreeThreads + threadIdx.x; c < n; c += gridDim.x * kFreeThreads) {
        const int32_t page = tables[r * table_stride + c];
        if (static_cast<uint32_t>(page) < static_cast<uint32_t>(n_pages)) used[page] = 1;
    }
}

// Bytes that are zero among this thread's 16 pages from page0 on (those past the pool's are not).
__device__ inline uint32_t free_bits(const u32x4* used, int64_t thread, int32_t n_pages) {
    const int64_t page0 = thread * 16;
    if (page0 >= n_pages) return 0;
    const u32x4 x = used[thread];
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) bits |= (((x[e >> 2] >> (8 * (e & 3))) & 1u) ^ 1u) << e;
    return n_pages - page0 < 16 ? bits & ((1u << (n_pages - page0)) - 1) : bits;
}

__global__ void __launch_bounds__(kFreeThreads) free_count_kernel(const u32x4* used, int32_t n_pages, int32_t* counts) {
    __shared__ int32_t part[kFreeThreads / 64];
    const int tid = threadIdx.x;
    int32_t n = __popc(free_bits(used, static_cast<int64_t>(blockIdx.x) * kFreeThreads + tid, n_pages));
#pragma unroll
    for (int d = 32; d > 0; d /= 2) n += __shfl_xor(n, d);
    if ((tid & 63) == 0) part[tid >> 6] = n;
    __syncthreads();
    if (tid == 0) counts[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

__global__ void __launch_bounds__(kFreeThreads) free_list_kernel(const u32x4* used, int32_t n_pages, int32_t groups,
                                                                 const int32_t* counts, int32_t* list, int32_t* start) {
    __shared__ int32_t s_before[kFreeThreads / 64], s_all[kFreeThreads / 64], s_wave[kFreeThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t group = blockIdx.x;
    int32_t before = 0, all = 0;
    for (int32_t g = tid; g < groups; g += kFreeThreads) {
        const int32_t n = counts[g];
        all += n;
        if (g < group) before += n;
    }
    const int64_t thread = static_cast<int64_t>(group) * kFreeThreads + tid;
    const uint32_t bits = free_bits(used, thread, n_pages);
    int32_t sum = __popc(bits);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int32_t up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
        before += __shfl_xor(before, d);
        all += __shfl_xor(all, d);
    }
    if (lane == 63) s_wave[wave] = sum;
    if (lane == 0) {
        s_before[wave] = before;
        s_all[wave] = all;
    }
    __syncthreads();
    before = all = 0;
#pragma unroll
    for (int w = 0; w < kFreeThreads / 64; ++w) {
        before += s_before[w];
        all += s_all[w];
        if (w < wave) sum += s_wave[w];
    }
    const int32_t first = n_pages - all;
    if (group == 0 && tid == 0) *start = first;
    int32_t at = first + before + sum - __popc(bits);
    for (int e = 0; e < 16; ++e) {
        const int64_t page = thread * 16 + e;
        if ((bits >> e) & 1) list[at++] = static_cast<int32_t>(page);
        if (page < first) list[page] = -1;
    }
}

}  // namespace
}  // namespace kvr

using namespace kvr;

extern "C" int64_t kvr_pools_size(void) { return sizeof(kvr_pools); }

extern "C" int kvr_keep_rows(const kvr_pools* p, const kvr_step_desc* d, const int32_t* path, const int32_t* kept,
                             void* stream) {
    int st = check_pools(p);
    if (st == KVR_OK) st = check_step(d);
    if (st != KVR_OK) return st;
    if (!path || !kept) return KVR_E_NULL_POINTER;
    if (p->page_size != d->page_size || p->n_slots != d->n_slots) return KVR_E_INVALID_ARGUMENT;
    KeepArgs a;
    a.row_starts = d->row_starts;
    a.slots = d->slots;
    a.positions = d->positions;
    a.tables = d->tables;
    a.table_stride = d->table_stride;
    a.path = path;
    a.kept = kept;
    a.table_width = d->table_width;
    for (int32_t first = 0; first < p->layers; first += kMaxLayers) {
        const int32_t layers = p->layers - first < kMaxLayers ? p->layers - first : kMaxLayers;
        a.p = pool_args(p, first, layers);
        keep_rows_kernel<<<dim3(d->requests, 2 * layers), kKeepThreads, 0, as_stream(stream)>>>(a);
    }
    return launch_status();
}

extern "C" int64_t kvr_fork_desc_size(void) { return sizeof(kvr_fork_desc); }

extern "C" int kvr_fork_requests(const kvr_pools* p, const kvr_fork_desc* d, void* stream) {
    const int st = check_pools(p);
    if (st != KVR_OK) return st;
    if (!d || !d->sources || !d->lengths || !d->tables || !d->out_lengths || !d->out_tables || !d->status ||
        !d->pages_taken || (d->free_count > 0 && !d->free_pages))
        return KVR_E_NULL_POINTER;
    if (d->count <= 0 || d->count > kForkMax || d->requests <= 0 || d->requests > kForkMax || d->table_width <= 0 ||
        d->free_count < 0)
        return KVR_E_UNSUPPORTED_SHAPE;
    if (static_cast<int64_t>(d->table_width) * p->page_size > (int64_t(1) << 30)) return KVR_E_UNSUPPORTED_SHAPE;
    const unsigned parts = static_cast<unsigned>(ceil_div(p->page_size, kCopyRows));
    if (parts > 65535) return KVR_E_UNSUPPORTED_SHAPE;
    if (d->table_stride < d->table_width || d->out_stride < d->table_width) return KVR_E_BAD_STRIDE;
    ForkArgs f;
    f.d = *d;
    f.page_log2 = __builtin_ctz(static_cast<unsigned>(p->page_size));
    f.n_pages = static_cast<int32_t>(p->n_slots / p->page_size);
    const int64_t blocks = ceil_div(d->count, kForkThreads / 64);
    fork_tables_kernel<<<static_cast<unsigned>(blocks), kForkThreads, 0, as_stream(stream)>>>(f);
    CopyArgs a;
    a.sources = d->sources;
    a.out_lengths = d->out_lengths;
    a.tables = d->tables;
    a.out_tables = d->out_tables;
    a.table_stride = d->table_stride;
    a.out_stride = d->out_stride;
    for (int32_t first = 0; first < p->layers; first += kMaxLayers) {
        const int32_t layers = p->layers - first < kMaxLayers ? p->layers - first : kMaxLayers;
        a.p = pool_args(p, first, layers);
        fork_copy_kernel<<<dim3(d->count, 2 * layers, parts), kCopyThreads, 0, as_stream(stream)>>>(a);
    }
    return launch_status();
}

extern "C" int64_t kvr_free_pages_workspace_bytes(int32_t n_pages) {
    if (n_pages <= 0) return KVR_E_UNSUPPORTED_SHAPE;
    return ceil_div(n_pages, 16) * 16 + free_groups(n_pages) * 4;
}

extern "C" int kvr_free_pages(const int32_t* lengths, const int32_t* tables, int64_t table_stride, int32_t requests,
                              int32_t table_width, int32_t page_size, int32_t n_pages, int32_t* list, int32_t* start,
                              void* workspace, int64_t workspace_bytes, void* stream) {
    const int64_t need = kvr_free_pages_workspace_bytes(n_pages);
    if (need < 0) return static_cast<int>(need);
    if (requests <= 0 || requests > KVR_STEP_MAX_REQUESTS || table_width <= 0 || page_size < kStepMinPage ||
        (page_size & (page_size - 1)))
        return KVR_E_UNSUPPORTED_SHAPE;
    if (table_stride < table_width) return KVR_E_BAD_STRIDE;
    if (!lengths || !tables || !list || !start) return KVR_E_NULL_POINTER;
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < need) return KVR_E_WORKSPACE_TOO_SMALL;
    hipStream_t s = as_stream(stream);
    u32x4* const used = static_cast<u32x4*>(workspace);
    const int64_t words = ceil_div(n_pages, 16);
    int32_t* const counts = reinterpret_cast<int32_t*>(used + words);
    const unsigned groups = static_cast<unsigned>(free_groups(n_pages));
    free_clear_kernel<<<groups, kFreeThreads, 0, s>>>(used, words);
    const unsigned across = static_cast<unsigned>(ceil_div(table_width, kFreeThreads) < 64 ? ceil_div(table_width, kFreeThreads) : 64);
    free_mark_kernel<<<dim3(across, requests), kFreeThreads, 0, s>>>(
        lengths, tables, table_stride, table_width, __builtin_ctz(static_cast<unsigned>(page_size)), n_pages,
        reinterpret_cast<uint8_t*>(used));
    free_count_kernel<<<groups, kFreeThreads, 0, s>>>(used, n_pages, counts);
    free_list_kernel<<<groups, kFreeThreads, 0, s>>>(used, n_pages, static_cast<int32_t>(groups), counts, list, start);
    return launch_status();
}
