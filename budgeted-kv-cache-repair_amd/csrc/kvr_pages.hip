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
constexpr int kXcds = 8;

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
// Accepted rows. Row path[i] >= i becomes row i: a thread moves one 16-byte piece of every row, 8 rows read
// before 8 are written. A batch's targets lie below the sources of the rows behind it, so nothing is
// overwritten before it has been read. A block has a request's rows of one tensor, and an XCD an eighth of
// the tensors: the requests' rows of a tensor lie all over it, and an XCD that visits few tensors finds more
// of their addresses' translations (337 rows of 64 requests, 32 layers: 26.6 us with each XCD in all tensors,
// 24.6 so). 88 MB read and written in a graph's 23 us are 3.8 TB/s; with nothing to move the launch takes 8.
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
    int32_t requests;
    int32_t tensors;  // of this launch
};

__global__ void __launch_bounds__(kKeepThreads) keep_rows_kernel(KeepArgs a) {
    __shared__ int64_t from[kKeepRows], to[kKeepRows];
    __shared__ int32_t s_bad;
    const int tid = threadIdx.x;
    const int32_t block = blockIdx.x, of_xcd = block / kXcds;
    const int32_t r = of_xcd % a.requests, tensor = of_xcd / a.requests * kXcds + block % kXcds;
    if (tensor >= a.tensors) return;
    const int32_t start = a.row_starts[r], rows = a.row_starts[r + 1] - start;
    int32_t n = min(a.kept[r], rows);
    if (n <= 0) return;
    const int64_t length = a.positions[start];  // node 0 is the first behind the committed tokens
    if (length < 0) return;
    const int which = tensor & 1;
    char* const pool = a.p.pool[which][tensor >> 1];
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
// Forked requests, one launch: every block finds all of the new requests out by itself (their sources, which
// of them come first, the free pages of the others), so that none waits for another; then the blocks share
// the rows of the new tables and the copies. Copies pass the caches (nontemporal): 22 last pages of 32
// layers, 99 MB read and written, 39.5 us, 5.0 TB/s; 15 of 9 rows, 16 MB, 10.9 us; in a
// graph 15 of 8 rows take 9.8, and 3.7 with nothing to copy: the launch and the reads that find a copy out, each of
// which waits for the one before it. One launch for all instead of one for the plan and one for the copies: 64 beams
// 103 -> 41.6 us (a call; other draws, which copy more pages, up to 50.6).
// ---------------------------------------------------------------------------
constexpr int kForkThreads = 256;
constexpr int kForkMax = KVR_STEP_MAX_REQUESTS;
constexpr int kForkBlocks = 2048;
constexpr int kForkPieces = 4 * kForkThreads;  // 16-byte pieces of a block's copy

struct ForkArgs {
    PoolArgs p;
    kvr_fork_desc d;
    int32_t tensors;   // of this launch
    int32_t chunks;    // copies of a whole page of a tensor
    int32_t tables;    // 1: the launch that writes the new requests
};

__global__ void __launch_bounds__(kForkThreads) fork_kernel(ForkArgs a) {
    extern __shared__ int32_t lds[];
    __shared__ int32_t wave_sums[kForkThreads / 64];
    __shared__ int32_t s_taken;
    const kvr_fork_desc& d = a.d;
    int32_t* const first = lds;                  // [requests] the first output that continues a request
    int32_t* const source = first + d.requests;  // [count] of an output that is one; -1
    int32_t* const length = source + d.count;    // [count]
    int32_t* const own = length + d.count;       // [count] its own last page; -1: none
    int32_t* const copy = own + d.count;         // [count] the outputs that have one, in order
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t log2 = a.p.page_log2, P = 1 << log2;
    const int32_t each = (d.count + kForkThreads - 1) / kForkThreads, from = min(tid * each, d.count);
    const int32_t to = min(from + each, d.count);
    for (int32_t r = tid; r < d.requests; r += kForkThreads) first[r] = INT32_MAX;
    if (tid == 0) s_taken = 0;
    const int32_t skip = d.free_start ? *d.free_start : 0;
    const int32_t given = skip < 0 || skip > d.free_count ? 0 : d.free_count - skip;
    __syncthreads();
    const bool tells = a.tables && blockIdx.x == 0;
    for (int32_t i = from; i < to; ++i) {
        int32_t src = d.sources[i], status = KVR_STEP_OK, len = 0;
        if (src < -1 || src >= d.requests) {
            status = KVR_STEP_INVALID;
        } else if (src >= 0) {
            len = d.lengths[src];
            if (len < 0)
                status = KVR_STEP_INVALID;
            else if (len > static_cast<int64_t>(d.table_width) << log2)
                status = KVR_STEP_TOO_LONG;
            else
                atomicMin(&first[src], i);  // a smallest value: the order is no matter
        }
        source[i] = status == KVR_STEP_OK ? src : -1;
        length[i] = status == KVR_STEP_OK ? len : 0;
        if (tells) d.status[i] = status;
    }
    __syncthreads();
    int32_t mine = 0;
    for (int32_t i = from; i < to; ++i) {
        const int32_t src = source[i], len = length[i];
        int32_t page = -1;
        if (src >= 0 && (len & (P - 1)) && first[src] != i) page = d.tables[src * d.table_stride + (len >> log2)];
        own[i] = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.p.n_pages) ? 0 : -1;
        mine += own[i] == 0;
    }
    int32_t at = mine;
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const int32_t up = __shfl_up(at, s);
        if (lane >= s) at += up;
    }
    if (lane == 63) wave_sums[wave] = at;
    __syncthreads();
    at -= mine;
    for (int w = 0; w < wave; ++w) at += wave_sums[w];
    for (int32_t i = from; i < to; ++i) {
        if (own[i] == 0) {
            if (at < given) {
                own[i] = d.free_pages[skip + at];
                copy[at] = i;
                atomicMax(&s_taken, at + 1);
            } else {
                own[i] = source[i] = -1;
                length[i] = 0;
                if (tells) d.status[i] = KVR_STEP_NO_PAGES;
            }
            ++at;
        }
        if (tells) d.out_lengths[i] = length[i];
    }
    __syncthreads();
    const int32_t copies = s_taken;
    if (tells && tid == 0) *d.pages_taken = copies;
    // ---- the rows of the new tables, a wave each ----
    if (a.tables)
        for (int32_t i = blockIdx.x * (kForkThreads / 64) + wave; i < d.count; i += gridDim.x * (kForkThreads / 64)) {
            const int32_t r = source[i], n = (length[i] + P - 1) >> log2;
            // one that copies has a last page of its own, whatever stands in the free list
            const bool last = (length[i] & (P - 1)) && r >= 0 && first[r] != i;
            for (int32_t c = lane; c < d.table_width; c += 64) {
                int32_t page = c < n ? d.tables[r * d.table_stride + c] : -1;
                if (last && c == n - 1 && static_cast<uint32_t>(page) < static_cast<uint32_t>(a.p.n_pages)) page = own[i];
                d.out_tables[i * d.out_stride + c] = page;
            }
        }
    // ---- the copies: a block has some pieces of a page of one tensor ----
    const int64_t items = static_cast<int64_t>(copies) * a.tensors * a.chunks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int32_t chunk = static_cast<int32_t>(item % a.chunks), rest = static_cast<int32_t>(item / a.chunks);
        const int32_t tensor = rest % a.tensors, i = copy[rest / a.tensors], which = tensor & 1;
        const int32_t rows = length[i] & (P - 1), per_head = rows * a.p.pieces, all = a.p.kv_heads * per_head;
        const int32_t fresh = own[i];
        if (chunk * kForkPieces >= all || static_cast<uint32_t>(fresh) >= static_cast<uint32_t>(a.p.n_pages)) continue;
        const int32_t old = d.tables[source[i] * d.table_stride + (length[i] >> log2)];
        char* const pool = a.p.pool[which][tensor >> 1];
        const int64_t head = a.p.head[which], stride = a.p.row[which];
        const char* const src = pool + (static_cast<int64_t>(old) << log2) * stride;
        char* const dst = pool + (static_cast<int64_t>(fresh) << log2) * stride;
        u32x4 x[4];
        int64_t off[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t c = chunk * kForkPieces + e * kForkThreads + tid;
            const uint32_t h = c / per_head, in = c - h * per_head, row = in / a.p.pieces;
            off[e] = c < static_cast<uint32_t>(all) ? h * head + row * stride + (in - row * a.p.pieces) * 16 : -1;
            if (off[e] >= 0) x[e] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + off[e]));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (off[e] >= 0) __builtin_nontemporal_store(x[e], reinterpret_cast<u32x4*>(dst + off[e]));
    }
}

// ---------------------------------------------------------------------------
// The free list. Small pools and tables: one block with a bit a page in LDS. 4096 entries and pages 7.4 us in
// a graph and 7.5 by calls one after another, with the three launches below 10.6 and 12.4; 16384 of each 11.5
// and 10.2, with three 10.4 and 12.9; 31000 18.4 and 17.0, with three 10.6 and 13.
// ---------------------------------------------------------------------------
constexpr int kFewThreads = 1024;
constexpr int32_t kFewPages = 16384;
constexpr int64_t kFewEntries = 16384;

__global__ void __launch_bounds__(kFewThreads) free_few_kernel(const int32_t* lengths, const int32_t* tables,
                                                               int64_t table_stride, int32_t requests, int32_t width,
                                                               int32_t page_log2, int32_t n_pages, int32_t* list,
                                                               int32_t* start) {
    __shared__ uint64_t used[kFewPages / 64];
    __shared__ int32_t s_word[kFewPages / 64];  // free pages before each word
    __shared__ int32_t s_wave[kFewThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t words = (n_pages + 63) / 64;
    // this thread's word of the map: pages that are none count as used
    if (tid < words) used[tid] = n_pages - tid * 64 < 64 ? ~uint64_t(0) << (n_pages - tid * 64) : 0;
    __syncthreads();
    const int32_t entries = requests * width;
    for (int32_t e = tid; e < entries; e += kFewThreads) {
        const int32_t r = e / width, c = e - r * width, len = lengths[r];
        const int32_t page = tables[r * table_stride + c];
        const bool held = len > 0 && c < static_cast<int32_t>((static_cast<int64_t>(len) + (1 << page_log2) - 1) >> page_log2);
        if (held && static_cast<uint32_t>(page) < static_cast<uint32_t>(n_pages))
            atomicOr(reinterpret_cast<uint32_t*>(used) + (page >> 5), 1u << (page & 31));  // any order: the same bits
    }
    __syncthreads();
    const int32_t mine = tid < words ? __popcll(~used[tid]) : 0;
    int32_t sum = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int32_t up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    if (lane == 63) s_wave[wave] = sum;
    __syncthreads();
    int32_t all = 0;
#pragma unroll
    for (int w = 0; w < kFewThreads / 64; ++w) {
        if (w < wave) sum += s_wave[w];
        all += s_wave[w];
    }
    if (tid < words) s_word[tid] = sum - mine;
    __syncthreads();
    const int32_t first = n_pages - all;
    if (tid == 0) *start = first;
    for (int32_t w = wave; w < words; w += kFewThreads / 64) {
        const uint64_t free = ~used[w];
        const int32_t page = w * 64 + lane;
        if ((free >> lane) & 1) list[first + s_word[w] + __popcll(free & ((uint64_t(1) << lane) - 1))] = page;
        if (page < first) list[page] = -1;
    }
}

// Others, three launches, each a round trip or two: a byte a page says whether a request holds it (many may
// say so at once: the same value, and no atomics), groups of pages count theirs that are free, and each
// writes them behind those of the groups before it and clears its bytes for the next call.
constexpr int kFreeThreads = 256;
constexpr int kFreeGroup = 16 * kFreeThreads;  // pages of a block: 16 bytes a thread

int64_t free_groups(int32_t n_pages) { return ceil_div(n_pages, kFreeGroup); }

// A group's count (at most 4096) as it stands in the workspace: seven bits a byte, the lowest of each zero. What a call
// leaves there is no held page to a call of a larger pool, whose bytes may lie where these counts do.
__device__ inline int32_t pack_count(int32_t n) { return (n & 127) << 1 | (n >> 7) << 9; }
__device__ inline int32_t count_of(int32_t packed) { return (packed >> 1 & 127) | (packed >> 9) << 7; }

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

// Of 16 pages from page0 on those whose bytes are zero (pages past the pool's are none).
__device__ inline uint32_t free_bits(u32x4 x, int64_t page0, int32_t n_pages) {
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) bits |= (((x[e >> 2] >> (8 * (e & 3))) & 1u) ^ 1u) << e;
    const int64_t here = n_pages - page0;
    return here <= 0 ? 0 : here < 16 ? bits & ((1u << here) - 1) : bits;
}

__global__ void __launch_bounds__(kFreeThreads) free_count_kernel(const u32x4* used, int32_t n_pages, int32_t* counts) {
    __shared__ int32_t part[kFreeThreads / 64];
    const int tid = threadIdx.x;
    const int64_t thread = static_cast<int64_t>(blockIdx.x) * kFreeThreads + tid;
    const bool in = thread * 16 < n_pages;
    int32_t n = __popc(free_bits(in ? used[thread] : u32x4{0u, 0u, 0u, 0u}, thread * 16, n_pages));
#pragma unroll
    for (int d = 32; d > 0; d /= 2) n += __shfl_xor(n, d);
    if ((tid & 63) == 0) part[tid >> 6] = n;
    __syncthreads();
    if (tid == 0) counts[blockIdx.x] = pack_count(part[0] + part[1] + part[2] + part[3]);
}

__global__ void __launch_bounds__(kFreeThreads) free_list_kernel(u32x4* used, int32_t n_pages, int32_t groups,
                                                                 const int32_t* counts, int32_t* list, int32_t* start) {
    __shared__ int32_t s_before[kFreeThreads / 64], s_all[kFreeThreads / 64], s_wave[kFreeThreads / 64];
    __shared__ int32_t s_list[kFreeGroup];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int32_t group = blockIdx.x;
    const int64_t thread = static_cast<int64_t>(group) * kFreeThreads + tid;
    const bool in = thread * 16 < n_pages;
    const u32x4 x = in ? used[thread] : u32x4{0u, 0u, 0u, 0u};
    int32_t before = 0, all = 0;
    for (int32_t g = tid; g < groups; g += kFreeThreads) {
        const int32_t n = count_of(counts[g]);
        all += n;
        if (g < group) before += n;
    }
    const uint32_t bits = free_bits(x, thread * 16, n_pages);
    if (in) used[thread] = u32x4{0u, 0u, 0u, 0u};
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
    int32_t here = 0;
#pragma unroll
    for (int w = 0; w < kFreeThreads / 64; ++w) {
        before += s_before[w];
        all += s_all[w];
        if (w < wave) sum += s_wave[w];
        here += s_wave[w];
    }
    const int32_t first = n_pages - all;
    if (group == 0 && tid == 0) *start = first;
    // the group's pages in LDS, so that neighbouring threads write neighbouring values
    int32_t at = sum - __popc(bits);
    for (uint32_t left = bits; left; left &= left - 1) s_list[at++] = static_cast<int32_t>(thread * 16) + __builtin_ctz(left);
    __syncthreads();
    for (int32_t e = tid; e < here; e += kFreeThreads) list[first + before + e] = s_list[e];
    const int32_t page0 = group * kFreeGroup;
    for (int32_t e = tid; e < kFreeGroup; e += kFreeThreads)
        if (static_cast<int64_t>(page0) + e < first) list[page0 + e] = -1;
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
    a.requests = d->requests;
    for (int32_t first = 0; first < p->layers; first += kMaxLayers) {
        const int32_t layers = p->layers - first < kMaxLayers ? p->layers - first : kMaxLayers;
        a.p = pool_args(p, first, layers);
        a.tensors = 2 * layers;
        const int64_t rounds = ceil_div(a.tensors, kXcds);
        keep_rows_kernel<<<static_cast<unsigned>(rounds * kXcds * d->requests), kKeepThreads, 0, as_stream(stream)>>>(a);
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
    if (d->table_stride < d->table_width || d->out_stride < d->table_width) return KVR_E_BAD_STRIDE;
    ForkArgs a;
    a.d = *d;
    const size_t lds = (static_cast<size_t>(d->requests) + 4 * static_cast<size_t>(d->count)) * 4;
    static LdsGrant grant;
    // with room for the static part; the most that any call needs
    if (!grant.ok(fork_kernel, lds <= 64512 ? lds : static_cast<size_t>(kForkMax) * 5 * 4)) return KVR_E_LAUNCH_FAILED;
    for (int32_t first = 0; first < p->layers; first += kMaxLayers) {
        const int32_t layers = p->layers - first < kMaxLayers ? p->layers - first : kMaxLayers;
        a.p = pool_args(p, first, layers);
        a.tensors = 2 * layers;
        a.chunks = static_cast<int32_t>(ceil_div(static_cast<int64_t>(p->kv_heads) * a.p.pieces * p->page_size, kForkPieces));
        a.tables = first == 0;
        const int64_t most = static_cast<int64_t>(d->count) * a.tensors * a.chunks;
        fork_kernel<<<static_cast<unsigned>(most < kForkBlocks ? most : kForkBlocks), kForkThreads, lds, as_stream(stream)>>>(a);
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
    const int32_t page_log2 = __builtin_ctz(static_cast<unsigned>(page_size));
    if (n_pages <= kFewPages && static_cast<int64_t>(requests) * table_width <= kFewEntries) {
        free_few_kernel<<<1, kFewThreads, 0, s>>>(lengths, tables, table_stride, requests, table_width, page_log2, n_pages,
                                                  list, start);
        return launch_status();
    }
    u32x4* const used = static_cast<u32x4*>(workspace);
    int32_t* const counts = reinterpret_cast<int32_t*>(used + ceil_div(n_pages, 16));
    const unsigned groups = static_cast<unsigned>(free_groups(n_pages));
    const int64_t across = ceil_div(table_width, kFreeThreads);
    free_mark_kernel<<<dim3(static_cast<unsigned>(across < 64 ? across : 64), requests), kFreeThreads, 0, s>>>(
        lengths, tables, table_stride, table_width, page_log2, n_pages, reinterpret_cast<uint8_t*>(used));
    free_count_kernel<<<groups, kFreeThreads, 0, s>>>(used, n_pages, counts);
    free_list_kernel<<<groups, kFreeThreads, 0, s>>>(used, n_pages, static_cast<int32_t>(groups), counts, list, start);
    return launch_status();
}
