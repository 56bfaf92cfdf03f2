// Attention of chunks of new tokens (kvr_step_plan.hip's rows, any number a request)
// over each request's paged cache:
//   out[h, t] = softmax_{j <= L + t}(scale q[h, t] . k[h / G, slot(j)]) @ v[h / G, slot(j)]
//
// What bounds it: the matrix work, 4 D operations a query row and key, from some 100 query rows of
// a KV head on; below, the read of K and V, each once for the 256 query rows (token x query head of
// the KV head) of a tile, and the latency of two launches. A work list shares all tiles' steps of
// 128 keys evenly among one worker a CU and KV head, so that a few long tiles or many of unequal
// length keep all CUs; a tile that is cut between workers leaves partial (m, l, O), which
// chunk_merge_kernel joins.
//
// A block is eight waves, two a SIMD, each with 32 of the 256 rows: one wave's exponentials then
// run while the other's matrix instructions do, which a wave's own order can not give (some five
// vector instructions hide behind a 32x32x16 product, and a sub-tile has twice as many a product).
// K and V go by asynchronous loads straight to LDS, 64 keys a stage, three stages ahead in a ring
// of four: one barrier a stage, for no wave writes what another still reads. S^T = K Q^T and O^T +=
// V^T P^T: a lane then has all its scores in one row, its maximum and sum need one exchange at the
// end, and P is the second product's operand as it stands, without a way through LDS; V is read
// transposed. Fp32 statistics, one pass with a running maximum that moves only when a score exceeds
// it by 2^8 (fp16: 2^3). P is rounded to the inputs' type before it weighs V (its low half would
// cost the second product again) and is summed as rounded, so that the weights of a row add up to
// one; in fp16 a power of two lifts it above the type's smallest steps.
//
// Measured: 4096 rows over 28672 + 4096 tokens, 32 / 8 heads of 128, bf16: 1754 - 1861 us, 1.11 - 1.18 PFLOP/s (a
// library product of 8192^3 1.27 to 1.46; the clock falls to 1.7 - 1.95 GHz under either; the
// matrix units are busy 58% of the CUs' cycles), 294 MB read from HBM where K and V are 134, each
// by some XCDs; 20 requests of 1 to 1500 rows over up to 8192 tokens 1077 - 1192 us, 1.0 PFLOP/s;
// 96 rows over 2048 tokens 18 us + 4 us of the merge; five requests with heads of 64 (half the
// matrix work for each exponential) 64 - 75 us, 0.45 - 0.52 PFLOP/s. Four waves of 64 rows, one a SIMD,
// which read each fragment of K and V once for two products, were faster only on the first (1847 us
// to 1917, tiles not yet dealt by requests); the others took 1304 us to 1261, 23.0 to 20.9 and 93
// to 73.
#include "kvr_attention_tiles.h"
#include "kvr_step.h"
#include "kvrepair_serve.h"

#include <type_traits>

namespace kvr {
namespace {

typedef const __attribute__((address_space(4))) int32_t uniform_i32;  // read through the scalar cache
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr int kChunkWaves = 8;
constexpr int kChunkThreads = 64 * kChunkWaves;
constexpr int kWaveRows = 32;
constexpr int kTileRows = kWaveRows * kChunkWaves;  // query rows of a block
constexpr int kSub = 32;                            // keys of a sub-tile
constexpr int kRowAlign = 256;                      // LDS addresses of stages: whole rows of K and V
constexpr int kVoteLds = 256;                       // static LDS, of the block's votes

// ---------------------------------------------------------------------------
// The work list. A request of T rows has ceil(T G / 256) tiles; a tile whose last row sees n keys
// is ceil(n / 128) + 1 units (one for its start). Tiles are put in order, those of the longest
// requests first, and dealt out to the workers of a KV head, one to each in turn, there and back:
// those of a request then run at the same time and read its K and V from one XCD's L2. As many
// rounds are dealt as leave no worker with more than its even share; what is left of the line of
// tiles is cut where the workers' shares end, so that all end together. Where dealing out all tiles
// leaves no worker with more than 1 / 32 and 8 units above its share, none is cut: partial results
// of a tile are 130 KB written and read again (6 requests of 100 to 900 rows 81.6 us cut, 74.2 not;
// 2048 rows over no tokens 68.1 and 66.3; with 12 units 4 requests of 500 to 700 rows, heads of 64,
// 72.0 instead of 70.4). A cut tile's pieces are consecutive workers'; the first has partial slot 2
// worker + 1, the others, each the first of its worker's cut pieces, 2 worker.
//
// int32: header {items, cut tiles, units of a share, tiles, rounds dealt, 0, ...}; workers + 1
// x {first item}, padded to 8; items x {request, first key, end key, partial slot or -1, committed
// tokens, rows (failed requests: minus rows), first packed row, first query row}; cut tiles x {worker of the
// first piece, pieces, first packed row, first query row, rows, 0, 0, 0}; tiles + 1 x {first unit}.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 1024;
constexpr int kPlanPer = KVR_STEP_MAX_REQUESTS / kPlanThreads;

struct ChunkShape {
    int64_t workers;
    int64_t tiles;     // room
    int64_t items;     // one a tile, and one more at each share's end
    int64_t partials;
    int64_t splits;
    int64_t ints;
};

ChunkShape chunk_shape(const kvr_step_desc* d, int32_t q_heads, int32_t kv_heads) {
    const int64_t group = q_heads / kv_heads;
    ChunkShape s;
    s.workers = kv_heads <= kStepCus ? kStepCus / kv_heads : 1;
    s.tiles = static_cast<int64_t>(d->rows) * group / kTileRows + d->requests;
    s.items = s.tiles + s.workers;
    s.partials = s.workers > 1 ? 2 * s.workers : 0;
    s.splits = s.tiles < s.workers ? s.tiles : s.workers;
    s.ints = kStepHeader + step_worker_ints(s.workers) + (s.items + s.splits) * kStepItem + s.tiles + 1;
    return s;
}

// Sizes of a chunk plan that 32 bits and the work list hold (a status).
int check_chunk(const kvr_step_desc* d, int32_t q_heads, int32_t kv_heads) {
    const int st = check_step(d);
    if (st != KVR_OK) return st;
    if (d->parents || q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads || q_heads > 65536)
        return KVR_E_UNSUPPORTED_SHAPE;
    const int64_t keys = static_cast<int64_t>(d->table_width) * d->page_size;
    if (static_cast<int64_t>(d->rows) * (q_heads / kv_heads) > INT32_MAX - kTileRows) return KVR_E_UNSUPPORTED_SHAPE;
    if (chunk_shape(d, q_heads, kv_heads).tiles * (keys / kStepKeys + 2) > (int64_t(1) << 30))
        return KVR_E_UNSUPPORTED_SHAPE;
    return KVR_OK;
}

struct ChunkPlanArgs {
    const int32_t* lengths;
    const int32_t* status;
    const int32_t* row_starts;
    int32_t* schedule;
    int32_t requests;
    int32_t group;
    int32_t workers;
    int32_t items;
    int32_t splits;
};

constexpr int kSorted = kPlanThreads;  // most requests that are put in order: one a thread
constexpr int kMaxWorkers = kStepCus;
constexpr int32_t kCutUnits = 8;

struct ChunkPlanShared {
    int32_t tile[KVR_STEP_MAX_REQUESTS + 1];  // first tile of each request, in the tiles' order
    int32_t request[KVR_STEP_MAX_REQUESTS];   // ... and which it is
    int64_t keys[kSorted];
    int32_t cap[kMaxWorkers + 1];             // first unit of each worker's cut of the line
    int32_t item[kMaxWorkers];                // ... first item
    int32_t wave_sums[kPlanThreads / 64];
    int32_t rounds, top;
};

// Exclusive sum over the block of one value a thread; returns the total too.
__device__ inline int32_t block_exclusive(int32_t x, int32_t* wave_sums, int32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int32_t sum = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int32_t up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    if (lane == 63) wave_sums[wave] = sum;
    __syncthreads();
    int32_t before = sum - x;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 64; ++w) {
        const int32_t s = wave_sums[w];
        if (w < wave) before += s;
        total += s;
    }
    __syncthreads();
    return before;
}

__global__ void __launch_bounds__(kPlanThreads) chunk_schedule_kernel(ChunkPlanArgs a) {
    __shared__ ChunkPlanShared s;
    const int tid = threadIdx.x, R = a.requests, W = a.workers;
    auto rows_of = [&](int32_t r) { return a.row_starts[r + 1] - a.row_starts[r]; };
    auto failed = [&](int32_t r) { return a.status[r] != KVR_STEP_OK; };
    // one tile of no keys for a failed request's rows
    auto tiles_of = [&](int32_t r) {
        const int32_t rows = rows_of(r);
        return rows == 0 ? 0 : failed(r) ? 1 : (rows * a.group + kTileRows - 1) / kTileRows;
    };
    // ---- the requests' order ----
    if (R <= kSorted) {
        // a bitonic sort, the longest first, one request a thread: partners of one wave by shuffles, others through LDS
        // (counting each one's rank took 38 us for 1024 requests, this 8)
        // Unsorted: 20 requests of 1 to 1500 rows 1157 us instead of 1118, 600 of 1 to 200 1070 instead of 1033, 1000
        // of 1 to 60 512 instead of 503.
        int64_t key = -1;
        if (tid < R) key = (static_cast<int64_t>(failed(tid) ? 0 : a.lengths[tid] + rows_of(tid)) << 10) | (kSorted - 1 - tid);
        int32_t n = 1;
        while (n < R) n *= 2;
#pragma unroll 1
        for (int32_t size = 2; size <= n; size *= 2)
#pragma unroll 1
            for (int32_t apart = size / 2; apart > 0; apart /= 2) {
                int64_t other;
                if (apart < 64) {
                    other = __shfl_xor(key, apart);
                } else {
                    s.keys[tid] = key;
                    __syncthreads();
                    other = s.keys[tid ^ apart];
                    __syncthreads();
                }
                const bool larger = ((tid & apart) == 0) == ((tid & size) == 0);
                key = (other > key) == larger ? other : key;
            }
        if (tid < R) s.request[tid] = kSorted - 1 - static_cast<int32_t>(key & (kSorted - 1));
    } else {
        for (int32_t r = tid; r < R; r += kPlanThreads) s.request[r] = r;
    }
    __syncthreads();
    int32_t tiles[kPlanPer], mine = 0, n_tiles;
#pragma unroll
    for (int e = 0; e < kPlanPer; ++e) {
        const int i = tid * kPlanPer + e;
        tiles[e] = i < R ? tiles_of(s.request[i]) : 0;
        mine += tiles[e];
    }
    int32_t at = block_exclusive(mine, s.wave_sums, n_tiles);
#pragma unroll
    for (int e = 0; e < kPlanPer; ++e) {
        const int i = tid * kPlanPer + e;
        if (i < R) s.tile[i] = at;
        at += tiles[e];
    }
    if (tid == 0) {
        s.tile[R] = n_tiles;
        s.rounds = INT32_MAX;
        s.top = 0;
    }
    __syncthreads();
    int32_t* const first_of = a.schedule + kStepHeader;
    int32_t* const work = first_of + step_worker_ints(W);
    int32_t* const cuts = work + static_cast<int64_t>(a.items) * kStepItem;
    int32_t* const units = cuts + static_cast<int64_t>(a.splits) * kStepItem;
    struct Tile {
        int32_t request, first, keys;  // its first query row, the keys that its last row sees
    };
    auto tile_at = [&](int32_t t) -> Tile {
        // the last request whose first tile is at or before t: one with tiles; its last tile, the longest, is first
        int32_t lo = 0, hi = R;
        while (hi - lo > 1) {
            const int32_t mid = (lo + hi) >> 1;
            if (s.tile[mid] <= t)
                lo = mid;
            else
                hi = mid;
        }
        const int32_t r = s.request[lo];
        if (failed(r)) return {r, 0, 0};
        const int32_t first = (s.tile[lo + 1] - 1 - t) * kTileRows;
        return {r, first, a.lengths[r] + (min(first + kTileRows, rows_of(r) * a.group) - 1) / a.group + 1};
    };
    // ---- each tile's first unit ----
    int32_t all = 0;
    for (int32_t base = 0; base < n_tiles; base += kPlanThreads) {
        const int32_t t = base + tid;
        const int32_t n = t < n_tiles ? 1 + (tile_at(t).keys + kStepKeys - 1) / kStepKeys : 0;
        int32_t total;
        const int32_t before = block_exclusive(n, s.wave_sums, total);
        if (t < n_tiles) units[t] = all + before;
        all += total;
    }
    if (tid == 0) units[n_tiles] = all;
    __syncthreads();
    // ---- rounds that are dealt out ----
    const int32_t even = (all + W - 1) / W, every = (n_tiles + W - 1) / W;
    auto dealt = [&](int32_t k) { return k * W + (k & 1 ? W - 1 - tid : tid); };  // this worker's tile of round k
    // each(k, units of this worker's tile of round k) for the first n rounds
    auto tiles_dealt = [&](int32_t n, auto each) {
        constexpr int kAhead = 16;  // loads in flight
        for (int32_t k0 = 0; k0 < n; k0 += kAhead) {
            int32_t u[kAhead];
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                const int32_t t = dealt(min(k0 + e, n - 1));
                u[e] = t < n_tiles ? units[t + 1] - units[t] : 0;
            }
#pragma unroll
            for (int e = 0; e < kAhead; ++e)
                if (k0 + e < n) each(k0 + e, u[e]);
        }
    };
    if (tid < W) {
        int32_t load = 0, fits = -1;
        tiles_dealt(every, [&](int32_t k, int32_t u) {
            load += u;
            if (load > even && fits < 0) fits = k;
        });
        atomicMin(&s.rounds, fits < 0 ? every : fits);  // smallest and largest values: the order is no matter
        atomicMax(&s.top, load);
    }
    __syncthreads();
    // a last round that is not whole is dealt only with all
    int32_t rounds = min(s.rounds, n_tiles / W);
    if (n_tiles >= W && s.top <= even + even / 32 + kCutUnits) rounds = every;
    const int32_t share = rounds > 0 && rounds < every ? even + 1 : max(even, 1);  // each has a unit of the line
    const int32_t line = min(rounds * W, n_tiles), line0 = units[line], rest = all - line0;
    int32_t load = 0;
    if (tid < W) tiles_dealt(rounds, [&](int32_t, int32_t u) { load += u; });
    int32_t total;
    const int32_t cap0 = block_exclusive(tid < W && rest > 0 ? share - load : 0, s.wave_sums, total);
    if (tid < W) s.cap[tid] = min(cap0, rest);
    if (tid == 0) s.cap[W] = rest;
    __syncthreads();
    // ---- each worker's items ----
    const bool works = tid < W;
    const int32_t from = works ? s.cap[tid] : 0, to = works ? s.cap[tid + 1] : 0;
    int32_t t0 = line;  // the tile of the line that holds `from`
    if (from < to) {
        int32_t lo = line, hi = n_tiles;
        while (hi - lo > 1) {
            const int32_t mid = (lo + hi) >> 1;
            if (units[mid] - line0 <= from)
                lo = mid;
            else
                hi = mid;
        }
        t0 = lo;
    }
    // steps [begin, end) of tile t, which starts at unit u of the line, that are this worker's; empty ones are no piece
    auto piece = [&](int32_t u, int32_t steps, int32_t& begin, int32_t& end) -> bool {
        begin = min(max(from - u - 1, 0), steps);
        end = min(max(to - u - 1, 0), steps);
        return steps > 0 ? begin < end : from <= u && u < to;
    };
    const int32_t whole_tiles = works && rounds > 0 ? rounds - (dealt(rounds - 1) >= n_tiles) : 0;
    int32_t count = whole_tiles, cut = 0;
    if (works) {
        for (int32_t t = t0; t < n_tiles && from < to && units[t] - line0 < to; ++t) {
            int32_t begin, end;
            const int32_t u = units[t] - line0, steps = units[t + 1] - units[t] - 1;
            if (!piece(u, steps, begin, end)) continue;
            ++count;
            cut += begin == 0 && end < steps;
        }
    }
    int32_t n_items, n_cut;
    int32_t item = block_exclusive(count, s.wave_sums, n_items);
    const int32_t place = block_exclusive(cut, s.wave_sums, n_cut);
    if (works) s.item[tid] = first_of[tid] = item;
    item += whole_tiles;
    if (tid == 0) {
        first_of[W] = n_items;
        a.schedule[0] = n_items;
        a.schedule[1] = n_cut;
        a.schedule[2] = share;
        a.schedule[3] = n_tiles;
        a.schedule[4] = rounds;
    }
    auto put = [&](int32_t item, int32_t t, int32_t begin, int32_t end, int32_t part) -> Tile {
        const Tile tile = tile_at(t);
        const int32_t rows = rows_of(tile.request);
        const bool none = failed(tile.request);
        int32_t* const out = work + static_cast<int64_t>(item) * kStepItem;
        out[0] = tile.request;
        out[1] = min(begin * kStepKeys, tile.keys);
        out[2] = min(end * kStepKeys, tile.keys);
        out[3] = part;
        out[4] = none ? 0 : a.lengths[tile.request];
        out[5] = none ? -rows : rows;
        out[6] = a.row_starts[tile.request];
        out[7] = tile.first;
        return tile;
    };
    __syncthreads();
    for (int32_t t = tid; t < line; t += kPlanThreads) {
        const int32_t k = t / W, turn = t - k * W;
        put(s.item[k & 1 ? W - 1 - turn : turn] + k, t, 0, units[t + 1] - units[t] - 1, -1);
    }
    if (!works) return;
    for (int32_t t = t0; t < n_tiles && from < to && units[t] - line0 < to; ++t) {
        int32_t begin, end;
        const int32_t u = units[t] - line0, steps = units[t + 1] - units[t] - 1;
        if (!piece(u, steps, begin, end)) continue;
        const bool whole = begin == 0 && end == steps;
        const Tile tile = put(item++, t, begin, end, whole ? -1 : begin == 0 ? step_partial(tid, 0) : step_partial(tid - 1, 1));
        if (whole || begin > 0) continue;
        // its last step is the worker's whose cut holds that unit
        int32_t lo = tid, hi = W;
        while (hi - lo > 1) {
            const int32_t mid = (lo + hi) >> 1;
            if (s.cap[mid] <= u + steps)
                lo = mid;
            else
                hi = mid;
        }
        int32_t* const p = cuts + static_cast<int64_t>(place) * kStepItem;
        p[0] = tid;
        p[1] = lo - tid + 1;
        p[2] = a.row_starts[tile.request];
        p[3] = tile.first;
        p[4] = rows_of(tile.request);
    }
}

// ---------------------------------------------------------------------------
// Attention.
// ---------------------------------------------------------------------------
struct ChunkArgs {
    const char* q;
    const char* k;
    const char* v;
    char* out;
    int64_t qs[2], os[2];           // {head, row} element strides
    int64_t k_head, v_head;         // bytes
    uint32_t k_row, v_row;          // bytes of a row's stride
    uint32_t k_page, v_page;        // ... of a page
    const int32_t* schedule;
    const int32_t* tables;
    float* part_o;                  // [partial][kv head][256][D], unnormalised
    float* part_ml;                 // ... [2]: running maximum (log2 units) and sum (-1: scores of -inf alone)
    int64_t table_stride;
    const int32_t* row_starts;
    int32_t items;
    int32_t workers;
    int32_t requests;
    int32_t rows;
    int32_t zero_rest;
    int32_t page_log2;
    int32_t n_pages;
    int32_t kv_heads;
    int32_t group;
    float scale_log2;               // scale * log2(e)
};

template <typename T> struct wide_mma;
template <> struct wide_mma<bf16_t> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    __device__ static inline f32x16 mma(v8 a, v8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
    // sum + the two packed values
    __device__ static inline float add2(uint32_t p, float sum) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, 0x3f803f80u), sum, false);
    }
};
template <> struct wide_mma<f16_t> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    __device__ static inline f32x16 mma(v8 a, v8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
    __device__ static inline float add2(uint32_t p, float sum) {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, p), __builtin_bit_cast(v2, 0x3c003c00u), sum, false);
    }
};

typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;

__device__ inline uint32_t lds_address(const char* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) const char*)p));
}

// Exponent bits of an element: all ones for infinities and NaN.
template <typename T> constexpr uint32_t kExponentBits = 0x7f80u;
template <> constexpr uint32_t kExponentBits<f16_t> = 0x7c00u;

template <typename T>
__device__ inline uint32_t any_special(u32x4 x) {
    uint32_t found = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        found |= ((x[e] & kExponentBits<T>) == kExponentBits<T>) | (((x[e] >> 16) & kExponentBits<T>) == kExponentBits<T>);
    return found;
}

template <int N>
__device__ inline void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// The pages of an item's keys: entries of its request's row of the block table, read
// through the scalar cache. Keys past the item's have its last page; a page outside the
// pool is read as the pool's last (the careful way masks its keys).
struct ChunkPages {
    uniform_i32* table;
    int32_t first, last, log2;
    uint32_t top;

    __device__ inline ChunkPages(const ChunkArgs& a, int32_t request, int32_t key_begin, int32_t key_end)
        : table(reinterpret_cast<uniform_i32*>(reinterpret_cast<uint64_t>(a.tables + request * a.table_stride))),
          first(key_begin >> a.page_log2), last((key_end - 1) >> a.page_log2), log2(a.page_log2),
          top(static_cast<uint32_t>(a.n_pages - 1)) {}
    __device__ inline uint32_t of(int32_t key) const {
        return min(static_cast<uint32_t>(table[min(key >> log2, last)]), top);
    }
    __device__ inline bool outside(int32_t key) const {
        return static_cast<uint32_t>(table[min(key >> log2, last)]) > top;
    }
    // Whether any page lies outside the pool; the threads of a block look at some each.
    __device__ inline bool any_outside(int tid) const {
        const int32_t* const row = reinterpret_cast<const int32_t*>(reinterpret_cast<uint64_t>(table));
        bool found = false;
        for (int32_t e = first + tid; e <= last; e += kChunkThreads) found |= static_cast<uint32_t>(row[e]) > top;
        return __syncthreads_or(found);
    }
};

template <int D>
struct ChunkCfg {
    static constexpr int c8 = D / 8;                    // 16-byte pieces of a row
    static constexpr int kKeys = 64;                    // of a stage
    static constexpr int kTensor = kKeys * D * 2;       // K or V of a stage
    static constexpr int kStage = 2 * kTensor;
    static constexpr int kRing = 4;                     // stages
    static constexpr int kLds = kRing * kStage;
    static constexpr int kLoadRows = 1024 / (D * 2);    // rows of a load
    static constexpr int kWaveKeys = kKeys / kChunkWaves;      // rows that a wave loads: all in one page
    static constexpr int kLoads = kWaveKeys / kLoadRows;       // of K or V, a wave
    // Row r's 16-byte piece p lies at piece p ^ swz(r): 8 rows at one piece, as K is read, then lie on different banks,
    // and so do 4 rows x 2 pieces, 16 lanes of a transposing read of V. Not so 32 lanes, 4 rows x 4 pieces: two rows share
    // their banks (a third of LDS's busy cycles are conflicts, 126 of 378 M for 4096 rows over 32768 tokens).
    __device__ static constexpr int kswz(int r) { return r & (c8 - 1); }
    __device__ static constexpr int vswz(int r) { return (2 * r) & (c8 - 1); }
};

// A wave's 32 query rows. Lane (lq, h) = (lane % 32, lane / 32) holds row lq's scores of keys
// 8 (i / 4) + 4 h + i % 4, i < 16, of a sub-tile, and of O dims 32 dt + 8 (i / 4) + 4 h + i % 4.
template <typename T, int D>
struct ChunkWave {
    using M = wide_mma<T>;
    using R = mma_t<T>;
    using L = Lift<T, true>;
    using C = ChunkCfg<D>;
    using v8 = typename M::v8;
    static constexpr int KS = D / 16;  // k steps of QK^T
    static constexpr int DT = D / 32;  // d tiles of PV

    v8 qf[KS];
    f32x16 o[DT];
    float m_run, m_neg, m_thr, l_run;
    // of the sub-tiles in the pipeline
    v8 kf[KS], vf[2][DT];
    f32x16 s[2];
    uint32_t p[8];
    // K row lq, piece h (k step ks: 2 ks more, which the swizzle leaves a change of two bits); V row
    // 4 h + (lane % 16) / 4, dims 16 ((lane / 16) % 2) + 4 (lane % 4) (d tile dt: four pieces more, likewise)
    uint32_t koff, voff;

    __device__ inline void init(int lane) {
        const int lq = lane & 31, h = lane >> 5;
        koff = (lq * C::c8 + (h ^ C::kswz(lq))) * 16;
        const int r = 4 * h + ((lane & 15) >> 2), d0 = 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
        voff = (r * C::c8 + ((d0 >> 3) ^ C::vswz(r))) * 16 + (d0 & 4) * 2;
        m_run = -INFINITY;
        m_neg = L::kLog2;
        m_thr = -INFINITY;
        l_run = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[dt][i] = 0.f;
    }

    // LDS addresses of a sub-tile's first fragments. Those of the others in a row differ by bits of the offset in the row,
    // changed by XOR: rows, and with them the dynamic LDS behind the static part, start at multiples of their size.
    __device__ inline uint32_t k_at(const char* Ks) const { return lds_address(Ks) + koff; }
    __device__ inline uint32_t v_at(const char* Vs) const { return lds_address(Vs) + voff; }

    __device__ static inline v8 read_k(uint32_t k, int ks) {
        return __builtin_bit_cast(v8, *(lds_u32x4*)(uintptr_t)(k ^ (ks << 5)));
    }
    // keys 16 s + 4 h .. + 4 and 16 s + 8 + 4 h .. + 4 of dim 32 dt + lq
    __device__ static inline v8 read_v(uint32_t v, int dt, int s) {
        lds_s16x4* const at = (lds_s16x4*)(uintptr_t)(v ^ (dt << 6));
        const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at + 16 * s * D * 2 / 8);
        const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(at + (16 * s + 8) * D * 2 / 8);
        return __builtin_bit_cast(v8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
    }

    __device__ inline f32x16 scores(const char* Ks) const {
        f32x16 sc;
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = 0.f;
        const uint32_t k = k_at(Ks);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) sc = M::mma(read_k(k, ks), qf[ks], sc);
        return sc;
    }

    // the largest of this lane's scores, scaled (scale_log2 > 0)
    __device__ static inline float largest(const f32x16& sc, float scale_log2) {
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[i]);
        return mx * scale_log2;
    }

    __device__ inline void rescale_if(float mx) {
        if (__any(mx > m_thr)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = mx > m_thr ? mx : m_run;
            // 1 if unmoved, 0 from -inf; a row with no visible key keeps m = -inf
            const float alpha = __builtin_amdgcn_exp2f(m_run - (m_new == -INFINITY ? 0.f : m_new));
            m_run = m_new;
            m_neg = L::kLog2 - (m_new == -INFINITY ? 0.f : m_new);
            m_thr = m_new + L::kHead;
            l_run *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
        }
    }

    // word w of the packed weights: scores 2 w and 2 w + 1, rounded
    __device__ inline uint32_t weight_pair(const f32x16& sc, int w, float scale_log2) const {
        return R::round2(__builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * w], scale_log2, m_neg)),
                         __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * w + 1], scale_log2, m_neg)));
    }
    __device__ static inline v8 half(const uint32_t (&pw)[8], int s) {
        return __builtin_bit_cast(v8, u32x4{pw[4 * s], pw[4 * s + 1], pw[4 * s + 2], pw[4 * s + 3]});
    }

    // ---- Sub-tiles whose keys every row sees, software-pipelined: while the vector units make one's weights, the
    // matrix units make the next one's scores, and its maximum goes beside this one's weighted values.
    // Fragments are read half a sub-tile before their first use; the scheduling barriers keep the order.

    // weights of the scores in s[J], this sub-tile's V into vf, and with NEXT the next one's scores from kf
    template <int J, bool NEXT>
    __device__ inline void weights_scores(const char* Vs, float scale_log2) {
        constexpr int W = 8 / KS;
        // of the two waves of a SIMD the one that has only matrix work goes first
        __builtin_amdgcn_s_setprio(0);
        const uint32_t v = v_at(Vs);
        f32x16 zero;
#pragma unroll
        for (int i = 0; i < 16; ++i) zero[i] = 0.f;
#pragma unroll
        for (int g = 0; g < KS; ++g) {
            if (NEXT) s[1 - J] = M::mma(kf[g], qf[g], g == 0 ? zero : s[1 - J]);
            vf[g / DT][g % DT] = read_v(v, g % DT, g / DT);
#pragma unroll
            for (int w = W * g; w < W * (g + 1); ++w) {
                p[w] = weight_pair(s[J], w, scale_log2);
                asm volatile("" : "+v"(p[w]));  // pinned here, not at its first use
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }

    // weighted values from vf, the sum of the weights, with NEXT the maximum of the next one's scores in s[1 - J],
    // and with KREAD the K of the one after it into kf
    template <int J, bool NEXT, bool KREAD>
    __device__ inline float values_max(const char* Ks, float scale_log2) {
        constexpr int G = 2 * DT;
        __builtin_amdgcn_s_setprio(1);
        const uint32_t k = KREAD ? k_at(Ks) : 0;
        float mx = -INFINITY;
#pragma unroll
        for (int g = 0; g < G; ++g) {
            o[g % DT] = M::mma(vf[g / DT][g % DT], half(p, g / DT), o[g % DT]);
            if (KREAD) kf[g] = read_k(k, g);
#pragma unroll
            for (int w = 8 / G * g; w < 8 / G * (g + 1); ++w) l_run = M::add2(p[w], l_run);
            if (NEXT && g >= G / 2) {
#pragma unroll
                for (int i = 32 / G * (g - G / 2); i < 32 / G * (g + 1 - G / 2); ++i) mx = fmaxf(mx, s[1 - J][i]);
                asm volatile("" : "+v"(mx));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        return mx * scale_log2;
    }

    // Fills the pipeline: the first sub-tile's scores, the second's K.
    __device__ inline void begin(const char* Ks, float scale_log2) {
        s[0] = scores(Ks);
        const uint32_t k = k_at(Ks + kSub * D * 2);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) kf[ks] = read_k(k, ks);
        rescale_if(largest(s[0], scale_log2));
    }

    // A stage's two sub-tiles; `landed` waits for the next one, which stands at next.
    template <bool NEXT, typename F>
    __device__ inline void stage(const char* Ks, const char* Vs, const char* next, float scale_log2, F landed) {
        weights_scores<0, true>(Vs, scale_log2);
        if (NEXT) landed();
        rescale_if(values_max<0, true, NEXT>(next, scale_log2));
        weights_scores<1, NEXT>(Vs + kSub * D * 2, scale_log2);
        const float mx = values_max<1, NEXT, NEXT>(next + kSub * D * 2, scale_log2);
        if (NEXT) rescale_if(mx);
    }

    // A sub-tile by itself. With MASK, rows see the keys up to `last`, and none those of `bad` halves (of 16 keys);
    // with `spill`, some value that only some rows see is an infinity or NaN: it is added key by key, to
    // the rows that see it.
    template <bool MASK>
    __device__ inline void step(const char* Ks, const char* Vs, float scale_log2, int32_t key0, int32_t last,
                                uint32_t bad, bool spill, int lane) {
        const int h = lane >> 5;
        f32x16 sc = scores(Ks);
        uint32_t seen = 0;
        if (MASK) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool ok = key0 + 8 * (i / 4) + 4 * h + i % 4 <= last && !((bad >> (i / 8)) & 1);
                sc[i] = ok ? sc[i] : -INFINITY;
                seen |= static_cast<uint32_t>(ok) << i;
            }
        }
        rescale_if(largest(sc, scale_log2));
        uint32_t pw[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            pw[w] = weight_pair(sc, w, scale_log2);
            l_run = M::add2(pw[w], l_run);
        }
        if (!MASK || !spill) {
            const uint32_t v = v_at(Vs);
#pragma unroll
            for (int g = 0; g < 2 * DT; ++g) o[g % DT] = M::mma(read_v(v, g % DT, g / DT), half(pw, g / DT), o[g % DT]);
            return;
        }
#pragma unroll 1
        for (int key = 0; key < kSub; ++key) {
            const int i = 4 * (key >> 3) + (key & 3), from = (lane & 31) + 32 * ((key >> 2) & 1);
            uint32_t word = 0;
#pragma unroll
            for (int w = 0; w < 8; ++w) word = w == i >> 1 ? pw[w] : word;
            const float weight = elem<T>::to_float(static_cast<uint16_t>(__shfl(word, from) >> (16 * (i & 1))));
            const bool ok = (__shfl(seen, from) >> i) & 1;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const int d0 = 32 * dt + 8 * g + 4 * h;
                    const uint16_t* const x = reinterpret_cast<const uint16_t*>(
                        Vs + (key * C::c8 + ((d0 >> 3) ^ C::vswz(key))) * 16 + (d0 & 4) * 2);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (ok) o[dt][4 * g + j] += weight * elem<T>::to_float(x[j]);
                }
        }
    }
};

// The item at `at` of the work list, for one KV head.
template <typename T, int D>
__device__ inline void chunk_item(const ChunkArgs& a, uniform_i32* at, int kv_head, char* smem) {
    using W = ChunkWave<T, D>;
    using C = ChunkCfg<D>;
    using E = elem<T>;
    using v8 = typename W::v8;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // no value of an item is kept over the loop of items
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lq = lane & 31, h = lane >> 5;
    const int32_t request = at[0], key_begin = at[1], key_end = at[2], part = at[3], length = at[4];
    const int32_t rows = at[5], row0 = at[6], first = at[7];
    if (rows < 0) {  // a failed request's rows become zero
        const int64_t per = static_cast<int64_t>(a.group) * (D / 4);
        for (int64_t e = tid; e < -rows * per; e += kChunkThreads) {
            const int64_t row = row0 + e / per, piece = e % per;
            const int64_t head = static_cast<int64_t>(kv_head) * a.group + piece / (D / 4);
            *reinterpret_cast<uint2*>(a.out + (head * a.os[0] + row * a.os[1] + piece % (D / 4) * 4) * 2) = uint2{0u, 0u};
        }
        return;
    }
    const int32_t live = min(rows * a.group - first, kTileRows);  // the tile's rows
    const int32_t mine = live - kWaveRows * wave;                 // this wave's and those of the waves behind it

    // ---- this wave's loads: rows kWaveKeys wave .. of a stage, all of one page ----
    const ChunkPages pages(a, request, key_begin, key_end);
    const int32_t n_st = (key_end - key_begin + C::kKeys - 1) / C::kKeys;
    const int lr = lane / C::c8, lc = lane % C::c8;
    const uint32_t page_mask = (1u << a.page_log2) - 1;
    const char* const kbase = a.k + kv_head * a.k_head;
    const char* const vbase = a.v + kv_head * a.v_head;
    uint32_t koff[C::kLoads], voff[C::kLoads];
#pragma unroll
    for (int l = 0; l < C::kLoads; ++l) {
        const int r = l * C::kLoadRows + lr;
        koff[l] = r * a.k_row + 16 * (lc ^ C::kswz(C::kWaveKeys * wave + r));
        voff[l] = r * a.v_row + 16 * (lc ^ C::vswz(C::kWaveKeys * wave + r));
    }
    int32_t issued = 0;  // stages
    auto issue = [&]() __attribute__((always_inline)) {
        const int32_t key = key_begin + C::kKeys * issued + C::kWaveKeys * wave;
        const uint32_t page = pages.of(key), row = key & page_mask;
        const char* const kp = kbase + (static_cast<uint64_t>(page) * a.k_page + row * a.k_row);
        const char* const vp = vbase + (static_cast<uint64_t>(page) * a.v_page + row * a.v_row);
        char* const to = smem + (issued % C::kRing) * C::kStage + C::kWaveKeys * wave * D * 2;
#pragma unroll
        for (int l = 0; l < C::kLoads; ++l) lds_dma16(kp, koff[l], to + l * 1024);
#pragma unroll
        for (int l = 0; l < C::kLoads; ++l) lds_dma16(vp, voff[l], to + C::kTensor + l * 1024);
        ++issued;
    };
    // stage i has landed, and every wave has come here; at most two stages behind it are in flight
    auto landed = [&](int32_t i) __attribute__((always_inline)) {
        if (issued - i > 2)
            wait_loads<4 * C::kLoads>();
        else if (issued - i > 1)
            wait_loads<2 * C::kLoads>();
        else
            wait_loads<0>();
        // what this wave has read of the stages before i has been used: nothing of it is in flight
        asm volatile("s_barrier" ::: "memory");
    };

    W w;
    w.init(lane);
    int32_t last;  // the last key that this lane's row sees
    {
        u32x4 raw[W::KS];
        const int32_t qr = first + min(kWaveRows * wave + lq, live - 1);
        const int64_t token = qr / a.group, head = static_cast<int64_t>(kv_head) * a.group + qr % a.group;
        last = length + static_cast<int32_t>(token);
#pragma unroll
        for (int ks = 0; ks < W::KS; ++ks)
            raw[ks] = *reinterpret_cast<const u32x4*>(a.q + (head * a.qs[0] + (row0 + token) * a.qs[1] + 16 * ks + 8 * h) * 2);
#pragma unroll 1
        while (issued < min(n_st, 3)) issue();
#pragma unroll
        for (int ks = 0; ks < W::KS; ++ks) {
            asm volatile("" : "+v"(raw[ks]));
            w.qf[ks] = __builtin_bit_cast(v8, raw[ks]);
        }
    }
    // the keys that all rows of the tile see, that all rows of this wave see, and the last that one of this wave's sees
    const int32_t common = length + first / a.group;
    const int32_t wave_common = length + (first + kWaveRows * wave) / a.group;
    const int32_t wave_last = length + (first + min(kWaveRows * wave + kWaveRows, live) - 1) / a.group;
    const int32_t tile_last = length + (first + live - 1) / a.group;

    const bool strange = pages.any_outside(tid);
    const int32_t plain = strange ? 0 : min(n_st, max(0, (common + 1 - key_begin) / C::kKeys));
    int32_t i = 0;
    if (plain > 0) {
        landed(0);
        // the next stage; the one after it goes where the one before this was
        auto turn = [&]() __attribute__((always_inline)) {
            landed(i + 1);
            if (issued < n_st) issue();
        };
        if (mine > 0) {
            w.begin(smem, a.scale_log2);
#pragma unroll 1
            for (; i + 1 < plain; ++i) {
                const char* const Ks = smem + (i % C::kRing) * C::kStage;
                w.template stage<true>(Ks, Ks + C::kTensor, smem + ((i + 1) % C::kRing) * C::kStage, a.scale_log2, turn);
            }
            const char* const Ks = smem + (i % C::kRing) * C::kStage;
            w.template stage<false>(Ks, Ks + C::kTensor, Ks, a.scale_log2, [] {});
        } else {
#pragma unroll 1
            for (; i + 1 < plain; ++i) turn();
        }
        ++i;
    }
#pragma unroll 1
    for (; i < n_st; ++i) {
        landed(i);
        while (issued < min(n_st, i + 3)) issue();
        const int32_t key0 = key_begin + C::kKeys * i;
        uint32_t bad = 0;  // halves (16 keys) outside the pool
        if (strange) {
#pragma unroll
            for (int half_of = 0; half_of < C::kKeys / 16; ++half_of)
                if (pages.outside(key0 + 16 * half_of)) bad |= 1u << half_of;
        }
        char* const Ks = smem + (i % C::kRing) * C::kStage;
        char* const Vs = Ks + C::kTensor;
        // V rows that no row of the tile sees become zero (their weights are, and 0 * V must be)
        uint32_t special = 0;
        for (int e = tid; e < C::kKeys * C::c8; e += kChunkThreads) {
            const int r = e / C::c8;
            u32x4* const p = reinterpret_cast<u32x4*>(Vs + e * 16);
            if (((bad >> (r >> 4)) & 1) || key0 + r > tile_last)
                *p = u32x4{0u, 0u, 0u, 0u};
            else if (key0 + r > common)
                special |= any_special<T>(*p);
        }
        const bool spill = __syncthreads_or(special != 0);
        if (mine <= 0) continue;
#pragma unroll 1
        for (int j = 0; j < C::kKeys / kSub; ++j) {
            const int32_t from = key0 + kSub * j;
            if (from > wave_last) break;
            const char* const ks = Ks + kSub * j * D * 2;
            const char* const vs = Vs + kSub * j * D * 2;
            if (bad == 0 && from + kSub - 1 <= wave_common)
                w.template step<false>(ks, vs, a.scale_log2, from, last, 0u, false, lane);
            else
                w.template step<true>(ks, vs, a.scale_log2, from, last, (bad >> (2 * j)) & 3u, spill, lane);
        }
    }

    // ---- the rows, or their partials ----
    const float sum = w.l_run + __shfl_xor(w.l_run, 32);
    const int32_t in_tile = kWaveRows * wave + lq;
    if (in_tile >= live) return;
    // a sum of zero: a row that sees no key of the item, or one all of whose scores are -inf
    bool seen = true;
    if (__any(sum == 0.f)) {
        int32_t key = key_begin;  // the first whose page lies in the pool
        while (strange && key < key_end && pages.outside(key)) key = ((key >> a.page_log2) + 1) << a.page_log2;
        seen = key <= min(last, key_end - 1);
    }
    if (part < 0) {
        const int32_t qr = first + in_tile;
        const int64_t row = row0 + qr / a.group, head = static_cast<int64_t>(kv_head) * a.group + qr % a.group;
        char* const dst = a.out + (head * a.os[0] + row * a.os[1]) * 2;
        const bool none = !seen;
        const float inv = 1.f / sum;  // scores of -inf alone: 0 / 0, as the softmax has it
#pragma unroll
        for (int dt = 0; dt < W::DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                uint32_t e[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) e[j] = none ? 0u : E::from_float(w.o[dt][4 * g + j] * inv);
                *reinterpret_cast<uint2*>(dst + (32 * dt + 8 * g + 4 * h) * 2) =
                    uint2{e[0] | (e[1] << 16), e[2] | (e[3] << 16)};
            }
    } else {
        const int64_t at_row = (static_cast<int64_t>(part) * a.kv_heads + kv_head) * kTileRows + in_tile;
#pragma unroll
        for (int dt = 0; dt < W::DT; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g)
                *reinterpret_cast<f32x4*>(a.part_o + at_row * D + 32 * dt + 8 * g + 4 * h) =
                    f32x4{w.o[dt][4 * g], w.o[dt][4 * g + 1], w.o[dt][4 * g + 2], w.o[dt][4 * g + 3]};
        if (h == 0) {
            a.part_ml[2 * at_row] = w.m_run;
            a.part_ml[2 * at_row + 1] = sum == 0.f && seen ? -1.f : sum;  // its weight is zero: the maximum is -inf
        }
    }
}

// A worker's items, one after another.
template <typename T, int D>
__global__ void __launch_bounds__(kChunkThreads) chunk_attention_kernel(ChunkArgs a) {
    extern __shared__ __align__(kRowAlign) char smem[];
    static_assert(__alignof__(smem) >= 2 * D && ChunkCfg<D>::kTensor % (2 * D) == 0, "fragments' addresses: ChunkWave");
    const int kv_head = blockIdx.x % a.kv_heads, worker = blockIdx.x / a.kv_heads;
    uniform_i32* first_of = reinterpret_cast<uniform_i32*>(reinterpret_cast<uint64_t>(a.schedule + kStepHeader + worker));
    const int32_t end = first_of[1];
    const int32_t* work = a.schedule + kStepHeader + step_worker_ints(a.workers);
#pragma unroll 1
    for (int32_t i = first_of[0]; i < end; ++i) {
        uniform_i32* at =
            reinterpret_cast<uniform_i32*>(reinterpret_cast<uint64_t>(work + static_cast<int64_t>(i) * kStepItem));
        chunk_item<T, D>(a, at, kv_head, smem);
        __syncthreads();  // the item's LDS has been read
    }
    if (a.zero_rest) {
        const int32_t total = a.row_starts[a.requests];
        const int64_t per = static_cast<int64_t>(a.group) * (D / 4);  // 8-byte pieces of a row
        const int64_t pieces = (a.rows - total) * per;
        for (int64_t e = static_cast<int64_t>(worker) * kChunkThreads + threadIdx.x; e < pieces;
             e += static_cast<int64_t>(a.workers) * kChunkThreads) {
            const int64_t row = total + e / per, piece = e % per;
            const int64_t head = static_cast<int64_t>(kv_head) * a.group + piece / (D / 4);
            *reinterpret_cast<uint2*>(a.out + (head * a.os[0] + row * a.os[1] + piece % (D / 4) * 4) * 2) = uint2{0u, 0u};
        }
    }
}

// The pieces of a cut tile's rows: D / 4 lanes a row, of which each first finds the weight of some pieces.
constexpr int kMergeThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) chunk_merge_kernel(ChunkArgs a) {
    using E = elem<T>;
    constexpr int kLanes = D / 4, kRows = kMergeThreads / kLanes;
    if (static_cast<int32_t>(blockIdx.y) >= a.schedule[1]) return;
    const int32_t* cut = a.schedule + kStepHeader + step_worker_ints(a.workers) +
                         static_cast<int64_t>(a.items + blockIdx.y) * kStepItem;
    const int32_t worker = cut[0], pieces = cut[1], row0 = cut[2], first = cut[3], rows = cut[4];
    const int32_t kv_head = blockIdx.x % a.kv_heads;
    const int32_t in_tile = blockIdx.x / a.kv_heads * kRows + threadIdx.x / kLanes, qr = first + in_tile;
    if (qr >= rows * a.group) return;  // all lanes of the row
    const int lane = threadIdx.x % kLanes;
    auto at_row = [&](int32_t p) {
        return (static_cast<int64_t>(step_partial(worker, p)) * a.kv_heads + kv_head) * kTileRows + in_tile;
    };
    float top = -INFINITY;
    for (int32_t p = lane; p < pieces; p += kLanes) top = fmaxf(top, a.part_ml[2 * at_row(p)]);
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
    const float use = top == -INFINITY ? 0.f : top;
    float l = 0.f;
    int seen = 0;  // whether some piece has a key of the row's
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int32_t base = 0; base < pieces; base += kLanes) {
        const int32_t here = min(pieces - base, kLanes);
        float weight = 0.f;
        if (lane < here) {
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * at_row(base + lane));
            weight = __builtin_amdgcn_exp2f(ml.x - use);
            l += ml.y * weight;
            seen |= ml.y != 0.f;
        }
        for (int32_t p = 0; p < here; p += 4) {
            f32x4 x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (p + e < here) x[e] = *reinterpret_cast<const f32x4*>(a.part_o + at_row(base + p + e) * D + 4 * lane);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float f = __shfl(weight, p + e, kLanes);
                if (p + e < here) o += x[e] * f;
            }
        }
    }
#pragma unroll
    for (int d = 1; d < kLanes; d *= 2) {
        l += __shfl_xor(l, d);
        seen |= __shfl_xor(seen, d);
    }
    const int64_t row = row0 + qr / a.group, head = static_cast<int64_t>(kv_head) * a.group + qr % a.group;
    const bool none = !seen;
    const float inv = 1.f / l;
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = none ? 0u : E::from_float(o[i] * inv);
    *reinterpret_cast<uint2*>(a.out + (head * a.os[0] + row * a.os[1] + 4 * lane) * 2) =
        uint2{e[0] | (e[1] << 16), e[2] | (e[3] << 16)};
}

template <typename T, int D>
int launch_chunk(const ChunkArgs& a, const ChunkShape& s, hipStream_t stream) {
    static LdsGrant grant;
    // with the static part heads of 64 need more than 64 KB too
    if (!grant.ok(chunk_attention_kernel<T, D>, ChunkCfg<D>::kLds + kVoteLds)) return KVR_E_LAUNCH_FAILED;
    chunk_attention_kernel<T, D><<<static_cast<unsigned>(a.kv_heads * s.workers), kChunkThreads, ChunkCfg<D>::kLds, stream>>>(a);
    if (s.workers > 1) {
        constexpr int kRows = kMergeThreads / (D / 4);
        chunk_merge_kernel<T, D><<<dim3(a.kv_heads * (kTileRows / kRows), static_cast<unsigned>(s.splits)), kMergeThreads, 0, stream>>>(a);
    }
    return launch_status();
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

}  // namespace
}  // namespace kvr

using namespace kvr;

extern "C" int64_t kvr_chunk_schedule_ints(const kvr_step_desc* d, int32_t q_heads, int32_t kv_heads) {
    const int st = check_chunk(d, q_heads, kv_heads);
    return st == KVR_OK ? chunk_shape(d, q_heads, kv_heads).ints : st;
}

extern "C" int kvr_chunk_schedule(const kvr_step_desc* d, int32_t q_heads, int32_t kv_heads, int32_t* schedule,
                                  void* stream) {
    const int st = check_chunk(d, q_heads, kv_heads);
    if (st != KVR_OK) return st;
    if (!schedule || !d->lengths) return KVR_E_NULL_POINTER;
    if (!aligned(schedule, 32)) return KVR_E_BAD_STRIDE;
    const ChunkShape s = chunk_shape(d, q_heads, kv_heads);
    ChunkPlanArgs a;
    a.lengths = d->lengths;
    a.status = d->status;
    a.row_starts = d->row_starts;
    a.schedule = schedule;
    a.requests = d->requests;
    a.group = q_heads / kv_heads;
    a.workers = static_cast<int32_t>(s.workers);
    a.items = static_cast<int32_t>(s.items);
    a.splits = static_cast<int32_t>(s.splits);
    chunk_schedule_kernel<<<1, kPlanThreads, 0, as_stream(stream)>>>(a);
    return launch_status();
}

extern "C" int64_t kvr_chunk_workspace_bytes(const kvr_step_desc* d, int32_t q_heads, int32_t kv_heads, int32_t head_dim) {
    const int st = check_chunk(d, q_heads, kv_heads);
    if (st != KVR_OK) return st;
    if (head_dim != 64 && head_dim != 128) return KVR_E_UNSUPPORTED_SHAPE;
    return chunk_shape(d, q_heads, kv_heads).partials * kv_heads * kTileRows * (head_dim + 2) * 4;
}

extern "C" int kvr_chunk_attention(const void* q, const void* k, const void* v, void* out, const kvr_step_desc* d,
                                   const int32_t* schedule, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                                   float scale, const int64_t strides[12], int32_t zero_rest, void* workspace,
                                   int64_t workspace_bytes, int32_t dtype, void* stream) {
    if (dtype != KVR_DTYPE_BF16 && dtype != KVR_DTYPE_F16) return KVR_E_UNSUPPORTED_DTYPE;
    const int64_t need = kvr_chunk_workspace_bytes(d, q_heads, kv_heads, head_dim);
    if (need < 0) return static_cast<int>(need);
    const float scale_log2 = scale * 1.4426950408889634f;
    if (!(scale > 0.f) || !isfinite(scale_log2)) return KVR_E_INVALID_ARGUMENT;
    if (!q || !k || !v || !out || !strides || !schedule) return KVR_E_NULL_POINTER;
    for (int t = 0; t < 4; ++t) {
        const int64_t* s = strides + 3 * t;
        const int64_t unit = t == 3 ? 4 : 8;
        // a load's row offsets fit 32 bits
        if (s[0] <= 0 || s[1] <= 0 || s[2] != 1 || s[0] % unit || s[1] % unit || s[1] > (int64_t(1) << 26))
            return KVR_E_BAD_STRIDE;
        // ... and a page of K or V
        if ((t == 1 || t == 2) && s[1] * 2 * d->page_size > UINT32_MAX) return KVR_E_BAD_STRIDE;
    }
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 8) || !aligned(schedule, 32))
        return KVR_E_BAD_STRIDE;
    if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need)) return KVR_E_WORKSPACE_TOO_SMALL;
    const ChunkShape s = chunk_shape(d, q_heads, kv_heads);
    ChunkArgs a;
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k);
    a.v = static_cast<const char*>(v);
    a.out = static_cast<char*>(out);
    for (int i = 0; i < 2; ++i) {
        a.qs[i] = strides[i];
        a.os[i] = strides[9 + i];
    }
    a.k_head = strides[3] * 2;
    a.v_head = strides[6] * 2;
    a.k_row = static_cast<uint32_t>(strides[4] * 2);
    a.v_row = static_cast<uint32_t>(strides[7] * 2);
    a.k_page = a.k_row * static_cast<uint32_t>(d->page_size);
    a.v_page = a.v_row * static_cast<uint32_t>(d->page_size);
    a.schedule = schedule;
    a.tables = d->tables;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + s.partials * kv_heads * kTileRows * head_dim;
    a.table_stride = d->table_stride;
    a.row_starts = d->row_starts;
    a.items = static_cast<int32_t>(s.items);
    a.workers = static_cast<int32_t>(s.workers);
    a.requests = d->requests;
    a.rows = d->rows;
    a.zero_rest = zero_rest != 0;
    a.page_log2 = __builtin_ctz(static_cast<unsigned>(d->page_size));
    a.n_pages = static_cast<int32_t>(d->n_slots / d->page_size);
    a.kv_heads = kv_heads;
    a.group = q_heads / kv_heads;
    a.scale_log2 = scale_log2;
    hipStream_t hs = as_stream(stream);
    if (dtype == KVR_DTYPE_BF16)
        return head_dim == 128 ? launch_chunk<bf16_t, 128>(a, s, hs) : launch_chunk<bf16_t, 64>(a, s, hs);
    return head_dim == 128 ? launch_chunk<f16_t, 128>(a, s, hs) : launch_chunk<f16_t, 64>(a, s, hs);
}
