// Attention of a step's rows (kvr_step_plan.hip) over each request's paged cache:
//   out[h, row] = softmax_j(scale q[h, row] . k[h / G, slot(j)]) @ v[h / G, slot(j)]
// j over the request's L committed tokens and the nodes (tokens L + u) whose bit
// the row's mask has: new tokens, chains and trees of drafted tokens alike.
//
// What bounds it: a request's rows (at most 64) times G query heads read the same
// K and V, so up to some 200 of them per KV head the time is that of reading K
// and V once, above that the MFMA's. Grid: (KV head and group of query rows, worker);
// the plan gives every worker, one a CU, the same share of all requests' keys, as
// items (runs of keys of one request) that a block works through; a request that is cut
// between workers leaves partial (m, l, O), which tree_merge_kernel joins.
//
// S^T = K Q^T and O^T += V^T P^T on the 16x16x32 MFMA, fp32 statistics, one pass
// with a running maximum that moves only when a score exceeds it by 2^8 (fp16: 2^3), so
// that the fp32 sums hold p; P enters PV as a hi + lo pair of 16-bit values, off by 2^-16
// of each p in bf16, and in fp16, where a power of two lifts it (Lift), by 2^-22 of it or
// 2^-37 of the row's largest. Only keys past the committed tokens, or of a
// page outside the pool, look at masks. K and V go straight from the cache to LDS
// (global_load_lds, nontemporal: 48 requests of up to 16k tokens 272 us without, 243
// with); a page of at least 16 slots holds whole 1 KB loads, so only the wave-uniform
// base of a load depends on the block table.
//
// Measured (32 query and 8 KV heads of 128, bf16, kernels alone): one token of each
// of 48 requests over 64 to 16k tokens 243 to 250 us = 6.6 TB/s of K and V, HBM reads 1.00
// of theirs; 7 to 26 drafted rows of 12 requests over 1k to 16k 95 to 111 us = 4.2 TB/s;
// 64 rows of one request over 128k 190 to 240 us by the card's clock, which falls under
// such work, = 0.95 PFLOP/s of MFMA work, a third of it the lo halves.
#include "kvr_attention_tiles.h"
#include "kvr_step.h"

#include <math.h>

#include <type_traits>

namespace kvr {
namespace {

typedef const __attribute__((address_space(4))) int32_t uniform_i32;  // read through the scalar cache

// ---------------------------------------------------------------------------
// Up to 32 query rows: four waves, each with all rows and every fourth 32-key
// sub-tile of an item, from a ring of its own in LDS: no wave waits for another
// before the four (m, l, O) are joined.
// ---------------------------------------------------------------------------
constexpr int kTreeWaves = 4;
constexpr int kTreeThreads = 64 * kTreeWaves;
constexpr int kSub = 32;             // keys of a sub-tile

// Exponent bits of an element: all ones for infinities and NaN.
template <typename T> constexpr uint32_t kExponent = 0x7f80u;
template <> constexpr uint32_t kExponent<f16_t> = 0x7c00u;

struct TreeArgs {
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
    const uint64_t* masks;
    float* part_o;   // [partial][kv head][row_groups * group rows][D], unnormalised
    float* part_ml;  // ... [2]: running maximum (log2 units) and sum
    int64_t table_stride;
    const int32_t* row_starts;
    int32_t items;   // room for items in the schedule
    int32_t workers;
    int32_t requests;
    int32_t rows;        // room for packed rows
    int32_t zero_rest;   // 1: rows of no request become zero
    int32_t table_width;
    int32_t page_log2;
    int32_t n_pages;
    int32_t kv_heads;
    int32_t group;       // query heads of a KV head
    int32_t row_groups;
    float scale_log2;    // scale * log2(e)
};

template <int N>
__device__ inline void wait_vm() {
    static_assert(N >= 0 && N < 64, "vmcnt is six bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// Whether any of four packed pairs is an infinity or NaN.
template <typename T>
__device__ inline uint32_t special_pairs(u32x4 x) {
    uint32_t found = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        found |= ((x[e] & kExponent<T>) == kExponent<T>) | (((x[e] >> 16) & kExponent<T>) == kExponent<T>);
    return found;
}

template <int D>
struct TreeCfg {
    static constexpr int c8 = D / 8;                 // 16-byte pieces of a row
    static constexpr int kTensor = kSub * D * 2;     // K or V of a sub-tile
    static constexpr int kStage = 2 * kTensor;
    static constexpr int kStages = D == 128 ? 2 : 4; // ring of a wave: 32 KB
    static constexpr int kRing = kStages * kStage;
    static constexpr int kRows = 64 / c8;            // rows of a load
    static constexpr int kLoads = kSub / kRows;      // loads of K or V
    static constexpr int kHalf = kLoads / 2;         // ... of 16 keys, which lie in one page
    // Row r's 16-byte piece p lies at piece p ^ swz(r): the 16-byte reads of K
    // (8 rows at one piece) and the transposing reads of V (4 rows x 2 pieces)
    // then spread over all banks.
    __device__ static constexpr int kswz(int r) { return r & (c8 - 1); }
    __device__ static constexpr int vswz(int r) { return (2 * r) & (c8 - 1); }
    static constexpr int kVariants = 16 / kRows < c8 / kRows ? 16 / kRows : c8 / kRows > 0 ? c8 / kRows : 1;
};


// A failed request's rows of one KV head's query heads become zero.
template <int D>
__device__ inline void zero_rows(const TreeArgs& a, int32_t kv_head, int32_t row0, int32_t rows, int threads) {
    for (int64_t e = threadIdx.x; e < static_cast<int64_t>(rows) * a.group * (D / 4); e += threads) {
        const int64_t qr = e / (D / 4);
        const int64_t row = row0 + qr / a.group, head = static_cast<int64_t>(kv_head) * a.group + qr % a.group;
        *reinterpret_cast<uint2*>(a.out + (head * a.os[0] + row * a.os[1] + e % (D / 4) * 4) * 2) = uint2{0u, 0u};
    }
}

// The pages of an item's keys: entries of its request's row of the block table,
// read through the scalar cache. Keys past the item's have its last page; a page
// outside the pool is read as the pool's last (the careful way masks its keys).
struct ItemPages {
    uniform_i32* table;
    int32_t first, last;  // entries of the item's keys
    int32_t log2;
    uint32_t top;         // pages of the pool - 1

    __device__ inline ItemPages(const TreeArgs& a, int32_t request, int32_t key_begin, int32_t key_end)
        : table(reinterpret_cast<uniform_i32*>(reinterpret_cast<uint64_t>(a.tables + request * a.table_stride))),
          first(key_begin >> a.page_log2), last((key_end - 1) >> a.page_log2), log2(a.page_log2),
          top(static_cast<uint32_t>(a.n_pages - 1)) {}
    __device__ inline uint32_t of(int32_t key) const {
        return min(static_cast<uint32_t>(table[min(key >> log2, last)]), top);
    }
    __device__ inline bool outside(int32_t key) const {
        return static_cast<uint32_t>(table[min(key >> log2, last)]) > top;
    }
    // Whether any page lies outside the pool: every wave looks at all of them.
    __device__ inline bool any_outside(int lane) const {
        const int32_t* const row = reinterpret_cast<const int32_t*>(reinterpret_cast<uint64_t>(table));
        bool found = false;
        for (int32_t e = first + lane; e <= last; e += 64) found |= static_cast<uint32_t>(row[e]) > top;
        return __any(found);
    }
};

// LDS of a block: the waves' rings, which the join of their (m, l, O) reuses.
template <int D, int TPW>
constexpr size_t tree_lds() {
    const size_t ring = static_cast<size_t>(kTreeWaves) * TreeCfg<D>::kRing;
    const size_t join = static_cast<size_t>(kTreeWaves) * TPW * (D / 16 * 1024 + 64 * 8);
    return (ring > join ? ring : join);
}

// O of one row tile plus P V of a 32-key sub-tile, key by key, so that a value
// reaches only the rows that see it (vis, bit 4 kt + i: key 16 kt + 4 lj + i).
template <typename T, int D>
__device__ inline void add_seen(f32x4 (&o)[D / 16], const char* Vs, const u32x4& hi, const u32x4& lo, uint32_t vis,
                                int lq, int lj) {
    using E = elem<T>;
    using C = PairCfg<D>;
#pragma unroll 1
    for (int key = 0; key < kPairSub; ++key) {
        const int from = ((key & 15) >> 2) * 16 + lq, e = (key >> 4) * 4 + (key & 3);
        uint32_t wh = 0, wl = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w)
            if (w == e >> 1) {
                wh = hi[w];
                wl = lo[w];
            }
        const uint32_t ph = __shfl(wh, from) >> (16 * (e & 1)), pl = __shfl(wl, from) >> (16 * (e & 1));
        const float weight = E::to_float(static_cast<uint16_t>(ph)) + E::to_float(static_cast<uint16_t>(pl));
        const bool ok = (__shfl(vis, from) >> e) & 1;
#pragma unroll
        for (int dt = 0; dt < D / 16; ++dt) {
            const int d0 = 16 * dt + 4 * lj;
            const uint16_t* x = reinterpret_cast<const uint16_t*>(
                Vs + (key * C::c8 + ((d0 >> 3) ^ C::vswz(key))) * 16 + (d0 & 4) * 2);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (ok) o[dt][i] += weight * E::to_float(x[i]);
        }
    }
}

// d tiles [dt0, dt0 + SL) of query row `qr` of a block: the result, or with several chunks its partial.
template <typename T, int D, int SL>
__device__ inline void put_row(const TreeArgs& a, const f32x4 (&res)[SL], float top, float sum, bool sees,
                               int32_t kv_head, int32_t group, int32_t group_rows, int32_t first, int32_t qr,
                               int32_t row0, int32_t part, int dt0, int lj) {
    using E = elem<T>;
    if (part < 0) {
        const int64_t row = row0 + (first + qr) / a.group;
        const int64_t head = static_cast<int64_t>(kv_head) * a.group + (first + qr) % a.group;
        char* const dst = a.out + (head * a.os[0] + row * a.os[1]) * 2;
        const bool none = !sees || sum == 0.f;
        const float inv = 1.f / sum;
#pragma unroll
        for (int j = 0; j < SL; ++j) {
            uint32_t e[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) e[i] = none ? 0u : E::from_float(res[j][i] * inv);
            *reinterpret_cast<uint2*>(dst + (16 * (dt0 + j) + 4 * lj) * 2) =
                uint2{e[0] | (e[1] << 16), e[2] | (e[3] << 16)};
        }
    } else {
        const int64_t at_row =
            ((static_cast<int64_t>(part) * a.kv_heads + kv_head) * a.row_groups + group) * group_rows + qr;
#pragma unroll
        for (int j = 0; j < SL; ++j)
            *reinterpret_cast<f32x4*>(a.part_o + at_row * D + 16 * (dt0 + j) + 4 * lj) = res[j];
        if (dt0 == 0 && lj == 0) {
            a.part_ml[2 * at_row] = top;
            a.part_ml[2 * at_row + 1] = sum;
        }
    }
}

// The item at `at` of the schedule, for one KV head and group of query rows.
template <typename T, int D, int TPW>
__device__ inline void tree_item(const TreeArgs& a, uniform_i32* at, int kv_head, int group, char* smem) {
    using M = mma_t<T>;
    using v8 = typename M::v8;
    using C = TreeCfg<D>;
    using L = Lift<T, true>;
    constexpr int DS = D / 32, DT = D / 16, NL = 2 * C::kLoads;
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // no value of an item is kept over the loop of items
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lq = lane & 15, lj = lane >> 4;
    const int32_t request = at[0], key_begin = at[1], key_end = at[2], part = at[3], length = at[4];
    const int32_t nodes = at[5], row0 = at[6], rows = at[7];
    const int32_t first = group * 16 * TPW;           // query rows [first, first + 16 TPW) of nodes * G
    const int32_t live = nodes * a.group - first;

    if (nodes == 0) {
        if (group == 0) zero_rows<D>(a, kv_head, row0, rows, kTreeThreads);
        return;
    }
    if (live <= 0) return;
    const int tiles = min(TPW, (live + 15) >> 4);     // tiles with rows

    // ---- this wave's loads: sub-tiles wave, wave + 4, ... of the run ----
    const int32_t n_sub = (key_end - key_begin + kSub - 1) / kSub;
    const ItemPages pages(a, request, key_begin, key_end);
    char* const ring = smem + wave * C::kRing;
    const char* const kbase = a.k + kv_head * a.k_head;
    const char* const vbase = a.v + kv_head * a.v_head;
    const int lr = lane / C::c8, lc = lane % C::c8;
    uint32_t koff[C::kVariants], voff[C::kVariants];  // of load i: variant i mod kVariants
#pragma unroll
    for (int i = 0; i < C::kVariants; ++i) {
        koff[i] = lr * a.k_row + 16 * (lc ^ C::kswz(i * C::kRows + lr));
        voff[i] = lr * a.v_row + 16 * (lc ^ C::vswz(i * C::kRows + lr));
    }
    const uint32_t page_mask = (1u << a.page_log2) - 1;
    // sub-tile s, whose halves lie in pages p0 and p1
    auto load = [&](int32_t s, char* dst, uint32_t p0, uint32_t p1) __attribute__((always_inline)) {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint32_t page = half ? p1 : p0;
            const uint32_t row = (key_begin + kSub * s + 16 * half) & page_mask;
            const char* kp = kbase + (static_cast<uint64_t>(page) * a.k_page + row * a.k_row);
            const char* vp = vbase + (static_cast<uint64_t>(page) * a.v_page + row * a.v_row);
#pragma unroll
            for (int i = 0; i < C::kHalf; ++i) {
                lds_dma16_once(kp, koff[i % C::kVariants], dst + (half * C::kHalf + i) * 1024);
                kp += C::kRows * a.k_row;
            }
#pragma unroll
            for (int i = 0; i < C::kHalf; ++i) {
                lds_dma16_once(vp, voff[i % C::kVariants], dst + C::kTensor + (half * C::kHalf + i) * 1024);
                vp += C::kRows * a.v_row;
            }
        }
    };

    // ---- queries, masks, and the first stages, in one round trip ----
    u32x4 raw[TPW][DS];
    uint64_t mask[TPW];
#pragma unroll
    for (int t = 0; t < TPW; ++t) {
        const int32_t r = min(16 * t + lq, live - 1) + first;
        const int64_t row = row0 + r / a.group;
        const int64_t head = static_cast<int64_t>(kv_head) * a.group + r % a.group;
        mask[t] = a.masks[row];
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
            raw[t][ds] = *reinterpret_cast<const u32x4*>(a.q + (head * a.qs[0] + row * a.qs[1] + 32 * ds + 8 * lj) * 2);
    }
#pragma unroll
    for (int i = 0; i < C::kStages; ++i) {
        const int32_t s = wave + kTreeWaves * i, key0 = key_begin + kSub * s;
        if (s < n_sub) load(s, ring + i * C::kStage, pages.of(key0), pages.of(key0 + 16));
    }
    v8 qf[TPW][DS];
    uint64_t seen = 0;  // nodes that some row of the block attends to
#pragma unroll
    for (int t = 0; t < TPW; ++t) {
        if (16 * t + lq >= live) mask[t] = 0;
        seen |= mask[t];
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) {
            asm volatile("" : "+v"(raw[t][ds]));
            qf[t][ds] = __builtin_bit_cast(v8, mask[t] ? raw[t][ds] : u32x4{0u, 0u, 0u, 0u});
        }
    }
#pragma unroll
    for (int d = 1; d < 16; d *= 2) seen |= __shfl_xor(seen, d);

    f32x4 o[TPW][DT];
    float m_run[TPW], l_run[TPW];  // maximum: the same in the four lanes of a row; sum: of this lane's keys
#pragma unroll
    for (int t = 0; t < TPW; ++t) {
        m_run[t] = -INFINITY;
        l_run[t] = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    int32_t kfrag[DS], vfrag[DT];  // this lane's fragment reads: K row lq piece 4 ds + lj; V row 4 lj + (lq >> 2)
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) kfrag[ds] = (lq * C::c8 + ((4 * ds + lj) ^ C::kswz(lq))) * 16;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
        const int d0 = 16 * dt + 4 * (lq & 3), r = 4 * lj + (lq >> 2);
        vfrag[dt] = (r * C::c8 + ((d0 >> 3) ^ C::vswz(r))) * 16 + (d0 & 4) * 2;
    }

    // ---- one sub-tile; `masked`: it reaches past the committed tokens, or into a page outside the pool ----
    auto step = [&](char* Ks, auto masked, int32_t key0) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        char* const Vs = Ks + C::kTensor;
        v8 kf[DS][2];
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
                kf[ds][kt] = __builtin_bit_cast(v8, *reinterpret_cast<const u32x4*>(Ks + kfrag[ds] + 16 * kt * D * 2));
        uint32_t bad = 0;    // halves outside the pool
        bool spill = false;  // some value row that only some rows see holds an infinity or NaN
        if constexpr (kMasked) {
#pragma unroll
            for (int half = 0; half < 2; ++half)
                if (pages.outside(key0 + 16 * half)) bad |= 1u << half;
            // V rows that no row sees become zero (their weights are, and 0 * V must
            // be); two lanes a row, each half of its pieces
            const int r = lane >> 1;
            const int32_t u = key0 + r - length;
            const bool used = !((bad >> (r >> 4)) & 1) && (u < 0 || (u < 64 && ((seen >> (u & 63)) & 1)));
            uint32_t special = 0;
#pragma unroll
            for (int c = 0; c < C::c8 / 2; ++c) {
                u32x4* const p = reinterpret_cast<u32x4*>(Vs + (r * C::c8 + (lane & 1) * (C::c8 / 2) + c) * 16);
                if (!used)
                    *p = u32x4{0u, 0u, 0u, 0u};
                else if (u >= 0)
                    special |= special_pairs<T>(*p);
            }
            spill = __any(special != 0);
        }
        u32x4 hi[TPW], lo[TPW];
        uint32_t vis[TPW];  // bit 4 kt + i: key 16 kt + 4 lj + i is seen
#pragma unroll
        for (int t = 0; t < TPW; ++t) {
            if (t >= tiles) continue;
            f32x4 st[2];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                st[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ds = 0; ds < DS; ++ds) st[kt] = M::mma(kf[ds][kt], qf[t][ds], st[kt]);
            }
            if constexpr (kMasked) {
                vis[t] = 0;
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int32_t u = key0 + 16 * kt + 4 * lj + i - length;
                        const bool ok = mask[t] != 0 && !((bad >> kt) & 1) &&
                                        (u < 0 || (u < 64 && ((mask[t] >> (u & 63)) & 1)));
                        st[kt][i] = ok ? st[kt][i] : -INFINITY;
                        vis[t] |= static_cast<uint32_t>(ok) << (4 * kt + i);
                    }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) mx = fmaxf(mx, st[kt][i]);
            mx *= a.scale_log2;  // positive: the largest stays the largest
            if (__any(mx > m_run[t] + L::kHead)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float m_new = mx > m_run[t] + L::kHead ? mx : m_run[t];
                const float alpha = __builtin_amdgcn_exp2f(m_run[t] - (m_new == -INFINITY ? 0.f : m_new));
                m_run[t] = m_new;
                l_run[t] *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[t][dt] *= alpha;
            }
            const float neg = L::kLog2 - (m_run[t] == -INFINITY ? 0.f : m_run[t]);
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[e >> 2][e & 3], a.scale_log2, neg));
                l_run[t] += p[e];
            }
            uint32_t h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) M::split(p[2 * e], p[2 * e + 1], h[e], l[e]);
            hi[t] = u32x4{h[0], h[1], h[2], h[3]};
            lo[t] = u32x4{l[0], l[1], l[2], l[3]};
        }
        if (spill) {
#pragma unroll
            for (int t = 0; t < TPW; ++t)
                if (t < tiles) add_seen<T, D>(o[t], Vs, hi[t], lo[t], vis[t], lq, lj);
            return;
        }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(Vs + vfrag[dt]));
            const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(Vs + vfrag[dt] + 16 * D * 2));
            const v8 vf = __builtin_bit_cast(v8, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
            for (int t = 0; t < TPW; ++t)
                if (t < tiles) {
                    o[t][dt] = M::mma(vf, __builtin_bit_cast(v8, hi[t]), o[t][dt]);
                    o[t][dt] = M::mma(vf, __builtin_bit_cast(v8, lo[t]), o[t][dt]);
                }
        }
    };

    // sub-tile s has landed in `stage`; worked on, its buffer takes sub-tile s + kTreeWaves * kStages
    auto turn = [&](int32_t s, char* stage, auto masked) __attribute__((always_inline)) {
        const int32_t next = s + kTreeWaves * C::kStages, key0 = key_begin + kSub * s;
        const int32_t key1 = key_begin + kSub * min(next, n_sub - 1);
        const uint32_t p0 = pages.of(key1), p1 = pages.of(key1 + 16);
        __builtin_amdgcn_sched_barrier(0);
        // the later stages may still be in flight; behind the last refill any of them may be missing
        if (s + kTreeWaves * (C::kStages - 1) < n_sub)
            wait_vm<(C::kStages - 1) * NL>();
        else
            wait_vm<0>();
        step(stage, masked, key0);
        if (next < n_sub) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this stage has been read
            load(next, stage, p0, p1);
        }
    };
    // a page outside the pool anywhere in the run: all of it goes the careful way
    const bool strange = pages.any_outside(lane);
    const int32_t plain = strange ? 0 : min(n_sub, max(0, (length - key_begin) / kSub));
    int32_t s = wave, stage = 0;
#pragma unroll 1
    for (; s < plain; s += kTreeWaves) {
        turn(s, ring + stage, std::integral_constant<bool, false>{});
        stage = stage + C::kStage == C::kRing ? 0 : stage + C::kStage;
    }
#pragma unroll 1
    for (; s < n_sub; s += kTreeWaves) {
        turn(s, ring + stage, std::integral_constant<bool, true>{});
        stage = stage + C::kStage == C::kRing ? 0 : stage + C::kStage;
    }

    // ---- join: wave w owns d tiles [w DT / 4, (w + 1) DT / 4) of every row tile ----
    constexpr int SL = DT / kTreeWaves;
    f32x4* const xo = reinterpret_cast<f32x4*>(smem);  // [wave][tile][d tile][lane]
    float2* const xml = reinterpret_cast<float2*>(smem + static_cast<size_t>(kTreeWaves) * TPW * DT * 1024);
    __syncthreads();  // every ring is done with
#pragma unroll
    for (int t = 0; t < TPW; ++t) {
        if (t >= tiles) continue;
        float l = l_run[t];
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) xo[((wave * TPW + t) * DT + dt) * 64 + lane] = o[t][dt];
        xml[(wave * TPW + t) * 64 + lane] = float2{m_run[t], l};
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TPW; ++t) {
        if (t >= tiles) continue;
        float m[kTreeWaves], l[kTreeWaves], top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kTreeWaves; ++w) {
            const float2 ml = xml[(w * TPW + t) * 64 + lane];
            m[w] = ml.x;
            l[w] = ml.y;
            top = fmaxf(top, ml.x);
        }
        const float use = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
        f32x4 res[SL];
#pragma unroll
        for (int j = 0; j < SL; ++j) res[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kTreeWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(m[w] - use);
            sum += l[w] * f;
#pragma unroll
            for (int j = 0; j < SL; ++j) res[j] += xo[((w * TPW + t) * DT + wave * SL + j) * 64 + lane] * f;
        }
        if (16 * t + lq < live)
            put_row<T, D, SL>(a, res, top, sum, mask[t] != 0, kv_head, group, 16 * TPW, first, 16 * t + lq, row0, part,
                              wave * SL, lj);
    }
}

// ---------------------------------------------------------------------------
// More than 32 query rows: eight waves, each with 32 of the block's 32 U rows (two
// tiles: PairWave) and one of X = 8 / U key classes, over 128-key stages that all of
// them load and share, double-buffered. With U = 4 and 8 and heads of 128 a wave walks
// its two or four sub-tiles of a stage in the software-pipelined order of the head-pair
// kernel (26 drafted rows of 12 requests 104 -> 98 us). Four stages of half the
// size instead of two timed the same with U = 4, and 94 instead of 88 us with U = 2
// (16 drafted rows of 12 requests).
// ---------------------------------------------------------------------------
constexpr int kWideThreads = 512;

template <int D, int U>
struct WideCfg {
    static constexpr int kKeys = kPairStepKeys;  // of a stage
    static constexpr int kStage = PairCfg<D>::stage_bytes;
    static constexpr int kTensor = PairCfg<D>::tensor_bytes;
    static constexpr int kHalves = kKeys / 16;
    static constexpr int kLoads = PairCfg<D>::loads;  // of K or V, a wave
    static constexpr int kJoin = U == 8 ? 0 : 8 * 2 * (D / 16 * 1024 + 64 * 8);
    static constexpr int kLds = kJoin > 2 * kStage ? kJoin : 2 * kStage;
};

template <typename T, int D, int U>
__device__ inline void wide_item(const TreeArgs& a, uniform_i32* at, int kv_head, int group, char* smem) {
    using C = PairCfg<D>;
    using S = WideCfg<D, U>;
    using W = PairWave<T, D, true, true>;
    using v8 = typename W::v8;
    constexpr int X = 8 / U;               // key classes
    constexpr int DT = W::DT;
    constexpr int kRows = 512 / C::c8;     // rows that one load of the eight waves covers
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // no value of an item is kept over the loop of items
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lq = lane & 15, lj = lane >> 4;
    const int unit = wave % U, kq = wave / U;
    const int32_t request = at[0], key_begin = at[1], key_end = at[2], part = at[3], length = at[4];
    const int32_t nodes = at[5], row0 = at[6], rows = at[7];
    const int32_t first = group * 32 * U;
    const int32_t live = nodes * a.group - first;  // the block's rows
    if (nodes == 0) {
        if (group == 0) zero_rows<D>(a, kv_head, row0, rows, kWideThreads);
        return;
    }
    if (live <= 0) return;
    const int32_t mine = live - 32 * unit;         // rows of this wave and the ones behind it

    // ---- this wave's loads: rows l kRows + wave_row .. of a stage, all in one page ----
    const ItemPages item_pages(a, request, key_begin, key_end);
    const int wave_row = 64 * wave / C::c8;
    const int r0 = wave_row + lane / C::c8;
    const int c = lane % C::c8;
    const uint32_t koff = (lane / C::c8) * a.k_row + 16 * (c ^ C::kswz(r0));
    const uint32_t voff = (lane / C::c8) * a.v_row + 16 * (c ^ C::vswz(r0));
    const char* const kbase = a.k + kv_head * a.k_head;
    const char* const vbase = a.v + kv_head * a.v_head;
    const uint32_t page_mask = (1u << a.page_log2) - 1;
    const int32_t n_st = (key_end - key_begin + S::kKeys - 1) / S::kKeys;
    struct Pages {
        uint32_t of[S::kLoads];  // of this wave's loads
    };
    auto pages_of = [&](int32_t i) __attribute__((always_inline)) -> Pages {
        Pages p;
#pragma unroll
        for (int l = 0; l < S::kLoads; ++l) p.of[l] = item_pages.of(key_begin + S::kKeys * i + l * kRows + wave_row);
        return p;
    };
    // stage i into its buffer
    auto load = [&](int32_t i, const Pages& pages) __attribute__((always_inline)) {
        char* const stage = smem + (i & 1) * S::kStage;
#pragma unroll
        for (int l = 0; l < S::kLoads; ++l) {
            const uint32_t page = pages.of[l];
            const uint32_t row = (key_begin + S::kKeys * i + l * kRows + wave_row) & page_mask;
            lds_dma16_once(kbase + (static_cast<uint64_t>(page) * a.k_page + row * a.k_row), koff,
                           stage + (8 * l + wave) * 1024);
            lds_dma16_once(vbase + (static_cast<uint64_t>(page) * a.v_page + row * a.v_row), voff,
                           stage + S::kTensor + (8 * l + wave) * 1024);
        }
    };

    // ---- queries, masks and the first stage in one round trip ----
    W w;
    w.init(lq, lj);
    uint64_t mask[2], seen;
    {
        u32x4 raw[2][W::DS];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int32_t r = min(first + 32 * unit + 16 * t + lq, nodes * a.group - 1);
            const int64_t row = row0 + r / a.group;
            const int64_t head = static_cast<int64_t>(kv_head) * a.group + r % a.group;
            mask[t] = a.masks[row];
#pragma unroll
            for (int ds = 0; ds < W::DS; ++ds)
                raw[t][ds] = *reinterpret_cast<const u32x4*>(a.q + (head * a.qs[0] + row * a.qs[1] + 32 * ds + 8 * lj) * 2);
        }
        const uint64_t node = a.masks[row0 + min(lane, nodes - 1)];
        load(0, pages_of(0));
        asm volatile("" : "+v"(mask[0]), "+v"(mask[1]));
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if (16 * t + lq >= mine) mask[t] = 0;
#pragma unroll
            for (int ds = 0; ds < W::DS; ++ds) {
                asm volatile("" : "+v"(raw[t][ds]));
                w.qf[t][ds] = __builtin_bit_cast(v8, mask[t] ? raw[t][ds] : u32x4{0u, 0u, 0u, 0u});
            }
        }
        seen = __ballot(lane < nodes && node != 0);  // nodes that some row of the request attends to
    }
    Pages next = pages_of(1);

    // A sub-tile that reaches past the committed tokens, or into a page outside the pool.
    auto masked_step = [&](const char* Ks, const char* Vs, int32_t key0, uint32_t bad_halves, bool spill) {
        v8 kf[W::DS][2];
        w.read_k(Ks, kf);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            f32x4 st[2];
            w.qk(t, kf, st);
            uint32_t vis = 0;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int32_t u = key0 + 16 * kt + 4 * lj + i - length;
                    const bool ok = mask[t] != 0 && !((bad_halves >> kt) & 1) &&
                                    (u < 0 || (u < 64 && ((mask[t] >> (u & 63)) & 1)));
                    st[kt][i] = ok ? st[kt][i] : -INFINITY;
                    vis |= static_cast<uint32_t>(ok) << (4 * kt + i);
                }
            float x[2][4];
            w.rescale_if(t, w.row_max(st, a.scale_log2, x));
            u32x4 hi, lo;
            w.probs(t, x, a.scale_log2, hi, lo);
            if (!spill) {
                v8 vf[DT];
                w.read_v(Vs, vf);
                w.pv(t, vf, hi, lo);
                continue;
            }
            w.lsum[t] = W::M::mma(w.ones, __builtin_bit_cast(v8, hi), w.lsum[t]);
            w.lsum[t] = W::M::mma(w.ones, __builtin_bit_cast(v8, lo), w.lsum[t]);
            add_seen<T, D>(w.o[t], Vs, hi, lo, vis, lq, lj);
        }
    };

    // stage i has landed and every wave is past stage i - 1, whose buffer takes stage i + 1
    auto turn = [&](int32_t i) __attribute__((always_inline)) {
        wait_vm<0>();
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (i + 1 < n_st) {
            load(i + 1, next);
            next = pages_of(i + 2);
        }
    };
    // whole stages of committed tokens; with a page outside the pool anywhere all go the careful way
    const bool strange = item_pages.any_outside(lane);
    const int32_t plain = strange ? 0 : min(n_st, max(0, (length - key_begin) / S::kKeys));
    int32_t i = 0;
    for (; i < plain; ++i) {
        turn(i);
        const char* Ks = smem + (i & 1) * S::kStage;
        const char* Vs = Ks + S::kTensor;
        if (mine <= 0) continue;
        if constexpr (X < kPairSubs && D == 128) {
            w.template stage_pipelined<kPairSubs / X, X>(Ks + kPairSub * kq * D * 2, Vs + kPairSub * kq * D * 2, 0, INT32_MAX,
                                                        INT32_MAX, lj, a.scale_log2);
        } else {
#pragma unroll 1
            for (int j = kq; j < kPairSubs; j += X)
                w.step(Ks + kPairSub * j * D * 2, Vs + kPairSub * j * D * 2, false, 0, lj, a.scale_log2);
        }
    }
#pragma unroll 1
    for (; i < n_st; ++i) {
        turn(i);
        uint32_t bad = 0;  // halves (16 keys) outside the pool
#pragma unroll
        for (int h = 0; h < S::kHalves; ++h)
            if (item_pages.outside(key_begin + S::kKeys * i + 16 * h)) bad |= 1u << h;
        char* const Ks = smem + (i & 1) * S::kStage;
        char* const Vs = Ks + S::kTensor;
        const int32_t key0 = key_begin + S::kKeys * i;
        // V rows that no row of the request sees become zero (their weights are, and 0 * V must be)
        uint32_t special = 0;
        for (int e = tid; e < S::kKeys * C::c8; e += kWideThreads) {
            const int r = e / C::c8;
            const int32_t u = key0 + r - length;
            u32x4* const p = reinterpret_cast<u32x4*>(Vs + e * 16);
            if (((bad >> (r >> 4)) & 1) || !(u < 0 || (u < 64 && ((seen >> (u & 63)) & 1))))
                *p = u32x4{0u, 0u, 0u, 0u};
            else if (u >= 0)
                special |= special_pairs<T>(*p);
        }
        const bool spill = __syncthreads_or(special != 0);
        if (mine <= 0) continue;
#pragma unroll 1
        for (int j = kq; j < kPairSubs; j += X)
            if (key0 + kPairSub * j < key_end)
                masked_step(Ks + kPairSub * j * D * 2, Vs + kPairSub * j * D * 2, key0 + kPairSub * j,
                            (bad >> (2 * j)) & 3u, spill);
    }

    // ---- join the key classes of each unit: class kq owns d tiles [kq DT / X, (kq + 1) DT / X) ----
    constexpr int SL = DT / X;
    float l_run[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        float l = w.lsum[t][0];
        l += __shfl_xor(l, 16);
        l_run[t] = l + __shfl_xor(l, 32);
    }
    f32x4* const xo = reinterpret_cast<f32x4*>(smem);  // [wave][tile][d tile][lane]
    float2* const xml = reinterpret_cast<float2*>(smem + static_cast<size_t>(8) * 2 * DT * 1024);
    if constexpr (X > 1) {
        __syncthreads();  // every wave is done with the steps
        if (mine > 0) {
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) xo[((wave * 2 + t) * DT + dt) * 64 + lane] = w.o[t][dt];
                xml[(wave * 2 + t) * 64 + lane] = float2{w.m_run[t], l_run[t]};
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        f32x4 res[SL];
        float top = w.m_run[t], sum = l_run[t];
        if constexpr (X == 1) {
#pragma unroll
            for (int j = 0; j < SL; ++j) res[j] = w.o[t][j];
        } else {
            if (mine <= 0) break;
            float m[X], l[X];
            top = -INFINITY;
#pragma unroll
            for (int o = 0; o < X; ++o) {
                const float2 ml = xml[((o * U + unit) * 2 + t) * 64 + lane];
                m[o] = ml.x;
                l[o] = ml.y;
                top = fmaxf(top, ml.x);
            }
            const float use = top == -INFINITY ? 0.f : top;
            sum = 0.f;
#pragma unroll
            for (int j = 0; j < SL; ++j) res[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int o = 0; o < X; ++o) {
                const float f = __builtin_amdgcn_exp2f(m[o] - use);
                sum += l[o] * f;
#pragma unroll
                for (int j = 0; j < SL; ++j) res[j] += xo[(((o * U + unit) * 2 + t) * DT + kq * SL + j) * 64 + lane] * f;
            }
        }
        if (16 * t + lq < mine)
            put_row<T, D, SL>(a, res, top, sum, mask[t] != 0, kv_head, group, 32 * U, first, 32 * unit + 16 * t + lq,
                              row0, part, kq * SL, lj);
    }
}

// A worker's items, one after another. ROWS query rows a block.
template <typename T, int D, int ROWS>
__global__ void __launch_bounds__(ROWS <= 32 ? kTreeThreads : kWideThreads) tree_attention_kernel(TreeArgs a) {
    extern __shared__ __align__(16) char smem[];
    const int kv_head = blockIdx.x % a.kv_heads;
    const int group = blockIdx.x / a.kv_heads;
    uniform_i32* first_of = reinterpret_cast<uniform_i32*>(
        reinterpret_cast<uint64_t>(a.schedule + kStepHeader + blockIdx.y));
    const int32_t end = first_of[1];
    const int32_t* work = a.schedule + kStepHeader + step_worker_ints(a.workers);
#pragma unroll 1
    for (int32_t i = first_of[0]; i < end; ++i) {
        uniform_i32* at =
            reinterpret_cast<uniform_i32*>(reinterpret_cast<uint64_t>(work + static_cast<int64_t>(i) * kStepItem));
        if constexpr (ROWS <= 32)
            tree_item<T, D, ROWS / 16>(a, at, kv_head, group, smem);
        else
            wide_item<T, D, ROWS / 32>(a, at, kv_head, group, smem);
        __syncthreads();  // the item's LDS has been read
    }
    if (a.zero_rest) {
        const int32_t total = a.row_starts[a.requests];
        const int64_t per = static_cast<int64_t>(a.group) * (D / 4);  // 8-byte pieces of a row
        const int64_t pieces = (a.rows - total) * per;
        const int64_t part = static_cast<int64_t>(blockIdx.y) * a.row_groups + group;
        for (int64_t e = part * blockDim.x + threadIdx.x; e < pieces;
             e += static_cast<int64_t>(a.workers) * a.row_groups * blockDim.x) {
            const int64_t row = total + e / per, piece = e % per;
            const int64_t head = static_cast<int64_t>(kv_head) * a.group + piece / (D / 4);
            *reinterpret_cast<uint2*>(a.out + (head * a.os[0] + row * a.os[1] + piece % (D / 4) * 4) * 2) = uint2{0u, 0u};
        }
    }
}

// The chunks of a split request's row, in order: block = one query row of one
// split request, eight slices of the chunks joined through LDS. Latency: 3.6 us for one
// request's row, 8.3 for 26 rows of 12 (blocks of four rows took 7.0 there and 10.4
// instead of 8.9 for 64 rows of one request).
constexpr int kMergeThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(TreeArgs a, int32_t group_rows) {
    using E = elem<T>;
    constexpr int kLanes = D / 4;                       // threads of a row
    constexpr int kSlices = kMergeThreads / kLanes;
    __shared__ f32x4 so[kSlices][kLanes];
    __shared__ float2 sml[kSlices];
    if (static_cast<int32_t>(blockIdx.y) >= a.schedule[1]) return;
    const int32_t* split = a.schedule + kStepHeader + step_worker_ints(a.workers) +
                           static_cast<int64_t>(a.items) * kStepItem + blockIdx.y * kStepSplit;
    const int32_t worker = split[0], chunks = split[1], nodes = split[2], row0 = split[3];
    const int32_t rows_all = a.row_groups * group_rows;
    const int32_t kv_head = blockIdx.x / rows_all, qr = blockIdx.x % rows_all;
    if (qr >= nodes * a.group) return;
    const int lane = threadIdx.x % kLanes, slice = threadIdx.x / kLanes;
    float m = -INFINITY, l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int32_t c = slice; c < chunks; c += kSlices) {
        const int64_t r = (static_cast<int64_t>(step_partial(worker, c)) * a.kv_heads + kv_head) * rows_all + qr;
        const float mc = a.part_ml[2 * r], lc = a.part_ml[2 * r + 1];
        const f32x4 oc = *reinterpret_cast<const f32x4*>(a.part_o + r * D + 4 * lane);
        const float top = fmaxf(m, mc), use = top == -INFINITY ? 0.f : top;
        const float f = __builtin_amdgcn_exp2f(m - use), g = __builtin_amdgcn_exp2f(mc - use);
        l = l * f + lc * g;
        o = o * f + oc * g;
        m = top;
    }
    so[slice][lane] = o;
    if (lane == 0) sml[slice] = float2{m, l};
    __syncthreads();
    if (slice != 0) return;
    float top = -INFINITY;
#pragma unroll
    for (int s = 0; s < kSlices; ++s) top = fmaxf(top, sml[s].x);
    const float use = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 res = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < kSlices; ++s) {
        const float f = __builtin_amdgcn_exp2f(sml[s].x - use);
        sum += sml[s].y * f;
        res += so[s][lane] * f;
    }
    const int64_t row = row0 + qr / a.group, head = static_cast<int64_t>(kv_head) * a.group + qr % a.group;
    const bool none = a.masks[row] == 0 || sum == 0.f;
    const float inv = 1.f / sum;
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) e[i] = none ? 0u : E::from_float(res[i] * inv);
    *reinterpret_cast<uint2*>(a.out + (head * a.os[0] + row * a.os[1] + 4 * lane) * 2) =
        uint2{e[0] | (e[1] << 16), e[2] | (e[3] << 16)};
}

// ROWS query rows a block.
template <typename T, int D, int ROWS>
int launch_tree(const TreeArgs& a, const StepShape& s, hipStream_t stream) {
    const dim3 grid(static_cast<unsigned>(a.kv_heads * s.row_groups), static_cast<unsigned>(s.workers));
    constexpr size_t lds = ROWS <= 32 ? tree_lds<D, ROWS / 16>() : WideCfg<D, ROWS / 32>::kLds;
    static LdsGrant grant;
    if (!grant.ok(tree_attention_kernel<T, D, ROWS>, lds)) return KVR_E_LAUNCH_FAILED;
    tree_attention_kernel<T, D, ROWS><<<grid, ROWS <= 32 ? kTreeThreads : kWideThreads, lds, stream>>>(a);
    if (s.workers > 1) {
        const dim3 merge(static_cast<unsigned>(a.kv_heads * s.row_groups * s.group_rows), static_cast<unsigned>(s.splits));
        tree_merge_kernel<T, D><<<merge, kMergeThreads, 0, stream>>>(a, static_cast<int32_t>(s.group_rows));
    }
    return launch_status();
}

template <typename T, int D>
int launch_rows(const TreeArgs& a, const StepShape& s, hipStream_t stream) {
    switch (s.group_rows) {
        case 16: return launch_tree<T, D, 16>(a, s, stream);
        case 32: return launch_tree<T, D, 32>(a, s, stream);
        case 64: return launch_tree<T, D, 64>(a, s, stream);
        case 128: return launch_tree<T, D, 128>(a, s, stream);
        default: return launch_tree<T, D, 256>(a, s, stream);
    }
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

int check_tree(const kvr_step_desc* d, int32_t head_dim) {
    const int st = check_step(d);
    if (st != KVR_OK) return st;
    if (!d->schedule) return KVR_E_NULL_POINTER;
    return head_dim == 64 || head_dim == 128 ? KVR_OK : KVR_E_UNSUPPORTED_SHAPE;
}

}  // namespace
}  // namespace kvr

using namespace kvr;

extern "C" int64_t kvr_tree_workspace_bytes(const kvr_step_desc* d, int32_t head_dim) {
    const int st = check_tree(d, head_dim);
    if (st != KVR_OK) return st;
    const StepShape s = step_shape(d->requests, d->max_rows, d->q_heads, d->kv_heads);
    return s.partials * d->kv_heads * s.row_groups * s.group_rows * (head_dim + 2) * 4;
}

extern "C" int kvr_tree_attention(const void* q, const void* k, const void* v, void* out, const kvr_step_desc* d,
                                  int32_t head_dim, float scale, const int64_t strides[12], int32_t zero_rest,
                                  void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream) {
    if (dtype != KVR_DTYPE_BF16 && dtype != KVR_DTYPE_F16) return KVR_E_UNSUPPORTED_DTYPE;
    const int st = check_tree(d, head_dim);
    if (st != KVR_OK) return st;
    if (!(scale > 0.f) || !isfinite(scale)) return KVR_E_INVALID_ARGUMENT;
    if (!q || !k || !v || !out || !strides) return KVR_E_NULL_POINTER;
    for (int t = 0; t < 4; ++t) {
        const int64_t* s = strides + 3 * t;
        const int64_t unit = t == 3 ? 4 : 8;
        // a load's row offsets fit 32 bits
        if (s[0] <= 0 || s[1] <= 0 || s[2] != 1 || s[0] % unit || s[1] % unit || s[1] > (int64_t(1) << 26))
            return KVR_E_BAD_STRIDE;
        // ... and a page of K or V
        if ((t == 1 || t == 2) && s[1] * 2 * d->page_size > UINT32_MAX) return KVR_E_BAD_STRIDE;
    }
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 8)) return KVR_E_BAD_STRIDE;
    const int64_t need = kvr_tree_workspace_bytes(d, head_dim);
    if (need > 0 && (!workspace || !aligned(workspace, 16) || workspace_bytes < need)) return KVR_E_WORKSPACE_TOO_SMALL;
    const StepShape s = step_shape(d->requests, d->max_rows, d->q_heads, d->kv_heads);
    TreeArgs a;
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
    a.schedule = d->schedule;
    a.tables = d->tables;
    a.masks = d->masks;
    const int64_t part_rows = s.partials * d->kv_heads * s.row_groups * s.group_rows;
    a.part_o = static_cast<float*>(workspace);
    a.part_ml = a.part_o + part_rows * head_dim;
    a.table_stride = d->table_stride;
    a.row_starts = d->row_starts;
    a.items = static_cast<int32_t>(s.items);
    a.workers = static_cast<int32_t>(s.workers);
    a.requests = d->requests;
    a.rows = d->rows;
    a.zero_rest = zero_rest != 0;
    a.table_width = d->table_width;
    a.page_log2 = __builtin_ctz(static_cast<unsigned>(d->page_size));
    a.n_pages = static_cast<int32_t>(d->n_slots / d->page_size);
    a.kv_heads = d->kv_heads;
    a.group = d->q_heads / d->kv_heads;
    a.row_groups = static_cast<int32_t>(s.row_groups);
    a.scale_log2 = scale * 1.4426950408889634f;
    hipStream_t hs = as_stream(stream);
    if (dtype == KVR_DTYPE_BF16)
        return head_dim == 128 ? launch_rows<bf16_t, 128>(a, s, hs) : launch_rows<bf16_t, 64>(a, s, hs);
    return head_dim == 128 ? launch_rows<f16_t, 128>(a, s, hs) : launch_rows<f16_t, 64>(a, s, hs);
}
