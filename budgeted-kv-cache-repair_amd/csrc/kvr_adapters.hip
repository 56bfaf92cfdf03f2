// Projections with a low-rank adapter of each row's own beside the shared weights:
//   y[m, :] = W x_m + s_a B_a (A_a x_m)        a = ids[m]; W x_m alone where ids[m] names no adapter
// W: up to three weights, rows concatenated (q/k/v), each with its own A and B.
//
// What bounds it: up to some 200 rows reading W and, once each, the A_a and B_a of
// the adapters that the rows name; above that the matrix cores on W x. So W x runs
// on the projection kernels, and the adapters' two thin products go through the
// MFMA in tiles of 16 rows: a tile walks the distinct adapters that its rows name,
// so that rows of one adapter share its reads, and keeps of each product the
// columns of its rows.
//
//   up to 64 rows (kvr_gemm.hip):   the projection, with blocks behind its own for t = A_a x (kvr_adapters.h):
//                                   both leave fp32 partials, one a slice of k
//                                   adapter_up_kernel      y = sum of W x's partials + s_a B_a t
//   up to 256 (kvr_gemm_tiled.hip): the projection, left as partials; adapter_down_kernel, adapter_up_kernel
//   more:                           adapter_down_wide_kernel, adapter_pack_kernel    t, packed
//                                   the projection, which adds s_a B_a t to its sums (AdapterEpilogue)
//
// Measured (kernels alone, bf16): 1 row of q/k/v, 4096 to 6144, rank 16, 14.1 + 5.8 us,
// 3.6 TB/s in the first launch; 64 rows of 14336 to 4096 with 64 adapters of rank 16
// 31 + 9 us, 5.1 TB/s in the first; 4096 rows of q/k/v with rank 64, 31 + 8 + 216 to 237
// us by the card's clock, 0.9 to 1.0 PFLOP/s in the projection (180 to 209 without adapters).
//
// t enters the second product as a hi + lo pair of 16-bit values side by side in
// one MFMA (16 ranks of hi, the same 16 of lo), so it is not rounded to the input
// type. No sum depends on the order in which blocks end.
#include "kvr_adapters.h"
#include "kvr_gemm_tiled.h"
#include "kvrepair_step.h"

namespace kvr {
namespace {

constexpr int kAdapterThreads = 64 * kAdapterWaves;
constexpr int kMaxRank = 512;
constexpr int kMaxDownSplits = 32;
constexpr int kWideRows = 64;                        // rows of a block of adapter_down_wide_kernel
constexpr int32_t kWideRanks = 192;                  // its ranks, where there are more than 64
constexpr int kMaxWideSplits = 8;

// The next adapter of several tiles' rows, -1 when none is left.
template <int N>
__device__ inline int32_t next_adapter(const int32_t (&id)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint64_t waiting = __ballot(id[i] >= 0);
        if (waiting) return __builtin_amdgcn_readlane(id[i], __builtin_ctzll(waiting));
    }
    return -1;
}

// The power of two that brings the largest |t| of 16 ranks (this lane's 8 and those
// of the lane group beside it) to [0.5, 1): fp16's hi + lo pair then keeps 22 bits
// of it, whatever its size. bf16 has fp32's exponents and needs none.
template <typename T>
__device__ inline int adapter_exponent(const float (&t)[8]) {
    if constexpr (!__is_same(T, f16_t)) return 0;
    float top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(t[e]));
    top = fmaxf(top, __shfl_xor(top, 16));
    return __builtin_amdgcn_frexp_expf(top);  // 0 of zero and infinity
}

// Eight 16-bit values of t 2^-exponent: the rounded ones, or what these leave.
template <typename T>
__device__ inline u32x4 hi_or_lo(const float (&t)[8], int exponent, bool lo) {
    using E = elem<T>;
    uint32_t bits[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float v = __builtin_ldexpf(t[e], -exponent);
        const uint32_t head = E::from_float(v);
        const float of_head = E::to_float(static_cast<uint16_t>(head));
        const uint32_t rest = __builtin_isinf(of_head) ? 0u : E::from_float(v - of_head);
        bits[e] = lo ? rest : head;
    }
    return u32x4{bits[0] | (bits[1] << 16), bits[2] | (bits[3] << 16), bits[4] | (bits[5] << 16),
                 bits[6] | (bits[7] << 16)};
}

// Block = (64 columns, 16 rows), a wave 16 columns: the sum of W x's partials in
// split order, then the distinct adapters of the rows, eight at a time. MFMA
// roles: A = 16 rows of B_a (columns of y), 16 ranks twice; B = [hi | lo] of 16
// ranks of t. Latency: 5.8 us for 1 row, 8.8 for 64 (all ranks' t summed first, and B_a
// of the next 16 ranks in flight beside the MFMAs: 6.6 and 10.0).
template <typename T>
__global__ void __launch_bounds__(kAdapterThreads) adapter_up_kernel(AdapterArgs a) {
    using G = tile_t<T>;
    using E = elem<T>;
    using v8 = typename G::v8;
    constexpr int kBatch = 8;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lq = lane & 15, lj = lane >> 4;
    const int32_t columns = (a.n + 63) / 64;
    const int32_t tile = blockIdx.x % columns;
    const int32_t n0 = tile * 64 + wave * 16;
    __shared__ f32x4 sums[kAdapterWaves][2][64];
    const int32_t row = blockIdx.x / columns * 16 + lq;
    const int32_t row_in = row < a.m ? row : a.m - 1;
    const int32_t id = adapter_of(a, row);
    const uint32_t firsts = first_rows(id, lq);
    const float scale = id >= 0 ? a.scales[id] : 0.f;
    const float* at = a.base + (static_cast<int64_t>(tile) * a.splits * a.base_rows + row_in) * 64 + wave * 16 + 4 * lj;
    const int64_t step = static_cast<int64_t>(a.base_rows) * 64;
    f32x4 acc = *reinterpret_cast<const f32x4*>(at);  // past the last column: of the last partial tile, never written
#pragma unroll 4
    for (int s = 1; s < a.splits; ++s) acc += *reinterpret_cast<const f32x4*>(at + s * step);
    const int64_t inner = static_cast<int64_t>(a.weights) * a.rank;
    const int32_t col = n0 + lq;
    const int half = lj & 1;  // ranks 8 half .. of a chunk of 16; lanes of lj >= 2 hold lo
    const u32x4 zero = {0u, 0u, 0u, 0u};
    for (int w = 0; firsts != 0 && w < a.weights; ++w) {
        const int32_t begin = w ? a.end[w - 1] : 0, end = a.end[w];
        if (end <= tile * 64 || begin >= min(tile * 64 + 64, a.n)) continue;  // the same in all waves
        const int32_t rows_w = end - begin;
        const bool col_in = col >= begin && col < end;
        const char* const up = a.up[w] + static_cast<int64_t>(col_in ? col - begin : 0) * a.rank * 2;
        for (int r0 = 0; r0 < a.rank; r0 += kRankTile) {
            const int r = r0 + 8 * half;
            const bool in = col_in && r < a.rank;
            uint32_t left = firsts;
            u32x4 bf[kBatch];
            int32_t ad[kBatch];
            // the batch's rows of B, -1 behind the last adapter
            auto batch = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                    ad[b] = left ? __builtin_amdgcn_readlane(id, __builtin_ctz(left)) : -1;
                    bf[b] = zero;
                    if (left && in)
                        bf[b] = *reinterpret_cast<const u32x4*>(up + (static_cast<int64_t>(ad[b]) * rows_w * a.rank + r) * 2);
                    left &= left - 1;
                }
            };
            batch();
            // t of the rows: every wave sums a quarter of the slices, then the four in order
            f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
            if (id >= 0 && r < a.rank) {
                const float* from = a.inner + static_cast<int64_t>(row) * inner + static_cast<int64_t>(w) * a.rank + r;
                const int64_t split = a.m * inner;
#pragma unroll 4
                for (int s = wave; s < a.down_splits; s += kAdapterWaves) {
                    lo += *reinterpret_cast<const f32x4*>(from + s * split);
                    hi += *reinterpret_cast<const f32x4*>(from + s * split + 4);
                }
            }
            sums[wave][0][lane] = lo;
            sums[wave][1][lane] = hi;
            __syncthreads();
            lo = sums[0][0][lane];
            hi = sums[0][1][lane];
#pragma unroll
            for (int o = 1; o < kAdapterWaves; ++o) {
                lo += sums[o][0][lane];
                hi += sums[o][1][lane];
            }
            __syncthreads();
            float t[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = (e < 4 ? lo[e] : hi[e - 4]) * scale;
            const int exponent = adapter_exponent<T>(t);
            const v8 tf = __builtin_bit_cast(v8, hi_or_lo<T>(t, exponent, lj >= 2));
            f32x4 found = {0.f, 0.f, 0.f, 0.f};
            for (;;) {
#pragma unroll
                for (int b = 0; b < kBatch; ++b) {
                    const f32x4 none = {0.f, 0.f, 0.f, 0.f};
                    const f32x4 d = G::mma(__builtin_bit_cast(v8, bf[b]), tf, none);
                    found = id >= 0 && id == ad[b] ? d : found;
                }
                if (!left) break;
                batch();
            }
            // what an infinity or NaN of one weight or adapter makes of a product stays
            // in its own columns and rows
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int32_t c = n0 + 4 * lj + i;
                if (id >= 0 && c >= begin && c < end) acc[i] += __builtin_ldexpf(found[i], exponent);
            }
        }
    }
    if (row >= a.m) return;
    uint16_t* y = reinterpret_cast<uint16_t*>(a.y) + static_cast<int64_t>(row) * a.ldy + n0 + 4 * lj;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n0 + 4 * lj + i < a.n) y[i] = E::from_float(acc[i]);
}

// The inner products of up to kSomeRows rows.
template <typename T>
__global__ void __launch_bounds__(kAdapterThreads) adapter_down_kernel(AdapterArgs a) {
    adapter_down_block<T, tile_t<T>>(a, blockIdx.x);
}

// More than kSomeRows rows: block = (64 rows, 64 RT ranks of all weights' one after
// another, slice of k); wave w has RT tiles of 16 ranks for all rows. Stages of 64 k
// of the ranks and of x go straight into LDS, three in flight, as in the tiled
// projection (read from memory by each wave, 4096 rows of 4096 k and 192 ranks took
// 56 us). Rows of a prompt name one or two adapters; every adapter that the block's
// rows name is a pass over the slice.
constexpr int kWideStages = 4;

template <int RT>
constexpr int wide_stage_bytes() { return (64 * RT + kWideRows) * kRowBytes; }

template <typename T, int RT>
__global__ void __launch_bounds__(kAdapterThreads) adapter_down_wide_kernel(AdapterArgs a) {
    using G = tile_t<T>;
    using v8 = typename G::v8;
    constexpr int kTiles = kWideRows / 16, kStage = wide_stage_bytes<RT>();
    constexpr int kRankGroups = 64 * RT / kGroupRows, kGroups = kRankGroups + kWideRows / kGroupRows;
    constexpr int L = kGroups / kAdapterWaves;  // loads of a stage, a wave
    static_assert(kGroups % kAdapterWaves == 0, "every wave loads as much");
    extern __shared__ __align__(16) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lq = lane & 15, lj = lane >> 4;
    const int32_t ranks = a.weights * a.rank;
    const int32_t g0 = blockIdx.y * 64 * RT;
    const int32_t m0 = blockIdx.x * kWideRows;
    const int32_t k0 = blockIdx.z * a.turns * kStageK;
    const int32_t steps = min(a.turns, (a.k - k0) / kStageK);  // k is a multiple of 64
    int32_t id[kTiles];
#pragma unroll
    for (int i = 0; i < kTiles; ++i) id[i] = adapter_of(a, m0 + 16 * i + lq);

    // ---- this wave's loads: group g = 8 rows of [ranks | x] ----
    const int lr = lane >> 3;
    const char* base[L];   // of an adapter's pool (ranks: the weight's, first adapter), or of x
    uint32_t off[L], dst[L];
#pragma unroll
    for (int l = 0; l < L; ++l) {
        const int g = wave + l * kAdapterWaves;
        const int piece = (lane & 7) ^ swz((g * kGroupRows + lr) & 15);
        if (g < kRankGroups) {
            // a weight's ranks are a multiple of 8: a group is of one weight
            const int32_t rank = min(g0 + g * kGroupRows, ranks - kGroupRows), w = rank / a.rank;
            const char* const pool = w == 0 ? a.down[0] : w == 1 ? a.down[1] : a.down[2];
            base[l] = uniform(pool + (static_cast<int64_t>(rank - w * a.rank) * a.k + k0) * 2);
            off[l] = static_cast<uint32_t>(lr * a.k * 2 + piece * 16);
        } else {
            const int32_t row = (g - kRankGroups) * kGroupRows + lr;
            base[l] = uniform(a.x + (static_cast<int64_t>(m0) * a.ldx + k0) * 2);
            off[l] = static_cast<uint32_t>(min(row, a.m - 1 - m0) * a.ldx * 2) + piece * 16;
        }
        dst[l] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(
            reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)smem) + g * 1024));
    }
    const char* frag[2];  // this lane's fragment reads of row lq, k 32 kk + 8 lj
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) frag[kk] = smem + lq * kRowBytes + (((kk * 4 + lj) ^ swz(lq)) * 16);

    for (int32_t ad = next_adapter(id); ad >= 0; ad = next_adapter(id)) {
        uint32_t here = 0;  // row tiles that name it
#pragma unroll
        for (int i = 0; i < kTiles; ++i) here |= __any(id[i] == ad) ? 1u << i : 0u;
        const int64_t of_adapter = static_cast<int64_t>(ad) * a.rank * a.k * 2;
        auto load = [&](int32_t s) __attribute__((always_inline)) {
#pragma unroll
            for (int l = 0; l < L; ++l) {
                const bool rank = wave + l * kAdapterWaves < kRankGroups;
                load_lds(uniform(base[l] + (rank ? of_adapter : 0) + static_cast<int64_t>(s) * kRowBytes), off[l],
                         dst[l] + s % kWideStages * kStage);
            }
        };
        f32x4 acc[RT][kTiles];
#pragma unroll
        for (int g = 0; g < RT; ++g)
#pragma unroll
            for (int i = 0; i < kTiles; ++i) acc[g][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int32_t s = 0; s < kWideStages - 1; ++s)
            if (s < steps) load(s);
        for (int32_t s = 0; s < steps; ++s) {
            if (s + kWideStages - 2 < steps)
                wait_vm<(kWideStages - 2) * L>();
            else
                wait_vm<0>();
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            // every wave is past stage s - 1, whose buffer takes stage s + kWideStages - 1
            if (s + kWideStages - 1 < steps) load(s + kWideStages - 1);
            const int at = s % kWideStages * kStage;
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                u32x4 af[RT], xf[kTiles];
#pragma unroll
                for (int g = 0; g < RT; ++g)
                    af[g] = *reinterpret_cast<const u32x4*>(frag[kk] + at + (wave * RT + g) * 16 * kRowBytes);
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
                    xf[i] = *reinterpret_cast<const u32x4*>(frag[kk] + at + (64 * RT + 16 * i) * kRowBytes);
#pragma unroll
                for (int i = 0; i < kTiles; ++i)
                    if ((here >> i) & 1)
#pragma unroll
                        for (int g = 0; g < RT; ++g)
                            acc[g][i] = G::mma(__builtin_bit_cast(v8, af[g]), __builtin_bit_cast(v8, xf[i]), acc[g][i]);
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");  // the last stages have been read
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
            if (id[i] != ad) continue;
            float* const to = a.inner + (blockIdx.z * static_cast<int64_t>(a.m) + m0 + 16 * i + lq) * ranks;
#pragma unroll
            for (int g = 0; g < RT; ++g) {
                const int32_t rank = g0 + (wave * RT + g) * kRankTile + 4 * lj;
                if (rank < ranks) *reinterpret_cast<f32x4*>(to + rank) = acc[g][i];
            }
            id[i] = -1;
        }
    }
}

// t of more than kSomeRows rows as the epilogue reads it: the sum of the slices, scaled,
// chunks of 16 ranks as 16 hi and 16 lo values. A row's ranks of one weight by a
// group of `width` lanes (a power of two).
template <typename T>
__global__ void __launch_bounds__(kAdapterThreads) adapter_pack_kernel(AdapterArgs a, int32_t width) {
    using E = elem<T>;
    constexpr int kMost = kMaxRank / 64;
    const int32_t chunks = (a.rank + kRankTile - 1) / kRankTile;
    const int64_t unit = (static_cast<int64_t>(blockIdx.x) * kAdapterThreads + threadIdx.x) / width;
    const int lane = threadIdx.x % width;
    const int64_t row = unit / a.weights;
    const int32_t w = static_cast<int32_t>(unit - row * a.weights);
    const int32_t id = row < a.m ? adapter_of(a, static_cast<int32_t>(row)) : -1;
    const float scale = id >= 0 ? a.scales[id] : 0.f;
    const int64_t ranks = static_cast<int64_t>(a.weights) * a.rank;
    const float* const from = a.inner + row * ranks + static_cast<int64_t>(w) * a.rank;
    float v[kMost], top = 0.f;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int r = lane + i * width;
        v[i] = 0.f;
        if (id >= 0 && r < a.rank) {
            float sum = from[r];
            for (int s = 1; s < a.down_splits; ++s) sum += from[s * a.m * ranks + r];
            v[i] = sum * scale;
        }
        top = fmaxf(top, fabsf(v[i]));
    }
    int exponent = 0;
    if constexpr (__is_same(T, f16_t)) {
        for (int d = 1; d < width; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        // none where hi + lo keep 22 bits of the largest without: its place is [2^-3, 2^15)
        exponent = __builtin_amdgcn_frexp_expf(top);
        if (exponent >= -2 && exponent <= 15) exponent = 0;
        if (id >= 0 && lane == 0) a.exponents[row * a.weights + w] = exponent;
    }
    if (id < 0) return;
    uint16_t* const to = a.packed + (row * a.weights + w) * chunks * 32;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int r = lane + i * width;
        if (r >= chunks * kRankTile) break;
        const float x = __builtin_ldexpf(v[i], -exponent);
        const uint16_t head = E::from_float(x);
        const float of_head = E::to_float(head);
        to[r / kRankTile * 32 + r % kRankTile] = head;
        to[r / kRankTile * 32 + 16 + r % kRankTile] = __builtin_isinf(of_head) ? 0 : E::from_float(x - of_head);
    }
}

// s_a B_a t added to the tiled projection's sums. A tile whose rows all name one
// adapter and whose columns are one weight's, as most of a prompt's, has them as more
// stages of its walk over k: of x's side 32 ranks of packed t, of the weights' side the
// same ranks of B_a, each 16 twice. Any other tile adds them to its sums when these
// are done: for each weight of a wave's columns and each adapter of its rows, chunk
// by chunk of 16 ranks, which the tile's last stage cannot hide (4096 rows of q/k/v with rank
// 64: none with an adapter 180 to 209 us, six adapters' rows in runs 237, each row
// another's 269 to 275; the tiles where two runs meet are what the runs wait for).
struct AdapterEpilogue {
    static constexpr bool kAdds = true;
    AdapterArgs p;

    struct Tile {
        int32_t stages = 0;   // of 32 ranks
        int32_t adapter = -1, weight = 0;
        bool sums = false;    // the sums take it
    };

    // What the tile of rows m0 .. and columns n0 .. does, the same in every wave.
    template <typename T, int BM, int BN>
    __device__ inline Tile tile(int split, int m0, int n0, int lane) const {
        Tile t;
        if (split != 0) return t;
        while (t.weight + 1 < p.weights && n0 >= p.end[t.weight]) ++t.weight;
        const bool whole = p.rank % 32 == 0 && min(n0 + BN, p.n) <= p.end[t.weight];
        t.adapter = __builtin_amdgcn_readfirstlane(adapter_of(p, m0));
        bool one = true, any = false;
        for (int32_t r = lane; r < BM && m0 + r < p.m; r += 64) {
            const int32_t id = adapter_of(p, m0 + r);
            one &= id == t.adapter;
            any |= id >= 0;
            if (__is_same(T, f16_t) && whole && id >= 0)  // stages have no place for a power of two
                one &= p.exponents[static_cast<int64_t>(m0 + r) * p.weights + t.weight] == 0;
        }
        any = __any(any);
        if (any && whole && __all(one))
            t.stages = p.rank / 32;
        else
            t.sums = any;
        return t;
    }

    // Base and lane offset of the loads of stage e: 8 columns from `col`, lane row lr, 16-byte piece.
    __device__ inline void weights(const Tile& t, int e, int col, int lr, int piece, int32_t columns, const char*& base,
                                   uint32_t& off) const {
        const int32_t begin = t.weight ? p.end[t.weight - 1] : 0, rows_w = p.end[t.weight] - begin;
        const int32_t c = (col < columns ? col : p.end[t.weight] - kGroupRows) - begin;  // past the last: never written
        base = p.up[t.weight] + ((static_cast<int64_t>(t.adapter) * rows_w + c) * p.rank + 32 * e) * 2;
        off = static_cast<uint32_t>(lr * p.rank * 2 + (piece >> 2) * 32 + (piece & 1) * 16);
    }
    // ... of row m0 + row of x.
    __device__ inline void rows(const Tile& t, int e, int m0, int row, int piece, const char*& base, uint32_t& off) const {
        const int32_t row_bytes = p.weights * (p.rank / kRankTile) * 64;  // whole chunks
        base = reinterpret_cast<const char*>(p.packed) + static_cast<int64_t>(m0) * row_bytes +
               t.weight * (p.rank / kRankTile) * 64 + e * kRowBytes;
        off = static_cast<uint32_t>(min(row, p.m - 1 - m0) * row_bytes + piece * 16);
    }

    template <typename T, int TM, int TN>
    __device__ inline void add(f32x4 (&acc)[TM][TN], int m0, int n0, int lq, int lj) const {
        using G = tile_t<T>;
        using v8 = typename G::v8;
        const int32_t chunks = (p.rank + kRankTile - 1) / kRankTile;
        const u32x4 zero = {0u, 0u, 0u, 0u};
        for (int w = 0; w < p.weights; ++w) {
            const int32_t begin = w ? p.end[w - 1] : 0, end = p.end[w];
            if (end <= n0 || begin >= n0 + 16 * TN) continue;
            const int32_t rows_w = end - begin;
            int32_t id[TM];
            float power[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                id[i] = adapter_of(p, m0 + 16 * i + lq);
                power[i] = 1.f;
                if (__is_same(T, f16_t) && id[i] >= 0)
                    power[i] = __builtin_ldexpf(1.f, p.exponents[static_cast<int64_t>(m0 + 16 * i + lq) * p.weights + w]);
            }
            for (int32_t ad = next_adapter(id); ad >= 0; ad = next_adapter(id)) {
                for (int32_t c = 0; c < chunks; ++c) {
                    const int r = c * kRankTile + 8 * (lj & 1);
                    u32x4 tf[TM], bf[TN];
#pragma unroll
                    for (int j = 0; j < TN; ++j) {
                        const int32_t col = n0 + 16 * j + lq;
                        bf[j] = zero;
                        if (col >= begin && col < end && r < p.rank)
                            bf[j] = *reinterpret_cast<const u32x4*>(
                                p.up[w] + ((static_cast<int64_t>(ad) * rows_w + (col - begin)) * p.rank + r) * 2);
                    }
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
                        tf[i] = zero;
                        if (id[i] == ad)
                            tf[i] = *reinterpret_cast<const u32x4*>(
                                p.packed + ((static_cast<int64_t>(m0 + 16 * i + lq) * p.weights + w) * chunks + c) * 32 + 8 * lj);
                    }
#pragma unroll
                    for (int i = 0; i < TM; ++i) {
                        if (!__any(id[i] == ad)) continue;
#pragma unroll
                        for (int j = 0; j < TN; ++j) {
                            const f32x4 none = {0.f, 0.f, 0.f, 0.f};
                            const f32x4 d = G::mma(__builtin_bit_cast(v8, bf[j]), __builtin_bit_cast(v8, tf[i]), none);
                            // weights end at multiples of 8 columns; what an infinity or NaN of
                            // one weight or adapter makes stays in its own columns and rows
                            const int32_t col = n0 + 16 * j + 4 * lj;
                            if (id[i] == ad && col >= begin && col < end) {
#pragma unroll
                                for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(d[e], power[i], acc[i][j][e]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < TM; ++i)
                    if (id[i] == ad) id[i] = -1;
            }
        }
    }
};

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

constexpr int32_t kFewRows = 64;   // rows of one call of the streaming kernel
// Up to here the tiled projection leaves its sums to adapter_up_kernel, and each 16 rows
// make the inner products of their own adapters: what a step's rows, each request with its
// adapter, take (q/k/v of 4096 with rank 64: 72 rows of 64 adapters 64 instead of 296 us, 256
// rows 152 instead of 310; a run of 4 rows each 103 instead of 141). Rows that share
// an adapter share less: 256 rows of one 68 instead of 44 us, 72 rows 39 instead of 35, of
// rank 16 46 instead of 40 and 28 instead of 32. At 512 rows one adapter costs 100 instead
// of 57, runs of 8 rows 114 instead of 117.
constexpr int32_t kSomeRows = 256;

int64_t total_rows(int32_t n_weights, const int32_t* rows) {
    if (n_weights < 1 || n_weights > 3 || !rows) return KVR_E_INVALID_ARGUMENT;
    int64_t total = 0;
    for (int i = 0; i < n_weights; ++i) {
        if (rows[i] <= 0) return KVR_E_UNSUPPORTED_SHAPE;
        total += rows[i];
    }
    return total > (1 << 24) ? KVR_E_UNSUPPORTED_SHAPE : total;
}

bool takes_tiled(int32_t m, int32_t n_weights, const int32_t* rows, int64_t total, int32_t k) {
    bool ok = m > kFewRows && tiled_linear_ok(m, static_cast<int32_t>(total), k);
    for (int i = 0; i < n_weights; ++i) ok = ok && rows[i] % 8 == 0;
    return ok;
}

struct AdapterPlan {
    bool tiled, some;            // the tiled projection; ... leaving its sums to adapter_up_kernel
    TiledChoice choice;
    int32_t call_rows;           // rows of one pass: all, or the streaming kernel's 64
    int32_t down_splits, turns;
    int64_t base_bytes, inner_bytes, packed_bytes, exponent_bytes;
    int64_t bytes() const { return base_bytes + inner_bytes + packed_bytes + exponent_bytes; }
};

// strides: whether the call's suit the tiled projections.
int plan_adapters(int32_t m, int32_t n_weights, const int32_t* rows, int32_t k, int32_t rank, bool strides,
                  AdapterPlan* p) {
    const int64_t total = total_rows(n_weights, rows);
    if (total < 0) return static_cast<int>(total);
    if (m <= 0 || m > kTiledMaxRows || k <= 0 || k % 8 || k > (1 << 24) || rank <= 0 || rank % 8 || rank > kMaxRank)
        return KVR_E_UNSUPPORTED_SHAPE;
    if (ceil_div(total, 64) * ceil_div(m, 16) > INT32_MAX) return KVR_E_UNSUPPORTED_SHAPE;
    const int64_t tiles = ceil_div(total, kPartialTileCols) * kPartialTileCols * 4;
    p->tiled = strides && takes_tiled(m, n_weights, rows, total, k);
    p->some = p->tiled && m <= kSomeRows;
    p->call_rows = p->tiled || m <= kFewRows ? m : kFewRows;
    p->packed_bytes = p->exponent_bytes = 0;
    if (p->tiled) p->choice = tiled_choice(m, static_cast<int32_t>(total), k);
    if (p->tiled && !p->some) {
        p->base_bytes = p->choice.splits > 1 ? tiles * p->choice.splits * m : 0;
        // slices of k until every CU has a block, 256 k at least
        const int64_t blocks = ceil_div(m, kWideRows) * ceil_div(n_weights * rank, kWideRanks);
        const int32_t steps = k / kStageK;
        int64_t want = ceil_div(256, blocks);
        if (want > kMaxWideSplits) want = kMaxWideSplits;
        if (want > steps / 4) want = steps / 4 > 1 ? steps / 4 : 1;
        p->turns = static_cast<int32_t>(ceil_div(steps, want));
        p->down_splits = static_cast<int32_t>(ceil_div(steps, p->turns));
        p->packed_bytes = static_cast<int64_t>(m) * n_weights * ceil_div(rank, kRankTile) * 64;
        p->exponent_bytes = ceil_div(static_cast<int64_t>(m) * n_weights, 4) * 16;
    } else {
        p->base_bytes = p->some ? tiles * p->choice.splits * m
                                : tiles * kvr_linear_splits(p->call_rows, static_cast<int32_t>(total), k) * kPartialTileRows;
        const int64_t slices = ceil_div(k, kDownSlice);
        p->turns = static_cast<int32_t>(ceil_div(slices, kMaxDownSplits));
        p->down_splits = static_cast<int32_t>(ceil_div(slices, p->turns));
    }
    p->inner_bytes = static_cast<int64_t>(p->down_splits) * p->call_rows * n_weights * rank * 4;
    return KVR_OK;
}

template <typename T>
int launch_up(const AdapterArgs& a, hipStream_t s) {
    const unsigned blocks = static_cast<unsigned>(ceil_div(a.n, 64) * ceil_div(a.m, 16));
    adapter_up_kernel<T><<<blocks, kAdapterThreads, 0, s>>>(a);
    return launch_status();
}

template <typename T>
int launch_few(AdapterArgs a, const void* const* w, const int32_t* rows, const int64_t* ldw, float* base,
               int64_t base_bytes, int32_t dtype, hipStream_t s) {
    const int st = linear_partials_with_down(a, w, rows, ldw, base, base_bytes, dtype, s, &a.splits);
    if (st != KVR_OK) return st;
    a.base_rows = kPartialTileRows;
    return launch_up<T>(a, s);
}

// The partials of W x are in a.base.
template <typename T>
int launch_some(const AdapterArgs& a, hipStream_t s) {
    adapter_down_kernel<T><<<static_cast<unsigned>(adapter_down_blocks(a)), kAdapterThreads, 0, s>>>(a);
    const int st = launch_status();
    return st != KVR_OK ? st : launch_up<T>(a, s);
}

template <typename T, int RT>
int launch_down_wide(const AdapterArgs& a, hipStream_t s) {
    constexpr int lds = kWideStages * wide_stage_bytes<RT>();
    static LdsGrant grant;
    if (!grant.ok(adapter_down_wide_kernel<T, RT>, lds)) return KVR_E_LAUNCH_FAILED;
    const dim3 grid(static_cast<unsigned>(ceil_div(a.m, kWideRows)),
                    static_cast<unsigned>(ceil_div(a.weights * a.rank, 64 * RT)), static_cast<unsigned>(a.down_splits));
    adapter_down_wide_kernel<T, RT><<<grid, kAdapterThreads, lds, s>>>(a);
    return launch_status();
}

template <typename T>
int launch_many(const AdapterArgs& a, const TiledArgs& t, const TiledChoice& choice, hipStream_t s) {
    int st = a.weights * a.rank <= 64 ? launch_down_wide<T, 1>(a, s) : launch_down_wide<T, kWideRanks / 64>(a, s);
    if (st != KVR_OK) return st;
    int32_t width = 16;
    while (width < 64 && width < a.rank) width *= 2;
    const int64_t threads = static_cast<int64_t>(a.m) * a.weights * width;
    adapter_pack_kernel<T><<<static_cast<unsigned>(ceil_div(threads, kAdapterThreads)), kAdapterThreads, 0, s>>>(a, width);
    st = launch_status();
    if (st != KVR_OK) return st;
    return launch_tiled<T>(t, AdapterEpilogue{a}, choice.tile, true, s);
}

}  // namespace
}  // namespace kvr

using namespace kvr;

extern "C" int64_t kvr_adapter_linear_workspace_bytes(int32_t m, int32_t n_weights, const int32_t* rows, int32_t k,
                                                      int32_t rank) {
    // the call's strides are not known here: room for either projection
    AdapterPlan p, q;
    int st = plan_adapters(m, n_weights, rows, k, rank, true, &p);
    if (st != KVR_OK || !p.tiled) return st != KVR_OK ? st : p.bytes();
    st = plan_adapters(m, n_weights, rows, k, rank, false, &q);
    return st != KVR_OK ? st : p.bytes() > q.bytes() ? p.bytes() : q.bytes();
}

extern "C" int kvr_adapter_linear(const void* x, int32_t n_weights, const void* const* w, const int32_t* rows,
                                  const int64_t* ldw, const void* const* down, const void* const* up,
                                  const float* scales, int32_t n_adapters, int32_t rank, const int32_t* ids, void* y,
                                  int32_t m, int32_t k, int64_t ldx, int64_t ldy, void* workspace,
                                  int64_t workspace_bytes, int32_t dtype, void* stream) {
    if (dtype != KVR_DTYPE_BF16 && dtype != KVR_DTYPE_F16) return KVR_E_UNSUPPORTED_DTYPE;
    AdapterPlan p;
    int st = plan_adapters(m, n_weights, rows, k, rank, true, &p);
    if (st != KVR_OK) return st;
    if (n_adapters <= 0) return KVR_E_UNSUPPORTED_SHAPE;
    if (!x || !w || !ldw || !down || !up || !scales || !ids || !y) return KVR_E_NULL_POINTER;
    for (int i = 0; i < n_weights; ++i) {
        if (!w[i] || !down[i] || !up[i]) return KVR_E_NULL_POINTER;
        if (ldw[i] < k || ldw[i] % 8 || !aligned(w[i], 16) || !aligned(down[i], 16) || !aligned(up[i], 16))
            return KVR_E_BAD_STRIDE;
    }
    AdapterArgs a;
    memset(&a, 0, sizeof(a));
    a.n = static_cast<int32_t>(total_rows(n_weights, rows));
    if (ldx < k || ldx % 8 || ldy < a.n || !aligned(x, 16) || !aligned(y, 2)) return KVR_E_BAD_STRIDE;
    if (p.tiled) {
        constexpr int64_t kMaxLd = int64_t(1) << 21;  // a tile's byte offsets fit 32 bits
        bool strides = ldx <= kMaxLd && ldy % 4 == 0 && aligned(y, 8);
        for (int i = 0; i < n_weights; ++i) strides = strides && ldw[i] <= kMaxLd;
        st = strides ? KVR_OK : plan_adapters(m, n_weights, rows, k, rank, false, &p);
        if (st != KVR_OK) return st;
    }
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < p.bytes()) return KVR_E_WORKSPACE_TOO_SMALL;
    char* at = static_cast<char*>(workspace);
    float* const base = reinterpret_cast<float*>(at);
    a.base = base;
    a.inner = reinterpret_cast<float*>(at += p.base_bytes);
    a.packed = reinterpret_cast<uint16_t*>(at += p.inner_bytes);
    a.exponents = reinterpret_cast<int32_t*>(at += p.packed_bytes);
    a.x = static_cast<const char*>(x);
    a.y = static_cast<char*>(y);
    a.m = m;
    a.ids = ids;
    a.scales = scales;
    a.ldx = ldx;
    a.ldy = ldy;
    a.weights = n_weights;
    a.adapters = n_adapters;
    a.rank = rank;
    a.k = k;
    a.down_splits = p.down_splits;
    a.turns = p.turns;
    int32_t column = 0;
    for (int i = 0; i < n_weights; ++i) {
        a.down[i] = static_cast<const char*>(down[i]);
        a.up[i] = static_cast<const char*>(up[i]);
        a.end[i] = column += rows[i];
    }
    hipStream_t s = as_stream(stream);
    if (p.some) {
        st = tiled_partials(x, n_weights, w, rows, ldw, m, k, ldx, base, p.choice, dtype, stream);
        if (st != KVR_OK) return st;
        a.splits = p.choice.splits;
        a.base_rows = m;
        return dtype == KVR_DTYPE_BF16 ? launch_some<bf16_t>(a, s) : launch_some<f16_t>(a, s);
    }
    if (p.tiled) {
        const TiledArgs t = tiled_args(x, n_weights, w, rows, ldw, y, m, k, ldx, ldy, base, p.choice);
        return dtype == KVR_DTYPE_BF16 ? launch_many<bf16_t>(a, t, p.choice, s) : launch_many<f16_t>(a, t, p.choice, s);
    }
    for (int32_t from = 0; from < m; from += p.call_rows) {
        a.m = m - from < p.call_rows ? m - from : p.call_rows;
        a.x = static_cast<const char*>(x) + static_cast<int64_t>(from) * ldx * 2;
        a.y = static_cast<char*>(y) + static_cast<int64_t>(from) * ldy * 2;
        a.ids = ids + from;
        st = dtype == KVR_DTYPE_BF16 ? launch_few<bf16_t>(a, w, rows, ldw, base, p.base_bytes, dtype, s)
                                     : launch_few<f16_t>(a, w, rows, ldw, base, p.base_bytes, dtype, s);
        if (st != KVR_OK) return st;
    }
    return KVR_OK;
}
