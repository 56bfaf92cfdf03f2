// The inner products of few rows with their own adapters (kvr_adapters.hip), which up to
// 64 rows run as more blocks of the streaming projection's launch (kvr_gemm.hip):
// reading W is what that waits for, and these read beside it.
#pragma once

#include "kvr_internal.h"

namespace kvr {

struct AdapterArgs;
// linear_partials of a.x and the adapters' inner products a.inner, one launch.
int linear_partials_with_down(const AdapterArgs& a, const void* const* w, const int32_t* rows, const int64_t* ldw,
                              void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream,
                              int32_t* splits_out);

constexpr int kAdapterWaves = 4;
constexpr int kRankTile = 16;
constexpr int kRankTiles = 4;                        // rank tiles of one block
constexpr int kRankBlock = kRankTile * kRankTiles;
constexpr int kDownSlice = 512;                      // k of a wave's turn: 16 MFMAs
constexpr int kSlotGroups = 16 / kAdapterWaves;      // a tile of 16 rows names at most 16 adapters, one a wave

struct AdapterArgs {
    const char* x;             // [m][ldx]
    const char* down[3];       // [adapters][rank][k]
    const char* up[3];         // [adapters][rows_i][rank]
    const float* scales;       // [adapters]
    const int32_t* ids;        // [m]
    float* inner;              // [down_splits][m][weights * rank] fp32
    const float* base;         // W x: [ceil(rows / 64)][splits][base_rows][64] fp32
    char* y;                   // [m][ldy]
    int64_t ldx, ldy;
    int32_t end[3];            // concatenated row boundaries of the weights
    int32_t weights, adapters, rank;
    int32_t m, k, n;
    int32_t down_splits, turns;  // turns of kDownSlice of a split; adapter_down_wide_kernel: of 64 k
    uint16_t* packed;          // tiles that add to their sums: [m][weights * chunks][16 hi | 16 lo]
    int32_t* exponents;        // ... fp16: [m][weights]
    int32_t splits, base_rows;
};

namespace {

__device__ inline int32_t adapter_of(const AdapterArgs& a, int32_t row) {
    const int32_t id = row < a.m ? a.ids[row] : -1;
    return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.adapters) ? id : -1;
}

// Of the 16 rows of a wave's tile (row lq, repeated over the four lane groups) the
// first ones of each adapter: a bit a row.
__device__ inline uint32_t first_rows(int32_t id, int lq) {
    bool first = id >= 0;
#pragma unroll
    for (int j = 0; j < 15; ++j)
        if (j < lq && __builtin_amdgcn_readlane(id, j) == id) first = false;
    return static_cast<uint32_t>(__ballot(first)) & 0xffffu;
}

// MFMA roles: A = 16 ranks of A_a (lane: rank lq, k 8 lj ..), B = 16 rows of x
// (lane: row lq, k 8 lj ..); D: lane holds t of row lq at ranks 4 lj + i. Block =
// (16 rows, weight, 64 ranks and four of the tile's adapters, slice of k), a wave
// one adapter: all of a slice's loads of a rank tile are in flight at once (one
// adapter after another left each waiting for its own: 23 us for 64 adapters of
// rank 16 over 14336 k, 12 so). G: the MFMA of T. Waves behind the fourth leave.
template <typename T, typename G>
__device__ inline void adapter_down_block(const AdapterArgs& a, int block) {
    using v8 = typename G::v8;
    typedef float f32x4 __attribute__((ext_vector_type(4)));
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (wave >= kAdapterWaves) return;
    const int lq = lane & 15, lj = lane >> 4;
    const int row_tiles = (a.m + 15) / 16, rank_blocks = (a.rank + kRankBlock - 1) / kRankBlock;
    const int row_tile = block % row_tiles;
    block /= row_tiles;
    const int slot = block % kSlotGroups * kAdapterWaves + wave;
    block /= kSlotGroups;
    const int r0 = block % rank_blocks * kRankBlock;
    block /= rank_blocks;
    const int w = block % a.weights, split = block / a.weights;
    const int32_t row = row_tile * 16 + lq;
    const int32_t id = adapter_of(a, row);
    uint32_t firsts = first_rows(id, lq);
    for (int i = 0; i < slot; ++i) firsts &= firsts - 1;
    if (!firsts) return;
    const int32_t ad = __builtin_amdgcn_readlane(id, __builtin_ctz(firsts));
    const char* const base = a.down[w] + static_cast<int64_t>(ad) * a.rank * a.k * 2;
    const char* const xrow = a.x + static_cast<int64_t>(row < a.m ? row : a.m - 1) * a.ldx * 2;
    const int tiles = min(kRankTiles, (a.rank - r0 + kRankTile - 1) / kRankTile);
    const u32x4 zero = {0u, 0u, 0u, 0u};
    f32x4 acc[kRankTiles];
#pragma unroll
    for (int i = 0; i < kRankTiles; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int turn = 0; turn < a.turns; ++turn) {
        const int32_t k0 = (split * a.turns + turn) * kDownSlice + 8 * lj;
        if (k0 - 8 * lj >= a.k) break;
        u32x4 xf[16];
#pragma unroll
        for (int s = 0; s < 16; ++s)  // k is a multiple of 8
            xf[s] = k0 + 32 * s < a.k ? *reinterpret_cast<const u32x4*>(xrow + static_cast<int64_t>(k0 + 32 * s) * 2) : zero;
#pragma unroll
        for (int i = 0; i < kRankTiles; ++i) {
            if (i >= tiles) break;
            const int r = r0 + i * kRankTile + lq;
            const char* const arow = base + (static_cast<int64_t>(min(r, a.rank - 1)) * a.k + k0) * 2;
            u32x4 af[16];
#pragma unroll
            for (int s = 0; s < 16; ++s)
                af[s] = k0 + 32 * s < a.k ? *reinterpret_cast<const u32x4*>(arow + 64 * s) : zero;
#pragma unroll
            for (int s = 0; s < 16; ++s)
                acc[i] = G::mma(__builtin_bit_cast(v8, af[s]), __builtin_bit_cast(v8, xf[s]), acc[i]);
        }
    }
    if (id != ad) return;
    const int64_t inner = static_cast<int64_t>(a.weights) * a.rank;
    float* const to = a.inner + (split * static_cast<int64_t>(a.m) + row) * inner + static_cast<int64_t>(w) * a.rank;
#pragma unroll
    for (int i = 0; i < kRankTiles; ++i) {
        const int r = r0 + i * kRankTile + 4 * lj;
        if (i < tiles && r < a.rank) *reinterpret_cast<f32x4*>(to + r) = acc[i];  // the rank is a multiple of 8
    }
}

inline int64_t adapter_down_blocks(const AdapterArgs& a) {
    return ceil_div(a.m, 16) * kSlotGroups * ceil_div(a.rank, kRankBlock) * a.weights * a.down_splits;
}

}  // namespace
}  // namespace kvr
