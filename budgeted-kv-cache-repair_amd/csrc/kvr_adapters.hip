// Projections with a low-rank adapter of each row's own beside the shared weights:
//   y[m, :] = W x_m + s_a B_a (A_a x_m)        a = ids[m]; W x_m alone where ids[m] names no adapter
// W: up to three weights, rows concatenated (q/k/v), each with its own A and B.
//
// What bounds it: up to some 200 rows reading W and, once each, the A_a and B_a of
// the adapters that the rows name; above that the matrix cores on W x. So W x runs
// on the projection kernels (kvr_gemm.hip, kvr_gemm_tiled.hip), which leave their
// fp32 sums, and the adapters' two thin products go through the MFMA in tiles of
// 16 rows: a tile walks the distinct adapters that its rows name, so that rows of
// one adapter share its reads, and keeps of each product the columns of its rows.
//
//   adapter_down_kernel   t = A_a x: fp32 partials, one a slice of k
//   adapter_up_kernel     y = sum of W x's partials + s_a B_a t, rounded once
//
// t enters the second product as a hi + lo pair of 16-bit values side by side in
// one MFMA (16 ranks of hi, the same 16 of lo), so it is not rounded to the input
// type. No sum depends on the order in which blocks end.
#include "kvr_internal.h"
#include "kvrepair_step.h"

#include <string.h>

namespace kvr {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct adapter_t;
template <> struct adapter_t<bf16_t> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    __device__ static inline f32x4 mma(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
template <> struct adapter_t<f16_t> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    __device__ static inline f32x4 mma(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};

constexpr int kAdapterWaves = 4;
constexpr int kAdapterThreads = 64 * kAdapterWaves;
constexpr int kRankTile = 16;
constexpr int kRankTiles = 4;                        // rank tiles of one block
constexpr int kRankBlock = kRankTile * kRankTiles;
constexpr int kMaxRank = 512;
constexpr int kDownStep = 128;                       // k of a wave's turn: four MFMAs
constexpr int kDownTurn = kDownStep * kAdapterWaves; // ... of a block's

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
    int32_t down_splits, turns;  // turns of kDownTurn of a split
    int32_t splits, base_rows;
};

// The next adapter that some of the wave's rows still wait for, or -1. `id`: of
// this lane's row, -1 once done; rows repeat over the four lane groups.
__device__ inline int32_t next_adapter(int32_t id) {
    const uint64_t waiting = __ballot(id >= 0);
    if (!waiting) return -1;
    return __builtin_amdgcn_readlane(id, __builtin_ctzll(waiting));
}

__device__ inline int32_t adapter_of(const AdapterArgs& a, int32_t row) {
    const int32_t id = row < a.m ? a.ids[row] : -1;
    return static_cast<uint32_t>(id) < static_cast<uint32_t>(a.adapters) ? id : -1;
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

// MFMA roles: A = 16 ranks of A_a (lane: rank lq, k 8 lj ..), B = 16 rows of x
// (lane: row lq, k 8 lj ..); D: lane holds t of row lq at ranks 4 lj + i. Block =
// (16 rows, weight and 64 ranks, slice of k); its waves take 128 k in turn.
template <typename T>
__global__ void __launch_bounds__(kAdapterThreads) adapter_down_kernel(AdapterArgs a) {
    using G = adapter_t<T>;
    using v8 = typename G::v8;
    __shared__ f32x4 sums[kAdapterWaves][kRankTiles][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lq = lane & 15, lj = lane >> 4;
    const int rank_blocks = (a.rank + kRankBlock - 1) / kRankBlock;
    const int w = blockIdx.y / rank_blocks, r0 = blockIdx.y % rank_blocks * kRankBlock;
    const int32_t row = blockIdx.x * 16 + lq;
    const int32_t mine = adapter_of(a, row);
    if (!__any(mine >= 0)) return;  // the waves have the same rows: all leave
    const int tiles = min(kRankTiles, (a.rank - r0 + kRankTile - 1) / kRankTile);
    const int32_t k0 = blockIdx.z * a.turns * kDownTurn;
    const char* xrow = a.x + static_cast<int64_t>(row < a.m ? row : a.m - 1) * a.ldx * 2;
    f32x4 t[kRankTiles];
#pragma unroll
    for (int i = 0; i < kRankTiles; ++i) t[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    int32_t id = mine;
    for (int32_t ad = next_adapter(id); ad >= 0; ad = next_adapter(id)) {
        const char* base = a.down[w] + static_cast<int64_t>(ad) * a.rank * a.k * 2;
        f32x4 acc[kRankTiles];
#pragma unroll
        for (int i = 0; i < kRankTiles; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int turn = 0; turn < a.turns; ++turn) {
            const int32_t kw = k0 + turn * kDownTurn + wave * kDownStep;
            if (kw >= a.k) break;
            u32x4 xf[4], af[kRankTiles][4];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int32_t kk = kw + 32 * s + 8 * lj;
                const bool in = kk < a.k;  // k is a multiple of 8
                const u32x4 zero = {0u, 0u, 0u, 0u};
                xf[s] = in ? *reinterpret_cast<const u32x4*>(xrow + static_cast<int64_t>(kk) * 2) : zero;
#pragma unroll
                for (int i = 0; i < kRankTiles; ++i) {
                    const int r = r0 + i * kRankTile + lq;
                    af[i][s] = zero;
                    if (in && r < a.rank)
                        af[i][s] = *reinterpret_cast<const u32x4*>(base + (static_cast<int64_t>(r) * a.k + kk) * 2);
                }
            }
#pragma unroll
            for (int i = 0; i < kRankTiles; ++i)
                if (i < tiles)
#pragma unroll
                    for (int s = 0; s < 4; ++s)
                        acc[i] = G::mma(__builtin_bit_cast(v8, af[i][s]), __builtin_bit_cast(v8, xf[s]), acc[i]);
        }
        const bool its = id == ad;
#pragma unroll
        for (int i = 0; i < kRankTiles; ++i) t[i] = its ? acc[i] : t[i];
        if (its) id = -1;
    }
#pragma unroll
    for (int i = 0; i < kRankTiles; ++i) sums[wave][i][lane] = t[i];
    __syncthreads();
    if (wave >= tiles || mine < 0) return;
    f32x4 sum = sums[0][wave][lane];
#pragma unroll
    for (int o = 1; o < kAdapterWaves; ++o) sum += sums[o][wave][lane];
    const int r = r0 + wave * kRankTile + 4 * lj;
    const int64_t inner = static_cast<int64_t>(a.weights) * a.rank;
    if (r < a.rank)  // the rank is a multiple of 8
        *reinterpret_cast<f32x4*>(a.inner + (blockIdx.z * static_cast<int64_t>(a.m) + row) * inner +
                                  static_cast<int64_t>(w) * a.rank + r) = sum;
}

// Block = (64 columns, 16 rows), a wave 16 columns: the sum of W x's partials in
// split order, then the distinct adapters of the rows. MFMA roles: A = 16 rows
// of B_a (columns of y), 16 ranks twice; B = [hi | lo] of 16 ranks of t.
template <typename T>
__global__ void __launch_bounds__(kAdapterThreads) adapter_up_kernel(AdapterArgs a) {
    using G = adapter_t<T>;
    using E = elem<T>;
    using v8 = typename G::v8;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lq = lane & 15, lj = lane >> 4;
    const int32_t columns = (a.n + 63) / 64;
    const int32_t tile = blockIdx.x % columns;
    const int32_t n0 = tile * 64 + wave * 16;
    if (n0 >= a.n) return;
    const int32_t row = blockIdx.x / columns * 16 + lq;
    const int32_t row_in = row < a.m ? row : a.m - 1;
    const float* at = a.base + (static_cast<int64_t>(tile) * a.splits * a.base_rows + row_in) * 64 + wave * 16 + 4 * lj;
    const int64_t step = static_cast<int64_t>(a.base_rows) * 64;
    f32x4 acc = *reinterpret_cast<const f32x4*>(at);
    for (int s = 1; s < a.splits; ++s) acc += *reinterpret_cast<const f32x4*>(at + s * step);
    const int32_t mine = adapter_of(a, row);
    if (__any(mine >= 0)) {
        const float scale = mine >= 0 ? a.scales[mine] : 0.f;
        const int64_t inner = static_cast<int64_t>(a.weights) * a.rank;
        const int32_t col = n0 + lq;
        const int half = lj & 1;  // ranks 8 half .. of a chunk of 16; lanes of lj >= 2 hold lo
        for (int w = 0; w < a.weights; ++w) {
            const int32_t begin = w ? a.end[w - 1] : 0, end = a.end[w];
            if (end <= n0 || begin >= min(n0 + 16, a.n)) continue;
            const bool col_in = col >= begin && col < end;
            const int32_t rows_w = end - begin;
            for (int r0 = 0; r0 < a.rank; r0 += kRankTile) {
                const int r = r0 + 8 * half;
                float t[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                if (mine >= 0 && r < a.rank) {
                    const float* from = a.inner + static_cast<int64_t>(row) * inner + static_cast<int64_t>(w) * a.rank + r;
                    f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
                    for (int s = 0; s < a.down_splits; ++s) {
                        lo += *reinterpret_cast<const f32x4*>(from + s * a.m * inner);
                        hi += *reinterpret_cast<const f32x4*>(from + s * a.m * inner + 4);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) t[e] = (e < 4 ? lo[e] : hi[e - 4]) * scale;
                }
                const int exponent = adapter_exponent<T>(t);
                const u32x4 tf = hi_or_lo<T>(t, exponent, lj >= 2);
                f32x4 found = {0.f, 0.f, 0.f, 0.f};
                int32_t id = mine;
                for (int32_t ad = next_adapter(id); ad >= 0; ad = next_adapter(id)) {
                    u32x4 bf = {0u, 0u, 0u, 0u};
                    if (col_in && r < a.rank)
                        bf = *reinterpret_cast<const u32x4*>(
                            a.up[w] + ((static_cast<int64_t>(ad) * rows_w + (col - begin)) * a.rank + r) * 2);
                    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
                    const f32x4 d = G::mma(__builtin_bit_cast(v8, bf), __builtin_bit_cast(v8, tf), zero);
                    const bool its = id == ad;
                    found = its ? d : found;
                    if (its) id = -1;
                }
                // what an infinity or NaN of one weight or adapter makes of a product stays
                // in its own columns and rows
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int32_t c = n0 + 4 * lj + i;
                    if (mine >= 0 && c >= begin && c < end) acc[i] += __builtin_ldexpf(found[i], exponent);
                }
            }
        }
    }
    if (row >= a.m) return;
    uint16_t* y = reinterpret_cast<uint16_t*>(a.y) + static_cast<int64_t>(row) * a.ldy + n0 + 4 * lj;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (n0 + 4 * lj + i < a.n) y[i] = E::from_float(acc[i]);
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

constexpr int32_t kStreamRows = 64;  // rows of one call of the streaming kernel

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
    bool ok = m > kStreamRows && tiled_linear_ok(m, static_cast<int32_t>(total), k);
    for (int i = 0; i < n_weights; ++i) ok = ok && rows[i] % 8 == 0;
    return ok;
}

struct AdapterPlan {
    bool tiled;
    int32_t call_rows;           // rows of one pass: all, or the streaming kernel's 64
    int32_t down_splits, turns;
    int64_t base_bytes, inner_bytes;
};

int plan_adapters(int32_t m, int32_t n_weights, const int32_t* rows, int32_t k, int32_t rank, AdapterPlan* p) {
    const int64_t total = total_rows(n_weights, rows);
    if (total < 0) return static_cast<int>(total);
    if (m <= 0 || m > kTiledMaxRows || k <= 0 || k % 8 || k > (1 << 24) || rank <= 0 || rank % 8 || rank > kMaxRank)
        return KVR_E_UNSUPPORTED_SHAPE;
    if (ceil_div(total, 64) * ceil_div(m, 16) > INT32_MAX) return KVR_E_UNSUPPORTED_SHAPE;
    p->tiled = takes_tiled(m, n_weights, rows, total, k);
    p->call_rows = p->tiled || m <= kStreamRows ? m : kStreamRows;
    const int64_t tiles = ceil_div(total, kPartialTileCols) * kPartialTileCols * 4;
    if (p->tiled)
        p->base_bytes = tiles * tiled_splits(m, static_cast<int32_t>(total), k) * m;
    else
        p->base_bytes = tiles * kvr_linear_splits(p->call_rows, static_cast<int32_t>(total), k) * kPartialTileRows;
    // slices of k until some four blocks a CU, one turn at least
    const int32_t all = static_cast<int32_t>(ceil_div(k, kDownTurn));
    const int64_t blocks = ceil_div(p->call_rows, 16) * n_weights * ceil_div(rank, kRankBlock);
    const int32_t want = static_cast<int32_t>(ceil_div(1024, blocks));
    p->turns = static_cast<int32_t>(ceil_div(all, want < all ? want : all));
    p->down_splits = static_cast<int32_t>(ceil_div(all, p->turns));
    p->inner_bytes = static_cast<int64_t>(p->down_splits) * p->call_rows * n_weights * rank * 4;
    return KVR_OK;
}

template <typename T>
int launch_down(const AdapterArgs& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(ceil_div(a.m, 16)),
                    static_cast<unsigned>(a.weights * ceil_div(a.rank, kRankBlock)), static_cast<unsigned>(a.down_splits));
    adapter_down_kernel<T><<<grid, kAdapterThreads, 0, s>>>(a);
    return launch_status();
}

template <typename T>
int launch_up(const AdapterArgs& a, hipStream_t s) {
    const unsigned blocks = static_cast<unsigned>(ceil_div(a.n, 64) * ceil_div(a.m, 16));
    adapter_up_kernel<T><<<blocks, kAdapterThreads, 0, s>>>(a);
    return launch_status();
}

}  // namespace
}  // namespace kvr

using namespace kvr;

extern "C" int64_t kvr_adapter_linear_workspace_bytes(int32_t m, int32_t n_weights, const int32_t* rows, int32_t k,
                                                      int32_t rank) {
    AdapterPlan p;
    const int st = plan_adapters(m, n_weights, rows, k, rank, &p);
    return st != KVR_OK ? st : p.base_bytes + p.inner_bytes;
}

extern "C" int kvr_adapter_linear(const void* x, int32_t n_weights, const void* const* w, const int32_t* rows,
                                  const int64_t* ldw, const void* const* down, const void* const* up,
                                  const float* scales, int32_t n_adapters, int32_t rank, const int32_t* ids, void* y,
                                  int32_t m, int32_t k, int64_t ldx, int64_t ldy, void* workspace,
                                  int64_t workspace_bytes, int32_t dtype, void* stream) {
    if (dtype != KVR_DTYPE_BF16 && dtype != KVR_DTYPE_F16) return KVR_E_UNSUPPORTED_DTYPE;
    AdapterPlan p;
    int st = plan_adapters(m, n_weights, rows, k, rank, &p);
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
    if (!workspace || !aligned(workspace, 16) || workspace_bytes < p.base_bytes + p.inner_bytes)
        return KVR_E_WORKSPACE_TOO_SMALL;
    float* base = static_cast<float*>(workspace);
    a.inner = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.base_bytes);
    a.base = base;
    a.scales = scales;
    a.ldx = ldx;
    a.ldy = ldy;
    a.weights = n_weights;
    a.adapters = n_adapters;
    a.rank = rank;
    a.k = k;
    a.down_splits = p.down_splits;
    a.turns = p.turns;
    int32_t at = 0;
    for (int i = 0; i < n_weights; ++i) {
        a.down[i] = static_cast<const char*>(down[i]);
        a.up[i] = static_cast<const char*>(up[i]);
        a.end[i] = at += rows[i];
    }
    hipStream_t s = as_stream(stream);
    for (int32_t from = 0; from < m; from += p.call_rows) {
        a.m = m - from < p.call_rows ? m - from : p.call_rows;
        a.x = static_cast<const char*>(x) + static_cast<int64_t>(from) * ldx * 2;
        a.y = static_cast<char*>(y) + static_cast<int64_t>(from) * ldy * 2;
        a.ids = ids + from;
        st = dtype == KVR_DTYPE_BF16 ? launch_down<bf16_t>(a, s) : launch_down<f16_t>(a, s);
        if (st != KVR_OK) return st;
        st = (p.tiled ? tiled_partials : linear_partials)(a.x, n_weights, w, rows, ldw, a.m, k, ldx, base, p.base_bytes,
                                                          dtype, stream, &a.splits);
        a.base_rows = p.tiled ? a.m : kPartialTileRows;
        if (st != KVR_OK) return st;
        st = dtype == KVR_DTYPE_BF16 ? launch_up<bf16_t>(a, s) : launch_up<f16_t>(a, s);
        if (st != KVR_OK) return st;
    }
    return KVR_OK;
}
