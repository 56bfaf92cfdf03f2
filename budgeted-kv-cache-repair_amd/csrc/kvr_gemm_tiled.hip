// Projection GEMMs of more packed refresh rows than the streaming kernel of
// kvr_gemm.hip serves (gfx950 MFMA):
//   y[m, r] = sum_k x[m, k] * w[r, k]      bf16 / fp16, fp32 accumulation
// i.e. the q/k/v/o and MLP projections of the decoder layers (transformers
// 5.15.0 models/llama/modeling_llama.py:165-175, 243-252) for 65 rows up to a
// whole suffix. As in the streaming kernel one launch takes up to three weights
// (rows concatenated) or a gate/up pair with the SiLU-gated product in its
// epilogue, a residual can be added, and K can be split, the fp32 partials
// being summed by the consumer (fresh-row epilogue, residual + RMSNorm) or by
// tiled_reduce_kernel. Kernels and tiles are in kvr_gemm_tiled.h.
//
// What bounds it: reading the weights below ~200 rows (0.44 GB per layer of an
// 8B model), the matrix cores above. So the block tile follows the row count:
// every weight byte is read from HBM by as few blocks as LDS allows (the tile
// covers all rows up to 288), and the tile and the K split are chosen together
// so that the grid fills the 256 CUs in whole rounds (choose()).
//
// A stage of 64 k (128-byte rows, whole cache lines) of both operands goes
// straight from global memory to LDS (global_load_lds_dwordx4, no registers),
// 2 to 4 stages deep; LDS is full, so a CU runs one block (two of the smallest
// tile). Fragments of the next 32 k are read while the current ones are
// multiplied; at the turn of a stage every wave holds its last fragments, so
// after the barrier the stage's buffer is refilled at once, its loads and the
// next reads issued one by one between the MFMAs (in a burst before them
// 256 x 256 ran 5% slower; spread over the whole half step the last loads came
// too late, 3-5%: three quarters is best). 16-byte pieces are swizzled by row
// (SQ_LDS_BANK_CONFLICT counts none).
//
// Measured in the refreshes (us for the four projections of one 8B layer, from their
// kernel traces): 71 rows 100, 141 rows (fp16) 123, 282 rows 182, 1383 rows (Qwen3
// shape) 537, 15104 rows 5120 = 1.29 PFLOP/s; hipBLASLt's separate q, k, v, o, gate,
// up, down, SiLU and residual launches, timed alone, took 210, 230, 270 and 560 for
// the first four. Gate/up at 71 rows 44.6 us = 5.3 TB/s of weights, at 15104 rows
// 1.31 PFLOP/s: the matrix cores are busy 69% of the cycles of an engine clock that
// falls to 1.7 GHz; the rest are the turns of the stages and their LDS reads.
#include "kvr_gemm_tiled.h"

namespace kvr {
namespace {

using Choice = TiledChoice;

// The tile and K split with the least modelled time, of a model fitted to 260
// measured projections (q/k/v, o, gate/up, down of 8B shapes, 65 to 8192 rows;
// the choice is 0.7% slower than the fastest tile on average, 19% at most):
// blocks run in rounds of 32 CUs per XCD, a round costs its stages plus 2.1 us
// (2.3 us more for the gated epilogue); against it stands the weight stream,
// 5.9 TB/s with every CU loading, 7.0 nontemporal; both overlap as a 2-norm.
// Split partials cost 0.16 us/MB to write and 0.2 in their consumer. The
// smallest tile has no place beside other x tiles: two of its blocks share a CU.
Choice model_choice(int32_t m, int32_t rows, int32_t k, bool gated) {
    const int32_t steps = k / kStageK;
    Choice best{0, 1, steps};
    double least = 1e30;
    for (int t = 0; t < kTileCount; ++t) {
        const Tile& tile = kTiles[t];
        const int64_t tiles_m = ceil_div(m, tile.bm);
        if (smallest_tile(tile.bm, tile.bn) && tiles_m > 1) continue;
        const int64_t tiles = tiles_m * ceil_div(rows, tile.bn);
        const bool once = tiles_m == 1 && tile.bm <= kStreamRows;
        for (int32_t want = 1; want <= kMaxSplits; want *= 2) {
            if (want > 1 && (gated || steps / want < kMinSplitSteps)) break;
            const int32_t split_steps = static_cast<int32_t>(ceil_div(steps, want));
            const int32_t splits = static_cast<int32_t>(ceil_div(steps, split_steps));
            const int64_t blocks = tiles * splits;
            const int64_t rounds = ceil_div(ceil_div(blocks, kXcds), kCusPerXcd);
            const double work = rounds * (split_steps * static_cast<double>(tile.step_us) + (gated ? 4.4 : 2.1));
            const double busy = blocks < 256 ? static_cast<double>(blocks) / 256 : 1.0;
            const double stream = static_cast<double>(rows) * k * 2 / (once ? 7.0e6 : 5.9e6) / sqrt(busy);
            double us = sqrt(work * work + stream * stream);
            if (splits > 1) us += static_cast<double>(m) * rows * 4 * splits * 0.36e-6;
            if (us < least) {
                least = us;
                best = Choice{t, splits, split_steps};
            }
            if (blocks >= 1024) break;  // more splits only add partials
        }
    }
    return best;
}

// model_choice (~1 us of host time), remembered per thread for the few
// projections that a forward runs layer after layer.
Choice choose(int32_t m, int32_t rows, int32_t k, bool gated) {
    struct Entry {
        int32_t m, rows, k, gated;
        Choice choice;
    };
    constexpr int kEntries = 8;
    static thread_local Entry memo[kEntries] = {};
    static thread_local int next = 0;
    for (const Entry& e : memo)
        if (e.m == m && e.rows == rows && e.k == k && e.gated == (gated ? 1 : 0)) return e.choice;
    const Choice c = model_choice(m, rows, k, gated);
    memo[next] = Entry{m, rows, k, gated ? 1 : 0, c};
    next = (next + 1) % kEntries;
    return c;
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Rows of the weights of one call in total, or a negative status.
int64_t total_rows(int32_t n_weights, const int32_t* rows, bool gated) {
    if (n_weights < 1 || n_weights > 3 || !rows) return KVR_E_INVALID_ARGUMENT;
    if (gated && (n_weights != 2 || rows[0] != rows[1])) return KVR_E_UNSUPPORTED_SHAPE;
    int64_t total = 0;
    for (int i = 0; i < n_weights; ++i) {
        if (rows[i] <= 0 || rows[i] % kGroupRows) return KVR_E_UNSUPPORTED_SHAPE;
        total += rows[i];
    }
    return total > (1 << 24) ? KVR_E_UNSUPPORTED_SHAPE : total;
}

}  // namespace

bool tiled_linear_ok(int32_t m, int32_t rows, int32_t k) {
    return m > 0 && m <= kTiledMaxRows && rows > 0 && rows % kGroupRows == 0 && rows <= (1 << 24) && k > 0 &&
           k % kStageK == 0 && k <= (1 << 24);
}

int64_t tiled_workspace_bytes(int32_t m, int32_t rows, int32_t k) {
    if (!tiled_linear_ok(m, rows, k)) return KVR_E_UNSUPPORTED_SHAPE;
    const Choice c = choose(m, rows, k, false);
    return c.splits == 1 ? 0 : ceil_div(rows, kPartialTileCols) * kPartialTileCols * c.splits * m * 4;
}

TiledChoice tiled_choice(int32_t m, int32_t rows, int32_t k) { return choose(m, rows, k, false); }

int tiled_partials(const void* x, int32_t n_weights, const void* const* w, const int32_t* rows, const int64_t* ldw,
                   int32_t m, int32_t k, int64_t ldx, float* partial, const TiledChoice& c, int32_t dtype,
                   void* stream) {
    TiledArgs a = tiled_args(x, n_weights, w, rows, ldw, nullptr, m, k, ldx, 0, partial, c);
    a.keep = 1;
    hipStream_t s = as_stream(stream);
    return dtype == KVR_DTYPE_BF16 ? launch_tiled<bf16_t>(a, NoEpilogue{}, c.tile, false, s)
                                   : launch_tiled<f16_t>(a, NoEpilogue{}, c.tile, false, s);
}

int tiled_linear(const void* x, int32_t n_weights, const void* const* w, const int32_t* rows, const int64_t* ldw,
                 void* y, int32_t m, int32_t k, int64_t ldx, int64_t ldy, int32_t epilogue, const void* residual,
                 int64_t ldr, void* workspace, int64_t workspace_bytes, int32_t dtype, void* stream, bool reduce,
                 int32_t* splits_out) {
    if (dtype != KVR_DTYPE_BF16 && dtype != KVR_DTYPE_F16) return KVR_E_UNSUPPORTED_DTYPE;
    if (epilogue != KVR_LINEAR_CONCAT && epilogue != KVR_LINEAR_SILU_GATE && epilogue != KVR_LINEAR_RESIDUAL)
        return KVR_E_INVALID_ARGUMENT;
    const bool gated = epilogue == KVR_LINEAR_SILU_GATE;
    const int64_t total = total_rows(n_weights, rows, gated);
    if (total < 0) return static_cast<int>(total);
    if (!tiled_linear_ok(m, static_cast<int32_t>(total), k)) return KVR_E_UNSUPPORTED_SHAPE;
    if (!w || !ldw) return KVR_E_INVALID_ARGUMENT;
    const int64_t n_out = gated ? rows[0] : total;
    constexpr int64_t kMaxLd = int64_t(1) << 21;  // a tile's byte offsets fit 32 bits
    if (ldx < k || ldx % 8 || ldx > kMaxLd || ldy < n_out || ldy % 4) return KVR_E_BAD_STRIDE;
    for (int i = 0; i < n_weights; ++i)
        if (ldw[i] < k || ldw[i] % 8 || ldw[i] > kMaxLd) return KVR_E_BAD_STRIDE;
    if (epilogue == KVR_LINEAR_RESIDUAL) {
        if (!residual) return KVR_E_NULL_POINTER;
        if (ldr < n_out || ldr % 4 || !aligned(residual, 8)) return KVR_E_BAD_STRIDE;
        if (!reduce) return KVR_E_INVALID_ARGUMENT;  // partial consumers take plain sums
    }
    if (!x || !y) return KVR_E_NULL_POINTER;
    if (!aligned(x, 16) || !aligned(y, 8)) return KVR_E_BAD_STRIDE;
    for (int i = 0; i < n_weights; ++i) {
        if (!w[i]) return KVR_E_NULL_POINTER;
        if (!aligned(w[i], 16)) return KVR_E_BAD_STRIDE;
    }
    const Choice c = choose(m, static_cast<int32_t>(total), k, gated);
    if (c.splits > 1 && (!workspace || !aligned(workspace, 16) ||
                         workspace_bytes < tiled_workspace_bytes(m, static_cast<int32_t>(total), k)))
        return KVR_E_WORKSPACE_TOO_SMALL;
    TiledArgs a = tiled_args(x, n_weights, w, rows, ldw, y, m, k, ldx, ldy, workspace, c);
    a.gated = gated ? 1 : 0;
    a.res = epilogue == KVR_LINEAR_RESIDUAL ? static_cast<const char*>(residual) : nullptr;
    a.ldr = ldr;
    if (splits_out) *splits_out = c.splits;
    hipStream_t s = as_stream(stream);
    return dtype == KVR_DTYPE_BF16 ? launch_tiled<bf16_t>(a, NoEpilogue{}, c.tile, reduce, s)
                                   : launch_tiled<f16_t>(a, NoEpilogue{}, c.tile, reduce, s);
}

}  // namespace kvr

using namespace kvr;

extern "C" int kvr_internal_tiled_choice(int32_t m, int32_t rows, int32_t k, int32_t gated, int32_t out[4]) {
    if (!out || !tiled_linear_ok(m, rows, k)) return KVR_E_UNSUPPORTED_SHAPE;
    const Choice c = model_choice(m, rows, k, gated != 0);
    out[0] = kTiles[c.tile].bm;
    out[1] = kTiles[c.tile].bn;
    out[2] = m <= kTiles[c.tile].bm && kTiles[c.tile].bm <= kStreamRows;
    out[3] = c.splits;
    return KVR_OK;
}

extern "C" int64_t kvr_tiled_linear_workspace_bytes(int32_t m, int32_t rows, int32_t k) {
    return tiled_workspace_bytes(m, rows, k);
}

extern "C" int kvr_tiled_linear_multi(const void* x, int32_t n_weights, const void* const* w, const int32_t* rows,
                                      const int64_t* ldw, void* y, int32_t m, int32_t k, int64_t ldx, int64_t ldy,
                                      int32_t epilogue, const void* residual, int64_t ldr, void* workspace,
                                      int64_t workspace_bytes, int32_t dtype, void* stream) {
    return tiled_linear(x, n_weights, w, rows, ldw, y, m, k, ldx, ldy, epilogue, residual, ldr, workspace,
                        workspace_bytes, dtype, stream, true, nullptr);
}
