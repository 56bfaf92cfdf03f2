// Verification of drafted tokens against the target's probabilities, and the
// answer drawn from what is left after the last token that holds.
//
// Node t of a request hangs on node a (the highest set bit of its mask below t).
// It is taken
//   drafts as they are:          sum_{s<t} p_a(x_s) <= u_a < sum_{s<=t} p_a(x_s)   (s: its siblings, in order)
//   drawn from a draft's q_a:    u_a q_a(x_t) < p_a(x_t)
// and kept when all of its ancestors are, which its mask tells: the nodes of the mask
// are all taken. With w_i = p_a(i) without the tokens that hang on the last kept
// a, max(p_a(i) - q_a(i), 0), or p_a(i), the answer is the first i with
// sum_{j<=i} w_j > draw * sum_j w_j.
//
// Products of two fp32 values are exact in fp64, and the sums' own order moves no
// decision by more than 2^-50 of the whole: all of it is fp64, which costs no time
// beside the reads.
//
// What bounds it: for few requests and short rows a chain of some ten dependent reads, for many the
// read of one row of p (and q) each. Lane t of a wave is node t of a request and the walk is
// ballots and masks; then waves sum parts of 1024 tokens of what is left, every lane 16 values with
// all its loads in flight; a wave finds the part that holds the draw among the parts' sums (a lane
// adds up neighbouring ones, a sum over the wave, and the lane that passes the target walks its
// own), reads that part again and finds the token likewise. Rows of more than 2^20 tokens have
// longer parts, which are cut in sixteen until 1024 are left. Short rows: one block of 16 waves a
// request, one launch (8 trees of 32003 tokens 13.3 us in a graph). Long rows: several blocks, each
// of which walks by itself, then one that draws (64 chains of 128256 tokens with draft
// probabilities: sums 13.8 us, 66 MB read, 4.8 TB/s; draw 6.0).
#include "kvr_internal.h"
#include "kvr_step.h"
#include "kvrepair_serve.h"

#include <math.h>

namespace kvr {
namespace {

constexpr int kVerifyThreads = 1024;
constexpr int kVerifyWaves = kVerifyThreads / 64;
constexpr int kVerifyBlocks = 16;  // most of a request
constexpr int32_t kPartTokens = 1024;  // of a part that a wave walks
constexpr int32_t kParts = 1024;       // most of a row

constexpr int32_t kVerifyVocab = int32_t(1) << 30;  // what lies behind the last part fits 32 bits

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // rows start on any fp32 address

struct VerifyArgs {
    const float* p;
    const float* q;  // null: drafts as they are
    int64_t ld, ldd;
    const int64_t* tokens;
    const float* uniforms;
    const float* draws;
    const int32_t* row_starts;
    const uint64_t* masks;
    int32_t* kept;
    int32_t* path;
    int64_t* answers;
    struct Walked* walked;  // of a request; with several blocks
    double* sums;           // ... and the sums of its row's parts
    int32_t vocab;
    int32_t rows;
    int32_t requests;
    int32_t blocks;
    int32_t parts, part;    // parts of a row, and their tokens
};

// What counts of an entry, and of the difference of two: what is positive and finite. An entry of q is never looked at
// by itself: a negative one adds to the difference, with an infinite or NaN one nothing of it counts.
__device__ inline double weight(float p) { return p < INFINITY ? fmaxf(p, 0.f) : 0.f; }
__device__ inline double weight(float p, float q) {
    const double left = fmax(static_cast<double>(p) - static_cast<double>(q), 0.0);
    return fabsf(p) < INFINITY && fabsf(q) < INFINITY ? left : 0.0;
}

enum VerifyMode { kWhole = 0, kWithout = 1, kMinus = 2 };

// What is left of a row. A lane holds one of the tokens that do not count (kWithout), -1 for none.
struct Left {
    const float* p;
    const float* q;
    int32_t hangs;
    int32_t vocab;
    int mode;

    // The tokens in [begin, end) that do not count, one after another, the same in all lanes.
    template <typename F>
    __device__ inline void each_out(int32_t begin, int32_t end, F f) const {
        if (mode != kWithout) return;
        uint64_t some = __ballot(hangs >= begin && hangs < end);
        while (some) {
            f(__builtin_amdgcn_readlane(hangs, __builtin_ctzll(some)));
            some &= some - 1;
        }
    }

    template <bool MINUS>
    __device__ inline double sum_of(int32_t begin, int32_t end, int lane) const {
        constexpr int kAhead = kPartTokens / 256;  // 16-byte loads in flight, of either row
        double s = 0.0;
        for (; begin < end; begin += 256 * kAhead) {
            f32x4u a[kAhead], b[kAhead];
            const int32_t i = begin + 4 * lane;
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                a[e] = b[e] = f32x4u{0.f, 0.f, 0.f, 0.f};
                const int32_t j = i + 256 * e;
                if (j + 4 <= end) {
                    a[e] = *reinterpret_cast<const f32x4u*>(p + j);
                    if (MINUS) b[e] = *reinterpret_cast<const f32x4u*>(q + j);
                } else if (j < end) {
#pragma unroll
                    for (int k = 0; k < 3; ++k)
                        if (j + k < end) {
                            a[e][k] = p[j + k];
                            if (MINUS) b[e][k] = q[j + k];
                        }
                }
            }
            each_out(begin, min(begin + 256 * kAhead, end), [&](int32_t token) {
#pragma unroll
                for (int e = 0; e < kAhead; ++e)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (i + 256 * e + k == token) a[e][k] = 0.f;
            });
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                if (begin + 256 * e >= end) break;  // the same for all lanes
#pragma unroll
                for (int k = 0; k < 4; ++k) s += MINUS ? weight(a[e][k], b[e][k]) : weight(a[e][k]);
            }
        }
#pragma unroll
        for (int d = 32; d > 0; d /= 2) s += __shfl_xor(s, d);
        return s;
    }
    // The sum over [begin, end), at most the vocabulary's, by a wave: the same in every lane.
    __device__ inline double sum(int32_t begin, int32_t end, int lane) const {
        return mode == kMinus ? sum_of<true>(begin, end, lane) : sum_of<false>(begin, end, lane);
    }
};

// Exclusive sums over the wave of one value a lane; returns the total too.
__device__ inline double wave_exclusive(double x, int lane, double& total) {
    double sum = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const double up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    total = __shfl(sum, 63);
    const double before = __shfl_up(sum, 1);
    return lane > 0 ? before : 0.0;
}

// The first lane with something in it at which the running sum exceeds `target`, or else the last with something in it
// (63 where there is none).
__device__ inline int first_over(double x, double before, double target) {
    const uint64_t some = __ballot(x > 0.0), over = __ballot(x > 0.0 && before + x > target);
    return over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : 63;
}

// By a wave: the first of the n sums at which the running sum from `before` on exceeds `target`, as
// above; `before` becomes the sum ahead of it.
__device__ inline int32_t pick(const double* sums, int32_t n, double target, double& before, int lane) {
    const int32_t each = (n + 63) / 64, at = lane * each;
    double mine = 0.0, total;
    for (int32_t k = at; k < min(at + each, n); ++k) mine += sums[k];
    double run = before + wave_exclusive(mine, lane, total);
    const int found = first_over(mine, run, target);
    int32_t k = at, best = at;
    double best_run = run;
    for (; k < min(at + each, n); ++k) {
        if (sums[k] > 0.0) {
            best = k;
            best_run = run;
            if (run + sums[k] > target) break;
        }
        run += sums[k];
    }
    before = __shfl(best_run, found);
    return __shfl(best, found);
}

// What the walk down a request's nodes finds.
struct Walked {
    int32_t last;   // the last kept node; -1: none
    int32_t count;  // nodes that hang on it
    int32_t hangs[64];  // their tokens
};

// The nodes of request r, by one wave; with `put` it writes what is kept.
__device__ inline void walk(const VerifyArgs& a, int32_t r, bool put, Walked& w) {
    const int lane = threadIdx.x & 63;
    const int32_t start = a.row_starts[r], n = a.row_starts[r + 1] - start;
    const bool node = lane < n;
    const uint64_t mask = node ? a.masks[start + lane] : 0;
    const int64_t named = node ? a.tokens[start + lane] : -1;
    const int32_t token = named >= 0 && named < a.vocab ? static_cast<int32_t>(named) : -1;
    const uint64_t above = mask & ~(uint64_t(1) << lane);
    const int up = above ? 63 - __builtin_clzll(above) : -1;
    const bool real = lane > 0 && up >= 0 && (mask & 1);
    float p = 0.f, q = 0.f, u = 0.f;
    if (real) {
        u = a.uniforms[start + up];
        if (token >= 0) {
            p = a.p[(start + up) * a.ld + token];
            if (a.q) q = a.q[(start + up) * a.ldd + token];
        }
    }
    p = static_cast<float>(weight(p));
    // siblings before this node: whether one has its token, whether there is one, and their sum
    bool again = false, first = true;
    double ahead = 0.0;
    if (__any(real && up != lane - 1)) {  // a chain has none
        uint64_t rest = __ballot(real), before = 0;  // `before`: nodes with a sibling behind them
        while (rest) {
            const uint64_t same = __ballot(real && up == __builtin_amdgcn_readlane(up, __builtin_ctzll(rest)));
            before |= same & ~(uint64_t(1) << (63 - __builtin_clzll(same)));
            rest &= ~same;
        }
        while (before) {
            const int s = __builtin_ctzll(before);
            before &= before - 1;
            const bool sibling = real && lane > s && up == __builtin_amdgcn_readlane(up, s);
            again |= sibling && token == __builtin_amdgcn_readlane(token, s);
            first &= !sibling;
            // all before node s have been seen; a token that came before does not count again
            const float its = __uint_as_float(__builtin_amdgcn_readlane(again ? 0u : __float_as_uint(p), s));
            if (sibling) ahead += static_cast<double>(its);
        }
    }
    const double chance = p;
    bool taken = real && !again && chance > 0.0;
    if (a.q)
        taken = taken && first && static_cast<double>(u) * static_cast<double>(q) < chance;
    else
        taken = taken && u < ahead + chance && !(ahead > 0.0 && u < ahead);
    const uint64_t flags = __ballot(taken) | 1;
    const uint64_t on = __ballot(mask != 0 && (mask & 1) && (mask & ~flags) == 0);
    const int count = __popcll(on), last = on ? 63 - __builtin_clzll(on) : -1;
    const uint64_t below = (uint64_t(1) << lane) - 1;
    if (put) {
        for (int32_t i = count + lane; i < n; i += 64) a.path[start + i] = -1;
        if ((on >> lane) & 1) a.path[start + __popcll(on & below)] = lane;
        if (lane == 0) a.kept[r] = count;
    }
    const bool child = real && up == last;
    const uint64_t children = __ballot(child);
    if (child) w.hangs[__popcll(children & below)] = token;
    if (lane == 0) {
        w.last = last;
        w.count = __popcll(children);
    }
}

__device__ inline void clear_rest(const VerifyArgs& a) {  // the path of rows of no request
    for (int32_t i = a.row_starts[a.requests] + threadIdx.x; i < a.rows; i += kVerifyThreads) a.path[i] = -1;
}

__device__ inline Left left_of(const VerifyArgs& a, int32_t r, const Walked& w) {
    const int64_t row = a.row_starts[r] + w.last;
    Left left;
    left.p = a.p + row * a.ld;
    left.q = a.q ? a.q + row * a.ldd : nullptr;
    left.hangs = (threadIdx.x & 63) < w.count ? w.hangs[threadIdx.x & 63] : -1;
    left.vocab = a.vocab;
    left.mode = w.count == 0 ? kWhole : a.q ? kMinus : kWithout;
    return left;
}

// Tokens of a part of the row: 1024, or a multiple of it, so that at most 1024 parts have a sum.
__host__ __device__ inline int32_t part_tokens(int32_t vocab) {
    return (vocab + kPartTokens * kParts - 1) / (kPartTokens * kParts) * kPartTokens;
}

// The sums of parts first, first + step, ... up to `end` by a wave.
__device__ inline void sum_parts(const Left& left, double* sums, int32_t first, int32_t end, int32_t step, int32_t part,
                                 int lane) {
    for (int32_t k = first; k < end; k += step) {
        const double mine = left.sum(k * part, min(k * part + part, left.vocab), lane);
        if (lane == 0) sums[k] = mine;
    }
}

// The sum of n sums by a wave, the same in every lane.
__device__ inline double add_up(const double* sums, int32_t n, int lane) {
    double mine = 0.0, total;
    for (int32_t k = lane; k < n; k += 64) mine += sums[k];
    wave_exclusive(mine, lane, total);
    return total;
}

// The answer of request r by a block: `sums` are those of the `n` parts of `part` tokens, and `whole` their sum. A part
// of more than 1024 tokens is cut in sixteen, again and again.
__device__ inline void draw(const VerifyArgs& a, int32_t r, const Left& left, const double* sums, int32_t n, int32_t part,
                            double whole, double* pieces) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const double target = static_cast<double>(a.draws[r]) * whole;
    double before = 0.0;
    int32_t from = pick(sums, n, target, before, lane) * part, to = min(from + part, a.vocab);
    while (to - from > kPartTokens) {
        const int32_t piece = (to - from + kVerifyWaves - 1) / kVerifyWaves, begin = min(from + wave * piece, to);
        const double mine = left.sum(begin, min(begin + piece, to), lane);
        __syncthreads();  // the sums before have been read
        if (lane == 0) pieces[wave] = mine;
        __syncthreads();
        from += pick(pieces, kVerifyWaves, target, before, lane) * piece;
        to = min(from + piece, to);
    }
    if (wave != 0) return;
    constexpr int kEach = kPartTokens / 64;
    float p[kEach], q[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const int32_t i = kEach * lane + k;
        const bool in = from + i < to;
        p[k] = in ? left.p[from + i] : 0.f;
        q[k] = in && left.mode == kMinus ? left.q[from + i] : 0.f;
    }
    left.each_out(from, to, [&](int32_t token) {
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (from + kEach * lane + k == token) p[k] = 0.f;
    });
    double w[kEach], mine = 0.0, total;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        w[k] = weight(p[k], q[k]);
        mine += w[k];
    }
    double run = before + wave_exclusive(mine, lane, total);
    const int found = first_over(mine, run, target);
    int32_t answer = kEach * lane;
    bool over = false;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        if (!over && w[k] > 0.0) {
            answer = kEach * lane + k;
            over = run + w[k] > target;
        }
        run += w[k];
    }
    if (lane == found) a.answers[r] = from + answer;
}

// What is left is drawn from, or the whole row where nothing is; `sums` are in LDS.
__device__ inline void finish(const VerifyArgs& a, int32_t r, Left& left, double* sums, int32_t n, int32_t part,
                              double* pieces) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    double whole = add_up(sums, n, lane);
    if (!(whole > 0.0) && left.mode != kWhole) {
        left.mode = kWhole;
        __syncthreads();
        sum_parts(left, sums, wave, n, kVerifyWaves, part, lane);
        __syncthreads();
        whole = add_up(sums, n, lane);
    }
    if (whole > 0.0)
        draw(a, r, left, sums, n, part, whole, pieces);
    else if (tid == 0)
        a.answers[r] = -1;
}

// A block a request.
__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(VerifyArgs a) {
    __shared__ double sums[kParts], pieces[kVerifyWaves];
    __shared__ Walked w;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.x;
    if (r == 0) clear_rest(a);
    if (wave == 0) walk(a, r, true, w);
    __syncthreads();
    if (w.last < 0) {
        if (tid == 0) a.answers[r] = -1;
        return;
    }
    Left left = left_of(a, r, w);
    sum_parts(left, sums, wave, a.parts, kVerifyWaves, a.part, lane);
    __syncthreads();
    finish(a, r, left, sums, a.parts, a.part, pieces);
}

// Long rows: `blocks` blocks a request share the sums of the row's parts, then one draws.
__global__ void __launch_bounds__(kVerifyThreads) verify_sums_kernel(VerifyArgs a) {
    __shared__ Walked w;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.y, block = blockIdx.x;
    if (r == 0 && block == 0) clear_rest(a);
    if (wave == 0) walk(a, r, block == 0, w);
    __syncthreads();
    if (block == 0 && tid < static_cast<int>(sizeof(Walked) / 4))
        reinterpret_cast<int32_t*>(a.walked + r)[tid] = reinterpret_cast<const int32_t*>(&w)[tid];
    if (w.last < 0) return;
    const Left left = left_of(a, r, w);
    sum_parts(left, a.sums + static_cast<int64_t>(r) * a.parts, block * kVerifyWaves + wave, a.parts,
              a.blocks * kVerifyWaves, a.part, lane);
}

__global__ void __launch_bounds__(kVerifyThreads) verify_draw_kernel(VerifyArgs a) {
    __shared__ double sums[kParts], pieces[kVerifyWaves];
    __shared__ Walked w;
    const int tid = threadIdx.x;
    const int r = blockIdx.x;
    if (tid < static_cast<int>(sizeof(Walked) / 4))
        reinterpret_cast<int32_t*>(&w)[tid] = reinterpret_cast<const int32_t*>(a.walked + r)[tid];
    if (tid < a.parts) sums[tid] = a.sums[static_cast<int64_t>(r) * a.parts + tid];
    __syncthreads();
    if (w.last < 0) {
        if (tid == 0) a.answers[r] = -1;
        return;
    }
    Left left = left_of(a, r, w);
    finish(a, r, left, sums, a.parts, a.part, pieces);
}

// Blocks of a request's row; 1: all in one launch. Measured, us by calls one after another / in a graph:
// - Rows of at most 32768 tokens have one: 8 trees of 32003 tokens 13.8 / 13.3, with four blocks 16.4 / 13.7 (the host's
//   part of a second launch is 3); 64 chains 15.1 / 13.2, 17.3 / 15.2.
// - Longer rows of up to 128 requests as many as give each CU two blocks: 64 chains of 128256 tokens 20.0 / 21.1, with
//   one block a CU 20.9 / 22.0; 128 of them 30.8 / 30.0, 32.0 / 31.0. More requests have one block each: 200 of them
//   43.5 / 40.7, with two 46.6 / 44.0.
// - A row has ceil(tokens / 16384) blocks at most, of 10923 to 16384 tokens each (of more where these are more than
//   16): 16 chains of 64000 tokens 17.3 / 12.6 with their four, with eight 17.5 / 13.4, with one 15.4 / 16.9; a
//   request of 128256 tokens 17.1 / 11.8 with its eight, with two 17.2 / 13.4, with one 17.1 / 17.2.
int32_t verify_blocks(int32_t requests, int32_t vocab) {
    if (vocab <= 32768) return 1;
    const int64_t most = requests <= kStepCus / 2 ? 2 * kStepCus / requests : 1, parts = ceil_div(vocab, 16384);
    const int64_t blocks = most < parts ? most : parts;
    return static_cast<int32_t>(blocks < 1 ? 1 : blocks < kVerifyBlocks ? blocks : kVerifyBlocks);
}

}  // namespace
}  // namespace kvr

using namespace kvr;

extern "C" int64_t kvr_verify_workspace_bytes(int32_t requests, int32_t vocab) {
    if (requests <= 0 || requests > KVR_STEP_MAX_REQUESTS || vocab <= 0 || vocab > kVerifyVocab)
        return KVR_E_UNSUPPORTED_SHAPE;
    const int64_t blocks = verify_blocks(requests, vocab);
    return blocks == 1 ? 0 : ceil_div(requests * static_cast<int64_t>(sizeof(Walked) + ceil_div(vocab, part_tokens(vocab)) * sizeof(double)), 16) * 16;
}

extern "C" int kvr_verify_drafts(const float* probs, int64_t ld, const float* draft_probs, int64_t ldd, int32_t vocab,
                                 const int64_t* tokens, const float* uniforms, const float* draws,
                                 const kvr_step_desc* d, int32_t* kept, int32_t* path, int64_t* answers, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
    const int st = check_step(d);
    if (st != KVR_OK) return st;
    if (!d->masks) return KVR_E_UNSUPPORTED_SHAPE;
    if (!probs || !tokens || !uniforms || !draws || !kept || !path || !answers) return KVR_E_NULL_POINTER;
    const int64_t need = kvr_verify_workspace_bytes(d->requests, vocab);
    if (need < 0) return static_cast<int>(need);
    if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15) || workspace_bytes < need))
        return KVR_E_WORKSPACE_TOO_SMALL;
    if (ld < vocab || (draft_probs && ldd < vocab)) return KVR_E_BAD_STRIDE;
    VerifyArgs a;
    a.p = probs;
    a.q = draft_probs;
    a.ld = ld;
    a.ldd = ldd;
    a.tokens = tokens;
    a.uniforms = uniforms;
    a.draws = draws;
    a.row_starts = d->row_starts;
    a.masks = d->masks;
    a.kept = kept;
    a.path = path;
    a.answers = answers;
    a.vocab = vocab;
    a.rows = d->rows;
    a.requests = d->requests;
    a.blocks = verify_blocks(d->requests, vocab);
    a.part = part_tokens(vocab);
    a.parts = static_cast<int32_t>(ceil_div(vocab, a.part));
    a.walked = static_cast<Walked*>(workspace);
    a.sums = reinterpret_cast<double*>(a.walked + d->requests);
    hipStream_t hs = as_stream(stream);
    if (a.blocks == 1) {
        verify_kernel<<<d->requests, kVerifyThreads, 0, hs>>>(a);
    } else {
        verify_sums_kernel<<<dim3(a.blocks, d->requests), kVerifyThreads, 0, hs>>>(a);
        verify_draw_kernel<<<d->requests, kVerifyThreads, 0, hs>>>(a);
    }
    return launch_status();
}
