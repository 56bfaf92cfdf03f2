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
// beside the reads. One block a request: lane t of its first wave is node t; then
// each of the 16 waves sums a sixteenth of the row, the sixteenth that holds the
// draw is cut in sixteen again, and a wave walks what is left.
#include "kvr_internal.h"
#include "kvr_step.h"
#include "kvrepair_serve.h"

#include <math.h>

namespace kvr {
namespace {

constexpr int kVerifyThreads = 1024;
constexpr int kVerifyWaves = kVerifyThreads / 64;

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
    int32_t vocab;
    int32_t rows;
    int32_t requests;
};

// A weight that counts: positive and finite.
__device__ inline double sane(double w) { return w > 0.0 && w < INFINITY ? w : 0.0; }

enum VerifyMode { kWhole = 0, kWithout = 1, kMinus = 2 };

// What is left of a row.
struct Left {
    const float* p;
    const float* q;
    const int32_t* hangs;  // tokens that do not count (kWithout)
    int32_t count;
    int32_t vocab;
    int mode;

    __device__ inline double at(int32_t i) const {
        if (mode == kMinus) return sane(static_cast<double>(p[i]) - static_cast<double>(q[i]));
        const double w = sane(p[i]);
        if (mode == kWithout)
            for (int32_t c = 0; c < count; ++c)
                if (hangs[c] == i) return 0.0;
        return w;
    }

    // The sum over [begin, end) by a wave, the same in every lane.
    __device__ inline double sum(int32_t begin, int32_t end, int lane) const {
        double s = 0.0;
        end = min(end, vocab);
        int32_t i = begin + 4 * lane;
        constexpr int kAhead = 4;
        for (; begin < end; begin += 256 * kAhead, i += 256 * kAhead) {
            f32x4u a[kAhead], b[kAhead];
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                a[e] = b[e] = f32x4u{0.f, 0.f, 0.f, 0.f};
                const int32_t j = i + 256 * e;
                if (j + 4 <= end) {
                    a[e] = *reinterpret_cast<const f32x4u*>(p + j);
                    if (mode == kMinus) b[e] = *reinterpret_cast<const f32x4u*>(q + j);
                } else {
                    for (int32_t k = 0; j + k < end; ++k) {
                        a[e][k] = p[j + k];
                        if (mode == kMinus) b[e][k] = q[j + k];
                    }
                }
            }
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                const int32_t j = i + 256 * e;
                if (mode == kWithout)
                    for (int32_t c = 0; c < count; ++c)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (hangs[c] == j + k) a[e][k] = 0.f;
#pragma unroll
                for (int k = 0; k < 4; ++k) s += sane(static_cast<double>(a[e][k]) - static_cast<double>(b[e][k]));
            }
        }
#pragma unroll
        for (int d = 32; d > 0; d /= 2) s += __shfl_xor(s, d);
        return s;
    }
};

// The first of the n sums with something in it at which the running sum (from `before` on) exceeds `target`,
// or else the last with something in it; `before` becomes the sum ahead of it.
__device__ inline int pick(const double* sums, int n, double target, double& before) {
    int found = 0;
    double run = before;
    for (int k = 0; k < n; ++k) {
        const double next = run + sums[k];
        if (sums[k] > 0.0) {
            found = k;
            before = run;
            if (next > target) break;
        }
        run = next;
    }
    return found;
}

__global__ void __launch_bounds__(kVerifyThreads) verify_kernel(VerifyArgs a) {
    __shared__ double sums[kVerifyWaves];
    __shared__ int32_t hangs[64];
    __shared__ int32_t s_last, s_hangs;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int r = blockIdx.x;
    const int32_t start = a.row_starts[r], n = a.row_starts[r + 1] - start;
    if (r == 0)  // rows of no request
        for (int32_t i = a.row_starts[a.requests] + tid; i < a.rows; i += kVerifyThreads) a.path[i] = -1;
    if (wave == 0) {
        const bool node = lane < n;
        const uint64_t mask = node ? a.masks[start + lane] : 0;
        const int64_t token = node ? a.tokens[start + lane] : -1;
        const uint64_t above = mask & ~(uint64_t(1) << lane);
        const int up = above ? 63 - __builtin_clzll(above) : -1;
        const bool real = lane > 0 && up >= 0 && (mask & 1);
        double chance = 0.0, drafted = 0.0;
        float u = 0.f;
        if (real) {
            u = a.uniforms[start + up];
            if (token >= 0 && token < a.vocab) {
                chance = sane(a.p[(start + up) * a.ld + token]);
                if (a.q) drafted = a.q[(start + up) * a.ldd + token];
            }
        }
        // siblings before this node: whether one has its token, whether there is one, and their sum
        bool again = false, first = true;
        double ahead = 0.0;
        const uint64_t nodes = __ballot(real);
        for (int s = 1; s < 63 && (nodes >> s) > 1; ++s) {
            const int64_t other = __shfl(token, s);
            const int hung = __shfl(up, s);
            const bool sibling = real && lane > s && ((nodes >> s) & 1) && hung == up;
            again |= sibling && other == token;
            first &= !sibling;
            const double its = __shfl(again ? 0.0 : chance, s);  // all before node s have been seen
            if (sibling) ahead += its;
        }
        bool taken = real && !again && chance > 0.0;
        if (a.q)
            taken = taken && first && static_cast<double>(u) * drafted < chance;
        else
            taken = taken && u < ahead + chance && !(u < ahead);
        const uint64_t flags = __ballot(taken) | 1;
        const uint64_t on = __ballot(mask != 0 && (mask & 1) && (mask & ~flags) == 0);
        const int count = __popcll(on), last = on ? 63 - __builtin_clzll(on) : -1;
        for (int32_t i = count + lane; i < n; i += 64) a.path[start + i] = -1;
        if ((on >> lane) & 1) a.path[start + __popcll(on & ((uint64_t(1) << lane) - 1))] = lane;
        const bool child = real && up == last;
        const uint64_t children = __ballot(child);
        if (child) hangs[__popcll(children & ((uint64_t(1) << lane) - 1))] =
            token >= 0 && token < a.vocab ? static_cast<int32_t>(token) : -1;
        if (lane == 0) {
            a.kept[r] = count;
            s_last = last;
            s_hangs = __popcll(children);
        }
    }
    __syncthreads();
    const int32_t last = s_last;
    if (last < 0) {
        if (tid == 0) a.answers[r] = -1;
        return;
    }
    Left left;
    left.p = a.p + (start + last) * a.ld;
    left.q = a.q ? a.q + (start + last) * a.ldd : nullptr;
    left.hangs = hangs;
    left.count = s_hangs;
    left.vocab = a.vocab;
    left.mode = left.count == 0 ? kWhole : a.q ? kMinus : kWithout;
    // a sixteenth of the row for each wave, in whole groups of 256 tokens
    const int32_t part = (a.vocab + kVerifyWaves * 256 - 1) / (kVerifyWaves * 256) * 256;
    double whole;
    for (;;) {
        const double mine = left.sum(min(wave * part, a.vocab), min((wave + 1) * part, a.vocab), lane);
        if (lane == 0) sums[wave] = mine;
        __syncthreads();
        whole = 0.0;
#pragma unroll
        for (int k = 0; k < kVerifyWaves; ++k) whole += sums[k];
        if (whole > 0.0 || left.mode == kWhole) break;
        left.mode = kWhole;  // nothing is left: the whole row
        __syncthreads();
    }
    if (!(whole > 0.0)) {
        if (tid == 0) a.answers[r] = -1;
        return;
    }
    const double target = static_cast<double>(a.draws[r]) * whole;
    double before = 0.0;
    const int32_t base = pick(sums, kVerifyWaves, target, before) * part, piece = part / kVerifyWaves;
    __syncthreads();
    {
        const int32_t from = min(base + wave * piece, a.vocab), to = min(from + piece, a.vocab);
        const double mine = left.sum(from, to, lane);
        if (lane == 0) sums[wave] = mine;
    }
    __syncthreads();
    const int32_t from = base + pick(sums, kVerifyWaves, target, before) * piece;
    if (wave != 0) return;
    // 64 tokens at a time: their running sum in every lane
    const int32_t to = min(from + piece, a.vocab);
    int32_t answer = -1;
    double run = before;
    for (int32_t i = from; i < to; i += 64) {
        const double w = i + lane < to ? left.at(i + lane) : 0.0;
        double sum = w;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const double up = __shfl_up(sum, d);
            if (lane >= d) sum += up;
        }
        const uint64_t some = __ballot(w > 0.0), over = __ballot(w > 0.0 && run + sum > target);
        if (some) answer = i + 63 - __builtin_clzll(some);
        if (over) {
            answer = i + __builtin_ctzll(over);
            break;
        }
        run += __shfl(sum, 63);
    }
    if (lane == 0) a.answers[r] = answer;
}

}  // namespace
}  // namespace kvr

using namespace kvr;

extern "C" int kvr_verify_drafts(const float* probs, int64_t ld, const float* draft_probs, int64_t ldd, int32_t vocab,
                                 const int64_t* tokens, const float* uniforms, const float* draws,
                                 const kvr_step_desc* d, int32_t* kept, int32_t* path, int64_t* answers, void* stream) {
    const int st = check_step(d);
    if (st != KVR_OK) return st;
    if (!d->masks) return KVR_E_UNSUPPORTED_SHAPE;
    if (!probs || !tokens || !uniforms || !draws || !kept || !path || !answers) return KVR_E_NULL_POINTER;
    // 16 waves' shares of the row fit 32 bits
    if (vocab <= 0 || vocab > (int32_t(1) << 30)) return KVR_E_UNSUPPORTED_SHAPE;
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
    verify_kernel<<<d->requests, kVerifyThreads, 0, as_stream(stream)>>>(a);
    return launch_status();
}
