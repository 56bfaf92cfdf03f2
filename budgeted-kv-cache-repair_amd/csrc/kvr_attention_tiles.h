// Device code that the attention kernels share: the MFMA with its hi + lo pairs, the
// direct loads into LDS, and a wave's work on staged 32-key sub-tiles of K and V for
// two 16-row query tiles (kvr_attention.hip: of two query heads; kvr_tree_attention.hip:
// consecutive query rows). The staged layout is described at kvr_attention.hip's
// head-pair kernel.
#pragma once

#include "kvr_internal.h"

#include <math.h>

namespace kvr {
namespace {

constexpr float kLazyLog2 = 8.f;           // lazy-rescale headroom (log2 units): p <= 256

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Probabilities enter the PV MFMA as a hi + lo pair of 16-bit values so they
// are not rounded to 16 bits (the reference Triton kernel keeps P in fp32,
// _indexed_triton.py:54-58). split() packs two probabilities: hi holds their
// 16-bit heads, lo the rounded remainders p - head. fp16's have no step below 2^-24:
// what is smaller than half of that is lost, unless Lift moves it up.
template <typename T> struct mma_t;
template <> struct mma_t<bf16_t> {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    __device__ static inline f32x4 mma(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // bf16 head = the upper half of the fp32 bits (truncation); p - head is exact
    // in fp32 and its RNE bf16 rounding leaves an error below 2^-16 |p|.
    // two probabilities rounded to bf16 (RNE), packed
    __device__ static inline uint32_t round2(float p0, float p1) {
        const f32x2 r = {p0, p1};
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));
    }
    __device__ static inline void split(float p0, float p1, uint32_t& hi, uint32_t& lo) {
        const uint32_t b0 = __float_as_uint(p0), b1 = __float_as_uint(p1);
        hi = __builtin_amdgcn_perm(b1, b0, 0x07060302u);
        const f32x2 r = {p0 - __uint_as_float(b0 & 0xffff0000u), p1 - __uint_as_float(b1 & 0xffff0000u)};
        lo = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, bf16x2));  // v_cvt_pk_bf16_f32 (RNE)
    }
};
template <> struct mma_t<f16_t> {
    typedef _Float16 v8 __attribute__((ext_vector_type(8)));
    __device__ static inline f32x4 mma(v8 a, v8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    __device__ static inline uint32_t round2(float p0, float p1) {
        return static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(p0))) |
               (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, static_cast<_Float16>(p1))) << 16);
    }
    __device__ static inline void split(float p0, float p1, uint32_t& hi, uint32_t& lo) {
        const _Float16 h0 = static_cast<_Float16>(p0), h1 = static_cast<_Float16>(p1);
        const _Float16 l0 = static_cast<_Float16>(p0 - static_cast<float>(h0));
        const _Float16 l1 = static_cast<_Float16>(p1 - static_cast<float>(h1));
        hi = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, h0)) |
             (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, h1)) << 16);
        lo = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, l0)) |
             (static_cast<uint32_t>(__builtin_bit_cast(uint16_t, l1)) << 16);
    }
};

constexpr int kPairSub = 32;                 // keys per sub-tile
constexpr int kPairSubs = 4;                 // sub-tiles staged per step
constexpr int kPairStepKeys = kPairSub * kPairSubs;
constexpr int kPairThreads = 512;

template <int D>
struct PairCfg {
    static constexpr int c8 = D / 8;                              // 16-byte pieces per row
    static constexpr int tensor_bytes = kPairStepKeys * D * 2;    // K or V of one step
    static constexpr int stage_bytes = 2 * tensor_bytes;          // K then V
    static constexpr int bytes = 2 * stage_bytes;                 // double-buffered
    static constexpr int pieces_per_wave = tensor_bytes / 16 / 8; // 16-byte pieces one wave loads per tensor
    static constexpr int loads = pieces_per_wave / 64;            // load instructions per wave per tensor
    static_assert(pieces_per_wave % 64 == 0, "whole load instructions");
    // Piece swizzles (XOR on the 16-byte piece index; rows are keys). K: 8
    // consecutive rows at one piece hit 8 distinct bank groups (a 16-byte read
    // serves 8 lanes per cycle). V: the transposing read serves 16 lanes per
    // cycle, 4 consecutive rows x 2 adjacent pieces, which 2 r spreads over 8
    // distinct bank groups.
    __host__ __device__ static constexpr int kswz(int r) { return r & (c8 - 1); }
    __host__ __device__ static constexpr int vswz(int r) { return (2 * r) & (c8 - 1); }
};

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

// clang warns of every M0 in a list of clobbers, as a register that it may use itself.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 16 bytes per lane from `src` (per-lane global address) to LDS at `dst` + 16 *
// lane (`dst` wave-uniform): global_load_lds_dwordx4, the LDS base in M0, which such a
// load may read one wait state after its write (s_nop: the compiler adds none here). Issued
// as inline assembly so the compiler's wait-count pass, which cannot tell these
// LDS writes from the stage being read, adds no vmcnt waits before LDS reads;
// the kernel waits for them itself (vmcnt(0), then a barrier) before reading.
__device__ inline void lds_dma16(const char* src, char* dst) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane(
        static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)dst)));
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(src), "s"(m0) : "memory", "m0");
}

// The same load from a wave-uniform base (SGPRs) plus a 32-bit per-lane byte
// offset: no per-lane address arithmetic.
__device__ inline void lds_dma16(const char* base, uint32_t off, char* dst) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane(
        static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)dst)));
    // the base is wave-uniform; reading it from the first lane keeps it in
    // SGPRs even where the compiler cannot prove that (free where it can).
    // readfirstlane returns int: each half goes through uint32_t so the low
    // half is zero-extended, not sign-extended, into the 64-bit address.
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(b))));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(b >> 32))));
    const uint64_t sb = (static_cast<uint64_t>(hi) << 32) | lo;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(sb), "s"(m0)
                 : "memory", "m0");
}

// The same with the nontemporal hint, for bytes that are read once.
__device__ inline void lds_dma16_once(const char* base, uint32_t off, char* dst) {
    const uint32_t m0 = __builtin_amdgcn_readfirstlane(
        static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) char*)dst)));
    const uint64_t b = reinterpret_cast<uint64_t>(base);
    const uint32_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(b))));
    const uint32_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(static_cast<uint32_t>(b >> 32))));
    const uint64_t sb = (static_cast<uint64_t>(hi) << 32) | lo;
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1 nt" ::"v"(off), "s"(sb), "s"(m0)
                 : "memory", "m0");
}

#pragma clang diagnostic pop

// The power of two that probabilities are made larger by before they are split, and how
// far (log2) a score may exceed the running maximum. A sum of weighted values and the sum
// of its weights take the same one, and their quotient loses it again. fp16 needs one: its
// pair has no step below 2^-24, which without one is 2^-24 of the largest weight, and a
// weight below half of that is lost. With 2^12 the pair is off by at most 2^-37 of the
// largest weight and 2^-22 of its own; 2^15 is the most that a probability reaches.
template <typename T, bool LIFT> struct Lift {
    static constexpr float kLog2 = 0.f, kHead = kLazyLog2;
};
template <> struct Lift<f16_t, true> {
    static constexpr float kLog2 = 12.f, kHead = 3.f;
};

// HILO: probabilities enter PV as a hi + lo pair of 16-bit values (fp32-class,
// the reference Triton kernel's precision); otherwise each is rounded to the
// input dtype before PV, as the SDPA path the packed executor replaces rounds it.
// LIFT: with Lift's power of two.
template <typename T, int D, bool HILO, bool LIFT = false>
struct PairWave {
    using L = Lift<T, LIFT>;
    using M = mma_t<T>;
    using v8 = typename M::v8;
    using C = PairCfg<D>;
    static constexpr int DS = D / 32;  // k-steps of the QK^T MFMA
    static constexpr int DT = D / 16;  // d tiles of the PV MFMA

    v8 qf[2][DS];
    f32x4 o[2][DT];
    f32x4 lsum[2];    // row sums of P as a 17th output tile: row 0 of O^T += ones . P^T
    float m_run[2];
    // kept with m_run, so the per-sub-tile work does not recompute them: the
    // exponent offset L::kLog2 - (m_run, or 0 while m_run = -inf) and the lazy-rescale
    // threshold m_run + L::kHead
    float m_neg[2], m_thr[2];
    int32_t pos;      // this lane's row position; -1 past the selected rows
    v8 ones;          // A operand of the row-sum tile: row 0 all ones, rows 1..15 zero
    // Per-lane byte offsets of this lane's fragment reads within a staged tile,
    // for sub-tile row 0 (every sub-tile starts at a multiple of 16 rows, so the
    // swizzle of a lane's rows does not depend on the sub-tile or key tile; those
    // add compile-time offsets). K: row lq, piece 4 ds + lj. V (transposing
    // reads): row 4 lj + (lq >> 2), dims 16 dt + 4 (lq & 3).
    int32_t koff[DS];
    int32_t voff[DT];

    // byte offsets of piece c of row r in the swizzled K and V tiles
    __device__ static inline int kpiece(int r, int c) { return (r * C::c8 + (c ^ C::kswz(r))) * 16; }
    __device__ static inline int vpiece(int r, int c) { return (r * C::c8 + (c ^ C::vswz(r))) * 16; }

    __device__ inline void init(int lq, int lj) {
        offsets(lq, lj);
        const uint16_t one = elem<T>::from_float(1.f);
        const uint32_t w = lq == 0 ? (static_cast<uint32_t>(one) | (static_cast<uint32_t>(one) << 16)) : 0u;
        ones = __builtin_bit_cast(v8, u32x4{w, w, w, w});
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            m_run[t] = -INFINITY;
            m_neg[t] = L::kLog2 - 0.f;
            m_thr[t] = -INFINITY + L::kHead;
            lsum[t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[t][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }

    __device__ inline void offsets(int lq, int lj) {
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) koff[ds] = kpiece(lq, 4 * ds + lj);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int d0 = 16 * dt + 4 * (lq & 3);
            voff[dt] = vpiece(4 * lj + (lq >> 2), d0 >> 3) + (d0 & 4) * 2;
        }
    }

    // K fragments of the sub-tile: [ds][kt], rows 16 kt + lq, pieces 4 ds + lj.
    __device__ inline void read_k(const char* Ks, v8 (&kf)[DS][2]) {
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
                kf[ds][kt] =
                    __builtin_bit_cast(v8, *reinterpret_cast<const u32x4*>(Ks + koff[ds] + 16 * kt * D * 2));
    }

    // S^T = K Q_t^T for head t: keys on the M axis, lane (lq, lj) gets keys
    // 16 kt + 4 lj + i of row lq.
    __device__ inline void qk(int t, const v8 (&kf)[DS][2], f32x4 (&st)[2]) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) st[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ds = 0; ds < DS; ++ds)
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) st[kt] = M::mma(kf[ds][kt], qf[t][ds], st[kt]);
    }

    // Scores past a row's position become -inf (the causal mask; only sub-tiles
    // that reach past the tile's first position need it).
    __device__ inline void apply_mask(f32x4 (&st)[2], int32_t key0, int lj) { apply_mask_at(st, key0, lj, pos); }

    // The same with the row's last visible key given (at most its position).
    __device__ static inline void apply_mask_at(f32x4 (&st)[2], int32_t key0, int lj, int32_t last) {
        const int32_t lim = last - key0 - 4 * lj;  // key 16 kt + 4 lj + i is visible iff 16 kt + i <= lim
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) st[kt][i] = (16 * kt + i <= lim) ? st[kt][i] : -INFINITY;
    }

    // Row maximum of head t's scores over this lane's keys, scaled.
    __device__ inline float row_max(const f32x4 (&st)[2], float scale_log2, float (&x)[2][4]) {
        float mx = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[kt][i] = st[kt][i];
                mx = fmaxf(mx, x[kt][i]);
            }
        return mx * scale_log2;  // scale_log2 > 0: the scaled maximum is the raw maximum scaled
    }

    // Lazy move of head t's reference maximum: it moves only when a score
    // exceeds it by more than L::kHead (so p <= 2^8, lifted 2^15, and the fp32 accumulators
    // cannot overflow); O and the row sums are rescaled then (rare).
    __device__ inline void rescale_if(int t, float mx) {
        if (__any(mx > m_thr[t])) {
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float m_new = (mx > m_thr[t]) ? mx : m_run[t];
            // 1 if unmoved, 0 from -inf; a row with no visible key keeps m = -inf
            const float alpha = __builtin_amdgcn_exp2f(m_run[t] - (m_new == -INFINITY ? 0.f : m_new));
            m_run[t] = m_new;
            m_neg[t] = L::kLog2 - (m_new == -INFINITY ? 0.f : m_new);
            m_thr[t] = m_new + L::kHead;
            lsum[t] *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[t][dt] *= alpha;
        }
    }

    // two probabilities as B-operand halves: hi (+ lo) or the rounded pair
    __device__ static inline void pack(float p0, float p1, uint32_t& hi, uint32_t& lo) {
        if (HILO)
            M::split(p0, p1, hi, lo);
        else
            hi = M::round2(p0, p1);
    }

    // P = exp2(scale x - m) of head t as the B operand(s) of the PV MFMA:
    // element 4h + i of lane (lq, lj) is key 16h + 4 lj + i.
    __device__ inline void probs(int t, float (&x)[2][4], float scale_log2, u32x4& phi, u32x4& plo) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[kt][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[kt][i], scale_log2, m_neg[t]));
        uint32_t hv[4], lv[4] = {0u, 0u, 0u, 0u};
        pack(x[0][0], x[0][1], hv[0], lv[0]);
        pack(x[0][2], x[0][3], hv[1], lv[1]);
        pack(x[1][0], x[1][1], hv[2], lv[2]);
        pack(x[1][2], x[1][3], hv[3], lv[3]);
        phi = u32x4{hv[0], hv[1], hv[2], hv[3]};
        plo = u32x4{lv[0], lv[1], lv[2], lv[3]};
    }

    // V^T fragments of the sub-tile: per d tile two transposing reads give keys
    // 4 lj .. + 4 and 16 + 4 lj .. + 4 of dim 16 dt + lq.
    __device__ inline void read_v(const char* Vs, v8 (&vf)[DT]) {
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const s16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(Vs + voff[dt]));
            const s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(Vs + voff[dt] + 16 * D * 2));
            vf[dt] = __builtin_bit_cast(v8, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }

    // O_t^T += V^T P_t^T and the row sums.
    __device__ inline void pv(int t, const v8 (&vf)[DT], const u32x4& phi, const u32x4& plo) {
        const v8 bh = __builtin_bit_cast(v8, phi), bl = __builtin_bit_cast(v8, plo);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            o[t][dt] = M::mma(vf[dt], bh, o[t][dt]);
            if (HILO) o[t][dt] = M::mma(vf[dt], bl, o[t][dt]);
        }
        lsum[t] = M::mma(ones, bh, lsum[t]);
        if (HILO) lsum[t] = M::mma(ones, bl, lsum[t]);
    }

    // PV(0) with P(1) interleaved in source order: after the two MFMAs of each
    // d tile one probability of head 1 is computed (and, every other tile, a
    // pair is split), so the VALU work issues while the MFMAs execute.
    __device__ inline void pv0_probs1(const v8 (&vf)[DT], const u32x4& h0, const u32x4& l0, float (&x1)[2][4],
                                      float scale_log2, u32x4& h1, u32x4& l1) {
        const v8 bh = __builtin_bit_cast(v8, h0), bl = __builtin_bit_cast(v8, l0);
        float p[8];
        uint32_t hv[4], lv[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            o[0][dt] = M::mma(vf[dt], bh, o[0][dt]);
            if (HILO) o[0][dt] = M::mma(vf[dt], bl, o[0][dt]);
            if (dt < 8) {
                p[dt] = __builtin_amdgcn_exp2f(__builtin_fmaf(x1[dt >> 2][dt & 3], scale_log2, m_neg[1]));
                if (dt & 1) pack(p[dt - 1], p[dt], hv[dt >> 1], lv[dt >> 1]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (DT < 8) {  // head_dim 64: the remaining probabilities
#pragma unroll
            for (int e = DT; e < 8; ++e) {
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x1[e >> 2][e & 3], scale_log2, m_neg[1]));
                if (e & 1) pack(p[e - 1], p[e], hv[e >> 1], lv[e >> 1]);
            }
        }
        lsum[0] = M::mma(ones, bh, lsum[0]);
        if (HILO) lsum[0] = M::mma(ones, bl, lsum[0]);
        h1 = u32x4{hv[0], hv[1], hv[2], hv[3]};
        l1 = u32x4{lv[0], lv[1], lv[2], lv[3]};
    }

    // One 32-key sub-tile (Ks / Vs: its first staged K / V row) for both heads,
    // software-pipelined over the two heads so the MFMA work of one overlaps the
    // softmax of the other, each K and V fragment read once for both:
    //   read V, K;  QK(0);  QK(1);  [mask];  max, rescale (0, 1);  P(0);
    //   PV(0) || P(1);  PV(1)
    // MFMAs run asynchronously, so VALU work issued between them overlaps them;
    // the scheduling barriers keep this order.
    // mask: some key may lie beyond some row's position (wave-uniform).
    __device__ inline void step(const char* Ks, const char* Vs, bool mask, int32_t key0, int lj, float scale_log2) {
        v8 vf[DT];
        v8 kf[DS][2];
        read_v(Vs, vf);
        read_k(Ks, kf);
        __builtin_amdgcn_sched_barrier(0);
        compute(kf, vf, mask, key0, lj, scale_log2);
    }

    // The sub-tile's work once its K and V fragments are in registers.
    __device__ inline void compute(const v8 (&kf)[DS][2], const v8 (&vf)[DT], bool mask, int32_t key0, int lj,
                                   float scale_log2) {
        f32x4 s0[2], s1[2];
        float x0[2][4], x1[2][4];
        qk(0, kf, s0);
        qk(1, kf, s1);
        __builtin_amdgcn_sched_barrier(0);
        if (mask) {
            apply_mask(s0, key0, lj);
            apply_mask(s1, key0, lj);
        }
        rescale_if(0, row_max(s0, scale_log2, x0));
        rescale_if(1, row_max(s1, scale_log2, x1));
        finish_subtile(vf, x0, x1, scale_log2);
    }

    // P and PV of both heads from masked, rescaled scores x0 / x1.
    __device__ inline void finish_subtile(const v8 (&vf)[DT], float (&x0)[2][4], float (&x1)[2][4],
                                          float scale_log2) {
        u32x4 h0, l0, h1, l1;
        probs(0, x0, scale_log2, h0, l0);
        __builtin_amdgcn_sched_barrier(0);
        pv0_probs1(vf, h0, l0, x1, scale_log2, h1, l1);
        __builtin_amdgcn_sched_barrier(0);
        pv(1, vf, h1, l1);
    }

    // ---- Software-pipelined stage (one key class: the wave walks every
    // sub-tile of the stage). Sub-tile j's work is split so that the MFMAs of
    // one part issue beside the vector-ALU work of another:
    //   A: P of sub-tile j (both heads)       with the QK MFMAs of sub-tile j + 1
    //   B: PV of sub-tile j (and row sums)    with the row maxima of sub-tile j + 1
    //   C: the lazy rescale for sub-tile j + 1 (rare)
    // Every operation, operand and per-accumulator order is that of step():
    // the results are bit-identical, only independent instructions move.

    // scaled row maximum of one head's scores (the value row_max returns)
    __device__ static inline float scaled_max(const f32x4 (&st)[2], float scale_log2) {
        float mx = -INFINITY;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, st[kt][i]);
        return mx * scale_log2;
    }

    // V^T fragment of d tile dt (one tile of read_v).
    __device__ inline v8 read_v_tile(const char* Vs, int dt) {
        const s16x4 lo4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(Vs + voff[dt]));
        const s16x4 hi4 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(Vs + voff[dt] + 16 * D * 2));
        return __builtin_bit_cast(v8, __builtin_shufflevector(lo4, hi4, 0, 1, 2, 3, 4, 5, 6, 7));
    }

    // K fragment f of the sub-tile at Ks: k-step f / 2, key tile f % 2 (read_k's kf[f / 2][f % 2]).
    __device__ inline v8 read_k_frag(const char* Ks, int f) {
        return __builtin_bit_cast(v8, *reinterpret_cast<const u32x4*>(Ks + koff[f >> 1] + 16 * (f & 1) * D * 2));
    }

    // A: probabilities of both heads from scores c0 / c1 (maxima applied), each
    // computed before one QK MFMA of the next sub-tile (K tiles at Ks1) into
    // n0 / n1. The MFMAs go by K fragment, both heads in turn; fragments are
    // read three ahead, each freed after its second MFMA.
    __device__ inline void probs_qk(const f32x4 (&c0)[2], const f32x4 (&c1)[2], const char* Ks1, f32x4 (&n0)[2],
                                    f32x4 (&n1)[2], float scale_log2, u32x4& h0, u32x4& l0, u32x4& h1, u32x4& l1) {
        static_assert(DS == 4, "head_dim 128");
        constexpr int kAhead = 3;
        float p[16];
        uint32_t hv[8], lv[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
        v8 kf[2 * DS];
#pragma unroll
        for (int f = 0; f < kAhead; ++f) kf[f] = read_k_frag(Ks1, f);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) n0[kt] = n1[kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            // probability i: head i / 8, key 16 kt + 4 lj + e with (kt, e) = divmod(i % 8, 4)
            const int e = i & 7;
            const float s = i < 8 ? c0[e >> 2][e & 3] : c1[e >> 2][e & 3];
            p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s, scale_log2, m_neg[i >> 3]));
            if (i & 1) {
                pack(p[i - 1], p[i], hv[i >> 1], lv[i >> 1]);
                // pinned here: otherwise the compiler sinks the probabilities
                // to their first use in part B, past every QK MFMA (the lo
                // halves only where they exist: a pinned constant 0 costs a move)
                if (HILO)
                    asm volatile("" : "+v"(hv[i >> 1]), "+v"(lv[i >> 1]));
                else
                    asm volatile("" : "+v"(hv[i >> 1]));
            }
            // QK MFMA i: K fragment i / 2 (k-step i / 4, key tile (i / 2) % 2), head i % 2
            // (per accumulator the k-steps go in qk()'s order)
            const int f = i >> 1, ds = i >> 2, kt = f & 1;
            if (i & 1) {
                n1[kt] = M::mma(kf[f], qf[1][ds], n1[kt]);
                if (f + kAhead < 2 * DS) kf[f + kAhead] = read_k_frag(Ks1, f + kAhead);
            } else {
                n0[kt] = M::mma(kf[f], qf[0][ds], n0[kt]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        h0 = u32x4{hv[0], hv[1], hv[2], hv[3]};
        l0 = u32x4{lv[0], lv[1], lv[2], lv[3]};
        h1 = u32x4{hv[4], hv[5], hv[6], hv[7]};
        l1 = u32x4{lv[4], lv[5], lv[6], lv[7]};
    }

    // B: PV of both heads by d tile (V^T fragments read three tiles ahead from
    // Vs, each freed after its two heads' MFMAs), then the row sums; the next
    // sub-tile's scaled row maxima (n0 / n1, masked beforehand where needed)
    // are computed between the MFMAs.
    __device__ inline void pv_max(const char* Vs, const u32x4& h0, const u32x4& l0, const u32x4& h1,
                                  const u32x4& l1, const f32x4 (&n0)[2], const f32x4 (&n1)[2], float scale_log2,
                                  float (&mx)[2]) {
        constexpr int kAhead = 3;
        const v8 b[2][2] = {{__builtin_bit_cast(v8, h0), __builtin_bit_cast(v8, l0)},
                            {__builtin_bit_cast(v8, h1), __builtin_bit_cast(v8, l1)}};
        v8 vf[DT];
#pragma unroll
        for (int dt = 0; dt < kAhead; ++dt) vf[dt] = read_v_tile(Vs, dt);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            if (dt + kAhead < DT) vf[dt + kAhead] = read_v_tile(Vs, dt + kAhead);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                o[t][dt] = M::mma(vf[dt], b[t][0], o[t][dt]);
                if (HILO) o[t][dt] = M::mma(vf[dt], b[t][1], o[t][dt]);
            }
            if (dt == 1) {
                mx[0] = scaled_max(n0, scale_log2);
                asm volatile("" : "+v"(mx[0]));  // pinned between the MFMAs
            }
            if (dt == 3) {
                mx[1] = scaled_max(n1, scale_log2);
                asm volatile("" : "+v"(mx[1]));
            }
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            lsum[t] = M::mma(ones, b[t][0], lsum[t]);
            if (HILO) lsum[t] = M::mma(ones, b[t][1], lsum[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }

    // Mask (where a key can lie past a row's last visible key) and lazy rescale
    // of the scores of the sub-tile starting at key0, outside the pipelined parts.
    __device__ inline void mask_rescale(f32x4 (&s0)[2], f32x4 (&s1)[2], bool mask, int32_t key0, int lj,
                                        int32_t last, float scale_log2) {
        if (mask) {
            apply_mask_at(s0, key0, lj, last);
            apply_mask_at(s1, key0, lj, last);
        }
        rescale_if(0, scaled_max(s0, scale_log2));
        rescale_if(1, scaled_max(s1, scale_log2));
    }

    // Sub-tile J of the NS that the wave takes of a stage, STRIDE apart (scores of
    // J in c0 / c1, next scores into n0 / n1).
    template <int J, int NS, int STRIDE>
    __device__ inline void pipelined_subtile(const char* Ks, const char* Vs, int32_t key0, int32_t mask_from,
                                             int32_t last, int lj, float scale_log2, f32x4 (&c0)[2],
                                             f32x4 (&c1)[2], f32x4 (&n0)[2], f32x4 (&n1)[2]) {
        if (J + 1 < NS) {
            const int32_t key1 = key0 + kPairSub * STRIDE * (J + 1);
            u32x4 h0, l0, h1, l1;
            probs_qk(c0, c1, Ks + kPairSub * STRIDE * (J + 1) * D * 2, n0, n1, scale_log2, h0, l0, h1, l1);
            if (key1 + kPairSub > mask_from) {
                apply_mask_at(n0, key1, lj, last);
                apply_mask_at(n1, key1, lj, last);
            }
            float mx[2];
            pv_max(Vs + kPairSub * STRIDE * J * D * 2, h0, l0, h1, l1, n0, n1, scale_log2, mx);
            rescale_if(0, mx[0]);
            rescale_if(1, mx[1]);
        } else {
            v8 vf[DT];
            read_v(Vs + kPairSub * STRIDE * J * D * 2, vf);
            __builtin_amdgcn_sched_barrier(0);
            float x0[2][4], x1[2][4];
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x0[kt][i] = c0[kt][i];
                    x1[kt][i] = c1[kt][i];
                }
            finish_subtile(vf, x0, x1, scale_log2);
        }
    }

    // All kPairSubs sub-tiles of a staged step (or NS of them, STRIDE apart),
    // straight-line code (the accumulators stay in their registers): Ks / Vs the
    // first one's K and V tiles, key0 its first key. `last` is this lane's last
    // visible key (its row's position, and before the chunk's end); keys below
    // mask_from are visible to every row of the tile. Sub-tiles past the chunk's
    // end or the tile's causal limit are masked whole: their probabilities are 0
    // and they add exact zeros (V rows past the chunk's end are zeroed in LDS).
    template <int NS = kPairSubs, int STRIDE = 1>
    __device__ inline void stage_pipelined(const char* Ks, const char* Vs, int32_t key0, int32_t mask_from,
                                           int32_t last, int lj, float scale_log2) {
        static_assert(NS == 2 || NS == 4, "pairs of sub-tiles");
        f32x4 sa0[2], sa1[2], sb0[2], sb1[2];
        {
            v8 kf[DS][2];
            read_k(Ks, kf);
            __builtin_amdgcn_sched_barrier(0);
            qk(0, kf, sa0);
            qk(1, kf, sa1);
            __builtin_amdgcn_sched_barrier(0);
        }
        mask_rescale(sa0, sa1, key0 + kPairSub > mask_from, key0, lj, last, scale_log2);
        pipelined_subtile<0, NS, STRIDE>(Ks, Vs, key0, mask_from, last, lj, scale_log2, sa0, sa1, sb0, sb1);
        pipelined_subtile<1, NS, STRIDE>(Ks, Vs, key0, mask_from, last, lj, scale_log2, sb0, sb1, sa0, sa1);
        if constexpr (NS == 4) {
            pipelined_subtile<2, NS, STRIDE>(Ks, Vs, key0, mask_from, last, lj, scale_log2, sa0, sa1, sb0, sb1);
            pipelined_subtile<3, NS, STRIDE>(Ks, Vs, key0, mask_from, last, lj, scale_log2, sb0, sb1, sa0, sa1);
        }
    }
};

}  // namespace
}  // namespace kvr
