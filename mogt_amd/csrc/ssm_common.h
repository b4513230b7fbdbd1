// Selective state space scan, what its forward, backward and single-token
// kernels share: the problem as the kernels see it, row loads, the step size
// and the gate with their slopes.
//
//   dt_t = delta_t + bias  (softplus of it on request)         per channel
//   h_t  = exp(dt_t A) h_{t-1} + dt_t x_t B_t                  N states per channel
//   y_t  = C_t . h_t + D x_t,   out_t = y_t silu(z_t)
//
// A wave owns 64 channels of one group and NS states of each: a lane is a
// channel, its states sit in registers, and B_t and C_t, which a group's
// channels share, are the same for all lanes: the wave loads them once, spread
// over its lanes, and reads them back from LDS.
#pragma once

#include <type_traits>

#include "common.h"

namespace mogt {

constexpr float SSM_LOG2E = 1.4426950408889634f;
constexpr float SSM_LN2 = 0.6931471805599453f;

struct SsmArgs {
    const void *x, *delta, *z, *B, *C;
    const float *A, *skip, *bias, *h0;
    const void* lengths;
    int64_t xs, xb, ds, db, zs, zb, Bs, Bb, Cs, Cb;   // row and batch strides
    int L, D, N, per, nbk;                            // per: channels of a group; nbk: its 64-channel blocks
    int seg, nseg;                                    // steps of a segment, segments
    int softplus, len64;
};

// Steps of sequence b, within [0, L] whatever the array holds.
__device__ __forceinline__ int ssm_length(const SsmArgs& p, int b) {
    if (!p.lengths) return p.L;
    int64_t n = p.len64 ? static_cast<const int64_t*>(p.lengths)[b] : static_cast<const int32_t*>(p.lengths)[b];
    n = n < 0 ? 0 : n > p.L ? p.L : n;
    return __builtin_amdgcn_readfirstlane(static_cast<int>(n));
}

// States of a wave: all of them up to 16, where the waves of a work-group need
// no exchange; above that 8 each up to 32 and 16 each beyond.  The last wave's
// idle states (where N is not a multiple) read zeros.  Output and sums kernels
// over 8192 steps of 1024 channels, bf16: 12 states in one wave of 16 take 76 us
// and in two of 8 106; 24 states in waves of 8 121 and of 16 161; 32 states 135
// and 148; 40 states 215 in waves of 8 and 198 in waves of 16; 64 states 238 and 213.
constexpr int ssm_states_per_wave(int N) { return N <= 8 || (N > 16 && N <= 32) ? 8 : 16; }
inline int ssm_waves(int N) { return (N + ssm_states_per_wave(N) - 1) / ssm_states_per_wave(N); }

// Calls f with (NS, SPLIT, WHOLE) as integral constants for N states: NS of a
// wave, more than one wave, every wave holds NS of the N.
template <typename F>
void ssm_with_states(int N, F&& f) {
    auto with = [&](auto ns) {
        constexpr int NS = decltype(ns)::value;
        if (N == NS)
            f(ns, std::false_type(), std::true_type());
        else if (N < NS)
            f(ns, std::false_type(), std::false_type());
        else if (N % NS == 0)
            f(ns, std::true_type(), std::true_type());
        else
            f(ns, std::true_type(), std::false_type());
    };
    if (ssm_states_per_wave(N) == 16)
        with(std::integral_constant<int, 16>());
    else
        with(std::integral_constant<int, 8>());
}

// The B (and C) values of U steps, the same for every channel of a wave: each
// lane loads E of them into registers (while the steps before are computed),
// then the wave lays them out in LDS as [U][VALS] floats, from where every lane
// reads them all.  A vector instruction with a scalar operand runs at little
// more than half the rate of one with registers alone (4.3 against 2.5 cycles
// measured, and 2.4 for every scalar instruction that unpacks one), so the rows
// do not come through the scalar unit.  States from `left` on (not WHOLE) and
// steps past cnt (not FULL) are zero.
template <typename TB, int NS, int U, bool WITH_C, bool WHOLE>
struct SsmRows {
    static constexpr int VALS = WITH_C ? 2 * NS : NS;
    static constexpr int ALL = U * VALS, E = ALL < 64 ? 1 : ALL / 64;   // lanes past ALL repeat the first ones
    static_assert((ALL % 64 == 0 || 64 % ALL == 0) && NS % E == 0, "a lane's values lie in one row of B or of C");
    const TB* p;
    int64_t stride;
    int step, first, left;

    __device__ __forceinline__ SsmRows(const TB* B, int64_t Bs, const TB* C, int64_t Cs, int lane, int left_) {
        const int e = lane * E % ALL, k = e % VALS;
        step = e / VALS;
        first = k % NS;
        left = left_;
        stride = WITH_C && k >= NS ? Cs : Bs;
        p = (WITH_C && k >= NS ? C : B) + first + step * stride;
    }
    template <bool FULL>
    __device__ __forceinline__ void load(int64_t t, int cnt, float (&v)[E]) const {   // of the steps from row t on
        const TB* q = p + (t + (FULL ? 0 : min(cnt - 1 - step, 0))) * stride;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            v[i] = IO<TB>::ld(q[WHOLE ? i : min(i, max(left - 1 - first, -first))]);
            if ((!WHOLE && first + i >= left) || (!FULL && step >= cnt)) v[i] = 0.0f;
        }
    }
    static __device__ __forceinline__ void store(float* s, int lane, const float (&v)[E]) {
        Pack<float, E> pk;
#pragma unroll
        for (int i = 0; i < E; ++i) pk.v[i] = v[i];
        *reinterpret_cast<Pack<float, E>*>(s + lane * E % ALL) = pk;
    }
};

// Four values from LDS.
__device__ __forceinline__ void ssm_lds4(const float* s, float (&v)[4]) {
    const Pack<float, 4> q = *reinterpret_cast<const Pack<float, 4>*>(s);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = q.v[k];
}

// LDS accesses of one wave run in order; the compiler has to keep them so.
__device__ __forceinline__ void ssm_wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Element at a byte offset from a pointer that is the same for the whole wave:
// the scalar base and the 32-bit offset go into the memory instruction as they
// are (an index would be added up in 64-bit vector arithmetic first).
template <typename T>
__device__ __forceinline__ T ssm_ld(const T* base, uint32_t off) {
    return *reinterpret_cast<const T*>(reinterpret_cast<const char*>(base) + off);
}
template <typename T>
__device__ __forceinline__ void ssm_st(T* base, uint32_t off, T v) {
    *reinterpret_cast<T*>(reinterpret_cast<char*>(base) + off) = v;
}

// Keeps an offset out of the loop's address arithmetic: the compiler would carry
// base + offset from step to step as one 64-bit vector address per tensor.
__device__ __forceinline__ void ssm_offset(uint32_t& off) { asm volatile("" : "+v"(off)); }

// A lane's channel (byte offset) of the next U rows (of the first cnt where not
// FULL, the last of them again past it); the row pointer moves on by U rows.
template <typename T, int U, bool FULL>
__device__ __forceinline__ void ssm_load_rows(const T*& p, int64_t stride, uint32_t& off, int cnt, T (&v)[U]) {
    const T* q = p;
    ssm_offset(off);
#pragma unroll
    for (int i = 0; i < U; ++i) {
        v[i] = ssm_ld(q, off);
        if (FULL || i + 1 < cnt) q += stride;
    }
    p += U * stride;
}

// Zero past the first cnt of U steps.
template <int U>
__device__ __forceinline__ void ssm_mask(int cnt, float (&v)[U]) {
    if (cnt < U) {
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (i >= cnt) v[i] = 0.0f;
    }
}

// The compiler finishes these before it goes on, and starts no LDS read earlier.
// Left to itself it reads the rows of all steps of a block first and forms the
// decays of all states ahead, which takes the registers of several waves.
__device__ __forceinline__ void ssm_done(float& a) { asm volatile("" : "+v"(a) :: "memory"); }
template <int N>
__device__ __forceinline__ void ssm_done4(float (&v)[N], int n) {
    asm volatile("" : "+v"(v[n]), "+v"(v[n + 1]), "+v"(v[n + 2]), "+v"(v[n + 3]) :: "memory");
}

typedef float ssm_f4 __attribute__((ext_vector_type(4)));

// softplus(v) = max(v, 0) + log(1 + e) with e = exp(-|v|) <= 1: for the rounded
// u = 1 + e the part that u lost, e - (u - 1), is added to log(u), which keeps
// small results (v far below zero) as exact as e is: |v| + 2 half steps, one per
// unit of the rounded product |v| log2(e).  No selects: infinities and NaN pass as
// in the definition.
__device__ __forceinline__ float ssm_softplus(float v) {
    const float e = __builtin_amdgcn_exp2f(fabsf(v) * -SSM_LOG2E);
    const float u = 1.0f + e;
    return fmaxf(v, 0.0f) + fmaf(__builtin_amdgcn_logf(u), SSM_LN2, e - (u - 1.0f));
}

// Step sizes of U steps; zero past the first cnt: such a step leaves the state
// as it is.
template <typename T, int U>
__device__ __forceinline__ void ssm_steps(const T (&raw)[U], float bias, int softplus, int cnt, float (&dt)[U]) {
#pragma unroll
    for (int i = 0; i < U; ++i) dt[i] = IO<T>::ld(raw[i]) + bias;
    if (softplus) {
#pragma unroll
        for (int i = 0; i < U; ++i) dt[i] = ssm_softplus(dt[i]);
    }
    ssm_mask<U>(cnt, dt);
}

__device__ __forceinline__ float ssm_exp2(float v) { return __builtin_amdgcn_exp2f(v); }

// The square root of 2^x.  A segment's decay is 2^(A S) with a sum of step sizes: it
// may lie far outside fp32 (a growing state, A S > 128) where the state that it
// scales is zero or small and the product is in range.  Its root is kept within
// [2^-126, 2^127] and applied twice: zero stays zero and infinity infinity, and
// what a normal number times a decay beyond that gives is infinite or below 2^-124.
__device__ __forceinline__ float ssm_root(float x) {
    return ssm_exp2(__builtin_amdgcn_fmed3f(0.5f * x, -126.0f, 127.0f));
}
// r^2 h + v
__device__ __forceinline__ float ssm_fold(float r, float h, float v) { return fmaf(r, r * h, v); }

// What enters each segment, of one state of 64 channels: out[k] = h, then
// h = 2^(A S[k]) h + part[k], over the segments in order (BACK: from the last
// on); out may be part itself.  The first `formed` in that order have S and part.
// The waves take 16 neighbouring segments each, fold them (one decay for the sum
// of their S), and start from what the folds of the waves before them leave: a
// chain over all segments in one thread waited for memory every 32 of them.
constexpr int SSM_CARRY_U = 16, SSM_CARRY_WAVES = 16;
inline int ssm_carry_threads(int nseg) {
    const int waves = (nseg + SSM_CARRY_U - 1) / SSM_CARRY_U;
    return 64 * (waves < 1 ? 1 : waves > SSM_CARRY_WAVES ? SSM_CARRY_WAVES : waves);
}

template <bool BACK>
__device__ __forceinline__ void ssm_carry(float A, float h, const float* S, int64_t S_stride, const float* part,
                                          float* out, int64_t stride, int nseg, int formed, bool valid) {
    constexpr int U = SSM_CARRY_U;
    __shared__ float s_fold[2][SSM_CARRY_WAVES][2][64];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int W = __builtin_amdgcn_readfirstlane(blockDim.x >> 6);
    float Sv[U], e[U];
    auto at = [&](int j) { return static_cast<int64_t>(BACK ? nseg - 1 - j : j); };
    auto load = [&](int j) {
#pragma unroll
        for (int i = 0; i < U; ++i) Sv[i] = e[i] = 0.0f;
        if (j >= formed) return;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t k = at(min(j + i, formed - 1));
            Sv[i] = S[k * S_stride];
            e[i] = part[k * stride];
        }
    };
    load(w * U);
    for (int j0 = 0, buf = 0; j0 < nseg; j0 += W * U, buf ^= 1) {
        const int j = j0 + w * U;
        float a[U], v[U], sum = 0.0f, f = 0.0f;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            a[i] = ssm_root(Sv[i] * A);
            v[i] = e[i];
            sum += Sv[i];
            f = ssm_fold(a[i], f, v[i]);
        }
        if (j0 + W * U < nseg) load(j + W * U);
        s_fold[buf][w][0][lane] = ssm_root(sum * A);
        s_fold[buf][w][1][lane] = f;
        __syncthreads();   // a buffer is written again past the next one, when its readers are done
        float g = h;
        for (int m = 0; m < W; ++m) {
            if (m == w) g = h;
            h = ssm_fold(s_fold[buf][m][0][lane], h, s_fold[buf][m][1][lane]);
        }
        if (!valid) continue;
#pragma unroll
        for (int i = 0; i < U; ++i) {
            if (j + i >= nseg) break;
            out[at(j + i) * stride] = g;
            g = ssm_fold(a[i], g, v[i]);
        }
    }
}

}  // namespace mogt
