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
// channels share, are the same for all lanes: they come through the scalar
// loads and feed the vector instructions as scalar operands.
#pragma once

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

// NS consecutive values of a B or C row from state n0, the same for every
// lane; states past N read as zero.  Rows are in constant memory for the
// launch, so the loads are scalar.  bf16 rows are 4-byte aligned and N is even
// (checked on the host): a 32-bit word holds two states.
template <typename TB, int NS>
__device__ __forceinline__ void ssm_row(const TB* row, int n0, int N, float (&v)[NS]) {
    if constexpr (sizeof(TB) == 4) {
        typedef const __attribute__((address_space(4))) float* cptr;
        const cptr q = (cptr)reinterpret_cast<uintptr_t>(row + n0);
        if (N - n0 >= NS) {
#pragma unroll
            for (int i = 0; i < NS; ++i) v[i] = q[i];
        } else {
#pragma unroll
            for (int i = 0; i < NS; ++i) v[i] = n0 + i < N ? q[i] : 0.0f;
        }
    } else {
        typedef const __attribute__((address_space(4))) uint32_t* cptr;
        const cptr q = (cptr)reinterpret_cast<uintptr_t>(row + n0);
        uint32_t w[NS / 2];
        if (N - n0 >= NS) {
#pragma unroll
            for (int i = 0; i < NS / 2; ++i) w[i] = q[i];
        } else {
#pragma unroll
            for (int i = 0; i < NS / 2; ++i) w[i] = n0 + 2 * i < N ? q[i] : 0u;
        }
#pragma unroll
        for (int i = 0; i < NS / 2; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

// softplus(v) = log(1 + e^v), v itself past 20 (there the two agree in fp32).
// log(1 + e) / e for the rounded u = 1 + e is log(u) / (u - 1) to fp32
// accuracy, which keeps the small step sizes (e of 2^-10 and below) exact to a
// few ulp.
__device__ __forceinline__ float ssm_softplus(float v) {
    const float e = __builtin_amdgcn_exp2f(v * SSM_LOG2E);
    const float u = 1.0f + e, d = u - 1.0f;
    const float s = __builtin_amdgcn_logf(u) * SSM_LN2 * e * __builtin_amdgcn_rcpf(d);
    return v > 20.0f ? v : d == 0.0f ? e : s;
}

__device__ __forceinline__ float ssm_exp2(float v) { return __builtin_amdgcn_exp2f(v); }

}  // namespace mogt
