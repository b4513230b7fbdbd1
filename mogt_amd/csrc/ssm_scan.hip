// Selective state space scan, forward, and its single-token form (ssm_common.h
// has the recurrence).
//
// A sequence is cut into segments of `seg` steps, one wave each per 64 channels
// and 16 states:
//   sums    each segment but the last scans from a zero state and leaves its
//           end state and its sum of step sizes: the segment's decay is
//           exp(A sum dt), one exponential per state and segment.
//   out     each segment folds the sums of the segments before it (in order,
//           so results do not depend on timing) into its start state, scans
//           again and writes the outputs.
// With one segment only the second launch runs.  More than 16 states: the
// waves of a work-group take 16 each and add their parts of y through LDS.
//
// Bound: the vector unit.  A state and step take one exponential and about
// five further fp32 instructions, and the two launches form the exponentials
// twice; holding them (N fp32 values per element of x) would cost N/4 times
// the bytes of every input together.
#include <type_traits>

#include "ssm_common.h"

namespace mogt {

constexpr int SSM_U = 8;   // steps whose rows are loaded together

struct SsmFwd {
    SsmArgs a;
    void* out;          // [B, L, D]
    float* state;       // [B, D, N] or null
    float* carries;     // [B, nseg, N, D] or null: the state entering each segment
    float* part_h;      // [B, nseg, N, D]
    float* part_s;      // [B, nseg, D]
};

template <typename T, typename TB, int NS, bool SPLIT>
__global__ __launch_bounds__(SPLIT ? 512 : 64) void ssm_sums_kernel(SsmFwd f) {
    const SsmArgs& p = f.a;
    const int lane = threadIdx.x & 63;
    const int n0 = SPLIT ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * NS : 0;
    const int g = blockIdx.x / p.nbk;
    const int ci = (blockIdx.x - g * p.nbk) * 64 + lane;
    const bool valid = ci < p.per;
    const int c = g * p.per + (valid ? ci : p.per - 1);
    const int seg = blockIdx.y, b = blockIdx.z;
    const int t0 = seg * p.seg;
    const int te = min(t0 + p.seg, ssm_length(p, b));

    float A[NS], h[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        A[n] = n0 + n < p.N ? p.A[static_cast<int64_t>(c) * p.N + n0 + n] * SSM_LOG2E : 0.0f;
        h[n] = 0.0f;
    }
    const float bias = p.bias ? p.bias[c] : 0.0f;
    const T* px = static_cast<const T*>(p.x) + b * p.xb;
    const T* pd = static_cast<const T*>(p.delta) + b * p.db;
    const TB* pB = static_cast<const TB*>(p.B) + b * p.Bb + static_cast<int64_t>(g) * p.N;
    float S = 0.0f;
    for (int t = t0; t < te; t += SSM_U) {
        T xr[SSM_U], dr[SSM_U];
#pragma unroll
        for (int i = 0; i < SSM_U; ++i) {
            const int64_t tt = min(t + i, te - 1);
            xr[i] = (px + tt * p.xs)[c];
            dr[i] = (pd + tt * p.ds)[c];
        }
#pragma unroll
        for (int i = 0; i < SSM_U; ++i) {
            if (t + i >= te) break;
            float Bv[NS];
            ssm_row<TB, NS>(pB + (t + i) * p.Bs, n0, p.N, Bv);
            float dt = IO<T>::ld(dr[i]) + bias;
            if (p.softplus) dt = ssm_softplus(dt);
            const float w = dt * IO<T>::ld(xr[i]);
            S += dt;
#pragma unroll
            for (int n = 0; n < NS; ++n) h[n] = fmaf(ssm_exp2(dt * A[n]), h[n], w * Bv[n]);
        }
    }
    if (!valid) return;
    const int64_t row = static_cast<int64_t>(b) * p.nseg + seg;
    if (n0 == 0) f.part_s[row * p.D + c] = S;
#pragma unroll
    for (int n = 0; n < NS; ++n)
        if (n0 + n < p.N) f.part_h[(row * p.N + n0 + n) * p.D + c] = h[n];
}

template <typename T, typename TB, int NS, bool Z, bool SPLIT>
__global__ __launch_bounds__(SPLIT ? 512 : 64) void ssm_out_kernel(SsmFwd f) {
    extern __shared__ float s_y[];   // SPLIT: [2][waves][SSM_U][64]
    const SsmArgs& p = f.a;
    const int lane = threadIdx.x & 63;
    const int nb = SPLIT ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int NB = SPLIT ? __builtin_amdgcn_readfirstlane(blockDim.x >> 6) : 1;
    const int n0 = nb * NS;
    const int g = blockIdx.x / p.nbk;
    const int ci = (blockIdx.x - g * p.nbk) * 64 + lane;
    const bool valid = ci < p.per;
    const int c = g * p.per + (valid ? ci : p.per - 1);
    const int seg = blockIdx.y, b = blockIdx.z;
    const int len = ssm_length(p, b);
    const int t0 = seg * p.seg, t1 = min(t0 + p.seg, p.L);
    const int te = min(t1, len);

    float A[NS], h[NS];
    const int64_t cn = (static_cast<int64_t>(b) * p.D + c) * p.N + n0;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const bool in = n0 + n < p.N;
        A[n] = in ? p.A[static_cast<int64_t>(c) * p.N + n0 + n] * SSM_LOG2E : 0.0f;
        h[n] = in && p.h0 ? p.h0[cn + n] : 0.0f;
    }
    // the segments before this one; those past the sequence's end hold no step
    const int64_t row0 = static_cast<int64_t>(b) * p.nseg;
    for (int j = 0; j < seg && j * p.seg < len; ++j) {
        const float S = f.part_s[(row0 + j) * p.D + c];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const float e = n0 + n < p.N ? f.part_h[((row0 + j) * p.N + n0 + n) * p.D + c] : 0.0f;
            h[n] = fmaf(ssm_exp2(S * A[n]), h[n], e);
        }
    }
    if (f.carries && valid) {
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (n0 + n < p.N) f.carries[((row0 + seg) * p.N + n0 + n) * p.D + c] = h[n];
    }
    const float bias = p.bias ? p.bias[c] : 0.0f;
    const float skip = p.skip ? p.skip[c] : 0.0f;
    const T* px = static_cast<const T*>(p.x) + b * p.xb;
    const T* pd = static_cast<const T*>(p.delta) + b * p.db;
    const T* pz = static_cast<const T*>(p.z) + b * p.zb;
    const TB* pB = static_cast<const TB*>(p.B) + b * p.Bb + static_cast<int64_t>(g) * p.N;
    const TB* pC = static_cast<const TB*>(p.C) + b * p.Cb + static_cast<int64_t>(g) * p.N;
    T* po = static_cast<T*>(f.out) + static_cast<int64_t>(b) * p.L * p.D;
    int buf = 0;
    for (int t = t0; t < te; t += SSM_U) {
        T xr[SSM_U], dr[SSM_U], zr[SSM_U];
#pragma unroll
        for (int i = 0; i < SSM_U; ++i) {
            const int64_t tt = min(t + i, te - 1);
            xr[i] = (px + tt * p.xs)[c];
            dr[i] = (pd + tt * p.ds)[c];
            if constexpr (Z) zr[i] = (pz + tt * p.zs)[c];
        }
        auto finish = [&](int i, float y) {
            y = fmaf(skip, IO<T>::ld(xr[i]), y);
            if constexpr (Z) {
                const float z = IO<T>::ld(zr[i]);
                y *= z * sigmoid_hw(z);
            }
            if (valid) (po + static_cast<int64_t>(t + i) * p.D)[c] = IO<T>::st(y);
        };
#pragma unroll
        for (int i = 0; i < SSM_U; ++i) {
            if (t + i >= te) break;
            float Bv[NS], Cv[NS];
            ssm_row<TB, NS>(pB + (t + i) * p.Bs, n0, p.N, Bv);
            ssm_row<TB, NS>(pC + (t + i) * p.Cs, n0, p.N, Cv);
            float dt = IO<T>::ld(dr[i]) + bias;
            if (p.softplus) dt = ssm_softplus(dt);
            const float w = dt * IO<T>::ld(xr[i]);
            float y = 0.0f;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                h[n] = fmaf(ssm_exp2(dt * A[n]), h[n], w * Bv[n]);
                y = fmaf(Cv[n], h[n], y);
            }
            if constexpr (SPLIT)
                s_y[((buf * NB + nb) * SSM_U + i) * 64 + lane] = y;
            else
                finish(i, y);
        }
        if constexpr (SPLIT) {
            // two buffers: a wave writes one again only past the next barrier,
            // which every wave reaches after its reads of it
            __syncthreads();
#pragma unroll
            for (int i = 0; i < SSM_U; ++i) {
                if (t + i >= te) break;
                if (i % NB != nb) continue;
                float y = 0.0f;
                for (int k = 0; k < NB; ++k) y += s_y[((buf * NB + k) * SSM_U + i) * 64 + lane];
                finish(i, y);
            }
            buf ^= 1;
        }
    }
    if (nb == 0 && valid)   // rows past the sequence's length
        for (int t = max(t0, te); t < t1; ++t) (po + static_cast<int64_t>(t) * p.D)[c] = IO<T>::st(0.0f);
    if (f.state && seg == p.nseg - 1 && valid) {
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (n0 + n < p.N) f.state[cn + n] = h[n];
    }
}

// ---------------------------------------------------------------------------
// single token: four lanes per channel, each every fourth state
// ---------------------------------------------------------------------------
struct SsmStep {
    SsmArgs a;
    float* state;   // [B, D, N], updated
    void* out;      // [B, D]
    int batch;
};

template <typename T, typename TB>
__global__ __launch_bounds__(256) void ssm_step_kernel(SsmStep f) {
    const SsmArgs& p = f.a;
    const int q = threadIdx.x & 3;
    const int ci = blockIdx.x * 64 + (threadIdx.x >> 2);
    if (ci >= p.D) return;   // whole quads
    const int b = blockIdx.y;
    const int g = ci / p.per;
    const float x = IO<T>::ld((static_cast<const T*>(p.x) + b * p.xb)[ci]);
    float dt = IO<T>::ld((static_cast<const T*>(p.delta) + b * p.db)[ci]) + (p.bias ? p.bias[ci] : 0.0f);
    if (p.softplus) dt = ssm_softplus(dt);
    const float w = dt * x;
    float* h = f.state + (static_cast<int64_t>(b) * p.D + ci) * p.N;
    const float* A = p.A + static_cast<int64_t>(ci) * p.N;
    const TB* B = static_cast<const TB*>(p.B) + b * p.Bb + static_cast<int64_t>(g) * p.N;
    const TB* C = static_cast<const TB*>(p.C) + b * p.Cb + static_cast<int64_t>(g) * p.N;
    float y = 0.0f;
    for (int n = q; n < p.N; n += 4) {
        const float v = fmaf(ssm_exp2(dt * A[n] * SSM_LOG2E), h[n], w * IO<TB>::ld(B[n]));
        h[n] = v;
        y = fmaf(IO<TB>::ld(C[n]), v, y);
    }
    y += __shfl_xor(y, 1, 64);
    y += __shfl_xor(y, 2, 64);
    if (q != 0) return;
    y = fmaf(p.skip ? p.skip[ci] : 0.0f, x, y);
    if (p.z) {
        const float z = IO<T>::ld((static_cast<const T*>(p.z) + b * p.zb)[ci]);
        y *= z * sigmoid_hw(z);
    }
    (static_cast<T*>(f.out) + static_cast<int64_t>(b) * p.D)[ci] = IO<T>::st(y);
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int ssm_args(const mogt_ssm_problem* q, bool step, SsmArgs& a) {
    if (!q) return set_error(MOGT_E_INVALID, "null problem");
    if (q->batch < 0 || q->length < 0 || q->channels < 0 || q->states < 1 || q->groups < 1)
        return set_error(MOGT_E_INVALID, "bad sizes: batch %lld, length %lld, channels %lld, states %lld, groups %lld",
                         (long long)q->batch, (long long)q->length, (long long)q->channels, (long long)q->states,
                         (long long)q->groups);
    if (q->states > MOGT_SSM_MAX_STATES)
        return set_error(MOGT_E_INVALID, "%lld states: at most %d", (long long)q->states, MOGT_SSM_MAX_STATES);
    if (q->channels % q->groups != 0)
        return set_error(MOGT_E_INVALID, "%lld channels do not divide into %lld groups", (long long)q->channels,
                         (long long)q->groups);
    const bool f32 = q->io_dtype == MOGT_F32 && q->bc_dtype == MOGT_F32;
    const bool bf16 = q->io_dtype == MOGT_BF16 && (q->bc_dtype == MOGT_F32 || q->bc_dtype == MOGT_BF16);
    if (!f32 && !bf16) return set_error(MOGT_E_INVALID, "dtype codes %d, %d not supported", q->io_dtype, q->bc_dtype);
    if (q->lengths && q->lengths_bytes != 4 && q->lengths_bytes != 8)
        return set_error(MOGT_E_INVALID, "lengths of 4 or 8 bytes expected, got %d", q->lengths_bytes);
    // 32-bit steps and channels in the kernels; batch and segments are grid dimensions
    if (q->length >= (1ll << 30) || q->channels >= (1ll << 24) || q->batch > 65535)
        return set_error(MOGT_E_INVALID, "batch up to 65535, length below 2^30, channels below 2^24 expected");
    if (q->batch == 0 || q->channels == 0) return MOGT_OK;
    if (q->length > 0) {
        if (!q->x || !q->delta || !q->A || !q->B || !q->C) return set_error(MOGT_E_INVALID, "null input pointer");
        if (q->bc_dtype == MOGT_BF16 && !step) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(q->B) | reinterpret_cast<uintptr_t>(q->C);
            if ((at & 3) || ((q->B_row | q->B_batch | q->C_row | q->C_batch | q->states) & 1))
                return set_error(MOGT_E_INVALID, "bf16 B and C rows: 4-byte alignment and an even state count expected");
        }
    }
    a.x = q->x; a.delta = q->delta; a.z = q->z; a.B = q->B; a.C = q->C;
    a.A = q->A; a.skip = q->D; a.bias = q->delta_bias; a.h0 = q->initial_state;
    a.lengths = q->lengths;
    a.xs = q->x_row; a.xb = q->x_batch; a.ds = q->delta_row; a.db = q->delta_batch;
    a.zs = q->z_row; a.zb = q->z_batch;
    a.Bs = q->B_row; a.Bb = q->B_batch; a.Cs = q->C_row; a.Cb = q->C_batch;
    a.L = static_cast<int>(q->length);
    a.D = static_cast<int>(q->channels);
    a.N = static_cast<int>(q->states);
    a.per = static_cast<int>(q->channels / q->groups);
    a.nbk = (a.per + 63) / 64;
    a.softplus = q->softplus;
    a.len64 = q->lengths_bytes == 8;
    a.seg = a.nseg = 1;
    if (!step) {
        if (q->segment < 8 || q->segment % 8 != 0 || q->segment >= (1ll << 30))
            return set_error(MOGT_E_INVALID, "segment of %lld steps: a positive multiple of 8 expected",
                             (long long)q->segment);
        const int64_t nseg = (q->length + q->segment - 1) / q->segment;
        if (nseg > 65535) return set_error(MOGT_E_INVALID, "%lld segments: at most 65535", (long long)nseg);
        a.seg = static_cast<int>(q->segment);
        a.nseg = nseg > 0 ? static_cast<int>(nseg) : 1;
    }
    return MOGT_OK;
}

namespace {

template <typename T, typename TB, int NS, bool SPLIT>
int fwd_launch(const SsmFwd& f, int batch, hipStream_t st) {
    const SsmArgs& a = f.a;
    const int waves = SPLIT ? (a.N + NS - 1) / NS : 1;
    const int blocks = a.D / a.per * a.nbk;
    if (a.nseg > 1)
        ssm_sums_kernel<T, TB, NS, SPLIT><<<dim3(blocks, a.nseg - 1, batch), 64 * waves, 0, st>>>(f);
    const size_t lds = SPLIT ? sizeof(float) * 2 * waves * SSM_U * 64 : 0;
    const dim3 grid(blocks, a.nseg, batch);
    if (a.z)
        ssm_out_kernel<T, TB, NS, true, SPLIT><<<grid, 64 * waves, lds, st>>>(f);
    else
        ssm_out_kernel<T, TB, NS, false, SPLIT><<<grid, 64 * waves, lds, st>>>(f);
    return check_launch("mogt_ssm_scan_fwd");
}

template <typename T, typename TB>
int fwd_states(const SsmFwd& f, int batch, hipStream_t st) {
    if (f.a.N <= 8) return fwd_launch<T, TB, 8, false>(f, batch, st);
    if (f.a.N <= 16) return fwd_launch<T, TB, 16, false>(f, batch, st);
    return fwd_launch<T, TB, 16, true>(f, batch, st);
}

}  // namespace
}  // namespace mogt

using namespace mogt;

extern "C" size_t mogt_ssm_scan_workspace_bytes(int64_t batch, int64_t length, int64_t channels, int64_t states,
                                                int64_t segment) {
    if (batch <= 0 || channels <= 0 || states <= 0 || segment <= 0 || length <= segment) return 0;
    const int64_t nseg = (length + segment - 1) / segment;
    return static_cast<size_t>(batch * nseg * channels * (states + 1)) * sizeof(float);
}

extern "C" int mogt_ssm_scan_fwd(const mogt_ssm_problem* q, void* out, float* final_state, float* carries,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    SsmFwd f{};
    if (const int rc = ssm_args(q, false, f.a)) return rc;
    if (q->batch == 0 || q->channels == 0 || (q->length == 0 && !final_state)) return MOGT_OK;
    if (q->length > 0 && !out) return set_error(MOGT_E_INVALID, "null output pointer");
    const size_t need = mogt_ssm_scan_workspace_bytes(q->batch, q->length, q->channels, q->states, q->segment);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return set_error(MOGT_E_WORKSPACE, "workspace of %zu bytes expected, got %zu", need,
                         workspace ? workspace_bytes : 0);
    if (!f.a.A) return set_error(MOGT_E_INVALID, "null input pointer");
    f.out = out;
    f.state = final_state;
    f.carries = carries;
    f.part_h = static_cast<float*>(workspace);
    f.part_s = f.part_h + q->batch * f.a.nseg * q->channels * q->states;
    const int batch = static_cast<int>(q->batch);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q->io_dtype == MOGT_F32) return fwd_states<float, float>(f, batch, st);
    if (q->bc_dtype == MOGT_F32) return fwd_states<bf16_t, float>(f, batch, st);
    return fwd_states<bf16_t, bf16_t>(f, batch, st);
}

extern "C" int mogt_ssm_step(const mogt_ssm_problem* q, float* state, void* out, void* stream) {
    clear_error();
    SsmStep f{};
    if (const int rc = ssm_args(q, true, f.a)) return rc;
    if (q->length != 1) return set_error(MOGT_E_INVALID, "a step takes one token, length is %lld", (long long)q->length);
    if (q->batch == 0 || q->channels == 0) return MOGT_OK;
    if (!state || !out) return set_error(MOGT_E_INVALID, "null state or output pointer");
    f.state = state;
    f.out = out;
    const dim3 grid((f.a.D + 63) / 64, static_cast<unsigned>(q->batch));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q->io_dtype == MOGT_F32)
        ssm_step_kernel<float, float><<<grid, 256, 0, st>>>(f);
    else if (q->bc_dtype == MOGT_F32)
        ssm_step_kernel<bf16_t, float><<<grid, 256, 0, st>>>(f);
    else
        ssm_step_kernel<bf16_t, bf16_t><<<grid, 256, 0, st>>>(f);
    return check_launch("mogt_ssm_step");
}
