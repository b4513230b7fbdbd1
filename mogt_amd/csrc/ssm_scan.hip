// Selective state space scan, forward, and its single-token form (ssm_common.h
// has the recurrence).
//
// A sequence is cut into segments of `seg` steps, one wave each per 64 channels
// and 16 states:
//   sums    each segment but the last scans from a zero state and leaves its
//           end state and its sum of step sizes: the segment's decay is
//           exp(A sum dt), one exponential per state and segment.
//   carry   the segments' start states, in order;
//   out     each segment scans again from its start state and writes the
//           outputs.
// With one segment only the last launch runs.  More than 16 states: the waves of
// a work-group take 8 or 16 each and add their parts of y through LDS.
//
// Bound: instruction issue on the vector unit.  A state and step take a product,
// an exponential, a product and a multiply-add, and one more multiply-add for the
// output; the two launches form the exponentials twice (holding them, N fp32
// values per element of x, would cost N/4 times the bytes of every input
// together).  32768 steps of 2048 channels with 16 states, bf16: sums 194 us,
// carry 13, out 257, with 5.0 and 6.8 vector instructions per state and step (4
// and 5 of them the above), which at 4 cycles each and 8 an exponential add up to
// 94 % of the cycles; the bytes alone would take 103.  B and C as scalar operands, two channels a
// lane, the matrix unit for w B, and one launch of longer work-groups for short
// sequences were all slower.
#include <type_traits>

#include "ssm_common.h"

namespace mogt {

constexpr int SSM_U = 8;   // steps whose rows are loaded together

struct SsmFwd {
    SsmArgs a;
    void* out;          // [B, L, D]
    float* state;       // [B, D, N] or null
    float* carries;     // [B, nseg, N, D]: the state entering each segment; null if not wanted and not needed
    float* part_h;      // [B, nseg, N, D]
    float* part_s;      // [B, nseg, D]
};

// What a wave works on: its lane's channel, its states, its steps t0 .. te - 1 of
// sequence b.  Idle lanes (valid false) repeat the group's last channel.
template <typename T, typename TB, int NS, bool WHOLE>
struct SsmWave {
    const SsmArgs& p;
    int lane, n0, left, g, c, b, t0, t1, te, len;
    uint32_t off;
    bool valid;
    float A[NS], bias;

    __device__ __forceinline__ SsmWave(const SsmArgs& p_, int n0_, int seg)
        : p(p_), lane(threadIdx.x & 63), n0(n0_), left(p_.N - n0_), b(blockIdx.z) {
        g = blockIdx.x / p.nbk;
        const int ci = (blockIdx.x - g * p.nbk) * 64 + lane;
        valid = ci < p.per;
        c = g * p.per + (valid ? ci : p.per - 1);
        off = static_cast<uint32_t>(c) * static_cast<uint32_t>(sizeof(T));
        len = ssm_length(p, b);
        t0 = seg * p.seg;
        t1 = min(t0 + p.seg, p.L);
        te = min(t1, len);
        bias = p.bias ? p.bias[c] : 0.0f;
#pragma unroll
        for (int n = 0; n < NS; ++n)
            A[n] = WHOLE || n < left ? p.A[static_cast<int64_t>(c) * p.N + n0 + n] * SSM_LOG2E : 0.0f;
    }
    __device__ __forceinline__ const T* rows(const void* q, int64_t stride, int64_t batch) const {
        return static_cast<const T*>(q) + b * batch + t0 * stride;
    }
    __device__ __forceinline__ const TB* states(const void* q, int64_t batch) const {
        return static_cast<const TB*>(q) + b * batch + static_cast<int64_t>(g) * p.N + n0;
    }

    // h from the state it holds through the steps; returns the sum of step sizes.
    // lds: SsmRows<.., false, ..>::ALL floats of the wave's own.
    __device__ __forceinline__ float sums(float* lds, float (&h)[NS]) {
        constexpr int U = SSM_U;
        typedef SsmRows<TB, NS, U, false, WHOLE> Rows;
        const T *px = rows(p.x, p.xs, p.xb), *pd = rows(p.delta, p.ds, p.db);
        const TB* pB = states(p.B, p.Bb);
        const Rows bc(pB, p.Bs, pB, p.Bs, lane, left);
        T xr[U], dr[U];
        float rv[Rows::E], S = 0.0f;
        auto load = [&](int t) {   // the rows of the block at t
            const int cnt = te - t;
            if (cnt >= U) {
                ssm_load_rows<T, U, true>(px, p.xs, off, U, xr);
                ssm_load_rows<T, U, true>(pd, p.ds, off, U, dr);
                bc.template load<true>(t, U, rv);
            } else if (cnt > 0) {
                ssm_load_rows<T, U, false>(px, p.xs, off, cnt, xr);
                ssm_load_rows<T, U, false>(pd, p.ds, off, cnt, dr);
                bc.template load<false>(t, cnt, rv);
            }
        };
        load(t0);
        for (int t = t0; t < te; t += U) {
            const int cnt = te - t;
            float dt[U], w[U];
            ssm_steps<T, U>(dr, bias, p.softplus, cnt, dt);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                w[i] = dt[i] * IO<T>::ld(xr[i]);
                S += dt[i];
            }
            ssm_mask<U>(cnt, w);
            Rows::store(lds, lane, rv);
            ssm_wave_sync();
            load(t + U);
            float Bn[4];   // the next four values of B, read ahead
            ssm_lds4(lds, Bn);
#pragma unroll
            for (int i = 0; i < U; ++i) {
#pragma unroll
                for (int m = 0; m < NS; m += 4) {
                    const float Bv[4] = {Bn[0], Bn[1], Bn[2], Bn[3]};
                    if (i * NS + m + 4 < U * NS) ssm_lds4(lds + i * NS + m + 4, Bn);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        h[m + e] = fmaf(ssm_exp2(dt[i] * A[m + e]), h[m + e], w[i] * Bv[e]);
                    ssm_done4(h, m);
                }
            }
            ssm_wave_sync();
        }
        return S;
    }

    // h through the steps, their outputs written.  lds: SsmRows<.., true, ..>::ALL
    // floats of the wave's own; SPLIT: s_y [2][8][U][64] of the work-group's, whose
    // NB waves (this one the nb-th) hold the channel's other states.
    template <bool Z, bool SPLIT>
    __device__ __forceinline__ void outputs(void* out, float* lds, float* s_y, int nb, int NB, float (&h)[NS]) {
        constexpr int U = SSM_U;
        typedef SsmRows<TB, NS, U, true, WHOLE> Rows;
        const float skip = p.skip ? p.skip[c] : 0.0f;
        const T *px = rows(p.x, p.xs, p.xb), *pd = rows(p.delta, p.ds, p.db), *pz = rows(p.z, p.zs, p.zb);
        const Rows bc(states(p.B, p.Bb), p.Bs, states(p.C, p.Cb), p.Cs, lane, left);
        T* po = static_cast<T*>(out) + (static_cast<int64_t>(b) * p.L + t0) * p.D;
        T xr[U], dr[U], zr[U];
        float rv[Rows::E];
        auto load = [&](int t) {   // the rows of the block at t
            const int cnt = te - t;
            if (cnt >= U) {
                ssm_load_rows<T, U, true>(px, p.xs, off, U, xr);
                ssm_load_rows<T, U, true>(pd, p.ds, off, U, dr);
                if constexpr (Z) ssm_load_rows<T, U, true>(pz, p.zs, off, U, zr);
                bc.template load<true>(t, U, rv);
            } else if (cnt > 0) {
                ssm_load_rows<T, U, false>(px, p.xs, off, cnt, xr);
                ssm_load_rows<T, U, false>(pd, p.ds, off, cnt, dr);
                if constexpr (Z) ssm_load_rows<T, U, false>(pz, p.zs, off, cnt, zr);
                bc.template load<false>(t, cnt, rv);
            }
        };
        int buf = 0;
        load(t0);
        for (int t = t0; t < te; t += U, po += static_cast<int64_t>(U) * p.D) {
            const int cnt = te - t;
            // what a step needs of its channel: step size, written value, and the
            // factors of the output, out = gate y + gx
            float dt[U], w[U], gate[U], gx[U];
            ssm_steps<T, U>(dr, bias, p.softplus, cnt, dt);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                const float x = IO<T>::ld(xr[i]);
                w[i] = dt[i] * x;
                gate[i] = 1.0f;
                gx[i] = skip * x;
                if (Z && (!SPLIT || i % NB == nb)) {
                    const float z = IO<T>::ld(zr[i]);
                    gate[i] = z * sigmoid_hw(z);
                    gx[i] *= gate[i];
                }
            }
            ssm_mask<U>(cnt, w);
            Rows::store(lds, lane, rv);
            ssm_wave_sync();
            load(t + U);
            float Bn[4], Cn[4];   // the next four values of B and C, read ahead
            ssm_lds4(lds, Bn);
            ssm_lds4(lds + NS, Cn);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                float y = 0.0f;
#pragma unroll
                for (int m = 0; m < NS; m += 4) {
                    const float Bv[4] = {Bn[0], Bn[1], Bn[2], Bn[3]}, Cv[4] = {Cn[0], Cn[1], Cn[2], Cn[3]};
                    if (i * NS + m + 4 < U * NS) {
                        const int at = m + 4 < NS ? i * Rows::VALS + m + 4 : (i + 1) * Rows::VALS;
                        ssm_lds4(lds + at, Bn);
                        ssm_lds4(lds + at + NS, Cn);
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        h[m + e] = fmaf(ssm_exp2(dt[i] * A[m + e]), h[m + e], w[i] * Bv[e]);
                        y = fmaf(Cv[e], h[m + e], y);
                    }
                    ssm_done4(h, m);
                    ssm_done(y);
                }
                if constexpr (SPLIT)
                    s_y[((buf * 8 + nb) * U + i) * 64 + lane] = y;
                else
                    gx[i] = fmaf(gate[i], y, gx[i]);
            }
            if constexpr (SPLIT) {
                // two buffers: a wave writes one again only past the next barrier,
                // which every wave reaches after its reads of it
                __syncthreads();
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    if (i % NB != nb || i >= cnt) continue;
                    float y = 0.0f;
                    for (int m = 0; m < NB; ++m) y += s_y[((buf * 8 + m) * U + i) * 64 + lane];
                    if (valid) ssm_st<T>(po + static_cast<int64_t>(i) * p.D, off, IO<T>::st(fmaf(gate[i], y, gx[i])));
                }
                buf ^= 1;
            } else {
                ssm_wave_sync();
                if (valid) {
                    T* q = po;
                    ssm_offset(off);
                    if (cnt >= U) {
#pragma unroll
                        for (int i = 0; i < U; ++i, q += p.D) ssm_st<T>(q, off, IO<T>::st(gx[i]));
                    } else {
#pragma unroll
                        for (int i = 0; i < U; ++i, q += p.D)
                            if (i < cnt) ssm_st<T>(q, off, IO<T>::st(gx[i]));
                    }
                }
            }
        }
        if (nb == 0 && valid) {   // rows past the sequence's length
            T* pt = static_cast<T*>(out) + static_cast<int64_t>(b) * p.L * p.D + c;
            for (int t = max(t0, te); t < t1; ++t) pt[static_cast<int64_t>(t) * p.D] = IO<T>::st(0.0f);
        }
    }

    // The wave's states of a [B, D, N] tensor, and of segment seg of a
    // [B, nseg, N, D] one.
    __device__ __forceinline__ void read_state(const float* q, float (&h)[NS]) const {
        const int64_t cn = (static_cast<int64_t>(b) * p.D + c) * p.N + n0;
#pragma unroll
        for (int n = 0; n < NS; ++n) h[n] = q && (WHOLE || n < left) ? q[cn + n] : 0.0f;
    }
    __device__ __forceinline__ void write_state(float* q, const float (&h)[NS]) const {
        if (!q || !valid) return;
        const int64_t cn = (static_cast<int64_t>(b) * p.D + c) * p.N + n0;
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (WHOLE || n < left) q[cn + n] = h[n];
    }
    __device__ __forceinline__ int64_t segment_at(int seg) const {
        return ((static_cast<int64_t>(b) * p.nseg + seg) * p.N + n0) * p.D + c;
    }
    __device__ __forceinline__ void write_segment(float* q, int seg, const float (&h)[NS]) const {
        if (!q || !valid) return;
        q += segment_at(seg);
#pragma unroll
        for (int n = 0; n < NS; ++n)
            if (WHOLE || n < left) q[static_cast<int64_t>(n) * p.D] = h[n];
    }
};

template <typename T, typename TB, int NS, bool SPLIT, bool WHOLE>
__global__ __launch_bounds__(SPLIT ? 512 : 64) void ssm_sums_kernel(SsmFwd f) {
    constexpr int ALL = SsmRows<TB, NS, SSM_U, false, WHOLE>::ALL;
    __shared__ __align__(16) float s_rows[(SPLIT ? 8 : 1) * ALL];
    const int nb = SPLIT ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0, seg = blockIdx.y;
    SsmWave<T, TB, NS, WHOLE> w(f.a, nb * NS, seg);
    float h[NS] = {};
    const float S = w.sums(s_rows + nb * ALL, h);
    if (w.valid && nb == 0) f.part_s[(static_cast<int64_t>(w.b) * f.a.nseg + seg) * f.a.D + w.c] = S;
    w.write_segment(f.part_h, seg, h);
}

// The state entering each segment from the segments' sums (the last one's are not
// formed); `carries` may be part_h itself.
__global__ __launch_bounds__(64 * SSM_CARRY_WAVES) void ssm_carry_kernel(SsmFwd f) {
    const SsmArgs& p = f.a;
    const int ci = blockIdx.x * 64 + (threadIdx.x & 63), c = min(ci, p.D - 1), n = blockIdx.y, b = blockIdx.z;
    const int64_t cn = static_cast<int64_t>(c) * p.N + n, row0 = static_cast<int64_t>(b) * p.nseg;
    const int64_t at = (row0 * p.N + n) * p.D + c;
    ssm_carry<false>(p.A[cn] * SSM_LOG2E, p.h0 ? p.h0[static_cast<int64_t>(b) * p.D * p.N + cn] : 0.0f,
                     f.part_s + row0 * p.D + c, p.D, f.part_h + at, f.carries + at, static_cast<int64_t>(p.N) * p.D,
                     p.nseg, p.nseg - 1, ci < p.D);
}

template <typename T, typename TB, int NS, bool Z, bool SPLIT, bool WHOLE>
__global__ __launch_bounds__(SPLIT ? 512 : 64) void ssm_out_kernel(SsmFwd f) {
    constexpr int ALL = SsmRows<TB, NS, SSM_U, true, WHOLE>::ALL;
    __shared__ __align__(16) float s_rows[(SPLIT ? 8 : 1) * ALL];
    __shared__ float s_y[SPLIT ? 2 * 8 * SSM_U * 64 : 1];
    const int nb = SPLIT ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0, seg = blockIdx.y;
    const int NB = SPLIT ? __builtin_amdgcn_readfirstlane(blockDim.x >> 6) : 1;
    SsmWave<T, TB, NS, WHOLE> w(f.a, nb * NS, seg);
    float h[NS];
    if (f.a.nseg > 1) {
        const float* q = f.carries + w.segment_at(seg);
#pragma unroll
        for (int n = 0; n < NS; ++n) h[n] = WHOLE || n < w.left ? q[static_cast<int64_t>(n) * f.a.D] : 0.0f;
    } else {
        w.read_state(f.a.h0, h);
        w.write_segment(f.carries, 0, h);
    }
    w.template outputs<Z, SPLIT>(f.out, s_rows + nb * ALL, s_y, nb, NB, h);
    if (seg == f.a.nseg - 1) w.write_state(f.state, h);
}

// ---------------------------------------------------------------------------
// single token: four lanes per channel, each four consecutive states of every
// sixteen (VEC: states in whole aligned quads) or every fourth state.  Bound by
// reading and writing the states (a server's batch) or by latency (one sequence):
// 256 sequences of 2048 channels with 16 states 16.6 us (4.3 TB/s), one 3.1.  By
// single states the 256 take 33.6 us.  Four sequences a thread, which share A, were no
// faster at any batch (19.0 us for the 256, 5.1 against 3.7 for 16).
// ---------------------------------------------------------------------------
struct SsmStep {
    SsmArgs a;
    float* state;   // [B, D, N], updated
    void* out;      // [B, D]
};

template <typename T, typename TB, bool VEC>
__global__ __launch_bounds__(256) void ssm_step_kernel(SsmStep f) {
    constexpr int V = VEC ? 4 : 1;
    const SsmArgs& p = f.a;
    const int q = threadIdx.x & 3;
    const int c = blockIdx.x * 64 + (threadIdx.x >> 2);
    if (c >= p.D) return;   // whole quads
    const int64_t b = blockIdx.y;
    const int g = c / p.per;
    const float x = IO<T>::ld((static_cast<const T*>(p.x) + b * p.xb)[c]);
    float dt = IO<T>::ld((static_cast<const T*>(p.delta) + b * p.db)[c]) + (p.bias ? p.bias[c] : 0.0f);
    const float* A = p.A + static_cast<int64_t>(c) * p.N;
    float* h = f.state + (b * p.D + c) * p.N;
    const TB* B = static_cast<const TB*>(p.B) + b * p.Bb + static_cast<int64_t>(g) * p.N;
    const TB* C = static_cast<const TB*>(p.C) + b * p.Cb + static_cast<int64_t>(g) * p.N;
    float y = 0.0f;
    bool raw = p.softplus;
    for (int n = q * V; n < p.N; n += 4 * V) {
        const Pack<float, V> a = *reinterpret_cast<const Pack<float, V>*>(A + n);
        Pack<float, V> v = *reinterpret_cast<const Pack<float, V>*>(h + n);
        float Bv[V], Cv[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            Bv[e] = IO<TB>::ld(B[n + e]);
            Cv[e] = IO<TB>::ld(C[n + e]);
        }
        if (raw) dt = ssm_softplus(dt);   // after the first loads have gone out
        raw = false;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            v.v[e] = fmaf(ssm_exp2(dt * (a.v[e] * SSM_LOG2E)), v.v[e], dt * x * Bv[e]);
            y = fmaf(Cv[e], v.v[e], y);
        }
        *reinterpret_cast<Pack<float, V>*>(h + n) = v;
    }
    y += __shfl_xor(y, 1, 64);
    y += __shfl_xor(y, 2, 64);
    if (q != 0) return;
    float o = fmaf(p.skip ? p.skip[c] : 0.0f, x, y);
    if (p.z) {
        const float z = IO<T>::ld((static_cast<const T*>(p.z) + b * p.zb)[c]);
        o *= z * sigmoid_hw(z);
    }
    (static_cast<T*>(f.out) + b * p.D)[c] = IO<T>::st(o);
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
    // fewer than 2^32 threads along x; the gradient's work-groups have up to 5 waves for 17 to 40 states
    const int64_t blocks = q->groups * ((q->channels / q->groups + 63) / 64);
    const int64_t waves = q->states <= 16 ? 1 : q->states <= 40 ? (q->states + 7) / 8 : (q->states + 15) / 16;
    if (!step && blocks * 64 * waves >= (1ll << 32))
        return set_error(MOGT_E_INVALID, "%lld blocks of a group's 64 channels with %lld states: too many for a launch",
                         (long long)blocks, (long long)q->states);
    if (q->batch == 0 || q->channels == 0) return MOGT_OK;
    if (q->length > 0) {
        if (!q->x || !q->delta || !q->A || !q->B || !q->C) return set_error(MOGT_E_INVALID, "null input pointer");
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

template <typename T, typename TB>
int fwd_launch(const SsmFwd& f, int batch, hipStream_t st) {
    const SsmArgs& a = f.a;
    const int waves = ssm_waves(a.N), blocks = a.D / a.per * a.nbk;
    ssm_with_states(a.N, [&](auto ns, auto split, auto whole) {
        constexpr int NS = decltype(ns)::value;
        constexpr bool SPLIT = decltype(split)::value, WHOLE = decltype(whole)::value;
        if (a.nseg > 1) {
            ssm_sums_kernel<T, TB, NS, SPLIT, WHOLE><<<dim3(blocks, a.nseg - 1, batch), 64 * waves, 0, st>>>(f);
            ssm_carry_kernel<<<dim3((a.D + 63) / 64, a.N, batch), ssm_carry_threads(a.nseg), 0, st>>>(f);
        }
        const dim3 grid(blocks, a.nseg, batch);
        if (a.z)
            ssm_out_kernel<T, TB, NS, true, SPLIT, WHOLE><<<grid, 64 * waves, 0, st>>>(f);
        else
            ssm_out_kernel<T, TB, NS, false, SPLIT, WHOLE><<<grid, 64 * waves, 0, st>>>(f);
    });
    return check_launch("mogt_ssm_scan_fwd");
}

template <typename T, typename TB>
int step_launch(const SsmStep& f, int batch, hipStream_t st) {
    const SsmArgs& a = f.a;
    const bool vec = a.N % 4 == 0 && ((reinterpret_cast<uintptr_t>(f.state) | reinterpret_cast<uintptr_t>(a.A)) & 15) == 0;
    const dim3 grid((a.D + 63) / 64, batch);
    if (vec)
        ssm_step_kernel<T, TB, true><<<grid, 256, 0, st>>>(f);
    else
        ssm_step_kernel<T, TB, false><<<grid, 256, 0, st>>>(f);
    return check_launch("mogt_ssm_step");
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
    f.part_h = static_cast<float*>(workspace);
    f.carries = carries || need == 0 ? carries : f.part_h;
    f.part_s = f.part_h + q->batch * f.a.nseg * q->channels * q->states;
    const int batch = static_cast<int>(q->batch);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q->io_dtype == MOGT_F32) return fwd_launch<float, float>(f, batch, st);
    if (q->bc_dtype == MOGT_F32) return fwd_launch<bf16_t, float>(f, batch, st);
    return fwd_launch<bf16_t, bf16_t>(f, batch, st);
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
    const int batch = static_cast<int>(q->batch);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q->io_dtype == MOGT_F32) return step_launch<float, float>(f, batch, st);
    if (q->bc_dtype == MOGT_F32) return step_launch<bf16_t, float>(f, batch, st);
    return step_launch<bf16_t, bf16_t>(f, batch, st);
}
