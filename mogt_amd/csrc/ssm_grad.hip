// Selective state space scan, backward (ssm_common.h has the recurrence).
//
// With dy = dout silu(z), w = dt x and g the gradient of h_t:
//   g_t = C_t dy_t + a_{t+1} g_{t+1}                (a = exp(dt A))
//   dC_t = sum_d dy h      dB_t = sum_d g w         sums over a group's channels
//   dw = sum_n g B,  q = g a h_{t-1}                (q: gradient of dt A)
//   dx = dw dt + D dy,  ddt = dw x + sum_n q A,  dA = sum_t q dt,  dz = dout y silu'(z)
//
// States are not kept by the forward, only those entering each segment.
//   marks   scans each segment forward from its start state, leaves the state
//           entering every SSM_R steps and, in the same sweep, the segment's
//           share of the gradient of its start state: sum_t (prod_{s<=t} a_s) C_t dy_t.
//   grad    folds those shares of the segments after its own (last first) into
//           the gradient arriving at its end, then walks its blocks of SSM_R
//           steps backwards: the states of a block are formed again from its
//           mark and stay in registers while g runs through it.
//   sums    over the 64-channel blocks of a group (dB, dC) and over segments
//           and sequences (dA, dD, bias), in a fixed order.
// The sum of 2 NS products over the 64 channels of a wave is a halving
// exchange: each step adds two lanes' values and halves the count, so it takes
// about 2 instructions per product instead of 6.
#include <type_traits>

#include "ssm_common.h"

namespace mogt {

int ssm_args(const mogt_ssm_problem* q, bool step, SsmArgs& a);

constexpr int SSM_R = 8;   // steps between marks

struct SsmBwd {
    SsmArgs a;
    const void* dout;          // [B, L, D]
    const float* dfinal;       // [B, D, N] or null
    const float* carries;      // [B, nseg, N, D]
    void *dx, *ddelta, *dz;    // [B, L, D], each may be null
    float* dh0;                // [B, D, N] or null
    float* marks;              // [B, ceil(L / SSM_R), N, D]
    float* part_g;             // [B, nseg, N, D]
    float* part_s;             // [B, nseg, D]
    float* part_bc;            // [2][G nbk][B][L][N]: dB, dC of a 64-channel block
    float* part_a;             // [B nseg][N][D]
    float* part_d;             // [waves][B nseg][D]
    float* part_bias;          // [waves][B nseg][D]
    int batch, nblk;
};

// Sum of each of M values over the wave's lanes.  The halving steps leave
// value R * (lane / 4) + j, R = M / 16, in v[j] of each lane.
template <int M>
__device__ __forceinline__ void wave_sums(float (&v)[M]) {
    static_assert(M == 16 || M == 32, "16 or 32 values");
#pragma unroll
    for (int i = 0; i < M / 2; ++i) {   // lanes 32..63 keep the upper half of the values
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i + M / 2]), false,
                                                        false);
        v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
#pragma unroll
    for (int i = 0; i < M / 4; ++i) {   // odd rows of 16 lanes
        const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i + M / 4]), false,
                                                        false);
        v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
#pragma unroll
    for (int i = 0; i < M / 8; ++i) {   // lanes 8..15 of a row
        float r;
        asm("s_nop 1\n\t"
            "v_add_f32_dpp %0, %1, %1 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
            "v_add_f32_dpp %0, %2, %2 row_ror:8 row_mask:0xf bank_mask:0xc"
            : "=&v"(r) : "v"(v[i]), "v"(v[i + M / 8]));
        v[i] = r;
    }
#pragma unroll
    for (int i = 0; i < M / 16; ++i) {   // odd quads
        float r;
        asm("s_nop 1\n\t"
            "v_add_f32_dpp %0, %1, %1 row_half_mirror row_mask:0xf bank_mask:0x5\n\t"
            "v_add_f32_dpp %0, %2, %2 row_half_mirror row_mask:0xf bank_mask:0xa"
            : "=&v"(r) : "v"(v[i]), "v"(v[i + M / 16]));
        v[i] = r;
    }
#pragma unroll
    for (int i = 0; i < M / 16; ++i) {
        v[i] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v[i]), 0xB1, 0xf, 0xf, false));
        v[i] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v[i]), 0x4E, 0xf, 0xf, false));
    }
}

template <typename T, typename TB, int NS, bool Z, bool SPLIT>
__global__ __launch_bounds__(SPLIT ? 512 : 64) void ssm_marks_kernel(SsmBwd f) {
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
    const int64_t row = static_cast<int64_t>(b) * p.nseg + seg;

    float A[NS], h[NS], P[NS], G[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const bool in = n0 + n < p.N;
        A[n] = in ? p.A[static_cast<int64_t>(c) * p.N + n0 + n] * SSM_LOG2E : 0.0f;
        h[n] = in ? f.carries[(row * p.N + n0 + n) * p.D + c] : 0.0f;
        P[n] = 1.0f;
        G[n] = 0.0f;
    }
    const float bias = p.bias ? p.bias[c] : 0.0f;
    const T* px = static_cast<const T*>(p.x) + b * p.xb;
    const T* pd = static_cast<const T*>(p.delta) + b * p.db;
    const T* pz = static_cast<const T*>(p.z) + b * p.zb;
    const T* pg = static_cast<const T*>(f.dout) + static_cast<int64_t>(b) * p.L * p.D;
    const TB* pB = static_cast<const TB*>(p.B) + b * p.Bb + static_cast<int64_t>(g) * p.N;
    const TB* pC = static_cast<const TB*>(p.C) + b * p.Cb + static_cast<int64_t>(g) * p.N;
    float S = 0.0f;
    for (int t = t0; t < te; t += SSM_R) {
        T xr[SSM_R], dr[SSM_R], zr[SSM_R], gr[SSM_R];
#pragma unroll
        for (int i = 0; i < SSM_R; ++i) {
            const int64_t tt = min(t + i, te - 1);
            xr[i] = (px + tt * p.xs)[c];
            dr[i] = (pd + tt * p.ds)[c];
            gr[i] = (pg + tt * p.D)[c];
            if constexpr (Z) zr[i] = (pz + tt * p.zs)[c];
        }
        if (valid) {
            float* m = f.marks + ((static_cast<int64_t>(b) * f.nblk + t / SSM_R) * p.N + n0) * p.D + c;
#pragma unroll
            for (int n = 0; n < NS; ++n)
                if (n0 + n < p.N) m[static_cast<int64_t>(n) * p.D] = h[n];
        }
#pragma unroll
        for (int i = 0; i < SSM_R; ++i) {
            if (t + i >= te) break;
            float Bv[NS], Cv[NS];
            ssm_row<TB, NS>(pB + (t + i) * p.Bs, n0, p.N, Bv);
            ssm_row<TB, NS>(pC + (t + i) * p.Cs, n0, p.N, Cv);
            float dt = IO<T>::ld(dr[i]) + bias;
            if (p.softplus) dt = ssm_softplus(dt);
            const float w = dt * IO<T>::ld(xr[i]);
            float dy = IO<T>::ld(gr[i]);
            if constexpr (Z) {
                const float z = IO<T>::ld(zr[i]);
                dy *= z * sigmoid_hw(z);
            }
            S += dt;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const float a = ssm_exp2(dt * A[n]);
                h[n] = fmaf(a, h[n], w * Bv[n]);
                P[n] *= a;
                G[n] = fmaf(P[n], Cv[n] * dy, G[n]);
            }
        }
    }
    if (!valid) return;
    if (n0 == 0) f.part_s[row * p.D + c] = S;
#pragma unroll
    for (int n = 0; n < NS; ++n)
        if (n0 + n < p.N) f.part_g[(row * p.N + n0 + n) * p.D + c] = G[n];
}

template <typename T, typename TB, int NS, bool Z, bool SPLIT>
__global__ __launch_bounds__(SPLIT ? 512 : 64) void ssm_grad_kernel(SsmBwd f) {
    extern __shared__ float s_part[];   // SPLIT: [waves][3][SSM_R][64] parts of y, dw and sum q A
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
    const int64_t row0 = static_cast<int64_t>(b) * p.nseg;

    // gradient arriving at the segment's end; idle lanes hold zeros throughout
    float A[NS], gc[NS], dA[NS];
    const int64_t cn = (static_cast<int64_t>(b) * p.D + c) * p.N + n0;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const bool in = n0 + n < p.N;
        A[n] = in ? p.A[static_cast<int64_t>(c) * p.N + n0 + n] * SSM_LOG2E : 0.0f;
        gc[n] = in && valid && f.dfinal ? f.dfinal[cn + n] : 0.0f;
        dA[n] = 0.0f;
    }
    for (int j = (len - 1) / p.seg; j > seg && len > 0; --j) {
        const float S = f.part_s[(row0 + j) * p.D + c];
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const float e = n0 + n < p.N ? f.part_g[((row0 + j) * p.N + n0 + n) * p.D + c] : 0.0f;
            gc[n] = valid ? fmaf(ssm_exp2(S * A[n]), gc[n], e) : 0.0f;
        }
    }
    const float bias = p.bias ? p.bias[c] : 0.0f;
    const float skip = p.skip ? p.skip[c] : 0.0f;
    float d_skip = 0.0f, d_bias = 0.0f;
    const int64_t bl = static_cast<int64_t>(b) * p.L;
    const T* px = static_cast<const T*>(p.x) + b * p.xb;
    const T* pd = static_cast<const T*>(p.delta) + b * p.db;
    const T* pz = static_cast<const T*>(p.z) + b * p.zb;
    const T* pg = static_cast<const T*>(f.dout) + bl * p.D;
    const TB* pB = static_cast<const TB*>(p.B) + b * p.Bb + static_cast<int64_t>(g) * p.N;
    const TB* pC = static_cast<const TB*>(p.C) + b * p.Cb + static_cast<int64_t>(g) * p.N;
    T* ox = static_cast<T*>(f.dx) + bl * p.D;
    T* od = static_cast<T*>(f.ddelta) + bl * p.D;
    T* oz = static_cast<T*>(f.dz) + bl * p.D;
    // dB, dC rows of this 64-channel block
    const int64_t plane = static_cast<int64_t>(gridDim.x) * f.batch * p.L * p.N;
    float* pbc = f.part_bc + (static_cast<int64_t>(blockIdx.x) * f.batch * p.L + bl) * p.N + n0;

    auto block = [&](int t, auto full) {
        constexpr bool FULL = decltype(full)::value;
        float x[SSM_R], raw[SSM_R], z[SSM_R], go[SSM_R];
#pragma unroll
        for (int i = 0; i < SSM_R; ++i) {
            const int64_t tt = FULL ? t + i : min(t + i, te - 1);
            const bool on = valid && (FULL || t + i < te);
            x[i] = IO<T>::ld((px + tt * p.xs)[c]);
            raw[i] = IO<T>::ld((pd + tt * p.ds)[c]) + bias;
            go[i] = IO<T>::ld((pg + tt * p.D)[c]);
            z[i] = 0.0f;
            if constexpr (Z) z[i] = IO<T>::ld((pz + tt * p.zs)[c]);
            if (!on) x[i] = raw[i] = go[i] = z[i] = 0.0f;
        }
        float h0[NS], hs[SSM_R][NS], dt[SSM_R], y[SSM_R];
        const float* m = f.marks + ((static_cast<int64_t>(b) * f.nblk + t / SSM_R) * p.N + n0) * p.D + c;
#pragma unroll
        for (int n = 0; n < NS; ++n) h0[n] = valid && n0 + n < p.N ? m[static_cast<int64_t>(n) * p.D] : 0.0f;
#pragma unroll
        for (int i = 0; i < SSM_R; ++i) {
            if (!FULL && t + i >= te) break;
            float Bv[NS], Cv[NS];
            ssm_row<TB, NS>(pB + (t + i) * p.Bs, n0, p.N, Bv);
            if constexpr (Z) ssm_row<TB, NS>(pC + (t + i) * p.Cs, n0, p.N, Cv);
            dt[i] = p.softplus ? ssm_softplus(raw[i]) : raw[i];
            const float w = dt[i] * x[i];
            y[i] = 0.0f;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                hs[i][n] = fmaf(ssm_exp2(dt[i] * A[n]), i > 0 ? hs[i > 0 ? i - 1 : 0][n] : h0[n], w * Bv[n]);
                if constexpr (Z) y[i] = fmaf(Cv[n], hs[i][n], y[i]);
            }
        }
        auto finish = [&](int i, float yi, float dw, float qA) {
            float dy = go[i];
            const int64_t at = static_cast<int64_t>(t + i) * p.D;
            if constexpr (Z) {
                const float s = sigmoid_hw(z[i]);
                dy *= z[i] * s;
                if (f.dz && valid)
                    (oz + at)[c] = IO<T>::st(go[i] * fmaf(skip, x[i], yi) * (s * fmaf(z[i], 1.0f - s, 1.0f)));
            }
            float dd = fmaf(dw, x[i], qA * SSM_LN2);
            if (p.softplus) dd *= sigmoid_hw(raw[i]);
            d_skip = fmaf(dy, x[i], d_skip);
            d_bias += dd;
            if (valid) {
                if (f.dx) (ox + at)[c] = IO<T>::st(fmaf(dw, dt[i], skip * dy));
                if (f.ddelta) (od + at)[c] = IO<T>::st(dd);
            }
        };
#pragma unroll
        for (int i = SSM_R - 1; i >= 0; --i) {
            if (!FULL && t + i >= te) continue;
            float Bv[NS], Cv[NS], v[2 * NS];
            ssm_row<TB, NS>(pB + (t + i) * p.Bs, n0, p.N, Bv);
            ssm_row<TB, NS>(pC + (t + i) * p.Cs, n0, p.N, Cv);
            const float w = dt[i] * x[i];
            const float dy = Z ? go[i] * z[i] * sigmoid_hw(z[i]) : go[i];
            float dw = 0.0f, qA = 0.0f;
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                const float gn = fmaf(Cv[n], dy, gc[n]);
                v[n] = gn * w;
                v[NS + n] = dy * hs[i][n];
                dw = fmaf(gn, Bv[n], dw);
                gc[n] = gn * ssm_exp2(dt[i] * A[n]);
                const float q = gc[n] * (i > 0 ? hs[i > 0 ? i - 1 : 0][n] : h0[n]);
                qA = fmaf(q, A[n], qA);
                dA[n] = fmaf(q, dt[i], dA[n]);
            }
            if (f.part_bc) {
                wave_sums<2 * NS>(v);
                constexpr int R = NS / 8;
                const int j = lane & 3, k = R * (lane >> 2) + j, n = k % NS;
                if (j < R && n0 + n < p.N)
                    pbc[(k >= NS ? plane : 0) + static_cast<int64_t>(t + i) * p.N + n] = R == 2 && j == 1 ? v[R - 1] : v[0];
            }
            if constexpr (SPLIT) {
                float* s = s_part + (nb * 3 * SSM_R + i) * 64 + lane;
                s[0] = y[i];
                s[SSM_R * 64] = dw;
                s[2 * SSM_R * 64] = qA;
            } else {
                finish(i, y[i], dw, qA);
            }
        }
        if constexpr (SPLIT) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < SSM_R; ++i) {
                if (!FULL && t + i >= te) break;
                if (i % NB != nb) continue;
                float yi = 0.0f, dw = 0.0f, qA = 0.0f;
                for (int k = 0; k < NB; ++k) {
                    const float* s = s_part + (k * 3 * SSM_R + i) * 64 + lane;
                    yi += s[0];
                    dw += s[SSM_R * 64];
                    qA += s[2 * SSM_R * 64];
                }
                finish(i, yi, dw, qA);
            }
            __syncthreads();
        }
    };
    if (te > t0) {
        int t = t0 + (te - 1 - t0) / SSM_R * SSM_R;
        if (t + SSM_R > te) {
            block(t, std::integral_constant<bool, false>());
            t -= SSM_R;
        }
        for (; t >= t0; t -= SSM_R) block(t, std::integral_constant<bool, true>());
    }
    // rows past the sequence's length
    for (int t = max(t0, te); t < t1; ++t) {
        const int64_t at = static_cast<int64_t>(t) * p.D;
        if (nb == 0 && valid) {
            if (f.dx) (ox + at)[c] = IO<T>::st(0.0f);
            if (f.ddelta) (od + at)[c] = IO<T>::st(0.0f);
            if (Z && f.dz) (oz + at)[c] = IO<T>::st(0.0f);
        }
        if (f.part_bc && lane < 2 * NS && n0 + lane % NS < p.N)
            pbc[(lane >= NS ? plane : 0) + static_cast<int64_t>(t) * p.N + lane % NS] = 0.0f;
    }
    if (!valid) return;
    const int64_t row = row0 + seg;
#pragma unroll
    for (int n = 0; n < NS; ++n)
        if (n0 + n < p.N) {
            f.part_a[(row * p.N + n0 + n) * p.D + c] = dA[n];
            if (f.dh0 && seg == 0) f.dh0[cn + n] = gc[n];
        }
    const int64_t rows = static_cast<int64_t>(f.batch) * p.nseg;
    f.part_d[(nb * rows + row) * p.D + c] = d_skip;
    f.part_bias[(nb * rows + row) * p.D + c] = d_bias;
}

// dB, dC [B, L, G, N]: the sums over the 64-channel blocks of a group, in order.
template <typename TB>
__global__ __launch_bounds__(256) void ssm_bc_kernel(const float* part, TB* dB, TB* dC, int64_t rows, int G, int nbk,
                                                     int N) {
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;   // (row, n) of one group
    if (i >= rows * N) return;
    const int g = blockIdx.y;
    TB* out = blockIdx.z ? dC : dB;
    if (!out) return;
    const float* q = part + (static_cast<int64_t>(blockIdx.z) * G + g) * nbk * rows * N + i;
    float s = 0.0f;
    for (int k = 0; k < nbk; ++k) s += q[static_cast<int64_t>(k) * rows * N];
    const int64_t r = i / N;
    out[(r * G + g) * N + (i - r * N)] = IO<TB>::st(s);
}

// Column sums over rows of [rows][cols], in a fixed order: a work-group takes
// 64 columns, its 16 waves every 16th row each.  Column k goes to out[(k % D) *
// N + k / D] (state-major to channel-major).
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* part, float* out, int64_t rows, int64_t cols,
                                                           int64_t D, int64_t N) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t k = static_cast<int64_t>(blockIdx.x) * 64 + lane;
    float v = 0.0f;
    if (k < cols)
        for (int64_t r = w; r < rows; r += 16) v += part[r * cols + k];
    s[w][lane] = v;
    __syncthreads();
    if (w != 0 || k >= cols) return;
#pragma unroll
    for (int i = 1; i < 16; ++i) v += s[i][lane];
    out[(k % D) * N + k / D] = v;
}

int column_sums(const float* part, float* out, int64_t rows, int64_t D, int64_t N, hipStream_t st) {
    const int64_t cols = D * N;
    column_sums_kernel<<<static_cast<unsigned>((cols + 63) / 64), 1024, 0, st>>>(part, out, rows, cols, D, N);
    return check_launch("column sums");
}

namespace {

template <typename T, typename TB, int NS, bool SPLIT>
void grad_launch(const SsmBwd& f, hipStream_t st) {
    const SsmArgs& a = f.a;
    const int waves = SPLIT ? (a.N + NS - 1) / NS : 1;
    const dim3 grid(a.D / a.per * a.nbk, a.nseg, f.batch);
    const size_t lds = SPLIT ? sizeof(float) * 3 * waves * SSM_R * 64 : 0;
    if (a.z) {
        ssm_marks_kernel<T, TB, NS, true, SPLIT><<<grid, 64 * waves, 0, st>>>(f);
        ssm_grad_kernel<T, TB, NS, true, SPLIT><<<grid, 64 * waves, lds, st>>>(f);
    } else {
        ssm_marks_kernel<T, TB, NS, false, SPLIT><<<grid, 64 * waves, 0, st>>>(f);
        ssm_grad_kernel<T, TB, NS, false, SPLIT><<<grid, 64 * waves, lds, st>>>(f);
    }
}

template <typename T, typename TB>
void grad_states(const SsmBwd& f, hipStream_t st) {
    if (f.a.N <= 8)
        grad_launch<T, TB, 8, false>(f, st);
    else if (f.a.N <= 16)
        grad_launch<T, TB, 16, false>(f, st);
    else
        grad_launch<T, TB, 16, true>(f, st);
}

struct BwdSizes {
    size_t marks, seg, s, bc, d;   // floats of each part
    size_t total() const { return marks + 2 * seg + s + bc + 2 * d; }
};

BwdSizes bwd_sizes(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G, int64_t segment) {
    const int64_t nseg = L > 0 ? (L + segment - 1) / segment : 1;
    const int64_t ncb = G * ((D / G + 63) / 64), waves = N <= 16 ? 1 : (N + 15) / 16;
    BwdSizes z;
    z.marks = static_cast<size_t>(B * ((L + SSM_R - 1) / SSM_R) * N * D);
    z.seg = static_cast<size_t>(B * nseg * N * D);
    z.s = static_cast<size_t>(B * nseg * D);
    z.bc = static_cast<size_t>(2 * ncb * B * L * N);
    z.d = static_cast<size_t>(waves * B * nseg * D);
    return z;
}

}  // namespace
}  // namespace mogt

using namespace mogt;

extern "C" size_t mogt_ssm_scan_bwd_workspace_bytes(int64_t batch, int64_t length, int64_t channels, int64_t states,
                                                    int64_t groups, int64_t segment) {
    if (batch <= 0 || channels <= 0 || states <= 0 || segment <= 0 || length < 0 || groups <= 0 ||
        channels % groups != 0)
        return 0;
    return bwd_sizes(batch, length, channels, states, groups, segment).total() * sizeof(float);
}

extern "C" int mogt_ssm_scan_bwd(const mogt_ssm_problem* q, const void* dout, const float* dfinal_state,
                                 const float* carries, const mogt_ssm_gradients* out, void* workspace,
                                 size_t workspace_bytes, void* stream) {
    clear_error();
    SsmBwd f{};
    if (const int rc = ssm_args(q, false, f.a)) return rc;
    if (!out) return set_error(MOGT_E_INVALID, "null gradients");
    if (q->batch == 0 || q->channels == 0) return MOGT_OK;
    if (!carries || !q->A || (q->length > 0 && !dout)) return set_error(MOGT_E_INVALID, "null input pointer");
    if (out->dz && !q->z) return set_error(MOGT_E_INVALID, "a gradient of z without z");
    // one-dimensional grids of the sums
    if (q->batch * q->length * q->states >= (1ll << 32) || q->channels * q->states >= (1ll << 28))
        return set_error(MOGT_E_INVALID, "batch x length x states below 2^32 and channels x states below 2^28 expected");
    const BwdSizes n = bwd_sizes(q->batch, q->length, q->channels, q->states, q->groups, q->segment);
    if (!workspace || workspace_bytes < n.total() * sizeof(float))
        return set_error(MOGT_E_WORKSPACE, "workspace of %zu bytes expected, got %zu", n.total() * sizeof(float),
                         workspace ? workspace_bytes : 0);
    f.dout = dout;
    f.dfinal = dfinal_state;
    f.carries = carries;
    f.dx = out->dx;
    f.ddelta = out->ddelta;
    f.dz = out->dz;
    f.dh0 = out->dinitial_state;
    f.batch = static_cast<int>(q->batch);
    f.nblk = (f.a.L + SSM_R - 1) / SSM_R;
    f.marks = static_cast<float*>(workspace);
    f.part_g = f.marks + n.marks;
    f.part_a = f.part_g + n.seg;
    f.part_s = f.part_a + n.seg;
    float* bc = f.part_s + n.s;
    f.part_bc = out->dB || out->dC ? bc : nullptr;
    f.part_d = bc + n.bc;
    f.part_bias = f.part_d + n.d;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q->io_dtype == MOGT_F32)
        grad_states<float, float>(f, st);
    else if (q->bc_dtype == MOGT_F32)
        grad_states<bf16_t, float>(f, st);
    else
        grad_states<bf16_t, bf16_t>(f, st);
    if (const int rc = check_launch("mogt_ssm_scan_bwd")) return rc;
    const int64_t rows = q->batch * q->length;
    if (f.part_bc && rows > 0) {
        const dim3 grid(static_cast<unsigned>((rows * q->states + 255) / 256), static_cast<unsigned>(q->groups), 2);
        if (q->bc_dtype == MOGT_F32)
            ssm_bc_kernel<float><<<grid, 256, 0, st>>>(bc, static_cast<float*>(out->dB), static_cast<float*>(out->dC),
                                                       rows, static_cast<int>(q->groups), f.a.nbk, f.a.N);
        else
            ssm_bc_kernel<bf16_t><<<grid, 256, 0, st>>>(bc, static_cast<bf16_t*>(out->dB),
                                                        static_cast<bf16_t*>(out->dC), rows,
                                                        static_cast<int>(q->groups), f.a.nbk, f.a.N);
        if (const int rc = check_launch("mogt_ssm_scan_bwd")) return rc;
    }
    const int64_t parts = q->batch * f.a.nseg, waves = f.a.N <= 16 ? 1 : (f.a.N + 15) / 16;
    if (out->dA)
        if (const int rc = column_sums(f.part_a, out->dA, parts, q->channels, q->states, st)) return rc;
    if (out->dD)
        if (const int rc = column_sums(f.part_d, out->dD, waves * parts, q->channels, 1, st)) return rc;
    if (out->ddelta_bias)
        if (const int rc = column_sums(f.part_bias, out->ddelta_bias, waves * parts, q->channels, 1, st)) return rc;
    return MOGT_OK;
}
