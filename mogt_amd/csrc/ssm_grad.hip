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
//   carry   folds those shares, the last segment first, into the gradient
//           arriving at each segment's end.
//   grad    walks a segment's blocks of SSM_R steps backwards: the states of a
//           block are formed again from its mark and stay in registers while g
//           runs through it.
//   sums    over the 64-channel blocks of a group (dB, dC) and over segments
//           and sequences (dA, dD, bias), in a fixed order.
// 2 x 8192 steps of 1280 channels with 16 states, bf16: marks 123 us (4.1 TB/s:
// near the 5.2 of a large copy), carry 16, grad 305 (2.2 TB/s), sums 12 and 10.
// Bound of grad: the vector unit (69 % of the cycles) at two waves a SIMD, which is
// what a block's states leave room for: 21 vector instructions per state and step,
// 14 of them the formulas' and 3 the sums over channels.  Marks every 8 steps, 8 states a wave (85
// instead of 62 us at 4096 x 1024) and three waves a SIMD with a part of the states
// in scratch memory were slower; forming all decays twice to load the next block
// earlier changed nothing.
#include <type_traits>

#include "ssm_common.h"
#include "wide_grid.h"

namespace mogt {

int ssm_args(const mogt_ssm_problem* q, bool step, SsmArgs& a);

constexpr int SSM_R = 4;   // steps between marks

struct SsmBwd {
    SsmArgs a;
    const void* dout;          // [B, L, D]
    const float* dfinal;       // [B, D, N] or null
    const float* carries;      // [B, nseg, N, D]
    void *dx, *ddelta, *dz;    // [B, L, D], each may be null
    float* dh0;                // [B, D, N] or null
    float* marks;              // [B, ceil(L / SSM_R), ceil(D / 64), N, 64]: channel c at [c / 64][n][c % 64]
    float* part_g;             // [B, nseg, N, D]
    float* part_s;             // [B, nseg, D]
    float* part_bc;            // [G nbk][B][L][2][N]: dB, dC of a 64-channel block
    float* part_a;             // [B nseg][N + 2][D]: dA, dD, gradient of the bias
    int batch, nblk;
};

// Byte offset of a channel's first state in a row of marks.  The blocks go by the
// channel's number, not by the wave: a group of few channels takes no more room.
__device__ __forceinline__ uint32_t mark_offset(int c, int N) {
    return (static_cast<uint32_t>(c >> 6) * static_cast<uint32_t>(N) * 64u + static_cast<uint32_t>(c & 63)) * 4u;
}
__host__ __device__ inline int64_t mark_row(int64_t D, int64_t N) { return (D + 63) / 64 * 64 * N; }

// Sum of each of 32 values over the wave's lanes by halving steps; a lane gets
// value 2 * (lane / 4) + lane % 2.
__device__ __forceinline__ float wave_sums32(float (&v)[32], int lane) {
    constexpr int M = 32;
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
    const float even = v[0], odd = v[1];   // (an index would put the array into memory)
    return lane & 1 ? odd : even;
}

// Sum of each of 4 values over the lanes with the same lane % Q (4 or 8); a lane
// gets value 2 * (lane / 32) + (lane / 16) % 2.
template <int Q>
__device__ __forceinline__ float wave_sums4(const float (&u)[4]) {
    float v[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(u[i]), __float_as_uint(u[i + 2]), false, false);
        v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    const auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[0]), __float_as_uint(v[1]), false, false);
    float r = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    r += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(r), 0x128, 0xf, 0xf, false));   // row_ror:8
    if constexpr (Q == 4)
        r += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(r), 0x124, 0xf, 0xf, false));   // row_ror:4
    return r;
}

// Whether the grad kernel sums dB and dC through LDS: work-groups of many waves
// of 16 states have no room for it.
constexpr bool grad_via_lds(int NS, int OWN) { return NS == 8 || OWN > 1; }
constexpr int grad_row(int NS) { return 2 * NS + 4; }
constexpr int GRAD_ROWS = 65;   // of a buffer of products: a lane's each, and one for all idle lanes

template <typename T, typename TB, int NS, bool Z, bool SPLIT, bool WHOLE>
__global__ __launch_bounds__(SPLIT ? 512 : 64) void ssm_marks_kernel(SsmBwd f) {
    constexpr int U = SSM_R;
    typedef SsmRows<TB, NS, U, true, WHOLE> Rows;
    __shared__ __align__(16) float s_rows[(SPLIT ? 8 : 1) * Rows::ALL];
    const SsmArgs& p = f.a;
    const int lane = threadIdx.x & 63;
    const int nb = SPLIT ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int n0 = nb * NS, left = p.N - n0;
    const int g = blockIdx.x / p.nbk;
    const int ci = (blockIdx.x - g * p.nbk) * 64 + lane;
    const bool valid = ci < p.per;
    const int c = g * p.per + (valid ? ci : p.per - 1);
    uint32_t off = static_cast<uint32_t>(c) * static_cast<uint32_t>(sizeof(T));
    const int seg = blockIdx.y, b = blockIdx.z;
    const int t0 = seg * p.seg;
    const int te = min(t0 + p.seg, ssm_length(p, b));
    const int64_t row = static_cast<int64_t>(b) * p.nseg + seg;

    float A[NS], h[NS], P[NS], G[NS];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const bool in = WHOLE || n < left;
        A[n] = in ? p.A[static_cast<int64_t>(c) * p.N + n0 + n] * SSM_LOG2E : 0.0f;
        h[n] = in ? f.carries[(row * p.N + n0 + n) * p.D + c] : 0.0f;
        P[n] = 1.0f;
        G[n] = 0.0f;
    }
    const float bias = p.bias ? p.bias[c] : 0.0f;
    const T* px = static_cast<const T*>(p.x) + b * p.xb + t0 * p.xs;
    const T* pd = static_cast<const T*>(p.delta) + b * p.db + t0 * p.ds;
    const T* pz = static_cast<const T*>(p.z) + b * p.zb + t0 * p.zs;
    const T* pg = static_cast<const T*>(f.dout) + (static_cast<int64_t>(b) * p.L + t0) * p.D;
    const TB* pB = static_cast<const TB*>(p.B) + b * p.Bb + static_cast<int64_t>(g) * p.N + n0;
    const TB* pC = static_cast<const TB*>(p.C) + b * p.Cb + static_cast<int64_t>(g) * p.N + n0;
    const Rows rows(pB, p.Bs, pC, p.Cs, lane, left);
    const int64_t row_marks = mark_row(p.D, p.N);
    float* pm = f.marks + (static_cast<int64_t>(b) * f.nblk + t0 / SSM_R) * row_marks + n0 * 64;
    float* lds = s_rows + nb * Rows::ALL;
    uint32_t mark = mark_offset(c, p.N);
    T xr[U], dr[U], zr[U], gr[U];
    float rv[Rows::E], S = 0.0f;
    auto load = [&](int t) {   // the rows of the block at t
        const int cnt = te - t;
        if (cnt >= U) {
            ssm_load_rows<T, U, true>(px, p.xs, off, U, xr);
            ssm_load_rows<T, U, true>(pd, p.ds, off, U, dr);
            ssm_load_rows<T, U, true>(pg, p.D, off, U, gr);
            if constexpr (Z) ssm_load_rows<T, U, true>(pz, p.zs, off, U, zr);
            rows.template load<true>(t, U, rv);
        } else if (cnt > 0) {
            ssm_load_rows<T, U, false>(px, p.xs, off, cnt, xr);
            ssm_load_rows<T, U, false>(pd, p.ds, off, cnt, dr);
            ssm_load_rows<T, U, false>(pg, p.D, off, cnt, gr);
            if constexpr (Z) ssm_load_rows<T, U, false>(pz, p.zs, off, cnt, zr);
            rows.template load<false>(t, cnt, rv);
        }
    };
    load(t0);
    for (int t = t0; t < te; t += U) {
        const int cnt = te - t;
        float dt[U], w[U], dy[U];
        ssm_steps<T, U>(dr, bias, p.softplus, cnt, dt);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            w[i] = dt[i] * IO<T>::ld(xr[i]);
            dy[i] = IO<T>::ld(gr[i]);
            if constexpr (Z) {
                const float z = IO<T>::ld(zr[i]);
                dy[i] *= z * sigmoid_hw(z);
            }
            S += dt[i];
        }
        ssm_mask<U>(cnt, w);
        ssm_mask<U>(cnt, dy);
        Rows::store(lds, lane, rv);
        ssm_wave_sync();
        load(t + U);
        ssm_offset(mark);
#pragma unroll
        for (int n = 0; n < NS; ++n)   // idle lanes write the last channel's once more
            if (WHOLE || n < left) ssm_st<float>(pm + n * 64, mark, h[n]);
        pm += row_marks;
        float Bn[4], Cn[4];   // the next four values of B and C, read ahead
        ssm_lds4(lds, Bn);
        ssm_lds4(lds + NS, Cn);
#pragma unroll
        for (int i = 0; i < U; ++i) {
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
                    const int n = m + e;
                    const float a = ssm_exp2(dt[i] * A[n]);
                    h[n] = fmaf(a, h[n], w[i] * Bv[e]);
                    P[n] *= a;
                    G[n] = fmaf(P[n], Cv[e] * dy[i], G[n]);
                }
                ssm_done4(h, m);
                ssm_done4(G, m);
            }
        }
        ssm_wave_sync();
    }
    // The products of a growing state's decays leave fp32 where the gradient that
    // they carry need not (zero or small rows of it): such a share is formed again
    // from the segment's end, step by step, which scales by one decay at a time.
    bool beyond = false;
#pragma unroll
    for (int n = 0; n < NS; ++n) beyond |= !(fabsf(P[n]) < INFINITY) || !(fabsf(G[n]) < INFINITY);
    if (__any(beyond)) {
#pragma unroll
        for (int n = 0; n < NS; ++n) G[n] = 0.0f;
        // the row pointers stand behind the last block
        for (int t = t0 + (te - 1 - t0) / U * U; t >= t0; t -= U) {
            const int cnt = te - t;
            pd -= U * p.ds;
            pg -= static_cast<int64_t>(U) * p.D;
            const T *qd = pd, *qg = pg;
            ssm_load_rows<T, U, false>(qd, p.ds, off, cnt, dr);
            ssm_load_rows<T, U, false>(qg, p.D, off, cnt, gr);
            if constexpr (Z) {
                pz -= U * p.zs;
                const T* qz = pz;
                ssm_load_rows<T, U, false>(qz, p.zs, off, cnt, zr);
            }
            rows.template load<false>(t, cnt, rv);
            Rows::store(lds, lane, rv);
            ssm_wave_sync();
            float dt[U], dy[U];
            ssm_steps<T, U>(dr, bias, p.softplus, cnt, dt);
#pragma unroll
            for (int i = 0; i < U; ++i) {
                dy[i] = IO<T>::ld(gr[i]);
                if constexpr (Z) {
                    const float z = IO<T>::ld(zr[i]);
                    dy[i] *= z * sigmoid_hw(z);
                }
            }
            ssm_mask<U>(cnt, dy);
#pragma unroll
            for (int i = U - 1; i >= 0; --i) {
#pragma unroll
                for (int n = 0; n < NS; n += 4) {
                    float Cv[4];
                    ssm_lds4(lds + i * Rows::VALS + NS + n, Cv);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        G[n + e] = ssm_exp2(dt[i] * A[n + e]) * fmaf(Cv[e], dy[i], G[n + e]);
                    ssm_done4(G, n);
                }
            }
            ssm_wave_sync();
        }
    }
    if (!valid) return;
    if (n0 == 0) f.part_s[row * p.D + c] = S;
#pragma unroll
    for (int n = 0; n < NS; ++n)
        if (WHOLE || n < left) f.part_g[(row * p.N + n0 + n) * p.D + c] = G[n];
}

// The gradient arriving at each segment's end from the segments' shares, in
// place, the last segment first.
__global__ __launch_bounds__(64 * SSM_CARRY_WAVES) void ssm_carry_back_kernel(SsmBwd f) {
    const SsmArgs& p = f.a;
    const int ci = blockIdx.x * 64 + (threadIdx.x & 63), c = min(ci, p.D - 1), n = blockIdx.y, b = blockIdx.z;
    const int64_t cn = static_cast<int64_t>(c) * p.N + n, row0 = static_cast<int64_t>(b) * p.nseg;
    float* pg = f.part_g + (row0 * p.N + n) * p.D + c;
    ssm_carry<true>(p.A[cn] * SSM_LOG2E, f.dfinal ? f.dfinal[static_cast<int64_t>(b) * p.D * p.N + cn] : 0.0f,
                    f.part_s + row0 * p.D + c, p.D, pg, pg, static_cast<int64_t>(p.N) * p.D, p.nseg, p.nseg, ci < p.D);
}

// One work-group: 64 channels, a wave for NS of their states.  With several waves
// (SPLIT) what a step needs of its channel (step size, written value, gradient of
// y) is formed by one of them and shared through LDS; each adds its part of y, dw
// and sum q A there, and the step's owner finishes its outputs.  OWN: steps of a
// block that a wave owns.
//
// dB and dC are summed over the 64 channels through LDS: each lane leaves its 2 NS
// products in a row (padded to 16-byte accesses without bank conflicts) and adds 4
// values of NS / 2 rows, which leaves 4 values instead of 2 NS to exchange between
// lanes.  Idle lanes write to a row that is not read, and their own stay zero (their
// states repeat the last channel's, and zero times an infinity there would be NaN).
// KEEP: the decays of a block's last steps stay in registers beside its
// states; 16 states leave room for two steps of them, the others form them again
// on the way back.
template <typename T, typename TB, int NS, int OWN, bool Z, bool SPLIT, bool WHOLE>
__global__ __launch_bounds__(SPLIT ? 512 : 64) __attribute__((amdgpu_waves_per_eu(2)))
void ssm_grad_kernel(SsmBwd f) {
    constexpr int R = SSM_R;
    constexpr int KEEP = NS == 8 ? R : 2;   // of the last steps of a block
    constexpr bool VIA_LDS = grad_via_lds(NS, OWN);
    constexpr int ROW = grad_row(NS), QUADS = NS / 2;   // quads of products in a row
    typedef SsmRows<TB, NS, R, true, WHOLE> Rows;
    extern __shared__ __align__(16) float smem[];
    const SsmArgs& p = f.a;
    const int lane = threadIdx.x & 63;
    const int nb = SPLIT ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0;
    const int NB = SPLIT ? __builtin_amdgcn_readfirstlane(blockDim.x >> 6) : 1;
    const int n0 = nb * NS, left = p.N - n0;
    // SPLIT: [2][R][3][64] dt, w, dy and each wave's parts [R][3][64]; per wave
    // its rows and its products
    float* s_chan = smem;
    float* s_part = s_chan + 2 * R * 3 * 64;
    float* s_rows = smem + (SPLIT ? (2 + NB) * R * 3 * 64 : 0) + nb * Rows::ALL;
    float* s_prod = smem + (SPLIT ? (2 + NB) * R * 3 * 64 : 0) + NB * Rows::ALL + nb * (GRAD_ROWS * ROW);
    // a step's products are summed while the next ones are formed (2 x 8192 x 1280: 324
    // us instead of 334, one card): two buffers, for which only a work-group of one wave
    // has the room
    constexpr bool BEHIND = VIA_LDS && !SPLIT;
    const int g = blockIdx.x / p.nbk;
    const int ci = (blockIdx.x - g * p.nbk) * 64 + lane;
    const bool valid = ci < p.per;
    const int c = g * p.per + (valid ? ci : p.per - 1);
    uint32_t off = static_cast<uint32_t>(c) * static_cast<uint32_t>(sizeof(T)), mark = mark_offset(c, p.N);
    const int seg = blockIdx.y, b = blockIdx.z;
    const int len = ssm_length(p, b);
    const int t0 = seg * p.seg, t1 = min(t0 + p.seg, p.L);
    const int te = min(t1, len);
    const int64_t row = static_cast<int64_t>(b) * p.nseg + seg;

    // gradient arriving at the segment's end
    float A[NS], gc[NS], dA[NS];
    const int64_t cn = (static_cast<int64_t>(b) * p.D + c) * p.N + n0;
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        const bool in = WHOLE || n < left;
        A[n] = in ? p.A[static_cast<int64_t>(c) * p.N + n0 + n] * SSM_LOG2E : 0.0f;
        gc[n] = in ? f.part_g[(row * p.N + n0 + n) * p.D + c] : 0.0f;
        dA[n] = 0.0f;
    }
    const float bias = p.bias ? p.bias[c] : 0.0f;
    const float skip = p.skip ? p.skip[c] : 0.0f;
    float d_skip = 0.0f, d_bias = 0.0f;
    const int64_t bl = static_cast<int64_t>(b) * p.L;
    // the last block's first step, and the rows at it of the inputs and outputs
    int t = te > t0 ? t0 + (te - 1 - t0) / R * R : t0 - R;
    const T* px = static_cast<const T*>(p.x) + b * p.xb + t * p.xs;
    const T* pd = static_cast<const T*>(p.delta) + b * p.db + t * p.ds;
    const T* pz = static_cast<const T*>(p.z) + b * p.zb + t * p.zs;
    int64_t pg = (bl + t) * p.D;   // of dx, ddelta and dz
    const T* pdo = static_cast<const T*>(f.dout) + pg;
    const int64_t row_marks = mark_row(p.D, p.N);
    const float* pm = f.marks + (static_cast<int64_t>(b) * f.nblk + t / R) * row_marks + n0 * 64;
    const Rows rows(static_cast<const TB*>(p.B) + b * p.Bb + static_cast<int64_t>(g) * p.N + n0, p.Bs,
                    static_cast<const TB*>(p.C) + b * p.Cb + static_cast<int64_t>(g) * p.N + n0, p.Cs, lane, left);
    // dB, dC rows of this 64-channel block: a lane ends with value `mine` of
    // them, of step `slot` of every GROUP among the lanes with the same one
    constexpr int GROUP = 32 / NS;
    const int mine = VIA_LDS ? 4 * (lane & (QUADS - 1)) + 2 * (lane >> 5) + ((lane >> 4) & 1)
                             : 2 * (lane >> 2) + (lane & 1);
    const int slot = (lane / QUADS) & (GROUP - 1);
    const float* s_mine = s_prod + (lane / QUADS) * QUADS * ROW + (lane & (QUADS - 1)) * 4;
    const bool held = f.part_bc && (WHOLE || mine % NS < left) && (VIA_LDS || (lane & 2) == 0);
    uint32_t bc_off = ((mine >= NS ? p.N : 0) + n0 + mine % NS) * 4u;

    // inputs of the next block: the rows of the steps this wave owns, B and C,
    // the state it starts from
    T xr[OWN], dr[OWN], gr[OWN], zr[OWN];
    float rv[Rows::E], hm[NS];
    auto load_as = [&](auto full, int t) {   // the block at t; pointers move to the one before it
        constexpr bool FULL = decltype(full)::value;
        const int cnt = te - t;
        ssm_offset(off);
        ssm_offset(mark);
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int i = nb + k * NB, at = FULL && !SPLIT ? i : min(i, min(cnt, R) - 1);
            xr[k] = ssm_ld(px + at * p.xs, off);
            dr[k] = ssm_ld(pd + at * p.ds, off);
            gr[k] = ssm_ld(pdo + static_cast<int64_t>(at) * p.D, off);
            if constexpr (Z) zr[k] = ssm_ld(pz + at * p.zs, off);
        }
        rows.template load<FULL>(t, cnt, rv);
#pragma unroll
        for (int n = 0; n < NS; ++n) hm[n] = WHOLE || n < left ? ssm_ld(pm + n * 64, mark) : 0.0f;
        px -= R * p.xs;
        pd -= R * p.ds;
        pz -= R * p.zs;
        pdo -= static_cast<int64_t>(R) * p.D;
        pm -= row_marks;
    };
    auto load = [&](int t) {
        if (te - t >= R)
            load_as(std::true_type(), t);
        else
            load_as(std::false_type(), t);
    };
    float* s_own = s_prod + (valid ? lane : 64) * ROW;   // this lane's products
    const bool idle = !__all(valid);
    if (VIA_LDS && !valid) {
#pragma unroll
        for (int q = 0; q < (BEHIND ? 2 : 1); ++q)
            for (int k = 0; k < ROW; ++k) s_prod[(q * GRAD_ROWS + lane) * ROW + k] = 0.0f;
    }
    const int64_t bc_row = static_cast<int64_t>(blockIdx.x) * f.batch * p.L + bl;
    float* pbc = f.part_bc + (bc_row + t) * 2 * p.N;
    uint32_t bc_mine = bc_off + (VIA_LDS ? slot * 2 * p.N * 4u : 0u);
    if (t >= t0) load(t);
    for (int buf = 0; t >= t0; t -= R, buf ^= 1) {
        const int cnt = te - t;
        float* chan = s_chan + buf * R * 3 * 64 + lane;
        // of the owned steps: x, gradient of the output, raw step size, the gate
        float x[OWN], go[OWN], raw[OWN], z[OWN], dt_own[OWN];
        // gradient of y, and the gate's sigmoid
        auto grad_y = [&](int k, float& sig) {
            sig = Z ? sigmoid_hw(z[k]) : 0.0f;
            return Z ? go[k] * (z[k] * sig) : go[k];
        };
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int i = nb + k * NB;
            x[k] = IO<T>::ld(xr[k]);
            go[k] = IO<T>::ld(gr[k]);
            raw[k] = IO<T>::ld(dr[k]) + bias;
            dt_own[k] = p.softplus ? ssm_softplus(raw[k]) : raw[k];
            z[k] = Z ? IO<T>::ld(zr[k]) : 0.0f;
            if (cnt < R && i >= cnt) x[k] = go[k] = dt_own[k] = z[k] = 0.0f;
            if (SPLIT && i < R) {
                float sig;
                chan[(i * 3 + 0) * 64] = dt_own[k];
                chan[(i * 3 + 1) * 64] = dt_own[k] * x[k];
                chan[(i * 3 + 2) * 64] = grad_y(k, sig);
            }
        }
        Rows::store(s_rows, lane, rv);
        float h0[NS], hs[R][NS], a[KEEP][NS], dt[R];
#pragma unroll
        for (int n = 0; n < NS; ++n) h0[n] = hm[n];
        if constexpr (SPLIT)
            __syncthreads();
        else
            ssm_wave_sync();
        float Bn[4], Cn[4];   // the next four values of B and C, read ahead
        ssm_lds4(s_rows, Bn);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            dt[i] = SPLIT ? chan[(i * 3 + 0) * 64] : dt_own[SPLIT ? 0 : i];
            const float w = SPLIT ? chan[(i * 3 + 1) * 64] : dt[i] * x[SPLIT ? 0 : i];
#pragma unroll
            for (int m = 0; m < NS; m += 4) {
                const float Bv[4] = {Bn[0], Bn[1], Bn[2], Bn[3]};
                if (m + 4 < NS)
                    ssm_lds4(s_rows + i * Rows::VALS + m + 4, Bn);
                else   // on the way back the last step comes first
                    ssm_lds4(s_rows + min(i + 1, R - 1) * Rows::VALS, Bn);
                if (i == R - 1 && m + 4 == NS) ssm_lds4(s_rows + i * Rows::VALS + NS, Cn);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = m + e;
                    const float d = ssm_exp2(dt[i] * A[n]);
                    if (i >= R - KEEP) a[i >= R - KEEP ? i - (R - KEEP) : 0][n] = d;
                    hs[i][n] = fmaf(d, i > 0 ? hs[i > 0 ? i - 1 : 0][n] : h0[n], w * Bv[e]);
                }
                ssm_done4(hs[i], m);
            }
        }
        auto finish = [&](int k, float dy, float sig, float y, float dw, float qA) {   // outputs of an owned step
            const int64_t at = pg + static_cast<int64_t>(nb + k * NB) * p.D;
            float dd = fmaf(dw, x[k], qA * SSM_LN2);
            if (p.softplus) dd *= sigmoid_hw(raw[k]);
            d_skip = fmaf(dy, x[k], d_skip);
            d_bias += dd;
            if (!valid) return;
            if constexpr (Z) {
                if (f.dz)
                    ssm_st<T>(static_cast<T*>(f.dz) + at, off,
                              IO<T>::st(go[k] * fmaf(skip, x[k], y) * (sig * fmaf(z[k], 1.0f - sig, 1.0f))));
            }
            if (f.dx) ssm_st<T>(static_cast<T*>(f.dx) + at, off, IO<T>::st(fmaf(dw, dt_own[k], skip * dy)));
            if (f.ddelta) ssm_st<T>(static_cast<T*>(f.ddelta) + at, off, IO<T>::st(dd));
        };
        // this lane's part of a step's sums over the channels, from its products in
        // LDS; BEHIND: while the step before it in time is computed
        float kept = 0.0f, u[4];
        auto read_rows = [&](int i, int k, float (&r0)[4], float (&r1)[4]) {   // k and k + 1 of step i
            const float* q = s_mine + ((BEHIND ? i % 2 * GRAD_ROWS : 0) + k) * ROW;
            ssm_lds4(q, r0);
            ssm_lds4(q + ROW, r1);
        };
        auto add_rows = [&](int k, const float (&r0)[4], const float (&r1)[4]) {
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = (k > 0 ? u[e] + r0[e] : r0[e]) + r1[e];
        };
        auto put_sums = [&](int i) {
            const float s = wave_sums4<QUADS>(u);
            kept = slot == i % GROUP ? s : kept;
            if (i % GROUP == 0 && held && i + slot < cnt) ssm_st<float>(pbc + i * 2 * p.N, bc_mine, kept);
        };
#pragma unroll
        for (int i = R - 1; i >= 0; --i) {
            if (i < R - 1 && i == cnt - 1) {
                // The sequence's last step (its block is the first one here): the steps
                // behind it added their step size of zero times the end's state, which
                // may be infinite.
#pragma unroll
                for (int n = 0; n < NS; ++n) dA[n] = 0.0f;
#pragma unroll
                for (int n = 0; n < NS; n += 4) ssm_done4(dA, n);
            }
            float v[2 * NS];
            float sig = 0.0f;
            const float dy = SPLIT ? chan[(i * 3 + 2) * 64] : grad_y(SPLIT ? 0 : i, sig);
            const float w = SPLIT ? chan[(i * 3 + 1) * 64] : dt[i] * x[SPLIT ? 0 : i];
            if (i < R - KEEP) asm volatile("" : "+v"(dt[i]));   // no decays kept from the way there
            float y = 0.0f, dw = 0.0f, qA = 0.0f;
#pragma unroll
            for (int m = 0; m < NS; m += 4) {   // four states at a time
                ssm_f4 qb, qc;   // products of dB and dC
                const float Bv[4] = {Bn[0], Bn[1], Bn[2], Bn[3]}, Cv[4] = {Cn[0], Cn[1], Cn[2], Cn[3]};
                float r0[4], r1[4];   // of the step after
                if constexpr (BEHIND) {
                    if (i < R - 1) read_rows(i + 1, m / 2, r0, r1);
                }
                if (i > 0 || m + 4 < NS) {
                    const int at = m + 4 < NS ? i * Rows::VALS + m + 4 : (i - 1) * Rows::VALS;
                    ssm_lds4(s_rows + at, Bn);
                    ssm_lds4(s_rows + at + NS, Cn);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int n = m + e;
                    if constexpr (Z) y = fmaf(Cv[e], hs[i][n], y);
                    const float gn = fmaf(Cv[e], dy, gc[n]);
                    qb[e] = gn * w;
                    qc[e] = dy * hs[i][n];
                    dw = fmaf(gn, Bv[e], dw);
                    gc[n] = gn * (i >= R - KEEP ? a[i >= R - KEEP ? i - (R - KEEP) : 0][n] : ssm_exp2(dt[i] * A[n]));
                    const float q = gc[n] * (i > 0 ? hs[i > 0 ? i - 1 : 0][n] : h0[n]);
                    qA = fmaf(q, A[n], qA);
                    dA[n] = fmaf(q, dt[i], dA[n]);
                }
                if constexpr (VIA_LDS) {
                    float* q = s_own + (BEHIND ? i % 2 * GRAD_ROWS : 0) * ROW + m;
                    *reinterpret_cast<ssm_f4*>(q) = qb;
                    *reinterpret_cast<ssm_f4*>(q + NS) = qc;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[m + e] = qb[e];
                        v[NS + m + e] = qc[e];
                    }
                }
                ssm_done4(gc, m);
                ssm_done4(dA, m);
                ssm_done(qA);
                ssm_done(dw);
                if constexpr (Z) ssm_done(y);
                if constexpr (BEHIND) {
                    if (i < R - 1) add_rows(m / 2, r0, r1);
                }
            }
            if (f.part_bc) {
                if constexpr (VIA_LDS) {
                    ssm_wave_sync();
                    if (BEHIND && i < R - 1) put_sums(i + 1);
                    if (!BEHIND || i == 0) {
#pragma unroll
                        for (int k = 0; k < QUADS; k += 2) {
                            float r0[4], r1[4];
                            read_rows(i, k, r0, r1);
                            add_rows(k, r0, r1);
                        }
                        ssm_wave_sync();
                        put_sums(i);
                    }
                } else {
                    if (idle) {
#pragma unroll
                        for (int k = 0; k < 2 * NS; ++k) v[k] = valid ? v[k] : 0.0f;
                    }
                    const float s = wave_sums32(v, lane);
                    if (held && i < cnt) ssm_st<float>(pbc + i * 2 * p.N, bc_mine, s);
                }
            }
            if constexpr (SPLIT) {
                float* part = s_part + (nb * R + i) * 3 * 64 + lane;
                part[0] = y;
                part[64] = dw;
                part[128] = qA;
            } else if (i < cnt) {
                finish(SPLIT ? 0 : i, dy, sig, y, dw, qA);
            }
            // the next block's inputs take the registers of the states passed
            if (i == R - 2 && t - R >= t0) load(t - R);
        }
        if constexpr (SPLIT) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < OWN; ++k) {
                const int i = nb + k * NB;
                if (i >= R || i >= cnt) continue;
                float y = 0.0f, dw = 0.0f, qA = 0.0f;
                for (int m = 0; m < NB; ++m) {
                    const float* part = s_part + (m * R + i) * 3 * 64 + lane;
                    y += part[0];
                    dw += part[64];
                    qA += part[128];
                }
                float sig;
                const float dy = grad_y(k, sig);
                finish(k, dy, sig, y, dw, qA);
            }
        }
        pg -= static_cast<int64_t>(R) * p.D;
        pbc -= R * 2 * p.N;
        ssm_offset(bc_mine);
    }
    // rows past the sequence's length
    for (t = max(t0, te); t < t1; ++t) {
        const int64_t at = (bl + t) * p.D;
        if (nb == 0 && valid) {
            if (f.dx) (static_cast<T*>(f.dx) + at)[c] = IO<T>::st(0.0f);
            if (f.ddelta) (static_cast<T*>(f.ddelta) + at)[c] = IO<T>::st(0.0f);
            if (Z && f.dz) (static_cast<T*>(f.dz) + at)[c] = IO<T>::st(0.0f);
        }
        if (held) ssm_st<float>(f.part_bc + (bc_row + t) * 2 * p.N, bc_off, 0.0f);
    }
    if constexpr (SPLIT) {   // the first wave adds up the owned steps' sums
        __syncthreads();
        s_part[(nb * 2 + 0) * 64 + lane] = d_skip;
        s_part[(nb * 2 + 1) * 64 + lane] = d_bias;
        __syncthreads();
        d_skip = d_bias = 0.0f;
        for (int m = 0; m < NB; ++m) {
            d_skip += s_part[(m * 2 + 0) * 64 + lane];
            d_bias += s_part[(m * 2 + 1) * 64 + lane];
        }
    }
    if (!valid) return;
    float* pa = f.part_a + row * (p.N + 2) * p.D + c;
#pragma unroll
    for (int n = 0; n < NS; ++n)
        if (WHOLE || n < left) {
            pa[static_cast<int64_t>(n0 + n) * p.D] = dA[n];
            if (f.dh0 && seg == 0) f.dh0[cn + n] = gc[n];
        }
    if (nb == 0) {
        pa[static_cast<int64_t>(p.N) * p.D] = d_skip;
        pa[static_cast<int64_t>(p.N + 1) * p.D] = d_bias;
    }
}

// dB, dC [B, L, G, N]: the sums over the 64-channel blocks of a group, in order.
template <typename TB>
__global__ __launch_bounds__(256) void ssm_bc_kernel(const float* part, TB* dB, TB* dC, int64_t rows, int G, int nbk,
                                                     int N) {
    const int64_t i = wide_block() * 256 + threadIdx.x;   // (row, dB or dC, n) of one group
    const int64_t all = rows * 2 * N;
    if (i >= all) return;
    const int64_t r = i / (2 * N);
    const int k = static_cast<int>(i - r * (2 * N));
    TB* out = k < N ? dB : dC;
    if (!out) return;
    for (int g = blockIdx.z; g < G; g += gridDim.z) {
        const float* q = part + static_cast<int64_t>(g) * nbk * all + i;
        float s = 0.0f;
        for (int m = 0; m < nbk; ++m) s += q[m * all];
        out[(r * G + g) * N + (k < N ? k : k - N)] = IO<TB>::st(s);
    }
}

// Column sums over rows of [rows][K][D], in a fixed order: a work-group takes 64
// columns, its 16 waves every 16th row each.  Column (k, d) goes to a[d N + k]
// for k < N, then to b[d] and c[d]; each may be null.
__global__ __launch_bounds__(1024) void column_sums_kernel(const float* part, float* a, float* b, float* c, int64_t rows,
                                                           int64_t cols, int64_t D, int64_t N) {
    __shared__ float s[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int64_t i = wide_block() * 64 + lane;
    float v = 0.0f;
    if (i < cols)
        for (int64_t r = w; r < rows; r += 16) v += part[r * cols + i];
    s[w][lane] = v;
    __syncthreads();
    if (w != 0 || i >= cols) return;
#pragma unroll
    for (int m = 1; m < 16; ++m) v += s[m][lane];
    const int64_t k = i / D, d = i - k * D;
    if (k < N) {
        if (a) a[d * N + k] = v;
    } else if (k == N) {
        if (b) b[d] = v;
    } else if (c) {
        c[d] = v;
    }
}

int column_sums(const float* part, float* a, float* b, float* c, int64_t rows, int64_t K, int64_t D, int64_t N,
                hipStream_t st) {
    const int64_t cols = K * D;
    column_sums_kernel<<<wide_grid((cols + 63) / 64), 1024, 0, st>>>(part, a, b, c, rows, cols, D, N);
    return check_launch("column sums");
}

namespace {

// States of a wave of the grad kernel: 16 where one wave holds all, 8 from there
// to 40, and 16 beyond (more waves of 8 would not fit their products into 64 KB of
// LDS).  4096 steps of 1024 channels: 12 states in waves of 16 69 us and of 8 101,
// 16 states 62 and 85, 24 states 147 both, 32 states 130 and 107, 40 states 250
// both, 48 states 223 and 265.
constexpr int grad_states_per_wave(int64_t N) { return N > 8 && (N <= 16 || N > 40) ? 16 : 8; }
inline int grad_waves(int64_t N) {
    const int ns = grad_states_per_wave(N);
    return static_cast<int>((N + ns - 1) / ns);
}

template <typename T, typename TB, int NS, int OWN, bool SPLIT>
void grad_launch_as(const SsmBwd& f, hipStream_t st) {
    const SsmArgs& a = f.a;
    const int waves = grad_waves(a.N);
    const dim3 grid(a.D / a.per * a.nbk, a.nseg, f.batch);
    const size_t lds = sizeof(float) * ((SPLIT ? (2 + waves) * SSM_R * 3 * 64 : 0) + waves * SSM_R * 2 * NS +
                                        (grad_via_lds(NS, OWN) ? (SPLIT ? waves : 2) * GRAD_ROWS * grad_row(NS) : 0));
    const bool whole = a.N % NS == 0;
    if (a.z && whole)
        ssm_grad_kernel<T, TB, NS, OWN, true, SPLIT, true><<<grid, 64 * waves, lds, st>>>(f);
    else if (a.z)
        ssm_grad_kernel<T, TB, NS, OWN, true, SPLIT, false><<<grid, 64 * waves, lds, st>>>(f);
    else if (whole)
        ssm_grad_kernel<T, TB, NS, OWN, false, SPLIT, true><<<grid, 64 * waves, lds, st>>>(f);
    else
        ssm_grad_kernel<T, TB, NS, OWN, false, SPLIT, false><<<grid, 64 * waves, lds, st>>>(f);
}

template <typename T, typename TB>
void grad_launch(const SsmBwd& f, hipStream_t st) {
    const SsmArgs& a = f.a;
    const dim3 grid(a.D / a.per * a.nbk, a.nseg, f.batch);
    ssm_with_states(a.N, [&](auto ns, auto split, auto whole) {
        constexpr int NS = decltype(ns)::value;
        constexpr bool SPLIT = decltype(split)::value, WHOLE = decltype(whole)::value;
        if (a.z)
            ssm_marks_kernel<T, TB, NS, true, SPLIT, WHOLE><<<grid, 64 * ssm_waves(a.N), 0, st>>>(f);
        else
            ssm_marks_kernel<T, TB, NS, false, SPLIT, WHOLE><<<grid, 64 * ssm_waves(a.N), 0, st>>>(f);
    });
    ssm_carry_back_kernel<<<dim3((a.D + 63) / 64, a.N, f.batch), ssm_carry_threads(a.nseg), 0, st>>>(f);
    const int waves = grad_waves(a.N);
    if (grad_states_per_wave(a.N) == 8) {
        if (waves == 1)
            grad_launch_as<T, TB, 8, 4, false>(f, st);
        else if (waves < 4)
            grad_launch_as<T, TB, 8, 2, true>(f, st);
        else
            grad_launch_as<T, TB, 8, 1, true>(f, st);
    } else if (waves == 1) {
        grad_launch_as<T, TB, 16, 4, false>(f, st);
    } else if (waves < 4) {
        grad_launch_as<T, TB, 16, 2, true>(f, st);
    } else {
        grad_launch_as<T, TB, 16, 1, true>(f, st);
    }
}

struct BwdSizes {
    size_t marks, g, s, bc, a;   // floats of each part
    size_t total() const { return marks + g + s + bc + a; }
};

BwdSizes bwd_sizes(int64_t B, int64_t L, int64_t D, int64_t N, int64_t G, int64_t segment) {
    const int64_t nseg = L > 0 ? (L + segment - 1) / segment : 1;
    BwdSizes z;
    const int64_t ncb = G * ((D / G + 63) / 64);
    z.marks = static_cast<size_t>(B * ((L + SSM_R - 1) / SSM_R) * mark_row(D, N));
    z.g = static_cast<size_t>(B * nseg * N * D);
    z.s = static_cast<size_t>(B * nseg * D);
    z.bc = static_cast<size_t>(2 * ncb * B * L * N);
    z.a = static_cast<size_t>(B * nseg * (N + 2) * D);
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
    // a row of marks has 32-bit offsets
    if (q->batch * q->length * q->states >= (1ll << 31) || q->channels * q->states >= (1ll << 28))
        return set_error(MOGT_E_INVALID, "batch x length x states below 2^31 and channels x states below 2^28 expected");
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
    f.part_s = f.part_g + n.g;
    f.part_a = f.part_s + n.s;
    float* bc = f.part_a + n.a;
    f.part_bc = out->dB || out->dC ? bc : nullptr;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q->io_dtype == MOGT_F32)
        grad_launch<float, float>(f, st);
    else if (q->bc_dtype == MOGT_F32)
        grad_launch<bf16_t, float>(f, st);
    else
        grad_launch<bf16_t, bf16_t>(f, st);
    if (const int rc = check_launch("mogt_ssm_scan_bwd")) return rc;
    const int64_t rows = q->batch * q->length;
    if (f.part_bc && rows > 0) {
        const dim3 grid = wide_grid((rows * 2 * q->states + 255) / 256,
                                    static_cast<unsigned>(q->groups < 65535 ? q->groups : 65535));
        if (q->bc_dtype == MOGT_F32)
            ssm_bc_kernel<float><<<grid, 256, 0, st>>>(bc, static_cast<float*>(out->dB), static_cast<float*>(out->dC),
                                                       rows, static_cast<int>(q->groups), f.a.nbk, f.a.N);
        else
            ssm_bc_kernel<bf16_t><<<grid, 256, 0, st>>>(bc, static_cast<bf16_t*>(out->dB),
                                                        static_cast<bf16_t*>(out->dC), rows,
                                                        static_cast<int>(q->groups), f.a.nbk, f.a.N);
        if (const int rc = check_launch("mogt_ssm_scan_bwd")) return rc;
    }
    if (!out->dA && !out->dD && !out->ddelta_bias) return MOGT_OK;
    return column_sums(f.part_a, out->dA, out->dD, out->ddelta_bias, q->batch * f.a.nseg, q->states + 2, q->channels,
                       q->states, st);
}
