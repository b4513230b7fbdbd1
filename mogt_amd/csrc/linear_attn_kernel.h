// The chunked pass of linear attention (linear_attn.h has the mathematics), one
// work-group of four waves per segment, head and LA_NV value columns.
//
// Tiles (16x16 matrix instructions, D[row][column]: a lane holds column lane % 16
// and rows 4 (lane / 16) .. + 3):
//   pairs    D[s][t] = k_s . q_t, the lower triangle's tiles spread over the waves;
//            times the decay between the steps to LDS as rows t (bf16: pieces)
//   reads    D[v][t] += S q: a wave holds all rows of S for its 16 columns in
//            accumulators, whose layout is an operand's layout already
//   sums     D[v][t] += V P
//   writes   S = exp(c_T) S + K^T (w V): D[row of S][v]
// Operands that contract over steps are read transposed from LDS (bf16: the
// transposing LDS read).  S never leaves registers inside a segment.
#include "linear_attn.h"

namespace mogt {
namespace {

typedef float la_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 la_b8 __attribute__((ext_vector_type(8)));
typedef __bf16 la_b4 __attribute__((ext_vector_type(4)));
typedef short la_s4 __attribute__((ext_vector_type(4)));
typedef uint32_t la_u4 __attribute__((ext_vector_type(4)));

template <typename TI> struct LaOp;

template <> struct LaOp<bf16_t> {
    typedef la_b8 frag;
    static __device__ __forceinline__ la_f4 mma(frag a, frag b, la_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // column of the lane's chunk of four in a transposed tile read: of tile `tile`
    // of a state's rows (ROWS: two tiles hold 32 rows so that a lane's 2 x 4
    // accumulators are 8 consecutive rows, an operand's order), or natural
    template <bool ROWS>
    static __device__ __forceinline__ int tr_col(int tile, int lane) {
        return ROWS ? 32 * (tile >> 1) + 8 * (lane & 3) + 4 * (tile & 1) : 16 * tile + 4 * (lane & 3);
    }
    // elements (s0 + 8 g .. + 7, column lane % 16 of the tile) of rows s
    template <bool ROWS>
    static __device__ __forceinline__ frag tr(const bf16_t* p, int stride, int s0, int tile, int lane) {
        const bf16_t* q = p + (s0 + 8 * (lane >> 4) + ((lane & 15) >> 2)) * stride + tr_col<ROWS>(tile, lane);
        typedef __attribute__((address_space(3))) la_s4* lds;
        la_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(q));
        la_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(q + 4 * stride));
        return __builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // row of a state held by accumulator `tile`, register i
    static __device__ __forceinline__ int state_row(int tile, int i, int lane) {
        return 32 * (tile >> 1) + 8 * (lane >> 4) + 4 * (tile & 1) + i;
    }
    static __device__ __forceinline__ float value(frag f, int e) { return static_cast<float>(f[e]); }
};

template <> struct LaOp<float> {
    typedef la_f4 frag;
    static __device__ __forceinline__ la_f4 mma(frag a, frag b, la_f4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    template <bool ROWS>
    static __device__ __forceinline__ frag tr(const float* p, int stride, int s0, int tile, int lane) {
        const float* q = p + (s0 + 4 * (lane >> 4)) * stride + 16 * tile + (lane & 15);
        return frag{q[0], q[stride], q[2 * stride], q[3 * stride]};
    }
    static __device__ __forceinline__ int state_row(int tile, int i, int lane) { return 16 * tile + 4 * (lane >> 4) + i; }
    static __device__ __forceinline__ float value(frag f, int e) { return f[e]; }
};

// NP pieces of fp32 values: bf16 parts that add up to them, or the values
template <typename TI, int N>
__device__ __forceinline__ void la_split(float x, int e, typename LaOp<TI>::frag (&out)[N]) {
    if constexpr (std::is_same<TI, float>::value) {
        out[0][e] = x;
    } else {
#pragma unroll
        for (int p = 0; p < N; ++p) {
            const __bf16 h = static_cast<__bf16>(x);
            out[p][e] = h;
            if (p + 1 < N) x -= static_cast<float>(h);
        }
    }
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double la_dpp_add(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(u), CTRL, ROWS, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(u >> 32), CTRL, ROWS, 0xf, false);
    return x + __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// Inclusive sums over the 64 lanes; lanes shifted past a row's start add zero.
__device__ __forceinline__ double la_wave_sums(double x) {
    x = la_dpp_add<0x111, 0xf>(x);   // row_shr:1
    x = la_dpp_add<0x112, 0xf>(x);
    x = la_dpp_add<0x114, 0xf>(x);
    x = la_dpp_add<0x118, 0xf>(x);
    x = la_dpp_add<0x142, 0xa>(x);   // row_bcast:15 into rows 1 and 3
    x = la_dpp_add<0x143, 0xc>(x);   // row_bcast:31 into rows 2 and 3
    return x;
}

__device__ __forceinline__ double la_lane(double x, int lane) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(u), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(u >> 32), lane);
    return __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo);
}

// The rows of a chunk on their way from memory to LDS: W elements wide, 16 bytes
// at a time over the work-group's threads.
template <typename TI, int W>
struct LaTile {
    static constexpr int T = LaChunk<TI>::T, EPC = 16 / sizeof(TI), CPR = W / EPC;
    static constexpr int N = (T * CPR + LA_THREADS - 1) / LA_THREADS, STRIDE = W + LaChunk<TI>::PAD;
    la_u4 r[N];

    // row u of the chunk is step time(u); rows from `cnt` on and columns from `d` on are zero
    template <typename F>
    __device__ __forceinline__ void load(const LaRows& s, const TI* base, int cnt, int d, F&& time) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = threadIdx.x + LA_THREADS * i, u = id / CPR, c = id % CPR * EPC;
            la_u4 x = {0, 0, 0, 0};
            if (u < cnt && c < d) {
                const TI* p = base + time(u) * s.row + c;
                if (s.vec) {
                    x = *reinterpret_cast<const la_u4*>(p);
                } else {
                    union { la_u4 w; TI e[EPC]; } y;
                    y.w = x;
                    for (int e = 0; e < EPC; ++e)
                        if (c + e < d) y.e[e] = p[e];
                    x = y.w;
                }
            }
            r[i] = x;
        }
    }
    __device__ __forceinline__ void store(TI* lds) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = threadIdx.x + LA_THREADS * i;
            if (T * CPR % LA_THREADS == 0 || id < T * CPR)
                *reinterpret_cast<la_u4*>(lds + id / CPR * STRIDE + id % CPR * EPC) = r[i];
        }
    }
    // whether any element is infinite or NaN
    __device__ __forceinline__ bool wild() const {
        bool any = false;
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t w = r[i][j];
                if (sizeof(TI) == 2) any |= (w & 0x7f80u) == 0x7f80u;
                any |= (w & 0x7f800000u) == 0x7f800000u;
            }
        return any;
    }
};

template <typename TI, int DK, bool OUT>
struct LaLds {
    static constexpr int T = LaChunk<TI>::T, PAD = LaChunk<TI>::PAD, NP = LaChunk<TI>::NP;
    TI q[OUT ? T * (DK + PAD) : 8];
    TI k[T * (DK + PAD)];
    TI v[T * (LA_NV + PAD)];
    TI p[OUT ? NP * T * (T + PAD) : 8];
    float hi[T], lo[T];       // c_t in two parts: differences are as exact as their size
    float in[T], w[T];        // factors of the query's part and of the writes
    float end;                // exp(c_T)
    int wild;                 // 1 + the last chunk with an infinite or NaN value
    float dot[OUT ? 4 * T : 4];
};

template <typename TI, int DK, bool OUT>
__global__ __launch_bounds__(LA_THREADS, 2) void la_pass_kernel(LaArgs a) {
    typedef LaOp<TI> Op;
    typedef typename Op::frag Frag;
    constexpr int T = LaChunk<TI>::T, KS = LaChunk<TI>::KS, PAD = LaChunk<TI>::PAD, NP = LaChunk<TI>::NP;
    constexpr int TT = T / 16, RT = DK / 16, SK = DK + PAD, SV = LA_NV + PAD, SP = T + PAD, E = KS / 4;
    __shared__ __align__(16) LaLds<TI, DK, OUT> s;

    const int which = blockIdx.z / a.B, b = blockIdx.z - which * a.B, h = blockIdx.y;
    const LaPass& p = a.pass[which];
    // value blocks of one segment lie 8 work-groups apart, on one XCD
    const int seg = blockIdx.x / p.nvb, n0 = (blockIdx.x - seg * p.nvb) * LA_NV;
    if (seg >= (OUT ? a.nseg : a.nseg - 1)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grp = lane >> 4;
    const int n = la_length(a, b);
    const int64_t seq = static_cast<int64_t>(b) * a.H + h;
    // steps t0 .. t1 - 1 of the sequence; u counts them in pass order
    const int t0 = (p.reverse ? a.nseg - 1 - seg : seg) * a.seg, t1 = min(t0 + a.seg, n), cnt = max(t1 - t0, 0);

    const TI* qb = static_cast<const TI*>(p.q.p) + b * p.q.batch + h / p.q.div * p.q.head;
    const TI* kb = static_cast<const TI*>(p.k.p) + b * p.k.batch + h / p.k.div * p.k.head;
    const TI* vb = static_cast<const TI*>(p.v.p) + b * p.v.batch + h / p.v.div * p.v.head + n0;
    const float* gb = a.g + b * a.g_batch + h * a.g_head;
    const int nw = min(p.dn - n0, LA_NV);

    // the wave's 16 columns of the state
    la_f4 S[RT];
    const int col = n0 + 16 * wave + (lane & 15);
    float* slot = p.states ? p.states + (seq * (a.nseg + 1) + seg) * a.state : nullptr;
    {
        const float* from = !OUT ? nullptr : a.nseg > 1 ? slot : p.init ? p.init + seq * a.state : nullptr;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = Op::state_row(r, i, lane);
                const bool in = row < p.dc && col < p.dn;
                const int64_t at = static_cast<int64_t>(row) * p.rs + static_cast<int64_t>(col) * p.cs;
                S[r][i] = from && in ? from[at] : 0.0f;
                if (OUT && a.nseg == 1 && p.keep && slot && in) slot[at] = S[r][i];
            }
    }

    LaTile<TI, DK> tq, tk;
    LaTile<TI, LA_NV> tv;
    float gn = 0.0f;   // wave 0: g of the lane's step
    double total = 0.0;
    auto load = [&](int u0) {
        const int left = cnt - u0;
        auto time = [&](int u) { return static_cast<int64_t>(p.reverse ? t1 - 1 - u0 - u : t0 + u0 + u); };
        if (OUT) tq.load(p.q, qb, left, p.dc, time);
        tk.load(p.k, kb, left, p.dc, time);
        tv.load(p.v, vb, left, nw, time);
        if (wave == 0) {
            gn = 0.0f;
            if (lane < T && lane < left) {
                const int64_t t = time(lane) + (p.reverse ? 1 : 0);
                if (t < n) gn = gb[t * a.g_row];
            }
        }
    };
    if (threadIdx.x == 0) s.wild = 0;
    if constexpr (OUT && NP > 1) {   // the tiles above the diagonal that share a fragment with one below
#pragma unroll
        for (int piece = 0; piece < NP; ++piece)
            for (int tt = 0; tt < TT; tt += 2)
                for (int i = threadIdx.x; i < 256; i += LA_THREADS)
                    s.p[(piece * T + 16 * tt + (i >> 4)) * SP + 16 * (tt + 1) + (i & 15)] = 0;
    }
    load(0);
    for (int u0 = 0; u0 < cnt; u0 += T) {
        __syncthreads();   // the last chunk's reads are done
        if (OUT) tq.store(s.q);
        tk.store(s.k);
        tv.store(s.v);
        if (OUT && tv.wild()) s.wild = u0 + 1;
        if (wave == 0) {
            const double g2 = static_cast<double>(gn) * 1.4426950408889634;
            const double c = la_wave_sums(g2 < LA_LOG2_MIN ? LA_LOG2_MIN : g2), end = la_lane(c, 63);
            const float hi = static_cast<float>(c);
            if (lane < T) {
                s.hi[lane] = hi;
                s.lo[lane] = static_cast<float>(c - hi);
                s.in[lane] = p.qs * __builtin_amdgcn_exp2f(hi);
                s.w[lane] = p.ws * __builtin_amdgcn_exp2f(static_cast<float>(end - c));
            }
            if (lane == 0) s.end = __builtin_amdgcn_exp2f(static_cast<float>(end));
            total += end;
        }
        __syncthreads();
        if (u0 + T < cnt) load(u0 + T);

        la_f4 acc[OUT ? TT : 1];
        if constexpr (OUT) {
            // pairs
#pragma unroll
            for (int idx = 0; idx < TT * (TT + 1) / 2; ++idx) {
                if (idx % 4 != wave) continue;
                const int tt = idx < 1 ? 0 : idx < 3 ? 1 : idx < 6 ? 2 : 3, ts = idx - tt * (tt + 1) / 2;
                la_f4 d = {0, 0, 0, 0};
                const TI* kr = s.k + (16 * ts + (lane & 15)) * SK + E * grp;
                const TI* qr = s.q + (16 * tt + (lane & 15)) * SK + E * grp;
#pragma unroll
                for (int k = 0; k < DK; k += KS)
                    d = Op::mma(*reinterpret_cast<const Frag*>(kr + k), *reinterpret_cast<const Frag*>(qr + k), d);
                const int t = 16 * tt + (lane & 15), s0 = 16 * ts + 4 * grp;
                const float hi = s.hi[t], lo = s.lo[t];
                const la_f4 shi = *reinterpret_cast<const la_f4*>(s.hi + s0), slo = *reinterpret_cast<const la_f4*>(s.lo + s0);
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = __builtin_amdgcn_exp2f((hi - shi[i]) + (lo - slo[i]));
                    x[i] = s0 + i <= t ? d[i] * (p.ps * e) : 0.0f;
                }
#pragma unroll
                for (int piece = 0; piece < NP; ++piece) {
                    Pack<TI, 4> w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        w.v[i] = IO<TI>::st(x[i]);
                        if (piece + 1 < NP) x[i] -= IO<TI>::ld(w.v[i]);
                    }
                    *reinterpret_cast<Pack<TI, 4>*>(s.p + (piece * T + t) * SP + s0) = w;
                }
            }
            // reads
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) acc[tt] = la_f4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < DK / KS; ++k) {
                Frag sp[NP];
#pragma unroll
                for (int e = 0; e < E; ++e) la_split<TI>(S[(k * KS / 16) + e / 4][e & 3], e, sp);
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
                    const Frag qf = *reinterpret_cast<const Frag*>(s.q + (16 * tt + (lane & 15)) * SK + E * grp + k * KS);
#pragma unroll
                    for (int piece = 0; piece < NP; ++piece) acc[tt] = Op::mma(sp[piece], qf, acc[tt]);
                }
            }
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) acc[tt] *= s.in[16 * tt + (lane & 15)];
            __syncthreads();
        }

        Frag vf[T / KS], wv[T / KS][NP];
#pragma unroll
        for (int k = 0; k < T / KS; ++k) {
            vf[k] = Op::template tr<false>(s.v, SV, KS * k, wave, lane);
#pragma unroll
            for (int e = 0; e < E; ++e) la_split<TI>(Op::value(vf[k], e) * s.w[KS * k + E * grp + e], e, wv[k]);
        }
        if constexpr (OUT) {
            // sums
            if (s.wild != u0 + 1) {
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
#pragma unroll
                    for (int k = 0; k < (16 * tt + 15) / KS + 1; ++k)
#pragma unroll
                        for (int piece = 0; piece < NP; ++piece)
                            acc[tt] = Op::mma(vf[k], *reinterpret_cast<const Frag*>(s.p + (piece * T + 16 * tt + (lane & 15)) * SP + E * grp + KS * k), acc[tt]);
            } else {   // an infinite or NaN value must not meet the zeros of earlier steps
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
                    const int t = 16 * tt + (lane & 15);
                    for (int u = 0; u <= t; ++u) {
                        float x = 0.0f;
                        for (int piece = 0; piece < NP; ++piece) x += IO<TI>::ld(s.p[(piece * T + t) * SP + u]);
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            acc[tt][i] = fmaf(x, IO<TI>::ld(s.v[u * SV + 16 * wave + 4 * grp + i]), acc[tt][i]);
                    }
                }
            }
        }
        // writes
        const float end = s.end;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            la_f4 d = S[r] * end;
#pragma unroll
            for (int k = 0; k < T / KS; ++k) {
                const Frag kf = Op::template tr<true>(s.k, SK, KS * k, r, lane);
#pragma unroll
                for (int piece = 0; piece < NP; ++piece) d = Op::mma(kf, wv[k][piece], d);
            }
            S[r] = d;
        }
        if constexpr (OUT) {
            const int c0 = 16 * wave + 4 * grp;   // the lane's first column of the block
            const bool whole = p.dn % 4 == 0;
            const TI* xb = static_cast<const TI*>(p.x.p) + b * p.x.batch + h / p.x.div * p.x.head + n0 + c0;
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const int u = u0 + 16 * tt + (lane & 15);
                float dot = 0.0f;
                if (u < cnt && c0 < nw) {
                    const int64_t t = p.reverse ? t1 - 1 - u : t0 + u;
                    const int64_t at = ((static_cast<int64_t>(b) * a.L + t) * a.H + h) * p.dn + n0 + c0;
                    if (p.out) {
                        if (whole) {
                            if (p.out_f32) {
                                *reinterpret_cast<la_f4*>(static_cast<float*>(p.out) + at) = acc[tt];
                            } else {
                                Pack<TI, 4> w;
#pragma unroll
                                for (int i = 0; i < 4; ++i) w.v[i] = IO<TI>::st(acc[tt][i]);
                                *reinterpret_cast<Pack<TI, 4>*>(static_cast<TI*>(p.out) + at) = w;
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (c0 + i < nw) {
                                    if (p.out_f32)
                                        static_cast<float*>(p.out)[at + i] = acc[tt][i];
                                    else
                                        static_cast<TI*>(p.out)[at + i] = IO<TI>::st(acc[tt][i]);
                                }
                        }
                    }
                    if (p.dot) {
                        const TI* xr = xb + t * p.x.row;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (c0 + i < nw) dot = fmaf(IO<TI>::ld(xr[i]), acc[tt][i], dot);
                    }
                }
                if (p.dot) {
                    dot += __shfl_xor(dot, 16);
                    dot += __shfl_xor(dot, 32);
                    if (lane < 16) s.dot[wave * T + 16 * tt + lane] = dot;
                }
            }
            if (p.dot) {
                __syncthreads();
                const int u = u0 + threadIdx.x;
                if (threadIdx.x < T && u < cnt)
                    p.dot[(static_cast<int64_t>(n0 / LA_NV) * a.B * a.H + seq) * a.L + (p.reverse ? t1 - 1 - u : t0 + u)] =
                        (s.dot[threadIdx.x] + s.dot[T + threadIdx.x]) + (s.dot[2 * T + threadIdx.x] + s.dot[3 * T + threadIdx.x]);
            }
        }
    }

    if constexpr (OUT) {
        // rows past the sequence's length
        if (p.out) {
            const int from = max(t0, n), to = min(t0 + a.seg, a.L);
            for (int i = threadIdx.x; i < (to - from) * nw; i += LA_THREADS) {
                const int64_t t = from + i / nw;
                const int64_t at = ((static_cast<int64_t>(b) * a.L + t) * a.H + h) * p.dn + n0 + i % nw;
                if (p.out_f32)
                    static_cast<float*>(p.out)[at] = 0.0f;
                else
                    static_cast<TI*>(p.out)[at] = IO<TI>::st(0.0f);
            }
        }
    } else if (threadIdx.x == 0 && n0 == 0) {
        p.ctot[seq * a.nseg + seg] = static_cast<float>(total);
    }
    // the state after the segment: its own (sums), or the sequence's last
    float* after = !OUT || (seg == a.nseg - 1 && p.keep && p.states) ? slot + a.state : nullptr;
    float* last = OUT && seg == a.nseg - 1 && p.last ? p.last + seq * a.state : nullptr;
    if (after || last) {
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int row = Op::state_row(r, i, lane);
                if (row >= p.dc || col >= p.dn) continue;
                const int64_t at = static_cast<int64_t>(row) * p.rs + static_cast<int64_t>(col) * p.cs;
                if (after) after[at] = S[r][i];
                if (last) last[at] = S[r][i];
            }
    }
}

}  // namespace

// Launches the passes `pass[0 .. count - 1]` of `a`, which have one padded width.
template <typename TI>
void la_launch_passes(const LaArgs& a, int count, bool out, hipStream_t st) {
    int nvb = 0;
    for (int i = 0; i < count; ++i) nvb = a.pass[i].nvb > nvb ? a.pass[i].nvb : nvb;
    const dim3 grid(static_cast<unsigned>(out ? a.nseg : a.nseg - 1) * nvb, a.H, static_cast<unsigned>(a.B) * count);
    auto with = [&](auto width) {
        constexpr int W = decltype(width)::value;
        if (out)
            la_pass_kernel<TI, W, true><<<grid, LA_THREADS, 0, st>>>(a);
        else
            la_pass_kernel<TI, W, false><<<grid, LA_THREADS, 0, st>>>(a);
    };
    switch (la_width(a.pass[0].dc)) {
        case 32: with(std::integral_constant<int, 32>()); break;
        case 64: with(std::integral_constant<int, 64>()); break;
        default: with(std::integral_constant<int, 128>());
    }
}

}  // namespace mogt
