// The chunked pass of linear attention (linear_attn.h has the mathematics), one
// work-group per segment and head, a wave for CT times 16 value columns: four waves
// up to 64 columns; for 128 eight of 16, with a wave's registers halved and four
// waves a SIMD (kernels of 2 x 8192 steps of 16 heads of 128 with gradients, bf16: 521 us,
// with four waves of 32 columns 533; 32768 steps, forward: 309 and 301), but where loads
// are of single elements, which take more registers: those are four of 32.
//
// Tiles (16x16 matrix instructions, D[row][column]: a lane holds column lane % 16
// and rows 4 (lane / 16) .. + 3):
//   pairs    D[s][t] = k_s . q_t, the lower triangle's tiles spread over the waves;
//            times the decay between the steps to LDS as rows t (bf16: pieces)
//   reads    D[v][t] += S q: a wave holds all rows of S for its columns in
//            accumulators, which are operands as they are
//   sums     D[v][t] += V P
//   writes   S = exp(c_T) S + K^T (w V): D[row of S][v]
// Operands that contract over steps are read transposed from LDS (bf16: the
// transposing LDS read).  S never leaves registers inside a segment.
//
// 32768 steps of 16 heads of 128, bf16: sums 75 to 82 us (268 MB; without its
// products as long), outputs 180 to 206 us (537 MB; the vector unit, which splits the
// fp32 operands, is busy for 57 % of the cycles, the matrix unit 32 %, LDS 28 %, what
// is left are the waits between the steps above).  2 x 8192 steps of 12 heads of 64:
// sums 17 us, outputs 33, two gradients with their products 66 (100 MB each).
#include "linear_attn.h"

namespace mogt {
namespace {

typedef float la_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 la_b8 __attribute__((ext_vector_type(8)));
typedef short la_s4 __attribute__((ext_vector_type(4)));
typedef uint32_t la_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t la_u2 __attribute__((ext_vector_type(2)));
typedef float la_f2 __attribute__((ext_vector_type(2)));
typedef __bf16 la_b2 __attribute__((ext_vector_type(2)));
typedef uint16_t la_h2 __attribute__((ext_vector_type(2)));

template <typename TI> struct LaOp;

// LDS rows of W elements.  bf16: 16-byte chunk c of row r lies at place c ^ f(r),
// f a bit permutation of r % 16: 16 rows' pieces of one column fall into distinct
// banks, and so do the 8 rows by 32 bytes of a transposing read.  16 bytes after
// every 16 rows keep reads of rows 16 apart from being joined into one of two
// addresses, which takes twice the time of both (measured: 16 cycles against 8;
// the passes took 3 to 6 % longer).  fp32: 16 bytes of padding a row do it all.
//
// A fragment's contraction of KS elements is held 4 by 4: lane group g (lane / 16)
// has elements 4 g .. 4 g + 3 of every 16, which is an accumulator tile's row
// order, so that a state's tiles are operands as they are.
template <> struct LaOp<bf16_t> {
    typedef la_b8 frag;
    static constexpr int PAD = 8;   // after 16 rows
    template <int W> static constexpr int size(int rows) { return rows * W + rows / 16 * PAD; }
    template <int W>
    static __device__ __forceinline__ int twist(int row) {
        constexpr int N = W / 8;   // chunks of a row
        const int i = row / (16 / N) & (N - 1);
        return (i & (N / 2 - 1)) << 1 | i / (N / 2);
    }
    template <int W>
    static __device__ __forceinline__ int at(int row, int col) { return row * W + (row >> 4) * PAD + ((((col >> 3) ^ twist<W>(row)) << 3) | (col & 7)); }
    static __device__ __forceinline__ la_f4 mma(frag a, frag b, la_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    // 32 elements of a row from column c on, of both operands of a product of rows:
    // in any order
    template <int W>
    static __device__ __forceinline__ frag any(const bf16_t* p, int row, int c, int g) {
        return *reinterpret_cast<const frag*>(p + at<W>(row, c + 8 * g));
    }
    // in the order above
    template <int W>
    static __device__ __forceinline__ frag ordered(const bf16_t* p, int row, int c, int g) {
        const la_s4 lo = *reinterpret_cast<const la_s4*>(p + at<W>(row, c + 4 * g));
        const la_s4 hi = *reinterpret_cast<const la_s4*>(p + at<W>(row, c + 16 + 4 * g));
        return __builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // rows s .. s + 31 of column 16 tile + lane % 16, in the order above
    template <int W>
    static __device__ __forceinline__ frag column(const bf16_t* p, int s, int tile, int lane) {
        const bf16_t* q = p + at<W>(s + 4 * (lane >> 4) + ((lane & 15) >> 2), 16 * tile + 4 * (lane & 3));
        typedef __attribute__((address_space(3))) la_s4* lds;
        const la_s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(q));
        const la_s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(q + 16 * W + PAD));
        return __builtin_bit_cast(frag, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    // element e of the lane's is number order(e) + 4 g of the fragment's
    static constexpr int order(int e) { return (e & 3) + 16 * (e >> 2); }
    static __device__ __forceinline__ float value(frag f, int e) { return static_cast<float>(f[e]); }
    // x as the sum of N bf16 fragments, each the rest of those before rounded
    template <int N>
    static __device__ __forceinline__ void split(float (&x)[8], frag (&out)[N]) {
#pragma unroll
        for (int p = 0; p < N; ++p) {
            la_u4 w;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector((la_f2{x[e], x[e + 1]}), la_b2));
                w[e / 2] = u;
                if (p + 1 < N) {
                    x[e] -= __uint_as_float(u << 16);
                    x[e + 1] -= __uint_as_float(u & 0xffff0000u);
                }
            }
            out[p] = __builtin_bit_cast(frag, w);
        }
    }
};

template <> struct LaOp<float> {
    typedef la_f4 frag;
    template <int W> static constexpr int size(int rows) { return rows * (W + 4); }
    template <int W>
    static __device__ __forceinline__ int at(int row, int col) { return row * (W + 4) + col; }
    static __device__ __forceinline__ la_f4 mma(frag a, frag b, la_f4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
    template <int W>
    static __device__ __forceinline__ frag any(const float* p, int row, int c, int g) {
        return *reinterpret_cast<const frag*>(p + at<W>(row, c + 4 * g));
    }
    template <int W>
    static __device__ __forceinline__ frag ordered(const float* p, int row, int c, int g) { return any<W>(p, row, c, g); }
    template <int W>
    static __device__ __forceinline__ frag column(const float* p, int s, int tile, int lane) {
        const float* q = p + at<W>(s + 4 * (lane >> 4), 16 * tile + (lane & 15));
        constexpr int N = W + 4;
        return frag{q[0], q[N], q[2 * N], q[3 * N]};
    }
    static constexpr int order(int e) { return e; }
    static __device__ __forceinline__ float value(frag f, int e) { return f[e]; }
    template <int N>
    static __device__ __forceinline__ void split(float (&x)[4], frag (&out)[N]) { out[0] = frag{x[0], x[1], x[2], x[3]}; }
};

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

// Buffer loads and stores: a lane that has nothing there goes to an offset out of
// the range, reads zero and writes nothing, without a branch.
constexpr uint32_t LA_RANGE = 0x7fffffffu, LA_OUTSIDE = 0xffffff00u;
typedef __amdgpu_buffer_rsrc_t LaBuffer;

// (The address is the same for all lanes, which the compiler cannot see past a
// division; without that it loops over the lanes at every access.)
__device__ __forceinline__ LaBuffer la_buffer(const void* p) {
    const uint64_t u = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(u)), hi = __builtin_amdgcn_readfirstlane(static_cast<int>(u >> 32));
    return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(static_cast<uint64_t>(hi) << 32 | lo), 0, LA_RANGE, 0x00020000);
}

// x, which the compiler takes for a new value: what follows from it is formed again
// where it is needed (a shift or two), not held in registers through the loop.
__device__ __forceinline__ int la_again(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The rows of a chunk on their way from memory to LDS: W elements wide, 16 bytes
// at a time over the work-group's threads, or by their halves or single elements.
template <typename TI, int W, int THREADS, int VEC>
struct LaTile {
    static constexpr int T = LaChunk<TI>::T, EPC = 16 / sizeof(TI), CPR = W / EPC;
    static constexpr int N = (T * CPR + THREADS - 1) / THREADS;
    static constexpr int STEP = THREADS / CPR;   // rows between a thread's loads
    la_u4 r[N];

    static __device__ __forceinline__ int row(int me) { return me / CPR; }
    static __device__ __forceinline__ int column(int me) { return me % CPR * EPC; }

    // Row u of the chunk, `left` of them, lies at byte first + u * step of the
    // buffer; columns from `d` on are zero.
    __device__ __forceinline__ void load(int me, LaBuffer b, int first, int step, int left, int d) {
        const int c = column(me);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int u = row(me) + i * STEP;
            const uint32_t at = static_cast<uint32_t>(first) + static_cast<uint32_t>(u) * static_cast<uint32_t>(step) + c * static_cast<uint32_t>(sizeof(TI));
            if constexpr (VEC == LA_VECTORS) {
                r[i] = __builtin_amdgcn_raw_buffer_load_b128(b, ((u < left) & (c < d)) ? at : LA_OUTSIDE, 0, 0);
            } else if constexpr (VEC == LA_HALVES) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const la_u2 w = __builtin_amdgcn_raw_buffer_load_b64(b, ((u < left) & (c + 4 * e < d)) ? at + 8 * e : LA_OUTSIDE, 0, 0);
                    r[i][2 * e] = w[0];
                    r[i][2 * e + 1] = w[1];
                }
            } else if constexpr (sizeof(TI) == 4) {
#pragma unroll
                for (int e = 0; e < EPC; ++e)
                    r[i][e] = __builtin_amdgcn_raw_buffer_load_b32(b, ((u < left) & (c + e < d)) ? at + 4 * e : LA_OUTSIDE, 0, 0);
            } else {
#pragma unroll
                for (int e = 0; e < EPC; e += 2) {
                    const uint32_t x = __builtin_amdgcn_raw_buffer_load_b16(b, ((u < left) & (c + e < d)) ? at + 2 * e : LA_OUTSIDE, 0, 0);
                    const uint32_t y = __builtin_amdgcn_raw_buffer_load_b16(b, ((u < left) & (c + e + 1 < d)) ? at + 2 * e + 2 : LA_OUTSIDE, 0, 0);
                    r[i][e / 2] = (x & 0xffffu) | y << 16;
                }
            }
        }
    }
    __device__ __forceinline__ void store(int me, TI* lds) const {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (T % STEP == 0 || row(me) + i * STEP < T)
                *reinterpret_cast<la_u4*>(lds + LaOp<TI>::template at<W>(row(me) + i * STEP, column(me))) = r[i];
    }
    // whether any element is infinite or NaN
    __device__ __forceinline__ bool wild() const {
        la_h2 m = {0, 0};   // the greatest magnitudes' upper halves (bf16: of each half)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(la_h2, r[i][j] & 0x7fff7fffu));
        return (m[1] >= 0x7f80) | (sizeof(TI) == 2 && m[0] >= 0x7f80);
    }
};

// Pieces of an fp32 operand: three bf16 hold its 24 bits.
template <typename TI> constexpr int la_pieces() { return sizeof(TI) == 2 ? 3 : 1; }

template <typename TI, int DK, int CT, int WAVES, bool OUT, int NP>
struct LaLds {
    static constexpr int T = LaChunk<TI>::T;
    typedef LaOp<TI> Op;
    TI q[OUT ? Op::template size<DK>(T) : 8];
    TI k[Op::template size<DK>(T)];
    TI v[Op::template size<16 * CT * WAVES>(T)];
    TI p[OUT ? NP : 1][OUT ? Op::template size<T>(T) : 8];
    // of this chunk and the next, in turn:
    float hi[2][T], lo[2][T];   // c_t in two parts: differences are as exact as their size
    float in[2][T], w[2][T];    // factors of the query's part and of the writes
    float end[2];               // exp(c_T)
    float g[64];
    int wild;                 // 1 + the last chunk with an infinite or NaN value
    float dot[OUT ? WAVES * T : 4];
};

// Four fp32 values rounded to TI, and what is left of them.
__device__ __forceinline__ void la_pack4(float (&x)[4], Pack<float, 4>& w, bool) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w.v[i] = x[i];
}
__device__ __forceinline__ void la_pack4(float (&x)[4], Pack<bf16_t, 4>& w, bool rest) {
    la_u2 u;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        u[i / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector((la_f2{x[i], x[i + 1]}), la_b2));
        if (rest) {
            x[i] -= __uint_as_float(u[i / 2] << 16);
            x[i + 1] -= __uint_as_float(u[i / 2] & 0xffff0000u);
        }
    }
    w = __builtin_bit_cast(Pack<bf16_t, 4>, u);
}

// OUT: the outputs (else a segment's state from zero); DOT: with their rows'
// products; VEC: the least of the roles' rows; F32: fp32 outputs.
template <typename TI, int DK, int CT, int WAVES, bool OUT, bool DOT, int VEC, bool F32>
__global__ __launch_bounds__(64 * WAVES, la_waves_per_simd(DK, CT, WAVES)) void la_pass_kernel(LaArgs a) {
    typedef LaOp<TI> Op;
    typedef typename Op::frag Frag;
    constexpr int T = LaChunk<TI>::T, KS = LaChunk<TI>::KS, NP = la_pieces<TI>();
    constexpr int TT = T / 16, RT = DK / 16, NV = 16 * CT * WAVES, THREADS = 64 * WAVES;
    constexpr int E = KS / 4, ES = static_cast<int>(sizeof(TI));
    // Wide values: the next chunk's rows are loaded once the outputs' registers are free
    // (outputs of 32768 steps of 16 heads of 128: 218 us, loaded first and spilled 239).
    constexpr bool LATE = OUT && NV > 64 && (DOT || DK > 64);
    __shared__ __align__(16) LaLds<TI, DK, CT, WAVES, OUT, NP> s;

    const int which = __builtin_amdgcn_readfirstlane(blockIdx.z / a.B), b = blockIdx.z - which * a.B, h = blockIdx.y;
    const LaPass p = a.pass[which];   // a copy: its fields are read once
    const int seg = blockIdx.x;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = la_length(a, b);
    const int64_t seq = static_cast<int64_t>(b) * a.H + h;
    // steps t0 .. t1 - 1 of the sequence; u counts them in pass order, step t0 +
    // (reverse ? cnt - 1 - u : u)
    const bool reverse = p.reverse;
    const int t0 = (reverse ? a.nseg - 1 - seg : seg) * a.seg, t1 = min(t0 + a.seg, n), cnt = max(t1 - t0, 0);
    const int dc = p.dc, dn = p.dn;

    auto rows = [&](const LaRows& r) {
        return la_buffer(static_cast<const TI*>(r.p) + b * r.batch + h / r.div * r.head + t0 * r.row);
    };
    auto step = [&](const LaRows& r) { return static_cast<int>(reverse ? -r.row : r.row) * ES; };
    const LaBuffer bq = rows(p.q), bk = rows(p.k), bv = rows(p.v);
    const int sq = step(p.q), sk = step(p.k), sv = step(p.v);
    const LaBuffer bg = la_buffer(a.g + b * a.g_batch + h * a.g_head + t0 * a.g_row);
    const int sg = static_cast<int>(a.g_row) * 4;

    // the wave's columns of the state, of which a lane has lane % 16 and those 16 on
    la_f4 S[CT][RT];
    float* slot = p.states ? p.states + (seq * (a.nseg + 1) + seg) * a.state : nullptr;
    // The lane's elements of a state with the given strides: columns of `cs` apart,
    // four rows at a time where those lie together.
    auto each_state = [&](int rs, int cs, auto&& four, auto&& one) __attribute__((always_inline)) {
        const int l = la_again(tid & 63);
        if (rs == 1 && dc % 4 == 0) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const int row = 16 * r + 4 * (l >> 4), at = 16 * (CT * wave + c) + (l & 15);
                    const uint32_t byte = static_cast<uint32_t>(row + at * cs) * 4u;
                    four(S[c][r], ((row < dc) & (at < dn)) ? byte : LA_OUTSIDE);
                }
        } else {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int r = 0; r < RT; ++r)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int row = 16 * r + 4 * (l >> 4) + i, at = 16 * (CT * wave + c) + (l & 15);
                        const uint32_t byte = static_cast<uint32_t>(row * rs + at * cs) * 4u;
                        one(S[c][r], i, ((row < dc) & (at < dn)) ? byte : LA_OUTSIDE);
                    }
        }
    };
    auto write_state = [&](float* to, int rs, int cs) __attribute__((always_inline)) {
        const LaBuffer d = la_buffer(to);
        each_state(rs, cs, [&](la_f4 x, uint32_t at) __attribute__((always_inline)) { __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(la_u4, x), d, at, 0, 0); },
                   [&](la_f4 x, int i, uint32_t at) __attribute__((always_inline)) { __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(x[i]), d, at, 0, 0); });
    };
    auto read_state = [&](const float* from, int rs, int cs) __attribute__((always_inline)) {
        const LaBuffer d = la_buffer(from);
        each_state(rs, cs, [&](la_f4& x, uint32_t at) __attribute__((always_inline)) { x = __builtin_bit_cast(la_f4, __builtin_amdgcn_raw_buffer_load_b128(d, at, 0, 0)); },
                   [&](la_f4& x, int i, uint32_t at) __attribute__((always_inline)) { x[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(d, at, 0, 0)); });
    };
#pragma unroll
    for (int c = 0; c < CT; ++c)
#pragma unroll
        for (int r = 0; r < RT; ++r) S[c][r] = la_f4{0, 0, 0, 0};
    if constexpr (OUT) {
        if (a.nseg > 1)
            read_state(slot, p.rs, p.cs);
        else if (p.init)
            read_state(p.init + seq * a.state, p.user_rs, p.user_cs);
        if (a.nseg == 1 && p.keep && slot) write_state(slot, p.rs, p.cs);
    }

    LaTile<TI, DK, THREADS, VEC> tq, tk;
    LaTile<TI, NV, THREADS, VEC> tv;
    // One wave forms a chunk's decays while the others work on the chunk before.
    constexpr int DW = WAVES - 1;
    double total = 0.0;
    auto load_decay = [&](int u0, int lane) {   // g of the lane's step
        const int u = reverse ? cnt - u0 - lane : u0 + lane;
        const bool in = (wave == DW) & (lane < T) & (lane < cnt - u0) & (t0 + u < n);
        return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(bg, in ? static_cast<uint32_t>(u * sg) : LA_OUTSIDE, 0, 0));
    };
    auto decays = [&](float g, int buf, int lane) {
        const double g2 = static_cast<double>(g) * 1.4426950408889634;
        const double c = la_wave_sums(g2 < LA_LOG2_MIN ? LA_LOG2_MIN : g2), end = la_lane(c, 63);
        const float hi = static_cast<float>(c);
        // finite factors: growth keeps a state of zeros, or rows of zeros, what they are
        auto factor = [](double x) { return __builtin_amdgcn_exp2f(static_cast<float>(x > 127.0 ? 127.0 : x)); };
        if (lane < T) {
            s.hi[buf][lane] = hi;
            s.lo[buf][lane] = static_cast<float>(c - hi);
            s.in[buf][lane] = p.qs * factor(c);
            s.w[buf][lane] = p.ws * factor(end - c);
        }
        if (lane == 0) s.end[buf] = factor(end);
        total += end;
    };
    auto load = [&](int u0, int me) {
        const int left = cnt - u0, first = reverse ? cnt - 1 - u0 : u0;
        const int row = reverse ? -first : first;   // in steps of the signed strides
        if (OUT) tq.load(me, bq, row * sq, sq, left, dc);
        tk.load(me, bk, row * sk, sk, left, dc);
        tv.load(me, bv, row * sv, sv, left, dn);
    };
    if (threadIdx.x == 0) s.wild = 0;
    if constexpr (OUT && ES == 2) {   // the tiles above the diagonal that share a fragment with one below
#pragma unroll
        for (int piece = 0; piece < NP; ++piece)
            for (int tt = 0; tt < TT; tt += 2)
                if (threadIdx.x < 256) s.p[piece][Op::template at<T>(16 * tt + (threadIdx.x >> 4), 16 * (tt + 1) + (threadIdx.x & 15))] = 0;
    }
    constexpr int OS = F32 ? 4 : ES;
    const bool writes = p.out != nullptr;
    const int64_t out_row = static_cast<int64_t>(a.H) * dn;
    const LaBuffer bo = la_buffer(static_cast<char*>(p.out) + ((b * static_cast<int64_t>(a.L) + t0) * out_row + static_cast<int64_t>(h) * dn) * OS);
    const LaBuffer bx = DOT ? rows(p.x) : bo;
    const int so = static_cast<int>(reverse ? -out_row : out_row) * OS, sx = DOT ? step(p.x) : 0;
    float* dot = DOT ? p.dot + seq * a.L + t0 : nullptr;

    float gn = load_decay(0, tid & 63);
    load(0, tid);
    if (wave == DW) decays(gn, 0, tid & 63);
    gn = load_decay(T, tid & 63);
    int buf = 0;
    for (int u0 = 0; u0 < cnt; u0 += T, buf ^= 1) {
        const int me = la_again(tid), lane = me & 63, grp = lane >> 4;
        const int c0 = 16 * CT * wave + 4 * grp;   // the lane's outputs: columns c0 .. c0 + 3, c0 + 16 .. c0 + 19
        __syncthreads();   // the last chunk's reads are done
        if (wave == DW) s.g[lane] = gn;   // of the next chunk
        if (OUT) tq.store(me, s.q);
        tk.store(me, s.k);
        tv.store(me, s.v);
        if (OUT && tv.wild()) s.wild = u0 + 1;
        __syncthreads();
        gn = load_decay(u0 + 2 * T, lane);
        if constexpr (!LATE) load(u0 + T, me);   // past the last chunk: nothing is read
        __builtin_amdgcn_sched_barrier(0);   // the loads stay here, ahead of the work that hides them
        if (wave == DW) decays(s.g[lane], buf ^ 1, lane);
        const int first = reverse ? u0 + 1 - cnt : u0;   // the chunk's first row, in steps of the signed strides
        // the lane's rows of x
        Pack<TI, 4> xr[DOT ? CT : 1][DOT ? TT : 1];
        if constexpr (DOT) {
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) {
                    const int u = 16 * tt + (lane & 15), cc = c0 + 16 * c;
                    const uint32_t at = static_cast<uint32_t>(first + u) * static_cast<uint32_t>(sx) + cc * ES;
                    if constexpr (VEC) {
                        const uint32_t o = ((u0 + u < cnt) & (cc < dn)) ? at : LA_OUTSIDE;
                        if constexpr (ES == 2)
                            xr[c][tt] = __builtin_bit_cast(Pack<TI, 4>, __builtin_amdgcn_raw_buffer_load_b64(bx, o, 0, 0));
                        else
                            xr[c][tt] = __builtin_bit_cast(Pack<TI, 4>, __builtin_amdgcn_raw_buffer_load_b128(bx, o, 0, 0));
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t o = ((u0 + u < cnt) & (cc + i < dn)) ? at + i * ES : LA_OUTSIDE;
                            if constexpr (ES == 2)
                                xr[c][tt].v[i] = __builtin_bit_cast(TI, __builtin_amdgcn_raw_buffer_load_b16(bx, o, 0, 0));
                            else
                                xr[c][tt].v[i] = __builtin_bit_cast(TI, __builtin_amdgcn_raw_buffer_load_b32(bx, o, 0, 0));
                        }
                    }
                }
        }

        la_f4 acc[CT][OUT ? TT : 1];
        if constexpr (OUT) {
            // pairs: the waves take the tiles of the lower triangle in turn; the last wave,
            // which formed the decays, has the fewest
            constexpr int TILES = TT * (TT + 1) / 2;
#pragma unroll
            for (int j = 0; j < (TILES + WAVES - 1) / WAVES; ++j) {
                if (wave + WAVES * j >= TILES) break;
                const int idx = wave + WAVES * j;
                const int tt = idx < 1 ? 0 : idx < 3 ? 1 : idx < 6 ? 2 : 3, ts = idx - tt * (tt + 1) / 2;
                la_f4 d = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < DK; k += KS)
                    d = Op::mma(Op::template any<DK>(s.k, 16 * ts + (lane & 15), k, grp), Op::template any<DK>(s.q, 16 * tt + (lane & 15), k, grp), d);
                const int t = 16 * tt + (lane & 15), s0 = 16 * ts + 4 * grp;
                const float hi = s.hi[buf][t], lo = s.lo[buf][t], ps = p.ps;
                const la_f4 shi = *reinterpret_cast<const la_f4*>(s.hi[buf] + s0), slo = *reinterpret_cast<const la_f4*>(s.lo[buf] + s0);
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = d[i] * (ps * __builtin_amdgcn_exp2f((hi - shi[i]) + (lo - slo[i])));
                    x[i] = s0 + i <= t ? y : 0.0f;
                }
#pragma unroll
                for (int piece = 0; piece < NP; ++piece) {
                    Pack<TI, 4> w;
                    la_pack4(x, w, piece + 1 < NP);
                    *reinterpret_cast<Pack<TI, 4>*>(s.p[piece] + Op::template at<T>(t, s0)) = w;
                }
            }
            // reads
#pragma unroll
            for (int c = 0; c < CT; ++c)
#pragma unroll
                for (int tt = 0; tt < TT; ++tt) acc[c][tt] = la_f4{0, 0, 0, 0};
#pragma unroll
            for (int k = 0; k < DK / KS; ++k) {
                Frag qf[TT];
#pragma unroll
                for (int tt = 0; tt < TT; ++tt)
                    qf[tt] = Op::template ordered<DK>(s.q, 16 * tt + (lane & 15), k * KS, grp);
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    Frag sp[NP];
                    float x[E];
#pragma unroll
                    for (int e = 0; e < E; ++e) x[e] = S[c][(k * KS / 16) + e / 4][e & 3];
                    Op::template split<NP>(x, sp);
#pragma unroll
                    for (int piece = 0; piece < NP; ++piece)
#pragma unroll
                        for (int tt = 0; tt < TT; ++tt) acc[c][tt] = Op::mma(sp[piece], qf[tt], acc[c][tt]);
                }
            }
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const float in = s.in[buf][16 * tt + (lane & 15)];
#pragma unroll
                for (int c = 0; c < CT; ++c) acc[c][tt] *= in;
            }
            __syncthreads();
        }

        Frag vf[CT][T / KS];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int k = 0; k < T / KS; ++k) vf[c][k] = Op::template column<NV>(s.v, KS * k, CT * wave + c, lane);
        if constexpr (OUT) {
            // sums
            if (s.wild != u0 + 1) {
#pragma unroll
                for (int k = 0; k < T / KS; ++k)
#pragma unroll
                    for (int piece = 0; piece < NP; ++piece)
#pragma unroll
                        for (int tt = KS * k / 16; tt < TT; ++tt) {
                            const Frag pf = Op::template ordered<T>(s.p[piece], 16 * tt + (lane & 15), KS * k, grp);
#pragma unroll
                            for (int c = 0; c < CT; ++c) acc[c][tt] = Op::mma(vf[c][k], pf, acc[c][tt]);
                        }
            } else {   // an infinite or NaN value must not meet the zeros of earlier steps
#pragma unroll
                for (int c = 0; c < CT; ++c)
#pragma unroll
                    for (int tt = 0; tt < TT; ++tt) {
                        const int t = 16 * tt + (lane & 15);
#pragma unroll 1
                        for (int u = 0; u <= t; ++u) {
                            float x = 0.0f;
#pragma unroll
                            for (int piece = 0; piece < NP; ++piece) x += IO<TI>::ld(s.p[piece][Op::template at<T>(t, u)]);
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                acc[c][tt][i] = fmaf(x, IO<TI>::ld(s.v[Op::template at<NV>(u, c0 + 16 * c + i)]), acc[c][tt][i]);
                        }
                    }
            }
            // the lane's rows t and columns
#pragma unroll
            for (int tt = 0; tt < TT; ++tt) {
                const int u = 16 * tt + (lane & 15);
                const bool in = writes & (u0 + u < cnt);
                float d = 0.0f;
#pragma unroll
                for (int c = 0; c < CT; ++c) {
                    const int cc = c0 + 16 * c;
                    const uint32_t at = static_cast<uint32_t>(first + u) * static_cast<uint32_t>(so) + cc * OS;
                    if constexpr (VEC) {
                        const uint32_t o = (in & (cc < dn)) ? at : LA_OUTSIDE;
                        if constexpr (F32) {
                            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(la_u4, acc[c][tt]), bo, o, 0, 0);
                        } else {
                            Pack<bf16_t, 4> w;
                            float x[4] = {acc[c][tt][0], acc[c][tt][1], acc[c][tt][2], acc[c][tt][3]};
                            la_pack4(x, w, false);
                            __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(la_u2, w), bo, o, 0, 0);
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const uint32_t o = (in & (cc + i < dn)) ? at + i * OS : LA_OUTSIDE;
                            if constexpr (F32)
                                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(acc[c][tt][i]), bo, o, 0, 0);
                            else
                                __builtin_amdgcn_raw_buffer_store_b16(f32_to_bf16(acc[c][tt][i]), bo, o, 0, 0);
                        }
                    }
                    if constexpr (DOT) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) d = fmaf(IO<TI>::ld(xr[c][tt].v[i]), acc[c][tt][i], d);
                    }
                }
                if constexpr (DOT) {
                    d += __shfl_xor(d, 16);
                    d += __shfl_xor(d, 32);
                    if (lane < 16) s.dot[wave * T + u] = d;
                }
            }
        }
        if constexpr (LATE) load(u0 + T, me);
        // writes
        const float end = s.end[buf];
#pragma unroll
        for (int c = 0; c < CT; ++c)
#pragma unroll
            for (int r = 0; r < RT; ++r) S[c][r] *= end;
#pragma unroll
        for (int k = 0; k < T / KS; ++k) {
            float w[E];
#pragma unroll
            for (int e = 0; e < E; ++e) w[e] = s.w[buf][KS * k + 4 * grp + Op::order(e)];
            Frag wv[CT][NP];
#pragma unroll
            for (int c = 0; c < CT; ++c) {
                float x[E];
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] = Op::value(vf[c][k], e) * w[e];
                Op::template split<NP>(x, wv[c]);
            }
            // products of one tile lie apart: the next waits for the last's result
            constexpr int G = RT * CT < 4 ? RT : 4 / CT;
#pragma unroll
            for (int r0 = 0; r0 < RT; r0 += G) {
                Frag kf[G];
#pragma unroll
                for (int r = 0; r < G; ++r) kf[r] = Op::template column<DK>(s.k, KS * k, r0 + r, lane);
#pragma unroll
                for (int piece = 0; piece < NP; ++piece)
#pragma unroll
                    for (int r = 0; r < G; ++r)
#pragma unroll
                        for (int c = 0; c < CT; ++c) S[c][r0 + r] = Op::mma(kf[r], wv[c][piece], S[c][r0 + r]);
            }
        }
        if constexpr (OUT && DOT) {
            __syncthreads();
            const int u = u0 + threadIdx.x;
            if (threadIdx.x < T && u < cnt) {
                float x = 0.0f;
#pragma unroll
                for (int w = 0; w < WAVES; ++w) x += s.dot[w * T + threadIdx.x];
                dot[reverse ? cnt - 1 - u : u] = x;
            }
        }
    }

    if constexpr (OUT) {
        // rows past the sequence's length
        if (p.out) {
            const int from = max(t0, n), to = min(t0 + a.seg, a.L);
            for (int i = threadIdx.x; i < (to - from) * dn; i += THREADS) {
                const int64_t t = from + i / dn;
                const int64_t at = (b * static_cast<int64_t>(a.L) + t) * out_row + static_cast<int64_t>(h) * dn + i % dn;
                if constexpr (F32)
                    static_cast<float*>(p.out)[at] = 0.0f;
                else
                    static_cast<TI*>(p.out)[at] = IO<TI>::st(0.0f);
            }
        }
        if (seg == a.nseg - 1) {   // the sequence's last state
            if (p.keep && slot) write_state(slot + a.state, p.rs, p.cs);
            if (p.last) write_state(p.last + seq * a.state, p.user_rs, p.user_cs);
        }
    } else {   // the segment's own
        if (threadIdx.x == 64 * DW) p.ctot[seq * a.nseg + seg] = static_cast<float>(total);
        write_state(slot + a.state, p.rs, p.cs);
    }
}

}  // namespace

// Launches the passes `pass[0 .. count - 1]` of `a`, which are of one kind
// (la_one_kind).
template <typename TI>
void la_launch_passes(const LaArgs& a, int count, bool out, hipStream_t st) {
    int vec = LA_VECTORS;
    for (int i = 0; i < count; ++i) {
        const LaPass& p = a.pass[i];
        vec = min(vec, min(p.k.vec, p.v.vec));
        if (out) vec = min(vec, min(p.q.vec, p.dot ? p.x.vec : vec));
        if (out && reinterpret_cast<uintptr_t>(p.out) % 16 != 0) vec = LA_SINGLE;
    }
    const bool dot = out && a.pass[0].dot, f32 = out && a.pass[0].out_f32;
    const dim3 grid(out ? a.nseg : a.nseg - 1, a.H, static_cast<unsigned>(a.B) * count);
    auto with = [&](auto width, auto tiles, auto waves, auto whole) {
        constexpr int W = decltype(width)::value, N = decltype(tiles)::value, G = decltype(waves)::value;
        constexpr int V = decltype(whole)::value;
        constexpr bool F = sizeof(TI) == 4;
        if (!out)
            la_pass_kernel<TI, W, N, G, false, false, V, F><<<grid, 64 * G, 0, st>>>(a);
        else if (dot && f32)
            la_pass_kernel<TI, W, N, G, true, true, V, true><<<grid, 64 * G, 0, st>>>(a);
        else if (dot)
            la_pass_kernel<TI, W, N, G, true, true, V, F><<<grid, 64 * G, 0, st>>>(a);
        else
            la_pass_kernel<TI, W, N, G, true, false, V, F><<<grid, 64 * G, 0, st>>>(a);
    };
    typedef std::integral_constant<int, 1> one;
    typedef std::integral_constant<int, 2> two;
    typedef std::integral_constant<int, 4> four;
    typedef std::integral_constant<int, 8> eight;
    typedef std::integral_constant<int, LA_SINGLE> single;
    typedef std::integral_constant<int, sizeof(TI) == 2 ? LA_HALVES : LA_VECTORS> halves;
    typedef std::integral_constant<int, LA_VECTORS> vectors;
    auto pick = [&](auto width) {
        const bool narrow = !la_wide(a.pass[0].dn);
        if (vec == LA_VECTORS)
            narrow ? with(width, one(), four(), vectors()) : with(width, one(), eight(), vectors());
        else if (vec == LA_HALVES)
            narrow ? with(width, one(), four(), halves()) : with(width, one(), eight(), halves());
        else
            narrow ? with(width, one(), four(), single()) : with(width, two(), four(), single());
    };
    switch (la_width(a.pass[0].dc)) {
        case 32: pick(std::integral_constant<int, 32>()); break;
        case 64: pick(std::integral_constant<int, 64>()); break;
        default: pick(std::integral_constant<int, 128>());
    }
}

}  // namespace mogt
