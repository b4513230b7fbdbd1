// Matrix product on e4m3 operands with scales for blocks of 128 along K:
//   y[m][n] = sum_kb xs[m][kb] ws[n / 128][kb] sum_{k in block kb} x[m][k] w[n][k]
// x [M, K] with a scale for every row's block, w [N, K] with one for every 128 rows'
// block.  A block's products are added by one matrix instruction (16x16x128) into
// zeros, the block's sum is scaled and added in fp32 on the vector unit.
//
// The 8-bit instruction aligns the products it adds to the largest: a block's sum is
// off by up to 2^-13 of the sum of their magnitudes (1.4e-5 of it on normal rows, the
// same for the form of 32 values), which bf16 outputs of many rows take for twice the
// rate.  fp32 outputs and few rows (EXACT) widen the operands to bf16, which holds every
// e4m3 value, and add with the bf16 instruction to fp32's own accuracy.
//
// Tiles: a work-group of MW x NW waves, a wave 16 MT rows of x by 16 NT rows of w.
// D[row of w][row of x]: a lane's results are four consecutive outputs of one row,
// its row's scale one factor.  Stages of one block of K, two in LDS, filled by
// direct loads: 128-byte rows, their 16-byte chunks at places that give no bank
// conflicts (f8_twist).  A lane's 32 values of an operand are chunks g and g + 4 (g = lane /
// 16), the same of both operands, which is an order of the sum only.  Rows past the
// end and chunks past K load zeros.
//
// Up to 32 rows (one token of a batch): the weights are read once, straight into
// registers, by waves of 16 rows of w that share K; bound by their bytes.
//
// 32768 x 6144 x 2048 takes 406 to 438 us on different cards (2.03 to 1.88 PFLOP/s;
// torch's unscaled e4m3 product 340, its bf16 product 583), to fp32 794 to 829.  In a row
// of calls the card's power bounds it: of zeros the same product takes 360 us.  The matrix
// unit is busy for 43 % of the cycles, the vector unit, which adds 4 scaled results a
// product, for 40 %, LDS for 23 %; no order of loads, reads and products that was tried
// changes the time by more than 2 %.  To fp32 every wave widens the operands that it reads.
#include "lds_dma.h"
#include "wide_grid.h"

namespace mogt {
namespace {

typedef int f8_i8 __attribute__((ext_vector_type(8)));
typedef int f8_i4 __attribute__((ext_vector_type(4)));
typedef int f8_i2 __attribute__((ext_vector_type(2)));
typedef float f8_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 f8_b8 __attribute__((ext_vector_type(8)));
typedef __bf16 f8_b2 __attribute__((ext_vector_type(2)));

struct F8Gemm {
    const uint8_t *x, *w;
    const float *xs, *ws;
    void* y;
    int64_t M, ldx, ldy;
    int N, K, kb;
    int nm, nn;          // tiles
    int piece;           // bytes of a store: the most that rows of y are whole in, up to 16; 0: a tile's lie beyond 2^31 bytes
};

// A weight block's scale as 2^h times what is left, which is in [1, 2) for h of -100 to
// 103.  2^h goes to the operand (`power`: as the matrix instruction's 8-bit exponent, or
// as a float for the conversion to bf16), so that the row's scale times `rest` and the
// block's sum are normal numbers wherever the scaled sum is one: sums are 2^-18 to 2^25.
// (Both scales in one factor were subnormal for rows of 1e-36, and infinite times a sum
// of zero above 2^128.  Now only a row's scale above 2^110 times a block's above 2^103 is:
// those of sums that are not zero are infinite.)
struct F8Scale {
    float rest;
    int power;
};
template <bool EXACT> constexpr int F8_ONE = EXACT ? 127 << 23 : 127;
template <bool EXACT>
__device__ __forceinline__ F8Scale f8_part(float s) {
    const int e = __float_as_int(s) >> 23 & 255, h = min(max(e, 27), 230);
    return F8Scale{__builtin_ldexpf(s, 127 - h), EXACT ? h << 23 : h};
}

// An operand's 32 values of a lane as the matrix instruction takes them, times 2^h.
template <bool EXACT> struct F8Operand;
template <> struct F8Operand<false> {
    f8_i8 v;
    int power;
    __device__ __forceinline__ F8Operand() {}
    __device__ __forceinline__ F8Operand(f8_i4 lo, f8_i4 hi, int power)
        : v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, power(power) {}
};
template <> struct F8Operand<true> {
    f8_b8 v[4];
    __device__ __forceinline__ F8Operand() {}
    __device__ __forceinline__ F8Operand(f8_i4 lo, f8_i4 hi, int power) {
        const float scale = __int_as_float(power);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int u = i < 2 ? lo[2 * i + j] : hi[2 * i - 4 + j];
                const f8_b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, scale, false);
                const f8_b2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, scale, true);
                v[i][4 * j] = a[0];
                v[i][4 * j + 1] = a[1];
                v[i][4 * j + 2] = b[0];
                v[i][4 * j + 3] = b[1];
            }
    }
};

// the block's product of 16 rows of w by 16 rows of x
__device__ __forceinline__ f8_f4 f8_block(const F8Operand<false>& w, const F8Operand<false>& x) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, f8_f4{0, 0, 0, 0}, 0, 0, 0, w.power, 0, x.power);
}
__device__ __forceinline__ f8_f4 f8_block(const F8Operand<true>& w, const F8Operand<true>& x) {
    f8_f4 d = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], d, 0, 0, 0);
    return d;
}

// x, which the compiler takes for a new value: what follows from it is formed again
// where it is needed, not held in registers from tile to tile.
__device__ __forceinline__ int f8_again(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

// Chunk c of row r lies at place c ^ f8_twist(r): the 16 rows of a fragment's reads, two
// rows to the banks' width, fall into distinct banks.
__device__ __forceinline__ int f8_twist(int row) { return (row >> 1) & 7; }

template <bool F32>
__device__ __forceinline__ void f8_store(const F8Gemm& p, int64_t m, int n, f8_f4 v) {
    typedef typename std::conditional<F32, float, bf16_t>::type T;
    T* y = static_cast<T*>(p.y) + m * p.ldy + n;
    if (n + 4 <= p.N && p.ldy % 4 == 0) {
        Pack<T, 4> w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w.v[i] = IO<T>::st(v[i]);
        *reinterpret_cast<Pack<T, 4>*>(y) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.N) y[i] = IO<T>::st(v[i]);
    }
}

// `B` bytes from LDS to byte `at` of the buffer (an offset out of its range writes nothing)
template <int B>
__device__ __forceinline__ void f8_store_piece(const char* from, __amdgpu_buffer_rsrc_t to, uint32_t at) {
    if constexpr (B == 16)
        __builtin_amdgcn_raw_buffer_store_b128(*reinterpret_cast<const f8_i4*>(from), to, at, 0, 0);
    else if constexpr (B == 8)
        __builtin_amdgcn_raw_buffer_store_b64(*reinterpret_cast<const f8_i2*>(from), to, at, 0, 0);
    else if constexpr (B == 4)
        __builtin_amdgcn_raw_buffer_store_b32(*reinterpret_cast<const int*>(from), to, at, 0, 0);
    else
        __builtin_amdgcn_raw_buffer_store_b16(*reinterpret_cast<const int16_t*>(from), to, at, 0, 0);
}

// Tiles of work-group `bid` of `grid` (a multiple of 8, or all of n): its XCD (ids
// mod 8) takes a run of them, dealt to the XCD's work-groups in turn.
struct F8Walk {
    int next, step, end;
};
__device__ __forceinline__ F8Walk f8_walk(int n, int grid, int bid) {
    const int xcd = bid % 8, q = n / 8, rem = n % 8;
    const int first = xcd * q + min(xcd, rem);
    return F8Walk{first + bid / 8, (grid - xcd + 7) / 8, first + q + (xcd < rem ? 1 : 0)};
}

template <int MW, int NW, int MT, int NT, bool EXACT>
__global__ __launch_bounds__(64 * MW * NW) void f8_gemm_kernel(F8Gemm p) {
    typedef typename std::conditional<EXACT, float, bf16_t>::type TO;
    constexpr int BM = MW * MT * 16, BN = NW * NT * 16, WAVES = MW * NW, ROWS = BM + BN;
    constexpr int LOADS = ROWS / 8 / WAVES;   // 1 KB loads of a wave and stage
    constexpr int STAGE = ROWS * 128, OUTSIDE = 0x7ffffff0;
    static_assert(BM / 8 % WAVES == 0 && BN / 8 % WAVES == 0 && NT * 16 <= 128 && 128 % (NT * 16) == 0, "tile");
    static_assert(LOADS <= MT * NT, "a load beside each product");
    static_assert(WAVES % 2 == 0, "a wave's loads fill rows of one parity of eights");
    __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE];
    __shared__ float s_xs[2][BM];   // scales of the rows of x
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), grp = lane >> 4;
    const int wm = wave / NW, wn = wave % NW;
    const uint32_t lds0 = lds_addr(smem);
    const int twist = f8_twist(lane & 15);   // of every row the lane reads: they are 16 apart
    // place lane % 8 of row lane / 8 of a load takes the chunk that the twist puts there
    const int ch = ((lane & 7) ^ f8_twist((wave & 1) * 8 + (lane >> 3))) * 16;

    // the tile whose stages are being loaded
    int64_t m0;
    int n0, off[LOADS];
    lds_i32x4 rx, rw;
    const float *xs, *ws;
    auto enter = [&](int v) __attribute__((always_inline)) {
        // eight row blocks at a time (an XCD's L2 keeps their rows)
        const int group = 8 * p.nn, g = v / group, gm = min(p.nm - 8 * g, 8), in = v - g * group;
        const int mb = __builtin_amdgcn_readfirstlane(8 * g + in % gm), nb = __builtin_amdgcn_readfirstlane(in / gm);
        m0 = static_cast<int64_t>(mb) * BM;
        n0 = nb * BN;
        const int mrows = static_cast<int>(min(p.M - m0, static_cast<int64_t>(BM))), nrows = min(p.N - n0, BN), l = f8_again(lane);
        rx = lds_rsrc(p.x + m0 * p.ldx, static_cast<uint32_t>((mrows - 1) * p.ldx + p.K));
        rw = lds_rsrc(p.w + static_cast<int64_t>(n0) * p.K, static_cast<uint32_t>(nrows) * p.K);
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = (i * WAVES + wave) * 8 + (l >> 3);   // rows of x, then of w
            if (i < BM / 8 / WAVES)
                off[i] = r < mrows ? static_cast<int>(r * p.ldx) + ch : OUTSIDE;
            else
                off[i] = r - BM < nrows ? (r - BM) * p.K + ch : OUTSIDE;
        }
        // scales: a thread's row of x, and the wave's rows of w
        xs = p.xs + min(m0 + tid % BM, p.M - 1) * p.kb;
        ws = p.ws + static_cast<int64_t>(min(n0 + wn * NT * 16, p.N - 1) / 128) * p.kb;
    };
    float sx, sw;
    // load i of stage s of the tile into buffer `buf` (s < 0: none left, nothing is read)
    auto issue = [&](int i, int s, int buf) __attribute__((always_inline)) {
        const bool in = (s >= 0) & (s * 128 + ch < p.K) & (off[i] != OUTSIDE);
        lds_dma16(i < BM / 8 / WAVES ? rx : rw, in ? off[i] + s * 128 : OUTSIDE, 0,
                  lds0 + buf * STAGE + (i * WAVES + wave) * 1024);
    };

    F8Walk walk = f8_walk(p.nm * p.nn, gridDim.x, blockIdx.x);
    if (walk.next >= walk.end) return;
    enter(walk.next);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) issue(i, 0, 0);
    sw = ws[0];
    sx = xs[0];
    // stores of the tile before, issued after this one's first loads
    constexpr int OUT_ROW = NT * 16 * sizeof(TO), CH = OUT_ROW / 16, STORES = MT * 16 * OUT_ROW / 1024;
    bool stored = false;
    int buf = 0;
    while (true) {
        const int64_t m1 = m0;   // the tile being multiplied
        const int n1 = n0;
        const bool more = walk.next + walk.step < walk.end;
        f8_f4 acc[MT][NT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = f8_f4{0, 0, 0, 0};
        for (int s = 0; s < p.kb; ++s, buf ^= 1) {
            if (BM == 64 * WAVES || tid < BM) s_xs[buf][tid % BM] = sx;
            const F8Scale wscale = f8_part<EXACT>(sw);
            if (s == 0 && stored)
                lds_wait_vm<STORES>();
            else
                lds_wait_vm<0>();
            __syncthreads();
            // the lane's two chunks of a row, which lie 64 bytes apart (bit 2 of the place)
            const char* lo = smem + buf * STAGE + (lane & 15) * 128 + ((grp ^ twist) << 4);
            const char* hi = smem + buf * STAGE + (lane & 15) * 128 + (((grp ^ twist) << 4) ^ 64);
            auto frag = [&](int r, int power) __attribute__((always_inline)) {
                return F8Operand<EXACT>(*reinterpret_cast<const f8_i4*>(lo + r * 128), *reinterpret_cast<const f8_i4*>(hi + r * 128), power);
            };
            const float* const xscale = s_xs[buf] + wm * MT * 16 + (lane & 15);
            float f[MT];
            F8Operand<EXACT> w[NT], x[2];
#pragma unroll
            for (int j = 0; j < NT; ++j) w[j] = frag(BM + (wn * NT + j) * 16, wscale.power);
            x[0] = frag(wm * MT * 16, F8_ONE<EXACT>);
#pragma unroll
            for (int i = 0; i < MT; ++i) f[i] = xscale[16 * i] * wscale.rest;
            // the stage that loads meanwhile: this tile's next, or the next tile's first
            int stage = s + 1;
            if (stage == p.kb) {
                stage = more ? 0 : -1;
                if (more) {
                    walk.next += walk.step;
                    enter(walk.next);
                }
            }
            if (stage >= 0) {
                sw = ws[stage];
                sx = xs[stage];
            }
            __builtin_amdgcn_sched_barrier(0);
            // A product's result is there some 12 cycles after the next one has begun: it is
            // scaled three products later.  The order is held, or each would be waited for.
            constexpr int LAG = 3;
            f8_f4 d[LAG + 1];
#pragma unroll
            for (int t = 0; t < MT * NT + LAG; ++t) {
                if (t < MT * NT) {
                    const int i = t / NT, j = t % NT;
                    if (j == 0 && i + 1 < MT) x[(i + 1) & 1] = frag((wm * MT + i + 1) * 16, F8_ONE<EXACT>);
                    d[t % (LAG + 1)] = f8_block(w[j], x[i & 1]);
                }
                if (t < LOADS) issue(t, stage, buf ^ 1);
                if (t >= LAG) {
                    const int u = t - LAG, i = u / NT, j = u % NT;
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[u % (LAG + 1)][e], f[i], acc[i][j][e]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (p.piece) {
            // Through the last stage's LDS (no wave reads it any more), so that a row of the
            // wave's leaves in whole lines: straight from the registers 16 rows' 32 bytes a
            // store took 33 us a tile, more than its sixteen stages.  Rows that are not whole
            // 16 bytes leave in smaller pieces, coalesced all the same (4096 x 4098 x 2048, bf16:
            // 71 us, straight from the registers 100; 13577 x 3919 x 864: 107, 154).
            constexpr int ROOM = STAGE / WAVES / (16 * OUT_ROW), G = ROOM >= MT ? MT : ROOM >= 4 ? 4 : ROOM >= 2 ? 2 : 1;
            static_assert(ROOM >= 1 && MT % G == 0, "a tile's rows fit");
            __syncthreads();
            const int l = f8_again(lane);
            char* const mine = smem + (buf ^ 1) * STAGE + wave * (STAGE / WAVES / 16 * 16);
            const int left = static_cast<int>(min(p.M - m1, static_cast<int64_t>(BM))) - wm * MT * 16, nw = p.N - n1 - wn * NT * 16;
            const int ldy = static_cast<int>(p.ldy);
            const auto ry = __builtin_amdgcn_make_buffer_rsrc(
                static_cast<char*>(p.y) + (m1 * p.ldy + n1) * static_cast<int64_t>(sizeof(TO)), 0, 0x7fffffff, 0x00020000);
#pragma unroll
            for (int i0 = 0; i0 < MT; i0 += G) {
#pragma unroll
                for (int i = 0; i < G; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const int r = 16 * i + (l & 15), byte = (16 * j + 4 * (l >> 4)) * static_cast<int>(sizeof(TO));
                        Pack<TO, 4> v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v.v[e] = IO<TO>::st(acc[i0 + i][j][e]);
                        *reinterpret_cast<Pack<TO, 4>*>(mine + r * OUT_ROW + ((byte >> 4 ^ (r & (CH - 1))) << 4) + (byte & 15)) = v;
                    }
                // only the wave's own rows: its reads wait for its writes
                auto leave = [&](auto piece) __attribute__((always_inline)) {
                    constexpr int B = decltype(piece)::value, PR = OUT_ROW / B;   // pieces of a row
#pragma unroll 4
                    for (int k = 0; k < G * 16 * OUT_ROW / (64 * B); ++k) {
                        const int id = 64 * k + l, r = id / PR, byte = id % PR * B;
                        const int m = 16 * i0 + r, n = byte / static_cast<int>(sizeof(TO));
                        const uint32_t at = static_cast<uint32_t>((wm * MT * 16 + m) * ldy + wn * NT * 16 + n) * static_cast<uint32_t>(sizeof(TO));
                        const bool in = (m < left) & (n < nw);
                        f8_store_piece<B>(mine + r * OUT_ROW + ((byte >> 4 ^ (r & (CH - 1))) << 4) + (byte & 15), ry, in ? at : 0xffffff00u);
                    }
                };
                if (p.piece == 16)
                    leave(std::integral_constant<int, 16>());
                else if (p.piece == 8)
                    leave(std::integral_constant<int, 8>());
                else if (EXACT || p.piece == 4)
                    leave(std::integral_constant<int, 4>());
                else
                    leave(std::integral_constant<int, 2>());
            }
            stored = true;
        } else {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int64_t m = m1 + (wm * MT + i) * 16 + (lane & 15);
                if (m >= p.M) continue;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const int n = n1 + (wn * NT + j) * 16 + 4 * grp;
                    if (n < p.N) f8_store<EXACT>(p, m, n, acc[i][j]);
                }
            }
        }
        if (!more) return;
    }
}

// Few rows: a work-group's four waves take every fourth block of K of 16 rows of w, with
// the bf16 instruction for both outputs: the weights' bytes bound it, not the products
// (2048 columns by 6144, 8-bit and bf16 instruction: 16 rows 7.2 and 7.4 us, 32 rows 10.1
// and 10.2; 4096 by 32768, one row: 28.8 and 29.9).
template <int MT, bool F32>
__global__ __launch_bounds__(256) void f8_gemv_kernel(F8Gemm p) {
    __shared__ f8_f4 s_d[4][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grp = lane >> 4;
    const int n0 = min(static_cast<int>(wide_block()), (p.N - 1) / 16) * 16;   // work-groups too many repeat the last
    const uint8_t* wr = p.w + static_cast<int64_t>(min(n0 + (lane & 15), p.N - 1)) * p.K;
    const float* ws = p.ws + static_cast<int64_t>(n0 / 128) * p.kb;
    const uint8_t* xr[MT];
    const float* xs[MT];
    f8_f4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = min(static_cast<int64_t>(16 * i + (lane & 15)), p.M - 1);
        xr[i] = p.x + m * p.ldx;
        xs[i] = p.xs + m * p.kb;
        acc[i] = f8_f4{0, 0, 0, 0};
    }
    auto frag = [&](const uint8_t* row, int s, int power) {
        const int k = s * 128 + 16 * grp;
        f8_i4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        if (k < p.K) lo = *reinterpret_cast<const f8_i4*>(row + k);
        if (k + 64 < p.K) hi = *reinterpret_cast<const f8_i4*>(row + k + 64);
        return F8Operand<true>(lo, hi, power);
    };
#pragma unroll 4
    for (int s = wave; s < p.kb; s += 4) {
        const F8Scale wscale = f8_part<true>(ws[s]);
        const F8Operand<true> w = frag(wr, s, wscale.power);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const f8_f4 d = f8_block(w, frag(xr[i], s, F8_ONE<true>));
            const float f = xs[i][s] * wscale.rest;
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(d[e], f, acc[i][e]);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) s_d[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < MT; i += 4) {
        const f8_f4 d = (s_d[0][i][lane] + s_d[1][i][lane]) + (s_d[2][i][lane] + s_d[3][i][lane]);
        const int64_t m = 16 * i + (lane & 15);
        const int n = n0 + 4 * grp;
        if (m < p.M && n < p.N) f8_store<F32>(p, m, n, d);
    }
}

template <bool EXACT>
void f8_launch(F8Gemm& p, int cus, hipStream_t st) {
    if (p.M <= 32) {
        const dim3 grid = wide_grid((p.N + 15) / 16);
        if (p.M <= 16)
            f8_gemv_kernel<1, EXACT><<<grid, 256, 0, st>>>(p);
        else
            f8_gemv_kernel<2, EXACT><<<grid, 256, 0, st>>>(p);
        return;
    }
    auto tiles = [&](int bm, int bn) {
        p.nm = static_cast<int>((p.M + bm - 1) / bm);
        p.nn = (p.N + bn - 1) / bn;
        return p.nm * p.nn;
    };
    // The largest tile that fills the card: of 2048 columns of x (us, bf16 and fp32 outputs)
    //                 256 x 256, 128 x 256     128 x 128        64 x 128
    //   8192 x 6144   111      214             135  219         166  276
    //   4096 x 6144    66      108              68  109          84  141
    //   2048 x 6144    35       66              37   55          43   72
    //   4096 x 2048    33       38              26   39          32   46
    //   1024 x 6144    32       37              23   37          24   38
    //   2048 x 2048    32       34              18   26          18   26
    //     64 x 6144    28       31              15   22          11   16
    // and up to 32 rows the form without tiles: 32 x 6144 10.0 against 10.8 and 15.5, 16 x
    // 6144 7.2 against 10.8 and 15.3.
    const int each = EXACT ? 4 : 2;
    const int64_t row = p.ldy * each;
    p.piece = row * 256 >= 0x7fffff00 ? 0 : row % 16 == 0 ? 16 : row % 8 == 0 ? 8 : row % 4 == 0 ? 4 : 2;
    constexpr int BM = EXACT ? 128 : 256;
    if (tiles(BM, 256) >= (EXACT ? 2 * cus : cus * 3 / 4)) {
        const int n = tiles(BM, 256);
        f8_gemm_kernel<2, 4, BM / 32, 4, EXACT><<<n < cus ? n : cus, 512, 0, st>>>(p);
    } else if (tiles(128, 128) >= cus) {
        const int n = tiles(128, 128);
        f8_gemm_kernel<2, 2, 4, 4, EXACT><<<n < 2 * cus ? n : 2 * cus, 256, 0, st>>>(p);
    } else {
        const int n = tiles(64, 128);
        f8_gemm_kernel<2, 2, 2, 4, EXACT><<<n < 3 * cus ? n : 3 * cus, 256, 0, st>>>(p);
    }
}

}  // namespace
}  // namespace mogt

using namespace mogt;

extern "C" int mogt_linear_fp8(const void* x, int64_t ldx, const float* x_scale, const void* w, const float* w_scale,
                               void* y, int64_t rows, int64_t outputs, int64_t width, int out_dtype, void* stream) {
    clear_error();
    if (rows < 0 || outputs < 0 || width < 16 || width % 16 != 0 || ldx < width || ldx % 16 != 0)
        return set_error(MOGT_E_INVALID, "rows %lld of %lld (stride %lld), %lld outputs: a width and stride of whole 16 expected",
                         (long long)rows, (long long)width, (long long)ldx, (long long)outputs);
    if (out_dtype != MOGT_F32 && out_dtype != MOGT_BF16)
        return set_error(MOGT_E_INVALID, "output dtype %d not supported", out_dtype);
    if (ldx > (1 << 22) || outputs > (1 << 30) || rows > (1ll << 37))
        return set_error(MOGT_E_INVALID, "row stride %lld (at most 2^22), %lld outputs (2^30) or %lld rows (2^37) too large",
                         (long long)ldx, (long long)outputs, (long long)rows);
    if ((rows + 63) / 64 * ((outputs + 127) / 128) > 0x7fffffff)
        return set_error(MOGT_E_INVALID, "%lld rows by %lld outputs are too many tiles", (long long)rows, (long long)outputs);
    if (rows == 0 || outputs == 0) return MOGT_OK;
    if (!x || !x_scale || !w || !w_scale || !y) return set_error(MOGT_E_INVALID, "null pointer");
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(y)) & 15)
        return set_error(MOGT_E_INVALID, "operands and output must be 16-byte aligned");
    F8Gemm p{static_cast<const uint8_t*>(x), static_cast<const uint8_t*>(w), x_scale, w_scale, y, rows, ldx, outputs,
             static_cast<int>(outputs), static_cast<int>(width), static_cast<int>((width + 127) / 128), 0, 0, 0};
    int cus = 0;
    if (const int rc = device_cu_count(cus)) return rc;
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (out_dtype == MOGT_F32)
        f8_launch<true>(p, cus, st);
    else
        f8_launch<false>(p, cus, st);
    return check_launch("mogt_linear_fp8");
}
