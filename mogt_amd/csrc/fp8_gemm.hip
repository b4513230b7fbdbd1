// Matrix product on e4m3 operands with scales for blocks of 128 along K:
//   y[m][n] = sum_kb xs[m][kb] ws[n / 128][kb] sum_{k in block kb} x[m][k] w[n][k]
// x [M, K] with a scale for every row's block, w [N, K] with one for every 128 rows'
// block.  A block's products are added by one matrix instruction (16x16x128) into
// zeros, the block's sum is scaled and added in fp32 on the vector unit.
//
// The 8-bit instruction aligns the products it adds: a block's sum is off by about
// 1.4e-5 of it (measured on normal rows, the same for its form of 32 values), which
// a bf16 output does not show.  fp32 outputs (EXACT) widen the operands to bf16, which
// holds every e4m3 value, and add with the bf16 instruction, at half the rate, to
// fp32's own accuracy.
//
// Tiles: a work-group of MW x NW waves, a wave 16 MT rows of x by 16 NT rows of w.
// D[row of w][row of x]: a lane's results are four consecutive outputs of one row,
// its row's scale one factor.  Stages of one block of K, two in LDS, filled by
// direct loads: 128-byte rows, their 16-byte chunks at places that give no bank
// conflicts (f8_twist).  A lane's 32 values of an operand are chunks g and g + 4 (g = lane /
// 16), the same of both operands, which is an order of the sum only.  Rows past the
// end and chunks past K load zeros.
//
// Up to 64 rows (one token of a batch): the weights are read once, straight into
// registers, by waves of 16 rows of w that share K; bound by their bytes.
#include "lds_dma.h"

namespace mogt {
namespace {

typedef int f8_i8 __attribute__((ext_vector_type(8)));
typedef int f8_i4 __attribute__((ext_vector_type(4)));
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
};

// An operand's 32 values of a lane as the matrix instruction takes them.
template <bool EXACT> struct F8Operand;
template <> struct F8Operand<false> {
    f8_i8 v;
    __device__ __forceinline__ F8Operand() {}
    __device__ __forceinline__ F8Operand(f8_i4 lo, f8_i4 hi) : v{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]} {}
};
template <> struct F8Operand<true> {
    f8_b8 v[4];
    __device__ __forceinline__ F8Operand() {}
    __device__ __forceinline__ F8Operand(f8_i4 lo, f8_i4 hi) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int u = i < 2 ? lo[2 * i + j] : hi[2 * i - 4 + j];
                const f8_b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, false);
                const f8_b2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, 1.0f, true);
                v[i][4 * j] = a[0];
                v[i][4 * j + 1] = a[1];
                v[i][4 * j + 2] = b[0];
                v[i][4 * j + 3] = b[1];
            }
    }
};

// the block's product of 16 rows of w by 16 rows of x
__device__ __forceinline__ f8_f4 f8_block(const F8Operand<false>& w, const F8Operand<false>& x) {
    // scales of one (2^(127 - 127))
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w.v, x.v, f8_f4{0, 0, 0, 0}, 0, 0, 0, 0x7f7f7f7f, 0, 0x7f7f7f7f);
}
__device__ __forceinline__ f8_f4 f8_block(const F8Operand<true>& w, const F8Operand<true>& x) {
    f8_f4 d = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w.v[i], x.v[i], d, 0, 0, 0);
    return d;
}

// Chunk c of row r lies at place c ^ f8_twist(r): the 16 rows of a fragment's reads, two
// rows to the banks' width, fall into distinct banks.
__device__ __forceinline__ int f8_twist(int row) { return (row >> 1) & 7; }

template <bool EXACT>
__device__ __forceinline__ void f8_store(const F8Gemm& p, int64_t m, int n, f8_f4 v) {
    typedef typename std::conditional<EXACT, float, bf16_t>::type T;
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

template <int MW, int NW, int MT, int NT, bool EXACT>
__global__ __launch_bounds__(64 * MW * NW) void f8_gemm_kernel(F8Gemm p) {
    constexpr int BM = MW * MT * 16, BN = NW * NT * 16, WAVES = MW * NW, ROWS = BM + BN;
    constexpr int LOADS = ROWS / 8 / WAVES;   // 1 KB loads of a wave and stage
    static_assert(BM / 8 % WAVES == 0 && BN / 8 % WAVES == 0 && NT * 16 <= 128 && 128 % (NT * 16) == 0, "tile");
    __shared__ __attribute__((aligned(1024))) char smem[2 * ROWS * 128];
    __shared__ float s_xs[2][BM];   // scales of the rows of x
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), grp = lane >> 4;
    const int wm = wave / NW, wn = wave % NW;
    // an XCD takes a run of tiles, eight row blocks at a time (its L2 keeps their rows)
    int mb, nb;
    {
        const int n = p.nm * p.nn, xcd = blockIdx.x % 8, loc = blockIdx.x / 8, q = n / 8, rem = n % 8;
        const int v = (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + loc;
        const int group = 8 * p.nn, g = v / group, gm = min(p.nm - 8 * g, 8), in = v - g * group;
        mb = 8 * g + in % gm;
        nb = in / gm;
    }
    const int64_t m0 = static_cast<int64_t>(mb) * BM;
    const int n0 = nb * BN;
    const int mrows = static_cast<int>(min(p.M - m0, static_cast<int64_t>(BM))), nrows = min(p.N - n0, BN);
    const lds_i32x4 rx = lds_rsrc(p.x + m0 * p.ldx, static_cast<uint32_t>((mrows - 1) * p.ldx + p.K));
    const lds_i32x4 rw = lds_rsrc(p.w + static_cast<int64_t>(n0) * p.K, static_cast<uint32_t>(nrows) * p.K);
    const uint32_t lds0 = lds_addr(smem);
    // lane's place lane % 8 of row 8 i + lane / 8 takes the chunk that the twist puts there
    int chunk[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) chunk[i] = ((lane & 7) ^ f8_twist(8 * i + (lane >> 3))) * 16;
    constexpr int OUTSIDE = 0x7ffffff0;
    static_assert(WAVES % 2 == 0, "rows of one parity of eight a wave");
    const int ch = chunk[0] * (1 - (wave & 1)) + chunk[1] * (wave & 1);   // 8 (i WAVES + wave) rows on: the wave's parity
    int off[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = (i * WAVES + wave) * 8 + (lane >> 3);   // rows of x, then of w
        if (i < BM / 8 / WAVES)
            off[i] = r < mrows ? static_cast<int>(r * p.ldx) + ch : OUTSIDE;
        else
            off[i] = r - BM < nrows ? (r - BM) * p.K + ch : OUTSIDE;
    }
    auto issue = [&](int s) {
        const bool in = s * 128 + ch < p.K;
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            lds_dma16(i < BM / 8 / WAVES ? rx : rw, in && off[i] != OUTSIDE ? off[i] + s * 128 : OUTSIDE, 0,
                      lds0 + (s & 1) * (ROWS * 128) + (i * WAVES + wave) * 1024);
    };
    f8_f4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f8_f4{0, 0, 0, 0};
    // scales: a thread's row of x, and the wave's rows of w
    const float* xs = p.xs + min(m0 + tid % BM, p.M - 1) * p.kb;
    const float* ws = p.ws + static_cast<int64_t>(min(n0 + wn * NT * 16, p.N - 1) / 128) * p.kb;
    float sx = xs[0], sw = ws[0];
    issue(0);
    const int twist = f8_twist(lane & 15);   // of every row the lane reads: they are 16 apart
    for (int s = 0; s < p.kb; ++s) {
        if (BM == 64 * WAVES || tid < BM) s_xs[s & 1][tid % BM] = sx;
        lds_wait_vm<0>();
        __syncthreads();
        const float wscale = sw;
        if (s + 1 < p.kb) {
            issue(s + 1);
            sw = ws[s + 1];
            sx = xs[s + 1];
        }
        const char* st = smem + (s & 1) * (ROWS * 128);
        auto frag = [&](int r) {
            const char* q = st + (r + (lane & 15)) * 128;
            return F8Operand<EXACT>(*reinterpret_cast<const f8_i4*>(q + ((grp ^ twist) << 4)),
                                    *reinterpret_cast<const f8_i4*>(q + (((grp + 4) ^ twist) << 4)));
        };
        float f[MT];
        F8Operand<EXACT> w[NT], x[2];
#pragma unroll
        for (int j = 0; j < NT; ++j) w[j] = frag(BM + (wn * NT + j) * 16);
        x[0] = frag(wm * MT * 16);
#pragma unroll
        for (int i = 0; i < MT; ++i) f[i] = s_xs[s & 1][(wm * MT + i) * 16 + (lane & 15)] * wscale;
        // A product's result is there some 12 cycles after the next one has begun: it is
        // scaled three products later.  The order is held, or each would be waited for.
        constexpr int LAG = 3;
        f8_f4 d[LAG + 1];
#pragma unroll
        for (int t = 0; t < MT * NT + LAG; ++t) {
            if (t < MT * NT) {
                const int i = t / NT, j = t % NT;
                if (j == 0 && i + 1 < MT) x[(i + 1) & 1] = frag((wm * MT + i + 1) * 16);
                d[t % (LAG + 1)] = f8_block(w[j], x[i & 1]);
            }
            if (t >= LAG) {
                const int u = t - LAG, i = u / NT, j = u % NT;
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(d[u % (LAG + 1)][e], f[i], acc[i][j][e]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int64_t m = m0 + (wm * MT + i) * 16 + (lane & 15);
        if (m >= p.M) continue;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int n = n0 + (wn * NT + j) * 16 + 4 * grp;
            if (n < p.N) f8_store<EXACT>(p, m, n, acc[i][j]);
        }
    }
}

// Few rows: a work-group's four waves take every fourth block of K of 16 rows of w.
template <int MT, bool EXACT>
__global__ __launch_bounds__(256) void f8_gemv_kernel(F8Gemm p) {
    __shared__ f8_f4 s_d[4][MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), grp = lane >> 4;
    const int n0 = blockIdx.x * 16;
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
    auto frag = [&](const uint8_t* row, int s) {
        const int k = s * 128 + 16 * grp;
        f8_i4 lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
        if (k < p.K) lo = *reinterpret_cast<const f8_i4*>(row + k);
        if (k + 64 < p.K) hi = *reinterpret_cast<const f8_i4*>(row + k + 64);
        return F8Operand<EXACT>(lo, hi);
    };
#pragma unroll 4
    for (int s = wave; s < p.kb; s += 4) {
        const F8Operand<EXACT> w = frag(wr, s);
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            const f8_f4 d = f8_block(w, frag(xr[i], s));
            const float f = xs[i][s] * ws[s];
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
        if (m < p.M && n < p.N) f8_store<EXACT>(p, m, n, d);
    }
}

template <bool EXACT>
void f8_launch(F8Gemm& p, hipStream_t st) {
    if (p.M <= 64) {
        const unsigned grid = (p.N + 15) / 16;
        if (p.M <= 16)
            f8_gemv_kernel<1, EXACT><<<grid, 256, 0, st>>>(p);
        else if (p.M <= 32)
            f8_gemv_kernel<2, EXACT><<<grid, 256, 0, st>>>(p);
        else
            f8_gemv_kernel<4, EXACT><<<grid, 256, 0, st>>>(p);
        return;
    }
    auto tiles = [&](int bm, int bn) {
        p.nm = static_cast<int>((p.M + bm - 1) / bm);
        p.nn = (p.N + bn - 1) / bn;
        return p.nm * p.nn;
    };
    if constexpr (EXACT) {
        if (tiles(128, 256) >= 200) {
            f8_gemm_kernel<2, 4, 4, 4, EXACT><<<p.nm * p.nn, 512, 0, st>>>(p);
            return;
        }
    } else if (tiles(256, 256) >= 200) {
        f8_gemm_kernel<2, 4, 8, 4, EXACT><<<p.nm * p.nn, 512, 0, st>>>(p);
        return;
    }
    {
        tiles(64, 128);
        f8_gemm_kernel<2, 2, 2, 4, EXACT><<<p.nm * p.nn, 256, 0, st>>>(p);
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
             static_cast<int>(outputs), static_cast<int>(width), static_cast<int>((width + 127) / 128), 0, 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (out_dtype == MOGT_F32)
        f8_launch<true>(p, st);
    else
        f8_launch<false>(p, st);
    return check_launch("mogt_linear_fp8");
}
