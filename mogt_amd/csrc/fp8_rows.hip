// Rows and weights in e4m3 (OCP, 3 fraction bits, largest value 448) with a scale
// for each block of 128 values of a row, or of 128 rows by 128 values:
//   scale = max(largest |x| of the block / 448, 2^-126),   q = e4m3(x / scale)
// rounded to nearest even, so x is q * scale within half a step of the block's
// largest value, and a block of zeros is zeros.  A NaN stays one in its place; an
// infinity makes its block's scale infinite.  (The norm rounds its quotients from the
// scale in 64 bits; the quantisers divide by the scale that they store.)
//   add_rmsnorm_fp8  x' = x + s * z (bf16 z: the product rounded to bf16, as add_rmsnorm
//                    does), n = rmsnorm(x') * w, the rows n in 8 bits
//   quantize_rows    the rows of a matrix
//   quantize_blocks  128 x 128 blocks (weights, laid out once)
// Rows and weights in 8 bits: 32768 rows of 2048 take 71 us from bf16 (203 MB, 40 at a
// copy's rate) and 82 from fp32, a weight of 6144 x 2048, laid out once, 21 and 24.
// Four consecutive values a lane: half a wave is a block and its maximum five lane
// exchanges.  The norm takes one wave a row, which it holds in registers, in 64 bits
// from the update on, so that values at a border of the 8 bits fall where the
// definition's do: of 32768 rows of 2048 none falls elsewhere, in 32 bits about 50
// values do.  The root mean square is common to a block and cancels in
// q = 448 x' w / largest |x' w|.  Bound by HBM: those rows with bf16 z take 147 us,
// 5.0 TB/s (in 32 bits 140).
#include "common.h"
#include "wide_grid.h"

namespace mogt {
namespace {

constexpr int F8_BLOCK = 128;
constexpr float F8_MAX = 448.0f;
constexpr int F8_WAVES = 4;   // rows per work-group

__device__ __forceinline__ float f8_scale(float amax) { return fmaxf(amax / F8_MAX, 0x1p-126f); }

// four values as e4m3, nearest even; magnitudes are at most 448 (1 + 2^-23), which rounds to 448
__device__ __forceinline__ uint32_t f8_pack(const float (&v)[4]) {
    const int w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], w, true));
}
__device__ __forceinline__ uint32_t f8_pack(const float (&v)[4], float scale) {
    const float x[4] = {v[0] / scale, v[1] / scale, v[2] / scale, v[3] / scale};
    return f8_pack(x);
}

// the largest of the 32 lanes of a half wave
__device__ __forceinline__ float f8_block_max(float m) {
#pragma unroll
    for (int i = 16; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor(m, i));
    return m;
}

__device__ __forceinline__ float f8_max4(const float (&v)[4]) {
    return fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
}

template <int CTRL>
__device__ __forceinline__ double f8_dpp_max(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_mov_dpp(static_cast<int>(u), CTRL, 0xf, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_mov_dpp(static_cast<int>(u >> 32), CTRL, 0xf, 0xf, true);
    return fmax(x, __builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32 | lo));
}

__device__ __forceinline__ double f8_block_max(double m) {
    m = f8_dpp_max<0xb1>(m);    // lanes 1 apart
    m = f8_dpp_max<0x4e>(m);    // 2 apart
    m = f8_dpp_max<0x141>(m);   // mirrored in 8
    m = f8_dpp_max<0x140>(m);   // mirrored in 16
    const uint64_t u = __builtin_bit_cast(uint64_t, m);
    const uint32_t l = static_cast<uint32_t>(u), h = static_cast<uint32_t>(u >> 32);
    // the even rows of 16 lanes twice, and the odd ones
    const auto lo = __builtin_amdgcn_permlane16_swap(l, l, false, false), hi = __builtin_amdgcn_permlane16_swap(h, h, false, false);
    return fmax(__builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]),
                __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]));
}

// 1 / x for x > 0 to the last bits, 0 for infinity
__device__ __forceinline__ double f8_inverse(double x) {
    double r = __builtin_amdgcn_rcp(x);
    const double e = fma(-x, r, 1.0);
    r = fma(r, fma(e, e, e), r);
    return x > 0x1p1000 ? 0.0 : r;
}

// x with the bits below its first 20 in the last of them: exact in fp32, and on the
// side of a border of the 8 bits that x is on
__device__ __forceinline__ float f8_odd(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t hi = static_cast<uint32_t>(u >> 32) | min(static_cast<uint32_t>(u), 1u);
    return static_cast<float>(__builtin_bit_cast(double, static_cast<uint64_t>(hi) << 32));
}

// x, which the compiler takes for a new value: weights are loaded where they are
// used, not all held (90 registers against 112, 147 us against 157)
__device__ __forceinline__ int f8_again(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

struct F8Norm {
    const float* x;
    const void* z;
    const float* w;
    float* x_out;
    uint32_t* q;       // [rows, D] bytes
    float* scale;      // [rows, blocks]
    int64_t rows;
    int D, blocks;
    float zs, eps;
};

// VPL: vectors of four values a lane (D <= 256 VPL)
template <typename TZ, int VPL>
__global__ __launch_bounds__(64 * F8_WAVES) void f8_norm_kernel(F8Norm p) {
    const int lane = threadIdx.x & 63;
    const int64_t row = wide_block() * F8_WAVES + (threadIdx.x >> 6);
    if (row >= p.rows) return;
    const float* xr = p.x + row * p.D;
    const TZ* zr = static_cast<const TZ*>(p.z) + row * p.D;
    double v[VPL][4], ss = 0.0;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        const int c = (k * 64 + lane) * 4;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[k][e] = 0.0;
        if (c < p.D) {
            float x[4], zz[4];
            load_vec<float, 4>(xr + c, x);
            load_vec<TZ, 4>(zr + c, zz);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(TZ) == 4)
                    v[k][e] = fma(static_cast<double>(p.zs), static_cast<double>(zz[e]), static_cast<double>(x[e]));
                else
                    v[k][e] = static_cast<double>(x[e]) + static_cast<double>(IO<TZ>::ld(IO<TZ>::st(p.zs * zz[e])));
                ss = fma(v[k][e], v[k][e], ss);
                x[e] += IO<TZ>::ld(IO<TZ>::st(p.zs * zz[e]));
            }
            store_vec<float, 4>(p.x_out + row * p.D + c, x);
        }
    }
    for (int m = 32; m > 0; m >>= 1) ss += __shfl_xor(ss, m);
    const double inv = 1.0 / sqrt(ss / p.D + static_cast<double>(p.eps));
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        const int c = (k * 64 + f8_again(lane)) * 4;
        double u[4] = {0.0, 0.0, 0.0, 0.0};
        if (c < p.D) {
            float w[4];
            load_vec<float, 4>(p.w + c, w);
#pragma unroll
            for (int e = 0; e < 4; ++e) u[e] = v[k][e] * static_cast<double>(w[e]);
        }
        const double m = f8_block_max(fmax(fmax(fabs(u[0]), fabs(u[1])), fmax(fabs(u[2]), fabs(u[3]))));
        const double s = m * inv * (1.0 / F8_MAX);
        const bool least = !(s >= 0x1p-126);   // or NaN, which the values then are
        const double f = least ? inv * 0x1p126 : F8_MAX * f8_inverse(m);
        if (c < p.D) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = f8_odd(u[e] * f);
            p.q[(row * p.D + c) >> 2] = f8_pack(y);
            if ((lane & 31) == 0) p.scale[row * p.blocks + c / F8_BLOCK] = least ? 0x1p-126f : static_cast<float>(s);
        }
    }
}

// Half a wave per block of a row.
template <typename T>
__global__ __launch_bounds__(256) void f8_rows_kernel(const T* x, int64_t ldx, uint32_t* q, float* scale, int64_t total,
                                                      int D, int blocks) {
    const int64_t id = wide_block() * 8 + (threadIdx.x >> 5);
    const int64_t row = id / blocks;
    const int block = static_cast<int>(id - row * blocks), c = block * F8_BLOCK + (threadIdx.x & 31) * 4;
    const bool in = id < total && c < D;
    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (in) load_vec<T, 4>(x + row * ldx + c, v);
    const float s = f8_scale(f8_block_max(f8_max4(v)));
    if (in) {
        q[(row * D + c) >> 2] = f8_pack(v, s);
        if ((threadIdx.x & 31) == 0) scale[id] = s;
    }
}

// A work-group per 128 x 128 block: its maximum, then its values (read again from
// the caches).
template <typename T>
__global__ __launch_bounds__(256) void f8_blocks_kernel(const T* x, int64_t ldx, uint32_t* q, float* scale, int64_t rows,
                                                        int D) {
    __shared__ float s_max[4];
    const int64_t r0 = static_cast<int64_t>(blockIdx.y) * F8_BLOCK;
    const int c = blockIdx.x * F8_BLOCK + (threadIdx.x & 31) * 4, nr = static_cast<int>(min(rows - r0, static_cast<int64_t>(F8_BLOCK)));
    float m = 0.0f;
    for (int r = threadIdx.x >> 5; r < nr; r += 8)
        if (c < D) {
            float v[4];
            load_vec<T, 4>(x + (r0 + r) * ldx + c, v);
            m = fmaxf(m, f8_max4(v));
        }
    for (int i = 32; i > 0; i >>= 1) m = fmaxf(m, __shfl_xor(m, i));
    if ((threadIdx.x & 63) == 0) s_max[threadIdx.x >> 6] = m;
    __syncthreads();
    const float s = f8_scale(fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3])));
    for (int r = threadIdx.x >> 5; r < nr; r += 8)
        if (c < D) {
            float v[4];
            load_vec<T, 4>(x + (r0 + r) * ldx + c, v);
            q[((r0 + r) * D + c) >> 2] = f8_pack(v, s);
        }
    if (threadIdx.x == 0) scale[blockIdx.y * static_cast<int64_t>(gridDim.x) + blockIdx.x] = s;
}

template <typename TZ>
int f8_norm_launch(const F8Norm& p, hipStream_t st) {
    const int64_t blocks = (p.rows + F8_WAVES - 1) / F8_WAVES;
    if (blocks > WIDE_GRID_MAX) return set_error(MOGT_E_INVALID, "%lld rows are too many", (long long)p.rows);
    const dim3 grid = wide_grid(blocks);
    if (p.D <= 256)
        f8_norm_kernel<TZ, 1><<<grid, 64 * F8_WAVES, 0, st>>>(p);
    else if (p.D <= 1024)
        f8_norm_kernel<TZ, 4><<<grid, 64 * F8_WAVES, 0, st>>>(p);
    else if (p.D <= 2048)
        f8_norm_kernel<TZ, 8><<<grid, 64 * F8_WAVES, 0, st>>>(p);
    else
        f8_norm_kernel<TZ, 16><<<grid, 64 * F8_WAVES, 0, st>>>(p);
    return check_launch("mogt_add_rmsnorm_fp8_fwd");
}

template <typename T>
int f8_quantize_launch(const void* x, int64_t ld, void* q, float* scale, int64_t rows, int64_t dim, int block_rows,
                       hipStream_t st) {
    const int blocks = static_cast<int>((dim + F8_BLOCK - 1) / F8_BLOCK), D = static_cast<int>(dim);
    const T* xt = static_cast<const T*>(x);
    uint32_t* qt = static_cast<uint32_t*>(q);
    if (block_rows == 1) {
        const int64_t groups = (rows * blocks + 7) / 8;
        if (rows > (1ll << 40) || groups > WIDE_GRID_MAX)
            return set_error(MOGT_E_INVALID, "%lld rows of %lld are too many", (long long)rows, (long long)dim);
        f8_rows_kernel<T><<<wide_grid(groups), 256, 0, st>>>(xt, ld, qt, scale, rows * blocks, D, blocks);
    } else {
        const int64_t by = (rows + F8_BLOCK - 1) / F8_BLOCK;
        if (by > 65535) return set_error(MOGT_E_INVALID, "%lld rows: at most %d", (long long)rows, 65535 * F8_BLOCK);
        f8_blocks_kernel<T><<<dim3(blocks, static_cast<unsigned>(by)), 256, 0, st>>>(xt, ld, qt, scale, rows, D);
    }
    return check_launch("mogt_quantize_fp8");
}

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

}  // namespace
}  // namespace mogt

using namespace mogt;

extern "C" int mogt_add_rmsnorm_fp8_fwd(const float* x, const void* z, float scale, const float* weight, float* x_out,
                                        void* q, float* q_scale, int64_t rows, int64_t dim, float eps, int z_dtype,
                                        void* stream) {
    clear_error();
    if (rows < 0 || dim < 4 || dim > 4096 || dim % 4 != 0)
        return set_error(MOGT_E_INVALID, "rows %lld of %lld: a length that is a multiple of 4 up to 4096 expected",
                         (long long)rows, (long long)dim);
    if (z_dtype != MOGT_F32 && z_dtype != MOGT_BF16) return set_error(MOGT_E_INVALID, "z dtype %d not supported", z_dtype);
    if (rows == 0) return MOGT_OK;
    if (!x || !z || !weight || !x_out || !q || !q_scale) return set_error(MOGT_E_INVALID, "null pointer");
    if (!aligned(x, 16) || !aligned(x_out, 16) || !aligned(weight, 16) || !aligned(z, z_dtype == MOGT_BF16 ? 8 : 16) || !aligned(q, 4))
        return set_error(MOGT_E_INVALID, "rows of four values must be aligned");
    F8Norm p{x, z, weight, x_out, static_cast<uint32_t*>(q), q_scale, rows, static_cast<int>(dim),
             static_cast<int>((dim + F8_BLOCK - 1) / F8_BLOCK), scale, eps};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (z_dtype == MOGT_BF16) return f8_norm_launch<bf16_t>(p, st);
    return f8_norm_launch<float>(p, st);
}

extern "C" int mogt_quantize_fp8(const void* x, int64_t ld, void* q, float* q_scale, int64_t rows, int64_t dim, int dtype,
                                 int block_rows, void* stream) {
    clear_error();
    if (rows < 0 || dim < 4 || dim % 4 != 0 || dim > (1 << 30) || ld < dim)
        return set_error(MOGT_E_INVALID, "rows %lld of %lld (stride %lld): a length that is a multiple of 4 expected",
                         (long long)rows, (long long)dim, (long long)ld);
    if (dtype != MOGT_F32 && dtype != MOGT_BF16) return set_error(MOGT_E_INVALID, "dtype %d not supported", dtype);
    if (block_rows != 1 && block_rows != F8_BLOCK)
        return set_error(MOGT_E_INVALID, "blocks of %d rows: 1 or %d expected", block_rows, F8_BLOCK);
    if (rows == 0) return MOGT_OK;
    const size_t each = dtype == MOGT_BF16 ? 8 : 16;
    if (!x || !q || !q_scale) return set_error(MOGT_E_INVALID, "null pointer");
    if (!aligned(x, each) || ld % 4 != 0 || !aligned(q, 4)) return set_error(MOGT_E_INVALID, "rows of four values must be aligned");
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (dtype == MOGT_BF16) return f8_quantize_launch<bf16_t>(x, ld, q, q_scale, rows, dim, block_rows, st);
    return f8_quantize_launch<float>(x, ld, q, q_scale, rows, dim, block_rows, st);
}
