// Short causal depthwise convolution over channels-last rows, with its
// backward and its single-token form:
//   s_t = bias + sum_k w_k x_{t-K+1+k},  y_t = s_t or silu(s_t)
// and with ds = dy (silu'(s)):
//   dx_t = sum_k w_k ds_{t+K-1-k},  dw_k = sum_t ds_t x_{t-K+1+k},  dbias = sum_t ds_t.
//
// Bound: HBM (one read and one write of the rows; the backward reads x and dy
// and writes dx).  A lane owns VEC consecutive channels (16 bytes of a row
// where the rows allow it; 4 bf16 ones in the backward, whose windows and sums
// take the registers: 35 us against 45 with 8 at 4 x 4095 steps of 1280
// channels) and walks a stretch of steps with the last K - 1 rows in registers,
// so a row is read once per stretch plus K - 1 rows in front of it (and behind
// it in the backward), which the neighbouring wave has brought to the cache.
// The backward forms s again instead of keeping it.
// Measured, bf16, 4 taps: 32768 steps of 2048 channels 57 us (4.7 TB/s of the
// 5.2 that a large copy reaches here), 200 of 768 fp32 4.1; 4 x 4095 of 1280
// forward 23 us, backward 38 (3.3 TB/s; its vector instructions, 4 taps three
// times and the gate's slope, take 53 % of the cycles at 1.6 waves a SIMD, so
// neither memory nor the vector unit is full) and 3.8 for the sums; one token of
// 256 sequences of 2048 channels 5.3 us, of one 2.8.
#include <initializer_list>

#include "common.h"

namespace mogt {

int column_sums(const float* part, float* a, float* b, float* c, int64_t rows, int64_t K, int64_t D, int64_t N,
                hipStream_t st);

constexpr int CONV_U = 8;   // steps whose rows are loaded together

struct ConvArgs {
    const void* x;
    const float *w, *bias;
    const void *init, *lengths;
    int64_t xs, xb;
    int L, D, K, silu, len64;
    int steps, nchunk;
    void *y, *last;                       // forward outputs
    const void *dy, *dlast;               // backward inputs
    void *dx, *dinit;
    float* part;                          // [B nchunk][K + 1][D]: gradients of the taps, of the bias
};

__device__ __forceinline__ int conv_length(const ConvArgs& p, int b) {
    if (!p.lengths) return p.L;
    int64_t n = p.len64 ? static_cast<const int64_t*>(p.lengths)[b] : static_cast<const int32_t*>(p.lengths)[b];
    n = n < 0 ? 0 : n > p.L ? p.L : n;
    return __builtin_amdgcn_readfirstlane(static_cast<int>(n));
}

// Row t of the sequence with the K - 1 rows of the initial state before it.
template <typename T, int VEC>
__device__ __forceinline__ void conv_row(const ConvArgs& p, const T* px, int b, int t, int c, float (&v)[VEC]) {
    if (t >= 0) {
        load_vec<T, VEC>(px + t * p.xs + c, v);
    } else if (p.init && t >= 1 - p.K) {
        load_vec<T, VEC>(static_cast<const T*>(p.init) + (static_cast<int64_t>(b) * (p.K - 1) + p.K - 1 + t) * p.D + c,
                         v);
    } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = 0.0f;
    }
}

// KM: taps in registers; K == KM, or below it with the rest left out (never
// multiplied by zero: a row outside the window may hold an infinity).
template <typename T, int KM, int VEC>
__global__ __launch_bounds__(256) void conv_fwd_kernel(ConvArgs p) {
    const int lane = threadIdx.x & 63;
    const int chunk = blockIdx.y * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = (blockIdx.x * 64 + lane) * VEC;
    const int b = blockIdx.z;
    if (chunk >= p.nchunk || c >= p.D) return;
    const int K = KM == 8 ? p.K : KM;
    const int len = conv_length(p, b);
    const int t0 = chunk * p.steps, t1 = min(t0 + p.steps, p.L), te = min(t1, len);
    const T* px = static_cast<const T*>(p.x) + b * p.xb;
    T* py = static_cast<T*>(p.y) + static_cast<int64_t>(b) * p.L * p.D + c;

    float w[KM][VEC], bias[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        bias[e] = p.bias ? p.bias[c + e] : 0.0f;
#pragma unroll
        for (int k = 0; k < KM; ++k) w[k][e] = k < K ? p.w[static_cast<int64_t>(c + e) * K + k] : 0.0f;
    }
    if (chunk == 0 && p.last) {
        T* pl = static_cast<T*>(p.last) + static_cast<int64_t>(b) * (K - 1) * p.D + c;
        for (int j = 0; j < K - 1; ++j) {
            float v[VEC];
            conv_row<T, VEC>(p, px, b, len - (K - 1) + j, c, v);
            store_vec<T, VEC>(pl + static_cast<int64_t>(j) * p.D, v);
        }
    }
    // ext[i + k] is row t + i - (K - 1) + k
    float ext[KM - 1 + CONV_U][VEC];
#pragma unroll
    for (int k = 0; k < KM - 1; ++k)
        if (k < K - 1 && t0 < te) conv_row<T, VEC>(p, px, b, t0 - (K - 1) + k, c, ext[k]);
    for (int t = t0; t < te; t += CONV_U) {
        // the rows sit behind the K - 1 of the window, whatever K
        float row[CONV_U][VEC];
#pragma unroll
        for (int i = 0; i < CONV_U; ++i) load_vec<T, VEC>(px + min(t + i, te - 1) * p.xs + c, row[i]);
#pragma unroll
        for (int i = 0; i < CONV_U; ++i) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                if constexpr (KM == 8) {
#pragma unroll
                    for (int k = 0; k < KM - 1 + CONV_U; ++k)
                        if (k == K - 1 + i) ext[k][e] = row[i][e];
                } else {
                    ext[KM - 1 + i][e] = row[i][e];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < CONV_U; ++i) {
            if (t + i >= te) break;
            float s[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                s[e] = bias[e];
#pragma unroll
                for (int k = 0; k < KM; ++k)
                    if (k < K) s[e] = fmaf(w[k][e], ext[i + k][e], s[e]);
                if (p.silu) s[e] *= sigmoid_hw(s[e]);
            }
            store_vec<T, VEC>(py + static_cast<int64_t>(t + i) * p.D, s);
        }
#pragma unroll
        for (int k = 0; k < KM - 1; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) ext[k][e] = ext[CONV_U + k][e];
    }
    const float zero[VEC] = {};
    for (int t = max(t0, te); t < t1; ++t) store_vec<T, VEC>(py + static_cast<int64_t>(t) * p.D, zero);
}

// The gradient of s enters at step t, row t - (K - 1) then has all its terms and
// leaves.  The four waves of a work-group take neighbouring stretches and add
// their tap and bias sums, so one row of partial sums is written for all four.
constexpr int CONV_BWD_STEPS = 32;   // steps of a wave
constexpr int CONV_BWD_U = 4;        // rows loaded together, a block ahead

template <typename T, int KM, int VEC>
__global__ __launch_bounds__(256) void conv_bwd_kernel(ConvArgs p) {
    constexpr int U = CONV_BWD_U;
    __shared__ float s_sum[3][KM + 1][64 * VEC];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int chunk = blockIdx.y * 4 + wave;
    const int ci = (blockIdx.x * 64 + lane) * VEC;
    const bool valid = ci < p.D;
    const int c = valid ? ci : 0;
    const int b = blockIdx.z;
    const int K = KM == 8 ? p.K : KM;
    const int len = conv_length(p, b);
    const int t0 = chunk * CONV_BWD_STEPS, t1 = min(t0 + CONV_BWD_STEPS, p.L), te = min(t1, len);
    const T* px = static_cast<const T*>(p.x) + b * p.xb;
    const int64_t at = static_cast<int64_t>(b) * p.L * p.D + c;
    const T* pg = static_cast<const T*>(p.dy) + at;
    T* pdx = static_cast<T*>(p.dx) + at;

    // taps with the last at KM - 1 (a window's rows end at the same place) and,
    // for the way back, with the first at 0: the same array where K == KM
    float w[KM][VEC], first[KM][VEC], bias[VEC], dw[KM][VEC], db[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        bias[e] = p.bias ? p.bias[c + e] : 0.0f;
        db[e] = 0.0f;
#pragma unroll
        for (int k = 0; k < KM; ++k) {
            const int64_t q = static_cast<int64_t>(c + e) * K;
            w[k][e] = k >= KM - K ? p.w[q + k - (KM - K)] : 0.0f;
            first[k][e] = KM != 8 ? w[k][e] : k < K ? p.w[q + k] : 0.0f;
            dw[k][e] = 0.0f;
        }
    }
    // rows and gradients of s at steps t - (KM - 1) .. t + U - 1
    float xe[KM - 1 + U][VEC], ds[KM - 1 + U][VEC];
#pragma unroll
    for (int k = 0; k < KM - 1; ++k) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) xe[k][e] = ds[k][e] = 0.0f;
        if (k >= KM - K && chunk < p.nchunk) conv_row<T, VEC>(p, px, b, t0 - (KM - 1) + k, c, xe[k]);
    }
    const bool open = chunk == 0 && p.dinit;   // rows of the initial state leave too
    const int end = t0 < te || open ? te + K - 1 : t0;
    Pack<T, VEC> xr[U], gr[U];
    auto load = [&](int t) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int64_t r = min(t + i, len - 1);
            xr[i] = *reinterpret_cast<const Pack<T, VEC>*>(px + r * p.xs + c);
            gr[i] = *reinterpret_cast<const Pack<T, VEC>*>(pg + r * p.D);
        }
    };
    if (chunk < p.nchunk && t0 < end && len > 0) load(t0);
    for (int t = t0; t < end && chunk < p.nchunk; t += U) {
        float g[U][VEC];
#pragma unroll
        for (int i = 0; i < U; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const bool on = t + i < len;   // past the end: nothing was read
                xe[KM - 1 + i][e] = on ? IO<T>::ld(xr[i].v[e]) : 0.0f;
                g[i][e] = on ? IO<T>::ld(gr[i].v[e]) : 0.0f;
            }
        if (t + U < end && len > 0) load(t + U);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const bool on = t + i < len, own = t + i < te;
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                float d = g[i][e];
                if (p.silu) {
                    float s = bias[e];
#pragma unroll
                    for (int k = 0; k < KM; ++k)
                        if (k >= KM - K) s = fmaf(w[k][e], xe[i + k][e], s);
                    const float sg = sigmoid_hw(s);
                    d *= sg * fmaf(s, 1.0f - sg, 1.0f);
                }
                ds[KM - 1 + i][e] = on ? d : 0.0f;
            }
            if (own) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float d = ds[KM - 1 + i][e];
                    db[e] += d;
#pragma unroll
                    for (int k = 0; k < KM; ++k)
                        if (k >= KM - K) dw[k][e] = fmaf(d, xe[i + k][e], dw[k][e]);
                }
            }
            const int r = t + i - (K - 1);
            if (r >= te || (r < t0 && !open)) continue;
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                v[e] = 0.0f;
#pragma unroll
                for (int m = 0; m < KM; ++m)
                    if (m < K && t + i - m >= 0) v[e] = fmaf(first[m][e], ds[KM - 1 + i - m][e], v[e]);
            }
            if (p.dlast && r >= len - (K - 1)) {
                float q[VEC];
                load_vec<T, VEC>(static_cast<const T*>(p.dlast) +
                                     (static_cast<int64_t>(b) * (K - 1) + r - len + K - 1) * p.D + c, q);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] += q[e];
            }
            if (!valid) continue;
            if (r >= 0) {
                if (p.dx) store_vec<T, VEC>(pdx + static_cast<int64_t>(r) * p.D, v);
            } else {
                store_vec<T, VEC>(static_cast<T*>(p.dinit) + (static_cast<int64_t>(b) * (K - 1) + K - 1 + r) * p.D + c,
                                  v);
            }
        }
#pragma unroll
        for (int k = 0; k < KM - 1; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                xe[k][e] = xe[U + k][e];
                ds[k][e] = ds[U + k][e];
            }
    }
    if (p.dx && valid) {
        const float zero[VEC] = {};
        for (int t = max(t0, te); t < t1; ++t) store_vec<T, VEC>(pdx + static_cast<int64_t>(t) * p.D, zero);
    }
    if (wave > 0) {
#pragma unroll
        for (int k = 0; k < KM; ++k) store_vec<float, VEC>(&s_sum[wave - 1][k][lane * VEC], dw[k]);
        store_vec<float, VEC>(&s_sum[wave - 1][KM][lane * VEC], db);
    }
    __syncthreads();
    if (wave > 0 || !valid) return;
    const int64_t row = static_cast<int64_t>(b) * gridDim.y + blockIdx.y;
    float* part = p.part + row * (K + 1) * p.D + c;
#pragma unroll
    for (int k = 0; k <= KM; ++k) {
        if (k < KM - K) continue;
        float v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            v[e] = k < KM ? dw[k < KM ? k : 0][e] : db[e];
#pragma unroll
            for (int m = 0; m < 3; ++m) v[e] += s_sum[m][k][lane * VEC + e];
        }
        store_vec<float, VEC>(part + static_cast<int64_t>(k - (KM - K)) * p.D, v);
    }
}

// One token: a thread per channel; the state moves up by one row.
template <typename T>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvArgs p, T* state) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= p.D) return;
    const int b = blockIdx.y;
    T* q = state + static_cast<int64_t>(b) * (p.K - 1) * p.D + c;
    const T xr = (static_cast<const T*>(p.x) + b * p.xb)[c];
    float s = p.bias ? p.bias[c] : 0.0f;
    for (int k = 0; k < p.K - 1; ++k) {
        s = fmaf(p.w[static_cast<int64_t>(c) * p.K + k], IO<T>::ld(q[static_cast<int64_t>(k) * p.D]), s);
        q[static_cast<int64_t>(k) * p.D] = k + 2 < p.K ? q[static_cast<int64_t>(k + 1) * p.D] : xr;
    }
    s = fmaf(p.w[static_cast<int64_t>(c) * p.K + p.K - 1], IO<T>::ld(xr), s);
    if (p.silu) s *= sigmoid_hw(s);
    (static_cast<T*>(p.y) + static_cast<int64_t>(b) * p.D)[c] = IO<T>::st(s);
}

namespace {

int conv_steps(int64_t B, int64_t L, int64_t D, int vec) {
    // steps a wave walks: at most 32 (rows in front are read again), fewer
    // where the GPU would otherwise hold under 8 waves per CU.  Of 8, 16 and 32
    // steps, 200 of 768 channels fp32 take 4.2, 5.5 and 8.0 us, in bf16 2048 of 2048
    // 9.2, 12.8 and 16.4, 4 x 4095 of 1280 26.5, 23.7 and 25.3, 32768 of 2048 64.4,
    // 65 and 59.9 (one card, contiguous rows that rotate through 1.5 GB).
    const int64_t waves = B * ((D + 64 * vec - 1) / (64 * vec));
    int64_t s = 32;
    while (s > 8 && waves * ((L + s - 1) / s) < 2048) s /= 2;
    return static_cast<int>(s);
}

int conv_args(const mogt_short_conv_problem* q, ConvArgs& a) {
    if (!q) return set_error(MOGT_E_INVALID, "null problem");
    if (q->batch < 0 || q->length < 0 || q->channels < 0)
        return set_error(MOGT_E_INVALID, "bad sizes: batch %lld, length %lld, channels %lld", (long long)q->batch,
                         (long long)q->length, (long long)q->channels);
    if (q->taps < 1 || q->taps > 8) return set_error(MOGT_E_INVALID, "%lld taps: 1 to 8 expected", (long long)q->taps);
    if (q->io_dtype != MOGT_F32 && q->io_dtype != MOGT_BF16)
        return set_error(MOGT_E_INVALID, "dtype code %d not supported", q->io_dtype);
    if (q->lengths && q->lengths_bytes != 4 && q->lengths_bytes != 8)
        return set_error(MOGT_E_INVALID, "lengths of 4 or 8 bytes expected, got %d", q->lengths_bytes);
    if (q->length >= (1ll << 30) || q->channels >= (1ll << 24) || q->batch > 65535 ||
        (q->length + 31) / 32 > 4ll * 65535)
        return set_error(MOGT_E_INVALID, "batch up to 65535, length up to 8388480 and channels below 2^24 expected");
    if (q->batch > 0 && q->channels > 0 && (!q->weight || (q->length > 0 && !q->x)))
        return set_error(MOGT_E_INVALID, "null input pointer");
    a.x = q->x;
    a.w = q->weight;
    a.bias = q->bias;
    a.init = q->initial_state;
    a.lengths = q->lengths;
    a.xs = q->x_row;
    a.xb = q->x_batch;
    a.L = static_cast<int>(q->length);
    a.D = static_cast<int>(q->channels);
    a.K = static_cast<int>(q->taps);
    a.silu = q->silu;
    a.len64 = q->lengths_bytes == 8;
    return MOGT_OK;
}

// 16-byte vectors: every row starts on one and holds whole ones
bool conv_vectors(const mogt_short_conv_problem* q, std::initializer_list<const void*> others) {
    const int64_t n = q->io_dtype == MOGT_F32 ? 4 : 8;
    uintptr_t at = reinterpret_cast<uintptr_t>(q->x) | reinterpret_cast<uintptr_t>(q->initial_state);
    for (const void* o : others) at |= reinterpret_cast<uintptr_t>(o);
    return (at & 15) == 0 && q->channels % n == 0 && q->x_row % n == 0 && q->x_batch % n == 0;
}

template <typename T, int VEC>
int conv_fwd(ConvArgs& a, int batch, hipStream_t st) {
    a.steps = conv_steps(batch, a.L, a.D, VEC);
    a.nchunk = a.L > 0 ? (a.L + a.steps - 1) / a.steps : 1;
    const dim3 grid((a.D + 64 * VEC - 1) / (64 * VEC), (a.nchunk + 3) / 4, batch);
    switch (a.K) {
        case 2: conv_fwd_kernel<T, 2, VEC><<<grid, 256, 0, st>>>(a); break;
        case 3: conv_fwd_kernel<T, 3, VEC><<<grid, 256, 0, st>>>(a); break;
        case 4: conv_fwd_kernel<T, 4, VEC><<<grid, 256, 0, st>>>(a); break;
        default: conv_fwd_kernel<T, 8, VEC><<<grid, 256, 0, st>>>(a); break;
    }
    return check_launch("mogt_short_conv_fwd");
}

template <typename T, int VEC>
int conv_bwd(ConvArgs& a, int batch, hipStream_t st) {
    const dim3 grid((a.D + 64 * VEC - 1) / (64 * VEC), (a.nchunk + 3) / 4, batch);
    switch (a.K) {
        case 2: conv_bwd_kernel<T, 2, VEC><<<grid, 256, 0, st>>>(a); break;
        case 3: conv_bwd_kernel<T, 3, VEC><<<grid, 256, 0, st>>>(a); break;
        case 4: conv_bwd_kernel<T, 4, VEC><<<grid, 256, 0, st>>>(a); break;
        default: conv_bwd_kernel<T, 8, VEC><<<grid, 256, 0, st>>>(a); break;
    }
    return check_launch("mogt_short_conv_bwd");
}

// Work-groups along the sequence of the backward.
int64_t conv_bwd_groups(int64_t L) { return L > 0 ? (L + 4 * CONV_BWD_STEPS - 1) / (4 * CONV_BWD_STEPS) : 1; }

}  // namespace
}  // namespace mogt

using namespace mogt;

extern "C" int mogt_short_conv_fwd(const mogt_short_conv_problem* q, void* y, void* final_state, void* stream) {
    clear_error();
    ConvArgs a{};
    if (const int rc = conv_args(q, a)) return rc;
    if (q->batch == 0 || q->channels == 0) return MOGT_OK;
    if (q->taps == 1) final_state = nullptr;   // no rows
    if (q->length == 0 && !final_state) return MOGT_OK;
    if (q->length > 0 && !y) return set_error(MOGT_E_INVALID, "null output pointer");
    a.y = y;
    a.last = final_state;
    const bool vec = conv_vectors(q, {y, final_state});
    const int batch = static_cast<int>(q->batch);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q->io_dtype == MOGT_F32) return vec ? conv_fwd<float, 4>(a, batch, st) : conv_fwd<float, 1>(a, batch, st);
    return vec ? conv_fwd<bf16_t, 8>(a, batch, st) : conv_fwd<bf16_t, 1>(a, batch, st);
}

extern "C" size_t mogt_short_conv_bwd_workspace_bytes(int64_t batch, int64_t length, int64_t channels, int64_t taps) {
    if (batch <= 0 || channels <= 0 || taps <= 0 || length < 0) return 0;
    return static_cast<size_t>(batch * conv_bwd_groups(length) * (taps + 1) * channels) * sizeof(float);
}

extern "C" int mogt_short_conv_bwd(const mogt_short_conv_problem* q, const void* dy, const void* dfinal_state, void* dx,
                                   float* dweight, float* dbias, void* dinitial_state, void* workspace,
                                   size_t workspace_bytes, void* stream) {
    clear_error();
    ConvArgs a{};
    if (const int rc = conv_args(q, a)) return rc;
    if (q->batch == 0 || q->channels == 0) return MOGT_OK;
    if (q->length > 0 && !dy) return set_error(MOGT_E_INVALID, "null gradient pointer");
    const size_t need = mogt_short_conv_bwd_workspace_bytes(q->batch, q->length, q->channels, q->taps);
    if (!workspace || workspace_bytes < need)
        return set_error(MOGT_E_WORKSPACE, "workspace of %zu bytes expected, got %zu", need,
                         workspace ? workspace_bytes : 0);
    if (q->taps == 1) dfinal_state = dinitial_state = nullptr;
    a.dy = dy;
    a.dlast = dfinal_state;
    a.dx = dx;
    a.dinit = dinitial_state;
    a.nchunk = a.L > 0 ? (a.L + CONV_BWD_STEPS - 1) / CONV_BWD_STEPS : 1;
    const int64_t rows = q->batch * conv_bwd_groups(q->length);
    a.part = static_cast<float*>(workspace);
    const bool vec = conv_vectors(q, {dy, dfinal_state, dx, dinitial_state});
    const int batch = static_cast<int>(q->batch);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const int rc = q->io_dtype == MOGT_F32 ? (vec ? conv_bwd<float, 4>(a, batch, st) : conv_bwd<float, 1>(a, batch, st))
                                           : (vec ? conv_bwd<bf16_t, 4>(a, batch, st) : conv_bwd<bf16_t, 1>(a, batch, st));
    if (rc) return rc;
    if (!dweight && !dbias) return MOGT_OK;
    return column_sums(a.part, dweight, dbias, nullptr, rows, q->taps + 1, q->channels, q->taps, st);
}

extern "C" int mogt_short_conv_step(const mogt_short_conv_problem* q, void* state, void* y, void* stream) {
    clear_error();
    ConvArgs a{};
    if (const int rc = conv_args(q, a)) return rc;
    if (q->length != 1) return set_error(MOGT_E_INVALID, "a step takes one token, length is %lld", (long long)q->length);
    if (q->batch == 0 || q->channels == 0) return MOGT_OK;
    if (!y || (!state && q->taps > 1)) return set_error(MOGT_E_INVALID, "null state or output pointer");
    a.y = y;
    const dim3 grid((a.D + 255) / 256, static_cast<unsigned>(q->batch));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q->io_dtype == MOGT_F32)
        conv_step_kernel<float><<<grid, 256, 0, st>>>(a, static_cast<float*>(state));
    else
        conv_step_kernel<bf16_t><<<grid, 256, 0, st>>>(a, static_cast<bf16_t*>(state));
    return check_launch("mogt_short_conv_step");
}
