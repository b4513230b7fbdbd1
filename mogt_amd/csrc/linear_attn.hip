// Linear attention with a decay for each head: the states between segments, the
// gradient of the decays, shared heads' sums, the single-token form and the entry
// points (linear_attn.h has the mathematics, linear_attn_kernel.h the passes).
#include <initializer_list>

#include "linear_attn.h"
#include "wide_grid.h"

namespace mogt {

template <typename TI>
void la_launch_passes(const LaArgs& a, int count, bool out, hipStream_t st);
extern template void la_launch_passes<bf16_t>(const LaArgs&, int, bool, hipStream_t);
extern template void la_launch_passes<float>(const LaArgs&, int, bool, hipStream_t);

namespace {

// The states entering the segments, in place: slot 0 is the initial state, slot
// j + 1 = exp(c_j) slot j + what segment j wrote from zero.  A thread owns one
// element and reads 16 segments at once; `init` is [dk, dv], the segments' [dv, dk].
// 32 segments of 16 heads of 128 x 128, 67 MB: 13.9 us (4.8 TB/s; 32 at once, with
// half the waves, 16.2).
// A decay is its root applied twice, each finite: a state of a segment that grows
// is in range wherever the definition's is, and one of zeros stays zero.
__global__ __launch_bounds__(256) void la_carry_kernel(float* states, const float* ctot, const float* init, int nseg,
                                                       int dk, int dv) {
    constexpr int U = 16;
    const int e = blockIdx.x * 256 + threadIdx.x;
    const int state = dk * dv;
    const int64_t seq = blockIdx.y + static_cast<int64_t>(blockIdx.z) * gridDim.y;
    if (e >= state) return;
    float* q = states + seq * (nseg + 1) * state + e;
    const float* c = ctot + seq * nseg;
    float h = init ? init[seq * state + e % dk * dv + e / dk] : 0.0f;
    q[0] = h;
    for (int j = 0; j < nseg - 1; j += U) {
        float w[U], log2[U];   // all read before the first store, which the reads would wait for
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (j + i < nseg - 1) {
                w[i] = q[static_cast<int64_t>(j + i + 1) * state];
                log2[i] = c[j + i];
            }
#pragma unroll
        for (int i = 0; i < U; ++i)
            if (j + i < nseg - 1) {
                const float root = __builtin_amdgcn_exp2f(fminf(0.5f * log2[i], 127.0f));
                h = fmaf(root, root * h, w[i]);
                q[static_cast<int64_t>(j + i + 1) * state] = h;
            }
    }
}

struct LaDecay {
    const float *states, *rstates;   // [B, H, nseg + 1, state], in time order and in reverse
    const float *dot_q, *dot_k;      // [B, H, L]
    float* dg;                       // [B, L, H], or null
    double* part;                    // [H, B, nseg] sums of the segments, or null
    float* dinit;                    // [B, H, state], or null
    int dk;
    int have_last;                   // a gradient of the final state came in
};

// dg_s = sum_{t >= s} (q_t . dq_t - k_t . dk_t) within the segment, plus the
// product of the state after the segment and its gradient, which stands for
// every later step.  Bound by the states' bytes (2 x 8192 steps of 16 heads of 128:
// 67 MB, 19 us; of 12 heads of 64: 7.2 us).  Starting afresh at each segment keeps the differences of
// nearly equal sums short; they are added in 64 bits.
__global__ __launch_bounds__(256) void la_decay_kernel(LaArgs a, LaDecay d) {
    __shared__ double s_w[4];
    const int j = blockIdx.x, h = blockIdx.y, b = blockIdx.z, n = la_length(a, b);
    const int64_t seq = static_cast<int64_t>(b) * a.H + h;
    const int t0 = j * a.seg, t1 = min(t0 + a.seg, n), lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float* gb = a.g + b * a.g_batch + h * a.g_head;
    const float* R = d.rstates + (seq * (a.nseg + 1) + a.nseg - 1 - j) * a.state;   // gradient entering from later
    auto sum = [&](double x) {   // over the work-group
        for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
        __syncthreads();
        if (lane == 0) s_w[wave] = x;
        __syncthreads();
        return (s_w[0] + s_w[1]) + (s_w[2] + s_w[3]);
    };
    if (j == 0 && d.dinit) {   // its gradient, before the first step's decay (an empty sequence has none)
        const float* X = d.rstates + (seq * (a.nseg + 1) + a.nseg) * a.state;
        const float e = n > 0 ? __expf(gb[0]) : 1.0f;
        const int dv = a.state / d.dk;
        for (int i = threadIdx.x; i < a.state; i += 256)
            d.dinit[seq * a.state + i] = e == 0.0f ? 0.0f : e * X[i % dv * d.dk + i / dv];
    }
    if (!d.dg && !d.part) return;
    double carry = 0.0, total = 0.0;
    if (t0 < n && (t1 < n || d.have_last)) {
        const float* S = d.states + (seq * (a.nseg + 1) + j + 1) * a.state;
        double x = 0.0;
#pragma unroll 8
        for (int i = threadIdx.x; i < a.state; i += 256) x = fma(static_cast<double>(S[i]), static_cast<double>(R[i]), x);
        carry = sum(x);
        if (t1 < n) {
            const float g = gb[static_cast<int64_t>(t1) * a.g_row];
            carry = g <= LA_G_ZERO ? 0.0 : carry * exp(static_cast<double>(g));
        }
    }
    // from the segment's end, 256 steps at a time
    for (int hi = t1; hi > t0; hi -= 256) {
        const int t = hi - 1 - static_cast<int>(threadIdx.x);
        double x = 0.0;
        if (t >= t0) {
            const int64_t at = seq * a.L + t;
            x = static_cast<double>(d.dot_q[at]) - static_cast<double>(d.dot_k[at]);
        }
        for (int m = 1; m < 64; m <<= 1) {   // inclusive sums over the lanes
            const double y = __shfl_up(x, m);
            if (lane >= m) x += y;
        }
        __syncthreads();
        if (lane == 63) s_w[wave] = x;
        __syncthreads();
        for (int w = 0; w < wave; ++w) x += s_w[w];
        x += carry;
        carry += (s_w[0] + s_w[1]) + (s_w[2] + s_w[3]);
        if (t >= t0) {
            const double v = gb[static_cast<int64_t>(t) * a.g_row] <= LA_G_ZERO ? 0.0 : x;
            total += v;
            if (d.dg) d.dg[(static_cast<int64_t>(b) * a.L + t) * a.H + h] = static_cast<float>(v);
        }
    }
    if (d.dg)
        for (int t = max(t0, n) + static_cast<int>(threadIdx.x); t < min(t0 + a.seg, a.L); t += 256)
            d.dg[(static_cast<int64_t>(b) * a.L + t) * a.H + h] = 0.0f;
    if (d.part) {
        total = sum(total);
        if (threadIdx.x == 0) d.part[(static_cast<int64_t>(h) * a.B + b) * a.nseg + j] = total;
    }
}

// one decay a head: the sum of its segments' parts
__global__ __launch_bounds__(64) void la_decay_sum_kernel(const double* part, int64_t count, float* dg) {
    double x = 0.0;
    for (int64_t i = threadIdx.x; i < count; i += 64) x += part[blockIdx.x * count + i];
    for (int m = 32; m > 0; m >>= 1) x += __shfl_xor(x, m);
    if (threadIdx.x == 0) dg[blockIdx.x] = static_cast<float>(x);
}

// gradients of rows that `share` heads read: [rows, groups, share, d] fp32 to [rows, groups, d]
template <typename TI>
__global__ __launch_bounds__(256) void la_group_kernel(const float* dq, const float* dk, TI* to_q, TI* to_k, int64_t total,
                                                       int d, int share) {
    const int64_t i = wide_block() * 256 + threadIdx.x;
    TI* to = blockIdx.z ? to_k : to_q;
    if (i >= total || !to) return;
    const int64_t row = i / d;
    const float* p = (blockIdx.z ? dk : dq) + row * share * d + (i - row * d);
    float x = 0.0f;
    for (int j = 0; j < share; ++j) x += p[static_cast<int64_t>(j) * d];
    to[i] = IO<TI>::st(x);
}

// Single token: a work-group per sequence and head, a thread per V columns and
// every 256 / ceil(dv / V)-th row of the state; the rows' parts of the output
// are added through LDS.  The state is read and written once, in whole lines: 256
// sequences of 16 heads of 128 x 128, 541 MB, take 105 us, 5.2 TB/s.
struct LaStep {
    const void *q, *k, *v;
    const float* g;
    float* state;
    void* out;
    int64_t q_batch, q_head, k_batch, k_head, v_batch, v_head, g_batch, g_head;
    int H, div, dk, dv;
    float scale;
};

template <typename TI, int V>
__global__ __launch_bounds__(256) void la_step_kernel(LaStep p) {
    __shared__ float s_o[256 * V];
    const int h = blockIdx.x, b = blockIdx.y;
    const int cpr = (p.dv + V - 1) / V, rows = 256 / cpr, r0 = threadIdx.x / cpr, c = (threadIdx.x - r0 * cpr) * V;
    const TI* q = static_cast<const TI*>(p.q) + b * p.q_batch + h / p.div * p.q_head;
    const TI* k = static_cast<const TI*>(p.k) + b * p.k_batch + h / p.div * p.k_head;
    const TI* v = static_cast<const TI*>(p.v) + b * p.v_batch + h * p.v_head;
    float* S = p.state + (static_cast<int64_t>(b) * p.H + h) * p.dk * p.dv;
    const float decay = expf(p.g[b * p.g_batch + h * p.g_head]);
    float o[V] = {}, vv[V];
    if (r0 < rows) {
#pragma unroll
        for (int i = 0; i < V; ++i) vv[i] = IO<TI>::ld(v[c + i]);
        for (int r = r0; r < p.dk; r += rows) {
            const float kk = IO<TI>::ld(k[r]), qq = IO<TI>::ld(q[r]);
            Pack<float, V>* at = reinterpret_cast<Pack<float, V>*>(S + r * p.dv + c);
            Pack<float, V> x = *at;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                x.v[i] = fmaf(decay, x.v[i], kk * vv[i]);
                o[i] = fmaf(qq, x.v[i], o[i]);
            }
            *at = x;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) s_o[threadIdx.x * V + i] = o[i];
    __syncthreads();
    for (int j = threadIdx.x; j < p.dv; j += 256) {
        float x = 0.0f;
        for (int r = 0; r < rows; ++r) x += s_o[r * cpr * V + j];
        static_cast<TI*>(p.out)[(static_cast<int64_t>(b) * p.H + h) * p.dv + j] = IO<TI>::st(p.scale * x);
    }
}

int la_check(const mogt_linear_attn_problem* q) {
    if (!q) return set_error(MOGT_E_INVALID, "null problem");
    if (q->io_dtype != MOGT_F32 && q->io_dtype != MOGT_BF16)
        return set_error(MOGT_E_INVALID, "io_dtype %d not supported", q->io_dtype);
    if (q->batch < 0 || q->length < 0 || q->heads < 0 || q->groups < 1 || q->heads % q->groups != 0)
        return set_error(MOGT_E_INVALID, "batch %lld, length %lld, heads %lld in %lld groups", (long long)q->batch,
                         (long long)q->length, (long long)q->heads, (long long)q->groups);
    if (q->key_dim < 1 || q->key_dim > MOGT_LINEAR_ATTN_MAX_DIM || q->value_dim < 1 ||
        q->value_dim > MOGT_LINEAR_ATTN_MAX_DIM)
        return set_error(MOGT_E_INVALID, "key width %lld, value width %lld: 1 to %d expected", (long long)q->key_dim,
                         (long long)q->value_dim, MOGT_LINEAR_ATTN_MAX_DIM);
    if (q->batch > 21845 || q->heads > 65535 || q->length > (1ll << 30))
        return set_error(MOGT_E_INVALID, "batch %lld (at most 21845), heads %lld (65535) or length %lld (2^30) too large",
                         (long long)q->batch, (long long)q->heads, (long long)q->length);
    if (q->lengths && q->lengths_bytes != 4 && q->lengths_bytes != 8)
        return set_error(MOGT_E_INVALID, "lengths of %d bytes: 4 or 8 expected", q->lengths_bytes);
    if (q->batch * q->heads > 0 && q->length > 0 && (!q->q || !q->k || !q->v || !q->log_decay))
        return set_error(MOGT_E_INVALID, "null input pointer");
    return MOGT_OK;
}

int64_t la_segments(const mogt_linear_attn_problem* q) {
    const int64_t n = (q->length + q->segment - 1) / q->segment;
    return n > 0 ? n : 1;
}

// Rows of a segment are addressed by 32-bit byte offsets.
int la_check_rows(const mogt_linear_attn_problem* q) {
    const int64_t es = q->io_dtype == MOGT_BF16 ? 2 : 4, most = 0x7fffffff;
    const int64_t steps = q->segment < q->length ? q->segment : q->length;
    if (q->q_row < 0 || q->k_row < 0 || q->v_row < 0 || q->g_row < 0)
        return set_error(MOGT_E_INVALID, "negative row strides");
    int64_t row = q->heads * (q->key_dim > q->value_dim ? q->key_dim : q->value_dim) * 4 / es;   // of fp32 outputs
    for (const int64_t r : {q->q_row, q->k_row, q->v_row, q->g_row * 4 / es}) row = r > row ? r : row;
    if (row > most / es || row * es * (steps > 0 ? steps : 1) > most - 1024)
        return set_error(MOGT_E_INVALID, "segment of %lld rows %lld elements apart: below 2^31 bytes expected",
                         (long long)steps, (long long)row);
    return MOGT_OK;
}

int la_args(const mogt_linear_attn_problem* q, LaArgs& a) {
    if (const int rc = la_check(q)) return rc;
    const int chunk = q->io_dtype == MOGT_BF16 ? LaChunk<bf16_t>::T : LaChunk<float>::T;
    if (q->segment < chunk || q->segment % chunk != 0 || q->segment > (1 << 30))
        return set_error(MOGT_E_INVALID, "segment of %lld steps: a multiple of %d expected", (long long)q->segment, chunk);
    const int64_t nseg = la_segments(q);
    if (nseg > (1 << 20)) return set_error(MOGT_E_INVALID, "%lld segments: at most 2^20", (long long)nseg);
    if (const int rc = la_check_rows(q)) return rc;
    a.g = q->log_decay;
    a.g_row = q->g_row; a.g_batch = q->g_batch; a.g_head = q->g_head;
    a.lengths = q->lengths;
    a.len64 = q->lengths_bytes == 8;
    a.B = static_cast<int>(q->batch);
    a.L = static_cast<int>(q->length);
    a.H = static_cast<int>(q->heads);
    a.seg = static_cast<int>(q->segment);
    a.nseg = static_cast<int>(nseg);
    a.state = static_cast<int>(q->key_dim * q->value_dim);
    return MOGT_OK;
}

LaRows la_rows(const mogt_linear_attn_problem* q, const void* p, int64_t row, int64_t batch, int64_t head, int div,
               int64_t width) {
    const int64_t es = q->io_dtype == MOGT_BF16 ? 2 : 4;
    LaRows r;
    r.p = p;
    r.row = row; r.batch = batch; r.head = head;
    r.div = div;
    auto whole = [&](int64_t n) {
        return reinterpret_cast<uintptr_t>(p) % n == 0 && row % (n / es) == 0 && batch % (n / es) == 0 && head % (n / es) == 0 &&
               width % (n / es) == 0;
    };
    r.vec = whole(16) ? LA_VECTORS : es == 2 && whole(8) ? LA_HALVES : LA_SINGLE;
    return r;
}

// the roles' tensors
struct LaRoles {
    LaRows q, k, v, go;
};

LaRoles la_roles(const mogt_linear_attn_problem* q, const void* dout) {
    const int div = static_cast<int>(q->heads / q->groups);
    LaRoles r;
    r.q = la_rows(q, q->q, q->q_row, q->q_batch, q->q_head, div, q->key_dim);
    r.k = la_rows(q, q->k, q->k_row, q->k_batch, q->k_head, div, q->key_dim);
    r.v = la_rows(q, q->v, q->v_row, q->v_batch, q->v_head, 1, q->value_dim);
    r.go = la_rows(q, dout, q->heads * q->value_dim, q->length * q->heads * q->value_dim, q->value_dim, 1, q->value_dim);
    return r;
}

// a pass over query, key and value rows; `keys` whether the contraction is the
// keys' (states as they are), else the values' (transposed)
LaPass la_pass(const mogt_linear_attn_problem* q, const LaRows& query, const LaRows& key, const LaRows& value, bool keys) {
    LaPass p{};
    const int dk = static_cast<int>(q->key_dim), dv = static_cast<int>(q->value_dim);
    p.q = query; p.k = key; p.v = value; p.x = value;
    p.dc = keys ? dk : dv;
    p.dn = keys ? dv : dk;
    p.rs = keys ? 1 : dk;
    p.cs = keys ? dk : 1;
    p.user_rs = keys ? dv : 1;
    p.user_cs = keys ? 1 : dv;
    p.qs = p.ps = p.ws = 1.0f;
    return p;
}

void la_launch(const mogt_linear_attn_problem* q, const LaArgs& a, int count, bool out, hipStream_t st) {
    if (q->io_dtype == MOGT_BF16)
        la_launch_passes<bf16_t>(a, count, out, st);
    else
        la_launch_passes<float>(a, count, out, st);
}

void la_carry(const LaArgs& a, int dk, float* states, const float* ctot, const float* init, hipStream_t st) {
    la_carry_kernel<<<dim3((a.state + 255) / 256, a.H, a.B), 256, 0, st>>>(states, ctot, init, a.nseg, dk, a.state / dk);
}

size_t al(size_t x) { return round_up(x, 256); }

size_t la_states_bytes(const mogt_linear_attn_problem* q) {
    return al(static_cast<size_t>(q->batch * q->heads * (la_segments(q) + 1) * q->key_dim * q->value_dim) * 4);
}
size_t la_ctot_bytes(const mogt_linear_attn_problem* q) {
    return al(static_cast<size_t>(q->batch * q->heads * la_segments(q)) * 4);
}

}  // namespace
}  // namespace mogt

using namespace mogt;

extern "C" size_t mogt_linear_attn_workspace_bytes(const mogt_linear_attn_problem* q) {
    LaArgs a{};
    if (la_args(q, a) != MOGT_OK) return 0;
    return a.nseg > 1 ? la_states_bytes(q) + la_ctot_bytes(q) : 0;
}

extern "C" int mogt_linear_attn_fwd(const mogt_linear_attn_problem* q, void* out, float* final_state, float* carries,
                                    void* workspace, size_t workspace_bytes, void* stream) {
    clear_error();
    LaArgs a{};
    if (const int rc = la_args(q, a)) return rc;
    if (q->batch == 0 || q->heads == 0) return MOGT_OK;
    if (q->length > 0 && !out) return set_error(MOGT_E_INVALID, "null output pointer");
    const size_t need = a.nseg > 1 ? (carries ? 0 : la_states_bytes(q)) + la_ctot_bytes(q) : 0;
    if (need > 0 && (!workspace || workspace_bytes < need))
        return set_error(MOGT_E_WORKSPACE, "workspace of %zu bytes expected, got %zu", need, workspace ? workspace_bytes : 0);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const LaRoles r = la_roles(q, nullptr);
    LaPass& p = a.pass[0];
    p = la_pass(q, r.q, r.k, r.v, true);
    p.init = q->initial_state;
    p.ctot = static_cast<float*>(workspace);
    p.states = carries ? carries : need ? reinterpret_cast<float*>(static_cast<char*>(workspace) + la_ctot_bytes(q)) : nullptr;
    p.keep = carries != nullptr;
    p.last = final_state;
    p.out = out;
    if (a.nseg > 1) {
        la_launch(q, a, 1, false, st);
        la_carry(a, static_cast<int>(q->key_dim), p.states, p.ctot, p.init, st);
    }
    p.qs = p.ps = q->scale;
    la_launch(q, a, 1, true, st);
    return check_launch("mogt_linear_attn_fwd");
}

extern "C" size_t mogt_linear_attn_bwd_workspace_bytes(const mogt_linear_attn_problem* q) {
    LaArgs a{};
    if (la_args(q, a) != MOGT_OK) return 0;
    const size_t rows = static_cast<size_t>(q->batch) * q->length * q->heads;
    return la_states_bytes(q) + la_ctot_bytes(q) + 2 * al(rows * 4) +
           al(static_cast<size_t>(q->batch * q->heads * a.nseg) * 8) +
           (q->heads > q->groups ? 2 * al(rows * q->key_dim * 4) : 0);
}

extern "C" int mogt_linear_attn_bwd(const mogt_linear_attn_problem* q, const void* dout, const float* dfinal_state,
                                    const float* carries, const mogt_linear_attn_gradients* g, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    clear_error();
    LaArgs a{};
    if (const int rc = la_args(q, a)) return rc;
    if (!g) return set_error(MOGT_E_INVALID, "null gradients");
    if (q->batch == 0 || q->heads == 0) return MOGT_OK;
    if (!carries || (q->length > 0 && !dout)) return set_error(MOGT_E_INVALID, "null carries or gradient pointer");
    const size_t need = mogt_linear_attn_bwd_workspace_bytes(q);
    if (!workspace || workspace_bytes < need)
        return set_error(MOGT_E_WORKSPACE, "workspace of %zu bytes expected, got %zu", need, workspace ? workspace_bytes : 0);
    hipStream_t st = static_cast<hipStream_t>(stream);
    const size_t rows = static_cast<size_t>(q->batch) * q->length * q->heads;
    char* w = static_cast<char*>(workspace);
    auto take = [&](size_t bytes) {
        char* p = w;
        w += bytes;
        return p;
    };
    float* rstates = reinterpret_cast<float*>(take(la_states_bytes(q)));
    float* rctot = reinterpret_cast<float*>(take(la_ctot_bytes(q)));
    float* dot_q = reinterpret_cast<float*>(take(al(rows * 4)));
    float* dot_k = reinterpret_cast<float*>(take(al(rows * 4)));
    double* part = reinterpret_cast<double*>(take(al(static_cast<size_t>(q->batch * q->heads * a.nseg) * 8)));
    const bool shared = q->heads > q->groups;
    float* share_q = shared ? reinterpret_cast<float*>(take(al(rows * q->key_dim * 4))) : nullptr;
    float* share_k = shared ? reinterpret_cast<float*>(take(al(rows * q->key_dim * 4))) : nullptr;
    const LaRoles r = la_roles(q, dout);
    const bool need_g = g->dlog_decay != nullptr;

    LaPass dv = la_pass(q, r.k, r.q, r.go, true), dk = la_pass(q, r.v, r.go, r.q, false), dq = la_pass(q, r.go, r.v, r.k, false);
    dv.reverse = dk.reverse = 1;
    dv.init = dk.init = dfinal_state;
    dv.states = dk.states = rstates;
    dv.ctot = rctot;
    dv.ws = dk.ws = q->scale;
    dv.keep = 1;
    dv.out = g->dv;
    dk.ps = dv.ps = q->scale;
    dk.x = r.k;
    dk.out = shared && g->dk ? share_k : g->dk;
    dk.out_f32 = shared;
    dq.x = r.q;
    dq.init = q->initial_state;
    dq.states = const_cast<float*>(carries);
    dq.qs = dq.ps = q->scale;
    dq.out = shared && g->dq ? share_q : g->dq;
    dq.out_f32 = shared;
    // formed in any case: a row's gradient does not depend on which others are asked for
    dk.dot = dot_k;
    dq.dot = dot_q;
    if (a.nseg > 1 && (g->dv || g->dk || need_g || g->dinitial_state)) {   // dq takes the forward's states alone
        a.pass[0] = dv;
        la_launch(q, a, 1, false, st);
        la_carry(a, static_cast<int>(q->key_dim), rstates, rctot, dfinal_state, st);
    }
    // every pass that is asked for; the decays' gradient takes the products of
    // dq and dk, it and the initial state's the gradients of the states
    LaPass todo[3];
    int count = 0;
    if (g->dv || need_g || g->dinitial_state) todo[count++] = dv;
    if (g->dk || need_g) todo[count++] = dk;
    if (g->dq || need_g) todo[count++] = dq;
    for (int i = 0; i < count;) {   // those of one kind in one launch
        int m = 0;
        do
            a.pass[m++] = todo[i++];
        while (i < count && la_one_kind(a.pass[0], todo[i]));
        la_launch(q, a, m, true, st);
    }
    if (need_g || g->dinitial_state) {
        LaDecay d{};
        d.states = carries;
        d.rstates = rstates;
        d.dot_q = dot_q;
        d.dot_k = dot_k;
        d.dk = static_cast<int>(q->key_dim);
        d.have_last = dfinal_state != nullptr;
        d.dinit = g->dinitial_state;
        if (need_g) {
            if (q->decay_per_head)
                d.part = part;
            else
                d.dg = g->dlog_decay;
        }
        la_decay_kernel<<<dim3(need_g ? a.nseg : 1, a.H, a.B), 256, 0, st>>>(a, d);
        if (d.part)
            la_decay_sum_kernel<<<a.H, 64, 0, st>>>(part, static_cast<int64_t>(a.B) * a.nseg, g->dlog_decay);
    }
    if (shared) {
        const int share = static_cast<int>(q->heads / q->groups), d = static_cast<int>(q->key_dim);
        const int64_t total = q->batch * q->length * q->groups * q->key_dim;
        if (total > 0 && (g->dq || g->dk)) {
            const dim3 grid = wide_grid((total + 255) / 256, 2);
            if (q->io_dtype == MOGT_BF16)
                la_group_kernel<bf16_t><<<grid, 256, 0, st>>>(share_q, share_k, static_cast<bf16_t*>(g->dq),
                                                              static_cast<bf16_t*>(g->dk), total, d, share);
            else
                la_group_kernel<float><<<grid, 256, 0, st>>>(share_q, share_k, static_cast<float*>(g->dq),
                                                             static_cast<float*>(g->dk), total, d, share);
        }
    }
    return check_launch("mogt_linear_attn_bwd");
}

extern "C" int mogt_linear_attn_step(const mogt_linear_attn_problem* q, float* state, void* out, void* stream) {
    clear_error();
    if (const int rc = la_check(q)) return rc;
    if (q->length != 1) return set_error(MOGT_E_INVALID, "a step takes one token, length is %lld", (long long)q->length);
    if (q->batch == 0 || q->heads == 0) return MOGT_OK;
    if (!state || !out) return set_error(MOGT_E_INVALID, "null state or output pointer");
    LaStep p;
    p.q = q->q; p.k = q->k; p.v = q->v;
    p.g = q->log_decay;
    p.state = state;
    p.out = out;
    p.q_batch = q->q_batch; p.q_head = q->q_head;
    p.k_batch = q->k_batch; p.k_head = q->k_head;
    p.v_batch = q->v_batch; p.v_head = q->v_head;
    p.g_batch = q->g_batch; p.g_head = q->g_head;
    p.H = static_cast<int>(q->heads);
    p.div = static_cast<int>(q->heads / q->groups);
    p.dk = static_cast<int>(q->key_dim);
    p.dv = static_cast<int>(q->value_dim);
    p.scale = q->scale;
    const bool vec = q->value_dim % 4 == 0 && (reinterpret_cast<uintptr_t>(state) & 15) == 0;
    const dim3 grid(p.H, static_cast<unsigned>(q->batch));
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (q->io_dtype == MOGT_BF16) {
        if (vec)
            la_step_kernel<bf16_t, 4><<<grid, 256, 0, st>>>(p);
        else
            la_step_kernel<bf16_t, 1><<<grid, 256, 0, st>>>(p);
    } else {
        if (vec)
            la_step_kernel<float, 4><<<grid, 256, 0, st>>>(p);
        else
            la_step_kernel<float, 1><<<grid, 256, 0, st>>>(p);
    }
    return check_launch("mogt_linear_attn_step");
}
