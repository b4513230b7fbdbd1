// Linear attention with a decay for each head, per sequence and head
//   S_t = exp(g_t) S_{t-1} + k_t v_t^T   (dk x dv, fp32),   o_t = scale S_t^T q_t
// and its gradients.  One pass of the form
//   out_t = sum_{s <= t} exp(c_t - c_s) (q_t . k_s) v_s,   c_t = g_1 + ... + g_t,
// serves the forward and, with the roles of the rows exchanged, every gradient:
//   o   query q,  key k,  value v,  forwards
//   dq  query do, key v,  value k,  forwards, on the same states transposed
//   dk  query v,  key do, value q,  backwards in time
//   dv  query k,  key q,  value do, backwards, dk's states transposed
// Backwards the decay between neighbours is the later one's, and none lies
// before the last step.  The gradient of g follows from the rows' products
// (la_decay_kernel).
//
// Chunked form: inside a chunk of LA_T steps, with c from its start and S the
// state before it,
//   out_t = exp(c_t) S^T q_t + sum_{s <= t} exp(c_t - c_s) (q_t . k_s) v_s
//   S'    = exp(c_T) S + sum_s k_s (exp(c_T - c_s) v_s)^T
// all of them matrix products.  Sequences are cut into segments of whole chunks:
// sums (each segment's S' from zero), carry (the states entering the segments,
// in order), out (each segment from its state, chunk by chunk).
#pragma once

#include <type_traits>

#include "common.h"

namespace mogt {

// log2 of the least decay: exp(g) is zero in fp32 far above it, and sums over a
// chunk stay exact to 2^-33 in 64 bits (g = -inf is this and not NaN)
constexpr double LA_LOG2_MIN = -16384.0;
// exp(g) is zero in fp32 at and below this g (2^-150 rounds to zero)
constexpr float LA_G_ZERO = -103.972084f;

template <typename TI> struct LaChunk;
// Steps of a chunk and the contraction of one operand fragment (a lane holds KS /
// 4 consecutive elements).
template <> struct LaChunk<bf16_t> { static constexpr int T = 64, KS = 32; };
template <> struct LaChunk<float> { static constexpr int T = 32, KS = 16; };

// Loads of rows: 16 bytes, 8 bytes (bf16), an element.  Kernels of 2 x 8192 steps of 12
// heads of 100 x 100, bf16, forward: 127 us by halves, 268 by elements (an instruction for
// each, eight for 16 bytes); 128 x 128 by vectors 131.
constexpr int LA_SINGLE = 0, LA_HALVES = 1, LA_VECTORS = 2;

struct LaRows {      // rows of one role: element strides, and the heads that share them
    const void* p;
    int64_t row, batch, head;
    int div;         // head h reads h / div
    int vec;         // LA_VECTORS, LA_HALVES or LA_SINGLE: what address, strides and width are whole in
};

struct LaPass {
    LaRows q, k, v, x;          // x: rows multiplied with the outputs for `dot`
    const float* init;          // state entering the first segment [B, H, dk, dv], or null: zero
    float* states;              // [B, H, nseg + 1, dv, dk]: states entering the segments in pass order, the last after all
    float* ctot;                // [B, H, nseg]: log2 of the segments' decays
    float* last;                // final state [B, H, dk, dv], or null
    void* out;                  // [B, L, H, dn], or null
    float* dot;                 // [B, H, L] sums over the columns of x_t * out_t, or null
    float qs, ps, ws;           // factors of the query's part, the pairs and the writes
    int dc, dn;                 // width of q and k, of v
    int rs, cs;                 // strides of the rows (dc) and columns (dn) of one of `states`
    int user_rs, user_cs;       // ... of `init` and `last`, [dk, dv]
    int reverse, out_f32, keep; // keep: this pass leaves the first and last of `states`
};

struct LaArgs {
    LaPass pass[3];
    const float* g;
    const void* lengths;
    int64_t g_row, g_batch, g_head;
    int B, L, H, seg, nseg, len64;
    int state;                  // dk * dv
};

__device__ __forceinline__ int la_length(const LaArgs& a, int b) {
    if (!a.lengths) return a.L;
    int64_t n = a.len64 ? static_cast<const int64_t*>(a.lengths)[b] : static_cast<const int32_t*>(a.lengths)[b];
    n = n < 0 ? 0 : n > a.L ? a.L : n;
    return __builtin_amdgcn_readfirstlane(static_cast<int>(n));
}

// Padded contraction width of a pass and whether its values are wide, which its kernel
// is built for; the waves of a SIMD that the kernel's registers are held to, by its tiles
// of 16 value columns a wave and its waves.
inline int la_width(int dc) { return dc <= 32 ? 32 : dc <= 64 ? 64 : 128; }
inline bool la_wide(int dn) { return dn > 64; }
constexpr int la_waves_per_simd(int width, int tiles, int waves) { return waves == 8 ? 4 : tiles == 2 || width > 64 ? 2 : 3; }

inline bool la_one_kind(const LaPass& a, const LaPass& b) {
    return la_width(a.dc) == la_width(b.dc) && la_wide(a.dn) == la_wide(b.dn) && !a.dot == !b.dot && a.out_f32 == b.out_f32;
}

}  // namespace mogt
