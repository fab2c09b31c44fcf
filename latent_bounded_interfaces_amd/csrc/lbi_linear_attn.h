// Linear attention with a decay for each head: what its launches are described by, and the kernel over chunks of 64 tokens.
//
// One recurrence, read in the order in which the tokens are taken:
//   X_i = l X_{i-1} + b_i c_i^T,   out_i = a_i X_i,   X [Da, Dc],  l = exp(log_decay)
// The forward pass is (a, b, c) = (q, k, v); of the pullback, with g the cotangent of out,
//   dq = (g, v, k),   dk = (v, g, q) and dv = (k, q, g) from the last token to the first,
// so one kernel does all four.  Over a chunk of C = 64 tokens, with X the state in front of it,
//   out_i = l^(i+1) a_i X + sum over j <= i of l^(i-j) (a_i . b_j) c_j,    X' = l^C X + sum over j of b_j (l^(C-1-j) c_j)^T:
// four products on the matrix cores.  No power of l has a negative exponent.  A chain that starts with the cotangent of a last state, which
// meets the last token undiminished, has one l less in its readouts and one more in its sums (`shift`).
#pragma once

#include "lbi_attn_mfma.h"

namespace lbi {
namespace linear_attn {

using attn_mfma::Mma;
using attn_mfma::u32x2;
using attn_mfma::u32x4;

constexpr int CHUNK = 64;
constexpr int MOST_DIM = 128;

// Strides in elements: sequence, direction, head, token.  `group` neighbouring heads share one of the tensor's.
struct View {
    const void* p;
    int64_t sb, sp, sh, st;
    int group;
};
struct States {  // fp32; strides of sequence, direction, head, row and column
    float* p;
    int64_t sb, sp, sh, sr, sc;
};
struct Chain {
    View a, b, c, out;
    States first, last;            // p NULL: zero, not wanted
    float first_scale, last_scale;  // of what is read and written there
    float scale;                    // of out
    int Da, Dc, reverse, shift;
};
constexpr int MOST_CHAINS = 3;
struct Call {
    Chain chain[MOST_CHAINS];
    const float* log_decay;  // [H]
    const void* lengths;     // [B], NULL: T; 8 bytes each if lengths_wide
    float* segment_states;   // [chains, B, P, H, slots, Da, Dc]
    int chains, lengths_wide;
    int B, P, H, T;
    int segments, segment;  // tokens of one, a multiple of CHUNK
    int halved, half;       // each segment's state comes in two slots, of so many tokens (a multiple of CHUNK) and of the rest
    int joined;             // a launch of its own makes the states behind the segments of what these add; never with halves
    __host__ __device__ int slots() const { return (segments - 1) << halved; }
    __host__ __device__ int slot_at(int s) const { return (s >> halved) * segment + (s & halved) * half; }  // the first token of slot s
};

// l^n x of `log` = n log l: x + x (l^n - 1) near 1, where rounding l^n would add up over many steps, and x l^n from a half on, where what it leaves of x
// would be lost in the difference.
struct Fade {
    float by, kept;
    __device__ __forceinline__ explicit Fade(float log) : by(log > -0.6931472f ? expm1f(log) : expf(log)), kept(log > -0.6931472f ? 1.0f : 0.0f) {}
    __device__ __forceinline__ float of(float x) const { return fmaf(x, by, x * kept); }
};

}  // namespace linear_attn
}  // namespace lbi
