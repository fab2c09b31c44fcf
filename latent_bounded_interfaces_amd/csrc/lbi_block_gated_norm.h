// Launches of lbi_block_gated_norm_kernel.h: what they are described by, a source for each type.
#pragma once

#include "lbi_common.h"

namespace lbi {
namespace block_norm {

// What a workgroup leaves of the three sums over rows, [slabs, D] each.
struct Partials { float *post, *pre, *gate; };

// Gates, rows of one, and the slabs that they are cut into: as many in all as fill the chip a few times, none across two gates.
struct Plan {
    int64_t gates, per_gate;
    int slabs_per_gate, slab;
    int64_t slabs() const { return gates * slabs_per_gate; }
};
struct Forward {
    const void *branch, *residual, *gate, *post_weight, *weight;
    void *normed, *residual_out;
    int64_t rows, D, per_gate;
    float eps, residual_scale;
    int post_wide, wide;
};
struct Pullback {
    const void *g_normed, *branch, *residual_out, *g_residual_out, *gate, *post_weight, *weight;
    void *g_branch, *g_residual, *g_gate;  // g_gate: of a gate for each row
    Partials partials;
    Plan plan;
    int64_t D;
    float eps, residual_scale;
    int each, post_wide, wide;
};
// same: the residual stream is in the branch's type, fp32 otherwise
int forward_f32(const Forward& f, hipStream_t stream);
int forward_f16(const Forward& f, bool same, hipStream_t stream);
int forward_bf16(const Forward& f, bool same, hipStream_t stream);
int pullback_f32(const Pullback& f, hipStream_t stream);
int pullback_f16(const Pullback& f, bool same, hipStream_t stream);
int pullback_bf16(const Pullback& f, bool same, hipStream_t stream);

}  // namespace block_norm
}  // namespace lbi
