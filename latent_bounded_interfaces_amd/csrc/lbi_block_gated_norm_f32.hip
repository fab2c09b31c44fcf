// The norms behind and before a block, fp32 branches.
#include "lbi_block_gated_norm_kernel.h"

namespace lbi {
namespace block_norm {

int forward_f32(const Forward& f, hipStream_t stream) { return forward<float, float>(f, stream); }
int pullback_f32(const Pullback& f, hipStream_t stream) { return pullback<float, float>(f, stream); }

}  // namespace block_norm
}  // namespace lbi
